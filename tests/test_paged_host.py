"""Host-side parts of the paged cache's kernels, compiled with the host compiler: arithmetic at the
ends of its range and the launch helpers, against fakes of the CUDA calls."""

import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "submission_folder_b200", "csrc")


def _run(tmp_path, source):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(source)
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-pthread", "-I", CSRC,
                    "-I", os.path.join(cuda, "include"), str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True)


def test_shares_of_a_request_cover_its_rows(tmp_path):
    """Every row of a request belongs to one part and no part steps outside, for requests that ask for
    nearly 2^31 tokens as for small ones; a refused request has only the rows of the step."""
    r = _run(tmp_path, r'''
#include "ckv_share.h"
#include <stdio.h>
#include <initializer_list>
int main() {
  const int32_t top = 2147483647, asks[] = {0, 1, 5, 127, 128, 129, 4096, 1 << 20, top - 128, top - 64, top - 1, top};
  for (int32_t ask : asks)
    for (int32_t granted : {0, 1})
      for (int32_t t0 : {0, 7, 5000, top})
        for (int32_t total : {0, 8, 5000, 70000, top})
          for (int32_t parts : {1, 2, 3, 63, 64}) {
            const int32_t give = granted ? ask : 0;
            uint32_t at = 0;
            const uint32_t rows = total > t0 ? total - t0 : 0, want = give ? give : (uint32_t)ask < rows ? ask : rows;
            for (int32_t part = 0; part < parts; ++part) {
              const ckv::Share s = ckv::share_of(ask, give, t0, total, part, parts);
              if (s.from != at || s.to < s.from || (uint64_t)s.to + 128 > 0xffffffffull) return printf("%d %d\n", ask, part), 1;
              at = s.to;
            }
            if (at != want) return printf("%d %d %d %d: %u\n", ask, t0, total, parts, at), 1;
          }
  return 0;
}
''')
    assert r.returncode == 0, r.stdout + r.stderr


def test_shared_memory_is_opted_in_on_each_device(tmp_path):
    """The limit belongs to a (kernel, device) pair: one device's opt-in says nothing of another's."""
    r = _run(tmp_path, r'''
#include "ckv_smem.h"
#include <stdio.h>
#include <map>
static int now = 0, calls = 0, broken = 0;
static std::map<std::pair<int, const void*>, int> limit;
extern "C" cudaError_t cudaGetDevice(int* d) { *d = now; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int bytes) {
  if (broken || a != cudaFuncAttributeMaxDynamicSharedMemorySize) return cudaErrorInvalidValue;
  ++calls;
  limit[{now, f}] = bytes;
  return cudaSuccess;
}
int main() {
  static int f, g;
  for (int round = 0; round < 2; ++round)
    for (now = 0; now < 9; ++now) {
      if (ckv::ensure_dynamic_smem(&f, 196608) != cudaSuccess || (limit[{now, &f}] != 196608)) return printf("device %d\n", now), 1;
      if (ckv::ensure_dynamic_smem(&f, 1000) != cudaSuccess || (limit[{now, &f}] != 196608)) return printf("lowered\n"), 1;
    }
  if (calls != 9) return printf("%d calls\n", calls), 1;
  broken = 1;
  now = 3;
  if (ckv::ensure_dynamic_smem(&g, 1000) != cudaErrorInvalidValue) return printf("hidden error\n"), 1;
  broken = 0;
  if (ckv::ensure_dynamic_smem(&g, 1000) != cudaSuccess || calls != 10) return printf("kept error\n"), 1;
  return 0;
}
''')
    assert r.returncode == 0, r.stdout + r.stderr
