"""Build ``libckv.so`` and ``_ckv_torch.so`` in-tree for sm_100a (``python -m submission_folder_b200.build``)."""

from __future__ import annotations

import importlib.util
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")


def torch_headers() -> bool:
    """Whether the headers that ``_ckv_torch.so`` is compiled against are there."""
    if not os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")):
        return False
    spec = importlib.util.find_spec("torch")
    return spec is not None and os.path.exists(os.path.join(os.path.dirname(spec.origin), "include", "torch", "csrc", "api",
                                                            "include", "torch", "types.h"))


def _make(target: str, verbose: bool) -> None:
    jobs = str(max(1, min(8, os.cpu_count() or 1)))
    cmd = ["make", "-C", CSRC, "-j", jobs, f"PYTHON={sys.executable}", target]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose or res.returncode != 0:
        sys.stdout.write(res.stdout)
        sys.stderr.write(res.stderr)
    if res.returncode != 0:
        raise RuntimeError(f"building {os.path.basename(target)} failed")


def build(verbose: bool = False) -> str:
    """Run the csrc Makefile (nvcc -gencode arch=compute_100a,code=sm_100a); returns the library's path.
    ``_ckv_torch.so``, which only the paged cache's calls on tensors need, is left out with a message
    where the headers of Python or torch are missing."""
    _make("../libckv.so", verbose)
    if torch_headers():
        _make("torch", verbose)
    else:
        sys.stderr.write("_ckv_torch.so was not built: the headers of Python or torch are missing\n")
    return os.path.join(HERE, "libckv.so")


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))
