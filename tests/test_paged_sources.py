"""Properties of the paged cache's kernels that only a reader sees: a run would show their loss by chance."""

import os
import re


CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "submission_folder_b200", "csrc")


def _source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_a_warp_clears_only_its_own_entries():
    """Before the CTA's first barrier an entry of the merge list is written by one warp alone, its owner."""
    text = _source("ckv_attend.cu")
    body = text[text.index("k_attend(const AttArgs p)"):]
    body = body[:body.index("__syncthreads()")]
    written = re.findall(r"s_entry\[((?!2 \* kWarps\])[^\]]*)\]", body)
    assert len(written) == 2 and all(w.startswith("2 * wid +") for w in written)
    assert body.index("__syncwarp()") > body.index("s_entry[2 * wid + lane].used = 0")


def test_kernels_placed_early_use_plain_loads():
    """A kernel that is resident while its predecessor runs reads through loads that the wait orders."""
    for name in ("ckv_tables.cu", "ckv_rotary.cu", "ckv_cache.cu", "ckv_attend.cu"):
        text = _source(name)
        for other in ("__ldg", "__ldcg", "__ldca", "__ldcs", "ld.global.nc", "__restrict__"):
            assert other not in text, (name, other)
        assert text.count("__global__") <= text.count("after_previous();") + text.count("turns_of(a, t0, nt, rot_cs);"), name
