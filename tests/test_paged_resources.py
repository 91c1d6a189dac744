"""Register, scratch and LDS budgets of the paged-batch kernels (as test_kernel_resources.py for the others).  The
attention kernels use every register of a wavefront that has a SIMD to itself; what does not fit is a few words of the
place on the line, kept through a piece -- none in, or ahead of, the tile loops, where a reload waits for the DMA."""
import re

import pytest

from aubier_amd import build as B

from test_kernel_resources import LDS_MAX, pytestmark, resources  # noqa: F401

BUDGET = {                                                   # (VGPR spills, scratch bytes per lane)
    "kqkv_paged.hip": {"kqkv_paged_kernel": (8, 48), "kqkv_paged_merge_kernel": (0, 0), "kqkv_paged_merge_few_kernel": (0, 0)},
    "paged_ops.hip": {"pages_kernel": (0, 0), "kvrows_kernel": (0, 0)},
}


@pytest.mark.parametrize("src", sorted(BUDGET))
def test_budgets(src):
    seen = set()
    for name, r in resources(B.CSRC / src).items():
        print(name[:110], r)
        assert r.get("lds", 0) <= LDS_MAX, name
        for frag, (spills, scratch) in BUDGET[src].items():
            if re.search(r"\d" + frag + r"[IE]", name):
                seen.add(frag)
                assert r["vspill"] <= spills and r["scratch"] <= scratch, (name, r)
    assert seen == set(BUDGET[src])
