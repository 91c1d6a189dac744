"""Register, scratch and LDS budgets of the kernels around a batch's attention (as test_kernel_resources.py for the others)."""
import re

import pytest

from aubier_amd import build as B

from test_kernel_resources import LDS_MAX, pytestmark, resources  # noqa: F401

# kernel -> (VGPR spills, scratch bytes per lane).  Norms of rows over 12,288 values hold more than a workgroup's registers.
BUDGET = {
    "mul_i8.hip": {"direct_kernel": (0, 0), "split_kernel": (0, 0), "sum_kernel": (0, 0), "tile_kernel": (0, 0)},
    "row_ops.hip": {r"norm_kernelILi(?!1024ELi[48])\d+": (0, 0), "norm_kernelILi1024ELi4": (32, 128), "norm_kernelILi1024ELi8": (200, 800), "qrope_kernel": (0, 0)},
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
