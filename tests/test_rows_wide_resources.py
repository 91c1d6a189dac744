"""Registers of the norms of rows over 12,288 values, as they are built: up to 16,384 values without a spill, wider ones with at most
25 registers of one (with 200 a row of 24,576 took 55 us instead of 20); and one kernel of each for few rows and for many."""
import re

from aubier_amd import build as B

from test_kernel_resources import pytestmark, resources  # noqa: F401

BUDGET = {4: (0, 0), 8: (25, 104)}          # groups of four values a thread -> (VGPR spills, scratch bytes per lane)


def test_wide_norms():
    seen = set()
    for name, r in resources(B.CSRC / "row_ops.hip").items():
        m = re.search(r"norm_kernelILi1024ELi([48])ELb([01])ELi(\d)ELb([01])E", name)
        if m is None:
            continue
        groups, x, res, one = (int(g) for g in m.groups())
        spills, scratch = BUDGET[groups]
        assert r["vspill"] <= spills and r["scratch"] <= scratch, (name, r)
        assert (groups, x, res) not in seen, name
        seen.add((groups, x, res))
    assert seen == {(g, x, res) for g in BUDGET for x in (0, 1) for res in range(4)}
