"""The int8 rows of a norm next to the borders between two integers, where v = r * pre takes 48 bits and 127 v more than a double
holds: every integer against exact fractions."""
from fractions import Fraction

import pytest
import torch

import aubier_amd as A

pytestmark = pytest.mark.gpu
F32, I8 = torch.float32, torch.int8

# (r, pre) of a row's largest value, then of one whose 127 v / top lies below a border by less than 3e-14: products of the
# doubles round both sides of 127 v < (q + 1/2) top to the same number
BELOW = [
    (14890795, 10692262, 16314516, 7569127), (14188498, 12261905, 8720609, 12645608), (14074134, 12204187, 7952041, 13691281),
    (14070533, 11266195, 9626899, 16401675), (15089474, 14082210, 11908501, 16087538), (14598439, 15142689, 13425164, 14326773),
    (11319778, 15053266, 9820875, 15096526), (9223131, 11887717, 5180255, 16582311), (10942725, 10656737, 5895859, 12537034),
    (12933303, 11914640, 5142349, 15926813), (13737795, 13615753, 12298787, 15148974), (15559308, 16241523, 11562662, 13853240),
]
# the largest value 254 * 2^30, and values on the borders themselves: half away from zero
TIES = (254 << 10, 1 << 20, [(2 * q + 1) << 10 for q in range(0, 127, 9)])


def want_i8(r, pre):
    """Exact integers of rows r * pre."""
    out = []
    for row in r.double().tolist():
        v = [Fraction(a) * Fraction(b) for a, b in zip(row, pre.double().tolist())]
        top = max(abs(x) for x in v)
        out.append([int(abs(x) * 127 / top + Fraction(1, 2)) * (1 if x >= 0 else -1) for x in v])
    return torch.tensor(out, dtype=I8)


def check(dev, r, pre, n):
    wide = torch.zeros((r.shape[0], n))
    wide[:, n - r.shape[1]:] = r
    w = torch.zeros(n)
    w[n - r.shape[1]:] = pre
    want = want_i8(r, pre)
    zeros = torch.zeros_like(wide)
    for kw in ({}, dict(res=zeros.to(dev)), dict(res=zeros.half().to(dev), res_out=torch.empty_like(wide, device=dev))):
        _, h, s = A.ggml_m4_norm(wide.to(dev), w.to(dev), 0.0, dtype=I8, **kw)
        got = h.cpu()
        assert (got[:, :n - r.shape[1]] == 0).all() and torch.isfinite(s).all()
        assert torch.equal(got[:, n - r.shape[1]:], want), (got[:, n - r.shape[1]:], want)


@pytest.mark.parametrize("n", [8, 1536, 7168, 16384, 32768])
def test_below_a_border(dev, n):
    """From the plain range of f32 and from near its ends, where the quotient is taken in 64 bits."""
    for ta, tb, a, b in BELOW:
        r = torch.tensor([ta, a, -a, a + 1, a - 1], dtype=F32)
        pre = torch.tensor([tb, b, b, b, b], dtype=F32)
        rows = torch.stack([r, -r, r * 2.0 ** 40, r * 2.0 ** -30])
        for e in (0, 70, -120):
            check(dev, torch.nn.functional.pad(rows, (0, 3)), torch.nn.functional.pad(pre * 2.0 ** e, (0, 3)), n)


@pytest.mark.parametrize("n", [16, 4096])
def test_on_a_border(dev, n):
    ta, tb, a = TIES
    r, pre = torch.tensor([ta, *a], dtype=F32), torch.tensor([tb] * (1 + len(a)), dtype=F32)
    assert len(a) == 15
    check(dev, torch.stack([r, -r, r * 2.0 ** 90, r * 2.0 ** -130]), pre, n)


def test_many_rows(dev):
    """Rows one after another in a workgroup."""
    ta, tb, a, b = BELOW[0]
    r = torch.tensor([ta, a, -a, a - 1], dtype=F32).expand(3000, 4)
    pre = torch.tensor([tb, b, b, b], dtype=F32)
    _, h, _ = A.ggml_m4_norm(r.contiguous().to(dev), pre.to(dev), 0.0, dtype=I8)
    assert (h.cpu() == want_i8(r[:1], pre)).all()
