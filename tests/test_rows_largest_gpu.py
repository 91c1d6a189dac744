"""The operators around a batch's attention at the ends of what they take: rows that lie more than 4 GiB apart, the most rows and
channels."""
import pytest
import torch

import aubier_amd as A

from rows_util import EPS, YARN, int8_64, near, norm64, rope64
from test_mul_i8_gpu import check, make

pytestmark = pytest.mark.gpu
F32, F16, I8 = torch.float32, torch.float16, torch.int8
GIB = 1 << 30


def far(dev, shape, stride, dtype, fill=None):
    """A tensor [rows, ...] whose rows lie `stride` bytes apart in memory that is not touched otherwise."""
    es = torch.empty((), dtype=dtype).element_size()
    inner = 1
    for s in shape[1:]:
        inner *= s
    buf = torch.empty((shape[0] - 1) * stride // es + inner, dtype=dtype, device=dev)
    t = buf.as_strided(shape, (stride // es,) + tuple(torch.empty(shape[1:]).stride()))
    return t if fill is None else t.copy_(fill)


def test_norm_far_rows(dev):
    g = torch.Generator().manual_seed(1)
    x, res, pre = torch.randn((6, 1024), generator=g), torch.randn((6, 1024), generator=g).half(), torch.randn(1024, generator=g).to(dev)
    fx, fr = far(dev, (6, 1024), GIB, F32, x), far(dev, (6, 1024), GIB + 64, F16, res)
    out, ro = far(dev, (6, 1024), GIB + 16, F32), far(dev, (6, 1024), GIB - 16, F32)
    want = A.ggml_m4_norm(x.to(dev), pre, EPS, res=res.to(dev), res_out=torch.empty((6, 1024), device=dev))
    got = A.ggml_m4_norm(fx, pre, EPS, res=fr, out=out, res_out=ro)
    assert all(torch.equal(a, b) for a, b in zip(got[:2], want[:2]))
    near(got[1], norm64(ro.contiguous(), pre, EPS)[2], 2.0 ** -24 * (1 + 2.0 ** -10) + 2.0 ** -24)
    q, s = A.ggml_m4_rows_i8(fx, out=far(dev, (6, 1024), GIB + 4, I8))
    assert torch.equal(q, int8_64(x.double())[0].to(dev))
    pieces = far(dev, (6, 128, 8), GIB, F32, x.view(6, 128, 8)).permute(1, 0, 2)        # pieces, not rows, far apart
    q, s = A.ggml_m4_rows_i8(pieces)
    assert torch.equal(q, int8_64(x.view(6, 128, 8).permute(1, 0, 2).flatten(1).double())[0].to(dev))


@pytest.mark.parametrize("rows,n,k", [(1200, 70, 144), (20, 1200, 144), (1200, 1200, 48)])
def test_mul_far_rows(dev, rows, n, k):
    """Operand rows 4 MiB apart, more than 4 GiB in all, and the result's rows 5 MiB apart."""
    a = make(dev, rows, n, k, 5)
    w = far(dev, (n, k), 4 << 20, I8, a[0]) if n > 1000 else a[0]
    x = far(dev, (rows, k), 4 << 20, I8, a[2]) if rows > 1000 else a[2]
    out = far(dev, (rows, n), 5 << 20, F32)
    assert torch.equal(A.ggml_m4_mul_i8(w, a[1], x, a[3], out=out), A.ggml_m4_mul_i8(*a))
    check(a, out.contiguous())


def test_qrope_far_rows(dev):
    g = torch.Generator().manual_seed(2)
    q, pos = torch.randn((6, 5, 64), generator=g).to(dev), torch.arange(6, dtype=torch.int32, device=dev) * 1000
    rope = A.rope_params(n_dims=64, **YARN)
    want = A.ggml_m4_qrope(q, pos, rope)
    got = A.ggml_m4_qrope(far(dev, (6, 5, 64), GIB, F32, q), pos, rope, out=far(dev, (6, 5, 64), GIB + 256, F32))
    assert torch.equal(got, want)


def test_most_rows(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    x, pre = torch.randn((1 << 24, 4), device=dev, generator=g), torch.ones(4, device=dev)
    h = A.ggml_m4_norm(x, pre, EPS, dtype=I8)[1:]
    plain = A.ggml_m4_rows_i8(x)
    for at in (0, 1 << 23, (1 << 24) - 100000):
        part = slice(at, at + 100000)
        want = int8_64(x[part].double())
        assert torch.equal(plain[0][part], want[0]) and torch.equal(h[0][part], want[0])
        near(plain[1][part], want[1], 2.0 ** -24, 2.0 ** -150)
        near(h[1][part], norm64(x[part], pre, EPS)[3][1], 2.0 ** -23)
    q, pos = torch.randn((1 << 22, 1, 32), device=dev, generator=g), torch.arange(1 << 22, dtype=torch.int32, device=dev)
    got = A.ggml_m4_qrope(q, pos, A.rope_params(n_dims=32, **YARN))
    for at in (0, (1 << 22) - 1000):
        part = slice(at, at + 1000)
        pair = (q[part][..., 0::2].abs() + q[part][..., 1::2].abs()).double().repeat_interleave(2, -1) * 1.6
        assert ((got[part].double() - rope64(q[part], pos[part], YARN)).abs() <= pair * (3.2 + 8) * 2.0 ** -24).all()


@pytest.mark.parametrize("rows,n", [(1 << 22, 3), (5, 1 << 22), (300, 1 << 20)])
def test_most_rows_and_channels_of_a_product(dev, rows, n):
    a = make(dev, rows, n, 32, 6)
    got = A.ggml_m4_mul_i8(*a, dtype=F16)
    for r0, c0 in ((0, 0), (max(0, rows - 5000), max(0, n - 5000))):
        part = (a[0][c0:c0 + 5000], a[1][c0:c0 + 5000], a[2][r0:r0 + 5000], a[3][r0:r0 + 5000])
        check(part, got[r0:r0 + 5000, c0:c0 + 5000], F16)
