"""The product of int8 rows and weights (mla_m4_mul_i8) against exact integer sums."""
import ctypes
import math

import pytest
import torch

import aubier_amd as A

from rows_util import half_step, near

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


def ints(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)


def make(dev, rows, n, k, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 3 * n + 7 * k)
    return (ints(g, n, k).to(dev), torch.exp(torch.randn(n, generator=g)).to(dev) / 50, ints(g, rows, k).to(dev),
            torch.exp(torch.randn(rows, generator=g)).to(dev) / 50)


def want64(w, ws, x, xs):
    """Sums of whole numbers below 2^53: exact in any order."""
    return torch.matmul(x.double(), w.double().t().contiguous()) * xs.double()[:, None] * ws.double()


def check(a, got, what=""):
    """The sum rounded to f32 and two products, 2^-24 each; then the stored type's rounding."""
    rel, small = half_step(got.dtype)
    want = want64(*a)
    if got.dtype == F16:                                # past the middle of 65504, the largest, and the next step is an infinity
        want = torch.where(want.abs() >= 65520, torch.copysign(torch.full_like(want, math.inf), want), want)
    near(got, want, 3.01 * 2.0 ** -24 + (rel * (1 + 2.0 ** -10) if got.dtype == F16 else 0), small, what)


@pytest.mark.parametrize("rows", [1, 2, 4, 5, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 255, 257, 513])
@pytest.mark.parametrize("n,k", [(1, 16), (3, 48), (16, 64), (17, 80), (100, 128), (255, 272), (257, 1040), (576, 7168), (1030, 1536)])
def test_sizes(dev, rows, n, k):
    a = make(dev, rows, n, k)
    for dtype in (F32, F16):
        check(a, A.ggml_m4_mul_i8(*a, dtype=dtype), dtype)


@pytest.mark.parametrize("k", [16, 32, 48, 64, 80, 112, 128, 144, 240, 256, 272, 384, 400, 512, 528, 1008, 1024, 1040, 2048, 4112, 16384])
@pytest.mark.parametrize("rows,n", [(1, 40), (40, 40), (300, 520)])
def test_depths(dev, k, rows, n):
    a = make(dev, rows, n, k, 1)
    check(a, A.ggml_m4_mul_i8(*a), k)


@pytest.mark.parametrize("rows,n,k", [(2000, 4096, 512), (777, 6200, 2064), (8191, 129, 144), (64, 24576, 1536), (5000, 2112, 160), (300, 2, 7168)])
def test_large(dev, rows, n, k):
    a = make(dev, rows, n, k, 2)
    for dtype in (F32, F16):
        check(a, A.ggml_m4_mul_i8(*a, dtype=dtype), dtype)


@pytest.mark.parametrize("rows,n,k", [
    (1, 24577, 1552), (31, 24570, 1536), (32, 576, 7184), (48, 2112, 7168), (64, 2100, 7152), (100, 570, 7168), (64, 7168, 4096), (61, 7150, 4112),
    (128, 7168, 4096), (125, 7100, 4080), (60, 24576, 1536), (64, 7168, 16384), (300, 7168, 4096), (290, 7101, 4112), (130, 7168, 16384),
    (200, 24576, 1536), (1000, 7168, 4096), (1030, 4100, 4112), (3000, 4096, 528), (4001, 2112, 1040),
    (300, 24576, 1536), (389, 24570, 1552), (1401, 7100, 2064), (515, 24007, 528)])
def test_forms(dev, rows, n, k):
    """Shapes that the forms of the product share out among them, with and without a workspace, into rows at odd places."""
    a = make(dev, rows, n, k, 3)
    got = A.ggml_m4_mul_i8(*a)
    check(a, got)
    need = A.mul_i8_workspace_bytes(a[0], a[2])
    assert need <= 1 << 24
    work = torch.full((need + 16,), 99, dtype=torch.uint8, device=dev)
    buf = torch.full((rows, n + 3), 7.0, device=dev)
    assert torch.equal(A.ggml_m4_mul_i8(*a, out=buf[:, 1:n + 1], workspace=work[:max(need, 16)]), got)
    assert (buf[:, 0] == 7).all() and (buf[:, n + 1:] == 7).all() and (work[max(need, 16):] == 99).all()
    check(a, A.ggml_m4_mul_i8(*a, dtype=F16))


def test_without_a_workspace(dev):
    """The C entry point given none: the same bits; one that is too small is refused."""
    a = make(dev, 64, 576, 7168)
    want = A.ggml_m4_mul_i8(*a)
    need = A.mul_i8_workspace_bytes(a[0], a[2])
    assert need > 0
    with pytest.raises(A.MlaM4Error) as e:
        A.ggml_m4_mul_i8(*a, workspace=torch.empty(need - 1, dtype=torch.uint8, device=dev))
    assert e.value.status == -5
    out = torch.empty_like(want)
    v = [A.view(t) for t in (*a, out)]
    assert A.load_library().mla_m4_mul_i8(*(ctypes.byref(t) for t in v), None, 0, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_the_longest_sums(dev, rows):
    """131,056 products of -128 by -128 and of -128 by 127."""
    k = 131056
    w = torch.full((70, k), -128, dtype=torch.int8, device=dev)
    x = torch.full((rows, k), -128, dtype=torch.int8, device=dev)
    w[1::2] = 127
    one = lambda m: torch.ones(m, device=dev)  # noqa: E731
    check((w, one(70), x, one(rows)), A.ggml_m4_mul_i8(w, one(70), x, one(rows)))


@pytest.mark.parametrize("rows", [1, 3, 37, 150, 400])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_views(dev, rows, dtype):
    """Operands and result inside wider tensors; nothing beside the result is written."""
    g = torch.Generator().manual_seed(rows)
    n, k = 333, 208
    wb, xb = ints(g, n, k + 112).to(dev), ints(g, rows, k + 48).to(dev)
    _, ws, _, xs = make(dev, rows, n, k)
    for pad in (1, 4, 8, 16):
        buf = torch.full((rows, n + 3 * pad), 7.0, dtype=dtype, device=dev)
        out = buf[:, pad:pad + n]
        a = (wb[:, 32:32 + k], ws, xb[:, 16:16 + k], xs)
        assert A.ggml_m4_mul_i8(*a, out=out) is out
        check(a, out)
        assert (buf[:, :pad] == 7).all() and (buf[:, pad + n:] == 7).all()


def test_scales(dev):
    """NaN and infinite scales reach their row or channel and no other; tiny and huge ones."""
    for rows in (3, 40, 300):
        w, ws, x, xs = make(dev, rows, 100, 256)
        xs[1], ws[7] = math.nan, math.inf
        got = A.ggml_m4_mul_i8(w, ws, x, xs)
        assert torch.isnan(got[1]).all() and not torch.isnan(got[0, :7]).any() and not torch.isfinite(got[:, 7]).any()
        there = torch.ones(100, dtype=torch.bool, device=dev)
        there[7] = False
        keep = torch.arange(rows, device=dev) != 1
        check((w[there], ws[there], x[keep], xs[keep]), got[keep][:, there])
        xs[:], ws[:] = 2.0 ** -60, 2.0 ** 60
        assert torch.equal(A.ggml_m4_mul_i8(w, ws, x, xs).double(), want64(w, ws, x, xs).float().double())
        xs[:], ws[:] = 2.0 ** -100, 2.0 ** -40          # subnormal results
        near(A.ggml_m4_mul_i8(w, ws, x, xs), want64(w, ws, x, xs), 3.01 * 2.0 ** -24, 2.0 ** -150)
        xs[:], ws[:] = 1.0, 1.0                         # past f16's range
        want = want64(w, ws, x, xs).float().half()
        assert torch.equal(A.ggml_m4_mul_i8(w, ws, x, xs, dtype=F16), want)


def test_columns_stand_alone(dev):
    """Each result is its row's and its channel's alone: the same bits whatever else is in the call."""
    w, ws, x, xs = make(dev, 400, 700, 528)
    all_ = A.ggml_m4_mul_i8(w, ws, x, xs)
    for rows in ((0, 1), (5, 7), (0, 64), (100, 229), (390, 400)):
        for cols in ((0, 1), (3, 19), (128, 300), (699, 700)):
            r, c = slice(*rows), slice(*cols)
            assert torch.equal(A.ggml_m4_mul_i8(w[c], ws[c], x[r], xs[r]), all_[r, c]), (rows, cols)


def test_streams_and_graphs(dev):
    """Two streams at once; a captured call replayed with the program's own work between the replays."""
    a, b = make(dev, 70, 1000, 1040), make(dev, 300, 900, 2048)
    ya, yb = A.ggml_m4_mul_i8(*a), A.ggml_m4_mul_i8(*b)
    s = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for st, args, out in zip(s, (a, b), got):
            with torch.cuda.stream(st):
                out.append(A.ggml_m4_mul_i8(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(y, ya) for y in got[0]) and all(torch.equal(y, yb) for y in got[1])
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(ya)
    with torch.cuda.graph(graph, stream=s[0]):
        A.ggml_m4_mul_i8(*a, out=out)
    for i in range(4):
        a[3].mul_(0.5)
        want = A.ggml_m4_mul_i8(*a)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
