"""Norms with gate and residual, int8 rows and q's rope (mla_m4_norm, mla_m4_rows_i8, mla_m4_qrope) against their
definitions in 64 bits."""
from fractions import Fraction

import math

import pytest
import torch

import aubier_amd as A

from rows_util import EPS, PLAIN, YARN, half_step, int8_64, near, norm64, rope64

pytestmark = pytest.mark.gpu
F32, F16, I8 = torch.float32, torch.float16, torch.int8


def inputs(dev, rows, n, x=F32, res=F32, gate="channel", post=True, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * rows + n)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    spread = torch.exp(1.5 * r(rows, 1))
    return dict(x=(r(rows, n) * spread).to(x).to(dev), pre=(1 + 0.3 * r(n)).to(dev), post=(0.5 + 0.2 * r(n)).to(dev) if post else None,
                gate={"none": None, "channel": r(n), "row": r(rows, 1), "full": r(rows, n), "one": r(1)}[gate].to(dev) if gate != "none" else None,
                res=(r(rows, n) * spread).to(res).to(dev) if res is not None else None)


def check_norm(i, scale=1.0, dtype=F32, got=None, **kw):
    r, h, s = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], scale=scale, dtype=dtype, **kw) if got is None else got
    stored = kw["res_out"].dtype if kw.get("res_out") is not None else i["res"].dtype if i["res"] is not None else None
    rr, exact, hh, (q, step) = norm64(i["x"], i["pre"], EPS, i["post"], i["gate"], i["res"], scale, stored)
    if stored is not None:
        rel, small = half_step(stored)
        near(r, exact, rel * (1 + 2 ** -10) + 2.0 ** -24, small, "r")          # f16 by way of f32: 2^-24 more
        # the rest is of r as it is stored
        rr, _, hh, (q, step) = norm64(r, i["pre"], EPS, store=stored)
    else:
        assert r is None
    if dtype is None:
        assert h is None and s is None
    elif dtype == I8:
        if stored is not None:
            assert torch.equal(h, q), int((h != q).sum())
        else:                                                                 # r is in the kernel alone: at most a step of f32 off
            assert float((h.int() - q.int()).abs().max()) <= 1 and float((h != q).double().mean()) < 1e-4
        near(s, step, 2.0 ** -24 + (0 if stored is not None else 2.0 ** -22), 2.0 ** -150, "scale")
    else:
        # one rounding; of an r that is not stored its own 2^-24 before (twice: the reference may round the other way)
        rel, small = half_step(dtype)
        near(h, hh, rel * (1 + 2 ** -10) + 2.0 ** -24 + (0 if stored is not None else 2.0 ** -23), small, "h")
    return r, h, s


@pytest.mark.parametrize("n", [4, 8, 60, 252, 256, 260, 1020, 1024, 1028, 4092, 4096, 4100, 7168, 8192, 8196, 16384, 20000, 32764, 32768])
@pytest.mark.parametrize("rows", [1, 3, 65])
@pytest.mark.parametrize("dtype", [F32, F16, I8])
def test_norm_sizes(dev, n, rows, dtype):
    check_norm(inputs(dev, rows, n), dtype=dtype, scale=0.75)


@pytest.mark.parametrize("x", [F32, F16])
@pytest.mark.parametrize("res", [None, F32, F16])
@pytest.mark.parametrize("gate", ["none", "channel", "row", "full", "one"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, I8, None])
def test_norm_parts(dev, x, res, gate, post, dtype):
    if res is None and dtype is None:
        return
    check_norm(inputs(dev, 37, 1536, x, res, gate, post), dtype=dtype, scale=-0.5)


@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("rows", [1, 255, 256, 257, 1024, 3001])
def test_norm_rows(dev, pre, rows):
    """From few rows to many, and the norm after the residual left out."""
    i = inputs(dev, rows, 512, F16)
    if not pre:
        i["pre"] = None
    for dtype in (F32, I8):
        check_norm(i, dtype=dtype)


@pytest.mark.parametrize("n,rows", [(4, 20000), (256, 9000), (260, 9000), (512, 6001), (516, 5000), (1024, 5000), (1536, 4500), (2048, 4400), (2052, 2100), (2560, 2100), (4096, 2100),
                                    (5120, 1100), (6144, 1100), (7168, 1030), (8192, 600), (12288, 600), (12292, 600), (16384, 530), (32768, 530)])
@pytest.mark.parametrize("x,res", [(F32, F32), (F16, F16), (F32, None)])
def test_norm_many_rows(dev, n, rows, x, res):
    """More rows than workgroups at once, at each width's split; the residual's place taken by r."""
    i = inputs(dev, rows, n, x, res, "row")
    check_norm(i, dtype=I8)
    if res is not None:
        want, mine = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], dtype=F16), i["res"].clone()
        got = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=mine, res_out=mine, dtype=F16)
        assert got[0] is mine and all(torch.equal(a, b) for a, b in zip(got[:2], want[:2]))


@pytest.mark.parametrize("n", [128, 1536, 4096, 7168, 16384])
@pytest.mark.parametrize("rows", [64, 3000])
def test_norm_bad_rows_beside(dev, n, rows):
    """Rows behind a batch hold anything: NaN and infinities in every third row change no other row."""
    i = inputs(dev, rows, n)
    want = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], dtype=I8), A.ggml_m4_rows_i8(i["x"])
    for k, v in enumerate((math.nan, math.inf, -math.inf)):
        i["x"][k::9] = v
    good = torch.ones(rows, dtype=torch.bool, device=dev)
    for k in range(3):
        good[k::9] = False
    got = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], dtype=I8), A.ggml_m4_rows_i8(i["x"])
    for g, w in zip(got, want):
        assert all(torch.equal(a[good], b[good]) for a, b in zip(g, w)) and torch.isnan(g[-1][~good]).all() and (g[-2][~good] == 0).all()


def test_norm_into_given(dev):
    """Outputs of other types than the default, into views whose padding stays, and r in the place of the residual."""
    i = inputs(dev, 33, 260)
    for rt in (F32, F16):
        for dt in (F32, F16, I8):
            ro, out = torch.full((33, 300), 7, dtype=rt, device=dev), torch.full((33, 300), 7, dtype=dt, device=dev)
            sc = torch.full((40,), 7.0, device=dev)
            r, h, s = check_norm(i, dtype=F32, scale=2.0, got=None, res_out=ro[:, 8:268], out=out[:, 12:272], out_scale=sc[3:36] if dt == I8 else None) \
                if dt == F32 else A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], scale=2.0, res_out=ro[:, 8:268],
                                                 out=out[:, 12:272], out_scale=sc[3:36] if dt == I8 else None)
            if dt != F32:
                check_norm(i, scale=2.0, dtype=dt, got=(r, h, s), res_out=ro[:, 8:268])
            assert r.data_ptr() == ro[:, 8:].data_ptr() and h.data_ptr() == out[:, 12:].data_ptr()
            for t, a, b in ((ro, 8, 268), (out, 12, 272)):
                assert (t[:, :a] == 7).all() and (t[:, b:] == 7).all()
            assert (sc[:3] == 7).all() and (sc[36:] == 7).all()
    want = A.ggml_m4_norm(i["x"], i["pre"], EPS, res=i["res"], dtype=I8)
    res = i["res"].clone()
    got = A.ggml_m4_norm(i["x"], i["pre"], EPS, res=res, res_out=res, dtype=I8)
    assert got[0] is res and all(torch.equal(a, b) for a, b in zip(got, want))
    y = i["x"].clone()                                                        # the block's output and the residual are one tensor
    near(A.ggml_m4_norm(y, i["pre"], EPS, res=y)[0], 2 * y.double(), 0)


def test_norm_strided(dev):
    """Rows inside wider ones, as the parts of a product's rows: x, the residual and a gate for each value."""
    wide = inputs(dev, 21, 2112, gate="full")
    i = dict(x=wide["x"][:, 64:1600], res=wide["res"][:, :1536], gate=wide["gate"][:, 576:], pre=wide["pre"][4:1540], post=wide["post"][:1536])
    for dtype in (F32, F16, I8):
        check_norm(i, dtype=dtype)


def test_norm_nonfinite(dev):
    """A row with a NaN or an infinity, and the rows beside it; rows of zeros; the largest and the smallest values."""
    i = inputs(dev, 9, 1024, gate="none", post=False)
    for r, v in enumerate((math.nan, math.inf, -math.inf)):
        i["x"][r, 700] = v
    i["x"][3], i["res"][3] = 0, 0
    i["x"][4] *= 1e30
    i["res"][4] *= 1e30
    i["x"][5] *= 1e-38
    i["res"][5] *= 1e-38
    i["x"][6] = 0
    i["x"][6, 3] = 2.0 ** -149
    i["res"][6] = 0
    r, h, s = A.ggml_m4_norm(i["x"], i["pre"], EPS, res=i["res"], dtype=I8)
    assert torch.isnan(s[:3]).all() and (h[:3] == 0).all() and float(s[3]) == 0 and (h[3] == 0).all()
    assert int(h[6, 3].abs()) == 127 and int((h[6] != 0).sum()) == 1
    good = slice(3, None)
    check_norm({**i, "x": i["x"][good], "res": i["res"][good]}, dtype=I8, got=(r[good], h[good], s[good]))
    r, h, _ = A.ggml_m4_norm(i["x"], i["pre"], EPS, res=i["res"])
    assert torch.isnan(h[0]).all() and torch.isnan(h[1, 700]) and torch.isnan(h[2, 700]) and (h[1, :700] == 0).all()
    check_norm({**i, "x": i["x"][good], "res": i["res"][good]}, got=(r[good], h[good], None))
    # an f16 residual that overflows is stored as an infinity, and the norm is of what is stored
    r, h, s = A.ggml_m4_norm(torch.full((1, 64), 65000.0, device=dev), i["pre"][:64], EPS, res=torch.full((1, 64), 65000.0, device=dev).half(), dtype=I8)
    assert torch.isinf(r).all() and torch.isnan(s).all() and (h == 0).all()


# ------------------------------------------------------------------------------------ int8 rows
def check_i8(x, got):
    q, s = got
    flat = x.flatten(1)
    wq, ws = int8_64(flat.double())
    assert q.dtype == I8 and q.shape == flat.shape and torch.equal(q, wq), int((q != wq).sum())
    near(s, ws, 2.0 ** -24, 2.0 ** -150)


@pytest.mark.parametrize("shape", [(1, 4), (5, 256), (3, 1028), (64, 7168), (2, 32768), (300, 4096), (2, 1, 128), (7, 3, 4), (48, 32, 128), (9, 40, 128), (130, 128, 256), (9000, 256), (4500, 3, 512), (1100, 6144), (600, 100, 128), (530, 32768)])
@pytest.mark.parametrize("x", [F32, F16])
def test_rows_i8(dev, shape, x):
    g = torch.Generator().manual_seed(len(shape) + shape[0])
    v = (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn((shape[0],) + (1,) * (len(shape) - 1), generator=g))).to(x).to(dev)
    check_i8(v, A.ggml_m4_rows_i8(v))


@pytest.mark.parametrize("x", [F32, F16])
def test_rows_i8_strided(dev, x):
    """The heads' pieces as wv_b leaves them, every other head, parts of wider rows; into a view."""
    g = torch.Generator().manual_seed(5)
    o = torch.randn((12, 31, 136), generator=g).to(x).to(dev)
    for v in (o.permute(1, 0, 2), o.permute(1, 0, 2)[:, ::3], o.permute(1, 0, 2)[:, :, 4:132], o[:, :, :128], o[:, 5], o[3:4, :5]):
        check_i8(v, A.ggml_m4_rows_i8(v))
    buf, s = torch.full((31, 2048), 9, dtype=I8, device=dev), torch.empty(31, device=dev)
    v = o.permute(1, 0, 2)[:, :, :128]
    q, _ = A.ggml_m4_rows_i8(v, out=buf[:, 16:16 + 12 * 128], scale=s)
    check_i8(v, (q, s))
    assert (buf[:, :16] == 9).all() and (buf[:, 16 + 12 * 128:] == 9).all()
    check_i8(o[0, :1].expand(6, 136), A.ggml_m4_rows_i8(o[0, :1].expand(6, 136)))      # one row six times


def test_rows_i8_borders(dev):
    """Values on and next to the borders between two integers: every quotient against exact fractions."""
    tops = [127.0, 1.0, 254.0, 2.0 ** -100, 3.0, 0.1, 1e38, 127 * 2.0 ** -149]
    rows = []
    for t in tops:
        t = float(torch.tensor(t, dtype=F32))
        v = [t]
        for k in range(0, 127):
            mid = torch.tensor((k + 0.5) * t / 127, dtype=torch.float64).float()
            v += [float(mid), float(torch.nextafter(mid, torch.tensor(math.inf))), -float(torch.nextafter(mid, torch.tensor(-math.inf)))]
        rows.append(v + [0.0] * (384 - len(v)))
    x = torch.tensor(rows, dtype=F32)
    q, s = A.ggml_m4_rows_i8(x.to(dev))
    for r, row in enumerate(x.tolist()):
        top = max(Fraction(abs(v)) for v in row)
        for c, v in enumerate(row):
            steps = abs(Fraction(v)) * 127 / top
            want = int(steps + Fraction(1, 2)) * (1 if v >= 0 else -1)
            assert int(q[r, c]) == want, (r, c, v, int(q[r, c]), want)
    near(s.cpu(), x.double().abs().amax(1) / 127, 2.0 ** -24, 2.0 ** -150)


def test_rows_i8_nonfinite(dev):
    x = torch.randn((6, 512), generator=torch.Generator().manual_seed(1)).to(dev)
    x[0, 5], x[1, 511], x[2, 0], x[3] = math.nan, math.inf, -math.inf, 0
    for v in (x, x.half()):
        q, s = A.ggml_m4_rows_i8(v)
        assert torch.isnan(s[:3]).all() and (q[:4] == 0).all() and float(s[3]) == 0
        check_i8(v[4:], (q[4:], s[4:]))


# ------------------------------------------------------------------------------------ rope of q
def rope_bound(x, dtype):
    """The angle's part of a turn rounded to f32 (at most half a turn: pi 2^-24 in the angle), sine and cosine to 2 steps, the
    magnitude's product (and its own rounding) and two products and a sum: 8 roundings of 2^-24 beside |x0| + |x1|, times 1.6
    for the magnitude; then the stored type's."""
    pair = (x[..., 0::2].abs() + x[..., 1::2].abs()).double().repeat_interleave(2, -1) * 1.6
    return pair * (math.pi + 8) * 2.0 ** -24 + (0 if dtype == F32 else pair * 2.0 ** -11 + 2.0 ** -25)


@pytest.mark.parametrize("rows,heads,n", [(1, 1, 32), (1, 32, 64), (3, 5, 64), (64, 32, 64), (65, 40, 64), (7, 128, 64), (5, 3, 96), (5, 9, 256), (2, 1024, 32), (1001, 16, 64), (20000, 3, 64)])
@pytest.mark.parametrize("x", [F32, F16])
@pytest.mark.parametrize("out", [F32, F16])
@pytest.mark.parametrize("rp", [YARN, PLAIN])
def test_qrope(dev, rows, heads, n, x, out, rp):
    g = torch.Generator().manual_seed(rows + heads)
    wide = torch.randn((rows, heads, 128 + n), generator=g).to(x).to(dev)
    pos = torch.randint(0, 200000, (rows,), generator=g, dtype=torch.int32)
    pos[0] = 10 ** 7
    qcur = torch.full((rows, heads, 512 + n), 7, dtype=out, device=dev)
    got = A.ggml_m4_qrope(wide[:, :, 128:], pos.to(dev), A.rope_params(n_dims=n, **rp), out=qcur[:, :, 512:])
    assert got.data_ptr() == qcur[:, :, 512:].data_ptr() and (qcur[:, :, :512] == 7).all()
    want = rope64(wide[:, :, 128:], pos.to(dev), rp)
    assert ((got.double() - want).abs() <= rope_bound(wide[:, :, 128:], out)).all(), float((got.double() - want).abs().max())


def test_qrope_in_place_and_new(dev):
    g = torch.Generator().manual_seed(3)
    q, pos = torch.randn((9, 4, 64), generator=g).to(dev), torch.arange(9, dtype=torch.int32, device=dev) * 77
    rope = A.rope_params(n_dims=64, **YARN)
    want = A.ggml_m4_qrope(q, pos, rope)
    assert want.dtype == F32 and want.shape == q.shape and torch.equal(want[0, :, :], A.ggml_m4_qrope(q[:1], pos[:1], rope)[0])
    mine = q.clone()
    assert A.ggml_m4_qrope(mine, pos, rope, out=mine) is mine and torch.equal(mine, want)
    heads_first = torch.empty((4, 9, 64), device=dev)
    A.ggml_m4_qrope(q, pos, rope, out=heads_first.permute(1, 0, 2))
    assert torch.equal(heads_first.permute(1, 0, 2), want)
    q[2, 1, 8] = math.nan                                                     # reaches its pair and nothing else
    got = A.ggml_m4_qrope(q, pos, rope)
    assert torch.isnan(got[2, 1, 8:10]).all() and int(torch.isnan(got).sum()) == 2
