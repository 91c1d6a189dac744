"""The two ways from Python to the operators around a batch's attention, the compiled module and ctypes: the same results, outputs
and errors; other streams than the current one's work."""
import pytest
import torch

import aubier_amd as A
from aubier_amd import ops

from rows_util import EPS, YARN

pytestmark = pytest.mark.gpu
F32, F16, I8 = torch.float32, torch.float16, torch.int8


@pytest.fixture(params=["compiled", "ctypes"])
def way(request, monkeypatch):
    there = ops._calls()
    assert there
    monkeypatch.setattr(ops, "_native", there if request.param == "compiled" else False)
    if request.param == "ctypes":
        monkeypatch.setattr(ops, "_calls", lambda: False)
    return request.param


def inputs(dev):
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g).to(dev)  # noqa: E731
    return dict(x=r(70, 512), res=r(70, 512).half(), pre=r(512), post=r(512), gate=r(70, 1), o=r(4, 70, 128), w=r(576, 512), q=r(70, 4, 192),
                pos=torch.arange(70, dtype=torch.int32, device=dev) * 100)


def run(i, out=False):
    dev = i["x"].device
    e = lambda *s, dtype=F32: torch.empty(s, dtype=dtype, device=dev)  # noqa: E731
    kw = dict(res_out=e(70, 512, dtype=F16), out=e(70, 512, dtype=I8), out_scale=e(70)) if out else {}
    r, h, hs = A.ggml_m4_norm(i["x"], i["pre"], EPS, post=i["post"], gate=i["gate"], res=i["res"], scale=0.5, dtype=I8, **kw)
    assert not out or (r is kw["res_out"] and h is kw["out"] and hs is kw["out_scale"])
    none, h16, no_scale = A.ggml_m4_norm(i["x"], i["pre"], EPS, dtype=F16)
    assert none is None and no_scale is None and h16.dtype == F16 and r.dtype == F16
    r_only, no_h, _ = A.ggml_m4_norm(i["x"], None, EPS, res=i["res"], dtype=None)
    assert no_h is None
    w, ws = A.ggml_m4_rows_i8(i["w"])
    kw = dict(out=e(70, 512, dtype=I8), scale=e(70)) if out else {}
    q, qs = A.ggml_m4_rows_i8(i["o"].permute(1, 0, 2), **kw)
    assert not out or (q is kw["out"] and qs is kw["scale"])
    y = e(70, 576, dtype=F16) if out else None
    got = A.ggml_m4_mul_i8(w, ws, h, hs, dtype=F16, out=y, workspace=torch.empty(1 << 24, dtype=torch.uint8, device=dev) if out else None)
    assert not out or got is y
    pe = torch.zeros((70, 4, 64), device=dev) if out else None
    rope = A.ggml_m4_qrope(i["q"][:, :, 128:], i["pos"], A.rope_params(n_dims=64, **YARN), out=pe)
    assert not out or rope is pe
    return [r, h, hs, h16, r_only, w, ws, q, qs, got, rope]


@pytest.mark.parametrize("out", [False, True])
def test_same_results(dev, out, monkeypatch):
    i = inputs(dev)
    compiled = run(i, out)
    monkeypatch.setattr(ops, "_native", False)
    monkeypatch.setattr(ops, "_calls", lambda: False)
    for a, b in zip(compiled, run(i, out)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_errors(dev, way):
    i = inputs(dev)
    x, pre = i["x"], i["pre"]
    w, ws = A.ggml_m4_rows_i8(i["w"])
    h, hs = A.ggml_m4_rows_i8(x)
    rope = A.rope_params(n_dims=64, **YARN)
    calls = [
        (-1, lambda: A.ggml_m4_norm(x, pre.cpu(), EPS)), (-1, lambda: A.ggml_m4_norm(x.cpu(), pre, EPS)), (-2, lambda: A.ggml_m4_norm(x.double(), pre, EPS)),
        (-2, lambda: A.ggml_m4_norm(x, pre, EPS, dtype=torch.bfloat16)), (-3, lambda: A.ggml_m4_norm(x[0], pre, EPS)), (-3, lambda: A.ggml_m4_norm(x[:, None], pre, EPS)),
        (-3, lambda: A.ggml_m4_norm(x, pre[:256], EPS)), (-4, lambda: A.ggml_m4_norm(x.t().contiguous().t(), pre, EPS)), (-6, lambda: A.ggml_m4_norm(x, pre, -1.0)),
        (-1, lambda: A.ggml_m4_norm(x, pre, EPS, dtype=None)), (-2, lambda: A.ggml_m4_norm(x, pre, EPS, out_scale=hs)),
        (-2, lambda: A.ggml_m4_norm(x, pre, EPS, gate=i["gate"].half())), (-3, lambda: A.ggml_m4_norm(x, pre, EPS, out=torch.empty((70, 256), device=dev))),
        (-2, lambda: A.ggml_m4_rows_i8(h)), (-3, lambda: A.ggml_m4_rows_i8(x[0])), (-3, lambda: A.ggml_m4_rows_i8(x[None, None])), (-1, lambda: A.ggml_m4_rows_i8(x, scale=hs.cpu())),
        (-2, lambda: A.ggml_m4_mul_i8(w.float(), ws, h, hs)), (-3, lambda: A.ggml_m4_mul_i8(w, ws, h[0], hs)), (-3, lambda: A.ggml_m4_mul_i8(w[:, :256].contiguous(), ws, h, hs)),
        (-1, lambda: A.ggml_m4_mul_i8(w, ws.cpu(), h, hs)), (-3, lambda: A.ggml_m4_mul_i8(w, ws, h, hs[:3])),
        (-5, lambda: A.ggml_m4_mul_i8(w, ws, h, hs, workspace=torch.empty(1 << 24, dtype=torch.uint8))),
        (-5, lambda: A.ggml_m4_mul_i8(w, ws, h, hs, workspace=torch.empty((64, 1 << 18), dtype=torch.uint8, device=dev)[:, ::2])),
        (-5, lambda: A.ggml_m4_mul_i8(w, ws, h, hs, workspace=torch.empty((1 << 24) + 8, dtype=torch.uint8, device=dev)[8:])),
        (-1, lambda: A.ggml_m4_qrope(i["q"][:, :, 128:], i["pos"].cpu(), rope)), (-3, lambda: A.ggml_m4_qrope(i["q"], i["pos"], rope)),
        (-2, lambda: A.ggml_m4_qrope(i["q"][:, :, 128:], i["pos"].long(), rope)),
        (-6, lambda: A.ggml_m4_qrope(i["q"][:, :, 128:], i["pos"], A.rope_params(n_dims=64, **{**YARN, "beta_fast": 0.0}))),
    ]
    for n, (status, call) in enumerate(calls):
        with pytest.raises(A.MlaM4Error) as e:
            call()
        assert e.value.status == status, (way, n, e.value.status)


def test_no_tensors_at_all(dev):
    calls, s, i = ops._calls(), torch.cuda.current_stream().cuda_stream, inputs(dev)
    for bad in (lambda: calls.norm(1, None, None, None, 1.0, None, 1e-6, None, None, None, 0, s), lambda: calls.norm(i["x"], None, None, None, "x", None, 1e-6, None, None, None, 0, s),
                lambda: calls.norm(i["x"]), lambda: calls.rows_i8(None, None, None, s), lambda: calls.rows_i8(i["x"]), lambda: calls.mul_i8(i["x"], 2, 3, 4, None, 0, None, s),
                lambda: calls.mul_i8(), lambda: calls.qrope(i["q"], None, 0, None, s), lambda: calls.qrope(i["q"], i["pos"], 0)):
        with pytest.raises(TypeError):
            bad()


def test_streams(dev, way):
    """On another stream, behind and ahead of work of its own; two streams at once with different inputs."""
    i = inputs(dev)
    want = run(i)
    j = {k: v.flip(0).contiguous() if k in ("x", "res", "gate", "q", "pos") else v for k, v in i.items()}
    want_j = run(j)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for s, a, g in zip(streams, (i, j), got):
            with torch.cuda.stream(s):
                g.append(run(a))
    torch.cuda.synchronize()
    for g, w in zip(got, (want, want_j)):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_graphs(dev, way):
    """All four captured, replayed over changed inputs with eager work between."""
    i = inputs(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(i)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = run(i)
    for k in range(4):
        i["x"].mul_(-1.5)
        i["o"].add_(0.25)
        i["q"].neg_()
        i["pos"].add_(3)
        want = run(i)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
