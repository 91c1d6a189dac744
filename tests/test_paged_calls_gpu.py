"""The two ways from Python to the paged operators, the compiled module and ctypes: the same results, outputs and errors."""
import ctypes

import pytest
import torch

import aubier_amd as A
from aubier_amd import ops

from paged_util import Batch, SCALE, check

pytestmark = pytest.mark.gpu

RP = dict(freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, eps=1e-6, n_ctx_orig=4096)


def test_the_compiled_module_is_there():
    assert ops._calls()


@pytest.fixture(params=["compiled", "ctypes"])
def way(request, monkeypatch):
    monkeypatch.setattr(ops, "_native", ops._calls() if request.param == "compiled" else False)
    if request.param == "ctypes":
        monkeypatch.setattr(ops, "_calls", lambda: False)
    return request.param


def step(dev, cache="f16", out=False):
    """pages, rows and attention of one batch; everything that comes back."""
    b = Batch(dev, [70, 0, 300], [1, 5, 2], 16, dk=320, H=8, cache=cache, seed=1, poison=1.0, spare=8)
    table, free = b.table.clone(), torch.arange(100, 140, dtype=torch.int32, device=dev)
    kw = dict(slot=torch.empty(9, dtype=torch.int64, device=dev), pos=torch.empty(9, dtype=torch.int32, device=dev),
              used=torch.empty(2, dtype=torch.int32, device=dev)) if out else {}
    slot, pos, used = A.ggml_m4_pages(b.past, b.new, free, table, 16, 9, **kw)
    assert not out or (slot is kw["slot"] and pos is kw["pos"] and used is kw["used"])
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn((9, 320), generator=g).to(dev), torch.randn(256, generator=g).to(dev)
    # (rows into cells of the batch's own, as its pages stand)
    r = torch.arange(9, device=dev)
    cells = torch.where(r < 8, r * 3, -1)
    kcur = torch.empty((9, 320), device=dev) if out else None
    got = A.ggml_m4_kvrows(x, w, b.kc, cells, pos, A.rope_params(n_dims=64, **RP), out=kcur)
    assert not out or got is kcur
    o = torch.full((8, 8, 256), 7.0, device=dev) if out else None
    kqv = A.ggml_m4_kqkv_paged(b.kc, b.q, b.past, b.new, b.table, 16, SCALE, out=o,
                               workspace=torch.empty(1 << 26, dtype=torch.uint8, device=dev) if out else None)
    assert (kqv is o) if out else (kqv.dtype == torch.float16 and kqv.shape == (8, 8, 256))
    return [table, slot, pos, used, got, b.kc.blocks if cache == "q8" else b.kc, kqv.float()]


@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("out", [False, True])
def test_same_results(dev, cache, out, monkeypatch):
    there = ops._calls()
    compiled = step(dev, cache, out)
    monkeypatch.setattr(ops, "_native", False)
    monkeypatch.setattr(ops, "_calls", lambda: False)
    by_ctypes = step(dev, cache, out)
    assert there
    for a, b in zip(compiled, by_ctypes):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_errors(dev, way):
    b = Batch(dev, [70, 0, 300], [1, 5, 2], 16, dk=320, H=8, seed=1, poison=1.0)
    args = dict(kcache=b.kc, q=b.q, past=b.past, n_new=b.new, table=b.table, page_size=16, kq_scale=SCALE)
    for status, bad in ((-1, dict(past=b.past.cpu())), (-1, dict(q=b.q.cpu())), (-2, dict(kcache=b.kc.double())), (-2, dict(n_new=b.new.long())),
                        (-3, dict(table=b.table[None, None])), (-3, dict(q=b.q[0])), (-4, dict(past=torch.zeros(6, dtype=torch.int32, device=dev)[::2])),
                        (-6, dict(page_size=17)), (-6, dict(kq_scale=float("inf"))), (-2, dict(prefix=torch.zeros(2, device=dev))),
                        (-5, dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev))), (-8, dict(q=torch.zeros((8, 1025, 320), dtype=torch.float16, device=dev)))):
        with pytest.raises(A.MlaM4Error) as e:
            A.ggml_m4_kqkv_paged(**{**args, **bad})
        assert e.value.status == status, (way, bad.keys(), e.value.status)
    free = torch.arange(9, dtype=torch.int32, device=dev)
    for status, bad in ((-6, dict(page_size=20)), (-1, dict(free=free.cpu())), (-2, dict(free=free.float())), (-3, dict(used=free))):
        with pytest.raises(A.MlaM4Error) as e:
            A.ggml_m4_pages(**{**dict(past=b.past, n_new=b.new, free=free, table=b.table.clone(), page_size=16, n_rows=9), **bad})
        assert e.value.status == status, (way, bad.keys())
    x, rope = torch.zeros((9, 320), device=dev), A.rope_params(n_dims=64, **RP)
    for status, bad in ((-3, dict(kv_norm=torch.zeros(200, device=dev))), (-2, dict(slot=torch.zeros(9, dtype=torch.int32, device=dev))),
                        (-6, dict(rope=A.rope_params(n_dims=64, **{**RP, "eps": -1.0})))):
        with pytest.raises(A.MlaM4Error) as e:
            A.ggml_m4_kvrows(**{**dict(x=x, kv_norm=torch.zeros(256, device=dev), kcache=b.kc, slot=torch.zeros(9, dtype=torch.int64, device=dev),
                                       pos=torch.zeros(9, dtype=torch.int32, device=dev), rope=rope), **bad})
        assert e.value.status == status, (way, bad.keys())


def test_no_tensors_at_all(dev):
    b = Batch(dev, [70], [1], 16, dk=320, H=8, seed=1)
    calls, stream = ops._calls(), torch.cuda.current_stream().cuda_stream
    for bad in ([None, 0, b.q], [[1], 0, b.q], [b.kc, "x", b.q], [b.kc, 0, 3]):
        with pytest.raises(TypeError):
            calls.kqkv_paged(*bad, b.past, b.new, b.table, 16, 1.0, None, None, 256, None, stream)
    with pytest.raises(TypeError):
        calls.kqkv_paged(b.kc, 0, b.q, b.past, b.new, b.table, 16, 1.0, 5, None, 256, None, stream)
    with pytest.raises(TypeError):
        calls.kqkv_paged(b.kc, 0, b.q)
    with pytest.raises(TypeError):
        calls.pages(b.past, b.new, b.past, b.table, 16, 9, "slot", None, None, stream)
    with pytest.raises(TypeError):
        calls.kvrows(b.q, b.q, b.kc, 0, b.past, 1, ctypes.addressof(ctypes.c_int(0)), None, stream)


def test_streams_and_graphs(dev, way):
    b = Batch(dev, [700, 30], [1, 4], 16, dk=320, H=16, seed=5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = b.run()
    side.synchronize()
    check(b, got, way)
    g, out = torch.cuda.CUDAGraph(), b.out()
    with torch.cuda.graph(g, stream=side):
        b.run(out)
    for _ in range(3):
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)
