"""An attention layer of a paged batch by the framework's operators alone, from one block's output to the next block's input:
norm with the residual, int8 products, the rope of q beside the absorbed part, KV rows, attention over pages, wv_b, int8 rows, the
output projection and the norms behind it.  Every step against its plain form in 64 bits on what the step before left."""
import math

import pytest
import torch

import aubier_amd as A

from paged_util import Batch, SCALE, attend64, q8_f16, q8_rows
from rows_util import EPS, YARN, half_step, int8_64, near, norm64, rope64

pytestmark = pytest.mark.gpu
F32, F16, I8 = torch.float32, torch.float16, torch.int8


class Layer:
    """A batch of requests over a pool of pages and a layer's weights; step() runs it for n_rows rows, padded."""

    def __init__(self, dev, past, new, n_rows, dk=576, H=16, cache="f16", seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.dk, self.dv, self.H, self.n_rows, self.cache = dk, {576: 512, 320: 256}[dk], H, n_rows, cache
        self.dn, self.dr, self.lat, self.n = {576: 128, 320: 64}[dk], 64, 384, 1024
        self.b = Batch(dev, past, [0] * len(past), 16, dk=dk, H=H, cache=cache, spare=60, max_pages=24, pad=n_rows, q_type=F32, seed=seed, poison=0.5)
        held = set(self.b.table[self.b.table >= 0].tolist())
        self.free = torch.tensor([i for i in range(60 + len(held)) if i not in held], dtype=torch.int32, device=dev)
        self.new = torch.tensor(new, dtype=torch.int32, device=dev)
        self.x, self.res = r(n_rows, self.n).to(dev), r(n_rows, self.n).to(dev)
        w = lambda n: (1 + 0.2 * r(n)).to(dev)  # noqa: E731
        self.pre, self.post, self.gate, self.q_norm, self.kv_norm, self.pre2 = w(self.n), w(self.n), w(self.n), w(self.lat), w(self.dv), w(self.n)
        weights = lambda n, k: A.ggml_m4_rows_i8((r(n, k) / math.sqrt(k)).to(dev))  # noqa: E731
        self.w_a, self.w_q, self.w_o = weights(self.lat + dk, self.n), weights(H * (self.dn + self.dr), self.lat), weights(self.n, H * 128)
        self.w_kb = (r(H, self.dv, self.dn) / math.sqrt(self.dn)).to(dev) if dk == 576 else \
            A.Q8_0(q8_rows(r(H * self.dv, 64) / 8).view(H, self.dv, -1).to(dev), 64)
        self.w_vb = A.Q8_0(q8_rows(r(H * 128, self.dv) / 16).view(H, 128, -1).to(dev), self.dv)
        self.qcur = torch.zeros((n_rows, H, dk), device=dev)
        self.kqv = torch.zeros((H, n_rows, self.dv), device=dev)
        self.rope = A.rope_params(n_dims=64, **YARN)
        self.got = {}

    def step(self):
        s, g = self, self.got
        g["slot"], g["pos"], g["used"] = A.ggml_m4_pages(s.b.past, s.new, s.free, s.b.table, 16, s.n_rows)
        g["r"], g["h"], g["hs"] = A.ggml_m4_norm(s.x, s.pre, EPS, post=s.post, gate=s.gate, res=s.res, scale=0.5, dtype=I8)
        g["a"] = A.ggml_m4_mul_i8(*s.w_a, g["h"], g["hs"])
        _, g["ql"], g["qls"] = A.ggml_m4_norm(g["a"][:, :s.lat], s.q_norm, EPS, dtype=I8)
        g["q"] = A.ggml_m4_mul_i8(*s.w_q, g["ql"], g["qls"])
        q = g["q"].view(s.n_rows, s.H, s.dn + s.dr)
        A.ggml_m4_qrope(q[:, :, s.dn:], g["pos"], s.rope, out=s.qcur[:, :, s.dv:])
        A.ggml_m4_wkb(s.w_kb, q[:, :, :s.dn], out=s.qcur[:, :, :s.dv])
        g["kcur"] = A.ggml_m4_kvrows(g["a"][:, s.lat:], s.kv_norm, s.b.kc, g["slot"], g["pos"], s.rope)
        A.ggml_m4_kqkv_paged(s.b.kc, s.qcur, s.b.past, s.new, s.b.table, 16, SCALE, out=s.kqv)
        g["o"] = A.ggml_m4_phase_wvb(s.w_vb, s.kqv)
        g["oi"], g["ois"] = A.ggml_m4_rows_i8(g["o"].permute(1, 0, 2))
        g["y"] = A.ggml_m4_mul_i8(*s.w_o, g["oi"], g["ois"])
        g["r2"], g["h2"], _ = A.ggml_m4_norm(g["y"], s.pre2, EPS, post=s.post, res=g["r"], dtype=F16)
        return g

    def moves_on(self):
        """The lengths and the free list behind a step."""
        taken = int(self.got["used"][0])
        self.b.past += self.new
        self.free.copy_(torch.cat([self.free[taken:], self.free[:taken]]))

    def check(self):
        s, g, n = self, self.got, int(self.new.sum())
        live = slice(0, n)
        r, exact, _, (q, step) = norm64(s.x, s.pre, EPS, s.post, s.gate, s.res, 0.5)
        near(g["r"], exact, 2.0 ** -24 * (1 + 2.0 ** -10))
        _, _, _, (q, step) = norm64(g["r"], s.pre, EPS)
        assert torch.equal(g["h"], q)
        near(g["hs"], step, 2.0 ** -23)
        mul = lambda w, x, xs: (x.double() @ w[0].double().t().contiguous()) * xs.double()[:, None] * w[1].double()  # noqa: E731
        near(g["a"], mul(s.w_a, g["h"], g["hs"]), 3.01 * 2.0 ** -24)
        _, _, _, (q, step) = norm64(g["a"][:, :s.lat], s.q_norm, EPS)
        assert torch.equal(g["ql"], q)
        near(g["q"], mul(s.w_q, g["ql"], g["qls"]), 3.01 * 2.0 ** -24)
        q = g["q"].view(s.n_rows, s.H, -1)
        pe = q[:, :, s.dn:]
        pair = (pe[..., 0::2].abs() + pe[..., 1::2].abs()).double().repeat_interleave(2, -1) * 1.6
        assert ((s.qcur[:, :, s.dv:].double() - rope64(pe, g["pos"], YARN)).abs() <= pair * (math.pi + 8) * 2.0 ** -24).all()
        assert torch.equal(s.qcur[:, :, :s.dv], A.ggml_m4_wkb(s.w_kb, q[:, :, :s.dn]))
        values = q8_f16(s.b.kc.blocks) if s.cache == "q8" else s.b.kc
        stored = values[g["slot"][live]]
        assert torch.equal(stored, q8_f16(q8_rows(g["kcur"][live])) if s.cache == "q8" else g["kcur"][live].half())
        b = s.b
        b.values, b.q, b.new, b.rows = values, s.qcur, s.new, n
        ref, tol = attend64(b)
        assert ((s.kqv[:, live].double() - ref).abs() <= tol).all()
        q, step = int8_64(g["o"].permute(1, 0, 2).flatten(1).double())
        assert torch.equal(g["oi"], q)
        near(g["ois"], step, 2.0 ** -24)
        near(g["y"], mul(s.w_o, g["oi"], g["ois"]), 3.01 * 2.0 ** -24)
        r2, exact, _, _ = norm64(g["y"], s.pre2, EPS, s.post, None, g["r"])
        near(g["r2"], exact, 2.0 ** -24 * (1 + 2.0 ** -10))
        rel, small = half_step(F16)
        near(g["h2"], norm64(g["r2"], s.pre2, EPS)[2], rel * (1 + 2.0 ** -9), small)


@pytest.mark.parametrize("dk", [576, 320])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("past,new,pad", [([40, 0, 31, 100], [1, 5, 1, 3], 3), ([0], [1], 0), ([17] * 20, [1] * 20, 12), ([3, 60], [130, 1], 0)])
def test_layer(dev, dk, cache, past, new, pad):
    s = Layer(dev, past, new, sum(new) + pad, dk, 16 if dk == 576 else 32, cache)
    s.step()
    s.check()
    s.moves_on()
    s.new.copy_(torch.tensor([1] * len(new)))               # and a step of decodes behind it, in the same room for rows
    s.step()
    s.check()


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_captured(dev, cache):
    """A graph of the layer, replayed with other lengths and inputs and the program's own work between, against eager runs; rows
    behind the batch hold NaN, which reaches no other row."""
    past, new, n_rows = [40, 0, 31, 100], [1, 5, 1, 3], 13
    s, e = (Layer(dev, past, new, n_rows, cache=cache, seed=4) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = s.b.table.clone(), (s.b.kc.blocks if cache == "q8" else s.b.kc).clone()
    with torch.cuda.stream(side):
        s.step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.step()
    s.b.table.copy_(keep[0])
    (s.b.kc.blocks if cache == "q8" else s.b.kc).copy_(keep[1])
    gen = torch.Generator().manual_seed(9)
    for lengths in (new, [1, 1, 1, 1], [2, 0, 4, 1], [0, 1, 0, 0]):
        n = sum(lengths)
        x = torch.randn((n_rows, s.n), generator=gen)
        x[n:] = math.nan
        for layer in (s, e):
            layer.x.copy_(x)
            layer.new.copy_(torch.tensor(lengths))
            layer.kqv[:, n:] = math.nan
        graph.replay()
        e.step()
        torch.cuda.synchronize()
        for k in ("slot", "pos", "used"):
            assert torch.equal(s.got[k], e.got[k])
        for k in ("r", "h", "hs", "a", "ql", "q", "kcur", "oi", "ois", "y", "r2", "h2"):
            a, b = s.got[k][:n], e.got[k][:n]
            assert torch.equal(a, b) and (a.dtype == I8 or torch.isfinite(a).all()), (k, lengths)
        assert torch.equal(s.kqv[:, :n], e.kqv[:, :n]) and torch.isnan(s.got["hs"][n:]).all() and torch.isnan(s.got["r2"][n:]).all()
        for layer in (s, e):
            layer.moves_on()
