"""Page bookkeeping and batched KV rows (mla_m4_pages, mla_m4_kvrows) against plain forms on the host, and a whole step:
pages, rows, WKB, attention over pages, wv_b."""
import math

import numpy as np
import pytest
import torch

import aubier_amd as A

from paged_util import Batch, SCALE, attend64, q8_f16, q8_rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------ pages
def pages_host(past, new, free, table, page, n_rows):
    table, slot, pos, taken, mp = table.clone(), [], [], 0, table.shape[1]
    for b, (p, n) in enumerate(zip(past, new)):
        p, n = max(p, 0), max(n, 0)
        n = min(n, n_rows - len(slot))
        have = min(-(-p // page), mp)
        for j in range(have, min(-(-(p + n) // page), mp)):
            table[b, j] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n):
            j = (p + i) // page
            pid = int(table[b, j]) if j < mp else -1
            slot.append(pid * page + (p + i) % page if pid >= 0 else -1)
            pos.append(p + i)
    rows = len(slot)
    return (table, torch.tensor(slot + [-1] * (n_rows - rows)), torch.tensor(pos + [0] * (n_rows - rows), dtype=torch.int32),
            torch.tensor([min(taken, len(free)), rows], dtype=torch.int32))


def run_pages(dev, past, new, free, table, page, n_rows):
    t = table.to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    slot, pos, used = A.ggml_m4_pages(i32(past), i32(new), i32(free), t, page, n_rows)
    return t.cpu(), slot.cpu(), pos.cpu(), used.cpu()


@pytest.mark.parametrize("n_seq", [1, 2, 63, 64, 65, 255, 257, 1000, 4096])
@pytest.mark.parametrize("page", [16, 64, 65536])
@pytest.mark.parametrize("kind", ["decode", "mixed", "chunk"])
def test_pages(dev, n_seq, page, kind):
    rng = np.random.default_rng(n_seq + page)
    past = rng.integers(0, 5 * page + 3, n_seq).tolist()
    past[0] = 0
    if kind == "decode":
        new = [1] * n_seq
    elif kind == "mixed":
        new = rng.integers(0, 5, n_seq).tolist()
    else:
        new = [0] * n_seq
        new[n_seq // 2], new[-1] = 3000, 1
    mp = -(-(max(past) + max(new)) // page) + 1
    table = torch.from_numpy(rng.integers(0, 10 ** 6, (n_seq, mp)).astype(np.int32))
    free = rng.permutation(10 ** 5)[:sum(new) + 7].tolist()
    for spare in (0, 13, 700):
        args = (past, new, free, table, page, sum(new) + spare or 1)
        for got, want, name in zip(run_pages(dev, *args), pages_host(*args), ("table", "slot", "pos", "used")):
            assert torch.equal(got, want), name


def test_pages_out_of_range(dev):
    """The list ends, the table is too narrow, rows for fewer tokens, lengths below zero, entries that are no pages."""
    table = torch.tensor([[5, -3, 9], [7, 7, 7], [1, 2, 3], [-1, -1, -1]], dtype=torch.int32)
    for past, new, free, n_rows in (([20, 16, 0, 15], [20, 17, 40, 2], [100, 101], 200),
                                    ([40, 0, 33, 47], [90, 3, 16, 5], [50, 51, 52, 53, 54, 55], 60),
                                    ([-5, 10, -2 ** 31, 0], [3, -7, 20, 1], [9, 8, 7], 100),
                                    ([0, 0, 0, 0], [2 ** 31 - 1] * 4, [4, 3, 2, 1], 50),
                                    ([0, 16, 32, 48], [0, 0, 0, 0], [], 3),
                                    ([0, 16, 32, 48], [1, 1, 1, 1], [], 4)):
        args = (past, new, free, table, 16, n_rows)
        for got, want, name in zip(run_pages(dev, *args), pages_host(*args), ("table", "slot", "pos", "used")):
            assert torch.equal(got, want), (past, name)


def test_pages_into_views(dev):
    wide = torch.full((3, 40), 77, dtype=torch.int32, device=dev)
    rows = torch.full((64,), 5, dtype=torch.int64, device=dev)
    t = wide[:, 3:10]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    A.ggml_m4_pages(i32([16, 0, 30]), i32([1, 20, 3]), i32([1, 2, 3, 4, 5]), t, 16, 24, slot=rows[8:32],
                    pos=torch.empty(24, dtype=torch.int32, device=dev))
    want = pages_host([16, 0, 30], [1, 20, 3], [1, 2, 3, 4, 5], torch.full((3, 7), 77, dtype=torch.int32), 16, 24)
    assert torch.equal(t.cpu(), want[0]) and torch.equal(rows[8:32].cpu(), want[1])
    assert (wide[:, :3] == 77).all() and (wide[:, 10:] == 77).all() and (rows[:8] == 5).all() and (rows[32:] == 5).all()


# ------------------------------------------------------------------------------------ batched KV rows
ROPES = [dict(freq_base=1e6, freq_scale=0.25, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, eps=1e-6, n_ctx_orig=8192),
         dict(freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.3, beta_fast=32.0, beta_slow=1.0, eps=1e-5, n_ctx_orig=4096)]


def kvrows64(x, w, pos, rp, d_r):
    x, w, pos = x.double().cpu(), w.double().cpu(), pos.double().cpu()
    dl = x.shape[1] - d_r
    lat = x[:, :dl] / torch.sqrt((x[:, :dl] ** 2).mean(1, keepdim=True) + rp["eps"]) * w
    p = torch.arange(d_r // 2, dtype=torch.float64)
    f = rp["freq_base"] ** (-2.0 * p / d_r)
    ms = rp["attn_factor"]
    f32 = np.float32
    if rp["ext_factor"]:
        def corr(rot):
            return d_r * math.log(rp["n_ctx_orig"] / (rot * 2 * math.pi)) / (2 * math.log(rp["freq_base"]))
        lo, hi = max(0.0, math.floor(corr(rp["beta_fast"]))), min(d_r - 1.0, math.ceil(corr(rp["beta_slow"])))
        mix = (1.0 - torch.clamp((p - lo) / max(0.001, hi - lo), 0.0, 1.0)) * rp["ext_factor"]
        f = f * (float(f32(rp["freq_scale"])) * (1.0 - mix) + mix)
        ms *= 1.0 + 0.1 * math.log(1.0 / rp["freq_scale"])
    else:
        f = f * rp["freq_scale"]
    th = pos[:, None] * f
    co, si = torch.cos(th) * ms, torch.sin(th) * ms
    x0, x1 = x[:, dl::2], x[:, dl + 1::2]
    return torch.cat([lat, torch.stack([x0 * co - x1 * si, x0 * si + x1 * co], 2).flatten(1)], 1)


def kvrows_bound(x, want, d_r):
    """f32: the mean of d_lat squares (their sum's rounding is at most d_lat 2^-24 of it, half of that after the root),
    a root, a quotient and two products, 2^-24 each; a rope pair: its angle's part of a turn rounded to f32 (at most
    2 pi 2^-25 of a turn's half), sine and cosine within 2 steps, a product and a sum each.  All beside |x0| + |x1|."""
    dl = x.shape[1] - d_r
    b = want.abs() * (dl / 2 + 8) * 2.0 ** -24
    pair = (x[:, dl::2].abs() + x[:, dl + 1::2].abs()).double().cpu().repeat_interleave(2, 1) * 1.6
    b[:, dl:] = pair * (math.pi / 2 + 8) * 2.0 ** -24
    return b + 1e-30


@pytest.mark.parametrize("n,d_r", [(576, 64), (320, 64), (64, 32), (1024, 256), (544, 32)])
@pytest.mark.parametrize("rows", [1, 3, 64, 1001])
@pytest.mark.parametrize("xt", [torch.float32, torch.float16])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("rope", [0, 1])
def test_kvrows(dev, n, d_r, rows, xt, cache, rope):
    g = torch.Generator().manual_seed(n + rows)
    rp = ROPES[rope]
    x = torch.randn((rows, n), generator=g).to(xt).to(dev)
    w = (1 + 0.25 * torch.randn(n - d_r, generator=g)).to(dev)
    n_cells = 2 * rows + 5
    slot = torch.randperm(n_cells, generator=g)[:rows]
    pos = torch.randint(0, 200000, (rows,), generator=g, dtype=torch.int32)
    if rows > 2:
        slot[1], slot[2], pos[0] = -1, n_cells, 10 ** 7
    before = torch.randn((n_cells, n), generator=g).half().to(dev)
    blocks = q8_rows(before.float())
    kc = A.Q8_0(blocks.clone(), n) if cache == "q8" else before.clone()
    got = A.ggml_m4_kvrows(x, w, kc, slot.to(dev), pos.to(dev), A.rope_params(n_dims=d_r, **rp))
    want = kvrows64(x, w, pos, rp, d_r)
    off = (got.double().cpu() - want).abs() / kvrows_bound(x, want, d_r)
    print(f"worst error / bound {float(off.max()):.3f}", flush=True)
    assert float(off.max()) <= 1.0
    # the cache: the launch's own Kcur, rounded; every other row as it was
    live = (slot >= 0) & (slot < n_cells)
    if cache == "q8":
        blocks[slot[live].to(dev)] = q8_rows(got)[live.to(dev)]
        assert torch.equal(kc.blocks, blocks)
    else:
        before[slot[live].to(dev)] = got.half()[live.to(dev)]
        assert torch.equal(kc, before)


def test_kvrows_agrees_with_kvwrite(dev):
    """The row that KV-write stores and the batched form's from KV-write's own product (its Kcur undone is not to be
    had, so: a product with one weight per output, which makes the gemv exact)."""
    g = torch.Generator().manual_seed(1)
    n_embd, dl, d_r = 4096, 256, 64
    cur = torch.zeros(n_embd)
    cur[:320] = torch.randint(-127, 128, (320,), generator=g).float()
    for blk in range(10):                                    # every 32-block has its 127: scale 1, quants exact
        cur[32 * blk] = 127.0
    wq = torch.zeros((320, n_embd // 32, 34), dtype=torch.uint8)
    one = torch.tensor([1.0]).half().view(torch.uint8)
    for o in range(320):
        wq[o, o // 32, :2] = one
        wq[o, o // 32, 2 + o % 32] = 1
    w = (1 + 0.25 * torch.randn(dl, generator=g)).to(dev)
    rp = A.rope_params(n_dims=d_r, **ROPES[0])
    for pos in (0, 5, 900):
        kc1, kc2 = (torch.zeros((4, 320), dtype=torch.float16, device=dev) for _ in range(2))
        at, p = torch.tensor([2], device=dev), torch.tensor([pos], dtype=torch.int32, device=dev)
        k1 = A.ggml_m4_phase_kvwrite(cur.to(dev), A.Q8_0(wq.flatten(1).to(dev), n_embd), w, kc1, at, p, rp)
        k2 = A.ggml_m4_kvrows(cur[None, :320].to(dev), w, kc2, at, p, rp)[0]
        # KV-write's angles are f32 products: off by up to pos 2^-23 radians, beside |x0| + |x1| <= 254 at a scale of 1.14
        assert (k1 - k2).abs().max() <= 1e-4 + 300 * (pos + 8) * 2.0 ** -22, pos
        assert (kc1.float() - kc2.float()).abs().max() <= 0.2


def test_kvrows_views_and_no_kcur(dev):
    g = torch.Generator().manual_seed(2)
    rp = A.rope_params(n_dims=64, **ROPES[0])
    x = torch.randn((5, 576), generator=g).to(dev)
    w = torch.ones(512, device=dev)
    slot, pos = torch.arange(5, device=dev), torch.arange(5, dtype=torch.int32, device=dev)
    kc = torch.zeros((6, 576), dtype=torch.float16, device=dev)
    k = A.ggml_m4_kvrows(x, w, kc, slot, pos, rp)
    wide = torch.full((5, 700), math.nan, device=dev)
    wide[:, 4:580] = x
    rows = torch.full((6, 600), 3.0, dtype=torch.float16, device=dev)
    out = torch.full((5, 592), 3.0, device=dev)
    A.ggml_m4_kvrows(wide[:, 4:580], w, rows[:, 8:584], slot, pos, rp, out=out[:, 8:584])
    assert torch.equal(out[:, 8:584], k) and torch.equal(rows[:5, 8:584], kc[:5]) and (rows[5] == 3).all()
    assert (out[:, :8] == 3).all() and (out[:, 584:] == 3).all() and (rows[:, :8] == 3).all() and (rows[:, 584:] == 3).all()
    lib, P = A.load_library(), A.ops._ptr
    kc2 = torch.zeros_like(kc)
    v = A.view
    import ctypes
    assert lib.mla_m4_kvrows(P(v(x)), P(v(w)), P(v(kc2)), P(v(slot)), P(v(pos)), ctypes.byref(rp), None,
                             torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(kc2, kc)


# ------------------------------------------------------------------------------------ a whole step
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("captured", [False, True])
def test_step(dev, cache, captured):
    """Two steps of a batch at the reference geometry: its pages, slots and rows, WKB, the attention over the pages and
    wv_b, eagerly and as a graph that is replayed with the second step's lengths."""
    g = torch.Generator().manual_seed(3)
    H, dk, dv, page, n_rows = 32, 320, 256, 16, 12
    past, new = [40, 0, 31, 16], [1, 5, 1, 3]
    b = Batch(dev, past, [0] * 4, page, dk=dk, H=H, cache=cache, spare=30, max_pages=6, pad=n_rows, q_type=torch.float32, seed=3, poison=0.5)
    held = set(b.table[b.table >= 0].tolist())
    free = torch.tensor([i for i in range(30 + len(held)) if i not in held], dtype=torch.int32, device=dev)
    rp, f = ROPES[0], torch.float32
    x = torch.randn((n_rows, dk), generator=g).to(dev)
    w = (1 + 0.25 * torch.randn(dv, generator=g)).to(dev)
    qraw = torch.randn((n_rows, H, 128), generator=g).to(dev)
    wkb = A.Q8_0(q8_rows(torch.randn((H * dv, 64), generator=g) / 8).view(H, dv, -1).to(dev), 64)
    wvb = A.Q8_0(q8_rows(torch.randn((H * 128, dv), generator=g) / 16).view(H, 128, -1).to(dev), dv)
    qcur = torch.zeros((n_rows, H, dk), dtype=f, device=dev)
    kqv, out = torch.zeros((H, n_rows, dv), dtype=f, device=dev), torch.zeros((H, n_rows, 128), dtype=f, device=dev)
    slot, pos = torch.empty(n_rows, dtype=torch.int64, device=dev), torch.empty(n_rows, dtype=torch.int32, device=dev)
    used, kcur = torch.empty(2, dtype=torch.int32, device=dev), torch.empty((n_rows, dk), dtype=f, device=dev)
    n_new = torch.tensor(new, dtype=torch.int32, device=dev)
    ws = torch.empty(max(16, A.kqkv_paged_workspace_bytes(b.kc, qcur, b.past, kqv)), dtype=torch.uint8, device=dev)

    def step():
        A.ggml_m4_pages(b.past, n_new, free, b.table, page, n_rows, slot=slot, pos=pos, used=used)
        A.ggml_m4_kvrows(x, w, b.kc, slot, pos, A.rope_params(n_dims=64, **rp), out=kcur)
        A.ggml_m4_wkb(wkb, qraw[:, :, :64], out=qcur[:, :, :dv])
        qcur[:, :, dv:].copy_(qraw[:, :, 64:])
        A.ggml_m4_kqkv_paged(b.kc, qcur, b.past, n_new, b.table, page, SCALE, out=kqv, workspace=ws)
        A.ggml_m4_phase_wvb(wvb, kqv, out=out)

    run = step
    if captured:
        saved = (b.table.clone(), b.kc.blocks.clone() if cache == "q8" else b.kc.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        b.table.copy_(saved[0])
        (b.kc.blocks if cache == "q8" else b.kc).copy_(saved[1])
        run = graph.replay
    table = b.table.cpu()
    for lengths in (new, [1, 2, 0, 1]):
        n_new.copy_(torch.tensor(lengths))
        run()
        torch.cuda.synchronize()
        want = pages_host(past, lengths, free.tolist(), table, page, n_rows)
        for got, ref in zip((b.table, slot, pos, used), want):
            assert torch.equal(got.cpu(), ref)
        n = sum(lengths)
        values = q8_f16(b.kc.blocks) if cache == "q8" else b.kc
        stored = values[slot[:n]]
        assert torch.equal(stored, q8_f16(q8_rows(kcur[:n])) if cache == "q8" else kcur[:n].half())
        b.values, b.q, b.new, b.rows = values, qcur, n_new, n
        ref, tol = attend64(b)
        assert ((kqv[:, :n].double() - ref).abs() <= tol).all()
        assert torch.equal(out, A.ggml_m4_phase_wvb(wvb, kqv))
        past = [p + k for p, k in zip(past, lengths)]
        table = want[0]
        b.past.copy_(torch.tensor(past))
        free.copy_(torch.cat([free[int(want[3][0]):], free[:int(want[3][0])]]))
