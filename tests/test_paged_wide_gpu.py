"""KQKV over the pages of a batch with so much to do that requests of more than 32 rows run in blocks of 128 (smaller
batches run in blocks of 32)."""
import math

import pytest
import torch

import aubier_amd as A

from paged_util import Batch, SCALE, attend64, check

pytestmark = pytest.mark.gpu

FEW_TILES = 1600                                             # of 32 rows by 64 keys: up to these, blocks of 32 rows


def wide(dev, past, new, page=16, H=40, **kw):
    b = Batch(dev, past, new, page, H=H, **{"dk": 320, **kw})
    assert sum(-(-n * H // 32) * ((p + n // 2) // 64 + 1) for p, n in zip(past, new)) > FEW_TILES
    return b


@pytest.mark.parametrize("q_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("dst", [torch.float16, torch.float32])
@pytest.mark.parametrize("dk", [576, 320])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_types(dev, q_type, dst, dk, cache):
    b = wide(dev, [9000, 40, 0, 4000], [9, 3, 2, 5], 64, dk=dk, cache=cache, q_type=q_type, pad=3, seed=3)
    check(b, b.run(b.out(dst)))


@pytest.mark.parametrize("H", [1, 7, 16, 33, 40, 64, 128, 200, 1024])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_heads(dev, H, cache):
    """Blocks that begin and end inside a token, the last ones of every number of rows."""
    n = max(2, -(-640 // H))
    b = wide(dev, [5300, 70, 3000], [n, 1, 1 + n // 2], 32, H=H, cache=cache, pad=1, seed=H)
    check(b, b.run(b.out(torch.float16)), f"H={H}")


@pytest.mark.parametrize("past,new", [([0], [900]), ([61, 700], [400, 300]), ([2500, 0, 64], [64, 300, 1]), ([7] * 40, [60] * 40),
                                      ([15000, 10, 20000], [6, 1, 1])])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_chunks(dev, past, new, cache):
    """Chunks of a prompt, most of whose tiles some rows see and others do not, beside single tokens."""
    b = wide(dev, past, new, 16, dk=320 if len(past) > 1 else 576, H=32, cache=cache, pad=5, seed=len(past))
    check(b, b.run(), f"{past} {new}")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_later_tokens_do_not_reach_earlier_ones(dev, bad, cache):
    if cache == "q8" and math.isinf(bad):
        pytest.skip("an infinite scale times a zero quant is NaN as well")
    for past, new, H, at in ((9000, 9, 40, 9004), (0, 700, 40, 333), (8190, 14, 32, 8193)):
        b = wide(dev, [past], [new], 16, H=H, cache=cache, seed=past + new, poison=1.0)
        want, tol = attend64(b)
        cell = int(b.table[0, at // 16]) * 16 + at % 16
        if cache == "f16":
            b.kc[cell] = bad
        else:
            b.kc.blocks[cell].unflatten(-1, (-1, 34))[:, 1] = 0x7e
        got = b.run()
        n = at - past
        assert ((got[:, :n].double() - want[:, :n]).abs() <= tol[:, :n]).all(), (past, new)
        if math.isnan(bad):
            assert torch.isnan(got[:, n:new]).all(), (past, new)


def test_pages_that_are_none(dev):
    b = wide(dev, [9000, 90, 200], [10, 3, 1], 16, seed=6)
    t = b.table.clone()
    t[0, 3:20], t[0, 100], t[0, 560:] = -1, 10 ** 9, -2 ** 31
    t[1, :6] = 2 ** 31 - 1
    t[2, :] = -1
    b.table = t
    b.kc[torch.isnan(b.kc)] = 1.0
    got = b.run()
    check(b, got)
    assert (got[:, 13] == 0).all()


def test_strides(dev):
    b = wide(dev, [9000, 500], [10, 2], 32, seed=12)
    big = torch.full((b.nt, 42, 344), math.nan, dtype=b.q.dtype, device=dev)
    big[:, 1:41, 8:328] = b.q
    b.q = big[:, 1:41, 8:328]
    rows = torch.full((b.kc.shape[0], 360), math.nan, dtype=torch.float16, device=dev)
    rows[:, 16:336] = b.kc
    b.kc = rows[:, 16:336]
    check(b, b.run(), "views")
    b.q = b.q.transpose(0, 1).contiguous().transpose(0, 1)         # heads outermost
    check(b, b.run(), "q by heads")


def test_captured_step_changes_its_blocks(dev):
    """The same graph over few tiles and many."""
    b = wide(dev, [9000, 130, 260], [9, 2, 1], 16, seed=14, pad=2, poison=1.0)
    out = b.out()
    ws = torch.empty(A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, out), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.run(out, workspace=ws)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.run(out, workspace=ws)
    for past, new in (([9000, 130, 260], [9, 2, 1]), ([500, 100, 0], [9, 0, 1]), ([8999, 0, 0], [9, 3, 0]), ([64, 64, 64], [1, 9, 2]), ([9000, 130, 260], [9, 2, 1])):
        b.past.copy_(torch.tensor(past))
        b.new.copy_(torch.tensor(new))
        b.rows = sum(new)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        check(b, replayed, f"replay {past}")
        assert torch.equal(replayed, b.run())


@pytest.mark.parametrize("dk,H,past,new,cache", [(576, 128, [9000, 33], [4, 3], "f16"), (320, 16, [3000, 10, 0], [1, 900, 1], "q8")])
def test_workspace(dev, dk, H, past, new, cache):
    b = wide(dev, past, new, 16, dk=dk, H=H, cache=cache, pad=2, seed=31)
    need = A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, b.out())
    big = torch.empty(need + (1 << 20), dtype=torch.uint8, device=dev)
    got = []
    for fill in (0, 255, 127):
        big.fill_(fill)
        room = torch.full((b.H * b.nt * b.dv + 4096,), 7.0, device=dev)
        b.run(room[:b.H * b.nt * b.dv].view(b.H, b.nt, b.dv), workspace=big[:need])
        assert (big[need:] == fill).all() and (room[b.H * b.nt * b.dv:] == 7.0).all()
        got.append(room[:b.H * b.nt * b.dv].view(b.H, b.nt, b.dv))
    check(b, got[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_scores_far_apart(dev):
    """Scores of some hundreds: the running maximum moves in many tiles."""
    b = wide(dev, [9000, 40], [10, 5], 16, seed=1, spread=30.0, poison=1.0)
    k = b.values
    got = b.run().double()
    r = 0
    for s, (p, n) in enumerate(zip(b.past_l, b.new_l)):
        for i in range(n):
            j = torch.arange(p + i + 1, device=dev)
            cell = b.table[s, j // 16].long() * 16 + j % 16
            w, v = torch.softmax(b.q[r].double() @ k[cell].double().t() * SCALE, dim=1), k[cell, :256].double()
            # f32 sums of 320 products of up to some thousands: scores within 2^-11, weights within 2^-10
            assert ((got[:, r] - w @ v).abs() <= 2.0 ** -8 * (w @ v.abs()) + 1e-4).all(), (s, i)
            r += 1
