"""KQKV over the pages of a batch (mla_m4_kqkv_paged) against 64 bits: lengths from one token to long ones, requests
without tokens, pages that end inside a tile, shared prefixes, ids that are no pages, NaN and infinities in cells that
nobody sees, other strides, streams, captured graphs.  paged_util.attend64 derives the bounds."""
import math

import pytest
import torch

import aubier_amd as A

from paged_util import Batch, SCALE, attend64, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dk", [576, 320])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("past,new,page", [
    ([0], [1], 16), ([1], [1], 64), ([62], [1], 16), ([63], [1], 64), ([64], [1], 32), ([199], [1], 128),
    ([0, 15, 16, 700], [1, 1, 1, 1], 16), ([5, 0, 300], [0, 1, 0], 64), ([2500], [1], 256)])
def test_single_tokens(dev, dk, cache, past, new, page):
    b = Batch(dev, past, new, page, dk=dk, cache=cache, pad=2, seed=len(past) + page)
    check(b, b.run(), f"{cache} {past}")


@pytest.mark.parametrize("H", [1, 3, 16, 31, 32, 33, 40, 64, 128, 200])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_heads(dev, H, cache):
    b = Batch(dev, [130, 7, 513], [1, 1, 2], 32, dk=320, H=H, cache=cache, pad=1, seed=H)
    check(b, b.run(b.out(torch.float16)), f"H={H}")


@pytest.mark.parametrize("q_type", [torch.float16, torch.float32])
@pytest.mark.parametrize("dst", [torch.float16, torch.float32])
@pytest.mark.parametrize("dk", [576, 320])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_types(dev, q_type, dst, dk, cache):
    b = Batch(dev, [500, 40, 0], [1, 3, 9], 64, dk=dk, H=40, cache=cache, q_type=q_type, pad=3, seed=3)
    check(b, b.run(b.out(dst)))
    b = Batch(dev, [400, 420, 330], [1, 1, 2], 64, dk=dk, H=32, cache=cache, q_type=q_type, prefix=320, share=3, seed=4)
    check(b, b.run(b.out(dst)))


@pytest.mark.parametrize("new", [[2], [4], [5, 1, 3], [17], [64, 1, 1], [200, 0, 1, 30]])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("past0", [0, 61, 1000])
def test_several_tokens(dev, new, cache, past0):
    past = [past0 + 13 * i for i in range(len(new))]
    b = Batch(dev, past, new, 16, dk=320 if past0 else 576, H=16 if past0 == 61 else 32, cache=cache, pad=5, seed=past0)
    check(b, b.run(), f"{past} {new}")


@pytest.mark.parametrize("prefix,share,past,new", [
    (64, 2, [64, 64], [1, 1]), (640, 5, [640, 641, 700, 900, 2000], [1, 1, 1, 1, 1]),
    (1008, 3, [1100, 1010, 1300, 50, 4000], [1, 4, 2, 1, 3]), (2048, 9, [2048 + 7 * i for i in range(9)], [1] * 9),
    (512, 2, [600, 512], [40, 1]), (48, 3, [60, 50, 48], [1, 1, 1])])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("dk,H", [(576, 32), (320, 40), (576, 16)])
def test_shared_prefix(dev, prefix, share, past, new, cache, dk, H):
    b = Batch(dev, past, new, 16, dk=dk, H=H, cache=cache, prefix=prefix, share=share, pad=1, seed=prefix)
    got = b.run()
    check(b, got, f"prefix {prefix}")
    check(b, b.run(prefix=False), "unshared")


@pytest.mark.parametrize("prefix", [[5000, 3], [-5, 2], [320, -1], [320, 0], [320, 1], [320, 900], [2 ** 31 - 1, 2 ** 31 - 1]])
def test_prefix_out_of_range(dev, prefix):
    """More cells or requests than there are, or fewer than none: the shared cells that all of them hold."""
    b = Batch(dev, [400, 420, 330], [1, 1, 2], 64, dk=320, prefix=320, share=3, seed=4)
    b.prefix = torch.tensor(prefix, dtype=torch.int32, device=dev)
    if prefix[0] > 320:                                      # a request whose table begins otherwise would be wrong
        b = Batch(dev, [320, 320, 320], [1, 1, 2], 64, dk=320, prefix=320, share=3, seed=4)
        b.prefix = torch.tensor(prefix, dtype=torch.int32, device=dev)
    check(b, b.run())


def test_many_requests(dev):
    past = [(37 * i * i) % 400 for i in range(700)]
    b = Batch(dev, past, [1 if i % 5 else 0 for i in range(700)], 16, dk=320, H=16, seed=9, pad=2)
    check(b, b.run())


def test_long_context(dev):
    b = Batch(dev, [70001, 12, 30000], [1, 1, 2], 128, dk=576, H=16, seed=5)
    check(b, b.run())


def test_pages_that_are_none(dev):
    """Ids below zero or past the pool: their keys are not seen; a request that has no other sees none and gets zeros."""
    b = Batch(dev, [300, 90, 200, 20], [1, 3, 1, 2], 16, dk=320, H=32, seed=6)
    t = b.table.clone()
    t[0, 3], t[0, 7], t[0, 18] = -1, 10 ** 9, -2 ** 31
    t[1, :6] = 2 ** 31 - 1
    t[2, 5:] = -7
    t[3, :] = -1
    b.table = t
    b.kc[torch.isnan(b.kc)] = 1.0
    got = b.run()
    check(b, got)
    assert (got[:, 5:7] == 0).all()


def test_lengths_out_of_range(dev):
    """Negative lengths count as none; cells past the table's width are not there; rows past nt are not."""
    b = Batch(dev, [100, 40, 30], [1, 1, 2], 16, dk=320, seed=7, poison=1.0)
    b.past[0] = -9
    b.new[1] = -3
    b.past[2] = 10 ** 9                                      # sees its whole table, whose tail is no page
    b.rows = 3
    check(b, b.run(), "past, new out of range")
    b = Batch(dev, [100, 40, 30], [1, 1, 2], 16, dk=320, seed=8)
    b.q, b.nt, b.rows = b.q[:3], 3, 3
    want, tol = attend64(Batch(dev, [100, 40, 30], [1, 1, 2], 16, dk=320, seed=8))
    got = b.run()
    assert ((got.double() - want[:, :3]).abs() <= tol[:, :3]).all()
    b.new[:] = 2 ** 31 - 1                                   # request 0 takes all three rows
    b.rows = 3
    b.kc[torch.isnan(b.kc)] = 1.0
    got = b.run()
    b.new[:] = torch.tensor([3, 0, 0])
    check(b, got, "new past nt")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_later_tokens_do_not_reach_earlier_ones(dev, bad, cache):
    """A cell that only later tokens of the request see: whatever it holds, the earlier ones' results stay the same,
    and those that see it take it in."""
    if cache == "q8" and math.isinf(bad):
        pytest.skip("an infinite scale times a zero quant is NaN as well")
    for past, new, H, at in ((60, 9, 32, 64), (0, 70, 40, 33), (500, 3, 16, 501), (126, 4, 8, 127)):
        b = Batch(dev, [past], [new], 16, dk=320, H=H, cache=cache, seed=past + new, poison=1.0)
        want, tol = attend64(b)
        cell = int(b.table[0, at // 16]) * 16 + at % 16
        if cache == "f16":
            b.kc[cell] = bad
        else:
            b.kc.blocks[cell].unflatten(-1, (-1, 34))[:, 1] = 0x7e
        got = b.run()
        n = at - past                                        # tokens that do not see it
        assert ((got[:, :n].double() - want[:, :n]).abs() <= tol[:, :n]).all(), (past, new)
        if math.isnan(bad):
            assert torch.isnan(got[:, n:new]).all(), (past, new)


def test_nan_stays_in_its_request(dev):
    b = Batch(dev, [200, 300, 90], [1, 1, 1], 16, dk=576, prefix=64, share=0, seed=11, poison=1.0)
    want, tol = attend64(b)
    b.kc[int(b.table[1, 3]) * 16 + 5, 100] = math.nan
    got = b.run()
    assert torch.isnan(got[:, 1]).all()
    for t in (0, 2):
        assert ((got[:, t].double() - want[:, t]).abs() <= tol[:, t]).all()
    b.kc[int(b.table[1, 3]) * 16 + 5, 100] = 1.0
    b.q[2, 4] = math.nan
    got = b.run()
    assert torch.isnan(got[4, 2]).all() and torch.isfinite(got[:4]).all() and torch.isfinite(got[5:]).all()


def test_strides(dev):
    b = Batch(dev, [90, 500, 33], [1, 2, 1], 32, dk=320, H=40, seed=12)
    big = torch.full((b.nt, 42, 344), math.nan, dtype=b.q.dtype, device=dev)
    big[:, 1:41, 8:328] = b.q
    b.q = big[:, 1:41, 8:328]
    wide = torch.full((3, 77), -5, dtype=torch.int32, device=dev)
    wide[:, 2:2 + b.table.shape[1]] = b.table
    b.table = wide[:, 2:2 + b.table.shape[1]]
    check(b, b.run(), "q and table views")
    rows = torch.full((b.kc.shape[0], 360), math.nan, dtype=torch.float16, device=dev)
    rows[:, 16:336] = b.kc
    b.kc = rows[:, 16:336]
    check(b, b.run(), "cache view")
    swapped = b.q.transpose(0, 1).contiguous().transpose(0, 1)     # heads outermost
    b.q = swapped
    check(b, b.run(), "q by heads")


def test_scores_far_apart(dev):
    """Scores of some hundreds: the running maximum moves in many tiles."""
    for seed in range(3):
        b = Batch(dev, [900, 40, 333], [1, 5, 2], 16, dk=320, seed=seed, spread=30.0, poison=1.0)
        k, v = b.values.float(), b.values[:, :256].float()
        got = b.run().double()
        r = 0
        for s, (p, n) in enumerate(zip(b.past_l, b.new_l)):
            for i in range(n):
                j = torch.arange(p + i + 1, device=dev)
                cell = b.table[s, j // 16].long() * 16 + j % 16
                w = torch.softmax(b.q[r].double() @ k[cell].double().t() * SCALE, dim=1)
                # f32 sums of 320 products of up to some thousands: scores within 2^-11, weights within 2^-10
                want = w @ v[cell].double()
                assert ((got[:, r] - want).abs() <= 2.0 ** -8 * (w @ v[cell].double().abs()) + 1e-4).all(), (seed, s, i)
                r += 1


def test_largest_offsets(dev):
    """A pool past 4 GiB, pages at its end."""
    page, n_pages, dk = 64, 62000, 576
    kc = torch.empty((page * n_pages, dk), dtype=torch.float16, device=dev)      # 4.57 GB
    assert kc.numel() * 2 > 2 ** 32
    b = Batch(dev, [1000, 300, 70], [1, 1, 2], page, dk=dk, seed=13)
    need = b.kc.shape[0]
    kc[-need:] = b.kc
    b.table = torch.where(b.table >= 0, b.table + (n_pages - need // page), b.table)
    small, b.kc = b.kc, kc
    got = b.run()
    b.kc, b.values = small, small
    b.table = torch.where(b.table >= 0, b.table - (n_pages - need // page), b.table)
    check(b, got)


def test_captured_step_replays_with_new_lengths(dev):
    b = Batch(dev, [700, 130, 260, 64], [1, 2, 1, 1], 16, dk=320, prefix=64, share=4, seed=14, pad=2, poison=1.0)
    out = b.out()
    ws = torch.empty(max(16, A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, out, b.prefix)), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.run(out, workspace=ws)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.run(out, workspace=ws)
    for past, new, prefix in (([700, 130, 260, 64], [1, 2, 1, 1], [64, 4]), ([500, 100, 0, 10], [0, 3, 1, 1], [0, 0]),
                              ([64, 64, 64, 64], [1, 1, 1, 0], [64, 3]), ([700, 130, 260, 64], [1, 2, 1, 1], [64, 4])):
        b.past.copy_(torch.tensor(past))
        b.new.copy_(torch.tensor(new))
        b.prefix.copy_(torch.tensor(prefix))
        b.rows = sum(new)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        check(b, replayed, f"replay {past}")
        assert torch.equal(replayed, b.run())


def test_two_streams(dev):
    bs = [Batch(dev, [3000 + i, 50], [1, 3], 16, dk=320, seed=20 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for b, st, o in zip(bs, streams, outs):
            with torch.cuda.stream(st):
                o.append(b.run())
    torch.cuda.synchronize()
    for b, o in zip(bs, outs):
        check(b, o[0])
        assert all(torch.equal(x, o[0]) for x in o)


@pytest.mark.parametrize("n_seq", [256, 257, 4096])
def test_most_requests(dev, n_seq):
    new = [(1, 0, 2, 0, 0)[i % 5] for i in range(n_seq)]
    b = Batch(dev, [(29 * i) % 90 for i in range(n_seq)], new, 16, dk=320, H=8, seed=n_seq, pad=1)
    check(b, b.run(), f"{n_seq} requests")
    b = Batch(dev, [0] * (n_seq - 1) + [500], [0] * (n_seq - 1) + [3], 16, dk=320, H=8, seed=n_seq)      # only the last
    check(b, b.run(), "only the last")


@pytest.mark.parametrize("H,past,new", [(1024, [70, 130], [1, 1]), (1, [300], [300]), (1, [5, 900, 64], [33, 1, 130]), (7, [1000], [64])])
def test_rows_across_blocks(dev, H, past, new):
    """Blocks of 128 rows that begin and end inside a token, tokens that begin and end inside a block."""
    b = Batch(dev, past, new, 32, dk=320, H=H, seed=H, pad=1)
    check(b, b.run(b.out(torch.float16)))


def test_no_tokens(dev):
    b = Batch(dev, [50, 0, 7], [0, 0, 0], 16, dk=320, seed=1, pad=4)
    assert (b.run() == 7.0).all()


@pytest.mark.parametrize("scale", [0.0, -0.05, 1e-30])
def test_scales(dev, scale):
    b = Batch(dev, [700, 20], [1, 6], 16, dk=320, seed=2)
    got = A.ggml_m4_kqkv_paged(b.kc, b.q, b.past, b.new, b.table, 16, scale, out=b.out()).double()
    k, r = b.values.double(), 0
    for s, (p, n) in enumerate(zip(b.past_l, b.new_l)):
        for i in range(n):
            j = torch.arange(p + i + 1, device=dev)
            kk = k[b.table[s, j // 16].long() * 16 + j % 16]
            w = torch.softmax(b.q[r].double() @ kk.t() * scale, dim=1)
            # f16 weights and records: 2^-11 each, twice the former
            assert ((got[:, r] - w @ kk[:, :256]).abs() <= 4 * 2.0 ** -11 * (w @ kk[:, :256].abs()) + 2.0 ** -24).all()
            r += 1


@pytest.mark.parametrize("dk,H,past,new,prefix,share,cache", [
    (576, 32, [2100, 2048, 2300, 40], [1, 4, 1, 1], 2048, 3, "f16"), (320, 16, [3000, 10, 0], [1, 200, 1], 0, 0, "q8"),
    (320, 40, [600, 513, 700], [2, 2, 2], 512, 3, "q8"), (576, 128, [900, 33], [1, 3], 0, 0, "f16")])
def test_workspace(dev, dk, H, past, new, prefix, share, cache):
    """What the workspace holds at the start does not matter, nothing behind it (or behind dst) is written, and a byte
    less is refused."""
    b = Batch(dev, past, new, 16, dk=dk, H=H, cache=cache, prefix=prefix, share=share, pad=2, seed=31)
    need = A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, b.out(), b.prefix)
    big = torch.empty(need + (1 << 20), dtype=torch.uint8, device=dev)
    got = []
    for fill in (0, 255, 127):
        big.fill_(fill)
        room = torch.full((b.H * b.nt * b.dv + 4096,), 7.0, device=dev)
        out = room[:b.H * b.nt * b.dv].view(b.H, b.nt, b.dv)
        b.run(out, workspace=big[:need])
        assert (big[need:] == fill).all() and (room[b.H * b.nt * b.dv:] == 7.0).all()
        got.append(out)
    check(b, got[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    for bad in (big[:need - 1], big[1:], big[:1].expand(need), big.cpu()):
        with pytest.raises(A.MlaM4Error) as e:
            b.run(workspace=bad)
        assert e.value.status == -5


def test_shared_cells_on_pages_that_are_none(dev):
    b = Batch(dev, [700, 650, 640], [1, 2, 1], 16, dk=320, H=40, prefix=640, share=3, seed=32)
    t = b.table.clone()
    t[:, 4], t[:, 39] = -1, 10 ** 6
    b.table = t
    b.kc[torch.isnan(b.kc)] = 1.0
    check(b, b.run())


def test_first_sharer_without_tokens(dev):
    """The shared cells are read through the table of the first request that has tokens; the others' tables, and what
    they hold, do not matter."""
    b = Batch(dev, [400, 420, 330, 500], [0, 1, 2, 1], 64, dk=320, prefix=320, share=4, seed=33)
    b.table[0] = -1
    b.past[0] = 3
    check(b, b.run())


def test_same_pages_twice(dev):
    """Two requests with one table (a forked conversation before it writes): each sees the same cells."""
    b = Batch(dev, [333, 100], [1, 1], 16, dk=320, seed=34, poison=1.0)
    b.table[1] = b.table[0]
    b.past[1] = 333
    b.q[1] = b.q[0]
    got = b.run()
    check(b, got)
    assert torch.equal(got[:, 0], got[:, 1])
