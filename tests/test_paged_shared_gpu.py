"""KQKV over the pages of a batch behind a long shared prefix, in batches that are large enough for the shared cells to
be taken once for all of them; what tells is that only the first sharer's table is followed there."""
import math

import pytest
import torch

import aubier_amd as A

from paged_util import Batch, SCALE, attend64, check

pytestmark = pytest.mark.gpu

N = 64


def many(dev, prefix=2560, n=N, extra=(), new=None, behind=300, **kw):
    """n requests behind the same prefix, up to `behind` cells more each, then the others."""
    past = [prefix + (37 * i * i) % behind for i in range(n)] + [p for p, _ in extra]
    new = (list(new) if new else [1] * n) + [t for _, t in extra]
    return Batch(dev, past, new, 16, prefix=prefix, share=n, **kw)


def run_followed_once(b, first=0, **kw):
    """Runs b with every other sharer's first pages replaced by ids that are none: where the shared cells are taken once,
    through request `first`, that makes no difference.  (Whole tiles only are: their last page or two stay.)"""
    whole, table = int(b.prefix[0]) // 64 * 4, b.table
    b.table = table.clone()
    for s in range(int(b.prefix[1])):
        if s != first:
            b.table[s, :whole] = -1
    got = b.run(**kw)
    b.table = table
    return got


@pytest.mark.parametrize("dk", [576, 320])
@pytest.mark.parametrize("cache", ["f16", "q8"])
@pytest.mark.parametrize("q_type,dst", [(torch.float16, torch.float32), (torch.float32, torch.float16)])
@pytest.mark.parametrize("H", [16, 32])
def test_taken_once(dev, dk, cache, q_type, dst, H):
    b = many(dev, dk=dk, H=H, cache=cache, q_type=q_type, pad=3, extra=[(700, 1), (0, 1), (50, 9)], seed=H)
    got = run_followed_once(b, out=b.out(dst))
    check(b, got, "shared")
    check(b, b.run(b.out(dst), prefix=False), "not shared")


@pytest.mark.parametrize("H,n,prefix", [(1, 64, 1600), (3, 200, 1008), (40, 64, 1290), (8, 130, 1999), (16, 4096 // 16, 640)])
def test_heads_across_blocks(dev, H, n, prefix):
    """Blocks of 128 shared rows that begin and end inside a token; prefixes that end inside a tile or a page."""
    b = many(dev, dk=320, H=H, n=n, prefix=prefix, behind=90, seed=n)
    check(b, run_followed_once(b), f"H={H}")


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_requests_without_tokens_and_of_several(dev, cache):
    """The first sharer that has tokens is followed; one that holds fewer cells has no tokens, so it does not count."""
    new = [(0, 0, 1, 2, 1, 3, 1, 0)[i % 8] for i in range(N)]
    b = many(dev, dk=320, H=16, new=new, cache=cache, extra=[(100, 2)], seed=3)
    b.past[0] = 3
    check(b, run_followed_once(b, first=2))


def test_fewer_cells_than_the_prefix(dev):
    """What all sharing requests with tokens hold is what is taken once: one of 1,300 cells leaves 20 tiles."""
    b = many(dev, dk=320, H=16, seed=4)
    want, tol = attend64(b)
    keep = b.past.clone()
    b.past[7] = 1300
    b.prefix[0] = 2000000000
    table = b.table.clone()
    for s in range(1, N):
        b.table[s, :80] = -1                                 # 20 tiles of 64 cells on pages of 16
    got = b.run()
    rows = [r for r in range(N) if r != 7]                   # one token each: row r is request r's
    assert ((got.double() - want).abs() <= tol)[:, rows].all()
    b.table = table
    check(b, got, "the shorter one")
    b.past = keep


def test_no_pages_among_shared_cells(dev):
    b = many(dev, dk=320, H=16, seed=5, poison=1.0)
    b.table[:N, 4], b.table[:N, 39] = -1, 10 ** 6
    check(b, run_followed_once(b))


def test_nan_in_shared_cells_reaches_all_that_share(dev):
    b = many(dev, dk=576, H=16, seed=6, extra=[(500, 1)], poison=1.0)
    b.kc[int(b.table[0, 50]) * 16 + 3, 7] = math.nan
    got = b.run()
    assert torch.isnan(got[:, :N]).all() and torch.isfinite(got[:, N:]).all()


def test_captured_step_starts_and_stops_sharing(dev):
    b = many(dev, dk=320, H=16, seed=7, pad=2, extra=[(90, 2)], poison=1.0)
    out = b.out()
    ws = torch.empty(A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, out, b.prefix), dtype=torch.uint8, device=dev)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.run(out, workspace=ws)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.run(out, workspace=ws)
    past = b.past.clone()
    for cells, requests, few in ((2560, N, False), (0, 0, False), (2560, N, True), (128, N, False), (2560, 40, False), (2560, N, False)):
        b.prefix.copy_(torch.tensor([cells, requests]))
        b.past.copy_(torch.where(torch.arange(N + 1, device=dev) % 3 == 0, 0, past) if few else past)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        check(b, replayed, f"{cells} {requests} {few}")
        assert torch.equal(replayed, b.run())


@pytest.mark.parametrize("dk,H,cache", [(576, 32, "f16"), (320, 40, "q8")])
def test_workspace_of_shared_cells(dev, dk, H, cache):
    b = many(dev, dk=dk, H=H, cache=cache, seed=8, pad=2, extra=[(30, 9)])
    need = A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, b.out(), b.prefix)
    big = torch.empty(need + (1 << 20), dtype=torch.uint8, device=dev)
    got = []
    for fill in (0, 255, 127):
        big.fill_(fill)
        room = torch.full((b.H * b.nt * b.dv + 4096,), 7.0, device=dev)
        got.append(run_followed_once(b, out=room[:b.H * b.nt * b.dv].view(b.H, b.nt, b.dv), workspace=big[:need]))
        assert (big[need:] == fill).all() and (room[b.H * b.nt * b.dv:] == 7.0).all()
    check(b, got[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_scale_of_any_sign_over_shared_cells(dev):
    b = many(dev, dk=320, H=16, seed=9)
    want, tol = attend64(b)
    b.q = -b.q                                               # (-q) (-scale)
    got = A.ggml_m4_kqkv_paged(b.kc, b.q, b.past, b.new, b.table, 16, -SCALE, prefix=b.prefix, out=b.out())
    assert ((got.double() - want).abs() <= tol).all()
