"""NaN and infinities in cells that tokens see, against the definition in 64 bits, element by element: a score of NaN or +inf
makes a row NaN; a cell of score -inf has weight 0, which makes NaN of the columns in which it is not finite and leaves
the others.  The same whichever way the batch is cut: blocks of 32 and of 128 rows, tiles that all rows see and tiles
that some do, results that go to dst at once and results that are merged."""
import math

import pytest
import torch

from paged_util import Batch, SCALE, attend64

INF, NAN = math.inf, math.nan


def definition(b, dst_type=torch.float32):
    """(out [H, rows, D_v], tolerance) as attend64, with NaN where the definition has it.  Scores of cells that hold a NaN or
    an infinity are summed element by element; the others' values enter the products, where they are finite."""
    v64 = b.values.double()
    past, new, table = b.past.tolist(), b.new.tolist(), b.table.tolist()
    out = torch.zeros((b.H, b.rows, b.dv), dtype=torch.float64, device=v64.device)
    tol = torch.zeros_like(out)
    u16, r = 2.0 ** -11, 0
    for s, (p, n) in enumerate(zip(past, new)):
        j = torch.arange(p + n, device=v64.device)
        k = v64[torch.tensor(table[s], device=v64.device)[j // b.page].long() * b.page + j % b.page]
        fine = torch.isfinite(k)
        clean, odd = torch.where(fine, k, 0.0), ~fine.all(1)
        for i in range(n):
            m = p + i + 1
            q = b.q[r].double()
            sc = q @ clean[:m].t() * SCALE
            at = odd[:m].nonzero()[:, 0]
            sc[:, at] = (q[:, None] * k[at][None]).sum(-1) * SCALE
            nan = (torch.isnan(sc) | (sc == INF)).any(1) | (sc == -INF).all(1)
            w = torch.softmax(torch.where(nan[:, None], torch.zeros_like(sc), sc), dim=1)
            v = clean[:m, :b.dv]
            o = w @ v
            o[:, (~fine[:m, :b.dv]).any(0)] = NAN
            o[nan] = NAN
            out[:, r] = o
            # attend64's bound
            size = (q.abs() @ clean[:m].abs().t() * SCALE).max(dim=1).values
            d = size * (b.dk + 1) * 2.0 ** -24 + (size * u16 if b.q.dtype == torch.float32 else 0.0)
            rel = 2 * torch.expm1(d) + 2 * u16 + m * 2.0 ** -32 + u16 + 2.0 ** -20 + (u16 if dst_type == torch.float16 else 2.0 ** -24)
            tol[:, r] = rel[:, None] * (w @ v.abs())
            r += 1
    return out, tol + 2.0 ** -24


def check(b, got, name=""):
    want, tol = definition(b, got.dtype)
    g = got[:, :b.rows].double()
    bad, ref = torch.isnan(g), torch.isnan(want)
    assert ref.any() and not ref.all(), "the case says nothing"
    assert torch.equal(bad, ref), (name, "NaN where there is none:", int((bad & ~ref).sum()), "none where there is:", int((ref & ~bad).sum()))
    off = torch.where(ref, 0.0, (g - want).abs() / tol)
    print(f"{name} {int(ref.sum())} NaN of {ref.numel()}, worst error / bound {float(off.max()):.3f}", flush=True)
    assert float(off.max()) <= 1.0, name
    assert (got[:, b.rows:] == 7.0).all()


def plant(b, seq, key, cols, value):
    """`value` in some columns of a request's key.  In 8 bits an infinity is a product past f16's largest value, beside zeros
    in the rest of its block, a NaN a block's scale."""
    cell = int(b.table[seq, key // b.page]) * b.page + key % b.page
    if b.cache == "f16":
        b.kc[cell, cols] = value
        return
    blocks = b.kc.blocks[cell].unflatten(-1, (-1, 34))
    for c in cols:
        blk = blocks[c // 32]
        if math.isnan(value):
            blk[0], blk[1] = 0, 0x7e
        else:
            blk[:] = 0
            blk[:2] = torch.tensor([600.0], dtype=torch.float16).view(torch.uint8).to(blk.device)
            blk[2 + c % 32] = 127 if value > 0 else 129      # -127
    b.values[cell] = _values(b.kc.blocks[cell])


def _values(row):
    from paged_util import q8_f16
    return q8_f16(row[None])[0]


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_the_oracle(cache):
    """definition() against the formula, product by product, on the host; attend64 where everything is finite."""
    b = Batch("cpu", [3, 20], [4, 1], 16, dk=320, H=3, cache=cache, seed=1, poison=1.0)
    want, tol = attend64(b)
    got, tol2 = definition(b)
    assert torch.equal(got, want) and torch.allclose(tol, tol2, rtol=1e-9)
    plant(b, 0, 5, [7], INF)
    plant(b, 0, 6, [290], -INF)
    plant(b, 1, 0, [3], -INF)
    plant(b, 1, 9, [100], INF)
    got, _ = definition(b)
    r = 0
    for s, (p, n) in enumerate(zip(b.past_l, b.new_l)):
        for i in range(n):
            j = torch.arange(p + i + 1)
            k = b.values[b.table[s, j // 16].long() * 16 + j % 16].double()
            w = torch.softmax((b.q[r].double()[:, None] * k[None]).sum(-1) * SCALE, dim=1)
            ref = (w[:, :, None] * k[None, :, :256]).sum(1)
            assert torch.equal(torch.isnan(ref), torch.isnan(got[:, r]))
            assert torch.allclose(ref, got[:, r], rtol=1e-9, equal_nan=True)
            r += 1


# past, new, H, and (request, key, columns, value): columns up to 255 are V's too
SEEN_BY_ALL = [([70, 130], [1, 1], 32, [(0, 3, [5], INF), (1, 70, [300], -INF)]),
               ([700], [1], 40, [(0, 100, [17], INF), (0, 650, [255, 31], -INF)]),
               ([20], [1], 16, [(0, 7, [0], -INF)])]
SEEN_BY_SOME = [([60], [9], 32, [(0, 66, [5], INF)]), ([60], [9], 32, [(0, 67, [290], -INF)]), ([60], [9], 32, [(0, 66, [64, 200], INF)]),
                ([60], [9], 32, [(0, 67, [130], NAN)]), ([0], [70], 40, [(0, 33, [255], -INF), (0, 50, [0], INF)]),
                ([500], [3], 16, [(0, 501, [8], -INF), (0, 502, [319], INF)]), ([5], [100], 1, [(0, 40, [9], INF), (0, 80, [33], -INF)]),
                ([20], [5], 16, [(0, 22, [12], INF)]), ([120, 8], [8, 3], 8, [(0, 126, [40], INF), (1, 9, [50], -INF)])]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(SEEN_BY_ALL) + len(SEEN_BY_SOME)))
@pytest.mark.parametrize("cache,q_type,dst", [("f16", torch.float16, torch.float32), ("f16", torch.float32, torch.float16),
                                              ("q8", torch.float32, torch.float32), ("q8", torch.float16, torch.float16)])
def test_blocks_of_32(dev, case, cache, q_type, dst):
    past, new, H, odd = (SEEN_BY_ALL + SEEN_BY_SOME)[case]
    for dk in (320, 576):
        b = Batch(dev, past, new, 16, dk=dk, H=H, cache=cache, q_type=q_type, seed=case, pad=1, poison=1.0)
        for at in odd:
            plant(b, *at)
        check(b, b.run(b.out(dst)), f"{dk} {past} {new}")


@pytest.mark.gpu
@pytest.mark.parametrize("past,new,H,odd", [
    ([9000], [9], 40, [(0, 9004, [5], INF)]), ([9000], [9], 40, [(0, 9003, [300], -INF), (0, 9006, [77, 78], INF)]),
    ([9000], [9], 40, [(0, 5000, [5], INF)]), ([0], [700], 40, [(0, 333, [200], -INF), (0, 600, [310], INF)]),
    ([8190], [14], 32, [(0, 8197, [255], INF)]), ([8190], [14], 32, [(0, 8198, [1], NAN)]),
    ([7] * 40, [60] * 40, 32, [(2, 30, [10], INF), (39, 65, [100], -INF), (20, 66, [290], INF)])])
@pytest.mark.parametrize("cache,q_type,dst", [("f16", torch.float16, torch.float32), ("f16", torch.float32, torch.float16),
                                              ("q8", torch.float32, torch.float32), ("q8", torch.float16, torch.float16)])
def test_blocks_of_128(dev, past, new, H, odd, cache, q_type, dst):
    for dk in (320, 576) if len(past) == 1 and cache == "f16" else (320,):
        b = Batch(dev, past, new, 16, dk=dk, H=H, cache=cache, q_type=q_type, seed=len(odd), pad=1, poison=1.0)
        assert sum(-(-n * H // 32) * ((p + n // 2) // 64 + 1) for p, n in zip(past, new)) > 1600
        for at in odd:
            plant(b, *at)
        check(b, b.run(b.out(dst)), f"{dk} {past} {new}")


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_behind_shared_cells(dev, cache):
    """In the shared cells, which all see, and in a request's own ones."""
    b = Batch(dev, [2560 + 7 * i for i in range(64)], [1 + i % 3 for i in range(64)], 16, dk=320, H=16, cache=cache, prefix=2560, share=64, seed=2, pad=1, poison=1.0)
    plant(b, 0, 1000, [90], INF)
    plant(b, 11, 2560 + 78, [20], -INF)
    check(b, b.run())


# cells whose tile holds nothing else that a row sees, or whole tiles of them: a piece of the row's keys without a score
ALONE = [([64], [1], 32, [(0, 64, [5], INF)]), ([64, 30], [1, 1], 32, [(0, 64, [290], INF), (1, 3, [300], INF)]),
         ([60], [9], 32, [(0, 64, [5], -INF)]), ([60, 640], [9, 1], 8, [(0, 64, [77, 130], INF), (1, 640, [9], INF)]),
         ([300], [1], 16, [(0, k, [70], INF) for k in range(64, 128)]), ([300, 9], [2, 1], 40, [(0, k, [300], INF) for k in range(128, 192)]),
         ([0, 20], [1, 1], 32, [(0, 0, [3], INF)]), ([0, 50], [3, 1], 32, [(0, 0, [300], -INF), (0, 1, [301], INF)]),
         ([30, 5], [1, 2], 16, [(0, k, [280], INF) for k in range(31)])]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(ALONE)))
@pytest.mark.parametrize("cache,q_type,dst", [("f16", torch.float16, torch.float32), ("q8", torch.float32, torch.float16)])
def test_pieces_without_a_score(dev, case, cache, q_type, dst):
    past, new, H, odd = ALONE[case]
    for dk in (320, 576):
        b = Batch(dev, past, new, 16, dk=dk, H=H, cache=cache, q_type=q_type, seed=case, pad=1, poison=1.0)
        if case == 8:                                        # every key of a request -inf for half its heads: 0 / 0
            b.q[0, ::2, 280] = b.q[0, ::2, 280].abs()
        for at in odd:
            plant(b, *at)
        check(b, b.run(b.out(dst)), f"{dk} {past} {new}")


@pytest.mark.gpu
@pytest.mark.parametrize("past,new,H,odd", [
    ([9024], [9], 40, [(0, 9024, [5], INF)]), ([9024], [9], 40, [(0, k, [k % 256], INF) for k in range(9024, 9030)]),
    ([7] * 40, [60] * 40, 32, [(i, 64, [100], -INF) for i in range(40)]),
    ([9024], [9], 40, [(0, k, [7], INF) for k in range(64 * 16, 64 * 30)]), ([0], [700], 40, [(0, 0, [300], INF), (0, 64, [7], INF), (0, 640, [9], -INF)])])
@pytest.mark.parametrize("cache,q_type,dst", [("f16", torch.float16, torch.float32), ("q8", torch.float32, torch.float16)])
def test_pieces_without_a_score_in_blocks_of_128(dev, past, new, H, odd, cache, q_type, dst):
    b = Batch(dev, past, new, 16, dk=320, H=H, cache=cache, q_type=q_type, seed=len(odd), pad=1, poison=1.0)
    assert sum(-(-n * H // 32) * ((p + n // 2) // 64 + 1) for p, n in zip(past, new)) > 1600
    for at in odd:
        plant(b, *at)
    check(b, b.run(b.out(dst)), f"{past} {new}")


@pytest.mark.gpu
@pytest.mark.parametrize("absent", [(0, 8), (4, 70), (0, 69)])
def test_without_a_score_and_without_a_page(dev, absent):
    """Keys whose pages are none are no keys: a row that sees only such gets zeros, one that sees others of score -inf NaN."""
    b = Batch(dev, [1100, 20], [3, 1], 16, dk=320, H=16, seed=5, pad=1, poison=1.0)
    b.q[:, :, 300] = b.q[:, :, 300].abs() + 0.1
    for k in range(1103):
        plant(b, 0, k, [300], -INF)
    b.table[0, absent[0]:absent[1]] = -1
    got = b.run()
    if absent == (0, 69):                                    # 1,104 cells: all of them
        assert (got[:, :3] == 0).all()
    else:
        assert torch.isnan(got[:, :3]).all()
    assert torch.isfinite(got[:, 3]).all() and (got[:, 4] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["nan", "inf", "column"])
@pytest.mark.parametrize("past,new,H", [([0, 30], [300, 2], 32), ([9000, 10], [9, 3], 40), ([5, 40], [90, 1], 1)])
def test_a_request_full_of_them(dev, what, past, new, H):
    """Every cell of a request NaN, infinite throughout, or infinite in one column."""
    b = Batch(dev, past, new, 16, dk=320, H=H, seed=H, pad=1, poison=1.0)
    j = torch.arange(past[0] + new[0], device=dev)
    cells = b.table[0, j // 16].long() * 16 + j % 16
    if what == "nan":
        b.kc[cells] = NAN
    elif what == "inf":
        b.kc[cells] = torch.where(b.kc[cells] > 0, INF, -INF).half()
    else:
        b.kc[cells, 7] = INF
    check(b, b.run(), what)
