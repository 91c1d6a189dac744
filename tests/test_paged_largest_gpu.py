"""The largest batches that the page bookkeeping and the attention take: 65,535 rows in one request and in thousands, and contexts whose tables
list the same pages again and again (a table may), so that positions pass 2^24 where the pool is small."""
import pytest
import torch

import aubier_amd as A

from paged_util import Batch, attend64

pytestmark = pytest.mark.gpu


def rows_of(b, rows):
    """Rows of a batch against 64 bits: attend64 over a batch of those tokens alone, one request each."""
    starts = [0]
    for n in b.new_l:
        starts.append(starts[-1] + n)
    pick = []
    for r in rows:
        s = max(i for i in range(len(b.new_l)) if starts[i] <= r and b.new_l[i] > 0)
        pick.append((s, b.past_l[s] + r - starts[s]))
    few = Batch.__new__(Batch)
    few.__dict__.update(b.__dict__)
    few.past = torch.tensor([p for _, p in pick], dtype=torch.int32)
    few.new = torch.ones(len(rows), dtype=torch.int32)
    few.table, few.q, few.rows, few.nt = b.table[[s for s, _ in pick]], b.q[rows], len(rows), len(rows)
    return attend64(few)


@pytest.mark.parametrize("past,new,H", [([0], [65535], 1), ([3], [65535], 2), ([(7 * i) % 50 for i in range(4095)], [16] * 4095, 3)])
def test_most_rows(dev, past, new, H):
    b = Batch(dev, past, new, 64, dk=320, H=H, seed=len(past), poison=1.0)
    got = b.run(b.out(torch.float16))
    assert torch.isfinite(got).all()
    rows = [0, 1, 63, 64, 127, 128, 12345, 32767, 32768, 40001, b.rows - 129, b.rows - 2, b.rows - 1]
    want, tol = rows_of(b, rows)
    assert ((got[:, rows].double() - want).abs() <= tol + 2.0 ** -11 * want.abs()).all()      # (an f16 result)


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_positions_past_24_bits(dev, cache):
    """A table of 4,200 times the same 64 pages of 64 cells, 17.2 million cells in whole rounds: the softmax over them is that over
    one round."""
    pages, rounds = 64, 4200
    b = Batch(dev, [pages * 64 - 1], [1], 64, dk=320, H=8, cache=cache, seed=1, poison=1.0, spare=0)
    once, tol = attend64(b)
    b.table = b.table.repeat(1, rounds).contiguous()
    b.past[0] = pages * 64 * rounds - 1
    assert int(b.past[0]) > 2 ** 24
    got = b.run().double()
    # a workgroup's piece is 1,050 tiles: 16 additions a tile to a lane's l, 4 to each of o, each off by at most 2^-24 of the
    # sum, so numerator and denominator by (16,800 + 4,200) 2^-24 of sum w |v| <= max |v| at most
    v = b.values[:, :256].double().abs().max()
    assert ((got - once).abs() <= tol + 21000 * 2.0 ** -24 * v).all()


def test_slots_of_the_largest_batch(dev):
    """65,535 rows over 4,096 requests through the page bookkeeping."""
    n = 4096
    past = torch.arange(n, dtype=torch.int32, device=dev) % 100
    new = torch.full((n,), 16, dtype=torch.int32, device=dev)
    new[-1] = 15
    table = torch.full((n, 8), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(n * 8, device=dev).to(torch.int32)
    held = (past.long() + 15) // 16
    at = torch.arange(8, device=dev)[None] < held[:, None]
    table[at] = torch.arange(int(held.sum()), dtype=torch.int32, device=dev) + n * 8
    first = table.clone()
    slot, pos, used = A.ggml_m4_pages(past, new, free, table, 16, 65535)
    rows = torch.arange(65535, device=dev)
    req = rows // 16
    p = past[req].long() + rows % 16
    assert torch.equal(pos.long(), p) and used.tolist() == [int(((past.long() + new + 15) // 16 - held).sum()), 65535]
    assert torch.equal(slot, table[req, p // 16].long() * 16 + p % 16) and (slot >= 0).all()
    assert torch.equal(table[at], first[at]) and torch.unique(slot).numel() == 65535
