"""KQKV over pages at the edges of a batch, where the shared cells are taken once: more requests than the prefix names or than
a workgroup has threads, tokens past the room for rows, tables that end with the shared cells; and batches most of whose
requests are idle."""
import pytest
import torch

from paged_util import Batch, attend64, check
from test_paged_shared_gpu import N, many

pytestmark = pytest.mark.gpu


def followed_once(b, sharers, first=0):
    """As test_paged_shared_gpu's run_followed_once, over `sharers` requests whatever the prefix says."""
    whole, table = int(b.prefix[0]) // 64 * 4, b.table
    b.table = table.clone()
    for s in range(sharers):
        if s != first:
            b.table[s, :whole] = -1
    got = b.run()
    b.table = table
    return got


@pytest.mark.parametrize("requests", [N + 1, 1000, 2 ** 31 - 1])
def test_prefix_of_more_requests_than_there_are(dev, requests):
    b = many(dev, dk=320, H=16, seed=11, pad=1)
    b.prefix[1] = requests
    check(b, followed_once(b, N), f"{requests}")


@pytest.mark.parametrize("n,H", [(257, 16), (600, 3), (1500, 1)])
@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_more_sharers_than_threads(dev, n, H, cache):
    """Several requests to a thread, some without tokens, others behind them that do not share."""
    new = [(1, 0, 2, 1, 0)[i % 5] for i in range(n)]
    b = many(dev, dk=320, H=H, n=n, prefix=640, behind=90, new=new, extra=[(100, 2), (0, 0), (7, 1)], cache=cache, seed=n, pad=2)
    check(b, followed_once(b, n), f"{n} requests")


@pytest.mark.parametrize("nt", [100, 64, 3])
def test_sharers_tokens_past_the_rows(dev, nt):
    """Rows end inside a sharer's tokens (100) or between two sharers' (64: 21 requests of 3 tokens and one of 1)."""
    new = [3] * 21 + [1] + [3] * (N - 22)
    b = many(dev, dk=320, H=40, new=new, seed=12)
    want, tol = attend64(b)
    b.q, b.nt = b.q[:nt].contiguous(), nt
    got = followed_once(b, N) if nt > 3 else b.run()         # (three rows do not make sharing pay)
    assert ((got.double() - want[:, :nt]).abs() <= tol[:, :nt]).all()


@pytest.mark.parametrize("cache", ["f16", "q8"])
def test_tables_that_end_with_the_shared_cells(dev, cache):
    """Every sharer holds as many cells as its table lists, all of them shared: nothing is left that is its own."""
    b = Batch(dev, [2559] * N, [1] * N, 16, dk=320, H=16, prefix=2560, share=N, cache=cache, seed=13, pad=1)
    assert b.table.shape[1] * 16 == 2560
    b.past += 1 + torch.arange(N, dtype=torch.int32, device=dev)
    check(b, followed_once(b, N), "all cells shared")


@pytest.mark.parametrize("n_seq,every", [(4096, 400), (4096, 1365), (900, 250)])
@pytest.mark.parametrize("H", [8, 128])
def test_hundreds_of_idle_requests_between(dev, n_seq, every, H):
    """Stretches of the work that go on from one request to the next with tokens, past hundreds without."""
    live = set(range(every // 2, n_seq, every)) | {n_seq - 1}
    past = [(900 if i % 2 else 130) + i % 77 if i in live else i % 3 for i in range(n_seq)]
    b = Batch(dev, past, [1 + i % 2 if i in live else 0 for i in range(n_seq)], 16, dk=320, H=H, seed=every, pad=1)
    check(b, b.run(), f"{len(live)} of {n_seq}")
    b = Batch(dev, [p * 9 if i in live else 0 for i, p in enumerate(past)], [1 if i in live else 0 for i in range(n_seq)], 64, dk=320, H=16, seed=every)
    check(b, b.run(), "longer")
