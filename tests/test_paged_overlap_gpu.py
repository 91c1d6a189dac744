"""Two captured calls that share a workspace and replay at once, which their user must not do: results are anything, but nothing
outside the calls' own memory is written, both end, and a call by itself is right afterwards.  What a call finds in its
workspace between its two launches is brought into range, so this is an ordinary run."""
import pytest
import torch

import aubier_amd as A

from paged_util import Batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shapes", ["long and short", "shared and not", "wide and narrow"])
def test_two_graphs_on_one_workspace(dev, shapes):
    if shapes == "long and short":
        bs = [Batch(dev, [9000, 50, 3000], [1, 1, 1], 16, dk=320, H=32, seed=1), Batch(dev, [70] * 40, [1] * 40, 16, dk=320, H=16, seed=2, pad=30)]
    elif shapes == "shared and not":
        bs = [Batch(dev, [2560 + 7 * i for i in range(64)], [1] * 64, 16, dk=320, H=16, prefix=2560, share=64, seed=3),
              Batch(dev, [500 + i for i in range(64)], [1] * 64, 16, dk=320, H=16, prefix=0, share=2, seed=4)]
    else:
        bs = [Batch(dev, [4000], [40], 16, dk=320, H=40, seed=5), Batch(dev, [8000, 20], [1, 2], 16, dk=320, H=8, seed=6)]
    guard = 1 << 16
    need = max(A.kqkv_paged_workspace_bytes(b.kc, b.q, b.past, b.out(), b.prefix) for b in bs)
    room = torch.full((need + 2 * guard,), 0xab, dtype=torch.uint8, device=dev)
    ws = room[guard:guard + need]
    rooms, outs, graphs, streams = [], [], [], []
    for b in bs:
        n = b.H * b.nt * b.dv
        rooms.append(torch.full((n + 2 * guard,), 7.0, device=dev))
        outs.append(rooms[-1][guard:guard + n].view(b.H, b.nt, b.dv))
    torch.cuda.synchronize()
    for b, out in zip(bs, outs):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            b.run(out, workspace=ws)
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            for _ in range(8):
                b.run(out, workspace=ws)
        torch.cuda.synchronize()
        streams.append(st)
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert (room[:guard] == 0xab).all() and (room[-guard:] == 0xab).all()
    for b, r, out, g in zip(bs, rooms, outs, graphs):
        assert (r[:guard] == 7.0).all() and (r[-guard:] == 7.0).all()
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(b, out, shapes)
