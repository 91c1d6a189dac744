"""Every form of the int8 product at the edges of what it is given, against exact integer sums (test_mul_i8_forms.py: that these shapes
reach them)."""
import ctypes

import pytest
import torch

import aubier_amd as A

from mul_forms_util import SHAPES
from test_mul_i8_gpu import check, make

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


@pytest.mark.parametrize("form,cut,shape", [(f, cut, s) for (f, cut), shapes in SHAPES.items() for s in shapes])
def test_form(dev, form, cut, shape):
    """Given a workspace of just its size and none at all: the same bits, and nothing written beside the result or the workspace;
    results in rows of their own and at odd places of wider ones."""
    rows, n, _ = shape
    a = make(dev, *shape, 11)
    lib, stream = A.load_library(), torch.cuda.current_stream().cuda_stream
    need = A.mul_i8_workspace_bytes(a[0], a[2])
    assert need > 0 or not cut
    for dtype in (F32, F16):
        whole = torch.full((rows, n), 7.0, dtype=dtype, device=dev)
        v = [A.view(t) for t in (*a, whole)]
        assert lib.mla_m4_mul_i8(*(ctypes.byref(t) for t in v), None, 0, stream) == 0
        check(a, whole, (form, "no workspace"))
        work = torch.full((need + 4096,), 99, dtype=torch.uint8, device=dev)
        for pad in (0, 3):
            buf = torch.full((rows, n + 2 * pad), 7.0, dtype=dtype, device=dev)
            out = buf[:, pad:pad + n]
            v = [A.view(t) for t in (*a, out)]
            assert lib.mla_m4_mul_i8(*(ctypes.byref(t) for t in v), work.data_ptr(), need, stream) == 0
            assert torch.equal(out, whole), (form, pad)
            assert (buf[:, :pad] == 7).all() and (buf[:, pad + n:] == 7).all() and (work[need:] == 99).all()
        if cut:
            assert (work[:need].view(torch.int32) != 0x63636363).any()


@pytest.mark.parametrize("form", ["SPLIT11", "SPLIT128"])
def test_cut_on_two_streams(dev, form):
    """A workspace each, at once; and a captured call replayed with the program's own work between."""
    shape = SHAPES[(form, True)][-1]
    a, b = make(dev, *shape, 12), make(dev, *shape, 13)
    want = A.ggml_m4_mul_i8(*a), A.ggml_m4_mul_i8(*b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for s, args, out in zip(streams, (a, b), got):
            with torch.cuda.stream(s):
                out.append(A.ggml_m4_mul_i8(*args))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(y, w) for y in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        y = A.ggml_m4_mul_i8(*a)
    for i in range(4):
        a[3].mul_(-0.5)
        w = A.ggml_m4_mul_i8(*a)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, w), i
