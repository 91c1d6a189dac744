"""Compiled calls under torch's dispatch modes: what a mode makes of a call's new tensors stays with that call."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

import aubier_amd as A
from aubier_amd import ops

pytestmark = pytest.mark.gpu

FIRST_CALL = """
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    import aubier_amd as A
    from aubier_amd import ops

    assert ops._calls()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")

    def pages():
        return A.ggml_m4_pages(i32(0, 5), i32(3, 1), i32(4, 5, 6, 7), torch.full((2, 3), -1, dtype=torch.int32, device="cuda"), 16, 4)

    with FakeTensorMode():
        x = torch.empty((3, 64), device="cuda")
        for call in (lambda: A.ggml_m4_rows_i8(x), lambda: A.ggml_m4_norm(x, x[0], 1e-6)):
            try:
                call()
            except (A.MlaM4Error, RuntimeError):
                pass
            else:
                raise SystemExit("a call without memory was taken")
    x = torch.arange(-96, 96, device="cuda").float().view(3, 64)
    q, s = A.ggml_m4_rows_i8(x)
    top = x.abs().amax(1, keepdim=True)
    want = torch.sign(x) * torch.floor((x.double() * 127 / top).abs() + 0.5)
    assert q.device == x.device and torch.equal(q.double(), want.double()) and torch.allclose(s, top[:, 0] / 127, rtol=2.0 ** -23, atol=0)
    slot, pos, used = pages()
    assert pos.device == x.device and pos.tolist() == [0, 1, 2, 5]
    print("whole")
"""


def test_first_call_of_a_process_under_a_fake_mode(dev):
    """It is refused, and the calls behind it are made as ever."""
    r = subprocess.run([sys.executable, "-c", textwrap.dedent(FIRST_CALL)], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True,
                       timeout=100)
    assert r.returncode == 0 and r.stdout.strip().endswith("whole"), r.stdout[-1000:] + r.stderr[-2000:]


def test_a_mode_sees_new_tensors(dev):
    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.new = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func is torch.ops.aten.empty.memory_format:
                self.new.append(out.data_ptr())
            return out

    assert ops._calls()
    x = torch.randn((5, 64), device=dev)
    want = A.ggml_m4_rows_i8(x)
    with Seen() as mode:
        got = A.ggml_m4_rows_i8(x)
    assert mode.new == [t.data_ptr() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = A.ggml_m4_rows_i8(x)
    assert len(mode.new) == 2 and all(torch.equal(a, b) for a, b in zip(again, want))
