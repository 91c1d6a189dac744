"""What a planner asks before it allocates (CPU): descriptors without data are sized as those with it."""
import ctypes

import torch

import aubier_amd as A
from aubier_amd import ops


def test_workspace_of_a_prefix_that_is_not_allocated():
    lib, i32 = A.load_library(), torch.int32
    kc, past = torch.zeros((64, 576), dtype=torch.float16), torch.zeros(64, dtype=i32)
    q, out = torch.empty((64, 32, 576), dtype=torch.float16), torch.empty((32, 64, 512), dtype=torch.float16)
    prefix = torch.zeros(2, dtype=i32)

    def need(prefix, bare):
        views = [ops.view(t) for t in (kc, q, past, prefix, out)]
        for v in views if bare else ():
            if v is not None:
                v.data = None
        return lib.mla_m4_kqkv_paged_workspace_bytes(*(ctypes.byref(v) if v is not None else None for v in views))

    assert need(prefix, True) == need(prefix, False) > need(None, True) == need(None, False) > 0
