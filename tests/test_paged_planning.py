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


def test_the_rows_of_one_head_end_inside_their_span():
    """128 rows of q are reached by 32-bit offsets, the last one's end too; a single head's stride says nothing of its length."""
    i32, h = torch.int32, torch.float16
    room = torch.empty((1 << 30) + (1 << 12), dtype=h)                           # (never touched)
    kc, past, table, out = torch.zeros((640, 576), dtype=h), torch.zeros(2, dtype=i32), torch.zeros((2, 9), dtype=i32), torch.zeros((1, 128, 512))

    def fits(token_bytes, head_bytes):
        q = room.as_strided((128, 1, 576), (token_bytes // 2, head_bytes // 2, 1))
        return A.supports_kqkv_paged(kc, q, past, past, table, 64, None, out)

    assert 127 * 16909296 + 1152 <= 2 ** 31 < 127 * 16909312 + 1152
    for head_bytes in (16, 1152):
        assert fits(16909296, head_bytes) and not fits(16909312, head_bytes)


def test_page_sizes_past_32_bits():
    """Refused, not taken for their lower 32 bits."""
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    for more in (0, 1 << 32, -(1 << 32), 1 << 40):
        assert (more == 0) == A.supports_pages(i32(4), i32(4), i32(9), i32(4, 8), 64 + more, torch.zeros(10, dtype=torch.int64), i32(10), i32(2))
        assert (more == 0) == A.supports_kqkv_paged(torch.zeros((640, 320), dtype=torch.float16), torch.zeros(3, 8, 320), i32(2), i32(2), i32(2, 9), 64 + more,
                                                    None, torch.zeros(8, 3, 256))
