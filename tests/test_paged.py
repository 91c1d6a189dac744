"""CPU tests of the paged operators' contracts: what their host checks refuse, without a launch."""
import ctypes

import pytest
import torch

import aubier_amd as A
from aubier_amd import ops


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


RP = dict(freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, eps=1e-6, n_ctx_orig=4096)


def pages(**kw):
    a = dict(past=i32(4), n_new=i32(4), free=i32(9), table=i32(4, 8), page_size=64, slot=torch.zeros(10, dtype=torch.int64),
             pos=i32(10), used=i32(2))
    a.update(kw)
    return A.supports_pages(**a)


def test_supports_pages():
    assert pages() and pages(free=i32(0)) and pages(table=i32(4, 30)[:, 2:9]) and pages(page_size=16) and pages(page_size=65536)
    for bad in (dict(n_new=i32(5)), dict(past=i32(4).long()), dict(past=i32(8)[::2]), dict(table=i32(3, 8)), dict(table=i32(4, 8).float()),
                dict(table=i32(8, 4).t()), dict(page_size=8), dict(page_size=48), dict(page_size=0), dict(page_size=-64),
                dict(page_size=131072), dict(slot=i32(10)), dict(pos=i32(9)), dict(used=i32(3)), dict(free=i32(9).float()),
                dict(free=i32(18)[::2]), dict(slot=torch.zeros(0, dtype=torch.int64), pos=i32(0)),
                dict(past=i32(4097), n_new=i32(4097), table=i32(4097, 1)), dict(table=i32(4, 70000), page_size=65536),
                dict(slot=torch.zeros(70000, dtype=torch.int64), pos=i32(70000))):
        assert not pages(**bad), bad


def rows(**kw):
    a = dict(x=torch.zeros(5, 576), kv_norm=torch.zeros(512), kcache=torch.zeros((20, 576), dtype=torch.float16),
             slot=torch.zeros(5, dtype=torch.int64), pos=i32(5), rope=A.rope_params(n_dims=64, **RP), out=torch.zeros(5, 576))
    a.update(kw)
    return A.supports_kvrows(**a)


def q8(n, ne0):
    return A.Q8_0(torch.zeros(n, ne0 // 32 * 34, dtype=torch.uint8), ne0)


def test_supports_kvrows():
    assert rows() and rows(x=torch.zeros((5, 576), dtype=torch.float16)) and rows(kcache=q8(20, 576)) and rows(out=None)
    for bad in (dict(x=torch.zeros(5, 575)), dict(x=torch.zeros(5, 577)[:, :576]), dict(x=torch.zeros(576, 5).t()),
                dict(x=torch.zeros((5, 576), dtype=torch.int32)), dict(kv_norm=torch.zeros(511)), dict(kv_norm=torch.zeros(513)[1:]),
                dict(kcache=torch.zeros(20, 576)), dict(kcache=q8(20, 320)), dict(kcache=torch.zeros((20, 320), dtype=torch.float16)),
                dict(slot=i32(5)), dict(slot=torch.zeros(4, dtype=torch.int64)), dict(pos=torch.zeros(5)), dict(out=torch.zeros(4, 576)),
                dict(out=torch.zeros((5, 576), dtype=torch.float16)), dict(rope=A.rope_params(n_dims=48, **RP)),
                dict(rope=A.rope_params(n_dims=0, **RP)), dict(rope=A.rope_params(n_dims=576, **RP)),
                dict(rope=A.rope_params(n_dims=64, **{**RP, "eps": float("nan")})),
                dict(rope=A.rope_params(n_dims=64, **{**RP, "freq_base": float("inf")})),
                dict(x=torch.zeros(5, 2048), out=torch.zeros(5, 2048), kv_norm=torch.zeros(1984),
                     kcache=torch.zeros((20, 2048), dtype=torch.float16))):
        assert not rows(**bad), bad


def test_supports_kvrows_row_limit():
    for n, ok in ((1 << 24, True), ((1 << 24) + 1, False)):
        # (nothing is read: the pages of these are never touched)
        assert ok == rows(x=torch.empty((n, 64), dtype=torch.float16), kv_norm=torch.zeros(32), kcache=torch.zeros((20, 64), dtype=torch.float16),
                          slot=torch.empty(n, dtype=torch.int64), pos=torch.empty(n, dtype=torch.int32), out=None,
                          rope=A.rope_params(n_dims=32, **RP))


def test_attention_workspace_stays_bounded():
    """Without shared cells the records number two per workgroup whatever the batch; what grows is 8 bytes a row."""
    kc, lens = torch.zeros((64, 576), dtype=torch.float16), i32(64)
    need = {}
    for nt in (1, 8000):
        for prefix in (None, i32(2)):
            q, out = torch.empty((nt, 16, 576), dtype=torch.float16), torch.empty((16, nt, 512), dtype=torch.float16)
            need[nt, prefix is not None] = A.kqkv_paged_workspace_bytes(kc, q, lens, out, prefix)
    record = 128 * (8 + 2 * 512)
    assert 512 * record <= need[1, False] <= need[8000, False] <= 512 * record + 9 * 16 * 8000
    assert need[8000, False] + 2 * 1000 * record <= need[8000, True] <= need[8000, False] + (256 + 2 * 1000 + 64) * record


def attn(dk=576, dv=512, **kw):
    a = dict(kcache=torch.zeros((640, dk), dtype=torch.float16), q=torch.zeros((3, 8, dk), dtype=torch.float16), past=i32(2), n_new=i32(2),
             table=i32(2, 9), page_size=64, prefix=None, out=torch.zeros((8, 3, dv)))
    a.update(kw)
    return A.supports_kqkv_paged(**a)


def test_supports_kqkv_paged():
    h = torch.float16
    assert attn() and attn(320, 256) and attn(prefix=i32(2)) and attn(kcache=q8(640, 576)) and attn(q=torch.zeros(3, 8, 576))
    assert attn(out=torch.zeros((8, 3, 512), dtype=h)) and attn(q=torch.zeros((3, 9, 600), dtype=h)[:, 1:, :576])
    for bad in (dict(out=torch.zeros(8, 3, 256)), dict(out=torch.zeros(8, 2, 512)), dict(out=torch.zeros((8, 3, 512), dtype=torch.int32)),
                dict(out=torch.zeros(3, 8, 512).transpose(0, 1)), dict(q=torch.zeros((3, 8, 320), dtype=h)), dict(q=torch.zeros((3, 8, 580), dtype=h)[:, :, :576]),
                dict(kcache=torch.zeros(640, 576)), dict(kcache=torch.zeros((640, 580), dtype=h)[:, :576]), dict(kcache=torch.zeros((63, 576), dtype=h)),
                dict(prefix=i32(3)), dict(prefix=torch.zeros(2)), dict(n_new=i32(3)), dict(table=i32(3, 9)), dict(page_size=63), dict(page_size=8),
                dict(dk=640, dv=512), dict(q=torch.zeros((3, 1025, 576), dtype=h), out=torch.zeros(1025, 3, 512))):
        assert not attn(**bad), bad


def test_supports_kqkv_paged_work_limit():
    """The places on the line of work are whole numbers in 64-bit floating point."""
    q, out = torch.empty((4096, 1024, 320), dtype=torch.float16), torch.empty((1024, 4096, 256), dtype=torch.float16)   # (never touched)
    kc = torch.zeros((65536, 320), dtype=torch.float16)
    for pages, ok in ((1 << 12, True), ((1 << 12) + 1, False), (1 << 14, False)):
        assert ok == attn(320, 256, q=q, out=out, kcache=kc, table=i32(2, pages), page_size=65536)


def test_entry_points_reject_before_launching():
    """Refused by the host's checks: nothing is launched, no pointer is followed."""
    lib, P = A.load_library(), lambda t: ctypes.byref(ops.view(t))  # noqa: E731
    p, n, t = i32(2), i32(2), i32(2, 4)
    s, o, u = torch.zeros(3, dtype=torch.int64), i32(3), i32(2)
    assert lib.mla_m4_pages(None, P(n), P(i32(3)), P(t), 64, P(s), P(o), P(u), None) == -1
    assert lib.mla_m4_pages(P(p), P(n), P(i32(3)), P(t), 60, P(s), P(o), P(u), None) == -6
    assert lib.mla_m4_pages(P(p), P(n), P(i32(3)), P(t), 64, P(s), P(o), None, None) == -1
    x, w, kc = torch.zeros(3, 320), torch.zeros(256), torch.zeros((9, 320), dtype=torch.float16)
    rp = A.rope_params(n_dims=64, **RP)
    assert lib.mla_m4_kvrows(P(x), P(w), P(kc), P(s), P(o), None, None, None) == -1
    assert lib.mla_m4_kvrows(P(x), P(w), P(kc), P(o), P(o), ctypes.byref(rp), None, None) == -2
    kc, q, out = torch.zeros((640, 320), dtype=torch.float16), torch.zeros(3, 8, 320), torch.zeros(8, 3, 256)
    nan = ctypes.c_float(float("nan"))
    args = (P(kc), P(q), P(p), P(n), P(t))
    assert lib.mla_m4_kqkv_paged(*args, 64, None, nan, P(out), None, 0, None) == -6
    assert lib.mla_m4_kqkv_paged(*args, 65, None, ctypes.c_float(1.0), P(out), None, 0, None) == -6
    assert lib.mla_m4_kqkv_paged(P(kc), P(q), P(p), P(n), None, 64, None, ctypes.c_float(1.0), P(out), None, 0, None) == -1


@pytest.mark.parametrize("call", ["pages", "rows", "attn"])
def test_host_tensors_are_refused(call):
    """The Python mirror refuses tensors that are not on one GPU (their pointers mean nothing to a kernel)."""
    with pytest.raises(A.MlaM4Error):
        if call == "pages":
            A.ggml_m4_pages(i32(2), i32(2), i32(3), i32(2, 4), 64, 5)
        elif call == "rows":
            A.ggml_m4_kvrows(torch.zeros(3, 320), torch.zeros(256), torch.zeros((9, 320), dtype=torch.float16),
                             torch.zeros(3, dtype=torch.int64), i32(3), A.rope_params(n_dims=64, **RP))
        else:
            A.ggml_m4_kqkv_paged(torch.zeros((640, 320), dtype=torch.float16), torch.zeros(3, 8, 320), i32(2), i32(2), i32(2, 4), 64, 1.0)
