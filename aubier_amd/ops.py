"""Python mirror of aubier's three custom ggml ops, calling the gfx950 kernels through the C ABI
of include/mla_m4.h (aubier_amd/libmla_m4.so).

Names and argument meaning follow the reference's op builders (vendor/llama.cpp/ggml/include/
ggml.h:1524-1586, ggml.c:3405-3539): ``ggml_m4_wkb(w_kb, q_nope)``, ``ggml_m4_kqkv(kcache, q,
mask, kq_scale)`` and the PHASE op's split-K merge ``ggml_m4_phase_merge(part)``.  A contract
violation raises :class:`MlaM4Error` (the ggml glue aborts instead, keeping the FATAL semantics).
There is no CPU path: without the built library every call raises.

Tensors are torch CUDA tensors in row-major order, i.e. with the ggml ``ne[]`` axes reversed:

=============  =========================  ==============================
op / operand   ggml ne (fastest first)    torch shape
=============  =========================  ==============================
W_kb           [d_n, D_v, H]              [H, D_v, d_n]
q_nope         [d_n, H, nt]               [nt, H, d_n] (a strided view is fine)
WKB dst        [D_v, H, nt]               [nt, H, D_v] (a view into Qcur is fine)
kcache         [D_k, n_kv]                [n_kv, D_k]  (f16 or f32)
q (Qcur)       [D_k, H, nt]               [nt, H, D_k]
mask           [n_kv, >= nt]              [>= nt, n_kv]
KQKV dst       [D_v, nt, H]               [H, nt, D_v]
partials       [64 + 16 D_v, S, nt, G]    [G, nt, S, 64 + 16 D_v]   (G = ceil(H / 32) head groups)
=============  =========================  ==============================
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from pathlib import Path
from typing import Optional

import torch

LIB_PATH = Path(__file__).resolve().parent / "libmla_m4.so"

TYPE_F32, TYPE_F16 = 0, 1
PART_HEADS = 32
MAX_SPLITS = 1024


def part_floats(d_v: int, kc_f16: bool = True) -> int:
    """4-byte words per split-K partial block (include/mla_m4.h MLA_M4_PART_FLOATS[_F32])."""
    return 64 + (16 if kc_f16 else 32) * d_v


PHASE_KVWRITE, PHASE_WVB, PHASE_MERGE = 0, 1, 2

STATUS = {
    0: "ok", -1: "null tensor or data pointer", -2: "unsupported element type",
    -3: "shape violates the op contract", -4: "strides/alignment violate the op contract",
    -5: "workspace missing or too small", -6: "scalar argument out of range",
    -7: "HIP launch failed", -8: "shape not implemented by these kernels",
    -9: "needs more than the static scratch holds (or its address is unavailable)",
}


class MlaM4Error(RuntimeError):
    def __init__(self, op: str, status: int):
        self.status = status
        super().__init__(f"{op}: {STATUS.get(status, 'unknown status')} ({status})")


class MlaTensor(ctypes.Structure):
    _fields_ = [
        ("data", ctypes.c_void_p),
        ("type", ctypes.c_int32),
        ("pad_", ctypes.c_int32),
        ("ne", ctypes.c_int64 * 4),
        ("nb", ctypes.c_size_t * 4),
    ]


class RopeParams(ctypes.Structure):
    """mla_m4_rope_params: op_params[1..9] of ggml_m4_phase_kvwrite."""
    _fields_ = [(n, ctypes.c_float) for n in ("freq_base", "freq_scale", "ext_factor", "attn_factor", "beta_fast",
                                               "beta_slow", "eps")] + [("n_dims", ctypes.c_int32), ("n_ctx_orig", ctypes.c_int32)]


_lib: Optional[ctypes.CDLL] = None

_EXPORTS = {
    "mla_m4_version": (ctypes.c_char_p, []),
    "mla_m4_status_str": (ctypes.c_char_p, [ctypes.c_int]),
    "mla_m4_wkb": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3 + [ctypes.c_void_p]),
    "mla_m4_kqkv": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3 + [ctypes.c_float, ctypes.POINTER(MlaTensor),
                                                                      ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "mla_m4_kqkv_noalloc": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3 + [ctypes.c_float, ctypes.POINTER(MlaTensor),
                                                                              ctypes.c_void_p]),
    "mla_m4_kqkv_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(MlaTensor)] * 3),
    "mla_m4_kqkv_default_splits": (ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int32]),
    "mla_m4_kqkv_partial": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3 + [ctypes.c_float, ctypes.c_int, ctypes.c_int64,
                                                                              ctypes.POINTER(MlaTensor), ctypes.c_void_p]),
    "mla_m4_phase_merge": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 2 + [ctypes.c_void_p]),
    "mla_m4_supports_wkb": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3),
    "mla_m4_supports_kqkv": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 4),
    "mla_m4_supports_phase": (ctypes.c_int, [ctypes.c_int32, ctypes.POINTER(MlaTensor), ctypes.POINTER(MlaTensor)]),
    "mla_m4_resolve_flag": (ctypes.c_int, [ctypes.c_int, ctypes.c_int]),
    "mla_m4_phase_wvb": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3 + [ctypes.c_void_p]),
    "mla_m4_supports_phase_wvb": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 3),
    "mla_m4_phase_kvwrite": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 6 + [ctypes.POINTER(RopeParams),
                                                                              ctypes.POINTER(MlaTensor), ctypes.c_void_p]),
    "mla_m4_supports_phase_kvwrite": (ctypes.c_int, [ctypes.POINTER(MlaTensor)] * 6 + [ctypes.POINTER(RopeParams),
                                                                                       ctypes.POINTER(MlaTensor)]),
    # (the operators of a paged batch take their descriptors by address, see _descriptors)
    "mla_m4_pages": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_int32] + [ctypes.c_void_p] * 4),
    "mla_m4_supports_pages": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_int32] + [ctypes.c_void_p] * 3),
    "mla_m4_kvrows": (ctypes.c_int, [ctypes.c_void_p] * 8),
    "mla_m4_supports_kvrows": (ctypes.c_int, [ctypes.c_void_p] * 7),
    "mla_m4_kqkv_paged": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p,
                                                                 ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "mla_m4_kqkv_paged_workspace_bytes": (ctypes.c_size_t, [ctypes.c_void_p] * 5),
    "mla_m4_supports_kqkv_paged": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_int32] + [ctypes.c_void_p] * 2),
    # (and those around its attention)
    "mla_m4_norm": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_float, ctypes.c_void_p, ctypes.c_float] + [ctypes.c_void_p] * 4),
    "mla_m4_supports_norm": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_float] + [ctypes.c_void_p] * 3),
    "mla_m4_rows_i8": (ctypes.c_int, [ctypes.c_void_p] * 4),
    "mla_m4_supports_rows_i8": (ctypes.c_int, [ctypes.c_void_p] * 3),
    "mla_m4_mul_i8": (ctypes.c_int, [ctypes.c_void_p] * 6 + [ctypes.c_size_t, ctypes.c_void_p]),
    "mla_m4_mul_i8_workspace_bytes": (ctypes.c_size_t, [ctypes.c_void_p] * 2),
    "mla_m4_supports_mul_i8": (ctypes.c_int, [ctypes.c_void_p] * 5),
    "mla_m4_qrope": (ctypes.c_int, [ctypes.c_void_p] * 5),
    "mla_m4_supports_qrope": (ctypes.c_int, [ctypes.c_void_p] * 4),
}


def load_library() -> ctypes.CDLL:
    """Load libmla_m4.so (raises if it has not been built: there is no fallback path)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(f"{LIB_PATH} is not built (python -m aubier_amd.build); the MLA ops have no CPU path")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in _EXPORTS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def exported_symbols() -> list[str]:
    return list(_EXPORTS)


# ------------------------------------------------------------------------------------ views
TYPE_Q8_0, TYPE_I8, TYPE_I32, TYPE_I64 = 8, 24, 26, 27
_DT = {torch.float32: (TYPE_F32, 4), torch.float16: (TYPE_F16, 2), torch.int8: (TYPE_I8, 1), torch.int32: (TYPE_I32, 4),
       torch.int64: (TYPE_I64, 8)}


class Q8_0:
    """A Q8_0 tensor (ggml block_q8_0: f16 scale + 32 int8 = 34 bytes per 32 elements): `blocks`
    is a uint8 tensor [..., ne0 / 32 * 34] of packed rows; the ggml shape is (ne0, reversed leading
    dims of `blocks`)."""

    def __init__(self, blocks: torch.Tensor, ne0: int):
        assert blocks.dtype == torch.uint8 and blocks.is_contiguous() and ne0 % 32 == 0
        assert blocks.shape[-1] == ne0 // 32 * 34
        self.blocks, self.ne0 = blocks, ne0

    @property
    def device(self):
        return self.blocks.device


def _view_q8(t: Q8_0) -> MlaTensor:
    v = MlaTensor()
    v.data = t.blocks.data_ptr()
    v.type = TYPE_Q8_0
    rows = list(reversed(t.blocks.shape[:-1]))
    shape = [t.ne0] + rows
    nb = [34, t.blocks.shape[-1]]
    for r in rows[:-1] if rows else []:
        nb.append(nb[-1] * r)
    while len(shape) < 4:
        shape.append(1)
    while len(nb) < 4:
        nb.append(nb[-1] * shape[len(nb) - 1])
    for i in range(4):
        v.ne[i] = int(shape[i])
        v.nb[i] = int(nb[i])
    return v


def view(t) -> Optional[MlaTensor]:
    """ggml-style view of a torch tensor: ne/nb are the reversed shape/strides (bytes)."""
    if t is None:
        return None
    if isinstance(t, Q8_0):
        return _view_q8(t)
    if t.dtype not in _DT:
        raise MlaM4Error("view", -2)
    if t.dim() > 4:
        raise MlaM4Error("view", -3)
    ty, es = _DT[t.dtype]
    v = MlaTensor()
    v.data = t.data_ptr()
    v.type = ty
    shape = list(reversed(t.shape))
    strides = [s * es for s in reversed(t.stride())]
    while len(shape) < 4:
        shape.append(1)
        strides.append(strides[-1] * shape[-2] if strides else es)
    for i in range(4):
        v.ne[i] = int(shape[i])
        v.nb[i] = int(strides[i])
    return v


def _ptr(v: Optional[MlaTensor]):
    return ctypes.byref(v) if v is not None else None


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _check(op: str, rc: int) -> None:
    if rc != 0:
        raise MlaM4Error(op, rc)


# The operators of a paged batch run once per layer or step on a handful of small tensors, so the host's time per call
# counts: a compiled module makes them (binding.cpp, 6 us), or else their descriptors are packed in one go instead of one
# ctypes structure each (24 -> 13 us a call).
_FIELDS = "Pii4q4Q"                         # struct mla_m4_tensor
_DESC_BYTES = struct.calcsize(_FIELDS)
_packers: dict = {}
_local = threading.local()                  # the library reads the descriptors during the call only


def _fields(op: str, t):
    """The values of view(t)'s fields."""
    if isinstance(t, Q8_0):
        if t.blocks.dim() != 2:
            raise MlaM4Error(op, -3)
        n, b = t.blocks.shape
        return (t.blocks.data_ptr(), TYPE_Q8_0, 0, t.ne0, n, 1, 1, 34, b, b * n, b * n)
    try:
        ty, es = _DT[t.dtype]
    except KeyError:
        raise MlaM4Error(op, -2) from None
    shape, stride = t.shape, t.stride()
    d = len(shape)
    if d == 1:
        n, b = shape[0], stride[0] * es
        return (t.data_ptr(), ty, 0, n, 1, 1, 1, b, b * n, b * n, b * n)
    if d == 2:
        n, b = shape[0], stride[0] * es
        return (t.data_ptr(), ty, 0, shape[1], n, 1, 1, stride[1] * es, b, b * n, b * n)
    if d == 3:
        n, b = shape[0], stride[0] * es
        return (t.data_ptr(), ty, 0, shape[2], shape[1], n, 1, stride[2] * es, stride[1] * es, b, b * n)
    raise MlaM4Error(op, -3)


def _descriptors(op: str, tensors):
    """The addresses of the tensors' descriptors (None for None) and the index of the one GPU they lie on; they stay
    valid until the thread's next call."""
    dev, values, at, n = None, [], [], 0
    base = getattr(_local, "base", None)
    if base is None:
        _local.buffer = ctypes.create_string_buffer(16 * _DESC_BYTES)
        base = _local.base = ctypes.addressof(_local.buffer)
    for t in tensors:
        if t is None:
            at.append(None)
            continue
        i = (t.blocks if isinstance(t, Q8_0) else t).get_device()
        if dev is None:
            dev = i
        if i != dev or i < 0:
            raise MlaM4Error(op, -1)
        values += _fields(op, t)
        at.append(base + n * _DESC_BYTES)
        n += 1
    packer = _packers.get(n)
    if packer is None:
        packer = _packers[n] = struct.Struct(_FIELDS * n)
    packer.pack_into(_local.buffer, 0, *values)
    return at, dev


def _run_on(op: str, dev: int, fn, *args):
    """fn(*args, the current stream of GPU dev) with that GPU as the current one."""
    if dev == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        raise MlaM4Error(op, rc)


_get_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _raw_stream(dev: int) -> int:
    return _get_raw_stream(dev) if _get_raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


_native = None


def _calls():
    """A batch's operators' calls as compiled from binding.cpp (13 -> 6 us of host time each), or False where that module is
    not built or was built for another PyTorch: then they go through ctypes, with the same results."""
    global _native
    if _native is None:
        lib = load_library()
        try:
            from . import _binding
        except ImportError:
            _native = False
        else:
            _binding.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
                "mla_m4_pages", "mla_m4_kvrows", "mla_m4_kqkv_paged", "mla_m4_kqkv_paged_workspace_bytes",
                "mla_m4_norm", "mla_m4_rows_i8", "mla_m4_mul_i8", "mla_m4_qrope", "mla_m4_mul_i8_workspace_bytes")))
            _native = _binding
    return _native


def _stream_of(op: str, t: torch.Tensor) -> int:
    dev = t.get_device()
    if dev < 0:
        raise MlaM4Error(op, -1)
    return _raw_stream(dev)


def _done(op: str, r):
    if type(r) is int:
        raise MlaM4Error(op, r)
    return r


# ------------------------------------------------------------------------------------ ops
def ggml_m4_wkb(w_kb, q_nope: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GGML_OP_M4_WKB: out[t, h, c] = sum_d w_kb[h, c, d] * q_nope[t, h, d].

    w_kb f32 [H, D_v, d_n] contiguous, or a Q8_0 with blocks [H, D_v, d_n / 32 * 34] (the
    reference's form: Q8_1 activation numerics); q_nope [nt, H, d_n] (strided view ok);
    out [nt, H, D_v] (a view into the Qcur buffer ok)."""
    lib = load_library()
    if out is None:
        H, D_v = (w_kb.blocks.shape[0], w_kb.blocks.shape[1]) if isinstance(w_kb, Q8_0) else (w_kb.shape[0], w_kb.shape[1])
        out = torch.empty((q_nope.shape[0], H, D_v), dtype=torch.float32, device=q_nope.device)
    vw, vq, vo = view(w_kb), view(q_nope), view(out)
    _check("ggml_m4_wkb", lib.mla_m4_wkb(_ptr(vw), _ptr(vq), _ptr(vo), _stream(q_nope)))
    return out


def kqkv_workspace_bytes(kcache: torch.Tensor, q: torch.Tensor, out: torch.Tensor) -> int:
    lib = load_library()
    return int(lib.mla_m4_kqkv_workspace_bytes(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(out))))


def _kc_width(kcache) -> int:
    """D_k of a cache: a torch tensor [n_kv, D_k] or a Q8_0 one (ne0)."""
    return kcache.ne0 if isinstance(kcache, Q8_0) else kcache.shape[1]


def _dv_of(kcache) -> int:
    """D_v of the op's output for a cache of width D_k: 512 for the 576-wide cache, 256 for the
    reference's 320-wide one, else D_k."""
    dk = _kc_width(kcache)
    return 512 if dk == 576 else (256 if dk == 320 else dk)


def _kc_f16_partials(kcache) -> bool:
    """Whether the partial records hold f16 o (F16 and Q8_0 caches) or f32 (F32 cache)."""
    return isinstance(kcache, Q8_0) or kcache.dtype == torch.float16


def ggml_m4_kqkv(kcache: torch.Tensor, q: torch.Tensor, mask: Optional[torch.Tensor], kq_scale: float,
                 out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GGML_OP_M4_KQKV: out[h, t, :] = softmax_j(kq_scale * q[t, h] . K[j] + mask[t, j]) . V[j, :D_v].

    kcache [n_kv, D_k] f16/f32, or Q8_0 (ne0 = D_k); q [nt, H, D_k] f32; mask [>= nt, n_kv] f32 or None;
    out [H, nt, D_v] f32 (D_v = 512 unless out is given).  workspace: optional uint8 device
    buffer (allocated here when None and the shape needs one)."""
    lib = load_library()
    if out is None:
        out = torch.empty((q.shape[1], q.shape[0], _dv_of(kcache)), dtype=torch.float32, device=q.device)
    vk, vq, vm, vo = view(kcache), view(q), view(mask), view(out)
    need = int(lib.mla_m4_kqkv_workspace_bytes(_ptr(vk), _ptr(vq), _ptr(vo)))
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _check("ggml_m4_kqkv", lib.mla_m4_kqkv(_ptr(vk), _ptr(vq), _ptr(vm), ctypes.c_float(kq_scale), _ptr(vo),
                                           ws_ptr, ws_bytes, _stream(q)))
    return out


NOALLOC_SCRATCH_BYTES = 32 << 20


def ggml_m4_kqkv_noalloc(kcache: torch.Tensor, q: torch.Tensor, mask: Optional[torch.Tensor], kq_scale: float,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ggml_m4_kqkv without a workspace: the library's static scratch holds the split-K partials
    (include/mla_m4.h mla_m4_kqkv_noalloc; calls that overlap on one GPU race)."""
    lib = load_library()
    if out is None:
        out = torch.empty((q.shape[1], q.shape[0], _dv_of(kcache)), dtype=torch.float32, device=q.device)
    _check("ggml_m4_kqkv_noalloc", lib.mla_m4_kqkv_noalloc(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(mask)),
                                                           ctypes.c_float(kq_scale), _ptr(view(out)), _stream(q)))
    return out


def ggml_m4_kqkv_partial(kcache: torch.Tensor, q: torch.Tensor, mask: Optional[torch.Tensor], kq_scale: float,
                         n_split: int, part: Optional[torch.Tensor] = None, d_v: int = 512) -> torch.Tensor:
    """Split-K pass 1 with an explicit split count: part [G, nt, n_split, 64 + 16 D_v] (f32 words)."""
    lib = load_library()
    if part is None:
        G = (q.shape[1] + PART_HEADS - 1) // PART_HEADS
        part = torch.empty((G, q.shape[0], n_split, part_floats(d_v, _kc_f16_partials(kcache))),
                           dtype=torch.float32, device=q.device)
    _check("ggml_m4_kqkv_partial", lib.mla_m4_kqkv_partial(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(mask)),
                                                           ctypes.c_float(kq_scale), int(n_split), int(d_v),
                                                           _ptr(view(part)), _stream(q)))
    return part


def ggml_m4_phase_merge(part: torch.Tensor, out: Optional[torch.Tensor] = None, n_head: Optional[int] = None,
                        d_v: int = 512) -> torch.Tensor:
    """GGML_OP_M4_PHASE phase 2: the split-K merge.  part [G, nt, S, 64 + 16 D_v] -> out [H, nt, D_v]."""
    lib = load_library()
    if out is None:
        H = n_head if n_head is not None else part.shape[0] * PART_HEADS
        out = torch.empty((H, part.shape[1], d_v), dtype=torch.float32, device=part.device)
    _check("ggml_m4_phase_merge", lib.mla_m4_phase_merge(_ptr(view(part)), _ptr(view(out)), _stream(part)))
    return out


def decode_partials(part, n_head: int, d_v: int = 512):
    """Split a partial buffer (numpy/torch, [G, nt, S, 64 + 16 D_v] f32 words; per (group, token)
    one record: the (m, l) pairs [32 heads][S], then the o / l blocks [S][32 heads][D_v]) into
    m [H, nt, S], l [H, nt, S] and o_norm [H, nt, S, D_v] (float32 numpy arrays)."""
    import numpy as np
    p = part.detach().cpu().numpy() if isinstance(part, torch.Tensor) else np.asarray(part)
    G, nt, S, W = p.shape
    rec = np.ascontiguousarray(p).reshape(G, nt, S * W)
    ml = rec[..., :2 * PART_HEADS * S].reshape(G, nt, PART_HEADS, S, 2)
    o = np.ascontiguousarray(rec[..., 2 * PART_HEADS * S:])
    if W == part_floats(d_v, True):
        o = o.view(np.float16)
    o = o.reshape(G, nt, S, PART_HEADS, d_v)
    m = np.moveaxis(ml[..., 0], 2, 1).reshape(G * PART_HEADS, nt, S)[:n_head]
    l = np.moveaxis(ml[..., 1], 2, 1).reshape(G * PART_HEADS, nt, S)[:n_head]
    o = np.moveaxis(o, 3, 1).reshape(G * PART_HEADS, nt, S, d_v)[:n_head].astype(np.float32)
    return m, l, o


def default_splits(n_kv: int, n_head: int = 32, kcache_type: int = TYPE_F16) -> int:
    return int(load_library().mla_m4_kqkv_default_splits(n_kv, n_head, kcache_type))


def supports_kqkv(kcache, q, mask, out) -> bool:
    lib = load_library()
    return bool(lib.mla_m4_supports_kqkv(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(mask)), _ptr(view(out))))


def supports_wkb(w_kb, q_nope, out) -> bool:
    lib = load_library()
    return bool(lib.mla_m4_supports_wkb(_ptr(view(w_kb)), _ptr(view(q_nope)), _ptr(view(out))))


def supports_phase(phase: int, src0, dst) -> bool:
    lib = load_library()
    return bool(lib.mla_m4_supports_phase(int(phase), _ptr(view(src0)), _ptr(view(dst))))


def resolve_flag(flag: int, gpu_core: bool) -> bool:
    """The tri-state enable flag (-1 AUTO, 0 off, 1 explicit); explicit without gpu_core raises."""
    rc = int(load_library().mla_m4_resolve_flag(int(flag), int(bool(gpu_core))))
    if rc < 0:
        raise MlaM4Error("resolve_flag", rc)
    return bool(rc)


def kq_scale_default(d_k_nope: int = 128, d_rope: int = 64) -> float:
    return 1.0 / math.sqrt(d_k_nope + d_rope)


# ---------------------------------------------------------------- PHASE 0 / 1 (reference geometry)
def ggml_m4_phase_wvb(w: Q8_0, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GGML_OP_M4_PHASE phase 1 (wv_b): w Q8_0 blocks [H, d_out, d_in / 32 * 34]; x f32 [H, nt, d_in]
    (the KQKV output layout) -> out [H, nt, d_out]."""
    lib = load_library()
    if out is None:
        out = torch.empty((x.shape[0], x.shape[1], w.blocks.shape[1]), dtype=torch.float32, device=x.device)
    _check("ggml_m4_phase_wvb", lib.mla_m4_phase_wvb(_ptr(view(w)), _ptr(view(x)), _ptr(view(out)), _stream(x)))
    return out


def rope_params(**kw) -> RopeParams:
    rp = RopeParams()
    for k, v in kw.items():
        setattr(rp, k, v)
    return rp


def ggml_m4_phase_kvwrite(cur: torch.Tensor, wkv_a: Q8_0, kv_norm: torch.Tensor, kcache: torch.Tensor,
                          kidx: torch.Tensor, pos: torch.Tensor, rope: RopeParams,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """GGML_OP_M4_PHASE phase 0 (KV-write): cur f32 [n_embd]; wkv_a Q8_0 blocks [n_out, n_embd/32*34];
    kv_norm f32 [d_lat]; kcache f16 [n_kv, n_out] or Q8_0 (rows of n_out / 32 blocks; row kidx[0]
    written in place, quantised as ggml's f32 -> q8_0 copy); kidx int64 [1]; pos int32 [1] -> Kcur
    f32 [n_out]."""
    lib = load_library()
    if out is None:
        out = torch.empty((wkv_a.blocks.shape[0],), dtype=torch.float32, device=cur.device)
    _check("ggml_m4_phase_kvwrite",
           lib.mla_m4_phase_kvwrite(_ptr(view(cur)), _ptr(view(wkv_a)), _ptr(view(kv_norm)), _ptr(view(kcache)),
                                    _ptr(view(kidx)), _ptr(view(pos)), ctypes.byref(rope), _ptr(view(out)),
                                    _stream(cur)))
    return out


def supports_phase_wvb(w, x, out) -> bool:
    return bool(load_library().mla_m4_supports_phase_wvb(_ptr(view(w)), _ptr(view(x)), _ptr(view(out))))


def supports_phase_kvwrite(cur, wkv_a, kv_norm, kcache, kidx, pos, rope: RopeParams, out) -> bool:
    return bool(load_library().mla_m4_supports_phase_kvwrite(_ptr(view(cur)), _ptr(view(wkv_a)), _ptr(view(kv_norm)),
                                                             _ptr(view(kcache)), _ptr(view(kidx)), _ptr(view(pos)),
                                                             ctypes.byref(rope), _ptr(view(out))))


# ------------------------------------------------------------------------------------ paged batches
def _page_size(n: int) -> int:
    """The page size for a call, 0 (which is refused) for what is no int32: ctypes would take its lower 32 bits."""
    return int(n) if -2 ** 31 <= n < 2 ** 31 else 0


def ggml_m4_pages(past: torch.Tensor, n_new: torch.Tensor, free: torch.Tensor, table: torch.Tensor, page_size: int, n_rows: int,
                  slot: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None, used: Optional[torch.Tensor] = None):
    """Block tables and slot maps from request lengths (include/mla_m4.h mla_m4_pages): past, n_new int32 [n_seq];
    free int32 [n_free], the ids that may be taken; table int32 [n_seq, max_pages], the new pages entered in place.
    Returns slot int64 [n_rows] (-1: no cell), pos int32 [n_rows] and used int32 [2] (pages taken, rows of the batch)."""
    calls = _native or _calls()
    if calls:
        return _done("ggml_m4_pages", calls.pages(past, n_new, free, table, page_size, n_rows, slot, pos, used,
                                                  _stream_of("ggml_m4_pages", table)))
    lib = load_library()
    dev = table.device
    slot = torch.empty(n_rows, dtype=torch.int64, device=dev) if slot is None else slot
    pos = torch.empty(n_rows, dtype=torch.int32, device=dev) if pos is None else pos
    used = torch.empty(2, dtype=torch.int32, device=dev) if used is None else used
    (p, n, f, t, s, o, u), gpu = _descriptors("ggml_m4_pages", (past, n_new, free, table, slot, pos, used))
    _run_on("ggml_m4_pages", gpu, lib.mla_m4_pages, p, n, f, t, _page_size(page_size), s, o, u)
    return slot, pos, used


def ggml_m4_kvrows(x: torch.Tensor, kv_norm: torch.Tensor, kcache, slot: torch.Tensor, pos: torch.Tensor, rope: RopeParams,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A batch's latent rows into the cache (include/mla_m4.h mla_m4_kvrows): x f32 or f16 [n_rows, d_lat + n_dims], the
    wkv_a product; kv_norm f32 [d_lat]; kcache f16 [n_cells, d_lat + n_dims] or Q8_0, row slot[r] written in place (none for
    a slot outside the cache); slot int64 [n_rows], pos int32 [n_rows] -> Kcur f32 [n_rows, d_lat + n_dims]."""
    calls = _native or _calls()
    if calls:
        kc, ne0 = (kcache.blocks, kcache.ne0) if isinstance(kcache, Q8_0) else (kcache, 0)
        return _done("ggml_m4_kvrows", calls.kvrows(x, kv_norm, kc, ne0, slot, pos, ctypes.addressof(rope), out,
                                                    _stream_of("ggml_m4_kvrows", x)))
    lib = load_library()
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    (vx, w, k, s, o, d), gpu = _descriptors("ggml_m4_kvrows", (x, kv_norm, kcache, slot, pos, out))
    _run_on("ggml_m4_kvrows", gpu, lib.mla_m4_kvrows, vx, w, k, s, o, ctypes.addressof(rope), d)
    return out


def kqkv_paged_workspace_bytes(kcache, q: torch.Tensor, past: torch.Tensor, out: torch.Tensor,
                               prefix: Optional[torch.Tensor] = None) -> int:
    return int(load_library().mla_m4_kqkv_paged_workspace_bytes(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(past)), _ptr(view(prefix)),
                                                                _ptr(view(out))))


def ggml_m4_kqkv_paged(kcache, q: torch.Tensor, past: torch.Tensor, n_new: torch.Tensor, table: torch.Tensor, page_size: int,
                       kq_scale: float, prefix: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                       workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """KQKV over the pages of a batch (include/mla_m4.h mla_m4_kqkv_paged): token i of request b sees the first
    past[b] + i + 1 cells of table[b].  kcache [n_cells, D_k] f16 or Q8_0; q [nt, H, D_k] f32 or f16; past, n_new int32
    [n_seq]; table int32 [n_seq, max_pages]; prefix int32 [2] (cells, requests) or None: the first requests' tables begin
    with the same pages, whose cells are then read once for all of them.  out [H, nt, D_v], of q's type unless given; rows
    behind the last request are left as they are (in a new `out`: not set).  workspace: optional uint8 device buffer."""
    calls = _native or _calls()
    if calls:
        kc, ne0 = (kcache.blocks, kcache.ne0) if isinstance(kcache, Q8_0) else (kcache, 0)
        return _done("ggml_m4_kqkv_paged", calls.kqkv_paged(kc, ne0, q, past, n_new, table, page_size, kq_scale, prefix, out, _dv_of(kcache),
                                                            workspace, _stream_of("ggml_m4_kqkv_paged", q)))
    lib = load_library()
    if out is None:
        out = torch.empty((q.shape[1], q.shape[0], _dv_of(kcache)), dtype=q.dtype, device=q.device)
    (vk, vq, vp, vn, vt, vf, vo), gpu = _descriptors("ggml_m4_kqkv_paged", (kcache, q, past, n_new, table, prefix, out))
    if workspace is None:
        need = lib.mla_m4_kqkv_paged_workspace_bytes(vk, vq, vp, vf, vo)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need > 0 else None
    elif workspace.get_device() != gpu or not workspace.is_contiguous():
        raise MlaM4Error("ggml_m4_kqkv_paged", -5)
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None else (None, 0)
    _run_on("ggml_m4_kqkv_paged", gpu, lib.mla_m4_kqkv_paged, vk, vq, vp, vn, vt, _page_size(page_size), vf, kq_scale, vo, ws_ptr, ws_bytes)
    return out


def supports_pages(past, n_new, free, table, page_size: int, slot, pos, used) -> bool:
    return bool(load_library().mla_m4_supports_pages(_ptr(view(past)), _ptr(view(n_new)), _ptr(view(free)), _ptr(view(table)),
                                                     _page_size(page_size), _ptr(view(slot)), _ptr(view(pos)), _ptr(view(used))))


def supports_kvrows(x, kv_norm, kcache, slot, pos, rope: RopeParams, out) -> bool:
    return bool(load_library().mla_m4_supports_kvrows(_ptr(view(x)), _ptr(view(kv_norm)), _ptr(view(kcache)), _ptr(view(slot)),
                                                      _ptr(view(pos)), ctypes.byref(rope), _ptr(view(out))))


def supports_kqkv_paged(kcache, q, past, n_new, table, page_size: int, prefix, out) -> bool:
    return bool(load_library().mla_m4_supports_kqkv_paged(_ptr(view(kcache)), _ptr(view(q)), _ptr(view(past)), _ptr(view(n_new)),
                                                          _ptr(view(table)), _page_size(page_size), _ptr(view(prefix)), _ptr(view(out))))


# ------------------------------------------------------------------------------------ around a batch's attention
_FLOAT_OR_I8 = {torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.int8: TYPE_I8}
_FLOAT = {torch.float32: TYPE_F32, torch.float16: TYPE_F16}


def _type_for(op: str, dtype, types) -> int:
    """The type's number; MlaM4Error where a result cannot have it."""
    try:
        return types[dtype]
    except KeyError:
        raise MlaM4Error(op, -2) from None


def ggml_m4_norm(x: torch.Tensor, pre: Optional[torch.Tensor], eps: float, post: Optional[torch.Tensor] = None,
                 gate: Optional[torch.Tensor] = None, res: Optional[torch.Tensor] = None, scale: float = 1.0,
                 dtype: Optional[torch.dtype] = torch.float32, res_out: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, out_scale: Optional[torch.Tensor] = None):
    """The norms before and after a block with the gate and the residual between them (include/mla_m4.h mla_m4_norm):
    y = rms(x) * post, r = res + scale * gate * y, h = rms(r) * pre; post, gate, res, pre None: that part is left out (res
    None: r = gate * y).  x f32 or f16 [rows, n], a block's output; post, pre f32 [n]; gate f32 [n], [rows, 1], [rows, n]
    or [1]; res f32 or f16 [rows, n].  Returns (r, h, h's scale): r of res's type, None without a res or res_out; h of
    `dtype` (None: no h), int8 with a scale f32 [rows], else None.  res_out may be res."""
    ty = -1 if dtype is None else _type_for("ggml_m4_norm", dtype, _FLOAT_OR_I8)
    calls = _native or _calls()
    if calls:
        return _done("ggml_m4_norm", calls.norm(x, post, gate, res, scale, pre, eps, res_out, out, out_scale, ty, _stream_of("ggml_m4_norm", x)))
    if x.dim() != 2:
        raise MlaM4Error("ggml_m4_norm", -3)
    lib = load_library()
    dev = x.device
    if res_out is None and res is not None:
        res_out = torch.empty(x.shape, dtype=res.dtype, device=dev)
    if out is None and dtype is not None:
        out = torch.empty(x.shape, dtype=dtype, device=dev)
    if out_scale is None and out is not None and out.dtype == torch.int8:
        out_scale = torch.empty(x.shape[0], dtype=torch.float32, device=dev)
    (vx, p, g, r, w, o, d, s), gpu = _descriptors("ggml_m4_norm", (x, post, gate, res, pre, res_out, out, out_scale))
    _run_on("ggml_m4_norm", gpu, lib.mla_m4_norm, vx, p, g, r, scale, w, eps, o, d, s)
    return res_out, out, out_scale


def ggml_m4_rows_i8(x: torch.Tensor, out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None):
    """Rows in int8 with a scale each (include/mla_m4.h mla_m4_rows_i8): x f32 or f16 [rows, n], or [rows, H, d] of any strides
    between pieces and rows (wv_b's result [H, rows, d], permuted) -> int8 [rows, n] or [rows, H d], f32 [rows].  Weights,
    whose rows are channels, are brought into this form by the same call."""
    calls = _native or _calls()
    if calls:
        return _done("ggml_m4_rows_i8", calls.rows_i8(x, out, scale, _stream_of("ggml_m4_rows_i8", x)))
    if x.dim() not in (2, 3):
        raise MlaM4Error("ggml_m4_rows_i8", -3)
    lib = load_library()
    if out is None:
        out = torch.empty((x.shape[0], x.shape[1] if x.dim() == 2 else x.shape[1] * x.shape[2]), dtype=torch.int8, device=x.device)
    if scale is None:
        scale = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    (vx, d, s), gpu = _descriptors("ggml_m4_rows_i8", (x, out, scale))
    _run_on("ggml_m4_rows_i8", gpu, lib.mla_m4_rows_i8, vx, d, s)
    return out, scale


def mul_i8_workspace_bytes(w: torch.Tensor, x: torch.Tensor) -> int:
    return int(load_library().mla_m4_mul_i8_workspace_bytes(_ptr(view(w)), _ptr(view(x))))


def ggml_m4_mul_i8(w: torch.Tensor, w_scale: torch.Tensor, x: torch.Tensor, x_scale: torch.Tensor,
                   dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The product of int8 rows and weights (include/mla_m4.h mla_m4_mul_i8): out[t, c] = x_scale[t] w_scale[c] sum_k w[c, k]
    x[t, k].  w int8 [N, K], w_scale f32 [N], x int8 [rows, K], x_scale f32 [rows] -> [rows, N] of `dtype` (f32 or f16) or in
    out.  workspace: optional uint8 device buffer (allocated here when None and the shape has a use for one)."""
    ty = _type_for("ggml_m4_mul_i8", dtype, _FLOAT)
    calls = _native or _calls()
    if calls:
        return _done("ggml_m4_mul_i8", calls.mul_i8(w, w_scale, x, x_scale, out, ty, workspace, _stream_of("ggml_m4_mul_i8", x)))
    if w.dim() != 2 or x.dim() != 2:
        raise MlaM4Error("ggml_m4_mul_i8", -3)
    lib = load_library()
    if out is None:
        out = torch.empty((x.shape[0], w.shape[0]), dtype=dtype, device=x.device)
    (vw, s, vx, t, d), gpu = _descriptors("ggml_m4_mul_i8", (w, w_scale, x, x_scale, out))
    if workspace is None:
        need = lib.mla_m4_mul_i8_workspace_bytes(vw, vx)
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device) if need > 0 else None
    elif workspace.get_device() != gpu or not workspace.is_contiguous():
        raise MlaM4Error("ggml_m4_mul_i8", -5)
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None else (None, 0)
    _run_on("ggml_m4_mul_i8", gpu, lib.mla_m4_mul_i8, vw, s, vx, t, d, ws_ptr, ws_bytes)
    return out


def ggml_m4_qrope(q: torch.Tensor, pos: torch.Tensor, rope: RopeParams, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rope parts of q (include/mla_m4.h mla_m4_qrope): q f32 or f16 [rows, H, n_dims], a view of a product's rows; pos int32
    [rows] -> [rows, H, n_dims], in out (a view into Qcur, or q itself) or a new f32 tensor."""
    calls = _native or _calls()
    if calls:
        return _done("ggml_m4_qrope", calls.qrope(q, pos, ctypes.addressof(rope), out, _stream_of("ggml_m4_qrope", q)))
    lib = load_library()
    if out is None:
        out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    (vq, p, d), gpu = _descriptors("ggml_m4_qrope", (q, pos, out))
    _run_on("ggml_m4_qrope", gpu, lib.mla_m4_qrope, vq, p, ctypes.addressof(rope), d)
    return out


def supports_norm(x, pre, eps: float, post=None, gate=None, res=None, res_out=None, out=None, out_scale=None) -> bool:
    v = [_ptr(view(t)) for t in (x, post, gate, res, pre, res_out, out, out_scale)]
    return bool(load_library().mla_m4_supports_norm(*v[:5], eps, *v[5:]))


def supports_rows_i8(x, out, scale) -> bool:
    return bool(load_library().mla_m4_supports_rows_i8(*(_ptr(view(t)) for t in (x, out, scale))))


def supports_mul_i8(w, w_scale, x, x_scale, out) -> bool:
    return bool(load_library().mla_m4_supports_mul_i8(*(_ptr(view(t)) for t in (w, w_scale, x, x_scale, out))))


def supports_qrope(q, pos, rope: RopeParams, out) -> bool:
    return bool(load_library().mla_m4_supports_qrope(_ptr(view(q)), _ptr(view(pos)), ctypes.byref(rope), _ptr(view(out))))
