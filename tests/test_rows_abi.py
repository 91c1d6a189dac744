"""What the operators around a batch's attention refuse (include/mla_m4.h mla_m4_norm, mla_m4_rows_i8, mla_m4_mul_i8,
mla_m4_qrope): host-side checks alone, no kernel is launched."""
import ctypes

import pytest
import torch

import aubier_amd as A
from aubier_amd import ops

from rows_util import EPS, YARN

F32, F16, I8 = torch.float32, torch.float16, torch.int8
z = torch.zeros


def refused(name, args, scalars=()):
    """The status of the entry point itself for descriptors of host tensors (nothing is launched: it is refused before)."""
    v = [A.view(a) if isinstance(a, torch.Tensor) else a for a in args]
    p = [ctypes.byref(t) if isinstance(t, ops.MlaTensor) else t for t in v]
    return getattr(A.load_library(), name)(*p, None)


def norm(**kw):
    d = dict(x=z(3, 64), post=None, gate=None, res=None, scale=1.0, pre=z(64), eps=EPS, res_out=None, out=z(3, 64), out_scale=None)
    d.update(kw)
    return refused("mla_m4_norm", [d[k] for k in ("x", "post", "gate", "res", "scale", "pre", "eps", "res_out", "out", "out_scale")])


@pytest.mark.parametrize("status,bad", [
    (-1, dict(out=None)), (-1, dict(x=None)), (-1, dict(out=z(3, 64, dtype=I8))),
    (-2, dict(x=z(3, 64, dtype=I8))), (-2, dict(res=z(3, 64, dtype=I8))), (-2, dict(res_out=z(3, 64, dtype=I8))), (-2, dict(out=z(3, 64, dtype=torch.int32))),
    (-2, dict(gate=z(64, dtype=F16))), (-2, dict(pre=z(64, dtype=F16))), (-2, dict(post=z(64, dtype=F16))),
    (-2, dict(out_scale=z(3))), (-2, dict(out=z(3, 64, dtype=I8), out_scale=z(3, dtype=F16))),
    (-3, dict(x=z(3, 62), pre=z(62), out=z(3, 62))), (-3, dict(res=z(3, 60))), (-3, dict(res=z(4, 64))), (-3, dict(out=z(2, 64))), (-3, dict(res_out=z(64))),
    (-3, dict(pre=z(60))), (-3, dict(post=z(2, 64))), (-3, dict(gate=z(32))), (-3, dict(gate=z(2, 64))), (-3, dict(gate=z(2, 1))),
    (-3, dict(x=z(2, 3, 64))), (-3, dict(out=z(3, 64, dtype=I8), out_scale=z(4))),
    (-4, dict(x=z(64, 3).t())), (-4, dict(x=z(3, 66)[:, :64])), (-4, dict(x=z(3, 68)[:, 1:65])), (-4, dict(out=z(1, 64).expand(3, 64))),
    (-4, dict(pre=z(65)[1:])), (-4, dict(pre=z(128)[::2])), (-4, dict(gate=z(3, 66)[:, :64])), (-4, dict(res=z(3, 66, dtype=F16)[:, :64])),
    (-4, dict(out=z(3, 66, dtype=I8)[:, :64], out_scale=z(3))), (-4, dict(out=z(3, 64, dtype=I8), out_scale=z(6)[::2])),
    (-6, dict(eps=-1.0)), (-6, dict(eps=float("nan"))), (-6, dict(eps=float("inf"))),
    (-8, dict(x=z(1, 32772), pre=z(32772), out=z(1, 32772))),
])
def test_norm(status, bad):
    assert norm(**bad) == status


def test_norm_rows_past_the_most():
    x = z(1, 4).expand(2 ** 24 + 1, 4)
    assert norm(x=x, pre=z(4), out=x) == -4              # rows in one place are no rows to write
    out = A.view(z(1, 4))
    for t in (out,):
        t.ne[1], t.nb[1] = 2 ** 24 + 1, 16
    assert refused("mla_m4_norm", [out, None, None, None, 1.0, A.view(z(4)), EPS, None, out, None]) == -8


def rows_i8(x, out, scale):
    return refused("mla_m4_rows_i8", [x, out, scale])


@pytest.mark.parametrize("status,args", [
    (-1, (None, z(3, 64, dtype=I8), z(3))), (-1, (z(3, 64), None, z(3))), (-1, (z(3, 64), z(3, 64, dtype=I8), None)),
    (-2, (z(3, 64, dtype=I8), z(3, 64, dtype=I8), z(3))), (-2, (z(3, 64), z(3, 64), z(3))), (-2, (z(3, 64), z(3, 64, dtype=I8), z(3, dtype=F16))),
    (-3, (z(3, 62), z(3, 62, dtype=I8), z(3))), (-3, (z(3, 64), z(3, 60, dtype=I8), z(3))), (-3, (z(3, 2, 32), z(2, 96, dtype=I8), z(2))),
    (-3, (z(3, 64), z(3, 64, dtype=I8), z(4))), (-3, (z(2, 3, 2, 32), z(3, 64, dtype=I8), z(3))), (-3, (z(3, 32, 2), z(3, 64, dtype=I8), z(3))),
    (-4, (z(64, 3).t(), z(3, 64, dtype=I8), z(3))), (-4, (z(3, 2, 33)[:, :, :32], z(3, 64, dtype=I8), z(3))), (-4, (z(3, 68)[:, 2:66], z(3, 64, dtype=I8), z(3))),
    (-4, (z(3, 64), z(3, 66, dtype=I8)[:, :64], z(3))), (-4, (z(3, 64), z(1, 64, dtype=I8).expand(3, 64), z(3))),
    (-8, (z(1, 32772), z(1, 32772, dtype=I8), z(1))), (-8, (z(1, 257, 128), z(1, 257 * 128, dtype=I8), z(1))),
])
def test_rows_i8(status, args):
    assert rows_i8(*args) == status


def mul(**kw):
    d = dict(w=z(5, 64, dtype=I8), ws=z(5), x=z(3, 64, dtype=I8), xs=z(3), out=z(3, 5))
    d.update(kw)
    v = [A.view(t) if isinstance(t, torch.Tensor) else t for t in d.values()]
    return A.load_library().mla_m4_mul_i8(*(ctypes.byref(t) if t is not None else None for t in v), None, 0, None)


@pytest.mark.parametrize("status,bad", [
    (-1, dict(w=None)), (-1, dict(ws=None)), (-1, dict(xs=None)), (-1, dict(out=None)),
    (-2, dict(w=z(5, 64))), (-2, dict(x=z(3, 64))), (-2, dict(out=z(3, 5, dtype=I8))), (-2, dict(ws=z(5, dtype=F16))), (-2, dict(xs=z(3, dtype=torch.int32))),
    (-3, dict(w=z(5, 72, dtype=I8), x=z(3, 72, dtype=I8))), (-3, dict(w=z(5, 48, dtype=I8))), (-3, dict(out=z(3, 4))), (-3, dict(out=z(4, 5))),
    (-3, dict(ws=z(4))), (-3, dict(xs=z(5))), (-3, dict(x=z(1, 3, 64, dtype=I8), out=z(1, 3, 5), w=z(2, 5, 64, dtype=I8))),
    (-3, dict(w=z(5, 8, dtype=I8), x=z(3, 8, dtype=I8))),
    (-4, dict(w=z(64, 5, dtype=I8).t())), (-4, dict(w=z(5, 72, dtype=I8)[:, :64])), (-4, dict(x=z(3, 96, dtype=I8)[:, 8:72])),
    (-4, dict(w=z(1, 64, dtype=I8).expand(5, 64))), (-4, dict(out=z(5, 3).t())), (-4, dict(out=z(1, 5).expand(3, 5))), (-4, dict(ws=z(10)[::2])),
    (-8, dict(w=z(5, 131072, dtype=I8), x=z(3, 131072, dtype=I8))),
])
def test_mul_i8(status, bad):
    assert mul(**bad) == status


def test_mul_i8_strides_past_the_most():
    w = A.view(z(5, 64, dtype=I8))
    w.nb[1] = 2 ** 22 + 16
    assert mul(w=w) == -8
    w.nb[1] = 2 ** 22
    assert A.load_library().mla_m4_supports_mul_i8(*(ctypes.byref(t) for t in (w, A.view(z(5)), A.view(z(3, 64, dtype=I8)), A.view(z(3)), A.view(z(3, 5)))))
    out = A.view(z(3, 5))
    out.nb[1] = 2 ** 62
    assert mul(out=out) == -4


def qrope(**kw):
    d = dict(q=z(3, 2, 64), pos=z(3, dtype=torch.int32), rope=A.rope_params(n_dims=64, **YARN), out=z(3, 2, 64))
    d.update(kw)
    v = [A.view(t) if isinstance(t, torch.Tensor) else t for t in d.values()]
    return A.load_library().mla_m4_qrope(*(ctypes.byref(t) if t is not None else None for t in v), None)


@pytest.mark.parametrize("status,bad", [
    (-1, dict(q=None)), (-1, dict(pos=None)), (-1, dict(rope=None)), (-1, dict(out=None)),
    (-2, dict(q=z(3, 2, 64, dtype=I8))), (-2, dict(out=z(3, 2, 64, dtype=torch.int32))), (-2, dict(pos=z(3, dtype=torch.int64))),
    (-3, dict(q=z(3, 2, 32))), (-3, dict(out=z(3, 2, 32))), (-3, dict(out=z(2, 3, 64))), (-3, dict(pos=z(2, dtype=torch.int32))),
    (-3, dict(rope=A.rope_params(n_dims=48, **YARN), q=z(3, 2, 48), out=z(3, 2, 48))),
    (-4, dict(q=z(3, 64, 2).transpose(1, 2))), (-4, dict(q=z(3, 2, 66)[:, :, :64])), (-4, dict(q=z(3, 2, 68)[:, :, 1:65])),
    (-4, dict(out=z(1, 2, 64).expand(3, 2, 64))), (-4, dict(out=z(3, 1, 64).expand(3, 2, 64))), (-4, dict(out=z(3, 2, 70)[:, :, :64])),
    (-6, dict(rope=A.rope_params(n_dims=64, **{**YARN, "freq_base": 0.0}))), (-6, dict(rope=A.rope_params(n_dims=64, **{**YARN, "freq_scale": float("nan")}))),
    (-6, dict(rope=A.rope_params(n_dims=64, **{**YARN, "n_ctx_orig": 0}))),
    (-8, dict(rope=A.rope_params(n_dims=288, **YARN), q=z(3, 2, 288), out=z(3, 2, 288))),
    (-8, dict(q=z(1, 1025, 64), out=z(1, 1025, 64), pos=z(1, dtype=torch.int32))),
])
def test_qrope(status, bad):
    assert qrope(**bad) == status


def test_no_rows():
    """A call of no rows is refused, whether its tensors have memory or not."""
    assert norm(x=z(0, 64), out=z(0, 64)) == -1 and mul(x=z(0, 64, dtype=I8), xs=z(0), out=z(0, 5)) == -1
    x, out = A.view(z(3, 64)), A.view(z(3, 64))
    x.ne[1] = out.ne[1] = 0
    assert norm(x=x, out=out) == -3
    x, out = A.view(z(3, 64, dtype=I8)), A.view(z(3, 5))
    x.ne[1] = out.ne[1] = 0
    assert mul(x=x, out=out) == -3


def test_supports():
    """What the mirrors accept: also descriptors whose data is not set yet."""
    assert A.supports_norm(z(3, 64), z(64), EPS, z(64), z(3, 1), z(3, 64, dtype=F16), z(3, 64, dtype=F16), z(3, 64, dtype=I8), z(3))
    assert A.supports_norm(z(3, 64), None, EPS, out=z(3, 64)) and not A.supports_norm(z(3, 64), None, EPS)
    assert A.supports_rows_i8(z(2, 3, 64).permute(1, 0, 2), z(3, 128, dtype=I8), z(3)) and not A.supports_rows_i8(z(3, 64), z(3, 64), z(3))
    assert A.supports_mul_i8(z(5, 64, dtype=I8), z(5), z(3, 64, dtype=I8), z(3), z(3, 5, dtype=F16))
    assert A.supports_qrope(z(3, 2, 192)[:, :, 128:], z(3, dtype=torch.int32), A.rope_params(n_dims=64, **YARN), z(3, 2, 576)[:, :, 512:])
    v = [A.view(t) for t in (z(5, 64, dtype=I8), z(5), z(3, 64, dtype=I8), z(3), z(3, 5))]
    for t in v:
        t.data = None
    assert A.load_library().mla_m4_supports_mul_i8(*(ctypes.byref(t) for t in v))
    assert A.load_library().mla_m4_mul_i8(*(ctypes.byref(t) for t in v), None, 0, None) == -1


def test_python_refuses():
    """Host tensors, types that a result cannot have, matrices that are none."""
    x, w, s = z(3, 64, dtype=I8), z(5, 64, dtype=I8), z(3)
    for status, call in ((-1, lambda: A.ggml_m4_norm(z(3, 64), z(64), EPS)), (-2, lambda: A.ggml_m4_norm(z(3, 64), z(64), EPS, dtype=torch.float64)),
                         (-1, lambda: A.ggml_m4_rows_i8(z(3, 64))), (-1, lambda: A.ggml_m4_mul_i8(w, z(5), x, s)),
                         (-2, lambda: A.ggml_m4_mul_i8(w, z(5), x, s, dtype=I8)),
                         (-1, lambda: A.ggml_m4_qrope(z(3, 2, 64), z(3, dtype=torch.int32), A.rope_params(n_dims=64, **YARN)))):
        with pytest.raises(A.MlaM4Error) as e:
            call()
        assert e.value.status == status
