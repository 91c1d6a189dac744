"""Plain forms in 64 bits of the operators around a batch's attention."""
import math

import torch

EPS = 2.0 ** -20
YARN = dict(freq_base=1e6, freq_scale=0.25, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, eps=1e-6, n_ctx_orig=8192)
PLAIN = dict(freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.25, beta_fast=32.0, beta_slow=1.0, eps=1e-5, n_ctx_orig=4096)


def int8_64(v):
    """f64 rows -> (int8, f64 scales) by the definition: half away from zero, NaN rows with scale NaN and zeros."""
    top = v.abs().amax(dim=1, keepdim=True)
    bad = ~torch.isfinite(v).all(dim=1, keepdim=True)
    t = torch.where((top > 0) & ~bad, v * 127.0 / torch.where(top > 0, top, torch.ones_like(top)), torch.zeros_like(v))
    q = (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8)
    return q, torch.where(bad, torch.full_like(top, math.nan), top / 127.0)[:, 0]


def rms64(z, eps=EPS):
    return z / torch.sqrt(z.square().mean(dim=1, keepdim=True) + eps)


def norm64(x, pre, eps, post=None, gate=None, res=None, scale=1.0, store=torch.float32):
    """(r as stored, r before it is rounded, h, (int8, scale) of h); store: r's type, None for one that is not rounded."""
    y = x.double()
    if post is not None:
        y = rms64(y, eps) * post.double()
    if gate is not None:
        y = y * gate.double()
    exact = y if res is None else res.double() + scale * y
    r = exact.float().to(store) if store is not None else exact.float()
    z = r.double()
    h = z if pre is None else rms64(z, eps) * pre.double()
    v = z if pre is None else z * pre.double()
    q, step = int8_64(v)
    if pre is not None:
        step = step / torch.sqrt(z.square().mean(dim=1) + eps)
    return r, exact, h, (q, step)


def rope64(x, pos, rp):
    n = x.shape[-1]
    p = torch.arange(n // 2, dtype=torch.float64, device=x.device)
    f = rp["freq_base"] ** (-2.0 * p / n)
    ms = rp["attn_factor"]
    if rp["ext_factor"]:
        def corr(rot):
            return n * math.log(rp["n_ctx_orig"] / (rot * 2 * math.pi)) / (2 * math.log(rp["freq_base"]))
        lo, hi = max(0.0, math.floor(corr(rp["beta_fast"]))), min(n - 1.0, math.ceil(corr(rp["beta_slow"])))
        mix = (1.0 - torch.clamp((p - lo) / max(0.001, hi - lo), 0.0, 1.0)) * rp["ext_factor"]
        f = f * (rp["freq_scale"] * (1.0 - mix) + mix)
        ms *= 1.0 + 0.1 * math.log(1.0 / rp["freq_scale"])
    else:
        f = f * rp["freq_scale"]
    th = pos.double()[:, None, None] * f
    co, si = torch.cos(th) * ms, torch.sin(th) * ms
    x0, x1 = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack([x0 * co - x1 * si, x0 * si + x1 * co], -1).flatten(-2)


def half_step(t):
    """Relative error of one rounding to a type, and the absolute one where it has only subnormals."""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def near(got, want, rel, small=0.0, what=""):
    """|got - want| <= rel |want| + small, and the same values that are not finite."""
    got, want = got.double(), want.double()
    there = torch.isfinite(want)
    assert torch.equal(there, torch.isfinite(got)) and torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~there & ~torch.isnan(want)], want[~there & ~torch.isnan(want)]), what
    d = (got - want).abs()[there] - rel * want.abs()[there] - small
    assert d.numel() == 0 or float(d.max()) <= 0, (what, float(d.max()), float((got - want).abs()[there].max()))
