"""A paged batch for the tests of the paged operators, and their plain forms in 64 bits, a request at a time."""
import math

import torch

import aubier_amd as A
from aubier_amd import inputs as I

GEOM = {576: 512, 320: 256}
SCALE = 1.0 / math.sqrt(192.0)


def q8_rows(x):
    """f32 rows [rows, ne0] -> block_q8_0 bytes, as ggml's f32 -> q8_0 copy (on the host: torch divides a GPU tensor by
    a number with a product by its reciprocal, which is not the quotient rounded once)."""
    return torch.from_numpy(I.q8_0_rows(x.cpu().numpy())).to(x.device)


def q8_f16(blocks):
    """block_q8_0 bytes -> f16(q d), the values the kernels compute with."""
    b = blocks.unflatten(-1, (-1, 34))
    d = b[..., :2].contiguous().view(torch.float16).float()
    return (d * b[..., 2:].contiguous().view(torch.int8).float()).half().flatten(-2)


class Batch:
    """Pages in no order, `spare` of them unused; cells that no token sees hold `poison` (f16 caches)."""

    def __init__(self, dev, past, new, page, dk=576, H=32, prefix=0, share=0, cache="f16", q_type=torch.float16, seed=0,
                 poison=math.nan, spare=3, pad=0, max_pages=None, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.page, self.dk, self.dv, self.H, self.cache = page, dk, GEOM[dk], H, cache
        self.past_l, self.new_l = list(past), list(new)
        need = [-(-(p + n) // page) for p, n in zip(past, new)]
        mp = max_pages or max(max(need), 1)
        whole = prefix // page
        owned = [n - (whole if 0 < b < share else 0) for b, n in enumerate(need)]
        n_pages = sum(owned) + spare
        perm = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((len(past), mp), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            ids = perm[:owned[b]]
            perm = perm[owned[b]:]
            if 0 < b < share:
                ids = table[0, :whole].tolist() + ids
            table[b, :n] = torch.tensor(ids, dtype=torch.int32)
        cells = n_pages * page
        kc = torch.randn((cells, dk), generator=g) * spread
        seen = torch.zeros(cells, dtype=torch.bool)
        for b, (p, n) in enumerate(zip(past, new)):
            j = torch.arange(p + n)
            seen[table[b, j // page].long() * page + j % page] = True
        kc = kc.half()
        if cache == "f16":
            kc[~seen] = poison
            self.kc = self.values = kc.to(dev)
        else:
            blocks = q8_rows(kc.float())
            if math.isnan(poison):                          # a NaN scale in every block
                bad = blocks[~seen].unflatten(-1, (-1, 34))
                bad[..., 0], bad[..., 1] = 0, 0x7e
                blocks[~seen] = bad.flatten(-2)
            self.values = q8_f16(blocks).to(dev)
            self.kc = A.Q8_0(blocks.to(dev), dk)
        nt = sum(new) + pad
        self.nt, self.rows = nt, sum(new)
        self.q = torch.randn((nt, H, dk), generator=g).to(q_type).to(dev)
        self.past = torch.tensor(past, dtype=torch.int32, device=dev)
        self.new = torch.tensor(new, dtype=torch.int32, device=dev)
        self.table = table.to(dev)
        self.prefix = torch.tensor([prefix, share], dtype=torch.int32, device=dev) if share else None

    def out(self, dtype=torch.float32, fill=7.0):
        return torch.full((self.H, self.nt, self.dv), fill, dtype=dtype, device=self.q.device)

    def run(self, out=None, prefix=True, **kw):
        return A.ggml_m4_kqkv_paged(self.kc, self.q, self.past, self.new, self.table, self.page, SCALE,
                                    prefix=self.prefix if prefix else None, out=self.out() if out is None else out, **kw)


def attend64(b: Batch, dst_type=torch.float32):
    """out [H, rows, D_v] in 64 bits and how far the kernel may be from it, element by element.

    The kernel's own roundings, each at most half a step: of q to f16 (only an f32 q is rounded), which moves a score by
    at most scale sum |q| |k| 2^-11 and by the f32 sum's rounding (D_k + 1 additions, 2^-24 each); of every weight to
    f16, which changes numerator and denominator by 2^-11 at most each (and by 2^-25 beside a largest weight of at least
    2^8 where it falls among f16's subnormals: keys x 2^-33); of a split's normalised output to f16 (2^-11); of the
    result (2^-11 for f16, 2^-24 for f32).  exp2 and the merge's factors: 2^-20 covers their few f32 roundings."""
    k64 = b.values.double()
    past, new, table = b.past.tolist(), b.new.tolist(), b.table.tolist()
    n_pages = k64.shape[0] // b.page
    out = torch.zeros((b.H, b.rows, b.dv), dtype=torch.float64, device=k64.device)
    tol = torch.zeros_like(out)
    u16 = 2.0 ** -11
    r = 0
    for s, (p, n) in enumerate(zip(past, new)):
        p, n = max(p, 0), max(n, 0)
        cap = len(table[s]) * b.page
        j = torch.arange(min(p + n, cap), device=k64.device)
        page = torch.tensor(table[s], device=k64.device)[j // b.page].long()
        ok = (page >= 0) & (page < n_pages)
        k = k64[(page * b.page + j % b.page)[ok]]
        j = j[ok]
        for i in range(n):
            kk = k[j < p + i + 1]
            if len(kk) == 0:
                continue
            q = b.q[r + i].double()
            sc = q @ kk.t() * SCALE
            w = torch.softmax(sc, dim=1)
            v = kk[:, :b.dv]
            out[:, r + i] = w @ v
            size = q.abs() @ kk.abs().t() * SCALE
            d = size.max(dim=1).values * (b.dk + 1) * 2.0 ** -24
            if b.q.dtype == torch.float32:
                d = d + size.max(dim=1).values * u16
            rel = 2 * torch.expm1(d) + 2 * u16 + len(kk) * 2.0 ** -32 + u16 + 2.0 ** -20
            rel = rel + (u16 if dst_type == torch.float16 else 2.0 ** -24)
            tol[:, r + i] = rel[:, None] * (w @ v.abs())
        r += n
    # a split's output and an f16 result may also fall among f16's subnormals (2^-25 each)
    return out, tol + 2.0 ** -24


def check(b: Batch, got, name=""):
    want, tol = attend64(b, got.dtype)
    g = got[:, :b.rows].double()
    assert torch.isfinite(g).all(), name
    off = (g - want).abs() / tol
    worst = float(off.max()) if off.numel() else 0.0
    print(f"{name} worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0, (name, worst)
    if b.nt > b.rows:                                        # rows behind the last request
        assert (got[:, b.rows:] == 7.0).all(), name
