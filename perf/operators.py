"""The work of the paged-batch operators, as a serving program runs them on one MI355X: a pool of cache pages
shared by the requests of a batch, and one decode, draft-check or prompt-chunk step over it.

Kinds (`"kind"` of a case):

* ``pages`` -- block tables and slot maps from request lengths: request b holds `past` cells and adds `n_new`
  tokens; the pages that it starts are taken from the free list, in request order, and every token gets its cell
  (`slot`) and position. A token without a page gets slot -1, as do the rows behind the last request.
* ``rows``  -- a batch's latent rows into the cache: RMS norm of the latent, YaRN rope of the rope part, the row
  stored at its slot (a row with slot -1 is not stored).
* ``attn``  -- attention of the step's tokens over the pages: token i of request b sees the first
  past[b] + i + 1 cells of its block table; the first `share` requests begin with the same `prefix` cells.
* ``step``  -- the three in turn, as a step uses them.

Geometries: ``base`` (KV row 576 = 512 latent + 64 rope) and ``ref`` (320 = 256 + 64). Caches: f16, and q8 (ggml's
block_q8_0: per 32 values an f16 scale and 32 int8). Latent values and q are scaled so that the scores have a
standard deviation of about 1.7, as they have behind a normalised latent and the 1 / sqrt(d) scale.
"""
import math

import torch

own = False

GEOM = {"base": dict(d_n=128, d_r=64, d_lat=512), "ref": dict(d_n=64, d_r=64, d_lat=256)}
ROPE = dict(freq_base=1e6, freq_scale=0.25, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
            eps=1e-6, n_ctx_orig=8192)
ROW_BYTES = {"f16": lambda dk: 2 * dk, "q8": lambda dk: dk // 32 * 34}


def _case(kind, name=None, **kw):
    c = {"kind": kind, "geom": "base", "cache": "f16", "heads": 32, "page": 64, "seqs": 1, "tok": 1, "chunk": 0,
         "prefix": 0, "share": 0, "lo": 0, "hi": 0, "pad": 0}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the page bookkeeping of an ordinary decode step: latency
        _case("pages", "pages_decode_64", seqs=64, lo=100, hi=8000),
        # of a step that checks drafts and takes in a long prompt, small pages, rows padded to a captured size
        _case("pages", "pages_mixed_500", seqs=500, page=16, tok=3, chunk=6000, lo=0, hi=5000, pad=309),
        # the rows of an ordinary decode step: latency
        _case("rows", "rows_decode_64", seqs=64, lo=100, hi=8000),
        # the rows of a long prompt chunk and some decodes beside it, far positions
        _case("rows", "rows_chunk_8000", seqs=30, chunk=7963, lo=100, hi=120000, pad=8),
        # the first tokens of one conversation: launches and latency
        _case("attn", "attn_one_200", page=16, seqs=1, lo=199, hi=199),
        # requests of very different lengths, nothing shared
        _case("attn", "attn_ragged_48", seqs=48, lo=300, hi=9000),
        # a batch behind one long document or system prompt
        _case("attn", "attn_prefix_64", seqs=64, prefix=32768, share=64, lo=50, hi=2000),
        # the reference geometry over the 8-bit cache, most requests behind a prefix that ends inside a tile
        _case("attn", "attn_prefix_q8_40", geom="ref", cache="q8", page=16, seqs=40, prefix=12000, share=37, lo=500, hi=6000),
        # four drafted tokens of each request checked in one step
        _case("attn", "attn_verify_16x4", seqs=16, tok=4, prefix=8192, share=16, lo=1000, hi=5000),
        # a prompt chunk beside decodes, heads that fill no whole group
        _case("attn", "attn_chunk_mixed", heads=40, page=32, seqs=9, chunk=700, lo=0, hi=3000),
        # a few very long contexts, 16 heads of a sharded model
        _case("attn", "attn_long_4", heads=16, page=128, seqs=4, lo=90000, hi=131000),
        # a whole step: pages, rows and attention over the 8-bit cache
        _case("step", "step_q8_32", cache="q8", seqs=32, prefix=4096, share=32, lo=100, hi=3500),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("pages", "rows", "attn", "attn", "attn", "step"))
    c = dict(geom=rng.choice(("base", "base", "ref")), cache=rng.choice(("f16", "f16", "q8")), page=rng.choice((16, 32, 64, 128)),
             prefix=0, share=0)
    if kind == "pages":
        c.update(seqs=_log(rng, 1, 500), tok=rng.choice((1, 1, 2, 3, 5)), chunk=rng.choice((0, _log(rng, 16, 6000))),
                 hi=_log(rng, 40, 8000), pad=rng.choice((0, rng.randint(1, 300))))
        return _case(kind, lo=rng.randint(0, c["hi"]), **c)
    if kind == "rows":
        c.update(cache="f16", seqs=_log(rng, 1, 100), chunk=rng.choice((0, _log(rng, 16, 7900))), hi=_log(rng, 40, 60000),
                 pad=rng.choice((0, rng.randint(1, 40))))
        return _case(kind, lo=rng.randint(0, c["hi"]), **c)
    c.update(heads=rng.choice((16, 32, 32, 40, 128)), seqs=_log(rng, 1, 64), tok=rng.choice((1, 1, 1, 2, 3, 4, 7)),
             chunk=rng.choice((0, 0, _log(rng, 16, 700))), hi=_log(rng, 40, 9000 if rng.random() < 0.8 else 100000))
    if kind == "step":
        c.update(heads=min(c["heads"], 40), tok=1, chunk=0)
    c["lo"] = rng.randint(0, c["hi"])
    if c["seqs"] > 1 and rng.random() < 0.6:
        c.update(prefix=_log(rng, 64, 32768), share=rng.randint(2, c["seqs"]))
    # at most the largest listed case: the cells a plain form lays out, and the products
    most = max(c["tok"], c["chunk"])
    while (c["seqs"] * (c["prefix"] + c["hi"] + most) > 1_500_000 or
           c["seqs"] * most * c["heads"] * (c["prefix"] + c["hi"] + most) > 700_000_000):
        if c["chunk"] > 100 or (c["chunk"] and c["seqs"] < 4):
            c["chunk"] = c["chunk"] // 2 if c["chunk"] > 30 else 0
        elif c["seqs"] > 1:
            c["seqs"] = c["seqs"] * 3 // 4
            c["share"] = min(c["share"], c["seqs"])
        else:
            c["hi"] //= 2
        c["lo"] = min(c["lo"], c["hi"])
        most = max(c["tok"], c["chunk"])
    return _case(kind, **c)


# ------------------------------------------------------------------------------------ sizes
def _lens(case):
    """(past, n_new) of every request: lengths spread between lo and hi, more short ones than long ones."""
    u = [((b + 1) * 0.6180339887) % 1.0 for b in range(case["seqs"])]
    past = [(case["prefix"] if b < case["share"] else 0) + case["lo"] + int((case["hi"] - case["lo"]) * x * x) for b, x in enumerate(u)]
    return past, [case["chunk"] if case["chunk"] and b == 0 else case["tok"] for b in range(case["seqs"])]


def _max_pages(case):
    past, new = _lens(case)
    return max(-(-(p + n) // case["page"]) for p, n in zip(past, new))


def _width(case):
    g = GEOM[case["geom"]]
    return g["d_lat"] + g["d_r"], g["d_lat"]


def work(case):
    past, new = _lens(case)
    rows = sum(new)
    dk, dv = _width(case)
    H, ps = case["heads"], case["page"]
    by = fl = 0
    if case["kind"] in ("pages", "step"):
        started = sum(-(-(p + n) // ps) - -(-p // ps) for p, n in zip(past, new))
        by += 8 * case["seqs"] + 8 * started + 12 * (rows + case["pad"])
    if case["kind"] in ("rows", "step"):
        by += rows * (4 * dk + 4 * dk + ROW_BYTES[case["cache"]](dk) + 12) + 4 * dv
        fl += rows * (4 * dv + 6 * (dk - dv))
    if case["kind"] in ("attn", "step"):
        shared = case["prefix"] // ps * ps if case["share"] > 1 else 0
        cells = sum(p + n for p, n in zip(past, new)) - shared * max(0, case["share"] - 1)
        pairs = sum(n * p + n * (n + 1) // 2 for p, n in zip(past, new))
        by += cells * ROW_BYTES[case["cache"]](dk) + cells // ps * 4 + rows * H * ((4 if case["kind"] == "step" else 2) * dk + 2 * dv)
        fl += 2 * H * pairs * (dk + dv)
    return {"bytes": by, "flops": fl}


# ------------------------------------------------------------------------------------ inputs
def _q8_rows(x):
    """f32 [rows, ne0] -> block_q8_0 bytes [rows, ne0 / 32 * 34]: d = max / 127, q = round(x / d), half away from zero."""
    b = x.reshape(x.shape[0], -1, 32)
    d = b.abs().amax(dim=2) / 127.0
    y = b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))[:, :, None]
    q = (torch.sign(y) * torch.floor(y.abs() + 0.5)).to(torch.int8)
    return torch.cat([d.to(torch.float16).view(torch.uint8).reshape(*d.shape, 2), q.view(torch.uint8)], dim=2).reshape(x.shape[0], -1)


def _q8_values(blocks, dtype):
    """block_q8_0 bytes [..., nb * 34] -> the values they stand for [..., nb * 32]."""
    b = blocks.reshape(*blocks.shape[:-1], -1, 34)
    d = b[..., :2].contiguous().view(torch.float16).to(dtype)
    return (d * b[..., 2:].contiguous().view(torch.int8).to(dtype)).flatten(-2)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    past, new = _lens(case)
    rows, n_seq, ps = sum(new), case["seqs"], case["page"]
    dk, dv = _width(case)
    mp = _max_pages(case)
    s = {"case": case, "page": ps, "rows": rows + case["pad"], "max_new": max(new), "max_keys": max(p + n for p, n in zip(past, new)),
         "scale": 1.0 / math.sqrt(GEOM[case["geom"]]["d_n"] + GEOM[case["geom"]]["d_r"])}
    s["past"] = torch.tensor(past, dtype=torch.int32, device="cuda")
    s["new"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    # the pool: pages in no order; the sharing requests' tables begin with the same ones
    fresh = case["kind"] in ("pages", "step")              # the step's own pages are still on the free list
    whole = case["prefix"] // ps                           # whole pages of the prefix: these are shared
    s["prefix"] = torch.tensor([whole * ps, case["share"]], dtype=torch.int32, device="cuda") if case["share"] else None
    col = torch.arange(mp, device="cuda")
    held = (s["past"] + (0 if fresh else 1) * s["new"] + ps - 1) // ps
    have = col[None, :] < held[:, None]
    shared = have & (col[None, :] < whole) & (torch.arange(n_seq, device="cuda")[:, None] < case["share"])
    first = torch.arange(n_seq, device="cuda")[:, None] == 0
    mine = have & (~shared | first)
    n_free = sum(-(-(p + n) // ps) - -(-p // ps) for p, n in zip(past, new)) + 5 if fresh else 0
    n_mine = sum(-(-(p if fresh else p + n) // ps) - (whole if 0 < b < case["share"] else 0) for b, (p, n) in enumerate(zip(past, new)))
    n_pages = n_mine + n_free + 3
    perm = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    order = (torch.cumsum(mine.reshape(-1).long(), 0) - 1).reshape(mine.shape)
    table = torch.where(mine, perm[order.clamp(min=0)], -torch.ones_like(perm[:1]))
    s["table"] = torch.where(shared, table[:1], table).contiguous()
    s["free"] = perm[n_mine:n_mine + n_free].contiguous()
    cells = n_pages * ps

    if case["kind"] == "rows":
        s["pos"] = (s["past"].repeat_interleave(s["new"].long()) + torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in new]))
        s["pos"] = torch.cat([s["pos"], torch.zeros(case["pad"], dtype=torch.int32, device="cuda")])
        cells = 2 * rows + 64
        slot = torch.randperm(cells, generator=gen, device="cuda")[:rows]
        s["slot"] = torch.cat([slot, -torch.ones(case["pad"], dtype=torch.int64, device="cuda")])
    if case["kind"] != "pages":
        kc = torch.randn((cells, dk), generator=gen, device="cuda")
        s["kc"] = _q8_rows(kc) if case["cache"] == "q8" else kc.to(torch.float16)
    if case["kind"] in ("rows", "step"):
        s["x"] = torch.randn((s["rows"], dk), generator=gen, device="cuda")
        s["norm"] = 1.0 + 0.25 * torch.randn((dv,), generator=gen, device="cuda")
    if case["kind"] in ("attn", "step"):
        # Qcur as WKB leaves it in a step, and rounded to f16 before the call elsewhere
        s["q"] = torch.randn((s["rows"], case["heads"], dk), generator=gen, device="cuda")
        s["q"] = s["q"] if case["kind"] == "step" else s["q"].to(torch.float16)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------------------------ the plain forms
def _pages(s):
    ps, table, n_rows = s["page"], s["table"], s["rows"]
    past, new = s["past"].long(), s["new"].long()
    have = (past + ps - 1) // ps
    take = (past + new + ps - 1) // ps - have
    first = torch.cumsum(take, 0) - take
    end = torch.cumsum(new, 0)
    r = torch.arange(n_rows, device=table.device)
    b = torch.searchsorted(end, r, right=True).clamp(max=len(new) - 1)
    p = past[b] + r - (end[b] - new[b])
    j = p // ps
    live = r < end[-1]
    nth = first[b] + j - have[b]
    mine = live & (j >= have[b])
    n_free = s["free"].numel()
    page = torch.where(mine, torch.where(nth < n_free, s["free"][nth.clamp(0, n_free - 1)], -1), table[b, j.clamp(max=table.shape[1] - 1)])
    # the row at a page's start enters it; the others write the same value again
    table.index_put_((torch.where(mine, b, b[:1]), torch.where(mine, j, j[:1])), torch.where(mine, page, page[:1]))
    slot = torch.where(live & (page >= 0), page.long() * ps + p % ps, -1)
    pos = torch.where(live, p, 0).to(torch.int32)
    used = torch.stack([torch.minimum(take.sum(), torch.full_like(take[0], n_free)), end[-1]]).to(torch.int32)
    return {"table": table, "slot": slot, "pos": pos, "used": used}


def _freqs(d_r, device):
    """Angle per position of every rope pair, and the scale of its cosine and sine (YaRN)."""
    p = torch.arange(d_r // 2, device=device, dtype=torch.float64)

    def corr(rot):
        return d_r * math.log(ROPE["n_ctx_orig"] / (rot * 2 * math.pi)) / (2 * math.log(ROPE["freq_base"]))

    lo, hi = max(0.0, math.floor(corr(ROPE["beta_fast"]))), min(d_r - 1.0, math.ceil(corr(ROPE["beta_slow"])))
    mix = (1.0 - torch.clamp((p - lo) / max(0.001, hi - lo), 0.0, 1.0)) * ROPE["ext_factor"]
    return (ROPE["freq_base"] ** (-2.0 * p / d_r) * (ROPE["freq_scale"] * (1.0 - mix) + mix),
            ROPE["attn_factor"] * (1.0 + 0.1 * math.log(1.0 / ROPE["freq_scale"])))


def _rows(s, slot, pos):
    dk, dv = _width(s["case"])
    x, kc = s["x"], s["kc"]
    lat = x[:, :dv] * torch.rsqrt(x[:, :dv].square().mean(dim=1, keepdim=True) + ROPE["eps"]) * s["norm"]
    freq, ms = _freqs(dk - dv, x.device)
    theta = pos.double()[:, None] * freq
    co, si = (torch.cos(theta) * ms).float(), (torch.sin(theta) * ms).float()
    x0, x1 = x[:, dv::2], x[:, dv + 1::2]
    kcur = torch.cat([lat, torch.stack([x0 * co - x1 * si, x0 * si + x1 * co], dim=2).flatten(1)], dim=1)
    stored = _q8_rows(kcur) if s["case"]["cache"] == "q8" else kcur.to(torch.float16)
    # rows without a slot: row 0's value to row 0's slot once more
    there = slot >= 0
    kc.index_put_((torch.where(there, slot, slot[:1]),), torch.where(there[:, None], stored, stored[:1]))
    return kcur


def _attend(s):
    q, table, ps, H = s["q"], s["table"], s["page"], s["case"]["heads"]
    dk, dv = _width(s["case"])
    past, new = s["past"].long(), s["new"].long()
    n_seq, m, n_rows = past.numel(), s["max_new"], s["rows"]
    end = torch.cumsum(new, 0)
    start = end - new
    i = torch.arange(m, device=q.device)
    key = torch.arange(s["max_keys"], device=q.device)
    seen = key[None, :] < (past + new)[:, None]
    cell = torch.where(seen, table[:, key // ps].long() * ps + key % ps, 0)
    k = s["kc"][cell]
    k = _q8_values(k, torch.float32) if s["case"]["cache"] == "q8" else k.float()
    qq = q[(start[:, None] + i).clamp(max=n_rows - 1)].float().reshape(n_seq, m * H, dk)
    sc = torch.matmul(qq, k.transpose(1, 2)).mul_(s["scale"]).view(n_seq, m, H, -1)
    sc.masked_fill_(~(key < (past[:, None] + i + 1)[:, :, None])[:, :, None, :], -math.inf)
    sc = sc.sub_(sc.amax(dim=-1, keepdim=True)).exp_()
    total = sc.sum(dim=-1, keepdim=True)
    o = torch.matmul(sc.view(n_seq, m * H, -1), k[:, :, :dv]).view(n_seq, m, H, dv).div_(total)
    r = torch.arange(n_rows, device=q.device)
    b = torch.searchsorted(end, r, right=True).clamp(max=n_seq - 1)
    return o[b, r - start[b]].permute(1, 0, 2).to(torch.float16).contiguous()


# ------------------------------------------------------------------------------------ the framework's calls
def _kcache(s):
    if s["case"]["cache"] == "q8":
        import aubier_amd as A
        return A.Q8_0(s["kc"], _width(s["case"])[0])
    return s["kc"]


def _own_pages(s):
    import aubier_amd as A
    slot, pos, used = A.ggml_m4_pages(s["past"], s["new"], s["free"], s["table"], s["page"], s["rows"])
    return {"table": s["table"], "slot": slot, "pos": pos, "used": used}


def _own_rows(s, slot, pos):
    import aubier_amd as A
    dk, dv = _width(s["case"])
    return A.ggml_m4_kvrows(s["x"], s["norm"], _kcache(s), slot, pos, A.rope_params(n_dims=dk - dv, **ROPE))


def _own_attend(s):
    import aubier_amd as A
    out = torch.empty((s["q"].shape[1], s["rows"], _width(s["case"])[1]), dtype=torch.float16, device="cuda")
    return A.ggml_m4_kqkv_paged(_kcache(s), s["q"], s["past"], s["new"], s["table"], s["page"], s["scale"], prefix=s["prefix"], out=out)


def run(state):
    pages, rows, attend = (_own_pages, _own_rows, _own_attend) if own else (_pages, _rows, _attend)
    kind = state["case"]["kind"]
    if kind == "pages":
        return pages(state)
    if kind == "rows":
        return {"kcur": rows(state, state["slot"], state["pos"]), "cache": state["kc"]}
    if kind == "attn":
        return {"kqv": attend(state)}
    p = pages(state)
    kcur = rows(state, p["slot"], p["pos"])
    return {**p, "kcur": kcur, "kqv": attend(state)}


# ------------------------------------------------------------------------------------ in 64 bits
def _rows64(s, slot, pos):
    """kcur [rows, D_k]: the rows before they are rounded for the cache."""
    dk, dv = _width(s["case"])
    x, w, n = s["x"].double(), s["norm"].double(), dk - dv
    lat = x[:, :dv] / torch.sqrt((x[:, :dv] ** 2).sum(1, keepdim=True) / dv + ROPE["eps"]) * w
    # rope pairs as complex numbers, turned by an angle that lies between the position's own and the
    # position's scaled by freq_scale, by where the pair's wavelength lies in the trained context
    base, pairs = ROPE["freq_base"], torch.arange(n // 2, device=x.device).double()
    bound = [math.log(ROPE["n_ctx_orig"] / (2 * math.pi * ROPE[k])) * n / (2 * math.log(base)) for k in ("beta_fast", "beta_slow")]
    lo, hi = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), n - 1)
    keep = (1 - ((pairs - lo) / max(hi - lo, 1e-3)).clamp(0, 1)) * ROPE["ext_factor"]
    own_angle = pos.to(x.device).double()[:, None] / base ** (2 * pairs / n)
    angle = own_angle * keep + own_angle * ROPE["freq_scale"] * (1 - keep)
    size = ROPE["attn_factor"] * (1 - 0.1 * math.log(ROPE["freq_scale"]))
    z = torch.view_as_complex(x[:, dv:].reshape(x.shape[0], -1, 2).contiguous()) * torch.polar(torch.full_like(angle, size), angle)
    return torch.cat([lat, torch.view_as_real(z).reshape(x.shape[0], -1)], dim=1)


def _blocks64(kcur):
    """block_q8_0 bytes of 64-bit rows."""
    v = kcur.unflatten(1, (-1, 32))
    top = v.abs().max(dim=2, keepdim=True).values / 127
    q = (v / torch.where(top == 0, torch.ones_like(top), top))
    q = torch.where(q < 0, torch.ceil(q - 0.5), torch.floor(q + 0.5)).to(torch.int8)
    return torch.cat([top.half().view(torch.uint8), q.view(torch.uint8)], dim=2).flatten(1)


def _values64(rows):
    v = rows.unflatten(1, (-1, 34))
    scale = (v[:, :, 0].long() + 256 * v[:, :, 1].long()).to(torch.int16).view(torch.float16).double()
    q = v[:, :, 2:].double()
    return (torch.where(q > 127, q - 256, q) * scale[:, :, None]).flatten(1)


def exact(case, seed):
    s = _inputs(case, seed)
    H, ps = case["heads"], case["page"]
    dk, dv = _width(case)
    if case["kind"] == "rows":
        kcur = _rows64(s, s["slot"], s["pos"])
        kc = s["kc"].double()
        n = s["rows"] - case["pad"]
        kc[s["slot"][:n]] = kcur[:n]
        return {"kcur": kcur, "cache": kc}

    def pages64():
        """The definition, a request at a time, on the host."""
        ps, n_rows = s["page"], s["rows"]
        table, free = s["table"].cpu(), s["free"].tolist()
        slot, pos, taken = [], [], 0
        for b, (p, n) in enumerate(zip(s["past"].tolist(), s["new"].tolist())):
            for i in range(n):
                j = (p + i) // ps
                if j * ps >= p and (p + i) % ps == 0:      # the request starts a page
                    table[b, j] = free[taken] if taken < len(free) else -1
                    taken += 1
                page = int(table[b, j])
                slot.append(page * ps + (p + i) % ps if page >= 0 else -1)
                pos.append(p + i)
        slot += [-1] * (n_rows - len(slot))
        used = [min(taken, len(free)), len(pos)]
        pos += [0] * (n_rows - len(pos))
        return {"table": table, "slot": torch.tensor(slot), "pos": torch.tensor(pos, dtype=torch.int32), "used": torch.tensor(used, dtype=torch.int32)}

    if case["kind"] == "pages":
        return pages64()
    kc, table, got = s["kc"], s["table"], {}
    if case["kind"] == "step":
        p = pages64()
        table, slot = p["table"].cuda(), p["slot"].cuda()
        kcur = _rows64(s, slot, p["pos"])
        kc[slot] = _blocks64(kcur) if case["cache"] == "q8" else kcur.to(torch.float16)
        got = {**p, "kcur": kcur}
    out = torch.zeros((H, s["rows"], dv), dtype=torch.float64, device="cuda")
    r = 0
    for b, (p, n) in enumerate(zip(*_lens(case))):
        key = torch.arange(p + n, device="cuda")
        k = kc[table[b, key // ps].long() * ps + key % ps]
        k = _values64(k) if case["cache"] == "q8" else k.double()
        kt, v = k.t().contiguous(), k[:, :dv].contiguous()
        for i in range(0, n, 64):                      # 64 tokens at a time
            e = min(n, i + 64)
            q = s["q"][r + i:r + e].double().reshape((e - i) * H, dk)
            x = (q @ kt * s["scale"]).view(e - i, H, -1)
            late = key[None, :] > (p + torch.arange(i, e, device="cuda"))[:, None]
            x = x.masked_fill(late[:, None, :], -math.inf)
            o = torch.softmax(x, dim=-1).view((e - i) * H, -1) @ v
            out[:, r + i:r + e] = o.view(e - i, H, dv).permute(1, 0, 2)
        r += n
    return {**got, "kqv": out}
