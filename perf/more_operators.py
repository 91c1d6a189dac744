"""The work of the operators around the attention of a paged batch, as a serving program runs them on one MI355X: the
norms and the residual before and after a block, the rows in 8-bit integers, their products, and the rope of q.

Kinds (`"kind"` of a case):

* ``norm``  -- rows between two blocks: y = rms(x) * post, r = res + scale * gate * y, h = rms(r) * pre.  r is stored as
  f32 or f16, h as f32, f16 or int8 with one scale a row (``out``).  Without a residual: h = rms(x) * pre.
* ``quant`` -- rows of several heads' pieces (the attention's output, [heads, rows, d] in memory) in int8, one scale a
  row: scale = max |x| / 127, q = round(127 x / max |x|), half away from zero.
* ``mul``   -- the product of int8 rows and int8 weights with a scale for each row (token) and each channel:
  y[t, n] = x_scale[t] * w_scale[n] * sum_k w[n, k] x[t, k].
* ``rope``  -- the rope parts of q into Qcur, beside the columns that the absorption of the other parts fills.
* ``into``  -- norm and product in turn: a block's input projections.
* ``out``   -- rows in int8, product, norm: from the attention's output to the next block's input.
"""
import math

import torch

own = False

EPS = 2.0 ** -20
ROPE = dict(freq_base=1e6, freq_scale=0.25, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
            eps=1e-6, n_ctx_orig=8192)
D_N, D_R, D_LAT, D_OUT = 128, 64, 512, 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "i8": torch.int8}


def _case(kind, name=None, **kw):
    c = {"kind": kind, "rows": 1, "n": 4096, "k": 4096, "heads": 32, "x": "f32", "res": "f32", "out": "f32", "post": True, "gate": "channel",
         "scale": 1.0}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # between two blocks of a decode step: latency
        _case("norm", "norm_decode_64", rows=64, n=7168, out="i8"),
        # of a prompt chunk, the block's output as an f16 product left it
        _case("norm", "norm_chunk_8000", rows=7993, n=4096, x="f16", out="i8", scale=0.5),
        # the attention's output of a decode step: latency
        _case("quant", "quant_decode_48", rows=48, heads=32),
        # of a prompt chunk, heads that make no power of two
        _case("quant", "quant_chunk_5000", rows=5003, heads=40),
        # one token's latent row: a few weights, latency
        _case("mul", "mul_one_576", rows=1, n=576, k=7168),
        # an output projection of a decode step: weights read once
        _case("mul", "mul_decode_64", rows=64, n=7168, k=4096, out="f16"),
        # the heads' q of a few hundred drafted tokens, a short sum
        _case("mul", "mul_verify_300", rows=300, n=24576, k=1536),
        # an output projection of a long prompt chunk: matrix instructions
        _case("mul", "mul_chunk_8000", rows=8000, n=7168, k=16384, out="f16"),
        # q of a decode step: latency
        _case("rope", "rope_decode_64", rows=64, heads=32),
        # q of a prompt chunk, as an f16 product left it
        _case("rope", "rope_chunk_5000", rows=5003, heads=40, x="f16"),
        # a decode step's input projections: the residual's norm, then q's and the cache's latents by one product
        _case("into", "into_32", rows=32, n=2112, k=7168),
        # from the attention's output of a prompt chunk to the next block's input
        _case("out", "out_4000", rows=4001, n=4096, heads=32, out="f16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(("norm", "quant", "mul", "mul", "mul", "rope", "into", "out"))
    wide = lambda: 16 * _log(rng, 16, 512)  # noqa: E731
    c = dict(x=rng.choice(("f32", "f16")), res=rng.choice(("f32", "f32", "f16")), post=rng.random() < 0.7, scale=rng.choice((1.0, 0.5, 0.25)),
             gate=rng.choice(("channel", "row", "none", "full")), heads=rng.choice((1, 8, 16, 32, 40, 64, 128)))
    if kind == "norm":
        c.update(rows=_log(rng, 1, 8000), n=rng.choice((4096, 7168, wide(), wide())), out=rng.choice(("f32", "f16", "i8", "i8")))
        if rng.random() < 0.3:
            c.update(res="none", gate="none", post=False)
    elif kind == "quant":
        c.update(rows=_log(rng, 1, 5000))
    elif kind == "mul":
        c.update(rows=_log(rng, 1, 8000), n=rng.choice((576, 4096, 7168, wide(), rng.randint(1, 4000))), k=rng.choice((1536, 4096, 7168, wide(), wide())),
                 out=rng.choice(("f32", "f16")))
        while c["rows"] * c["n"] > 60_000_000:
            c["rows"] = c["rows"] * 2 // 3
    elif kind == "rope":
        c.update(rows=_log(rng, 1, 8000), out=rng.choice(("f32", "f32", "f16")))
        while c["rows"] * c["heads"] > 400_000:
            c["rows"] = c["rows"] * 2 // 3
    elif kind == "into":
        c.update(rows=_log(rng, 1, 4000), n=rng.choice((2112, wide())), k=rng.choice((4096, 7168, wide())), out="f32")
    else:
        c.update(rows=_log(rng, 1, 4000), n=rng.choice((4096, 7168, wide())), out=rng.choice(("f32", "f16")))
    return _case(kind, **c)


# ------------------------------------------------------------------------------------ sizes
SIZE = {"f32": 4, "f16": 2, "i8": 1}


def _norm_bytes(rows, n, case, x, out):
    by = rows * n * (SIZE[x] + SIZE[out]) + 4 * n + (4 * rows if out == "i8" else 0)
    if case["res"] != "none":
        by += 2 * rows * n * SIZE[case["res"]]
    by += 4 * n if case["post"] else 0
    return by + 4 * {"channel": n, "row": rows, "full": rows * n, "none": 0}[case["gate"]]


def _mul_bytes(rows, n, k, out):
    return n * k + rows * k + 4 * (n + rows) + rows * n * SIZE[out]


def work(case):
    rows, n, k, H = case["rows"], case["n"], case["k"], case["heads"]
    if case["kind"] == "norm":
        return {"bytes": _norm_bytes(rows, n, case, case["x"], case["out"]), "flops": 10 * rows * n}
    if case["kind"] == "quant":
        return {"bytes": rows * H * D_OUT * (SIZE[case["x"]] + 1) + 4 * rows, "flops": 3 * rows * H * D_OUT}
    if case["kind"] == "mul":
        return {"bytes": _mul_bytes(rows, n, k, case["out"]), "flops": 2 * rows * n * k}
    if case["kind"] == "rope":
        return {"bytes": rows * (H * D_R * (SIZE[case["x"]] + SIZE[case["out"]]) + 4), "flops": 3 * rows * H * D_R}
    if case["kind"] == "into":     # x, residual, weights and scales in; r and the product out
        return {"bytes": _norm_bytes(rows, k, case, case["x"], "i8") - rows * (k + 4) + _mul_bytes(rows, n, k, "f32") - rows * (k + 4),
                "flops": 2 * rows * n * k + 10 * rows * k}
    k = H * D_OUT                  # the attention's output, weights and scales, residual in; r and h out
    return {"bytes": rows * k * SIZE[case["x"]] + n * (k + 4) + _norm_bytes(rows, n, case, "f32", case["out"]) - 4 * rows * n,
            "flops": 2 * rows * n * k + 10 * rows * n}


# ------------------------------------------------------------------------------------ inputs
def _int8_rows(x):
    """f32 [..., n] -> int8 and the rows' scales."""
    top = x.abs().amax(dim=-1, keepdim=True)
    return torch.round(x / top * 127.0).to(torch.int8), (top[..., 0] / 127.0)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, rows, H = case["kind"], case["rows"], case["heads"]
    s = {"case": case}

    def randn(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def hidden(n, typ):
        """Rows of a residual stream or a block's output: a few channels far above the others, rows of different sizes."""
        loud = torch.where(torch.rand((n,), generator=gen, device="cuda") < 0.004, 12.0, 1.0)
        return (randn(rows, n) * loud * torch.exp(0.5 * randn(rows, 1))).to(TYPES[typ])

    if kind in ("norm", "into", "out"):
        n = case["k"] if kind == "into" else case["n"]
        s["pre"] = 1.0 + 0.25 * randn(n)
        s["post"] = 0.5 + 0.125 * randn(n) if case["post"] else None
        shape = {"channel": (n,), "row": (rows, 1), "full": (rows, n)}.get(case["gate"])
        s["gate"] = 0.5 + 0.25 * randn(*shape) if shape else None
        s["res"] = hidden(n, case["res"]) if case["res"] != "none" else None
        if kind != "out":
            s["x"] = hidden(n, case["x"])
    if kind in ("quant", "out"):
        s["o"] = (randn(H, rows, D_OUT) * torch.exp(0.5 * randn(H, rows, 1))).to(TYPES[case["x"]])
    if kind in ("mul", "into", "out"):
        k = H * D_OUT if kind == "out" else case["k"]
        s["w"], s["w_scale"] = _int8_rows(randn(case["n"], k) / math.sqrt(k))
        if kind == "mul":
            s["q"], s["q_scale"] = _int8_rows(hidden(k, "f32"))
    if kind == "rope":
        s["pos"] = torch.randint(0, 120000, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        s["q"] = randn(rows, H, D_N + D_R).to(TYPES[case["x"]])            # the product's rows: the parts to absorb, then the rope parts
        s["qcur"] = torch.zeros((rows, H, D_LAT + D_R), dtype=TYPES[case["out"]], device="cuda")
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ------------------------------------------------------------------------------------ the plain forms
def _round_i8(v):
    """f64 [rows, n] -> int8, half away from zero, and the rows' largest magnitudes.  In 64 bits: a value next to a border
    between two integers falls on its side."""
    top = v.abs().amax(dim=1, keepdim=True)
    t = v * 127.0 / torch.where(top > 0, top, torch.ones_like(top))
    return (torch.sign(t) * torch.floor(t.abs() + 0.5)).to(torch.int8), top[:, 0]


def _norm(s, x, out):
    z = x.double()
    if s["post"] is not None:
        z = z * torch.rsqrt(z.square().mean(dim=1, keepdim=True) + EPS) * s["post"]
    if s["gate"] is not None:
        z = z * s["gate"]
    r = None
    if s["res"] is not None:
        r = (s["res"].double() + s["case"]["scale"] * z).to(s["res"].dtype)
        z = r.double()
    inv = torch.rsqrt(z.square().mean(dim=1, keepdim=True) + EPS)
    v = z * s["pre"]
    if out != "i8":
        return {"r": r, "h": (v * inv).to(TYPES[out])}
    q, top = _round_i8(v)
    return {"r": r, "h": q, "h_scale": (top * inv[:, 0] / 127.0).float()}


def _quant(o):
    x = o.permute(1, 0, 2).reshape(o.shape[1], -1).double()
    q, top = _round_i8(x)
    return {"q": q, "scale": (top / 127.0).float()}


def _mul(s, q, q_scale, out):
    # (sums of at most 16,384 products of zero mean: whole numbers far below 2^24, exact in 32 bits)
    y = torch.matmul(q.float(), s["w"].float().t())
    return y.mul_(q_scale[:, None]).mul_(s["w_scale"]).to(TYPES[out])


def _freqs(device):
    """Angle per position of every rope pair, and the scale of its cosine and sine (YaRN)."""
    p = torch.arange(D_R // 2, device=device, dtype=torch.float64)

    def corr(rot):
        return D_R * math.log(ROPE["n_ctx_orig"] / (rot * 2 * math.pi)) / (2 * math.log(ROPE["freq_base"]))

    lo, hi = max(0.0, math.floor(corr(ROPE["beta_fast"]))), min(D_R - 1.0, math.ceil(corr(ROPE["beta_slow"])))
    mix = (1.0 - torch.clamp((p - lo) / max(0.001, hi - lo), 0.0, 1.0)) * ROPE["ext_factor"]
    return (ROPE["freq_base"] ** (-2.0 * p / D_R) * (ROPE["freq_scale"] * (1.0 - mix) + mix),
            ROPE["attn_factor"] * (1.0 + 0.1 * math.log(1.0 / ROPE["freq_scale"])))


def _rope(s):
    freq, ms = _freqs(s["pos"].device)
    theta = s["pos"].double()[:, None] * freq
    co, si = (torch.cos(theta) * ms).float()[:, None], (torch.sin(theta) * ms).float()[:, None]
    x0, x1 = s["q"][:, :, D_N::2].float(), s["q"][:, :, D_N + 1::2].float()
    part = s["qcur"][:, :, D_LAT:]
    part.copy_(torch.stack([x0 * co - x1 * si, x0 * si + x1 * co], dim=3).flatten(2))
    return part


# ------------------------------------------------------------------------------------ the framework's calls
def _own_norm(s, x, out):
    import aubier_amd as A
    r, h, h_scale = A.ggml_m4_norm(x, s["pre"], EPS, post=s["post"], gate=s["gate"], res=s["res"], scale=s["case"]["scale"], dtype=TYPES[out])
    return {"r": r, "h": h, "h_scale": h_scale} if out == "i8" else {"r": r, "h": h}


def _own_quant(o):
    import aubier_amd as A
    q, scale = A.ggml_m4_rows_i8(o.permute(1, 0, 2))
    return {"q": q, "scale": scale}


def _own_mul(s, q, q_scale, out):
    import aubier_amd as A
    return A.ggml_m4_mul_i8(s["w"], s["w_scale"], q, q_scale, dtype=TYPES[out])


def _own_rope(s):
    import aubier_amd as A
    return A.ggml_m4_qrope(s["q"][:, :, D_N:], s["pos"], A.rope_params(n_dims=D_R, **ROPE), out=s["qcur"][:, :, D_LAT:])


def run(state):
    norm, quant, mul, rope = (_own_norm, _own_quant, _own_mul, _own_rope) if own else (_norm, _quant, _mul, _rope)
    s, case = state, state["case"]
    kind = case["kind"]
    if kind == "norm":
        return norm(s, s["x"], case["out"])
    if kind == "quant":
        return quant(s["o"])
    if kind == "mul":
        return {"y": mul(s, s["q"], s["q_scale"], case["out"])}
    if kind == "rope":
        return {"q_pe": rope(s)}
    if kind == "into":
        a = norm(s, s["x"], "i8")
        return {"r": a["r"], "y": mul(s, a["h"], a["h_scale"], "f32")}
    a = quant(s["o"])
    return norm(s, mul(s, a["q"], a["scale"], "f32"), case["out"])


# ------------------------------------------------------------------------------------ in 64 bits
def _rms64(z, w):
    return z / torch.sqrt((z ** 2).sum(1, keepdim=True) / z.shape[1] + EPS) * w.double()


def _i8_64(v):
    """The int8 values and scales of f64 rows, as f64."""
    top = torch.linalg.vector_norm(v, ord=math.inf, dim=1, keepdim=True)
    steps = torch.where(top == 0, torch.zeros_like(v), 127 * v / top)
    near = torch.trunc(steps + torch.copysign(torch.full_like(steps, 0.5), steps))
    return near, top[:, 0] / 127


def _norm64(s, x, out):
    y = x.double()
    if s["post"] is not None:
        y = _rms64(y, s["post"])
    if s["gate"] is not None:
        y = s["gate"].double() * y
    if s["res"] is None:
        r, y = None, y
    else:
        r = s["res"].double() + y * s["case"]["scale"]
        y = r.to(s["res"].dtype).double()              # the next norm is of the residual as it is stored
    if out != "i8":
        return {"r": r, "h": _rms64(y, s["pre"])}
    # the row's root scales all of its values alike: the integers are those of r * pre
    near, _ = _i8_64(y * s["pre"].double())
    _, step = _i8_64(_rms64(y, s["pre"]))
    return {"r": r, "h": near, "h_scale": step}


def _mul64(s, q, q_scale):
    return (q.double() * q_scale.double()[:, None]) @ (s["w"].double() * s["w_scale"].double()[:, None]).t().contiguous()


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _norm64(s, s["x"], case["out"])
    if kind in ("quant", "out"):
        near, step = _i8_64(s["o"].transpose(0, 1).flatten(1).double())
        if kind == "quant":
            return {"q": near, "scale": step}
        return _norm64(s, _mul64(s, near, step), case["out"])
    if kind == "mul":
        return {"y": _mul64(s, s["q"], s["q_scale"])}
    if kind == "into":
        a = _norm64(s, s["x"], "i8")
        return {"r": a["r"], "y": _mul64(s, a["h"], a["h_scale"])}
    # rope pairs as complex numbers, turned by an angle that lies between the position's own and the position's scaled by
    # freq_scale, by where the pair's wavelength lies in the trained context
    base, pairs = ROPE["freq_base"], torch.arange(D_R // 2, device="cuda").double()
    bound = [math.log(ROPE["n_ctx_orig"] / (2 * math.pi * ROPE[k])) * D_R / (2 * math.log(base)) for k in ("beta_fast", "beta_slow")]
    lo, hi = max(math.floor(bound[0]), 0), min(math.ceil(bound[1]), D_R - 1)
    keep = (1 - ((pairs - lo) / max(hi - lo, 1e-3)).clamp(0, 1)) * ROPE["ext_factor"]
    angle = s["pos"].double()[:, None] / base ** (2 * pairs / D_R)
    angle = (angle * keep + angle * ROPE["freq_scale"] * (1 - keep))[:, None]
    size = ROPE["attn_factor"] * (1 - 0.1 * math.log(ROPE["freq_scale"]))
    z = torch.view_as_complex(s["q"][:, :, D_N:].double().unflatten(2, (-1, 2)).contiguous()) * torch.polar(torch.full_like(angle, size), angle)
    return {"q_pe": torch.view_as_real(z).flatten(2)}
