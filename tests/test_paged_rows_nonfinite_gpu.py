"""NaN and infinities on their way into the cache (mla_m4_kvrows): what an f16 cache would hold as one must not become a number
in an 8-bit one."""
import math

import pytest
import torch

import aubier_amd as A

from paged_util import q8_f16

pytestmark = pytest.mark.gpu

RP = dict(freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0, eps=1e-6, n_ctx_orig=4096)


@pytest.mark.parametrize("n,d_r", [(576, 64), (320, 64)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("xt", [torch.float32, torch.float16])
def test_kvrows(dev, n, d_r, bad, xt):
    g = torch.Generator().manual_seed(n)
    rows, dl = 12, n - d_r
    x = torch.randn((rows, n), generator=g).to(xt).to(dev)
    # rows 0 .. 7: one value of the rope part; 8: one of the latent part; the others none
    cols = [dl, dl + 1, dl + 31, dl + 32, dl + 40, n - 2, n - 1, dl + 17]
    clean = x.clone()
    for r, c in enumerate(cols):
        x[r, c] = bad
    x[8, 70] = bad
    w = torch.ones(dl, device=dev)
    slot, pos = torch.arange(rows, device=dev), torch.arange(rows, dtype=torch.int32, device=dev) + 1
    rope = A.rope_params(n_dims=d_r, **RP)

    def run(x):
        f = torch.zeros((rows, n), dtype=torch.float16, device=dev)
        b = A.Q8_0(torch.zeros((rows, n // 32 * 34), dtype=torch.uint8, device=dev), n)
        k = A.ggml_m4_kvrows(x, w, f, slot, pos, rope)
        assert torch.equal(torch.isnan(k), torch.isnan(A.ggml_m4_kvrows(x, w, b, slot, pos, rope)))
        return k, f, b.blocks

    k, f, blocks = run(x)
    k0, f0, blocks0 = run(clean)
    odd = ~torch.isfinite(k)
    assert odd[:8].sum(1).tolist() == [2] * 8 and odd[8, 70] and not odd[9:].any()      # a rope pair; the latent part as its norm has it
    assert torch.equal(~torch.isfinite(f), odd)
    # 8 bits: blocks that hold one hold nothing finite, the others are as without it
    hit = odd.unflatten(1, (-1, 32)).any(2)
    values = q8_f16(blocks).unflatten(1, (-1, 32))
    assert not torch.isfinite(values[hit]).any()
    b, b0 = blocks.unflatten(1, (-1, 34)), blocks0.unflatten(1, (-1, 34))
    same = ~hit
    same[8] = False                                          # (its norm moved)
    assert torch.equal(b[same], b0[same])
