"""Inputs and error bounds shared by the tests of the 8-bit cache's operators."""

from __future__ import annotations

import torch

#: Half a rounding step of an output type, relative to the value.
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make_cache(blocks, block_size, kv_heads, dim, *, latent=False, seed=0, device="cuda", layout="thd"):
    """(k, v, k_scale, v_scale) with codes up to the type's largest and scales around 2**-6.

    ``layout`` "htd" stores each page head by head, and hands out the
    (block, token, head, dim) view of it."""
    g = torch.Generator().manual_seed(seed)

    def part():
        shape = (blocks, block_size, kv_heads, dim) if layout == "thd" else (blocks, kv_heads, block_size, dim)
        codes = (torch.randn(shape, generator=g) * 64).clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
        if layout == "htd":
            codes = codes.permute(0, 2, 1, 3)
        scale = torch.exp(torch.randn((blocks, kv_heads), generator=g) * 0.5) * 2.0**-6
        return codes, scale.to(device)

    k, ks = part()
    if latent:
        return k, None, ks, None
    v, vs = part()
    return k, v, ks, vs


def score_error(q, k_cache, k_scale, softmax_scale):
    """A bound on a score's absolute error in float32: the products' sum in
    blocks of 32 and their joining keep at least 23 bits of the largest partial
    sum, which is at most sum |q k| <= |q| |k|, over at most 18 blocks and the
    two or three parts of q; the factors' roundings add a few more units."""
    longest_q = float(q.double().norm(dim=-1).max())
    page = (k_cache.float().double().norm(dim=-1).amax(1) * k_scale.double()).nan_to_num(0.0)
    return 64 * 2.0**-23 * longest_q * float(page.max()) * abs(softmax_scale) + 2.0**-22


def assert_attention(out, lse, want, q, k_cache, k_scale, softmax_scale):
    """out within half a step of the output's type, plus what the weights' errors make.

    A weight enters the product as x = 2^(u - R + 5), with the tile's largest x
    in [2, 2^8.5], in parts of 8 bits. A first e4m3 part leaves at most
    max(2^-4 2^e, 2^-10) for x in [2^e, 2^(e + 1)); an e5m2 part leaves of a
    remainder r at most half a step of r's binade, which is 2^-3 of the
    binade's start, or 2^-17 below 2^-14. So two parts (bf16) leave at most
    max(2^-8 x, 2^-14), with 2^-11 x more from their way through fp16, and
    three (fp16) max(2^-12 x, 2^-17): relative errors of 2^-8 + 2^-11 and 2^-12
    in each weight, and 2^-15 and 2^-18 of the largest weight of that tile. The
    score's own error counts twice, in the weight and in the sum."""
    ref_out, ref_lse, spread, near = want
    u = HALF_STEP[out.dtype]
    relative, floor = {torch.bfloat16: (2.0**-8 + 2.0**-11, 2.0**-15), torch.float16: (2.0**-12, 2.0**-18)}[out.dtype]
    ds = score_error(q, k_cache, k_scale, softmax_scale)
    bound = u * ref_out.abs() + (relative + 2 * ds) * spread + floor * near + 1e-30
    error = (out.double() - ref_out).abs()
    bad = ~(error <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} outputs off, worst {float((error / bound).nan_to_num(9e9).max()):.3g} bounds"
    empty = ref_lse == -float("inf")
    assert bool((lse[empty] == -float("inf")).all()) and bool((out[empty] == 0).all())
    off = (lse.double() - ref_lse)[~empty].abs()
    assert off.numel() == 0 or float((off - 2.0**-22 * ref_lse[~empty].abs()).max()) <= ds + 2.0**-20
