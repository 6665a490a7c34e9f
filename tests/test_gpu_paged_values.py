"""What kata_paged_decode does with values of any size: V scales of int8 caches from the smallest fp16 number to the
largest, and long int8 caches head by head; each against a plain evaluation in 64 bits.

Elementwise bounds are relative to A = sum_j p_j |v_j| / l, the size of the terms an output is made of:
 - scores: q, codes and K scales are chosen so that every partial sum is exact; the exponent's argument (|x| < 32) is rounded three times, 3 * 32 * 2^-24 * ln 2, and ex2 is off by 2^-22. Both
   occur in numerator and denominator: 2 * (4.0e-6 + 2.4e-7) = 8.4e-6
 - p times the V scale in two fp16 terms: 2^-22, or 2^-25 of a number that is carried as 2^15 p v / (at most twice the tile's largest scale): 2^-40 of that scale a slot; in one term 2^-11 instead of 2^-22
 - products: up to 8 chained matrix instructions per tile, 2 * 2^-23 each; then one rounding a tile and four joins: 1,000 slots are below 64 tiles, 2^-18 in all
 together 8.4e-6 + 2.4e-7 + 1.9e-6 + 3.8e-6 < 2^-16; outputs add half a step of their type."""
import math

import pytest
import torch

from .test_gpu_paged import EPS, F8, _attend, _context, _gen, _kv, _randn, _rows, _score_error, capi  # noqa: F401

pytestmark = pytest.mark.gpu


def _exact_scores(ctx, g, T, n_seqs, q_step, k_scale):
    """Queries and int8 keys whose scores are sums of few-bit numbers: exact in fp32 in any order."""
    H, D = ctx.heads, ctx.head_dim
    q16 = (torch.randint(-1, 2, (n_seqs, T, H * D), generator=g, device="cuda") * q_step).half()
    k = ctx.plane(0, "k")
    k.copy_(torch.randint(-15, 16, k.shape, generator=g, device="cuda"))
    ctx.plane(0, "k_scale").fill_(k_scale)
    return q16


def _terms(ctx, seq, n, T, q16):
    """fp64: outputs and the sums of their terms' magnitudes, [T][heads][head_dim]."""
    KH, G, D = ctx.kv_heads, ctx.heads // ctx.kv_heads, ctx.head_dim
    k, v = _kv(ctx, 0, seq, n)
    q = q16.to(F8).view(T, KH, G, D)
    out, size = (torch.zeros(T, KH, G, D, dtype=F8, device="cuda") for _ in range(2))
    for t in range(T):
        m = n - T + 1 + t
        p = torch.softmax(torch.einsum("hgd,lhd->hgl", q[t], k[:m]), -1)
        out[t], size[t] = torch.einsum("hgl,lhd->hgd", p, v[:m]), torch.einsum("hgl,lhd->hgd", p, v[:m].abs())
    return out.view(T, KH * G, D), size.view(T, KH * G, D)


@pytest.mark.parametrize("layout,T", [((24, 4, 256), 1), ((24, 4, 256), 2), ((32, 8, 128), 1), ((16, 1, 128), 1)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [2.0 ** -24, 1e-6, 1e-5, 1e-3, 0.4, 500.0, "spread"])
@pytest.mark.parametrize("keys", ["mixed", "one heavy"])
def test_int8_values_of_any_size(capi, layout, T, out, scale, keys):  # noqa: F811
    H, KH, D = layout
    g = _gen(H + T)
    slots = [1000, 37, 5]
    ctx = _context(capi, slots, layout, 16, "int8", fill=g)
    q16 = _exact_scores(ctx, g, T, len(slots), 2.0 ** -5, 0.5)     # scores: multiples of 2^-6, standard deviation 1.8 (256) or 1.3
    ctx.plane(0, "v").copy_(torch.randint(1, 128, ctx.plane(0, "v").shape, generator=g, device="cuda"))   # of one sign: nothing cancels
    vs = ctx.plane(0, "v_scale")
    vs.copy_(scale * (1 + torch.rand(vs.shape, generator=g, device="cuda") / 64) if scale != "spread" else torch.exp2(torch.rand(vs.shape, generator=g, device="cuda") * 32 - 23.5))
    if keys == "one heavy":   # a key some 10 above the others (for the first head of each group) whose value is zero: all that comes out is what the others add
        for s, n in enumerate(slots):
            r = _rows(ctx, s, n)[0]
            ctx.plane(0, "k").view(-1, KH, D)[r] = (127 * q16[s, 0].view(KH, H // KH, D)[:, 0].sign()).to(torch.int8)
            ctx.plane(0, "v").view(-1, KH, D)[r] = 0
            ctx.plane(0, "k_scale").view(-1, KH)[r] = 2.0 ** -6 * 256 / D
    got = ctx.decode(0, range(len(slots)), slots, T, q16, out_dtype=out).view(len(slots), T, H, D)
    ctx.check()
    top = vs.double().max().item()
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[out]
    for s, n in enumerate(slots):
        ref, size = _terms(ctx, s, n, T, q16[s])
        bound = size * (2.0 ** -16 + (0.0 if out == torch.float32 else 2.0 ** -11)) + n * 2.0 ** -40 * 2 * top * 127 + EPS[out] * ref.abs() * 1.01 + tiny
        err = (got[s].to(F8) - ref).abs()
        assert (err <= bound).all(), (s, (err / bound).max().item())
    ctx.close()


@pytest.mark.parametrize("layout", [(24, 4, 256), (32, 8, 128)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slots,T", [([32768], 1), ([9001], 2), ([5000, 20011, 333], 1), ([4096] * 9, 1)])
def test_long_int8_caches_head_by_head(capi, layout, out, slots, T):  # noqa: F811
    """V of random signs: an error e of the p_j v_j, each its own, is an error e of the output's norm whatever the length. Of scores 2 * their error (numerator and
    denominator), of P 2^-11 in one term or 2^-18 with two and the sums, half a step of the output; twice that per token and head. The loss of one CTA's share of the longest cut (one of 37) would be 0.16."""
    H, KH, D = layout
    g = _gen(sum(slots) + T)
    ctx = _context(capi, slots, layout, 32, "int8", fill=g)
    q16 = (_randn(g, len(slots), T, H * D) / math.sqrt(D)).half()
    got = ctx.decode(0, range(len(slots)), slots, T, q16, out_dtype=out).view(len(slots), T, H, D)
    ctx.check()
    for s, n in enumerate(slots):
        ref, _, mag = _attend(ctx, 0, s, n, T, q16[s])
        d = 2 * _score_error(ctx, q16[s], mag, True) + EPS[out] + (2.0 ** -18 if out == torch.float32 else 2.0 ** -11)
        rel = (got[s].to(F8) - ref).norm(dim=-1) / ref.norm(dim=-1)
        assert (rel <= 2 * d).all(), (s, rel.max().item(), 2 * d)
    ctx.close()
