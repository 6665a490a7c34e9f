"""kata_paged_decode: token t of a call sees the slots below n_slots - T + 1 + t, and what lies in the others (the rows of the tokens behind it) has no part in it, whatever it is."""
import math

import pytest
import torch

from .test_gpu_paged import F8, _context, _gen, _randn, _rows, capi  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("layout", [(24, 4, 256), (32, 8, 128), (4, 4, 256), (16, 2, 256)])
@pytest.mark.parametrize("page,T", [(16, 2), (64, 3), (32, 8)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_later_tokens_row_has_no_part_in_an_earlier_token(capi, kv, layout, page, T, what):  # noqa: F811
    """The newest token's K and V hold no numbers (an activation that overflowed): the tokens before it do not see them. What they give is what they give beside a row of numbers: bit for bit, or (int8: the
    tile's largest V scale is another) up to 2^-40 of the largest scale and code per slot and some roundings of fp32."""
    H, KH, D = layout
    g = _gen(T + page)
    slots = [T, T + 1, 15, 16, 17, 33, 64, 65, 100, 1500]
    ctx = _context(capi, slots, layout, page, kv, fill=g, weights=True)
    q16 = (_randn(g, len(slots), T, H * D) / math.sqrt(D)).half()
    want = ctx.decode(0, range(len(slots)), slots, T, q16).view(len(slots), T, H, D)
    for s, n in enumerate(slots):
        last = _rows(ctx, s, n)[n - 1]
        for p in ("k", "v"):
            if kv == "fp16":
                ctx.plane(0, p).view(-1, KH, D)[last, :, ::3] = what
            else:
                ctx.plane(0, p + "_scale").view(-1, KH)[last] = what
    got = ctx.decode(0, range(len(slots)), slots, T, q16).view(len(slots), T, H, D)
    ctx.check()
    for s, n in enumerate(slots):
        a, b = got[s, :T - 1], want[s, :T - 1]
        assert torch.equal(a, b) if kv == "fp16" else ((a - b).abs() <= n * 2.0 ** -40 * 0.06 * 127 + 2.0 ** -21 * b.abs().max()).all(), s
    assert torch.isfinite(want).all()
    for s, n in enumerate(slots):   # the newest token sees its own row. (A K scale of +inf and a negative sum make its score -inf: weight 0, and 0 x inf is left open)
        last = _rows(ctx, s, n)[n - 1]
        own = torch.einsum("hgd,hd->hg", q16[s, T - 1].to(F8).view(KH, H // KH, D), ctx.plane(0, "k").view(-1, KH, D)[last].to(F8)).reshape(H)
        seen = got[s, T - 1, :, ::3] if kv == "fp16" else got[s, T - 1][own >= 0] if what == math.inf else got[s, T - 1]
        assert not torch.isfinite(seen).any(), s
    ctx.close()
