"""kata_paged_decode with scores so large that fp32 counts them in whole units: the heaviest key alone remains, nothing overflows."""
import pytest
import torch

from .test_gpu_paged import _context, _gen, _kv, _per_head, _randn, _rows, capi  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [(24, 4, 256), (32, 8, 128), (16, 1, 128)])
@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [2.0 ** 21, 2.0 ** 22 * 1.1, 1e7, 1.3e7, 1.9e7, 4e7, 1.7e8, 1e9])
def test_the_heaviest_key_alone_remains(capi, layout, kv, sign, size):  # noqa: F811
    """Scores are size * (1, or 31/32 to 1/32) and, for sign -1, the negatives of these with the heaviest at 1/32: the next one is at least size / 32 > 65,000 below. All of them are small integers times a power of two, times size's
    own fp16 rounding: the same in fp32 and 64 bits up to roundings, and exp of the difference is 0."""
    H, KH, D = layout
    g = _gen(int(size) % 1000)
    slots = [1, 31, 300]
    ctx = _context(capi, slots, layout, 16, kv, fill=g, weights=True)
    ctx.plane(0, "k").zero_()
    if kv == "int8":
        ctx.plane(0, "k_scale").fill_(256.0)
        ctx.plane(0, "v_scale").fill_(0.999 / 64)   # just below a power of two: P at the top of its range
    unit = 32 * 256.0 if kv == "int8" else 32 * 1024.0      # the key of weight 1: codes of 32, or values of 32 * 1024
    n_dims = next(n for n in range(1, D + 1) if size / unit / n <= 60000)
    heavy = []
    for s, n in enumerate(slots):
        r = _rows(ctx, s, n)
        part = torch.randint(1, 32, (n,), generator=g, device="cuda") if sign > 0 else torch.randint(2, 33, (n,), generator=g, device="cuda")
        heavy.append(n * 5 // 7)
        part[heavy[-1]] = 32 if sign > 0 else 1
        ctx.plane(0, "k").view(-1, KH, D)[r, :, :n_dims] = (sign * part * (1 if kv == "int8" else 1024))[:, None, None].to(ctx.plane(0, "k").dtype)
    q16 = torch.zeros(len(slots), 1, H, D, device="cuda", dtype=torch.float16)
    q16[..., :n_dims] = size / unit / n_dims
    got = ctx.decode(0, range(len(slots)), slots, 1, q16.view(len(slots), 1, H * D), accumulate=True).view(len(slots), H, D)
    ctx.check()
    for s, n in enumerate(slots):
        want = _kv(ctx, 0, s, n)[1][heavy[s]][:, None].expand(KH, H // KH, D).reshape(H, D)
        # one key: two fp16 terms of P, one product, and the division: 2^-21 in all; the weight is 1 per head
        assert ((got[s].double() - want).abs() <= 2.0 ** -21 * want.abs()).all(), (s, (got[s].double() - want).abs().max().item())
        w = _per_head(ctx, 0, "weight", s, n).double()
        one = torch.zeros_like(w)
        one[:, heavy[s]] = H // KH
        assert ((w - one).abs() <= 2.0 ** -20 * one).all(), s
    ctx.close()
