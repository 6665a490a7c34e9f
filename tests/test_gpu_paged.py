"""The paged cache on the GPU: prep with positions of up to three axes, attention over pages, accumulated attention weights, eviction, shared prefixes, rows taken over
from a contiguous context, each against a plain evaluation in 64 bits, and a run of them together.

Tolerances are those of the arithmetic: half a step of the output type (2^-11 fp16, 2^-8 bf16, 2^-24 fp32, relative), fp16 products summed in fp32
(an error of a score of at most 32 * 2^-23 of the sum of its terms' magnitudes: 16 chained matrix instructions of 16 terms), probabilities rounded to
fp16 for 16-bit outputs (2^-11), int8 codes carried with a bias of 1152 for those."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float64
EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def capi():
    from kata_b200 import capi as m
    assert torch.cuda.is_available()
    m.lib()
    return m


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _context(capi, slots, layout=(24, 4, 256), page=16, kv="fp16", fill=None, spare=3, n_layers=1, **kw):
    """A context whose sequences hold `slots` reserved slots, pages interleaved between them (16 slots at a time, round robin)."""
    H, KH, D = layout
    top = max(max(slots), 1)
    ctx = capi.PagedContext(n_layers, len(slots), sum(-(-s // page) for s in slots) + spare, page, min(top + 2 * page, 524288), heads=H, kv_heads=KH, head_dim=D, kv_mode=kv, rot_dim=kw.pop("rot_dim", 64), **kw)
    step = max(16, top // 8)
    for upto in range(step, top + step, step):
        for s, n in enumerate(slots):
            ctx.reserve(s, min(n, upto))
    if fill is not None:
        for l in range(n_layers):
            for p in ("k", "v"):
                t = ctx.plane(l, p)
                t.copy_(torch.randint(-127, 128, t.shape, generator=fill, device="cuda") if kv == "int8" else _randn(fill, *t.shape))
                if kv == "int8":
                    t = ctx.plane(l, p + "_scale")
                    t.copy_(0.01 + 0.02 * torch.rand(t.shape, generator=fill, device="cuda"))
    return ctx


def _rows(ctx, seq, n, device="cuda"):
    """Row of the pool (page * page_size + offset) of slots [0, n) of a sequence."""
    t = torch.tensor(ctx.pages(seq) or [0], device=device)
    s = torch.arange(n, device=device)
    return t[s // ctx.page_size] * ctx.page_size + s % ctx.page_size


def _kv(ctx, layer, seq, n):
    """Slots [0, n) of a sequence as fp64 values: k, v [n][kv_heads][head_dim]."""
    r, out = _rows(ctx, seq, n), []
    for p in ("k", "v"):
        x = ctx.plane(layer, p).reshape(-1, ctx.kv_heads, ctx.head_dim)[r].to(F8)
        out.append(x * ctx.plane(layer, p + "_scale").reshape(-1, ctx.kv_heads)[r].to(F8)[..., None] if ctx.kv_mode == "int8" else x)
    return out


def _per_head(ctx, layer, name, seq, n):
    """weight or age of slots [0, n): [kv_heads][n]."""
    r = _rows(ctx, seq, n)
    return ctx.plane(layer, name)[r // ctx.page_size, :, r % ctx.page_size].T


def _attend(ctx, layer, seq, n, T, q16):
    """fp64: outputs [T][heads][head_dim], the weights received [kv_heads][n], and the largest sum of |q k| term magnitudes."""
    KH, G, D = ctx.kv_heads, ctx.heads // ctx.kv_heads, ctx.head_dim
    k, v = _kv(ctx, layer, seq, n)
    q = q16.to(F8).view(T, KH, G, D)
    out, w, mag = torch.zeros(T, KH, G, D, dtype=F8, device="cuda"), torch.zeros(KH, n, dtype=F8, device="cuda"), 0.0
    for t in range(T):
        m = n - T + 1 + t
        if m <= 0:
            continue
        p = torch.softmax(torch.einsum("hgd,lhd->hgl", q[t], k[:m]), -1)
        out[t] = torch.einsum("hgl,lhd->hgd", p, v[:m])
        w[:, :m] += p.sum(1)
        mag = max(mag, torch.einsum("hgd,lhd->hgl", q[t].abs(), k[:m].abs()).max().item())
    return out.view(T, KH * G, D), w, mag


def _score_error(ctx, q16, mag, fine):
    """Largest error of a score: 32 * 2^-23 of its terms' magnitudes; biased int8 codes are up to 1279 instead of their own size."""
    if ctx.kv_mode == "int8" and not fine:
        mag = q16.float().view(-1, ctx.head_dim).abs().sum(-1).max().item() * 1279 * 0.03
    return 32 * 2.0 ** -23 * mag


def _check_out(ctx, got, ref, q16, mag, n, out_dtype):
    """got, ref [T][heads][head_dim] against each other, by norm: a relative error e of the probabilities moves the output by at most 2 e of its terms' norm."""
    fine = out_dtype == torch.float32
    d = 2 * _score_error(ctx, q16, mag, fine) + EPS[out_dtype] + (2.0 ** -18 if fine else 2.0 ** -11)
    if ctx.kv_mode == "int8" and not fine:   # the bias of the value codes, summed over n slots in fp32 and taken out again
        d += (n / 16 + 32) * 2.0 ** -23 * 1279 * 0.03 / max(ref.abs().mean().item(), 1e-3)
    assert torch.isfinite(got).all()
    rel = (got.to(F8) - ref).norm() / ref.norm().clamp_min(1e-30)
    assert rel.item() <= 2 * d, (rel.item(), 2 * d)
    assert (got.to(F8) - ref).abs().max().item() <= 40 * d * max(ref.abs().max().item(), 1e-30)


# ---------------------------------------------------------------------------------------------------------- decode
LAYOUTS = [(24, 4, 256), (32, 8, 128), (4, 4, 256), (16, 1, 128), (16, 2, 256), (6, 3, 128)]


@pytest.mark.parametrize("kv", ["fp16", "int8"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page,T,out", [(16, 1, torch.float32), (16, 2, torch.bfloat16), (32, 1, torch.float16), (64, 3, torch.float32), (128, 8, torch.bfloat16), (1024, 1, torch.float32)])
def test_decode_matches_64_bits(capi, layout, kv, page, T, out):
    g = _gen(layout[0] * 31 + page + T)
    slots = [1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 100, 129, 257, 700, 0]
    ctx = _context(capi, slots, layout, page, kv, fill=g)
    H, KH, D = layout
    q16 = (_randn(g, len(slots), T, H * D) / math.sqrt(D)).half()
    gate = _randn(g, len(slots), T, H * D) if layout[0] != 32 else None
    if kv == "fp16":   # nothing behind a sequence's end may matter
        for s, n in enumerate(slots):
            cap = len(ctx.pages(s)) * page
            r = _rows(ctx, s, cap)[n:]
            for p in ("k", "v"):
                ctx.plane(0, p).view(-1, KH, D)[r] = float("nan") if s % 2 else float("inf")
    got = ctx.decode(0, range(len(slots)), slots, T, q16, gate, out_dtype=out).view(len(slots), T, H, D)
    ctx.check()
    for s, n in enumerate(slots):
        ref, _, mag = _attend(ctx, 0, s, n, T, q16[s])
        if gate is not None:
            ref = ref * torch.sigmoid(gate[s].to(F8)).view(T, H, D)
        for t in range(T):
            if n - T + 1 + t <= 0:
                assert (got[s, t] == 0).all()
        _check_out(ctx, got[s], ref, q16[s], mag, n, out) if n else None
    ctx.close()


@pytest.mark.parametrize("kv,out", [("fp16", torch.float32), ("fp16", torch.float16), ("int8", torch.bfloat16), ("int8", torch.float32)])
@pytest.mark.parametrize("slots,T,page", [([9001], 1, 16), ([32768], 2, 64), ([5000, 20011, 333], 1, 32), ([4096] * 9, 1, 128)])
def test_decode_split_over_many_ctas(capi, kv, out, slots, T, page):
    g = _gen(sum(slots) + T)
    ctx = _context(capi, slots, page=page, kv=kv, fill=g)
    q16 = (_randn(g, len(slots), T, 6144) / 16).half()
    gate = _randn(g, len(slots), T, 6144)
    got = ctx.decode(0, range(len(slots)), slots, T, q16, gate, out_dtype=out)
    again = ctx.decode(0, range(len(slots)), slots, T, q16, gate, out_dtype=out)
    ctx.check()
    assert torch.equal(got, again)   # the split and the joins have one order
    for s, n in enumerate(slots):
        ref, _, mag = _attend(ctx, 0, s, n, T, q16[s])
        _check_out(ctx, got[s].view(T, 24, 256), ref * torch.sigmoid(gate[s].to(F8)).view(T, 24, 256), q16[s], mag, n, out)
    ctx.close()


def test_decode_of_a_full_batch_and_the_same_sequence_twice(capi):
    g = _gen(3)
    slots = [1 + 7 * i % 90 for i in range(256)]
    ctx = _context(capi, slots, (4, 2, 128), 16, fill=g)
    q16 = (_randn(g, 256, 1, 512) / 12).half()
    got = ctx.decode(0, range(256), slots, 1, q16)
    for s in (0, 100, 255):
        ref, _, mag = _attend(ctx, 0, s, slots[s], 1, q16[s])
        _check_out(ctx, got[s].view(1, 4, 128), ref, q16[s], mag, slots[s], torch.float32)
    two = ctx.decode(0, [100, 7, 100], [slots[100], slots[7], 3], 1, q16[[100, 7, 100]].contiguous())
    assert (two[:2] - got[[100, 7]]).abs().max() < 1e-5
    ref, _, mag = _attend(ctx, 0, 100, 3, 1, q16[100])
    _check_out(ctx, two[2].view(1, 4, 128), ref, q16[100], mag, 3, torch.float32)
    ctx.close()


@pytest.mark.parametrize("layout", [(24, 4, 256), (32, 8, 128)])
@pytest.mark.parametrize("kv,T,out", [("fp16", 1, torch.bfloat16), ("fp16", 2, torch.float32), ("int8", 1, torch.float32), ("int8", 1, torch.bfloat16), ("int8", 3, torch.float16)])
@pytest.mark.parametrize("order", ["mixed", "rising"])
def test_ragged_batches_pass_from_segment_to_segment(capi, layout, kv, T, out, order):
    """CTAs that work on many short segments, on parts of long ones and on whole ones in one launch; the weights of the same pass; the same bits again."""
    H, KH, D = layout
    r = random.Random(T * 7 + KH)
    slots = [0, 1, 7900, 17] + [r.choice([r.randint(1, 200), r.randint(200, 3000), r.randint(3000, 9000)]) for _ in range(36)]
    slots = sorted(slots) if order == "rising" else slots
    g = _gen(sum(slots))
    ctx = _context(capi, slots, layout, 32, kv, fill=g, weights=True)
    if kv == "fp16":
        for s, n in enumerate(slots):
            rows = _rows(ctx, s, len(ctx.pages(s)) * 32)[n:]
            for p in ("k", "v"):
                ctx.plane(0, p).view(-1, KH, D)[rows] = float("nan")
    q16 = (_randn(g, len(slots), T, H * D) / math.sqrt(D)).half()
    got = ctx.decode(0, range(len(slots)), slots, T, q16, out_dtype=out, accumulate=True)
    assert torch.equal(got, ctx.decode(0, range(len(slots)), slots, T, q16, out_dtype=out))
    ctx.check()
    for s, n in enumerate(slots):
        ref, w, mag = _attend(ctx, 0, s, n, T, q16[s])
        if n:
            _check_out(ctx, got[s].view(T, H, D), ref, q16[s], mag, n, out)
            tol = 2 * _score_error(ctx, q16[s], mag, True) + 2.0 ** -20
            assert (_per_head(ctx, 0, "weight", s, n).to(F8) - w).abs().le(tol * w + 2.0 ** -24).all()
        else:
            assert (got[s] == 0).all()
    ctx.close()


@pytest.mark.parametrize("D,kv", [(256, "fp16"), (256, "int8"), (128, "fp16"), (128, "int8")])
def test_decode_at_the_limits_of_heads_and_batch(capi, D, kv):
    """16 query heads on each of 16 KV heads, 256 sequences."""
    g = _gen(D)
    slots = [r % 41 for r in range(256)]
    ctx = _context(capi, slots, (256, 16, D), 16, kv, fill=g, weights=True)
    q16 = (_randn(g, 256, 2, 256 * D) / math.sqrt(D)).half()
    got = ctx.decode(0, range(256), slots, 2, q16, accumulate=True).view(256, 2, 256, D)
    ctx.check()
    for s in (0, 1, 2, 40, 128, 255):
        n = slots[s]
        ref, w, mag = _attend(ctx, 0, s, n, 2, q16[s])
        if n:
            _check_out(ctx, got[s], ref, q16[s], mag, n, torch.float32)
            tol = 2 * _score_error(ctx, q16[s], mag, True) + 2.0 ** -20
            assert (_per_head(ctx, 0, "weight", s, n).to(F8) - w).abs().le(tol * w + 2.0 ** -23).all()   # (two passes: a second sum)
        else:
            assert (got[s] == 0).all()
    ctx.close()


def test_two_graphs_of_one_context_replayed_in_turn(capi):
    """Graphs share the context's scratch; on one stream, one behind the other, each leaves it as the other needs it."""
    g = _gen(11)
    slots = [5000, 40, 2500, 0, 700]
    ctx = _context(capi, slots, fill=g, weights=True)
    q16 = (_randn(g, 5, 2, 6144) / 16).half()
    q = [q16, q16[2:4].contiguous()]
    ids, held = [list(range(5)), [2, 3]], [slots, [2400, 0]]
    want = [ctx.decode(0, ids[i], held[i], 2, q[i]) for i in range(2)]
    base = [(ctx.plane(0, "weight").zero_(), ctx.decode(0, ids[i], held[i], 2, q[i], accumulate=True), ctx.plane(0, "weight").clone())[2] for i in range(2)]
    ctx.plane(0, "weight").zero_()
    outs, graphs, s = [torch.zeros_like(x) for x in want], [], torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                ctx.decode(0, ids[i], held[i], 2, q[i], out=outs[i], accumulate=True)
            graphs.append(gr)
        for i in (0, 1, 1, 0):
            graphs[i].replay()
    torch.cuda.synchronize()
    ctx.check()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    w = 2 * (base[0].to(F8) + base[1].to(F8))
    assert (ctx.plane(0, "weight").to(F8) - w).abs().le(4 * 2.0 ** -24 * w).all()   # four sums, rounded
    ctx.close()


def test_large_scores_and_one_heavy_key(capi):
    """Scores of several hundred, and a key that takes all the weight: nothing overflows, small probabilities vanish."""
    g = _gen(4)
    ctx = _context(capi, [300], fill=g)
    q16 = (_randn(g, 1, 1, 6144) * 4).half()
    r = _rows(ctx, 0, 300)
    ctx.plane(0, "k").view(-1, 4, 256)[r[77]] = q16.view(4, 6, 256)[:, 0] * 4
    got = ctx.decode(0, [0], [300], 1, q16).view(1, 24, 256)
    ref, _, _ = _attend(ctx, 0, 0, 300, 1, q16[0])
    assert torch.isfinite(got).all() and (got.to(F8) - ref)[:, ::6].abs().max().item() < 1e-3   # the heads aimed at the heavy key: its V row alone
    ctx.close()


# ---------------------------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("layout,kv,page,T", [((24, 4, 256), "fp16", 16, 1), ((24, 4, 256), "fp16", 64, 2), ((24, 4, 256), "int8", 32, 5), ((32, 8, 128), "fp16", 16, 3), ((16, 1, 128), "int8", 16, 1), ((4, 4, 256), "fp16", 16, 8)])
def test_weights_are_the_summed_probabilities(capi, layout, kv, page, T):
    g = _gen(page + T)
    H, KH, D = layout
    slots = [1, 16, 33, 130, 1500, 0, 3]
    ctx = _context(capi, slots, layout, page, kv, fill=g, weights=True)
    ctx.plane(0, "weight").fill_(-7.0)
    for s, n in enumerate(slots):
        r = _rows(ctx, s, n)
        ctx.plane(0, "weight")[r // page, :, r % page] = 0.25
    q16 = (_randn(g, len(slots), T, H * D) / math.sqrt(D)).half()
    out = ctx.decode(0, range(len(slots)), slots, T, q16, accumulate=True)
    first = ctx.plane(0, "weight").clone()
    plain = ctx.decode(0, range(len(slots)), slots, T, q16)
    assert torch.equal(out, plain) and torch.equal(first, ctx.plane(0, "weight"))   # same output; without accumulate nothing is written
    ctx.decode(0, range(len(slots)), slots, T, q16, accumulate=True)
    ctx.check()
    touched = 0
    for s, n in enumerate(slots):
        _, w, mag = _attend(ctx, 0, s, n, T, q16[s])
        if not n:
            continue
        tol = 2 * _score_error(ctx, q16[s], mag, True) + 2.0 ** -20   # fp32 outputs: unbiased codes
        r = _rows(ctx, s, n)
        got1, got2 = first[r // page, :, r % page].T.to(F8), _per_head(ctx, 0, "weight", s, n).to(F8)
        assert ((got1 - 0.25) - w).abs().le(tol * w + 2.0 ** -24).all() and ((got2 - 0.25) - 2 * w).abs().le(2 * tol * w + 2.0 ** -23).all()
        touched += n * KH
    assert int((ctx.plane(0, "weight") == -7.0).sum()) == ctx.plane(0, "weight").numel() - touched   # slots no sequence holds are left alone
    ctx.close()


def test_weights_refuse_a_sequence_named_twice_and_contexts_without_them(capi):
    ctx = _context(capi, [20, 20], weights=True)
    q16 = torch.zeros(2, 1, 6144, dtype=torch.float16, device="cuda")
    with pytest.raises(capi.KataError) as e:
        ctx.decode(0, [1, 1], [20, 20], 1, q16, accumulate=True)
    assert e.value.code == 1
    bare = _context(capi, [20])
    for call in (lambda: bare.decode(0, [0], [20], 1, q16[:1], accumulate=True), lambda: bare.evict(0, [0], [20], 8, 20)):
        with pytest.raises(capi.KataError) as e:
            call()
        assert e.value.code == 3


# ---------------------------------------------------------------------------------------------------------- eviction
def _expected_eviction(w, age, n, keep, seen, sink, recent):
    """[kv_heads][n] weights and ages -> src [kv_heads][keep]."""
    KH = w.shape[0]
    src = torch.full((KH, keep), -1, dtype=torch.int32)
    for h in range(KH):
        if n <= keep:
            src[h, :n] = torch.arange(n, dtype=torch.int32)
            continue
        x, a = w[h].tolist(), age[h].tolist()
        key = [math.inf if a[j] < sink or a[j] >= seen - recent else (-math.inf if math.isnan(x[j]) else x[j]) for j in range(n)]
        nan = [math.isnan(x[j]) and not (a[j] < sink or a[j] >= seen - recent) for j in range(n)]
        order = sorted(range(n), key=lambda j: (nan[j], -key[j], j))
        kept = set(order[:keep])
        movers = iter(sorted(j for j in kept if j >= keep))
        for j in range(keep):
            src[h, j] = j if j in kept else next(movers)
    return src


@pytest.mark.parametrize("layout,kv,page", [((24, 4, 256), "fp16", 16), ((24, 4, 256), "int8", 64), ((32, 8, 128), "fp16", 32), ((16, 1, 128), "int8", 16)])
@pytest.mark.parametrize("slots,keep,sink,recent", [([40, 17, 16, 3, 0], 16, 0, 0), ([65, 64, 100, 33], 33, 4, 10), ([1000, 1001, 64], 64, 64, 0), ([2500, 700], 500, 1, 499), ([300], 1, 0, 0), ([300, 260], 299, 0, 7)])
def test_eviction_keeps_the_heaviest(capi, layout, kv, page, slots, keep, sink, recent):
    g = _gen(keep + page)
    H, KH, D = layout
    ctx = _context(capi, slots, layout, page, kv, fill=g, weights=True)
    w = ctx.plane(0, "weight")
    w.copy_((torch.rand(w.shape, generator=g, device="cuda") * 40).floor() / 8)     # many equal ones
    w[torch.rand(w.shape, generator=g, device="cuda") < 0.02] = float("nan")
    w[torch.rand(w.shape, generator=g, device="cuda") < 0.02] = float("inf")
    w[torch.rand(w.shape, generator=g, device="cuda") < 0.02] = -0.0
    seen = []
    for s, n in enumerate(slots):
        r = _rows(ctx, s, n)
        seen.append(n + 13 * s)
        if n:
            a = torch.stack([torch.randperm(seen[s], generator=g, device="cuda")[:n] for _ in range(KH)])
            ctx.plane(0, "age")[r // page, :, r % page] = a.T.int()
    names = ("k", "v", "weight", "age") + (("k_scale", "v_scale") if kv == "int8" else ())
    before = {p: ctx.plane(0, p).clone() for p in names}
    old = [{"kv": _kv(ctx, 0, s, n), "w": _per_head(ctx, 0, "weight", s, n).clone(), "a": _per_head(ctx, 0, "age", s, n).clone()} for s, n in enumerate(slots)]
    src = ctx.evict(0, range(len(slots)), slots, keep, seen, sink=sink, recent=recent)
    ctx.check()
    for s, n in enumerate(slots):
        want = _expected_eviction(old[s]["w"].cpu(), old[s]["a"].cpu(), n, keep, seen[s], sink, recent)
        assert torch.equal(src[s].cpu(), want)
        m = min(n, keep)
        if not m:
            continue
        at, h = src[s, :, :m].long(), torch.arange(KH, device="cuda")[:, None]
        for x, y in zip(_kv(ctx, 0, s, m), old[s]["kv"]):
            assert torch.equal(x.permute(1, 0, 2), y[at, h])
        assert torch.equal(_per_head(ctx, 0, "weight", s, m).contiguous().view(torch.int32), old[s]["w"].contiguous()[h, at].view(torch.int32))
        assert torch.equal(_per_head(ctx, 0, "age", s, m), old[s]["a"][h, at])
    # everything but the holes that were filled is as it was
    for p in names:
        x, y = ctx.plane(0, p), before[p]
        same = torch.ones(ctx.n_pages * page, KH, dtype=torch.bool, device="cuda")
        for s, n in enumerate(slots):
            if n > keep:
                filled = src[s] != torch.arange(keep, device="cuda")
                r = _rows(ctx, s, keep)
                for hh in range(KH):
                    same[r[filled[hh]], hh] = False
        a, b = (z.permute(0, 2, 1).reshape(-1, KH) if p in ("weight", "age") else z.reshape(-1, KH, *z.shape[3:]) for z in (x, y))
        assert torch.equal(a[same].contiguous().view(torch.uint8), b[same].contiguous().view(torch.uint8))
    ctx.close()


def test_eviction_of_several_layers_and_of_long_sequences(capi):
    """Layers in one call; more slots than the keys' share of shared memory holds."""
    g = _gen(9)
    slots, keep = [60000, 20000], 5000
    ctx = _context(capi, slots, (2, 2, 128), 256, weights=True, n_layers=3)
    for l in (1, 2):
        ctx.plane(l, "weight").copy_(torch.rand(ctx.plane(l, "weight").shape, generator=g, device="cuda").square())
        ctx.plane(l, "age").fill_(10)
        ctx.plane(l, "k").copy_(torch.arange(ctx.n_pages * 256, device="cuda").view(-1, 256, 1, 1).remainder(2048).expand_as(ctx.plane(l, "k")))
    old = {(l, s): (_per_head(ctx, l, "weight", s, n).clone(), _kv(ctx, l, s, n)[0]) for l in (1, 2) for s, n in enumerate(slots)}
    src = ctx.evict(1, [0, 1], slots, keep, 70000, recent=100, n_layers=2)
    ctx.check()
    assert tuple(src.shape) == (2, 2, 2, keep)
    for l in (1, 2):
        for s, n in enumerate(slots):
            w, k = old[l, s]
            order = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :keep]
            got = src[l - 1, s].long()
            assert torch.equal(got.sort(-1).values, order.sort(-1).values)
            stay = got < keep
            assert torch.equal(got[stay], torch.arange(keep, device="cuda").expand(2, keep)[stay])
            assert all((got[h][~stay[h]].diff() > 0).all() for h in range(2))
            assert torch.equal(_kv(ctx, l, s, keep)[0].permute(1, 0, 2), k[got, torch.arange(2, device="cuda")[:, None]])
    ctx.close()


def _expected_on_gpu(w, keep):
    """[kv_heads][n] weights -> src [kv_heads][keep], nothing protected."""
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :keep]
    kept = torch.zeros_like(w, dtype=torch.bool).scatter_(-1, order, True)
    src = torch.arange(keep, device=w.device).repeat(w.shape[0], 1)
    for h in range(w.shape[0]):
        src[h, ~kept[h, :keep]] = torch.nonzero(kept[h, keep:])[:, 0] + keep
    return src


@pytest.mark.parametrize("values", ["spread", "eighths", "equal", "sparse", "rising", "falling"])
@pytest.mark.parametrize("n,slots", [(1, 5120), (1, 5121), (2, 9999), (64, 1500), (40, 5300), (33, 12289), (1, 32768), (1, 32769), (1, 131072), (1, 131073), (1, 524288)])
def test_selection_of_any_size_and_any_ties(capi, n, slots, values):
    """One CTA or a cluster per head, bounds or a radix select, few and many heads: the same slots."""
    if n * slots > 100000 and values in ("rising", "sparse"):
        values = "spread"
    g = _gen(slots + n)
    ctx = _context(capi, [slots] * n, (2, 2, 128), 1024 if slots > 20000 else 64, weights=True, spare=0)
    mk = {"spread": lambda *s: torch.rand(s, generator=g, device="cuda").square(), "eighths": lambda *s: (torch.rand(s, generator=g, device="cuda") * 8).floor(), "equal": lambda *s: torch.zeros(s, device="cuda"),
          "sparse": lambda *s: torch.rand(s, generator=g, device="cuda") * (torch.rand(s, generator=g, device="cuda") < 0.1), "rising": lambda *s: torch.arange(s[-1], device="cuda").expand(s).float(),
          "falling": lambda *s: -torch.arange(s[-1], device="cuda").expand(s).float()}[values]
    w = mk(n, 2, slots)
    ctx.plane(0, "age").fill_(10 ** 6)
    page = ctx.page_size
    rows = torch.stack([_rows(ctx, s, slots) for s in range(n)])
    for keep in (1, slots // 8, slots // 2, slots - 1):
        for s in range(n):
            ctx.plane(0, "weight")[rows[s] // page, :, rows[s] % page] = w[s].T
        src = ctx.evict(0, range(n), [slots] * n, keep, 10 ** 7)
        ctx.check()
        for s in range(n):
            assert torch.equal(src[s].long(), _expected_on_gpu(w[s], keep)), (keep, s)
        assert torch.equal(torch.stack([_per_head(ctx, 0, "weight", s, keep) for s in range(n)]), w.gather(2, src.long()))
        ctx.plane(0, "age").fill_(10 ** 6)
    ctx.close()


def test_eviction_refusals(capi):
    ctx = _context(capi, [40, 40], weights=True)
    for kw, code in ((dict(keep=0), 2), (dict(keep=8, sink=5, recent=4), 2), (dict(keep=8, sink=-1), 2), (dict(keep=8, recent=-1), 2), (dict(keep=100000), 2)):
        with pytest.raises(capi.KataError) as e:
            ctx.evict(0, [0], [40], seen=40, src=torch.empty(1, 4, kw["keep"], dtype=torch.int32, device="cuda"), **kw)
        assert e.value.code == code
    for args, code in (((0, [0, 0], [40, 40], 8, 40), 1), ((1, [0], [40], 8, 40), 2), ((0, [2], [40], 8, 40), 2), ((0, [0], [49], 8, 40), 2), ((0, [0], [-1], 8, 40), 2), ((0, [0], [40], 8, -1), 2)):
        with pytest.raises(capi.KataError) as e:
            ctx.evict(*args)
        assert e.value.code == code
    with pytest.raises(capi.KataError) as e:
        ctx.evict(0, [0], [40], 8, 40, n_layers=2)
    assert e.value.code == 2


# ---------------------------------------------------------------------------------------------------------- prep
def _rotated(x, w, pos, axis_of, theta, rot):
    """fp64: x [n][T][heads][hd], pos [n][T][3] -> normed and rotated, and the pair magnitudes."""
    R = rot // 2
    y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.to(F8)
    if not R:
        return y, y.abs()
    f = torch.tensor([theta ** (-i / R) for i in range(R)], dtype=F8, device="cuda")
    ang = (pos.to(F8)[..., axis_of] * f)[:, :, None]
    a, b = y[..., :R], y[..., R:rot]
    m = (a.square() + b.square()).sqrt()
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), y[..., rot:]], -1), torch.cat([m, m, y[..., rot:].abs()], -1)


def _near16(got, ref, mag):
    """fp16 values of fp32 arithmetic: half a step, plus 2^-20 of the rotary pair's size for the norm (12 summation steps), the turn and the products."""
    return ((got.to(F8) - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -20 * mag + 2.0 ** -25).all()


AXES = {"text": ((32, 0, 0), False), "parts": ((8, 12, 12), False), "interleaved": ((11, 11, 10), True)}


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout,page", [((24, 4, 256), 16), ((32, 8, 128), 64), ((6, 3, 256), 32)])
@pytest.mark.parametrize("axes,rot", [("text", 64), ("parts", 64), ("interleaved", 64), ("whole", None), ("none", 0)])
def test_prep_matches_64_bits(capi, act, layout, page, axes, rot):
    g = _gen(7 + page)
    H, KH, D = layout
    n, T, slot0, theta = 3, 21, [0, 13, 40], 1e7 if axes != "whole" else 5e5
    rot = D if rot is None else rot
    sec, inter = AXES[axes] if axes in AXES else ((rot // 2, 0, 0), False) if axes == "none" else ((rot // 2 - 16, 6, 10), False)
    ctx = _context(capi, [s + T for s in slot0], layout, page, rot_dim=rot, theta=theta, sections=sec, interleaved=inter, weights=True)
    for p in ("k", "v"):
        ctx.plane(0, p).fill_(5.0)
    ctx.plane(0, "weight").fill_(3.0)
    ctx.plane(0, "age").fill_(-4)
    q, k, v = _randn(g, n, T, H, 2 * D).to(act), _randn(g, n, T, KH, D).to(act), _randn(g, n, T, KH, D).to(act)
    qn, kn = 1 + 0.05 * _randn(g, D), 1 + 0.05 * _randn(g, D)
    pos = torch.randint(0, 2 ** 31 - 1, (n, T, 3), generator=g, device="cuda", dtype=torch.int64)
    pos[0] //= 1 << 16
    pos[1] = -pos[1]
    age0 = [100, 13, 7]
    q16, _, gate = ctx.prep(0, range(n), slot0, T, q, k, v, qn, kn, axis_pos=pos.int().contiguous(), age0=age0)
    ctx.check()
    i = torch.arange(rot // 2, device="cuda")
    axis_of = torch.where((i % 3 == 1) & (i < 3 * sec[1]), 1, torch.where((i % 3 == 2) & (i < 3 * sec[2]), 2, 0)) if inter else torch.tensor([0] * sec[0] + [1] * sec[1] + [2] * sec[2], dtype=torch.long, device="cuda")
    rq, mq = _rotated(q[..., :D].to(F8), qn, pos, axis_of, theta, rot)
    rk, mk = _rotated(k.to(F8), kn, pos, axis_of, theta, rot)
    assert _near16(q16.view(n, T, H, D), rq / math.sqrt(D), mq / math.sqrt(D)) and torch.equal(gate.view(n, T, H, D), q[..., D:].float())
    left = torch.ones(ctx.n_pages * page, dtype=torch.bool, device="cuda")
    for s in range(n):
        r = _rows(ctx, s, slot0[s] + T)[slot0[s]:]
        left[r] = False
        assert _near16(ctx.plane(0, "k").view(-1, KH, D)[r], rk[s], mk[s]) and torch.equal(ctx.plane(0, "v").view(-1, KH, D)[r], v[s].half())
        assert (ctx.plane(0, "weight")[r // page, :, r % page] == 0).all()
        assert torch.equal(ctx.plane(0, "age")[r // page, :, r % page], (age0[s] + torch.arange(T, device="cuda"))[:, None].expand(T, KH).int())
    assert (ctx.plane(0, "k").view(-1, KH, D)[left] == 5).all() and (ctx.plane(0, "v").view(-1, KH, D)[left] == 5).all()   # nothing else is touched
    assert (ctx.plane(0, "weight").permute(0, 2, 1).reshape(-1, KH)[left] == 3).all() and (ctx.plane(0, "age").permute(0, 2, 1).reshape(-1, KH)[left] == -4).all()
    ctx.close()


@pytest.mark.parametrize("layout", [(24, 4, 256), (32, 8, 128)])
@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
def test_prep_int8_quantises_the_fp16_rows(capi, layout, act):
    g = _gen(11)
    H, KH, D = layout
    T, n = 37, 2
    k, v, kn = _randn(g, n, T, KH, D).to(act), _randn(g, n, T, KH, D).to(act), 1 + 0.05 * _randn(g, D)
    v[0, 3] = 0.0
    v[1, 5, 0, :] = 1e-6
    a, b = (_context(capi, [T] * n, layout, 32, kv) for kv in ("fp16", "int8"))
    for c in (a, b):
        assert c.prep(0, range(n), [0] * n, T, None, k, v, None, kn) == (None, None, None)   # K and V alone, text positions
        c.check()
    for s in range(n):
        r = _rows(a, s, T)
        for p in ("k", "v"):
            x = a.plane(0, p).view(-1, KH, D)[r].float()
            top = x.abs().amax(-1)
            sc = torch.where(top > 0, top / 127, torch.ones_like(top)).half()
            codes = torch.clamp(torch.round(x * (1 / sc.float())[..., None]), -127, 127).to(torch.int8)
            assert torch.equal(b.plane(0, p + "_scale").view(-1, KH)[_rows(b, s, T)], sc) and torch.equal(b.plane(0, p).view(-1, KH, D)[_rows(b, s, T)], codes)


def test_text_positions_are_three_equal_axes_and_agree_with_the_contiguous_prep(capi):
    g = _gen(12)
    T, start = 50, 1000
    q, k, v, qn, kn = _randn(g, 1, T, 12288), _randn(g, 1, T, 1024), _randn(g, 1, T, 1024), 1 + 0.05 * _randn(g, 256), 1 + 0.05 * _randn(g, 256)
    ctx, other = _context(capi, [T], sections=(11, 11, 10), interleaved=True), capi.AttnContext(1, [start + T])
    text = ctx.prep(0, [0], [0], T, q, k, v, qn, kn, age0=[start])
    rows = ctx.plane(0, "k").clone()
    pos = (start + torch.arange(T, device="cuda", dtype=torch.int32)).view(1, T, 1).expand(1, T, 3).contiguous()
    three = ctx.prep(0, [0], [0], T, q, k, v, qn, kn, axis_pos=pos)
    assert torch.equal(text[0], three[0]) and torch.equal(rows, ctx.plane(0, "k"))
    q16, _, gate = other.prep(0, [0], [start], T, q, k, v, qn, kn)
    # the contiguous prep forms its angles in fp32: at position 1050 off by at most 1050 * 2^-23 (product and frequency rounded); values below 8
    assert (q16.float() - text[0].float()).abs().max() <= 8 / 16 * (1050 * 2.0 ** -23 + 2.0 ** -11) and torch.equal(gate, text[2])


def test_prep_refusals(capi):
    ctx = _context(capi, [40, 40], (24, 4, 256), 16)
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    q, k, w = z(1, 4, 12288), z(1, 4, 1024), z(256)
    for call, code in ((lambda: ctx.prep(0, [0], [45], 4, q, k, k, w, w), 2), (lambda: ctx.prep(0, [0], [-1], 4, q, k, k, w, w), 2), (lambda: ctx.prep(1, [0], [0], 4, q, k, k, w, w), 2), (lambda: ctx.prep(0, [2], [0], 4, q, k, k, w, w), 2),
                       (lambda: ctx.prep(0, [0, 0], [0, 8], 2, z(2, 2, 12288), z(2, 2, 1024), z(2, 2, 1024), w, w), 1), (lambda: ctx.prep(0, [0], [0], 4, q, k, k, w, w, age0=[-1]), 2), (lambda: ctx.prep(0, [0], [0], 4, q, k, k, None, w), 1),
                       (lambda: ctx.prep(0, [0], [0], 1025, z(1, 1025, 12288), z(1, 1025, 1024), z(1, 1025, 1024), w, w), 2),
                       (lambda: ctx.prep(0, [0], [0], 1, None, z(1025)[1:].view(1, 1, 1024), z(1, 1, 1024), None, w), 1)):
        with pytest.raises(capi.KataError) as e:
            call()
        assert e.value.code == code
    for call in (lambda: ctx.prep(0, [0], [0], 4, q[..., :6144].contiguous(), k, k, w, w), lambda: ctx.prep(0, [0], [0], 4, q.half(), k, k, w, w), lambda: ctx.prep(0, [0], [0], 4, q, k, k, w, w, axis_pos=torch.zeros(1, 4, 3, device="cuda")),
                 lambda: ctx.prep(0, [0], [0, 1], 4, q, k, k, w, w), lambda: ctx.decode(0, [0], [4], 1, z(1, 6144))):
        with pytest.raises(ValueError):
            call()
    q16 = torch.zeros(1, 1, 6144, dtype=torch.float16, device="cuda")
    for call, code in ((lambda: ctx.decode(0, [0], [49], 1, q16), 2), (lambda: ctx.decode(0, [0], [-1], 1, q16), 2), (lambda: ctx.decode(1, [0], [4], 1, q16), 2), (lambda: ctx.decode(0, [0], [4], 9, torch.zeros(1, 9, 6144, dtype=torch.float16, device="cuda")), 2),
                       (lambda: ctx.decode(0, [], [], 1, q16[:0]), 1)):
        with pytest.raises(capi.KataError) as e:
            call()
        assert e.value.code == code


# ---------------------------------------------------------------------------------------------------------- pages
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_forked_prefix_is_shared_and_read_only(capi, kv):
    g = _gen(13)
    ctx = _context(capi, [100, 0, 0], page=32, kv=kv, fill=g, n_layers=2, spare=8)
    free = ctx.free_pages()
    ctx.fork(0, 1, 90)
    assert ctx.pages(1)[:2] == ctx.pages(0)[:2] and len(ctx.pages(1)) == 3 and ctx.pages(1)[2] != ctx.pages(0)[2] and ctx.free_pages() == free - 1
    q16 = (_randn(g, 1, 1, 6144) / 16).half()
    for l in (0, 1):
        for x, y in zip(_kv(ctx, l, 0, 90), _kv(ctx, l, 1, 90)):
            assert torch.equal(x, y)
        assert torch.equal(ctx.decode(l, [0], [90], 1, q16), ctx.decode(l, [1], [90], 1, q16))
    k, w = _randn(g, 1, 1, 1024), torch.ones(256, device="cuda")
    for seq, slot in ((0, 63), (1, 0)):
        with pytest.raises(capi.KataError) as e:
            ctx.prep(0, [seq], [slot], 1, None, k, k, None, w)
        assert e.value.code == 3
    before = _kv(ctx, 0, 0, 100)
    ctx.prep(0, [1], [90], 1, None, k, k, None, w)     # behind the shared pages: dst's own
    assert all(torch.equal(x, y) for x, y in zip(before, _kv(ctx, 0, 0, 100)))
    ctx.trim(1)
    ctx.prep(0, [0], [0], 1, None, k, k, None, w)      # its own again
    with pytest.raises(capi.KataError) as e:
        ctx.fork(0, 0, 10)
    assert e.value.code == 2
    with pytest.raises(capi.KataError) as e:
        _context(capi, [40, 0], weights=True).fork(0, 1, 40)
    assert e.value.code == 3


@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_prompt_goes_on_in_pages(capi, kv):
    """prep + prefill in a contiguous context, the rows taken over, the next token in pages: the same as going on in the contiguous one."""
    g = _gen(14)
    L = 150
    arena = capi.AttnContext(2, [200], kv_mode=kv)
    ctx = _context(capi, [L + 1], page=32, kv=kv, n_layers=2, weights=True)
    qn, kn = 1 + 0.05 * _randn(g, 256), 1 + 0.05 * _randn(g, 256)
    for l in (0, 1):
        arena.prep(l, [0], [0], L, None, _randn(g, 1, L, 1024), _randn(g, 1, L, 1024), None, kn, h0=24, nh=8)
        ctx.import_rows(l, 0, 0, 100, arena, l, 0, 0)
        ctx.import_rows(l, 0, 100, L - 100, arena, l, 0, 100)
        q, k, v = _randn(g, 1, 1, 12288), _randn(g, 1, 1, 1024), _randn(g, 1, 1, 1024)
        a16, _, ag = arena.prep(l, [0], [L], 1, q, k, v, qn, kn)
        p16, _, pg = ctx.prep(l, [0], [L], 1, q, k, v, qn, kn)
        want, got = arena.decode(l, [0], [L], 1, a16, ag), ctx.decode(l, [0], [L + 1], 1, p16, pg)
        arena.check(); ctx.check()
        assert (want - got).abs().max() < 2e-3 and (want - got).abs().mean() < 2e-4
        assert torch.equal(_per_head(ctx, l, "age", 0, L + 1), torch.arange(L + 1, device="cuda").expand(4, -1).int()) and (_per_head(ctx, l, "weight", 0, L + 1) == 0).all()
    for args, code in (((0, 0, 0, 201, arena, 0, 0, 0), 2), ((0, 0, 0, 10, arena, 0, 0, 195), 2), ((0, 0, 0, 0, arena, 0, 0, 0), 2), ((0, 0, 150, 11, arena, 0, 0, 0), 2), ((0, 0, 0, 1, arena, 2, 0, 0), 2), ((0, 0, 0, 1, arena, 0, 1, 0), 2), ((0, 0, 0, 1, arena, 0, 0, -1), 2)):
        with pytest.raises(capi.KataError) as e:
            ctx.import_rows(*args)
        assert e.value.code == code
    with pytest.raises(capi.KataError) as e:
        _context(capi, [10], kv="int8" if kv == "fp16" else "fp16", page=32).import_rows(0, 0, 0, 1, arena, 0, 0, 0)
    assert e.value.code == 3


def test_caller_owned_planes_and_a_pool_past_32_bit_offsets(capi):
    """Pools of the caller; a page whose byte and element offsets pass 2^32."""
    pages, page = 2200000, 16          # 35.2 M slots x 128 elements: 4.5e9 elements, 9 GB
    k, v = (torch.zeros(pages * page * 128, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx = capi.PagedContext(1, 2, pages, page, 524288, heads=2, kv_heads=1, head_dim=128, rot_dim=64, planes={"k": k, "v": v})
    ctx.reserve(0, 16)
    with pytest.raises(capi.KataError):
        ctx.reserve(0, 524289)
    L = capi.lib()
    # occupy the pages below with other sequences' tables would take thousands of calls: a context over the pool's end instead
    tail = 40
    last = {p: x.view(pages, page, 1, 128)[-tail:] for p, x in (("k", k), ("v", v))}
    big = capi.PagedContext(pages // tail, 1, tail, page, tail * page, heads=2, kv_heads=1, head_dim=128, rot_dim=64, planes={"k": k, "v": v})
    layer = pages // tail - 1
    big.reserve(0, 600)
    g = _gen(15)
    for x in last.values():
        x.copy_(_randn(g, *x.shape))
    q16 = (_randn(g, 1, 1, 256) / 11).half()
    got = big.decode(layer, [0], [600], 1, q16).view(1, 2, 128)
    ref, _, mag = _attend(big, layer, 0, 600, 1, q16[0])
    _check_out(big, got, ref, q16[0], mag, 600, torch.float32)
    kk = _randn(g, 1, 5, 1, 128)
    big.prep(layer, [0], [590], 5, None, kk, kk, None, torch.ones(128, device="cuda"))
    big.check()
    r = _rows(big, 0, 595)[590:]
    assert torch.equal(big.plane(layer, "v").view(-1, 128)[r], kk.view(5, 128).half())
    assert L.kata_paged_plane_ptr(big.h, layer, 0) == k.data_ptr() + 2 * layer * tail * page * 128
    with pytest.raises(ValueError):
        capi.PagedContext(1, 1, 4, 16, 64, planes={"k": k[:100]})


# ---------------------------------------------------------------------------------------------------------- streams and graphs
def test_captured_step_replays(capi):
    g = _gen(16)
    ctx = _context(capi, [700, 90], fill=g, page=32, weights=True)
    w, src = torch.ones(256, device="cuda"), torch.empty(2, 4, 64, dtype=torch.int32, device="cuda")
    q, k = _randn(g, 2, 1, 12288), _randn(g, 2, 1, 1024)
    q16, gate, out = torch.empty(2, 1, 6144, dtype=torch.float16, device="cuda"), torch.empty(2, 1, 6144, device="cuda"), torch.empty(2, 1, 6144, device="cuda")

    def step():
        ctx.plane(0, "weight").zero_()
        ctx.prep(0, [0, 1], [699, 89], 1, q, k, k, w, w, q16=q16, gate=gate)
        ctx.decode(0, [0, 1], [700, 90], 1, q16, gate, out=out, accumulate=True)
        ctx.evict(0, [1], [90], 64, 90, sink=2, recent=8, src=src[1:])

    keep = {p: ctx.plane(0, p).clone() for p in ("k", "v", "age")}
    step()
    want = (out.clone(), src[1].clone(), ctx.plane(0, "weight").clone(), ctx.plane(0, "k").clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for p, x in keep.items():
            ctx.plane(0, p).copy_(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
            with pytest.raises(capi.KataError) as e:
                ctx.reserve(1, 120)
            assert e.value.code == 3
        for _ in range(2):
            for p, x in keep.items():
                ctx.plane(0, p).copy_(x)
            out.zero_(); src.zero_()
            graph.replay()
        s.synchronize()
    got = (out, src[1], ctx.plane(0, "weight"), ctx.plane(0, "k"))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    ctx.check()


def test_several_calls_behind_one_another_on_another_stream(capi):
    """Layers back to back (each launched while the one before drains), on a stream of the caller's."""
    g = _gen(17)
    n_layers, slots = 6, [333, 2000, 17]
    ctx = _context(capi, slots, fill=g, page=16, n_layers=n_layers, weights=True)
    q16 = (_randn(g, n_layers, 3, 1, 6144) / 16).half()
    one = [ctx.decode(l, [0, 1, 2], slots, 1, q16[l]) for l in range(n_layers)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        two = [ctx.decode(l, [0, 1, 2], slots, 1, q16[l], accumulate=True) for l in range(n_layers)]
        s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    for l in range(n_layers):
        for i, n in enumerate(slots):
            total = _per_head(ctx, l, "weight", i, n).to(F8).sum(-1)
            assert (total - 6).abs().max() < 6 * (n + 16) * 2.0 ** -23 + 1e-5   # six heads, one token: the weights of a KV head add up to 6


# ---------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["fp16", "int8"])
def test_a_sequence_kept_within_a_budget(capi, kv):
    """Image and text tokens appended step by step, their attention weights summed, evicted whenever the budget is passed by a page; the attention over what is left is that of 64 bits over the same
    keys, and the keys that are left are those a plain bookkeeping keeps."""
    g = _gen(18)
    keep, page, sink, recent, steps = 96, 32, 4, 24, 120
    ctx = _context(capi, [keep + page + 8], page=page, kv=kv, weights=True, sections=(11, 11, 10), interleaved=True)
    qn, kn = 1 + 0.05 * _randn(g, 256), 1 + 0.05 * _randn(g, 256)
    first = torch.stack([torch.zeros(60, device="cuda"), torch.arange(60, device="cuda") // 10, torch.arange(60, device="cuda") % 10], -1).int().view(1, 60, 3)
    ctx.prep(0, [0], [0], 60, _randn(g, 1, 60, 12288), _randn(g, 1, 60, 1024), _randn(g, 1, 60, 1024), qn, kn, axis_pos=first)
    slots, seen, evictions = 60, 60, 0
    w = torch.zeros(4, 60, dtype=F8, device="cuda")
    age = torch.arange(60, device="cuda").expand(4, -1)
    for step in range(steps):
        T = 1 + step % 2
        pos = torch.full((1, T, 3), 60 + step, dtype=torch.int32, device="cuda")
        q16, _, gate = ctx.prep(0, [0], [slots], T, _randn(g, 1, T, 12288), _randn(g, 1, T, 1024), _randn(g, 1, T, 1024), qn, kn, axis_pos=pos, age0=[seen])
        slots, seen = slots + T, seen + T
        w = torch.cat([w, torch.zeros(4, T, dtype=F8, device="cuda")], 1)
        age = torch.cat([age, torch.arange(seen - T, seen, device="cuda").expand(4, -1)], 1)
        got = ctx.decode(0, [0], [slots], T, q16, gate, accumulate=True).view(T, 24, 256)
        ref, add, mag = _attend(ctx, 0, 0, slots, T, q16[0])
        _check_out(ctx, got, ref * torch.sigmoid(gate[0].to(F8)).view(T, 24, 256), q16[0], mag, slots, torch.float32)
        w = w + add
        assert (_per_head(ctx, 0, "weight", 0, slots).to(F8) - w).abs().max() < 1e-4 and torch.equal(_per_head(ctx, 0, "age", 0, slots), age.int())
        if slots >= keep + page:
            mine = _per_head(ctx, 0, "weight", 0, slots).clone()
            src = ctx.evict(0, [0], [slots], keep, seen, sink=sink, recent=recent)[0].long()
            assert torch.equal(src.cpu().int(), _expected_eviction(mine.cpu(), age.cpu(), slots, keep, seen, sink, recent))
            w, age, slots, evictions = w.gather(1, src), age.gather(1, src), keep, evictions + 1
            assert all(set(range(sink)) | set(range(seen - recent, seen)) <= set(a.tolist()) for a in age)
            ctx.trim(0, slots)
            assert len(ctx.pages(0)) == keep // page
            ctx.reserve(0, keep + page + 8)
    ctx.check()
    assert evictions >= 3
