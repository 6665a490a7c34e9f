"""Workloads of the paged-cache operators: the multi-axis rotary prep that appends to pages, attention of the newest
tokens over a paged cache (with or without the accumulation of the attention weights), and eviction from that cache.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, angles in 64) or, with ``own`` set,
through ``kata_b200.capi.PagedContext``. The pools, tables and activations are the same tensors either way.

Layouts are the two the library knows: 24 query / 4 KV heads of 256 (rotary part 64) and 32 / 8 heads of 128 (rotary
part 128). Context lengths follow the benchmark's decode configurations (8K, 16K to 32K), chunk lengths its prefill
configurations (512, 1024), and what lies between and below them.
"""
import math
import random

import torch

own = False

THETA = 1e7
EPS = 1e-6


def listed():
    return [
        # one new token of one sequence, behind an image: the latency of a decode step's first kernel
        _prep("prep_token_b1", n=1, T=1, hd=256, act="f32", kv="fp16", page=16, far=30000, sections="11,11,10", interleaved=True),
        # a prefill chunk of 1024 image tokens
        _prep("prep_image_chunk", n=1, T=1024, hd=256, act="bf16", kv="fp16", page=64, far=9000, sections="11,11,10", interleaved=True),
        # eight prompts of an odd length, values and keys quantised as they are appended
        _prep("prep_video_int8_b8", n=8, T=509, hd=256, act="f16", kv="int8", page=32, far=1000, sections="8,12,12", interleaved=False),
        # the latency of attention over a short conversation
        _decode("decode_short_b1", n=1, lo=517, hi=517, T=1, hd=256, kv="fp16", page=16, out="f32", gated=True, weights=False),
        # one long sequence: the cache's length has to be split over the whole GPU
        _decode("decode_long_b1", n=1, lo=32768, hi=32768, T=1, hd=256, kv="fp16", page=64, out="bf16", gated=True, weights=False),
        # eight sequences of 16K to 32K, two tokens each (a speculative pair)
        _decode("decode_pair_b8", n=8, lo=16384, hi=32768, T=2, hd=256, kv="fp16", page=16, out="f16", gated=True, weights=False),
        # a serving batch over an int8 cache, ragged from a few hundred to 32K
        _decode("decode_int8_b32", n=32, lo=300, hi=32768, T=1, hd=256, kv="int8", page=32, out="bf16", gated=True, weights=False),
        # the layout of 32 / 8 heads of 128, no output gate
        _decode("decode_h128_b16", n=16, lo=1000, hi=20000, T=1, hd=128, kv="fp16", page=128, out="f32", gated=False, weights=False),
        # the same attention while a cache budget is kept: the weights of all keys are summed up as well
        _decode("decode_weights_b8", n=8, lo=8192, hi=16384, T=1, hd=256, kv="fp16", page=32, out="bf16", gated=True, weights=True),
        # a budget of 4096 slots exceeded by one page: the regular small eviction of a running sequence
        _evict("evict_page_b1", n=1, lo=4160, hi=4160, keep=4096, hd=256, kv="fp16", page=64, sink=4, recent=512),
        # eight prompts of about 32K cut down to 4096 slots
        _evict("evict_prompt_b8", n=8, lo=30001, hi=32768, keep=4096, hd=256, kv="fp16", page=64, sink=4, recent=512),
        # an int8 cache cut in half
        _evict("evict_half_int8_b4", n=4, lo=16001, hi=16384, keep=8192, hd=256, kv="int8", page=32, sink=64, recent=1024),
    ]


def _prep(name, **c):
    return dict(c, op="prep", **({"name": name} if name else {}))


def _decode(name, **c):
    return dict(c, op="decode", **({"name": name} if name else {}))


def _evict(name, **c):
    return dict(c, op="evict", **({"name": name} if name else {}))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, hd, kv = rng.choice(["prep", "decode", "decode", "evict"]), rng.choice([256, 256, 128]), rng.choice(["fp16", "int8"])
    page = rng.choice([16, 32, 64, 128])
    if op == "prep":
        n = _log(rng, 1, 64)
        half = 32 if hd == 256 else 64
        a = rng.randint(1, half // 3)
        sections, interleaved = ("%d,%d,%d" % (half - 2 * a, a, a), True) if rng.random() < 0.5 else ("%d,%d,%d" % (half // 4, half // 2 - a, half // 4 + a), False)
        return _prep(None, n=n, T=_log(rng, 1, min(1024, 4096 // n)), hd=hd, act=rng.choice(["f32", "bf16", "f16"]), kv=kv, page=page, far=_log(rng, 1, 100000), sections=sections, interleaved=interleaved)
    if op == "decode":
        hi = _log(rng, 1, 32768)
        n = _log(rng, 1, max(1, min(64, 200000 // hi)))
        return _decode(None, n=n, lo=max(1, int(hi * rng.uniform(0.1, 1.0))), hi=hi, T=rng.choice([1, 1, 1, 2, 3, 8]), hd=hd, kv=kv, page=page, out=rng.choice(["f32", "bf16", "f16"]),
                       gated=rng.random() < 0.7, weights=rng.random() < 0.4)
    hi = _log(rng, 200, 32768)
    keep = max(8, int(hi * rng.uniform(0.05, 0.95)))
    return _evict(None, n=rng.randint(1, 8), lo=keep + 1 if keep + 1 <= hi else hi, hi=hi, keep=keep, hd=hd, kv=kv, page=page, sink=rng.randint(0, keep // 8), recent=rng.randint(0, keep // 2))


# ---------------------------------------------------------------------------------------------------------- inputs
_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _heads(c):
    return (24, 4) if c["hd"] == 256 else (32, 8)


def _rot(c):
    return 64 if c["hd"] == 256 else 128


def _lengths(c, lo, hi):
    """A length per sequence. They belong to the case, not to the seed: they say how large the pools are."""
    if c["n"] == 1:
        return [hi]
    r = random.Random(c["n"] * 1000003 + lo * 1009 + hi)
    return [r.randint(lo, hi) for _ in range(c["n"])]


def _tables(slots, page):
    """Pages as a server hands them out while its sequences grow side by side: every sequence takes an eighth of its pages
    at a time, lowest free page first. Returns the reservations in their order and one list of pages per sequence."""
    steps, tables, nxt = [], [[] for _ in slots], 0
    for r in range(1, 9):
        for b, L in enumerate(slots):
            upto = (L * r + 7) // 8
            need = -(-upto // page)
            steps.append((b, upto))
            for _ in range(need - len(tables[b])):
                tables[b].append(nxt)
                nxt += 1
    return steps, tables, nxt


def _cache(c, g, slots, fill):
    """The pools of one layer, and where each sequence's slots lie in them."""
    (_, kvh), hd, page = _heads(c), c["hd"], c["page"]
    steps, tables, n_pages = _tables(slots, page)
    shape = (n_pages, page, kvh, hd)
    s = {"c": c, "slots": slots, "steps": steps, "tables": tables, "n_pages": n_pages}
    if c["kv"] == "int8":
        mk = lambda: torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8) if fill else torch.zeros(shape, dtype=torch.int8, device="cuda")  # noqa: E731
        sc = lambda: ((0.01 + 0.02 * torch.rand(shape[:3], generator=g, device="cuda")) if fill else torch.zeros(shape[:3], device="cuda")).half()  # noqa: E731
        s["k"], s["v"], s["k_scale"], s["v_scale"] = mk(), mk(), sc(), sc()
    else:
        mk = lambda: torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) if fill else torch.zeros(shape, dtype=torch.float16, device="cuda")  # noqa: E731
        s["k"], s["v"] = mk(), mk()
    width = max(len(t) for t in tables)
    pad = torch.tensor([t + [0] * (width - len(t)) for t in tables], device="cuda")
    at = torch.arange(max(slots), device="cuda")
    s["rows"] = pad[:, at // page] * page + at % page            # [n][longest]: row of the pool, 0 behind a sequence's end
    s["len"] = torch.tensor(slots, device="cuda")
    return s


def _handle(s, sections=None, interleaved=False, gated=True, weights=False):
    from kata_b200 import capi
    c, (H, kvh) = s["c"], _heads(s["c"])
    ctx = capi.PagedContext(1, len(s["slots"]), s["n_pages"], c["page"], max(s["slots"]), heads=H, kv_heads=kvh, head_dim=c["hd"], kv_mode=c["kv"], rot_dim=_rot(c), theta=THETA,
                            sections=sections, interleaved=interleaved, gated=gated, weights=weights, planes={p: s[p] for p in ("k", "v", "k_scale", "v_scale", "weight", "age") if p in s})
    for b, upto in s["steps"]:
        ctx.reserve(b, upto)
    if any(ctx.pages(b) != t for b, t in enumerate(s["tables"])):
        raise RuntimeError("the context's pages are not the ones the workload's tables say")
    return ctx


def _axes(c):
    """The axis (0 time, 1 height, 2 width) each rotary frequency takes its position from."""
    st, sh, sw = (int(x) for x in c["sections"].split(","))
    if not c["interleaved"]:
        return torch.tensor([0] * st + [1] * sh + [2] * sw, device="cuda")
    i = torch.arange(st + sh + sw, device="cuda")
    return torch.where((i % 3 == 1) & (i < 3 * sh), 1, torch.where((i % 3 == 2) & (i < 3 * sw), 2, 0))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    (H, kvh), hd, n = _heads(c), c["hd"], c["n"]
    rand = lambda *sh: torch.randn(sh, generator=g, device="cuda")  # noqa: E731
    if c["op"] == "prep":
        T, dt = c["T"], _DT[c["act"]]
        before = _lengths(c, 0, 39)                                                                    # slots that earlier tokens hold
        s = _cache(c, g, [x + T for x in before], fill=False)
        s["slot0"] = before
        s["q"], s["kproj"], s["vproj"] = rand(n, T, H * 2 * hd).to(dt), rand(n, T, kvh * hd).to(dt), rand(n, T, kvh * hd).to(dt)
        s["qnorm"], s["knorm"] = 1 + 0.05 * rand(hd), 1 + 0.05 * rand(hd)
        base = torch.randint(0, c["far"] + 1, (n, 1), generator=g, device="cuda")
        i, gw, gh = torch.arange(T, device="cuda"), 26, 14                                             # frames of 14 x 26 patches
        s["pos"] = torch.stack([base + i // (gw * gh), base + i // gw % gh, base + i % gw], -1).int().contiguous()
        s["axis"] = _axes(c)
        s["new"] = torch.stack([s["rows"][b, x:x + T] for b, x in enumerate(before)])                   # [n][T]: the rows that are appended
        if own:
            s["ctx"] = _handle(s, sections=tuple(int(x) for x in c["sections"].split(",")), interleaved=c["interleaved"])
    elif c["op"] == "decode":
        T = c["T"]
        s = _cache(c, g, [max(x, T) for x in _lengths(c, c["lo"], c["hi"])], fill=True)
        s["q16"] = (rand(n, T, H * hd) / math.sqrt(hd)).half()
        s["gate"] = rand(n, T, H * hd) if c["gated"] else None
        if c["weights"]:
            s["weight"] = torch.rand((s["n_pages"], kvh, c["page"]), generator=g, device="cuda")
            s["age"] = torch.zeros((s["n_pages"], kvh, c["page"]), dtype=torch.int32, device="cuda")
            s["held"] = s["rows"][torch.arange(max(s["slots"]), device="cuda") < s["len"][:, None]]      # rows of the pool that hold a key, sequence after sequence
        if own:
            s["ctx"] = _handle(s, gated=c["gated"], weights=c["weights"])
    else:
        slots = _lengths(c, c["lo"], c["hi"])
        s = _cache(c, g, slots, fill=True)
        L, page = max(slots), c["page"]
        seen = 2 * L
        # ages: the newest `recent` tokens and a random choice of the older ones, in no order (earlier evictions moved them about)
        old = torch.rand((n, kvh, seen - c["recent"]), generator=g, device="cuda").argsort(-1)
        age = torch.cat([torch.arange(seen - c["recent"], seen, device="cuda").expand(n, kvh, -1), old], -1)
        age = age[..., :L].gather(-1, (torch.arange(L, device="cuda") + torch.randint(0, L, (n, kvh, 1), generator=g, device="cuda")) % L)
        w = torch.rand((n, kvh, L), generator=g, device="cuda").square() * 3                           # sums of attention weights: many small, few large,
        w = torch.where(torch.rand((n, kvh, L), generator=g, device="cuda") < 0.05, 0.0, w)             # some never attended at all
        at = torch.arange(L, device="cuda")
        valid = at < s["len"][:, None]
        s["seen"] = seen
        for name, x, dt in (("weight", w, torch.float32), ("age", age, torch.int32)):
            p = torch.zeros((s["n_pages"], page, kvh), dtype=dt, device="cuda")
            p.view(-1, kvh)[s["rows"][valid]] = x.permute(0, 2, 1)[valid].to(dt)
            s[name] = p.permute(0, 2, 1).contiguous()
            s[name + "0"] = s[name].clone()                                                            # as the decode steps before this call left it
        if own:
            s["ctx"] = _handle(s, weights=True)
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _values(codes, scale):
    return codes.float() * scale.float()[..., None]


def _flat(p):
    return p.view(-1, *p.shape[2:])


def _quantised(x):
    """Codes and scales of rows that are rounded to fp16 first: scale = fp16(max / 127), 1 for a row of zeros."""
    x = x.half().float()
    top = x.abs().amax(-1)
    scale = torch.where(top > 0, top / 127, torch.ones_like(top)).half()
    return torch.clamp(torch.round(x * (1 / scale.float())[..., None]), -127, 127).to(torch.int8), scale


def _plain_prep(s):
    c, (H, kvh), hd, R = s["c"], _heads(s["c"]), s["c"]["hd"], _rot(s["c"]) // 2
    n, T = s["pos"].shape[:2]
    freq = THETA ** (-torch.arange(R, dtype=torch.float64, device="cuda") / R)
    angle = s["pos"].double()[..., s["axis"]] * freq
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]

    def turned(x, w):
        x = x * (1 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()) * w
        a, b = x[..., :R], x[..., R:2 * R]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * R:]], -1)

    qg = s["q"].view(n, T, H, 2 * hd).float()
    q16 = (turned(qg[..., :hd], s["qnorm"]) / math.sqrt(hd)).half().view(n, T, -1)
    gate = qg[..., hd:].reshape(n, T, -1)
    k, v = turned(s["kproj"].view(n, T, kvh, hd).float(), s["knorm"]), s["vproj"].view(n, T, kvh, hd).float()
    if c["kv"] == "int8":
        (kc, ks), (vc, vs) = _quantised(k), _quantised(v)
        _flat(s["k"])[s["new"]], _flat(s["v"])[s["new"]], _flat(s["k_scale"])[s["new"]], _flat(s["v_scale"])[s["new"]] = kc, vc, ks, vs
    else:
        _flat(s["k"])[s["new"]], _flat(s["v"])[s["new"]] = k.half(), v.half()
    return q16, gate


def _plain_decode(s):
    c, (H, kvh), hd = s["c"], _heads(s["c"]), s["c"]["hd"]
    n, T = s["q16"].shape[:2]
    G, L = H // kvh, s["rows"].shape[1]
    k, v = (_flat(s[p])[s["rows"]].float() * (_flat(s[p + "_scale"])[s["rows"]].float()[..., None] if c["kv"] == "int8" else 1) for p in ("k", "v"))   # [n][L][kvh][hd]
    q = s["q16"].float().view(n, T, kvh, G, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, T * G, hd)
    x = (q @ k.permute(0, 2, 3, 1)).view(n, kvh, T, G, L)
    sees = torch.arange(L, device="cuda") < (s["len"][:, None] - T + 1 + torch.arange(T, device="cuda"))[:, :, None]   # [n][T][L]
    x = x.masked_fill(~sees[:, None, :, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(n, kvh, T * G, L) @ v.permute(0, 2, 1, 3)).view(n, kvh, T, G, hd).permute(0, 2, 1, 3, 4).reshape(n, T, -1)
    if s["gate"] is not None:
        o = o / (1 + (-s["gate"]).exp())
    if c["weights"]:
        got = p.sum((2, 3)).permute(0, 2, 1)[torch.arange(L, device="cuda") < s["len"][:, None]]          # [held rows][kvh]
        page, off = s["held"] // c["page"], s["held"] % c["page"]
        s["weight"][page, :, off] += got
    return o.to(_DT[c["out"]])


def _plain_evict(s):
    c, (_, kvh), page, keep = s["c"], _heads(s["c"]), s["c"]["page"], s["c"]["keep"]
    n, L = s["rows"].shape
    at, rows = torch.arange(L, device="cuda"), s["rows"][:, :, None].expand(n, L, kvh)
    h = torch.arange(kvh, device="cuda").expand(n, L, kvh)
    w, age = s["weight"][rows // page, h, rows % page].permute(0, 2, 1), s["age"][rows // page, h, rows % page].permute(0, 2, 1)   # [n][kvh][L]
    valid = (at < s["len"][:, None])[:, None]
    w = torch.where((age < c["sink"]) | (age >= s["seen"] - c["recent"]), math.inf, w).masked_fill(~valid, -math.inf)
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros(w.shape, dtype=torch.bool, device="cuda").scatter_(-1, best, True)
    hole, mover = ~kept & (at < keep), kept & (at >= keep)
    moved = torch.zeros((n, kvh, keep + 1), dtype=torch.long, device="cuda").scatter_(-1, torch.where(mover, mover.cumsum(-1) - 1, keep), at.expand(n, kvh, L))
    src = torch.where(hole, moved.gather(-1, (hole.cumsum(-1) - 1).clamp(0, keep)), at)[..., :keep]     # [n][kvh][keep]: where each slot's content comes from
    frm = s["rows"].gather(1, src.permute(0, 2, 1).reshape(n, -1)).view(n, keep, kvh)
    to, hk = s["rows"][:, :keep, None].expand(n, keep, kvh), torch.arange(kvh, device="cuda").expand(n, keep, kvh)
    for p in ("k", "v") + (("k_scale", "v_scale") if c["kv"] == "int8" else ()):
        _flat(s[p])[to, hk] = _flat(s[p])[frm, hk]
    for p in ("weight", "age"):
        s[p][to // page, hk, to % page] = s[p][frm // page, hk, frm % page]
    return src.int()


def run(s):
    c = s["c"]
    if c["op"] == "prep":
        if own:
            q16, _, gate = s["ctx"].prep(0, range(c["n"]), s["slot0"], c["T"], s["q"], s["kproj"], s["vproj"], s["qnorm"], s["knorm"], axis_pos=s["pos"])
        else:
            q16, gate = _plain_prep(s)
        if c["kv"] == "int8":   # the appended rows as the values they stand for
            return {"q16": q16, "gate": gate, "k": _values(_flat(s["k"])[s["new"]], _flat(s["k_scale"])[s["new"]]).half(), "v": _values(_flat(s["v"])[s["new"]], _flat(s["v_scale"])[s["new"]]).half()}
        return {"q16": q16, "gate": gate, "k": s["k"], "v": s["v"]}
    if c["op"] == "decode":
        if own:
            out = s["ctx"].decode(0, range(c["n"]), s["slots"], c["T"], s["q16"], s["gate"], out_dtype=_DT[c["out"]], accumulate=c["weights"])
        else:
            out = _plain_decode(s)
        return {"out": out, "weight": s["weight"]} if c["weights"] else {"out": out}
    s["weight"].copy_(s["weight0"])
    s["age"].copy_(s["age0"])
    if own:
        src = s["ctx"].evict(0, range(c["n"]), s["slots"], c["keep"], s["seen"], sink=c["sink"], recent=c["recent"])
    else:
        src = _plain_evict(s)
    return {p: x for p, x in (("src", src), *((q, s.get(q)) for q in ("k", "v", "k_scale", "v_scale", "weight", "age"))) if x is not None}


# ------------------------------------------------------------------------------------------------------------- work
def _mean_len(c):
    return c["hi"] if c["n"] == 1 else (c["lo"] + c["hi"]) / 2


def work(case):
    c, (H, kvh), hd = case, _heads(case), case["hd"]
    row = 2 * kvh * (hd * (1 if c["kv"] == "int8" else 2) + (2 if c["kv"] == "int8" else 0))           # K and V of one slot
    if c["op"] == "prep":
        tok, e = c["n"] * c["T"], 4 if c["act"] == "f32" else 2
        return {"bytes": tok * ((2 * H + 2 * kvh) * hd * e + H * hd * (2 + 4) + row + 12), "flops": tok * (H + kvh) * hd * 6}
    if c["op"] == "decode":
        keys = c["n"] * max(_mean_len(c), c["T"])
        io = c["n"] * c["T"] * H * hd * (2 + (4 if c["gated"] else 0) + (4 if c["out"] == "f32" else 2))
        return {"bytes": keys * (row + (8 * kvh if c["weights"] else 0)) + io, "flops": keys * c["T"] * H * hd * 4}
    L, keep = _mean_len(c), c["keep"]
    moved = c["n"] * keep * (1 - keep / L) * (1 - c["recent"] / keep)                                   # holes below the budget, filled from above it
    return {"bytes": c["n"] * L * kvh * 8 + c["n"] * keep * kvh * 4 + 2 * moved * (row + 8 * kvh), "flops": c["n"] * L * kvh * 4}


# ------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """From the definitions, sequence by sequence and in 64 bits."""
    s = prepare(case, seed)
    c, (H, kvh), hd, page = s["c"], _heads(s["c"]), case["hd"], case["page"]
    n, f8 = c["n"], torch.float64
    place = lambda b, j: (s["tables"][b][j // page], j % page)  # noqa: E731
    if c["op"] == "prep":
        T, half = c["T"], _rot(c) // 2
        q, kv = s["q"].view(n, T, H, 2, hd).to(f8), {"k": s["kproj"].view(n, T, kvh, hd).to(f8), "v": s["vproj"].view(n, T, kvh, hd).to(f8)}
        st, sh, sw = (int(x) for x in c["sections"].split(","))
        which = [0] * half
        for f in range(half):
            if c["interleaved"]:
                which[f] = 1 if f % 3 == 1 and f // 3 < sh else 2 if f % 3 == 2 and f // 3 < sw else 0
            else:
                which[f] = 0 if f < st else 1 if f < st + sh else 2
        ang = torch.stack([s["pos"][..., which[f]].to(f8) * math.pow(THETA, -f / half) for f in range(half)], -1)
        z = torch.polar(torch.ones_like(ang), ang)[:, :, None]

        def norm_and_turn(x, w):
            y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.to(f8)
            r = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * z
            return torch.cat([r.real, r.imag, y[..., 2 * half:]], -1)

        kv["k"] = norm_and_turn(kv["k"], s["knorm"])
        out = {"q16": (norm_and_turn(q[:, :, :, 0], s["qnorm"]) * hd ** -0.5).reshape(n, T, -1), "gate": q[:, :, :, 1].reshape(n, T, -1)}
        if c["kv"] == "int8":
            for name, x in kv.items():
                x = x.half().to(f8)
                big = x.abs().max(-1).values
                sc = torch.where(big == 0, 1.0, big / 127).half().to(f8)
                out[name] = (x / sc[..., None]).round().clamp(-127, 127) * sc[..., None]
            return out
        for name, x in kv.items():
            pool = torch.zeros(s[name].shape, dtype=f8, device="cuda")
            for b in range(n):
                pg, off = zip(*(place(b, s["slot0"][b] + t) for t in range(T)))
                pool[list(pg), list(off)] = x[b]
            out[name] = pool
        return out
    if c["op"] == "decode":
        T, G = c["T"], H // kvh
        out = torch.zeros(n, T, H, hd, dtype=f8, device="cuda")
        weight = s["weight"].to(f8) if c["weights"] else None
        for b, L in enumerate(s["slots"]):
            pg = torch.tensor(s["tables"][b], device="cuda")
            k, v = ((s[p][pg].to(f8) * (s[p + "_scale"][pg].to(f8)[..., None] if c["kv"] == "int8" else 1.0)).reshape(-1, kvh, hd)[:L] for p in ("k", "v"))
            q = s["q16"][b].to(f8).view(T, kvh, G, hd)
            for t in range(T):
                m = L - T + 1 + t
                p = torch.softmax(torch.einsum("hgd,lhd->hgl", q[t], k[:m]), -1)
                out[b, t] = torch.einsum("hgl,lhd->hgd", p, v[:m]).reshape(H, hd)
                if weight is not None:
                    full = torch.zeros(kvh, len(pg) * page, dtype=f8, device="cuda")
                    full[:, :m] = p.sum(1)
                    weight[pg] += full.view(kvh, len(pg), page).permute(1, 0, 2)
        out = out.view(n, T, H * hd)
        if s["gate"] is not None:
            out = out * torch.sigmoid(s["gate"].to(f8))
        return {"out": out, "weight": weight} if c["weights"] else {"out": out}
    # eviction moves bits and counts: everything it gives is exact already
    got = {p: s[p].clone() for p in ("k", "v", "k_scale", "v_scale", "weight", "age") if p in s}
    src = torch.zeros(n, kvh, c["keep"], dtype=torch.int32, device="cuda")
    for b, L in enumerate(s["slots"]):
        pg = torch.tensor(s["tables"][b], device="cuda")
        row = torch.arange(L, device="cuda")
        for h in range(kvh):
            w, age = s["weight"][pg, h].reshape(-1)[:L].to(f8), s["age"][pg, h].reshape(-1)[:L]
            w[(age < c["sink"]) | (age >= s["seen"] - c["recent"])] = math.inf
            rank = torch.argsort(-w, stable=True)
            stays = torch.zeros(L, dtype=torch.bool, device="cuda")
            stays[rank[:c["keep"]]] = True
            holes, movers = row[:c["keep"]][~stays[:c["keep"]]], row[c["keep"]:][stays[c["keep"]:]]
            from_ = row[:c["keep"]].clone()
            from_[holes] = movers
            src[b, h] = from_.int()
            for p, x in got.items():
                if p in ("weight", "age"):
                    x[pg[holes // page], h, holes % page] = s[p][pg[movers // page], h, movers % page]
                else:
                    x[pg[holes // page], holes % page, h] = s[p][pg[movers // page], movers % page, h]
    return {"src": src, **got}
