"""kata_attn_prep_axes: rotary positions of three axes over the contiguous cache, against a plain evaluation in 64 bits, and with equal positions
against kata_attn_prep byte for byte.

The kernel forms an angle in fp32 from an fp32 frequency: two roundings, 2^-23 of its size in all, and sine and cosine to 2 ulp. The norm is a sum of 256 squares, a division, a root and
two products (2^-19 relative covers them). fp16 rows add half a step (2^-11), int8 rows half a code step of a scale that is itself rounded to fp16."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F8 = torch.float64


@pytest.fixture(scope="module")
def capi():
    from kata_b200 import capi as m
    assert torch.cuda.is_available()
    m.lib()
    return m


def _inputs(seed, n, T, act):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return r(n, T, 24 * 512).to(act), r(n, T, 1024).to(act), r(n, T, 1024).to(act), 1 + 0.1 * r(256), 1 + 0.1 * r(256), g


def _axis_of(sections, interleaved):
    out = []
    for i in range(32):
        out.append((i % 3 if i % 3 and i < 3 * sections[i % 3] else 0) if interleaved else 0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2)
    return torch.tensor(out, device="cuda")


def _rotated(x, w, pos, axis):
    """fp64 norm and rotation of x [..., heads, 256]; pos [..., 3]. Also the magnitude of each rotated pair, and the largest angle."""
    x = x.to(F8)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.to(F8)
    f = 1e7 ** (-torch.arange(32, device="cuda", dtype=F8) / 32)
    ang = (pos[..., axis].to(F8) * f)[..., None, :]
    a, b = x[..., :32].clone(), x[..., 32:64].clone()
    mag = x.abs()
    mag[..., :32] = mag[..., 32:64] = torch.sqrt(a * a + b * b)
    x[..., :32], x[..., 32:64] = a * torch.cos(ang) - b * torch.sin(ang), a * torch.sin(ang) + b * torch.cos(ang)
    err = torch.full_like(x, 2.0 ** -19) * mag
    e = ang.abs() * 2.0 ** -23 + 2.0 ** -22
    err[..., :64] += mag[..., :64] * torch.cat([e, e], -1)
    return x, err


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kv", ["fp16", "int8", "int8v", "int8g"])
def test_equal_positions_give_the_same_bytes_as_prep(capi, kv, act):
    n, T, at = 2, 5, [0, 7]
    qf, k, v, qn, kn, _ = _inputs(1, n, T, act)
    a, b = capi.AttnContext(2, [32, 32], kv_mode=kv), capi.AttnContext(2, [32, 32], kv_mode=kv)
    pos = torch.tensor([[[at[s] + t] * 3 for t in range(T)] for s in range(n)], dtype=torch.int32, device="cuda")
    for sections, inter in (([32, 0, 0], False), ([12, 10, 10], True), ([8, 12, 12], False)):
        a.reset(); b.reset()
        q1, f1, g1 = a.prep(1, [0, 1], at, T, qf, k, v, qn, kn, want_q32=True)
        q2, f2, g2 = b.prep_axes(1, [0, 1], at, T, pos, sections, qf, k, v, qn, kn, interleaved=inter, q32=torch.empty_like(f1))
        assert torch.equal(q1, q2) and torch.equal(f1, f2) and torch.equal(g1, g2)
        for s in range(n):
            for p in range(a.kv_planes()):
                assert (a.plane_read(1, s, p, 0, 32) == b.plane_read(1, s, p, 0, 32)).all()
    a.check(); b.check()
    a.close(); b.close()


@pytest.mark.parametrize("sections,inter", [([12, 10, 10], True), ([8, 12, 12], False), ([32, 0, 0], False), ([0, 0, 32], False), ([30, 1, 1], True)])
@pytest.mark.parametrize("n,T", [(1, 1), (3, 33)])
def test_against_64_bits(capi, sections, inter, n, T):
    qf, k, v, qn, kn, g = _inputs(2 + T, n, T, torch.float32)
    at = [s * 3 for s in range(n)]
    pos = torch.randint(-50, 5000, (n, T, 3), generator=g, device="cuda", dtype=torch.int32)
    ctx = capi.AttnContext(1, [64] * n)
    q16, q32, gate = ctx.prep_axes(0, list(range(n)), at, T, pos, sections, qf, k, v, qn, kn, interleaved=inter, q32=torch.empty(n, T, 6144, device="cuda"))
    ax = _axis_of(sections, inter)
    q = qf.view(n, T, 24, 2, 256)
    ref, err = _rotated(q[..., 0, :], qn, pos, ax)
    assert ((q32.view(n, T, 24, 256).to(F8) - ref).abs() <= err + 2.0 ** -23 * ref.abs()).all()
    assert ((q16.view(n, T, 24, 256).to(F8) * 16 - ref).abs() <= err + 2.0 ** -11 * ref.abs() * 1.01 + 2.0 ** -20).all()   # (16 times the smallest subnormal's half)
    assert torch.equal(gate.view(n, T, 24, 256), q[..., 1, :])
    kr, kerr = _rotated(k.view(n, T, 4, 256), kn, pos, ax)
    for s in range(n):
        kc = torch.as_tensor(ctx.plane_read(0, s, 0, at[s], T).view("float16").reshape(T, 4, 256).copy()).cuda().to(F8)
        vc = torch.as_tensor(ctx.plane_read(0, s, 1, at[s], T).view("float16").reshape(T, 4, 256).copy()).cuda()
        assert ((kc - kr[s]).abs() <= kerr[s] + 2.0 ** -11 * kr[s].abs() * 1.01 + 2.0 ** -24).all()
        assert torch.equal(vc, v[s].view(T, 4, 256).half())
    ctx.check(); ctx.close()


def test_partial_head_slots_captured_and_read_by_decode(capi):
    """K and V alone, then the queries alone, inside one captured graph; decode reads them as it reads kata_attn_prep's rows."""
    T, at = 2, [6]
    qf, k, v, qn, kn, g = _inputs(9, 1, 8, torch.float32)
    pos = torch.randint(0, 90, (1, 8, 3), generator=g, device="cuda", dtype=torch.int32)
    sec = [12, 10, 10]
    a, b = capi.AttnContext(1, [16]), capi.AttnContext(1, [16])
    for c in (a, b):
        c.prep_axes(0, [0], [0], 6, pos[:, :6].contiguous(), sec, None, k[:, :6].contiguous(), v[:, :6].contiguous(), None, kn, interleaved=True, h0=24, nh=8)
    two = [x[:, 6:].contiguous() for x in (qf, k, v)]
    p2 = pos[:, 6:].contiguous()
    q16, _, gate = a.prep_axes(0, [0], at, T, p2, sec, *two, qn, kn, interleaved=True)
    want = a.decode(0, [0], at, T, q16, gate)
    q, gt, out = torch.zeros_like(q16), torch.zeros_like(gate), torch.zeros_like(want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            b.prep_axes(0, [0], at, T, p2, sec, None, two[1], two[2], None, kn, interleaved=True, h0=24, nh=8)
            b.prep_axes(0, [0], at, T, p2, sec, two[0], None, None, qn, None, interleaved=True, h0=0, nh=24, q16=q, gate=gt)
            b.decode(0, [0], at, T, q, gt, out=out)
        graph.replay()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(q, q16)
    a.check(); b.check()
    a.close(); b.close()


def test_refusals(capi):
    qf, k, v, qn, kn, _ = _inputs(4, 1, 2, torch.float32)
    ctx = capi.AttnContext(1, [8])
    pos = torch.zeros(1, 2, 3, dtype=torch.int32, device="cuda")
    for sections, inter in (([31, 0, 0], False), ([33, 0, 0], False), ([-1, 16, 17], False), ([0, 16, 16], True), ([2 ** 31 - 1, 2 ** 31 - 1, 34], False)):
        with pytest.raises(capi.KataError):
            ctx.prep_axes(0, [0], [0], 2, pos, sections, qf, k, v, qn, kn, interleaved=inter)
    for bad in (pos.long(), pos[:, :1], pos.cpu(), pos.expand(2, 2, 3)):
        with pytest.raises(ValueError):
            ctx.prep_axes(0, [0], [0], 2, bad, [32, 0, 0], qf, k, v, qn, kn)
    with pytest.raises(ValueError):
        ctx.prep_axes(0, [0], [0], 2, pos, [16, 16], qf, k, v, qn, kn)
    with pytest.raises(capi.KataError):   # rows behind the sequence's end
        ctx.prep_axes(0, [0], [7], 2, pos, [32, 0, 0], qf, k, v, qn, kn)
    assert ctx.L.kata_attn_prep_axes(ctx.h, 0, 1, None, None, 2, None, None, 0, None, None, None, 0, None, None, None, None, None, 0, 32, None) == 1
    import ctypes
    sec, one = (ctypes.c_int32 * 3)(32, 0, 0), (ctypes.c_int32 * 1)(0)
    at = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    assert ctx.L.kata_attn_prep_axes(ctx.h, 0, 1, one, one, 2, ctypes.c_void_p(pos.data_ptr() + 2), sec, 0, at(qf), at(k), at(v), 0, at(qn), at(kn), at(qf), None, at(qf), 0, 32, None) == 1   # positions off their boundary: nothing is launched
    ctx.check(); ctx.close()
