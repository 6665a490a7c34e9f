"""capi.PagedContext beside what surrounds it: contexts that rows are taken over from, tensors that alias its planes, ages after an eviction."""
import gc
import weakref

import pytest
import torch

from .test_gpu_paged import _context, _gen, _randn, capi  # noqa: F401

pytestmark = pytest.mark.gpu


def test_import_refuses_a_source_that_writes_some_of_the_kv_heads(capi):  # noqa: F811
    g = _gen(21)
    arena, ctx = capi.AttnContext(1, [64]), _context(capi, [40])
    kn, k = 1 + 0.05 * _randn(g, 256), _randn(g, 1, 20, 1024)
    ctx.plane(0, "k").fill_(3.0)
    arena.prep(0, [0], [0], 20, None, k, k, None, kn, h0=24, nh=8)
    for lo, n in ((0, 2), (3, 1)):
        arena.set_kv_heads(lo, n)
        with pytest.raises(capi.KataError) as e:
            ctx.import_rows(0, 0, 0, 20, arena, 0, 0, 0)
        assert e.value.code == 3
        torch.cuda.synchronize()
        assert (ctx.plane(0, "k") == 3).all()
    arena.set_kv_heads(0, 4)
    ctx.import_rows(0, 0, 0, 20, arena, 0, 0, 0)
    assert not (ctx.plane(0, "k") == 3).all()
    ctx.check()


@pytest.mark.parametrize("how", ["closed", "collected"])
def test_a_tensor_over_a_plane_keeps_its_memory(capi, how):  # noqa: F811
    ctx, arena = _context(capi, [40], weights=True), capi.AttnContext(1, [64])
    views = [ctx.plane(0, "k"), ctx.plane(0, "age")[1:, 2], arena.plane_tensor(0, 0, 0, 64)]   # (a view of an alias too)
    alive = [weakref.ref(ctx._native), weakref.ref(arena._native)]
    if how == "closed":
        ctx.close(), arena.close()
        with pytest.raises(capi.KataError):
            ctx.plane(0, "v")
    del ctx, arena
    gc.collect()
    assert all(r() is not None for r in alive)
    for i, v in enumerate(views):
        v.fill_(i + 1)
    other = torch.zeros(64 << 20, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert all(bool((v == i + 1).all()) for i, v in enumerate(views)) and not other.any()
    del views[2], v
    gc.collect()
    assert alive[0]() is not None and alive[1]() is None
    del views
    gc.collect()
    assert alive[0]() is None
