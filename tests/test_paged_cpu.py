"""Host side of the paged cache without a GPU: the page table (reserve, trim, fork), the decode kernel's work split, and what the C entries refuse
before they touch a device."""
import ctypes as C
import os
import random
import re

import pytest

from kata_b200 import build, capi

OK, ARG, RANGE, MODE, NOMEM = 0, 1, 2, 3, 6
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    build.build()
    return capi.lib()


class Pages:
    def __init__(self, L, n_pages, page_size, n_seqs, max_slots):
        self.L, self.p = L, C.c_void_p()
        assert L.kata_pages_create(n_pages, page_size, n_seqs, max_slots, C.byref(self.p)) == OK

    def get(self, seq):
        buf = (C.c_int32 * 64)()
        n = self.L.kata_pages_get(self.p, seq, buf, 64)
        assert n == self.L.kata_pages_count(self.p, seq)
        return list(buf)[:n]

    def fork(self, src, dst, n):
        f, t, s = C.c_int32(7), C.c_int32(7), C.c_int32(7)
        return self.L.kata_pages_fork(self.p, src, dst, n, C.byref(f), C.byref(t), C.byref(s)), (f.value, t.value, s.value)

    def free(self):
        return self.L.kata_pages_free_count(self.p)

    def owners(self, page):
        return self.L.kata_pages_owners(self.p, page)


def test_binding_lists_the_headers_symbols():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "kata_paged.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(kata_page[sd]_[a-z0-9_]+)\s*\(", src))
    assert names == set(capi.PAGED_EXPORTS)


def test_pages_are_handed_out_lowest_first_and_come_back(L):
    p = Pages(L, 6, 16, 3, 96)
    r, t = L.kata_pages_reserve, L.kata_pages_trim
    assert r(p.p, 0, 1) == OK and r(p.p, 1, 17) == OK and r(p.p, 0, 33) == OK
    assert p.get(0) == [0, 3, 4] and p.get(1) == [1, 2] and p.free() == 1
    assert r(p.p, 0, 5) == OK and p.get(0) == [0, 3, 4]            # never fewer
    assert r(p.p, 2, 17) == NOMEM and p.get(2) == [] and p.free() == 1   # all or nothing
    assert t(p.p, 1, 16) == OK and p.get(1) == [1] and p.free() == 2
    assert r(p.p, 2, 32) == OK and p.get(2) == [2, 5]
    assert t(p.p, 0, 0) == OK and p.get(0) == [] and p.free() == 3
    assert r(p.p, 1, 64) == OK and p.get(1) == [1, 0, 3, 4]
    for bad in ((-1, 1), (3, 1), (0, -1), (0, 97)):
        assert r(p.p, *bad) == RANGE
    assert t(p.p, 0, -1) == RANGE and t(p.p, 3, 0) == RANGE
    assert L.kata_pages_destroy(p.p) == OK


def test_fork_shares_whole_pages_and_copies_the_partial_one(L):
    p = Pages(L, 8, 16, 4, 128)
    assert L.kata_pages_reserve(p.p, 0, 50) == OK and p.get(0) == [0, 1, 2, 3]
    rc, copy = p.fork(0, 1, 40)
    assert rc == OK and copy == (2, 4, 8) and p.get(1) == [0, 1, 4]
    assert [p.owners(x) for x in range(6)] == [2, 2, 1, 1, 1, 0]
    assert p.fork(0, 2, 32) == (OK, (-1, -1, 0)) and p.get(2) == [0, 1] and p.owners(0) == 3
    assert p.fork(0, 2, 16)[0] == MODE                              # it holds pages already
    assert p.fork(0, 0, 16)[0] == RANGE and p.fork(0, 3, 65)[0] == RANGE and p.fork(0, 4, 1)[0] == RANGE and p.fork(5, 3, 1)[0] == RANGE
    assert p.fork(0, 3, 0) == (OK, (-1, -1, 0)) and p.get(3) == []
    free = p.free()
    assert L.kata_pages_trim(p.p, 0, 0) == OK and p.free() == free + 2   # pages 2 and 3; 0 and 1 have owners left
    assert L.kata_pages_trim(p.p, 1, 0) == OK and L.kata_pages_trim(p.p, 2, 0) == OK and p.free() == 8
    assert L.kata_pages_reserve(p.p, 0, 128) == OK and p.get(0) == list(range(8))
    assert p.fork(0, 1, 120) == (NOMEM, (-1, -1, 0)) and p.get(1) == [] and p.owners(0) == 1
    L.kata_pages_destroy(p.p)


def test_random_calls_keep_the_tables_consistent(L):
    rng = random.Random(5)
    p, model = Pages(L, 40, 32, 6, 32 * 20), {s: [] for s in range(6)}
    for _ in range(3000):
        s, n = rng.randrange(6), rng.randrange(0, 641)
        what, want = rng.choice("rtf"), -(-n // 32)
        used = {x for t in model.values() for x in t}
        free = sorted(set(range(40)) - used)
        if what == "r":
            rc, more = L.kata_pages_reserve(p.p, s, n), want - len(model[s])
            if more > len(free):
                assert rc == NOMEM
            else:
                assert rc == OK
                model[s] += free[:max(0, more)]
        elif what == "t":
            assert L.kata_pages_trim(p.p, s, n) == OK
            del model[s][want:]
        else:
            d = rng.randrange(6)
            rc, copy = p.fork(s, d, n)
            if d == s or n > 32 * len(model[s]):
                assert rc == RANGE
            elif model[d]:
                assert rc == MODE
            elif n % 32 and not free:
                assert rc == NOMEM
            else:
                assert rc == OK
                model[d] = model[s][:n // 32] + (free[:1] if n % 32 else [])
                assert copy == ((model[s][n // 32], free[0], n % 32) if n % 32 else (-1, -1, 0))
        assert all(p.get(x) == model[x] for x in range(6))
        count = [sum(t.count(x) for t in model.values()) for x in range(40)]
        assert [p.owners(x) for x in range(40)] == count and p.free() == count.count(0)
    L.kata_pages_destroy(p.p)


def test_page_table_refuses_what_it_cannot_hold(L):
    q = C.c_void_p()
    for bad in ((0, 16, 1, 1), (1, 8, 1, 1), (1, 24, 1, 1), (1, 2048, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0), (1, 16, 1, 524289)):
        assert L.kata_pages_create(*bad, C.byref(q)) == ARG and not q
    assert L.kata_pages_create(1, 16, 1, 1, None) == ARG and L.kata_pages_destroy(None) == ARG and L.kata_pages_reserve(None, 0, 1) == ARG
    assert L.kata_pages_count(None, 0) == -1 and L.kata_pages_get(None, 0, None, 0) == -1 and L.kata_pages_free_count(None) == -1 and L.kata_pages_owners(None, 0) == -1


def _plan(L, keys, kvh, tile, sm=148):
    n = len(keys)
    first, most = (C.c_int32 * (sm + 1))(), C.c_int32()
    c = L.kata_paged_decode_plan(n, (C.c_int32 * n)(*keys), kvh, tile, sm, first, sm + 1, C.byref(most))
    return c, list(first)[:c + 1], most.value


def test_work_split_covers_every_tile_once(L):
    rng = random.Random(7)
    shapes = [([0], 1, 16), ([1], 4, 16), ([16], 4, 16), ([17], 4, 32), ([32768], 4, 16), ([524288] * 3, 16, 16), ([5] * 256, 16, 32), ([0] * 256, 8, 16), ([100] * 37, 4, 16)]
    for _ in range(300):
        n = rng.randint(1, 256)
        top = rng.choice([1, 40, 1000, 33000])
        shapes.append(([rng.randint(0, top) for _ in range(n)] if rng.random() < 0.7 else [rng.randint(0, top)] * n, rng.randint(1, 16), rng.choice([16, 32])))
    for keys, kvh, tile in shapes:
        c, first, most = _plan(L, keys, kvh, tile)
        nt = [max(1, -(-k // tile)) for k in keys]
        assert 1 <= c <= 148 and first[0] == 0 and first[-1] == kvh * sum(nt) and all(a < b for a, b in zip(first, first[1:])), (keys, kvh, tile)
        import bisect
        worst, start = 0, 0
        for t in nt:
            for _ in range(kvh):
                worst = max(worst, bisect.bisect_right(first, start + t - 1) - bisect.bisect_right(first, start) + 1)
                start += t
        assert worst == most


def test_work_split_refuses_bad_arguments(L):
    assert _plan(L, [5], 0, 16)[0] == -1 and _plan(L, [5], 17, 16)[0] == -1 and _plan(L, [5], 4, 24)[0] == -1 and _plan(L, [-1], 4, 16)[0] == -1 and _plan(L, [524289], 4, 16)[0] == -1
    assert _plan(L, [5] * 257, 4, 16)[0] == -1


GOOD = dict(device=0, n_layers=1, n_seqs=2, n_pages=4, page_size=16, max_slots=64, heads=24, kv_heads=4, head_dim=256, kv_mode=0, rot_dim=64, section=(32, 0, 0), interleaved=0, flags=1, rope_theta=1e7)


def _create(L, **kw):
    v = dict(GOOD, **kw)
    v["section"] = (C.c_int32 * 3)(*v["section"])
    cfg = capi.PagedConfig(**{k: x for k, x in v.items() if k != "planes"})
    for i, x in enumerate(v.get("planes", ())):
        cfg.planes[i] = x
    h = C.c_void_p()
    return L.kata_paged_create(C.byref(cfg), C.byref(h))


@pytest.mark.parametrize("bad", [
    dict(n_layers=0), dict(n_seqs=0), dict(n_pages=0), dict(page_size=24), dict(page_size=8), dict(page_size=2048), dict(max_slots=0), dict(max_slots=524289),
    dict(heads=0), dict(heads=23), dict(kv_heads=0), dict(kv_heads=17, heads=17), dict(heads=68), dict(head_dim=64), dict(head_dim=192),
    dict(rot_dim=-16), dict(rot_dim=72), dict(rot_dim=272), dict(section=(31, 0, 0)), dict(section=(33, -1, 0)), dict(section=(16, 16, 1)), dict(section=(10, 11, 11), interleaved=1),
    dict(rope_theta=0.0), dict(rope_theta=float("nan")), dict(flags=4), dict(planes=(64,)),
])
def test_create_refuses(L, bad):
    assert _create(L, **bad) == ARG


def test_create_refuses_modes_and_sizes(L):
    assert _create(L, kv_mode=2) == MODE and _create(L, kv_mode=3) == MODE and _create(L, kv_mode=9) == MODE
    assert _create(L, n_pages=2 ** 31 - 1, page_size=1024) == RANGE
    h = C.c_void_p()
    assert L.kata_paged_create(None, C.byref(h)) == ARG and L.kata_paged_create(None, None) == ARG and not h


def test_null_contexts_are_refused(L):
    L.kata_paged_last_error.restype = C.c_char_p
    assert L.kata_paged_destroy(None) == ARG and L.kata_paged_check(None, None) == ARG and L.kata_paged_reserve(None, 0, 1, None) == ARG and L.kata_paged_trim(None, 0, 0) == ARG
    assert L.kata_paged_fork(None, 0, 1, 1, None) == ARG and L.kata_paged_prep(None, 0, 1, None, None, 1, None, None, None, None, None, 0, None, None, None, None, None) == ARG
    assert L.kata_paged_decode(None, 0, 1, None, None, 1, None, None, None, 0, 0, None) == ARG and L.kata_paged_evict(None, 0, 1, 1, None, None, None, 1, 0, 0, None, None) == ARG
    assert L.kata_paged_import(None, 0, 0, 0, 1, 0, None, 0, 0, 0, None) == ARG and L.kata_paged_last_error(None) == b"null context" and not L.kata_paged_plane_ptr(None, 0, 0)


def test_prep_axes_refuses_a_null_context(L):
    assert L.kata_attn_prep_axes(None, 0, 1, None, None, 1, None, None, 0, None, None, None, 0, None, None, None, None, None, 0, 32, None) == ARG
