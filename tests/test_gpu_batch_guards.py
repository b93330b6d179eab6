"""That a served batch's entries write nothing but their outputs and their workspace, whatever the device arrays hold: outputs
and workspaces lie between guards, rows have columns behind them that are not theirs, and what is read is compared with what
was put there."""
import numpy as np
import pytest

import _batch as B
import _decoder as D
import p2gemm as P

pytestmark = pytest.mark.gpu
EVERY = P.EVERY_KEY
BIG = 2 ** 31 - 1
GUARD = 1 << 16   # bytes before and behind


def rng_of(*key):
    return np.random.default_rng(list(repr(key).encode()))


class Between:
    """`nbytes` of 0xFF between guards of 0x5A."""

    def __init__(self, nbytes):
        self.n, self.buf = nbytes, P.DeviceBuffer(nbytes + 2 * GUARD)
        fill = np.full(nbytes + 2 * GUARD, 0x5A, np.uint8)
        fill[GUARD:GUARD + nbytes] = 0xFF
        self.buf.upload(fill)
        self.ptr = self.buf.ptr + GUARD

    def check(self, what=""):
        P.sync()
        for off in (0, GUARD + self.n):
            assert (self.buf.download(GUARD, np.uint8, offset=off) == 0x5A).all(), what

    def rows(self, shape, t):
        return self.buf.download(shape, D.np_type(t), offset=GUARD)


class Out(Between):
    """Rows of `width` elements at pitch width + pad."""

    def __init__(self, t, rows, width, pad=16):
        super().__init__(rows * (width + pad) * D.size(t))
        self.t, self.shape, self.width, self.ld = t, (rows, width + pad), width, width + pad

    def check(self, what=""):
        super().check(what)
        pads = np.ascontiguousarray(self.rows(self.shape, self.t)[:, self.width:])
        assert (pads.view(np.uint8) == 0xFF).all(), what


class Reads:
    """Arrays on the device that a call must leave as they are."""

    def __init__(self, *arrays):
        self.host = [np.ascontiguousarray(a) for a in arrays]
        self.dev = [D.device(a) for a in self.host]

    def __getitem__(self, i):
        return self.dev[i].ptr

    def check(self, what=""):
        P.sync()
        for h, d in zip(self.host, self.dev):
            assert np.array_equal(d.download(h.nbytes, np.uint8), h.view(np.uint8).reshape(-1)), what


def cache_reads(kept):
    r = Reads.__new__(Reads)
    r.host, r.dev = [kept.kc, kept.vc, kept.ks, kept.vs], kept.dev
    return r


def words(*values):
    return np.array(values, np.int64).astype(np.int32)


def wild(rng, shape, *among):
    return rng.choice(np.array((-1, -BIG, BIG, 0, *among), np.int64), shape).astype(np.int32)


STARTS = ((-5, 90, 12, BIG), (39, 39, 40, 41), (BIG, -1, 5, 0), (0, 10, 20, BIG), (-BIG, -BIG, BIG, BIG), (10, 20, 30, 35))


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh,Hk", ((64, 1), (128, 5)))
def test_rows(t, Dh, Hk):
    page, rows = 16, 40
    rng = rng_of("rows", t, Dh)
    table, pages = B.tables(rng, [3, 3, 3])
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    seen = cache_reads(kept)
    for tab in (table, wild(rng, table.shape, pages, pages - 1)):
        for starts in STARTS:
            r, k, v = Reads(words(*starts), tab), Out(t, rows, Hk * Dh), Out(t, rows, Hk * Dh)
            P.kv_rows_q8_dev(t, kept.c, rows, 3, r[0], r[1], tab.shape[1], k.ptr, k.ld, v.ptr, v.ld)
            for x in (k, v, r, seen):
                x.check(f"{t} {Dh} {starts}")
    # rows of no sequence are left as they were
    assert (np.ascontiguousarray(k.rows(k.shape, t)[:10]).view(np.uint8) == 0xFF).all()
    assert (np.ascontiguousarray(v.rows(v.shape, t)[35:]).view(np.uint8) == 0xFF).all()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("T", (40, 300))
def test_rope(t, T):
    H, Hk, Dh, page, pages = 4, 2, 64, 16, 3
    rng = rng_of("rope", t, T)
    qkv = D.rows(rng, t, T, (H + 2 * Hk) * Dh)
    gamma, freq, pos = rng.uniform(-1, 1, Dh).astype(np.float32), np.ones(Dh // 2, np.float32), wild(rng, T, 77)
    slots = rng.choice(np.array([-1, -BIG, BIG, pages * page, pages * page + 1], np.int64), T).astype(np.int32)
    at = rng.permutation(T)[:20]
    slots[at] = rng.permutation(pages * page)[:20]
    r, q, k = Reads(qkv, gamma, freq, pos, slots), Out(t, T, H * Dh), Out(t, T, Hk * Dh)
    n = pages * Hk * page
    codes, scales = [Between(n * Dh) for _ in range(2)], [Between(n * 4) for _ in range(2)]
    cache = P.KvCacheQ8(Hk, Dh, page, pages, codes[0].ptr, codes[1].ptr, scales[0].ptr, scales[1].ptr)
    P.qk_norm_rope_q8_dev(t, T, H, Hk, Dh, r[0], qkv.shape[1], r[1], r[1], 1e-6, Dh, False, r[2], r[3], q.ptr, q.ld, k.ptr, k.ld,
                          cache, r[4])
    for x in (r, q, k, *codes, *scales):
        x.check(f"{t} {T}")
    used = np.zeros((pages, page), bool)
    used[slots[at] // page, slots[at] % page] = True
    for c in codes:   # the other slots' codes
        got = c.buf.download((pages, Hk, page, Dh), np.uint8, offset=GUARD).transpose(0, 2, 1, 3)
        assert (got[~used] == 0xFF).all() and (got[used] != 0xFF).any()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("H,Hk", ((4, 2), (33, 1)))
def test_paged(t, H, Hk):
    page, Dh, n = 16, 64, 4
    rng = rng_of("paged", t, H)
    table, pages = B.tables(rng, [60] * n)
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    seen, q = cache_reads(kept), D.rows(rng, t, n, H * Dh)
    for tab in (table, wild(rng, table.shape, pages, pages - 1)):
        for lens in ((BIG, -BIG, 0, 961), (960, 1, 959, -1), (BIG, BIG, BIG, BIG)):
            for window, sinks in ((EVERY, 0), (1, EVERY), (100, 3)):
                for most in (960, EVERY):
                    need = P.attention_paged_q8_workspace_bytes(kept.c, n, H, most, window, sinks)
                    r, o, ws = Reads(q, tab, words(*lens)), Out(t, n, H * Dh), Between(need)
                    P.attention_paged_q8_dev(t, kept.c, n, H, r[0], H * Dh, r[1], tab.shape[1], r[2], most, 0.1, window, sinks,
                                             o.ptr, o.ld, ws.ptr if need else None, need)
                    for x in (r, o, ws, seen):
                        x.check(f"{t} {H} {lens} {window} {most}")


GROUPS = ((0, 5), (-BIG, BIG), (5, 0), (1, 2), (5, 0, 5), (0, 5, 0, 5), (5, 5, 0, 1, 0, 5), (4, 0, 3, 1, 2), (0, 2, 2, 5), None)


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("t,H,Hk", (("f32", 4, 2), ("f16", 4, 2), ("bf16", 64, 2), ("f16", 33, 1)))
def test_shared(kind, t, H, Hk):
    page, Dh, n = 16, 64, 5
    rng = rng_of("shared", kind, t, H)
    table, pages = B.tables(rng, [6] * n)
    if kind == "q8":
        kept = B.Kept.random(rng, pages, Hk, page, Dh)
        cache, seen, size = kept.c, cache_reads(kept), P.attention_shared_q8_workspace_bytes
    else:
        seen, size = Reads(*(D.rows(rng, t, pages, Hk, page, Dh) for _ in range(2))), P.attention_shared_workspace_bytes
        cache = P.KvCache(t, Hk, Dh, page, pages, seen[0], seen[1])
    q = D.rows(rng, t, n, H * Dh)
    for turn, starts in enumerate(GROUPS):
        st = rng.integers(0, n + 1, 200) if starts is None else np.array(starts)
        g = len(st) - 1
        for tab in (table, wild(rng, table.shape, pages, pages - 1)):
            for ms, mo in ((40, 60), (EVERY, EVERY), (0, 0)):
                shared = wild(rng, g, 40, 96, 97) if turn % 2 else np.full(g, 40, np.int32)
                lens = wild(rng, n, 50, 97) if ms else words(41, 50, 77, 96, 43)
                window, sinks = ((EVERY, 0), (30, 5))[turn % 2]
                need = size(cache, n, g, H, ms, mo, window, sinks)
                r, o, ws = Reads(q, st.astype(np.int64).astype(np.int32), shared, tab, lens), Out(t, n, H * Dh), Between(need)
                args = (cache, n, g, H, r[0], H * Dh, r[1], r[2], r[3], tab.shape[1], r[4], ms, mo, 0.1, window, sinks, o.ptr, o.ld,
                        ws.ptr, need)
                if kind == "q8":
                    P.attention_shared_q8_dev(t, *args)
                else:
                    P.attention_shared_dev(*args)
                for x in (r, o, ws, seen):
                    x.check(f"{kind} {t} {H} {st[:8]} {ms}")


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M,K,N,rank", ((1, 64, 70, 8), (5, 130, 64, 16), (33, 64, 131, 128), (300, 72, 200, 32), (600, 136, 133, 16),
                                       (577, 67, 64, 64)))
def test_adapters(t, M, K, N, rank):
    count = 3
    rng = rng_of("adapters", t, M, K)
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    for pad in (0, 8, 5):
        r = Reads(D.rows(rng, t, M, K), wild(rng, M, 1, 2, count), a, b, scale, D.rows(rng, t, M, N))
        ad = P.Adapters(t, count, rank, K, N, r[2], r[3], r[4])
        need = P.adapters_workspace_bytes(ad, M)
        y, ws = Out(t, M, N, pad), Between(need)
        P.adapters_add_dev(ad, M, r[0], K, r[1], r[5], N, y.ptr, y.ld, ws.ptr, need)
        for x in (r, y, ws):
            x.check(f"{t} {M} {K} {N} {rank} pad {pad}")
        none = (r.host[1] < 0) | (r.host[1] >= count)
        got = np.ascontiguousarray(y.rows(y.shape, t)[:, :N])
        assert np.array_equal(got[none].view(np.uint8), np.ascontiguousarray(r.host[5][none]).view(np.uint8))
