"""A served batch's step on the device against plain 64-bit forms (tests/_batch.py)."""
import numpy as np
import pytest

import _batch as B
import _decoder as D
import p2gemm as P

pytestmark = pytest.mark.gpu
EVERY = P.EVERY_KEY


def rng_of(*key):
    return np.random.default_rng(list(repr(key).encode()))


# ── the 8-bit cache: written ────────────────────────────────────────────────────────────────────────────────────

def rope_inputs(t, T, H, Hk, Dh, rot, key, far=100000):
    rng = rng_of(t, T, H, Dh, rot, key)
    qkv = D.rows(rng, t, T, (H + 2 * Hk) * Dh, scale=3.0)
    gq, gk = (rng.uniform(-1.5, 1.5, Dh).astype(np.float32) for _ in range(2))
    freq = (10000.0 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 1))).astype(np.float32)
    return rng, qkv, gq, gk, freq, rng.integers(0, far, T).astype(np.int32)


def run_rope(t, qkv, H, kept, gq, gk, eps, rot, inter, freq, pos, slots, keys=True, stream=None):
    """→ q, k (or None), and the cache's four arrays; the call without codes too, whose rows have to be the same bits."""
    T, W = qkv.shape
    Hk, Dh = kept.kc.shape[1], kept.kc.shape[3]
    dx, dgq, dgk, df, dp, ds = (D.device(a) for a in (qkv, gq, gk, freq, pos, np.asarray(slots, np.int32)))
    dq, dk = D.preset(t, (max(T, 1), H * Dh)), D.preset(t, (max(T, 1), Hk * Dh))
    P.qk_norm_rope_q8_dev(t, T, H, Hk, Dh, dx.ptr, W, dgq.ptr, dgk.ptr, eps, rot, inter, df.ptr, dp.ptr, dq.ptr, H * Dh,
                          dk.ptr if keys else None, Hk * Dh, kept.c, ds.ptr, stream)
    q, k = dq.download((T, H * Dh), D.np_type(t), stream), dk.download((T, Hk * Dh), D.np_type(t), stream) if keys else None
    eq, ek = D.preset(t, (max(T, 1), H * Dh)), D.preset(t, (max(T, 1), Hk * Dh))
    P.qk_norm_rope_dev(t, T, H, Hk, Dh, dx.ptr, W, dgq.ptr, dgk.ptr, eps, rot, inter, df.ptr, dp.ptr, eq.ptr, H * Dh,
                       ek.ptr, Hk * Dh, None, None, stream)
    assert np.array_equal(q.view(np.uint16), eq.download((T, H * Dh), D.np_type(t), stream).view(np.uint16))
    if keys:
        assert np.array_equal(k.view(np.uint16), ek.download((T, Hk * Dh), D.np_type(t), stream).view(np.uint16))
    return q, k, *kept.download(stream)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("T,H,Hk,Dh,rot,inter,page", ((1, 1, 1, 64, 64, False, 16), (21, 6, 3, 128, 128, True, 16),
                                                      (5, 8, 8, 128, 64, False, 64), (300, 4, 2, 64, 16, True, 32),
                                                      (7, 32, 8, 128, 0, False, 1024), (260, 5, 1, 128, 48, False, 256)))
def test_rope_q8(t, T, H, Hk, Dh, rot, inter, page):
    pages = -(-T // page) + 2
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "q8")
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    if T > 20:
        slots[4], slots[9], slots[13] = -1, pages * page, 2 ** 31 - 1   # rows that stay out of it
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    _, _, kc, vc, ks, vs = run_rope(t, qkv, H, kept, gq, gk, 1e-6, rot, inter, freq, pos, slots, keys=T % 2 == 1)
    x = D.to_f64(t, qkv).reshape(T, H + 2 * Hk, Dh)
    want, size_of = D.norm_rope(x[:, H:H + Hk], gk, 1e-6, rot, inter, freq, pos)
    off = D.rope_bound("f32", want, size_of, Dh)   # of the keys in 32 bits
    vcode, vscale = B.codes_of(x[:, H + Hk:].astype(np.float32))
    same = [a.copy() for a in (kept.kc, kept.vc, kept.ks, kept.vs)]
    for i, s in enumerate(slots):
        if not 0 <= s < pages * page:
            continue
        p, o = s // page, s % page
        # half a step, and what the key itself and its head's largest value may be off by
        top = np.abs(want[i]).max(1)
        assert (np.abs(ks[p, :, o] - top / 127) <= (off[i].max(1) + 2 * D.FP32 * top) / 127).all()
        value = kc[p, :, o].astype(np.float64) * ks[p, :, o].astype(np.float64)[:, None]
        most = 0.5 * ks[p, :, o].astype(np.float64)[:, None] * (1 + 512 * D.FP32) + off[i]
        assert (np.abs(value - want[i]) <= most).all(), (i, float((np.abs(value - want[i]) / most).max()))
        assert np.array_equal(vc[p, :, o], vcode[i]) and np.array_equal(vs[p, :, o], vscale[i])
        for a, b in zip(same, (kc, vc, ks, vs)):
            a[p, :, o] = b[p, :, o]
    for a, b in zip(same, (kc, vc, ks, vs)):
        assert np.array_equal(a, b)   # nothing else was written


@pytest.mark.parametrize("t", D.TYPES)
def test_rope_q8_zero_tiny_and_non_finite_heads(t):
    T, H, Hk, Dh, page = 6, 2, 2, 64, 16
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, 0, "odd")
    x = D.to_f64(t, qkv).reshape(T, H + 2 * Hk, Dh)
    x[0, H:] = 0.0
    x[1, H + Hk:] *= 2.0 ** -130                                  # below 2^-100 in every type
    x[2, H + Hk, 5], x[3, H + Hk + 1, 0], x[4, H, 63], x[5, H + 1, 7] = np.inf, np.nan, np.inf, -np.nan
    qkv = D.to_type(t, x.reshape(T, -1))
    kept = B.Kept.random(rng, 1, Hk, page, Dh)
    _, _, kc, vc, ks, vs = run_rope(t, qkv, H, kept, gq, gk, 1e-6, 0, False, freq, pos, np.arange(T))
    assert not kc[0, :, 0].any() and not vc[0, :, 0].any() and not ks[0, :, 0].any() and not vs[0, :, 0].any()
    assert not vc[0, :, 1].any() and not vs[0, :, 1].any() and (ks[0, :, 1] > 0).all()
    for sc, at in ((vs, (0, 2)), (vs, (1, 3)), (ks, (0, 4)), (ks, (1, 5))):
        assert np.isnan(sc[0, at[0], at[1]]) and np.isfinite(sc[0, 1 - at[0], at[1]])
    assert np.isfinite(vs[0, 1, 2]) and np.isfinite(ks[0, :, :4]).all()


@pytest.mark.parametrize("t", D.TYPES)
def test_rope_q8_many_rows_as_few(t):
    T, H, Hk, Dh, rot, page = 300, 6, 2, 64, 32, 32
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "many")
    slots = rng.permutation(10 * page)[:T].astype(np.int32)
    kept = B.Kept.random(rng, 10, Hk, page, Dh)
    whole = run_rope(t, qkv, H, kept, gq, gk, 1e-5, rot, True, freq, pos, slots)[2:]
    again = B.Kept(kept.kc, kept.vc, kept.ks, kept.vs)
    for a in range(0, T, 100):
        few = run_rope(t, qkv[a:a + 100], H, again, gq, gk, 1e-5, rot, True, freq, pos[a:a + 100], slots[a:a + 100])[2:]
    for a, b in zip(whole, few):
        assert np.array_equal(a, b)


# ── read back ───────────────────────────────────────────────────────────────────────────────────────────────────

def rows_want(t, kept, starts, table, rows):
    pages, Hk, page, Dh = kept.kc.shape
    out = []
    for c, sc in ((kept.kc, kept.ks), (kept.vc, kept.vs)):
        v = c.astype(np.float32) * sc[..., None]
        want = np.full((rows, Hk * Dh), 0xFFFF if t == "bf16" else np.nan, D.np_type(t))
        for s in range(len(starts) - 1):
            a, b = min(max(starts[s], 0), rows), min(max(starts[s + 1], 0), rows)
            for r in range(a, max(a, b)):
                n = r - a
                p = table[s, n // page] if n // page < table.shape[1] else -1
                x = v[p, :, n % page].reshape(-1) if 0 <= p < pages else np.zeros(Hk * Dh)
                want[r] = D.to_type(t, x)
        out.append(want)
    return out


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("lens,Hk,Dh,page,first,behind", (
    ((1,), 1, 64, 16, 0, 0), ((0, 5, 0, 0, 33, 16), 2, 128, 16, 3, 2), ((700, 0, 650), 3, 64, 32, 0, 0),
    ((2500, 1, 4000), 8, 128, 64, 0, 1), ((3,) * 70 + (0,) * 100 + (40, 7), 1, 128, 16, 1, 5)))
def test_rows_q8(t, lens, Hk, Dh, page, first, behind):
    rng = rng_of(t, lens, Hk, Dh)
    table, pages = B.tables(rng, [-(-n // page) for n in lens])
    starts = first + np.concatenate(([0], np.cumsum(lens)))
    rows = int(starts[-1]) + behind
    kept = B.fill_unwritten(B.Kept.random(rng, pages, Hk, page, Dh), table, lens)
    want = rows_want(t, kept, starts, table, rows)
    got = B.run_rows(t, kept, starts, table, rows, pad=16)
    for g, w in zip(got, want):
        g = np.ascontiguousarray(g[:, :Hk * Dh])
        inside = np.isfinite(D.to_f64(t, w))   # rows of no sequence stay what they were: bytes of 0xFF
        assert np.array_equal(g[inside], w[inside])
        assert (g.view(np.uint16).reshape(rows, -1)[~inside.any(1)] == 0xFFFF).all()
    assert (np.ascontiguousarray(got[0][:, Hk * Dh:]).view(np.uint16) == 0xFFFF).all()


def test_rows_q8_pages_that_are_not_there():
    t, Hk, Dh, page = "f32", 2, 64, 16
    rng = rng_of("holes")
    table, pages = B.tables(rng, [5, 2])
    table[0, 1], table[0, 4], table[1, 0] = -1, pages, 2 ** 31 - 1
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    table = np.ascontiguousarray(table[:, :5])
    starts = np.array([0, 100, 130])   # 100 tokens of 5 pages: the last 20 have none
    for g, w in zip(B.run_rows(t, kept, starts, table, 130), rows_want(t, kept, starts, table, 130)):
        assert np.array_equal(g, w) and not g[16:32].any() and not g[80:116].any() and g[0].any()


def test_rows_q8_starts_outside_the_rows():
    """Starts that lie outside [0, rows] or descend reach nothing outside the rows (what they mean is not defined)."""
    t, Hk, Dh, page, rows = "bf16", 1, 64, 16, 40
    rng = rng_of("starts")
    table, pages = B.tables(rng, [3, 3, 3])
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    for starts in ([-5, 90, 12, 2 ** 31 - 1], [39, 39, 40, 41], [2 ** 31 - 1, -1, 5, 0]):
        B.run_rows(t, kept, np.array(starts), table, rows)


@pytest.mark.parametrize("t", D.TYPES)
def test_rows_q8_most_rows_a_workgroup(t):
    """Sizes about where a workgroup takes one row, two, …, the most."""
    Hk, Dh, page = 1, 64, 64
    rng = rng_of("per", t)
    for rows in (2047, 2048, 4096 + 7, 70000):
        lens = (rows // 3, 1, rows - rows // 3 - 1)
        table, pages = B.tables(rng, [-(-n // page) for n in lens])
        kept = B.Kept.random(rng, pages, Hk, page, Dh)
        starts = np.concatenate(([0], np.cumsum(lens)))
        seq = np.searchsorted(starts, np.arange(rows), side="right") - 1
        at = np.arange(rows) - starts[seq]
        p = table[seq, at // page]
        for got, c, sc in zip(B.run_rows(t, kept, starts, table, rows), (kept.kc, kept.vc), (kept.ks, kept.vs)):
            want = c[p, :, at % page].astype(np.float32) * sc[p, :, at % page][..., None]
            assert np.array_equal(got, D.to_type(t, want.reshape(rows, -1)))


# ── attention over it ───────────────────────────────────────────────────────────────────────────────────────────

PAGED = [  # lengths, heads, key heads, page, window, sinks
    ((1,), 1, 1, 16, EVERY, 0), ((0, 5, 16, 17), 4, 2, 16, EVERY, 0), ((33, 100), 8, 8, 64, 20, 3),
    ((1000, 3, 257), 6, 1, 32, 64, 40), ((2500,), 8, 2, 256, EVERY, 0), ((700, 650), 40, 2, 16, 500, 16),
    ((3000, 1, 0, 1024), 2, 1, 1024, 1, 1), ((90,), 3, 3, 16, 32, 200), ((150, 31, 32, 33), 34, 1, 32, EVERY, 0)]


def paged_case(t, lens, H, Hk, page, Dh, key="p"):
    rng = rng_of(t, lens, H, page, Dh, key)
    table, pages = B.tables(rng, [-(-n // page) for n in lens])
    kept = B.fill_unwritten(B.Kept.random(rng, pages, Hk, page, Dh), table, lens)
    return D.rows(rng, t, len(lens), H * Dh), kept, table


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,H,Hk,page,window,sinks", PAGED)
def test_paged_q8(t, Dh, lens, H, Hk, page, window, sinks):
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh)
    want, bound = B.paged_want(t, q, *kept.values(), table, lens, H, 0.1, window, sinks, True)
    for split in (False, True):
        got = B.run_paged(t, q, kept, table, lens, H, 0.1, window, sinks, split)
        D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens} split {split}")
    for most in (1, 40000):   # planned for other lengths than those that come
        got = B.run_paged(t, q, kept, table, lens, H, 0.1, window, sinks, True, most)
        D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens} planned for {most}")


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_q8_pages_that_are_not_there(t):
    lens, H, Hk, page, Dh = (200, 64, 130), 4, 1, 16, 64
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "holes")
    table[0, 2], table[0, 11], table[1, :] = -1, kept.kc.shape[0], 2 ** 31 - 1
    want, bound = B.paged_want(t, q, *kept.values(), table, lens, H, 0.1, EVERY, 0, True)
    got = D.to_f64(t, B.run_paged(t, q, kept, table, lens, H, 0.1, EVERY, 0))
    D.check(got, want, bound, t)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_q8_lengths_outside_the_table(t):
    lens, H, Hk, page, Dh = (48, 20), 2, 1, 16, 64
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "long")
    table = np.ascontiguousarray(table[:, :3])
    table[1] = table[0]
    got = B.run_paged(t, q, kept, table, (1 << 30, -4), H, 0.1, EVERY, 0, True, 100)
    want = B.run_paged(t, q, kept, table, (48, 0), H, 0.1, EVERY, 0, True, 100)
    assert np.array_equal(got, want) and not want[1].any()


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_q8_scales_that_are_not_finite(t):
    """A NaN scale reaches the heads and sequences that see its token, and nothing else."""
    lens, H, Hk, page, Dh = (100, 90, 80), 4, 2, 16, 64
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "nan")
    clean = B.run_paged(t, q, kept, table, lens, H, 0.1, 50, 4)
    kept.ks[table[0, 90 // page], 0, 90 % page] = np.nan     # seen
    kept.vs[table[1, 3 // page], 1, 3 % page] = np.inf       # seen as one of the first
    kept.ks[table[2, 20 // page], :, 20 % page] = np.nan     # before the window
    kept.vs[table[2, 20 // page], :, 20 % page] = np.inf
    got = D.to_f64(t, B.run_paged(t, q, B.Kept(kept.kc, kept.vc, kept.ks, kept.vs), table, lens, H, 0.1, 50, 4))
    odd = ~np.isfinite(got.reshape(3, H, Dh))
    assert odd[0, :2].all() and not odd[0, 2:].any() and not odd[1, :2].any() and odd[1, 2:].any() and not odd[2].any()
    keep = ~odd.reshape(3, -1)
    assert np.array_equal(got[keep], D.to_f64(t, clean)[keep])


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_q8_large_scores_and_small_weights(t):
    """Scores up to 700 either way, and values of very different size beside them."""
    lens, H, Hk, page, Dh = (500, 77), 4, 2, 16, 128
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "large")
    kept.ks *= 10.0
    kept.vs *= (10.0 ** rng_of("decades").integers(-3, 4, kept.vs.shape)).astype(np.float32)
    kept = B.Kept(kept.kc, kept.vc, kept.ks, kept.vs)
    want, bound = B.paged_want(t, q, *kept.values(), table, lens, H, 1.0, EVERY, 0, True)
    D.check(D.to_f64(t, B.run_paged(t, q, kept, table, lens, H, 1.0, EVERY, 0)), want, bound, t)


@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,H,Hk", (((1100, 640), 4, 2), ((300, 17, 900), 8, 8)))
def test_paged_q8_fp32_on_the_whole(Dh, lens, H, Hk):
    """Relative 2-norm. As _decoder.ATTENTION_NORM counts, with three times as many products a score (8.7 in place of 5):
    sqrt(8.7² + 3² + 9.6² + 1) = 13.4, against 16 allowed."""
    q, kept, table = paged_case("f32", lens, H, Hk, 16, Dh, "whole")
    want, _ = B.paged_want("f32", q, *kept.values(), table, lens, H, 0.1, EVERY, 0, True)
    for split in (False, True):
        off = D.norm_off(B.run_paged("f32", q, kept, table, lens, H, 0.1, EVERY, 0, split).astype(np.float64), want)
        assert off <= D.ATTENTION_NORM, off


# ── shared prefixes ─────────────────────────────────────────────────────────────────────────────────────────────

SHARED = [  # groups of (shared, lengths); heads, key heads, page, window, sinks
    ([(40, (41, 50, 77))], 4, 2, 16, EVERY, 0),
    ([(375, (376,))], 1, 1, 16, EVERY, 0),
    ([(100, (101, 0, 30, 100, 400)), (0, (5, 60)), (33, (34,) * 9)], 6, 2, 32, EVERY, 0),
    ([(1000, tuple(range(1001, 1031)))], 8, 1, 64, EVERY, 0),
    ([(700, (701, 900, 1500)), (650, (2000,))], 8, 8, 16, 300, 0),
    ([(700, (701, 900, 1500, 640)), (10, (20, 300))], 4, 1, 16, 90, 25),
    ([(50, (300, 500)), (90, (95, 200))], 20, 1, 256, 64, 130),
    ([(2100, (2101, 2200, 3000) * 12)], 4, 4, 1024, EVERY, 7),
    ([(700, (701, 900, 640, 0, 1100, 33) * 7)], 8, 2, 16, 250, 70),      # many rows: tiles
    ([(333, (334,) * 33), (90, (95, 40) * 20), (1, (2,) * 50)], 16, 4, 32, EVERY, 0),
    ([(1500, (1501, 1600) * 40)], 4, 1, 64, 1300, 0)]


def shared_case(t, groups, H, Hk, page, Dh, key="s", before=0, behind=0):
    """Tables as a program has them: pages that a prefix fills are in every table of its group, the page that it ends in is
    each sequence's own from there on. before, behind: sequences of no group."""
    rng = rng_of(t, groups, H, page, Dh, key)
    lens = [9] * before + [n for _, g in groups for n in g] + [21] * behind
    starts, at = [before], before
    for _, g in groups:
        at += len(g)
        starts.append(at)
    needs = []
    for s in range(len(lens)):
        needs.append(-(-lens[s] // page))
    for g, (m, _) in enumerate(groups):   # the first one's row holds the whole prefix, whatever its own length
        if starts[g] < starts[g + 1]:
            needs[starts[g]] = max(needs[starts[g]], -(-m // page))
    table, pages = B.tables(rng, needs)
    for g, (m, _) in enumerate(groups):
        for s in range(starts[g] + 1, starts[g + 1]):
            n = min(m // page, needs[s])
            table[s, :n] = table[starts[g], :n]
    reach = list(lens)
    for g, (m, _) in enumerate(groups):
        if starts[g] < starts[g + 1]:
            reach[starts[g]] = max(reach[starts[g]], m)
    return rng, lens, starts, [m for m, _ in groups], table, pages, reach


def shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach):
    """(cache for the call, keys and values in 64 bits), anything in what no token was written to."""
    if kind == "q8":
        kept = B.fill_unwritten(B.Kept.random(rng, pages, Hk, page, Dh), table, reach)
        kept.c.keep = kept
        return (kept.c, *kept.values())
    kc, vc = (D.rows(rng, t, pages, Hk, page, Dh) for _ in range(2))
    used = np.zeros((pages, page), bool)
    for s, n in enumerate(reach):
        for j in range(n):
            used[table[s, j // page], j % page] = True
    nan = np.uint16(0x7FC0) if t == "bf16" else np.nan
    for a in (kc, vc):
        a[np.nonzero(~used)[0], :, np.nonzero(~used)[1]] = nan
    return B.row_cache(t, kc, vc), D.to_f64(t, kc), D.to_f64(t, vc)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("groups,H,Hk,page,window,sinks", SHARED)
def test_shared(t, kind, Dh, groups, H, Hk, page, window, sinks):
    rng, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh)
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, len(lens), H * Dh)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, window, sinks, kind == "q8", starts, shared)
    for plan in ((max(shared), max(lens)), (1, 1), (100000, 20000)):
        got = B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, window, sinks, *plan, pad=16)
        D.check(D.to_f64(t, got[:, :H * Dh]), want, bound, f"{t} {kind} {Dh} {groups} planned for {plan}")
        assert (np.ascontiguousarray(got[:, H * Dh:]).view(np.uint16) == 0xFFFF).all()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("kind", ("rows", "q8"))
def test_shared_sequences_of_no_group_and_empty_groups(t, kind):
    H, Hk, page, Dh = 4, 2, 16, 64
    groups = [(30, ()), (40, (41, 60)), (9, ()), (20, ()), (50, (51,)), (5, ())]
    rng, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh, before=2, behind=3)
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, len(lens), H * Dh)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    got = B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 50, 60)
    inside = np.isfinite(want).all(1)
    assert inside.tolist() == [False] * 2 + [True] * 3 + [False] * 3
    D.check(D.to_f64(t, got[inside]), want[inside], bound[inside], t)
    assert (np.ascontiguousarray(got[~inside]).view(np.uint16) == 0xFFFF).all()


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("n", (70, 200))
def test_shared_many_groups(kind, n):
    """More groups than lanes look for at once."""
    t, H, Hk, page, Dh = "f16", 2, 1, 16, 64
    groups = [(3 + g % 40, (4 + g % 40 + g % 7,) * (1 + g % 3)) for g in range(n)]
    rng, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh)
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, len(lens), H * Dh)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    D.check(D.to_f64(t, B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 43, 8)), want, bound, kind)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("H,Dh", ((2, 64), (20, 64), (40, 128)))
def test_shared_values_that_are_not_finite(t, H, Dh):
    """Infinities and NaN among the kept values reach the sequences that see them, and no others, in a prefix of which a
    window leaves each sequence another part, and in what is each one's own; few rows and many."""
    Hk, page, window = 1, 16, 60
    groups = [(100, (101, 120, 150, 190))]
    rng, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh, "odd")
    kc, vc = (D.rows(rng, t, pages, Hk, page, Dh) for _ in range(2))
    clean = B.run_shared(t, q := D.rows(rng, t, 4, H * Dh), B.row_cache(t, kc, vc), starts, shared, table, lens, H, 0.1,
                         window, 0, 100, 90)
    vc[table[0, 50 // page], 0, 50 % page, 3] = D.to_type(t, np.array([np.inf]))[0]     # seen by the first alone
    vc[table[0, 95 // page], 0, 95 % page, 7] = D.to_type(t, np.array([-np.inf]))[0]    # by three of them
    vc[table[2, 140 // page], 0, 140 % page, 9] = D.to_type(t, np.array([np.nan]))[0]   # of the third alone
    got = D.to_f64(t, B.run_shared(t, q, B.row_cache(t, kc, vc), starts, shared, table, lens, H, 0.1, window, 0, 100, 90))
    odd = np.zeros((4, H, Dh), bool)
    odd[0, :, 3] = odd[0, :, 7] = odd[1, :, 7] = odd[2, :, 7] = odd[2, :, 9] = True
    got = got.reshape(4, H, Dh)
    assert np.array_equal(~np.isfinite(got), odd)
    assert np.array_equal(got[~odd], D.to_f64(t, clean).reshape(4, H, Dh)[~odd])


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("H", (4, 64))
def test_shared_device_arrays_outside_their_ranges(kind, H):
    """Lengths, prefixes, pages and groups that no program means reach nothing outside the buffers."""
    t, Hk, page, Dh = "bf16", 2, 16, 64
    rng, lens, starts, shared, table, pages, reach = shared_case(t, [(40, (41, 50, 77))], H, Hk, page, Dh)
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, 3, H * Dh)
    big = 2 ** 31 - 1
    for st, sh, ln in (([0, 3], [big], [big, -big, 50]), ([0, 3], [-big], lens), ([-big, big], [40], lens),
                       ([3, 0], [40], lens), ([1, 2], [39], lens)):
        B.run_shared(t, q, cache, st, sh, table, ln, H, 0.1, EVERY, 0, 40, 60)
    wild = table.copy()
    wild[:] = rng.choice([-1, -big, big, pages, 0], wild.shape)
    B.run_shared(t, q, cache, starts, shared, wild, lens, H, 0.1, EVERY, 0, 40, 60)
    # a length beyond the table is the table's, a prefix beyond the lengths all of them
    full = np.ascontiguousarray(table[:, :2])
    a = B.run_shared(t, q, cache, starts, [10 ** 6], full, [10 ** 6, 20, 0], H, 0.1, EVERY, 0, 40, 60)
    b = B.run_shared(t, q, cache, starts, [32], full, [32, 20, 0], H, 0.1, EVERY, 0, 40, 60)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("H", (4, 64))
def test_shared_starts_that_descend(kind, H):
    """Groups whose starts go up and down, several of them and more than a wave looks at at once, reach nothing outside the
    buffers (what they mean is not defined), and a call behind one is right."""
    t, Hk, page, Dh = "bf16", 2, 16, 64
    rng, lens, starts, shared, table, pages, reach = shared_case(t, [(40, (41, 50, 77, 60, 43))], H, Hk, page, Dh, "down")
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, 5, H * Dh)
    for st in ([5, 0, 5], [0, 5, 0, 5], [5, 5, 0, 1, 0, 5], [4, 0, 3, 1, 2], list(rng.integers(0, 6, 200))):
        B.run_shared(t, q, cache, st, [40] * (len(st) - 1), table, lens, H, 0.1, EVERY, 0, 40, 60)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    D.check(D.to_f64(t, B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 40, 60)), want, bound, kind)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("H", (4, 48))
def test_shared_pages_that_are_not_there(t, kind, H):
    """Tokens of a page number outside the cache are not seen, in the prefix by nobody, behind it by their own sequence."""
    Hk, page, Dh = 2, 16, 64
    rng, lens, starts, shared, table, pages, reach = shared_case(t, [(200, (201, 230, 260, 150))], H, Hk, page, Dh, "holes")
    table[0, 3], table[0, 9], table[1, 13], table[2, 14] = -1, pages, 2 ** 31 - 1, -9
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, np.where((table < 0) | (table >= pages), 0, table), reach)
    q = D.rows(rng, t, 4, H * Dh)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    D.check(D.to_f64(t, B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 200, 60)), want, bound, t)


@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("kind", ("rows", "q8"))
def test_shared_fp32_on_the_whole(Dh, kind):
    """As test_paged_q8_fp32_on_the_whole."""
    H, Hk, page, t = 4, 2, 32, "f32"
    rng, lens, starts, shared, table, pages, reach = shared_case(t, [(700, (701, 800, 1000, 1090))], H, Hk, page, Dh, "whole")
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, len(lens), H * Dh)
    want, _ = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    off = D.norm_off(B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 700, 400).astype(np.float64),
                     want)
    assert off <= D.ATTENTION_NORM, off


# ── adapters ────────────────────────────────────────────────────────────────────────────────────────────────────

ADAPTERS = [  # M, K, N, rank, adapters
    (1, 64, 16, 8, 1), (1, 1024, 1024, 8, 4), (5, 77, 143, 16, 3), (16, 129, 65, 32, 2), (17, 256, 300, 64, 20),
    (33, 1000, 515, 128, 5), (100, 136, 7, 16, 4), (13, 4096, 257, 16, 13), (70, 1, 1, 8, 2), (3, 8192, 40, 32, 2),
    (600, 72, 200, 8, 3), (515, 520, 136, 16, 5), (700, 264, 72, 32, 40), (530, 1160, 64, 64, 2), (577, 128, 328, 128, 3),
    (513, 100, 131, 64, 4), (520, 136, 133, 32, 2), (514, 67, 64, 16, 2), (300, 264, 515, 16, 3), (257, 1024, 3, 8, 2),
    (290, 72, 200, 128, 5), (400, 130, 257, 64, 40), (256, 96, 64, 32, 3),
    (4, 64, 130, 128, 1), (2, 100, 70, 64, 2), (1, 32, 9, 32, 1), (16, 40, 100, 16, 16)]


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M,K,N,rank,count", ADAPTERS)
def test_adapters(t, M, K, N, rank, count):
    rng = rng_of(t, M, K, N, rank)
    x, z = D.rows(rng, t, M, K), D.rows(rng, t, M, N)
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    runs = np.sort(rng.integers(0, count, M))
    runs[M // 3:M // 2] = -1
    for index in (rng.integers(-1, count + 1, M), runs, np.full(M, count - 1)):
        want, bound = B.adapters_want(t, x, index, a, b, scale, z)
        got = B.run_adapters(t, x, index, a, b, scale, z)
        D.check(D.to_f64(t, got), want, bound, f"{t} {M} {K} {N} {rank}")
        none = (index < 0) | (index >= count)
        assert np.array_equal(got[none].view(np.uint16), z[none].view(np.uint16))
        same = B.run_adapters(t, x, index, a, b, scale, z, in_place=True)
        assert np.array_equal(same.view(np.uint16), got.view(np.uint16))


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M", (7, 37, 600))
def test_adapters_pitches_and_no_rows_before(t, M):
    K, N, rank, count = 200, 133, 16, 6
    rng = rng_of(t, "pitch")
    x, z = D.rows(rng, t, M, K), D.rows(rng, t, M, N)
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    index = rng.integers(-1, count, M)
    want = B.run_adapters(t, x, index, a, b, scale, z)
    for pads in ((8, 3, 5), (1, 0, 16), (3, 7, 0), (8, 11, 27)):   # of the last, rows are 16 bytes apart
        got = B.run_adapters(t, x, index, a, b, scale, z, pads=pads)
        exp, bound = B.adapters_want(t, x, index, a, b, scale, z)
        D.check(D.to_f64(t, got[:, :N]), exp, bound, str(pads))
        assert (np.ascontiguousarray(got[:, N:]).view(np.uint16) == 0xFFFF).all()
        in_place = B.run_adapters(t, x, index, a, b, scale, z, in_place=True, pads=pads)
        assert np.array_equal(in_place[:, :N].view(np.uint16), np.ascontiguousarray(got[:, :N]).view(np.uint16))
    assert want.shape == (M, N)
    alone, bound = B.adapters_want(t, x, index, a, b, scale, None)
    got = B.run_adapters(t, x, index, a, b, scale, None)
    D.check(D.to_f64(t, got), alone, bound, "no Z")
    assert not D.to_f64(t, got[index < 0]).any()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M", (7, 20, 300, 600))
def test_adapters_do_not_reach_other_rows(t, M):
    """Adapters and rows that are not finite change no row of another adapter; zeros of both signs and NaN of rows without
    an adapter stay as they are."""
    K, N, rank, count = 136, 70, 16, 5
    rng = rng_of(t, "others")
    x, z = D.rows(rng, t, M, K), D.rows(rng, t, M, N)
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    index = rng.integers(-1, count, M)
    index[:4] = (0, 2, 1, -1)
    z[3, :3] = D.to_type(t, np.array([-0.0, np.nan, np.inf]))
    clean = B.run_adapters(t, x, index, a, b, scale, z)
    a[2], b[3], scale[4] = D.to_type(t, np.full(a[2].shape, np.inf)), D.to_type(t, np.full(b[3].shape, np.nan)), np.inf
    x[0] = D.to_type(t, np.full(K, np.nan))
    got = B.run_adapters(t, x, index, a, b, scale, z)
    keep = (index < 2)
    keep[0] = False
    assert np.array_equal(got[keep].view(np.uint16), clean[keep].view(np.uint16))
    assert not np.isfinite(D.to_f64(t, got[~keep])).any()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M", (0, 9, 50, 600))
def test_no_adapters_at_all(t, M):
    """A set of none, and one that no row has: Z as it is."""
    rng = rng_of(t, "none")
    N = 128
    x, z = D.rows(rng, t, M, 64), D.rows(rng, t, M, N)
    a, b, scale = B.adapter_set(rng, t, 2, 16, 64, N)
    assert np.array_equal(B.run_adapters(t, x, np.full(M, 2), a, b, scale, z).view(np.uint16), z.view(np.uint16))
    dx, dz, di, dy = D.device(x), D.device(z), D.device(np.zeros(M, np.int32)), D.preset(t, (max(M, 1), N))
    ad = P.Adapters(t, 0, 16, 64, N, None, None, None)
    ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
    P.adapters_add_dev(ad, M, dx.ptr, 64, di.ptr, dz.ptr, N, dy.ptr, N, ws.ptr, ws.nbytes)
    assert np.array_equal(dy.download((M, N), D.np_type(t)).view(np.uint16), z.view(np.uint16))


@pytest.mark.parametrize("M,K,N,rank", ((40, 1024, 300, 64), (300, 1000, 64, 16), (5, 512, 700, 128), (600, 1024, 64, 64)))
def test_adapters_fp32_on_the_whole(M, K, N, rank):
    """Relative 2-norm of what the adapter adds: each product of the fp32 matrix unit may drop up to a step, rms 0.58 · 2 ·
    2^-24 of a sum that grows as a random walk: n products 1.15 · sqrt(n / 2) · 2^-24. A wave's quarter of K 256, 13; the
    rank 128, 9.2; waves, parts, the scale and the output 2: sqrt(13² + 9.2² + 2²) = 16.1, against 24 allowed."""
    rng = rng_of("whole", M, K)
    x = D.rows(rng, "f32", M, K)
    a, b, scale = B.adapter_set(rng, "f32", 3, rank, K, N)
    index = rng.integers(0, 3, M)
    want, _ = B.adapters_want("f32", x, index, a, b, scale, None)
    off = D.norm_off(B.run_adapters("f32", x, index, a, b, scale, None).astype(np.float64), want)
    assert off <= 24 * D.FP32, off


# ── offsets beyond 32 bits ──────────────────────────────────────────────────────────────────────────────────────

def test_cache_q8_beyond_32_bits():
    """A cache of more than 2^32 codes whose last pages are used, by every entry: the results of a small one."""
    t, H, Hk, Dh, page, pages, n = "bf16", 8, 8, 128, 1024, 4110, 1500
    assert pages * Hk * page * Dh > 1 << 32
    _, qkv, gq, gk, freq, pos = rope_inputs(t, n, H, Hk, Dh, Dh, "far pages")
    dx, dgq, dgk, df, dp = (D.device(a) for a in (qkv, gq, gk, freq, pos))
    outs = []
    for count, order in ((pages, (pages - 1, pages - 3)), (2, (1, 0))):
        dk, dv = (P.DeviceBuffer(count * Hk * page * Dh) for _ in range(2))
        ks, vs = (P.DeviceBuffer(count * Hk * page * 4) for _ in range(2))
        cache = P.KvCacheQ8(Hk, Dh, page, count, dk.ptr, dv.ptr, ks.ptr, vs.ptr)
        at = np.arange(n)
        ds = D.device((np.array(order)[at // page] * page + at % page).astype(np.int32))
        dt, dl = D.device(np.array([order], np.int32)), D.device(np.array([n], np.int32))
        dst, dg, dsh = (D.device(np.array(v, np.int32)) for v in ((0, n), (0, 1), (1100,)))
        dq = D.preset(t, (n, H * Dh))
        P.qk_norm_rope_q8_dev(t, n, H, Hk, Dh, dx.ptr, 3 * H * Dh, dgq.ptr, dgk.ptr, 1e-6, Dh, False, df.ptr, dp.ptr, dq.ptr,
                              H * Dh, None, 0, cache, ds.ptr)
        rk, rv, o1, o2 = (D.preset(t, (m, H * Dh)) for m in (n, n, 1, 1))
        P.kv_rows_q8_dev(t, cache, n, 1, dst.ptr, dt.ptr, 2, rk.ptr, H * Dh, rv.ptr, H * Dh)
        P.attention_paged_q8_dev(t, cache, 1, H, dq.ptr, H * Dh, dt.ptr, 2, dl.ptr, n, 0.1, EVERY, 0, o1.ptr, H * Dh)
        ws = P.Workspace(P.attention_shared_q8_workspace_bytes(cache, 1, 1, H, 1100, 400))
        P.attention_shared_q8_dev(t, cache, 1, 1, H, dq.ptr, H * Dh, dg.ptr, dsh.ptr, dt.ptr, 2, dl.ptr, 1100, 400, 0.1, EVERY,
                                  0, o2.ptr, H * Dh, ws.ptr, ws.nbytes)
        outs.append([b.download((m, H * Dh), np.uint16) for b, m in ((rk, n), (rv, n), (o1, 1), (o2, 1))])
    for far, near in zip(*outs):
        assert np.isfinite(D.to_f64(t, near)).all() and np.array_equal(far, near)


def test_adapters_beyond_32_bits():
    """The last of adapters whose values pass 2^32."""
    t, M, K, N, rank, count = "bf16", 3, 1 << 13, 1 << 13, 64, 8300
    assert count * rank * K > 1 << 32
    rng = rng_of("many adapters")
    a, b, scale = B.adapter_set(rng, t, 1, rank, K, N)
    x, z = D.rows(rng, t, M, K), D.rows(rng, t, M, N)
    want, bound = B.adapters_want(t, x, [0, -1, 0], a, b, scale, z)
    da, db = P.DeviceBuffer(count * rank * K * 2), P.DeviceBuffer(count * rank * N * 2)
    da.upload(a, offset=(count - 1) * rank * K * 2)
    db.upload(b, offset=(count - 1) * rank * N * 2)
    ds = D.device(np.full(count, scale[0], np.float32))
    dx, dz, di, dy = D.device(x), D.device(z), D.device(np.array([count - 1, count, count - 1], np.int32)), D.preset(t, (M, N))
    ad = P.Adapters(t, count, rank, K, N, da.ptr, db.ptr, ds.ptr)
    ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
    P.adapters_add_dev(ad, M, dx.ptr, K, di.ptr, dz.ptr, N, dy.ptr, N, ws.ptr, ws.nbytes)
    D.check(D.to_f64(t, dy.download((M, N), np.uint16)), want, bound)


def test_adapters_rows_far_apart():
    """Sixteen rows of Y that reach over 2^32 bytes, in place and from another Z."""
    t, M, K, N, rank, ldy = "f32", 257, 64, 64, 8, 72_000_000
    assert 15 * ldy * 4 > 1 << 32
    rng = rng_of("far rows")
    a, b, scale = B.adapter_set(rng, t, 3, rank, K, N)
    x, z, index = D.rows(rng, t, M, K), D.rows(rng, t, M, N), rng.integers(-1, 3, M)
    want, bound = B.adapters_want(t, x, index, a, b, scale, z)
    dx, dz, da, db, ds = (D.device(v) for v in (x, z, a, b, scale))
    di, dy = D.device(index.astype(np.int32)), P.DeviceBuffer(((M - 1) * ldy + N) * 4)
    ad = P.Adapters(t, 3, rank, K, N, da.ptr, db.ptr, ds.ptr)
    ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
    for in_place in (False, True):
        for m in range(M):
            dy.upload(z[m] if in_place else np.zeros(N, np.float32), offset=m * ldy * 4)
        P.adapters_add_dev(ad, M, dx.ptr, K, di.ptr, dy.ptr if in_place else dz.ptr, ldy if in_place else N, dy.ptr, ldy, ws.ptr,
                           ws.nbytes)
        got = np.stack([dy.download(N, np.float32, offset=m * ldy * 4) for m in range(M)])
        D.check(D.to_f64(t, got), want, bound, str(in_place))


# ── together, streams and graphs ────────────────────────────────────────────────────────────────────────────────

class Layer:
    """A decoder layer's attention step for a served batch: qkv by a 4-bit weight that all share and each request's adapter,
    norm and rotation into an 8-bit cache, attention behind the prefixes that groups share, the output projection."""
    H, Hk, DH, C, PAGE, WINDOW, SINKS, RANK, COUNT = 4, 2, 64, 256, 16, 200, 3, 16, 3

    def __init__(self, t, groups, shared, per, seed):
        """groups: starts; shared: tokens of each group's prefix, put into the cache here."""
        rng = rng_of(t, groups, shared, seed)
        W, n = (self.H + 2 * self.Hk) * self.DH, groups[-1]
        self.t, self.n, self.W, self.groups, self.shared = t, n, W, groups, shared
        self.wq, self.wo = D.q4_weight(rng, self.C, W, 64, True), D.q4_weight(rng, self.H * self.DH, self.C, 32, False)
        self.q4q, self.q4o = P.Q4Weight(*self.wq, self.C, W, 64), P.Q4Weight(*self.wo, self.H * self.DH, self.C, 32)
        self.ad = B.adapter_set(rng, t, self.COUNT, self.RANK, self.C, W)
        self.index = rng.integers(-1, self.COUNT, n).astype(np.int32)
        self.gq, self.gk = (rng.uniform(0.5, 1.5, self.DH).astype(np.float32) for _ in range(2))
        self.freq = (100.0 ** (-np.arange(0, self.DH, 2) / self.DH)).astype(np.float32)
        self.table, self.pages = B.tables(rng, [per] * n)
        for g, m in enumerate(shared):
            self.table[groups[g]:groups[g + 1], :m // self.PAGE] = self.table[groups[g], :m // self.PAGE]
        self.kept = B.fill_unwritten(B.Kept.random(rng, self.pages, self.Hk, self.PAGE, self.DH), self.table[groups[:-1]], shared)
        self.values0 = self.kept.values()
        self.most = per * self.PAGE
        dev = lambda a: D.device(np.ascontiguousarray(a))   # noqa: E731
        self.da, self.db, self.ds = (dev(a) for a in self.ad)
        self.set = P.Adapters(t, self.COUNT, self.RANK, self.C, W, self.da.ptr, self.db.ptr, self.ds.ptr)
        self.di, self.dg, self.dsh = dev(self.index), dev(np.array(groups, np.int32)), dev(np.array(shared, np.int32))
        self.dgq, self.dgk, self.df, self.dt = dev(self.gq), dev(self.gk), dev(self.freq), dev(self.table)
        self.dx, self.dqkv = D.preset(t, (n, self.C)), D.preset(t, (n, W))
        self.dq, self.do = D.preset(t, (n, self.H * self.DH)), D.preset(t, (n, self.H * self.DH))
        self.dpos, self.dslot, self.dlen = (dev(np.zeros(n, np.int32)) for _ in range(3))
        self.ws1 = P.Workspace(P.adapters_workspace_bytes(self.set, n))
        self.ws2 = P.Workspace(P.attention_shared_q8_workspace_bytes(self.kept.c, n, len(shared), self.H, max(shared),
                                                                     self.most, self.WINDOW, self.SINKS))

    def place(self, x, step):
        """The step's rows; every sequence's new token stands `step` places behind its prefix."""
        at = (np.repeat(self.shared, np.diff(self.groups)) + step).astype(np.int32)
        self.dx.upload(x)
        self.dpos.upload(at)
        self.dslot.upload((self.table[np.arange(self.n), at // self.PAGE] * self.PAGE + at % self.PAGE).astype(np.int32))
        self.dlen.upload(at + 1)

    def step(self, stream=None):
        t, n, H, Hk, DH = self.t, self.n, self.H, self.Hk, self.DH
        P.q4_gemv_dev(t, n, self.W, self.C, 0.05, self.dx.ptr, self.C, self.q4q, 0.0, self.dqkv.ptr, self.W, stream)
        P.adapters_add_dev(self.set, n, self.dx.ptr, self.C, self.di.ptr, self.dqkv.ptr, self.W, self.dqkv.ptr, self.W,
                           self.ws1.ptr, self.ws1.nbytes, stream)
        P.qk_norm_rope_q8_dev(t, n, H, Hk, DH, self.dqkv.ptr, self.W, self.dgq.ptr, self.dgk.ptr, 1e-6, DH, False,
                              self.df.ptr, self.dpos.ptr, self.dq.ptr, H * DH, None, 0, self.kept.c, self.dslot.ptr, stream)
        P.attention_shared_q8_dev(t, self.kept.c, n, len(self.shared), H, self.dq.ptr, H * DH, self.dg.ptr, self.dsh.ptr,
                                  self.dt.ptr, self.table.shape[1], self.dlen.ptr, max(self.shared), self.most, DH ** -0.5,
                                  self.WINDOW, self.SINKS, self.do.ptr, H * DH, self.ws2.ptr, self.ws2.nbytes, stream)
        P.q4_gemv_dev(t, n, self.C, H * DH, 0.05, self.do.ptr, H * DH, self.q4o, 1.0, self.dx.ptr, self.C, stream)

    def out(self, stream=None):
        return self.dx.download((self.n, self.C), D.np_type(self.t), stream)

    def plain(self, xs):
        """xs [steps][n][C] in 64 bits: the layer's outputs, nothing rounded in between."""
        wq = D.q4_values(*self.wq, self.C, self.W, 64) * 0.05
        wo = D.q4_values(*self.wo, self.H * self.DH, self.C, 32) * 0.05
        a, b = (D.to_f64(self.t, m) for m in self.ad[:2])
        S, H, Hk, DH = xs.shape[0], self.H, self.Hk, self.DH
        out = np.zeros(xs.shape)
        for s in range(self.n):
            g = np.searchsorted(self.groups, s, side="right") - 1
            m = self.shared[g]
            qkv, i = xs[:, s] @ wq, self.index[s]
            if i >= 0:
                qkv = qkv + float(self.ad[2][i]) * (xs[:, s] @ a[i].T @ b[i].T)
            qkv, pos = qkv.reshape(S, H + 2 * Hk, DH), m + np.arange(S)
            q, _ = D.norm_rope(qkv[:, :H], self.gq, 1e-6, DH, False, self.freq, pos)
            k, _ = D.norm_rope(qkv[:, H:H + Hk], self.gk, 1e-6, DH, False, self.freq, pos)
            pk, pv = (B.tokens(v, self.table[self.groups[g]], m)[0] for v in self.values0)
            k, v = np.concatenate((pk, k)), np.concatenate((pv, qkv[:, H + Hk:]))
            o, _ = D.attention("f32", q, k, v, D.visible(S, m + S, self.WINDOW, 0, self.SINKS), DH ** -0.5)
            out[:, s] = xs[:, s] + o.reshape(S, -1) @ wo
        return out


GROUPS, SHARES = [0, 3, 4, 9], [37, 0, 160]


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_token_by_token(t):
    """Forty tokens of nine sequences in three groups. Besides the roundings that a layer over rows has (8 half steps of the
    root mean square and 2^-16, as the layer of the decoder's tests), keys and values are off by half a step of 1 / 127 of
    their head's largest, which is up to 4 times its root mean square here: an rms of 4 / 127 / sqrt(12) = 0.9 % of theirs. A
    score's error from that is 0.9 % of |q| |k| / 8 (64 dimensions add up as a random walk): of q and k of norm 8 each
    (times their gains, up to 1.5 each) 0.16, a weight's relative error, of which the mean leaves at most its own size; with
    the values' 0.9 % and against a layer that changes its rows by its own size, 6 times 0.05 covers the largest entry."""
    L = Layer(t, GROUPS, SHARES, 16, "tokens")
    S = 40
    xs = D.rows(rng_of(t, "xs"), t, S, L.n, L.C)
    want = L.plain(D.to_f64(t, xs))
    for n in range(S):
        L.place(xs[n], n)
        L.step()
        got = D.to_f64(t, L.out())
        rms = np.sqrt((want[n] ** 2).mean())
        assert np.abs(got - want[n]).max() <= 6 * (8 * D.HALF[t] + 2.0 ** -16 + 0.05) * rms, \
            (n, np.abs(got - want[n]).max() / rms)


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_in_a_graph(t):
    """A captured step replayed for token after token, with eager work between: the bits of the eager step."""
    L, E = Layer(t, GROUPS, SHARES, 16, "graph"), Layer(t, GROUPS, SHARES, 16, "graph")
    S, s = 12, P.Stream()
    xs = D.rows(rng_of(t, "graph"), t, S, L.n, L.C)
    with P.Graph(s) as g:
        L.step(s.ptr)
    for n in range(S):
        L.place(xs[n], n)
        E.place(xs[n], n)
        P.sync()
        g.launch()
        s.sync()
        E.step()
        P.sync()
        assert np.array_equal(L.out(s.ptr).view(np.uint16), E.out().view(np.uint16)), n


def test_two_streams_at_once():
    t, S = "f16", 8
    both = [Layer(t, GROUPS, SHARES, 16, k) for k in ("one", "two")]
    alone = [Layer(t, GROUPS, SHARES, 16, k) for k in ("one", "two")]
    streams = [P.Stream(), P.Stream()]
    xs = D.rows(rng_of("two"), t, S, both[0].n, Layer.C)
    for n in range(S):
        for L in (*both, *alone):
            L.place(xs[n], n)
        P.sync()
        for L, s in zip(both, streams):
            L.step(s.ptr)
        for s in streams:
            s.sync()
        for L, A, s in zip(both, alone, streams):
            A.step()
            P.sync()
            assert np.array_equal(L.out(s.ptr), A.out())


@pytest.mark.parametrize("t", D.TYPES)
def test_prompt_chunk_over_kept_rows(t):
    """A prompt's second chunk: its keys and values go into the cache, everything kept comes back as rows, and windowed
    attention over these is what attention of the last token over the pages gives."""
    H, Hk, Dh, page, rot = 4, 2, 64, 16, 64
    past, chunk = (50, 0, 131), (20, 33, 7)
    lens = [p + c for p, c in zip(past, chunk)]
    T = sum(chunk)
    rng, qkv, gq, gk, freq, _ = rope_inputs(t, T, H, Hk, Dh, rot, "chunk")
    table, pages = B.tables(rng, [-(-n // page) for n in lens])
    kept = B.fill_unwritten(B.Kept.random(rng, pages, Hk, page, Dh), table, past)
    pos = np.concatenate([p + np.arange(c) for p, c in zip(past, chunk)]).astype(np.int32)
    seq = np.repeat(np.arange(3), chunk)
    slots = table[seq, pos // page] * page + pos % page
    q = run_rope(t, qkv, H, kept, gq, gk, 1e-6, rot, False, freq, pos, slots)[0]
    ks = np.concatenate(([0], np.cumsum(lens)))
    k, v = B.run_rows(t, kept, ks, table, int(ks[-1]))
    qs = np.concatenate(([0], np.cumsum(chunk)))
    o = D.run_window(t, q, k, v, H, Hk, Dh, 0.125, 60, 0, 2, qs, ks)
    last = np.ascontiguousarray(q[qs[1:] - 1])
    kept.kc, kept.vc, kept.ks, kept.vs = kept.download()
    got = B.run_paged(t, last, kept, table, lens, H, 0.125, 60, 2)
    want, bound = B.paged_want(t, last, *kept.values(), table, lens, H, 0.125, 60, 2, True)
    D.check(D.to_f64(t, got), want, bound, t)
    # rows are rounded to the type once more: a key's half step moves a score by at most half a step of sum |q k|
    mag = np.abs(D.to_f64(t, last)).max() * max(np.abs(x[np.isfinite(x)]).max() for x in kept.values()) * Dh * 0.125
    more = 2 * D.HALF[t] * (mag + 1) * np.abs(kept.values()[1][np.isfinite(kept.values()[1])]).max()
    assert (np.abs(D.to_f64(t, o[qs[1:] - 1]) - want) <= 2 * bound + more).all()


@pytest.mark.parametrize("t", D.TYPES)
def test_two_graphs_share_a_workspace(t):
    """Two captured calls with one workspace, replayed in turn on one stream, lengths changing between: each as it is alone."""
    rng = rng_of(t, "workspace")
    H, Hk, page, Dh, s, made = 4, 1, 16, 64, P.Stream(), []
    ws = P.Workspace(1 << 22)
    for groups in ([(900, (901, 1000, 1200))], [(30, (31, 40)), (500, (700,))]):
        _, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh, "ws")
        cache, K, V = shared_cache(rng, t, "q8", pages, Hk, page, Dh, table, reach)
        q = D.rows(rng, t, len(lens), H * Dh)
        bufs = [D.device(np.asarray(a, np.int32)) for a in (starts, shared, table, lens)]
        dq, do = D.device(q), D.preset(t, (len(lens), H * Dh))
        assert P.attention_shared_q8_workspace_bytes(cache, len(lens), len(shared), H, 900, 300) <= ws.nbytes
        with P.Graph(s) as g:
            P.attention_shared_q8_dev(t, cache, len(lens), len(shared), H, dq.ptr, H * Dh, bufs[0].ptr, bufs[1].ptr,
                                      bufs[2].ptr, table.shape[1], bufs[3].ptr, 900, 300, 0.1, EVERY, 0, do.ptr, H * Dh,
                                      ws.ptr, ws.nbytes, s.ptr)
        made.append((g, lens, bufs, do, lambda ln, a=(t, q, cache, starts, shared, table): B.run_shared(
            *a[:6], ln, H, 0.1, EVERY, 0, 900, 300), (cache, dq)))
    for turn in range(4):
        for g, lens, bufs, do, alone, _ in made:
            ln = [n - turn for n in lens]
            bufs[3].upload(np.asarray(ln, np.int32))
            P.sync()
            g.launch()
            s.sync()
            assert np.array_equal(do.download((len(lens), H * Dh), D.np_type(t)).view(np.uint16),
                                  alone(ln).view(np.uint16)), turn


def test_adapters_rows_very_far_apart():
    """Rows of Y so far apart that the size of sixteen, taken in 32 bits, is 0."""
    t, M, K, N, rank, ldy = "bf16", 257, 64, 64, 8, 1 << 28
    assert (16 * ldy) % (1 << 32) == 0
    rng = rng_of("very far rows")
    a, b, scale = B.adapter_set(rng, t, 3, rank, K, N)
    x, z, index = D.rows(rng, t, M, K), D.rows(rng, t, M, N), rng.integers(-1, 3, M)
    want, bound = B.adapters_want(t, x, index, a, b, scale, z)
    dx, dz, da, db, ds = (D.device(v) for v in (x, z, a, b, scale))
    di, dy = D.device(index.astype(np.int32)), P.DeviceBuffer(((M - 1) * ldy + N) * 2)
    ad = P.Adapters(t, 3, rank, K, N, da.ptr, db.ptr, ds.ptr)
    ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
    for m in range(M):
        dy.upload(np.full(N, 0xFFFF, np.uint16), offset=m * ldy * 2)
    P.adapters_add_dev(ad, M, dx.ptr, K, di.ptr, dz.ptr, N, dy.ptr, ldy, ws.ptr, ws.nbytes)
    got = np.stack([dy.download(N, np.uint16, offset=m * ldy * 2) for m in range(M)])
    D.check(D.to_f64(t, got), want, bound)


def test_rows_q8_more_workgroups_than_a_grid_is_wide():
    """2^29 rows and some, 137 GB of keys and values: tokens of three pages, again and again."""
    t, Hk, Dh, page, rows = "bf16", 1, 64, 1024, (1 << 29) + 5000
    rng = rng_of("many rows")
    kept = B.Kept.random(rng, 3, Hk, page, Dh)
    starts = np.array([0, 5, rows - 2000, rows - 7], np.int32)
    table = rng.integers(0, 3, (3, (1 << 19) + 8)).astype(np.int32)
    table[1, 700] = -1
    dk, dv = (P.DeviceBuffer(rows * Dh * 2) for _ in range(2))
    ds, dt = D.device(starts), D.device(table)
    some = np.unique(np.concatenate((np.arange(5, 3000), 700 * page + 5 + np.arange(-3, page + 3), rng.integers(5, rows, 300),
                                     (1 << 28) + np.arange(-40, 40), (1 << 29) + np.arange(-40, 40), rows - np.arange(2100, 1, -1))))
    behind = np.full((7, Dh), 0xFFFF, np.uint16)
    for d in (dk, dv):
        d.upload(behind, offset=(rows - 7) * Dh * 2)
    P.kv_rows_q8_dev(t, kept.c, rows, 3, ds.ptr, dt.ptr, table.shape[1], dk.ptr, Dh, dv.ptr, Dh)
    runs = np.split(some, np.nonzero(np.diff(some) > 1)[0] + 1)
    for d, c, sc in ((dk, kept.kc, kept.ks), (dv, kept.vc, kept.vs)):
        values = D.to_type(t, c[:, 0].astype(np.float32) * sc[:, 0, :, None])   # [page][place][Dh]
        assert np.array_equal(d.download((7, Dh), np.uint16, offset=(rows - 7) * Dh * 2), behind)
        for run in runs:
            run = run[run < rows - 7]
            if run.size == 0:
                continue
            s = np.searchsorted(starts, run, side="right") - 1
            at = run - starts[s]
            p = table[s, at // page]
            want = np.where((p >= 0)[:, None], values[np.maximum(p, 0), at % page], 0)
            assert np.array_equal(d.download((run.size, Dh), np.uint16, offset=int(run[0]) * Dh * 2), want), run[0]


@pytest.mark.parametrize("t", ("f16", "bf16"))
@pytest.mark.parametrize("Dh", (64, 128))
def test_q8_loses_no_more_than_the_outputs_rounding(t, Dh):
    """Relative 2-norm over many outputs. Rounding a value of mantissa m in [1, 2) to the type is off by an rms of eps / 2 / sqrt(3)
    of its power of two, that over m of the value: over all at most as if every m were 1. What comes before it is 2^-16 a weight
    and 32 bits. (Weights rounded to 8 bits would be as much again: over the limit, as m is spread.)"""
    H, Hk, page = 32, 8, 16
    lens = tuple(range(100, 900, 50))
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "rounding")
    want, _ = B.paged_want(t, q, *kept.values(), table, lens, H, 0.05, EVERY, 0, True)
    most = D.HALF[t] / 3 ** 0.5
    for split in (False, True):
        assert D.norm_off(D.to_f64(t, B.run_paged(t, q, kept, table, lens, H, 0.05, EVERY, 0, split)), want) <= most
    for per in (1, 16):   # 16 rows at a time, and 32
        groups = [(60, (61, 90, 300, 777) * per)]
        rng, lens, starts, shared, table, pages, reach = shared_case(t, groups, H, Hk, page, Dh, "rounding")
        cache, K, V = shared_cache(rng, t, "q8", pages, Hk, page, Dh, table, reach)
        q = D.rows(rng, t, len(lens), H * Dh)
        want, _ = B.paged_want(t, q, K, V, table, lens, H, 0.05, EVERY, 0, True, starts, shared)
        off = D.norm_off(D.to_f64(t, B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.05, EVERY, 0, 60, 717)), want)
        assert off <= most, (per, off)


# ── together, each stage from what the one before it left ───────────────────────────────────────────────────────

def codes_within(c, s, want, off):
    """Codes [.., Dh] and scales of heads that are `want` in 64 bits, of which what was put in may be off by `off`."""
    top = np.abs(want).max(-1)
    assert (np.abs(s - top / 127) <= (off.max(-1) + 2 * D.FP32 * top) / 127).all()
    s = s.astype(np.float64)[..., None]
    assert (np.abs(c * s - want) <= 0.5 * s * (1 + 512 * D.FP32) + off).all()


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_stage_by_stage(t):
    """Six tokens of the batch: each entry's outputs from what the entries before it really left, within that entry's own
    bounds. An adapter's part is many times those, so that none can be missing or another's."""
    L = Layer(t, GROUPS, SHARES, 16, "stages")
    n, H, Hk, DH = L.n, L.H, L.Hk, L.DH
    rng = rng_of(t, "stages")
    wq, wo = D.q4_values(*L.wq, L.C, L.W, 64), D.q4_values(*L.wo, H * DH, L.C, 32)
    shares = np.repeat(L.shared, np.diff(L.groups))
    for step in range(6):
        x = D.rows(rng, t, n, L.C)
        L.place(x, step)
        L.step()
        x64 = D.to_f64(t, x)
        z = x64 @ wq * 0.05
        of_z = D.q4_bound(t, x64, wq, z, 0.05, L.C)
        y, of_y = B.adapters_want(t, x, L.index, *L.ad, D.to_type(t, z))
        qkv = L.dqkv.download((n, L.W), D.np_type(t))
        got, bound = D.to_f64(t, qkv), of_y + (of_z + D.HALF[t] * np.abs(z)) * (1 + 2 * D.HALF[t])
        D.check(got, y, bound, f"{t} {step} qkv")
        has = L.index >= 0
        assert np.median((np.abs(y - z) / bound)[has]) > 20 and has.any()
        pos = shares + step
        heads = got.reshape(n, H + 2 * Hk, DH)
        wantq, size_of = D.norm_rope(heads[:, :H], L.gq, 1e-6, DH, False, L.freq, pos)
        q = L.dq.download((n, H * DH), D.np_type(t))
        D.check(D.to_f64(t, q).reshape(wantq.shape), wantq, D.rope_bound(t, wantq, size_of, DH), f"{t} {step} q")
        wantk, size_of = D.norm_rope(heads[:, H:H + Hk], L.gk, 1e-6, DH, False, L.freq, pos)
        L.kept.kc, L.kept.vc, L.kept.ks, L.kept.vs = L.kept.download()
        at, off = L.table[np.arange(n), pos // L.PAGE], pos % L.PAGE
        codes_within(L.kept.kc[at, :, off], L.kept.ks[at, :, off], wantk, D.rope_bound("f32", wantk, size_of, DH))
        vcode, vscale = B.codes_of(heads[:, H + Hk:].astype(np.float32))
        assert np.array_equal(L.kept.vc[at, :, off], vcode) and np.array_equal(L.kept.vs[at, :, off], vscale)
        want, bound = B.paged_want(t, q, *L.kept.values(), L.table, pos + 1, H, DH ** -0.5, L.WINDOW, L.SINKS, True, L.groups, L.shared)
        o = L.do.download((n, H * DH), D.np_type(t))
        D.check(D.to_f64(t, o), want, bound, f"{t} {step} o")
        o64 = D.to_f64(t, o)
        out = x64 + o64 @ wo * 0.05
        bound = D.q4_bound(t, o64, wo, out, 0.05, H * DH) + 2 * D.FP32 * (np.abs(x64) + np.abs(out))
        D.check(D.to_f64(t, L.out()), out, bound, f"{t} {step} out")


@pytest.mark.parametrize("t", D.TYPES)
def test_prompt_chunk_stage_by_stage(t):
    """As test_prompt_chunk_over_kept_rows, every row of the windowed attention, from the rows that were really read back."""
    H, Hk, Dh, page, rot = 4, 2, 64, 16, 64
    past, chunk = (50, 0, 131), (20, 33, 7)
    lens = [p + c for p, c in zip(past, chunk)]
    T = sum(chunk)
    rng, qkv, gq, gk, freq, _ = rope_inputs(t, T, H, Hk, Dh, rot, "chunk stages")
    table, pages = B.tables(rng, [-(-n // page) for n in lens])
    kept = B.fill_unwritten(B.Kept.random(rng, pages, Hk, page, Dh), table, past)
    pos = np.concatenate([p + np.arange(c) for p, c in zip(past, chunk)]).astype(np.int32)
    slots = table[np.repeat(np.arange(3), chunk), pos // page] * page + pos % page
    q, _, kept.kc, kept.vc, kept.ks, kept.vs = run_rope(t, qkv, H, kept, gq, gk, 1e-6, rot, False, freq, pos, slots)
    ks, qs = (np.concatenate(([0], np.cumsum(n))) for n in (lens, chunk))
    k, v = B.run_rows(t, kept, ks, table, int(ks[-1]))
    for got, want in zip((k, v), rows_want(t, kept, ks, table, int(ks[-1]))):
        assert np.array_equal(got, want)
    o = D.to_f64(t, D.run_window(t, q, k, v, H, Hk, Dh, 0.125, 60, 0, 2, qs, ks))
    for s in range(3):
        a, b = slice(qs[s], qs[s + 1]), slice(ks[s], ks[s + 1])
        want, bound = D.attention(t, *(D.to_f64(t, x).reshape(len(x), -1, Dh) for x in (q[a], k[b], v[b])),
                                  D.visible(chunk[s], lens[s], 60, 0, 2), 0.125)
        D.check(o[a].reshape(want.shape), want, bound, f"{t} {s}")


@pytest.mark.parametrize("H", (8, 96))
def test_shared_cache_of_rows_beyond_32_bits(H):
    """A prefix and own tokens in the last pages of a cache of more than 2^32 values, by 16 rows and by tiles: the results of a
    small one."""
    t, Hk, Dh, page, pages = "bf16", 8, 128, 1024, 4110
    assert pages * Hk * page * Dh > 1 << 32
    rng = rng_of("far rows of a cache")
    used = 3
    vals = [D.rows(rng, t, used, Hk, page, Dh) for _ in range(2)]
    lens, B_ = (1500, 1101, 2100), 3
    q = D.rows(rng, t, B_, H * Dh)
    outs = []
    for count, order in ((pages, (pages - 1, pages - 3, pages - 2)), (used, (0, 1, 2))):
        one = Hk * page * Dh * 2
        mem = [P.DeviceBuffer(count * one) for _ in range(2)]
        for m, v in zip(mem, vals):
            for i, p in enumerate(order):
                m.upload(v[i], offset=p * one)
        cache = P.KvCache(t, Hk, Dh, page, count, mem[0].ptr, mem[1].ptr)
        table = np.array([order] * B_, np.int32)
        outs.append(B.run_shared(t, q, cache, [0, B_], [1100], table, lens, H, 0.1, EVERY, 0, 1100, 1000))
    want, bound = B.paged_want(t, q, *(D.to_f64(t, v) for v in vals), table, lens, H, 0.1, EVERY, 0, False)
    D.check(D.to_f64(t, outs[1]), want, bound, str(H))
    assert np.array_equal(*outs)
