"""Calls of a served batch's entries that their documentation allows, at its ends: the most rows, sequences and groups, the widest
linears, rows that lie beside each other in one buffer, in place, replayed."""
import numpy as np
import pytest

import _batch as B
import _decoder as D
import p2gemm as P
from test_gpu_batch import paged_case, rng_of, rope_inputs, shared_cache, shared_case

pytestmark = pytest.mark.gpu
EVERY = P.EVERY_KEY


def bits(a):
    return np.ascontiguousarray(a).view(np.uint8)


# ── rows beside each other ──────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("t", D.TYPES)
def test_rows_beside_each_other(t):
    """Keys and values as columns of one buffer, and at pitches of their own: the same rows."""
    Hk, Dh, page, lens = 3, 64, 32, (70, 0, 33)
    rng = rng_of("beside", t)
    table, pages = B.tables(rng, [-(-n // page) for n in lens])
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    starts, rows, w = np.concatenate(([0], np.cumsum(lens))), sum(lens), Hk * Dh
    want = B.run_rows(t, kept, starts, table, rows)
    ds, dt = D.device(starts.astype(np.int32)), D.device(table)
    both = D.preset(t, (rows, 2 * w + 16))
    P.kv_rows_q8_dev(t, kept.c, rows, 3, ds.ptr, dt.ptr, table.shape[1], both.ptr, 2 * w + 16, both.ptr + (w + 8) * D.size(t),
                     2 * w + 16)
    got = both.download((rows, 2 * w + 16), D.np_type(t))
    assert np.array_equal(bits(got[:, :w]), bits(want[0])) and np.array_equal(bits(got[:, w + 8:2 * w + 8]), bits(want[1]))
    assert (bits(got[:, w:w + 8]) == 0xFF).all() and (bits(got[:, 2 * w + 8:]) == 0xFF).all()
    dk, dv = D.preset(t, (rows, w + 8)), D.preset(t, (rows, w + 64))
    P.kv_rows_q8_dev(t, kept.c, rows, 3, ds.ptr, dt.ptr, table.shape[1], dk.ptr, w + 8, dv.ptr, w + 64)
    for d, ld, x in ((dk, w + 8, want[0]), (dv, w + 64, want[1])):
        assert np.array_equal(bits(d.download((rows, ld), D.np_type(t))[:, :w]), bits(x))


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("T", (9, 300))
def test_rope_in_place(t, T):
    """Queries and keys in their own columns, values untouched: the same rows and codes."""
    H, Hk, Dh, page, rot = 4, 2, 64, 16, 32
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "place")
    pages = -(-T // page) + 1
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    one, two = (B.Kept(*(np.zeros(s, d) for s, d in (((pages, Hk, page, Dh), np.int8),) * 2 + (((pages, Hk, page), np.float32),) * 2))
                for _ in range(2))
    dx, dgq, dgk, df, dp, ds = (D.device(a) for a in (qkv, gq, gk, freq, pos, slots))
    W, es = qkv.shape[1], D.size(t)
    q, k = D.preset(t, (T, H * Dh)), D.preset(t, (T, Hk * Dh))
    P.qk_norm_rope_q8_dev(t, T, H, Hk, Dh, dx.ptr, W, dgq.ptr, dgk.ptr, 1e-6, rot, False, df.ptr, dp.ptr, q.ptr, H * Dh, k.ptr,
                          Hk * Dh, one.c, ds.ptr)
    P.qk_norm_rope_q8_dev(t, T, H, Hk, Dh, dx.ptr, W, dgq.ptr, dgk.ptr, 1e-6, rot, False, df.ptr, dp.ptr, dx.ptr, W,
                          dx.ptr + H * Dh * es, W, two.c, ds.ptr)
    got = dx.download((T, W), D.np_type(t))
    assert np.array_equal(bits(got[:, :H * Dh]), bits(q.download((T, H * Dh), D.np_type(t))))
    assert np.array_equal(bits(got[:, H * Dh:(H + Hk) * Dh]), bits(k.download((T, Hk * Dh), D.np_type(t))))
    assert np.array_equal(bits(got[:, (H + Hk) * Dh:]), bits(qkv[:, (H + Hk) * Dh:]))
    for a, b in zip(one.download(), two.download()):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("kind", ("paged", "rows", "q8"))
@pytest.mark.parametrize("H", (4, 48))
def test_queries_as_columns_of_wider_rows(t, kind, H):
    """q as the first columns of q | k | v rows, o as columns of wider ones: the same bits."""
    Hk, page, Dh, lens = 2, 16, 64, (60, 90, 41, 45)
    if kind == "paged":
        q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "wide")
        want = B.run_paged(t, q, kept, table, lens, H, 0.1, EVERY, 0)
        need = P.attention_paged_q8_workspace_bytes(kept.c, 4, H, 90)
    else:
        rng, lens, starts, shared, table, pages, reach = shared_case(t, [(40, lens)], H, Hk, page, Dh, "wide")
        cache, _, _ = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
        q = D.rows(rng, t, 4, H * Dh)
        want = B.run_shared(t, q, cache, starts, shared, table, lens, H, 0.1, EVERY, 0, 40, 50)
        need = (P.attention_shared_q8_workspace_bytes if kind == "q8" else P.attention_shared_workspace_bytes)(cache, 4, 1, H, 40, 50)
        dg, dsh = D.device(np.array(starts, np.int32)), D.device(np.array(shared, np.int32))
    W = (H + 2 * Hk) * Dh
    wide = np.full((4, W), 0x7FC0 if t == "bf16" else np.nan, D.np_type(t))
    wide[:, :H * Dh] = q
    dq, dt, dl, o, ws = D.device(wide), D.device(table), D.device(np.array(lens, np.int32)), D.preset(t, (4, W)), P.Workspace(need)
    if kind == "paged":
        P.attention_paged_q8_dev(t, kept.c, 4, H, dq.ptr, W, dt.ptr, table.shape[1], dl.ptr, 90, 0.1, EVERY, 0, o.ptr, W, ws.ptr, need)
    else:
        args = (cache, 4, 1, H, dq.ptr, W, dg.ptr, dsh.ptr, dt.ptr, table.shape[1], dl.ptr, 40, 50, 0.1, EVERY, 0, o.ptr, W, ws.ptr, need)
        if kind == "q8":
            P.attention_shared_q8_dev(t, *args)
        else:
            P.attention_shared_dev(*args)
    got = o.download((4, W), D.np_type(t))
    assert np.array_equal(bits(got[:, :H * Dh]), bits(want)) and (bits(got[:, H * Dh:]) == 0xFF).all()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M", (1, 20, 300, 600))
def test_adapters_on_columns(t, M):
    """Each of q, k and v of q | k | v rows has adapters of its own, in place, one call after the other: no column of the others
    is touched. Of a single row the pitches say nothing."""
    K, N, rank, count = 72, 64, 8, 3
    rng = rng_of("columns", t, M)
    x, z, index = D.rows(rng, t, M, K), D.rows(rng, t, M, 3 * N), rng.integers(-1, count, M)
    sets = [B.adapter_set(rng, t, count, rank, K, N) for _ in range(3)]
    dx, di, dy = D.device(x), D.device(index.astype(np.int32)), D.device(z)
    for i in (1, 2, 0):
        keep = [D.device(v) for v in sets[i]]
        ad = P.Adapters(t, count, rank, K, N, *(d.ptr for d in keep))
        ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
        at = dy.ptr + i * N * D.size(t)
        P.adapters_add_dev(ad, M, dx.ptr, K, di.ptr, at, 3 * N + (7 if M == 1 else 0), at, 3 * N, ws.ptr, ws.nbytes)
        P.sync()
    got = dy.download((M, 3 * N), D.np_type(t))
    for i in range(3):
        want, bound = B.adapters_want(t, x, index, *sets[i], z[:, i * N:(i + 1) * N])
        D.check(D.to_f64(t, got[:, i * N:(i + 1) * N]), want, bound, f"{t} {M} {i}")


# ── the most of everything ──────────────────────────────────────────────────────────────────────────────────────

def test_rows_of_thousands_of_sequences():
    t, Hk, Dh, page, n = "f16", 1, 64, 16, 20000
    rng = rng_of("thousands")
    lens = rng.integers(0, 4, n)
    lens[rng.integers(0, n, 20)] = 40
    starts = np.concatenate(([0], np.cumsum(lens)))
    rows, pages = int(starts[-1]), 50
    table = rng.integers(-1, pages + 1, (n, 3)).astype(np.int32)
    kept = B.Kept.random(rng, pages, Hk, page, Dh)
    seq = np.repeat(np.arange(n), lens)
    at = np.arange(rows) - starts[seq]
    p = table[seq, at // page]
    held = (p >= 0) & (p < pages)
    for got, c, sc in zip(B.run_rows(t, kept, starts, table, rows), (kept.kc, kept.vc), (kept.ks, kept.vs)):
        q = np.where(held, p, 0)
        want = c[q, 0, at % page].astype(np.float32) * sc[q, 0, at % page][:, None]
        assert np.array_equal(got, D.to_type(t, np.where(held[:, None], want, 0)))


def test_most_sequences():
    """65536 sequences of sixteen kinds: each what a call of the sixteen gives."""
    t, H, Hk, page, Dh, n = "bf16", 4, 2, 16, 64, 65536
    lens = (1, 0, 5, 16, 17, 40, 33, 2, 31, 32, 48, 7, 0, 20, 64, 50)
    q, kept, table = paged_case(t, lens, H, Hk, page, Dh, "most")
    want = B.run_paged(t, q, kept, table, lens, H, 0.1, 30, 3)
    kinds = np.arange(n) % 16
    got = B.run_paged(t, q[kinds], kept, np.ascontiguousarray(table[kinds]), np.array(lens)[kinds], H, 0.1, 30, 3)
    assert np.array_equal(got, want[kinds])


@pytest.mark.parametrize("kind", ("rows", "q8"))
def test_thousands_of_groups(kind):
    t, H, Hk, page, Dh, n = "bf16", 2, 1, 16, 64, 9000
    kinds = [(3, (4, 9)), (40, (41,)), (0, (5, 7, 2)), (17, (60, 17, 0, 18)), (33, ())]
    rng, lens, starts, shared, table, pages, reach = shared_case(t, kinds, H, Hk, page, Dh, "groups")
    cache, K, V = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, len(lens), H * Dh)
    want, bound = B.paged_want(t, q, K, V, table, lens, H, 0.1, EVERY, 0, kind == "q8", starts, shared)
    seqs = np.tile(np.arange(len(lens)), n // 5)
    st = np.concatenate(([0], np.cumsum(np.tile(np.diff(starts), n // 5))))
    got = B.run_shared(t, q[seqs], cache, st, np.tile(shared, n // 5), np.ascontiguousarray(table[seqs]), np.array(lens)[seqs], H, 0.1,
                       EVERY, 0, 40, 40)
    D.check(D.to_f64(t, got[:len(lens)]), want, bound, kind)
    assert np.array_equal(got, np.tile(got[:len(lens)], (n // 5, 1)))


def test_most_rows_of_adapters():
    """2^20 - 16 rows: each what calls of a few thousand give."""
    t, M, K, N, rank, count = "bf16", 16 * 65535, 64, 72, 8, 5
    rng = rng_of("most rows")
    x, z = D.rows(rng, t, 4096, K), D.rows(rng, t, 4096, N)
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    index = np.sort(rng.integers(-1, count, 4096))
    one = B.run_adapters(t, x, index, a, b, scale, z)
    want, bound = B.adapters_want(t, x, index, a, b, scale, z)
    D.check(D.to_f64(t, one), want, bound)
    of = np.arange(M) % 4096
    assert np.array_equal(B.run_adapters(t, x[of], index[of], a, b, scale, z[of]), one[of])


@pytest.mark.parametrize("M,K,N", ((2, 1 << 23, 3), (2, 40, 1 << 23), (20, (1 << 23) - 1, 5), (300, 16, (1 << 21) + 3)))
def test_widest_linears(M, K, N):
    t, rank, count = "bf16", 8, 2
    rng = rng_of("widest", M, K, N)
    x, z = D.rows(rng, t, M, K), D.rows(rng, t, 1, N)
    z = np.ascontiguousarray(np.broadcast_to(z, (M, N)))
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    index = rng.integers(-1, count, M)
    index[:2] = (1, 0)
    got = B.run_adapters(t, x, index, a, b, scale, z)
    for m in (0, 1, M // 2, M - 1):
        want, bound = B.adapters_want(t, x[m:m + 1], index[m:m + 1], a, b, scale, z[m:m + 1])
        D.check(D.to_f64(t, got[m:m + 1]), want, bound, str(m))


# ── again ───────────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M", (3, 40, 300, 600))
def test_adapters_replayed(t, M):
    """A captured call, in place, replayed with new rows and indexes, eager calls in between: their bits."""
    K, N, rank, count = 264, 200, 16, 4
    rng, s = rng_of("replayed", t, M), P.Stream()
    a, b, scale = B.adapter_set(rng, t, count, rank, K, N)
    da, db, dsc = (D.device(v) for v in (a, b, scale))
    ad = P.Adapters(t, count, rank, K, N, da.ptr, db.ptr, dsc.ptr)
    ws = P.Workspace(P.adapters_workspace_bytes(ad, M))
    dx, dy, di = D.preset(t, (M, K)), D.preset(t, (M, N)), D.device(np.zeros(M, np.int32))
    with P.Graph(s) as g:
        P.adapters_add_dev(ad, M, dx.ptr, K, di.ptr, dy.ptr, N, dy.ptr, N, ws.ptr, ws.nbytes, s.ptr)
    for turn in range(4):
        x, z, index = D.rows(rng, t, M, K), D.rows(rng, t, M, N), rng.integers(-1, count, M).astype(np.int32)
        dx.upload(x)
        dy.upload(z)
        di.upload(index)
        P.sync()
        g.launch()
        s.sync()
        got = dy.download((M, N), D.np_type(t))
        assert np.array_equal(bits(got), bits(B.run_adapters(t, x, index, a, b, scale, z))), turn


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("t,H", (("f32", 4), ("bf16", 4), ("bf16", 96), ("f16", 96)))
def test_shared_replayed(kind, t, H):
    """A captured call replayed with other groups, prefixes and lengths: the bits of eager calls."""
    Hk, page, Dh, s = 2, 16, 64, P.Stream()
    rng, lens, starts, shared, table, pages, reach = shared_case(t, [(100, (101, 130, 160)), (40, (41, 80))], H, Hk, page, Dh, "replay")
    cache, _, _ = shared_cache(rng, t, kind, pages, Hk, page, Dh, table, reach)
    q = D.rows(rng, t, 5, H * Dh)
    dq, dt, dg, dsh, dl = (D.device(np.asarray(v) if v is q else np.asarray(v, np.int32)) for v in (q, table, starts, shared, lens))
    need = (P.attention_shared_q8_workspace_bytes if kind == "q8" else P.attention_shared_workspace_bytes)(cache, 5, 2, H, 100, 60)
    ws, o = P.Workspace(need), D.preset(t, (5, H * Dh))
    args = (cache, 5, 2, H, dq.ptr, H * Dh, dg.ptr, dsh.ptr, dt.ptr, table.shape[1], dl.ptr, 100, 60, 0.1, EVERY, 0, o.ptr, H * Dh,
            ws.ptr, need, s.ptr)
    with P.Graph(s) as g:
        if kind == "q8":
            P.attention_shared_q8_dev(t, *args)
        else:
            P.attention_shared_dev(*args)
    for st, sh, ln in ((starts, shared, lens), ([0, 3, 3], [100, 0], [70, 0, 160, 0, 0]), ([0, 1, 5], [0, 30], [20, 35, 31, 41, 80]),
                       (starts, [64, 40], lens)):
        for d, v in ((dg, st), (dsh, sh), (dl, ln)):
            d.upload(np.asarray(v, np.int32))
        o.upload(np.full(o.nbytes, 0xFF, np.uint8))
        P.sync()
        g.launch()
        s.sync()
        got = o.download((5, H * Dh), D.np_type(t))
        assert np.array_equal(bits(got), bits(B.run_shared(t, q, cache, st, sh, table, ln, H, 0.1, EVERY, 0, 100, 60)))
