"""Plain 64-bit forms of a served batch's step (include/p2hip.h: p2h_qk_norm_rope_q8, p2h_kv_rows_q8,
p2h_attention_paged_q8, p2h_attention_shared, p2h_attention_shared_q8, p2h_adapters_add) and what their tests share.
Bounds are counted from the roundings a result goes through, as in _decoder.py."""
import numpy as np

import _decoder as D
import p2gemm as P

EVERY = P.EVERY_KEY


# ── the 8-bit cache ─────────────────────────────────────────────────────────────────────────────────────────────

def codes_of(x):
    """float32 heads [..., Dh] → (codes, scales) in 32 bits, each operation rounded as the header says."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(-1)
    some = top >= np.float32(2.0 ** -100)
    by = np.where(some, np.float32(127) / np.where(some, top, np.float32(1)), np.float32(0))
    return np.rint(x * by[..., None]).astype(np.int8), np.where(some, top / np.float32(127), np.float32(0))


class Kept:
    """An 8-bit cache on the host and on the device: codes [pages][Hk][page][Dh], scales [pages][Hk][page]."""

    def __init__(self, kc, vc, ks, vs):
        self.kc, self.vc, self.ks, self.vs = kc, vc, ks, vs
        self.dev = [D.device(a) for a in (kc, vc, ks, vs)]
        pages, Hk, page, Dh = kc.shape
        self.c = P.KvCacheQ8(Hk, Dh, page, pages, *(d.ptr for d in self.dev))

    @classmethod
    def random(cls, rng, pages, Hk, page, Dh):
        kc, vc = (rng.integers(-127, 128, (pages, Hk, page, Dh)).astype(np.int8) for _ in range(2))
        ks, vs = (rng.uniform(0.004, 0.02, (pages, Hk, page)).astype(np.float32) for _ in range(2))
        return cls(kc, vc, ks, vs)

    def download(self, stream=None):
        shapes = (self.kc.shape, self.vc.shape, self.ks.shape, self.vs.shape)
        return [d.download(s, t, stream) for d, s, t in zip(self.dev, shapes, (np.int8, np.int8, np.float32, np.float32))]

    def values(self):
        """Keys and values in 64 bits."""
        return [c.astype(np.float64) * s.astype(np.float64)[..., None] for c, s in ((self.kc, self.ks), (self.vc, self.vs))]


def fill_unwritten(kept, table, lens, only=None):
    """What no token was written to holds anything: codes of −128 and scales that are NaN."""
    page = kept.kc.shape[2]
    used = np.zeros(kept.ks.shape[::2], bool)
    for s, n in enumerate(lens):
        for t in range(n):
            p = table[s][t // page]
            if 0 <= p < used.shape[0]:
                used[p, t % page] = True
    at = np.nonzero(~used)
    for c, sc in ((kept.kc, kept.ks), (kept.vc, kept.vs)):
        c[at[0], :, at[1]] = -128
        sc[at[0], :, at[1]] = np.nan
    return Kept(kept.kc, kept.vc, kept.ks, kept.vs)


def run_rows(t, kept, starts, table, rows, pad=0, stream=None):
    Hk, Dh = kept.kc.shape[1], kept.kc.shape[3]
    ld = Hk * Dh + pad
    dk, dv = D.preset(t, (max(rows, 1), ld)), D.preset(t, (max(rows, 1), ld))
    ds, dt = D.device(np.asarray(starts, np.int32)), D.device(np.asarray(table, np.int32))
    P.kv_rows_q8_dev(t, kept.c, rows, len(starts) - 1, ds.ptr, dt.ptr, table.shape[1], dk.ptr, ld, dv.ptr, ld, stream)
    return [b.download((rows, ld), D.np_type(t), stream) for b in (dk, dv)]


def tables(rng, needs, spare=3, width=1):
    """Tables of pages in random order for sequences of that many pages each, entries behind them not pages."""
    order = rng.permutation(sum(needs) + spare)
    table = np.full((len(needs), max(max(needs, default=0), width) + 1), -7, np.int32)
    at = 0
    for s, n in enumerate(needs):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(needs) + spare


# ── attention ───────────────────────────────────────────────────────────────────────────────────────────────────

def attend(t, q, k, v, seen, scale, q8):
    """One query [H][Dh] over keys and values [n][Hk][Dh] in 64 bits → (o, bound). As _decoder.attention counts; codes of
    fp32 rows are multiplied in three pieces of the query, 3 · Dh additions a score and three for each weighted value, so
    three times its bound holds. (Parts without keys join exactly.)"""
    o, bound = D.attention(t, q[None], k, v, seen[None], scale)
    return o[0], bound[0] * (3 if q8 and t == "f32" else 1)


def tokens(cache, row, n):
    """Tokens 0 .. n − 1 of a table row from [pages][Hk][page][Dh] in 64 bits, and which of them a page holds."""
    pages, _, page, _ = cache.shape
    j = np.arange(n)
    p = np.asarray(row)[np.minimum(j // page, len(row) - 1)] if n else np.zeros(0, int)
    held = (p >= 0) & (p < pages) & (j // page < len(row))
    return np.where(held[:, None, None], cache[np.where(held, p, 0), :, j % page], 0.0), held


def paged_want(t, q, K, V, table, lens, H, scale, window, sinks, q8, groups=None, shared=None):
    """[B][H·Dh] in 64 bits and its bound; sequences of no group NaN. Values that no page holds or no mask lets through are
    not looked at."""
    Dh, page = K.shape[3], K.shape[2]
    want, bound = np.full((len(lens), H * Dh), np.nan), np.zeros((len(lens), H * Dh))
    for s, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * page)
        (k, held), (v, _) = tokens(K, table[s], n), tokens(V, table[s], n)
        if groups is not None:
            g = [i for i in range(len(groups) - 1) if groups[i] <= s < groups[i + 1]]
            if not g:
                continue
            m = min(max(shared[g[0]], 0), n)
            lead = table[groups[g[0]]]
            k[:m], held[:m] = tokens(K, lead, m)
            v[:m] = tokens(V, lead, m)[0]
        seen = D.visible(1, n, window, 0, sinks)[0] & held
        k, v = (np.where(seen[:, None, None], a, 0.0) for a in (k, v))
        o, e = attend(t, D.to_f64(t, q[s]).reshape(H, Dh), k, v, seen, scale, q8)
        want[s], bound[s] = o.reshape(-1), e.reshape(-1)
    return want, bound


def run_paged(t, q, kept, table, lens, H, scale, window, sinks, split=True, max_len=None, stream=None):
    Hk, Dh, B = kept.kc.shape[1], kept.kc.shape[3], q.shape[0]
    dq, dt, dl = D.device(q), D.device(np.asarray(table, np.int32)), D.device(np.asarray(lens, np.int32))
    do = D.preset(t, (max(B, 1), H * Dh))
    most = int(max(lens)) if max_len is None else max_len
    n = P.attention_paged_q8_workspace_bytes(kept.c, B, H, most, window, sinks) if split else 0
    ws = P.Workspace(n)
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    P.attention_paged_q8_dev(t, kept.c, B, H, dq.ptr, H * Dh, dt.ptr, table.shape[1], dl.ptr, most, scale, window, sinks,
                             do.ptr, H * Dh, ws.ptr if split else None, n, stream)
    return do.download((B, H * Dh), D.np_type(t), stream)


def row_cache(t, kc, vc):
    """A cache of rows on the device; keeps its buffers."""
    dk, dv = D.device(kc), D.device(vc)
    pages, Hk, page, Dh = kc.shape
    c = P.KvCache(t, Hk, Dh, page, pages, dk.ptr, dv.ptr)
    c.keep = (dk, dv)
    return c


def run_shared(t, q, cache, groups, shared, table, lens, H, scale, window, sinks, max_shared, max_own, pad=0, stream=None):
    """cache: a KvCache or a KvCacheQ8."""
    B, Dh = q.shape[0], cache.head_dim
    dq, dt, dl = D.device(q), D.device(np.asarray(table, np.int32)), D.device(np.asarray(lens, np.int32))
    dg, dsh = D.device(np.asarray(groups, np.int32)), D.device(np.asarray(shared, np.int32))
    ldo = H * Dh + pad
    do = D.preset(t, (max(B, 1), ldo))
    q8 = isinstance(cache, P.KvCacheQ8)
    need = (P.attention_shared_q8_workspace_bytes if q8 else P.attention_shared_workspace_bytes)(
        cache, B, len(shared), H, max_shared, max_own, window, sinks)
    ws = P.Workspace(need)
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    args = (cache, B, len(shared), H, dq.ptr, q.shape[1], dg.ptr, dsh.ptr, dt.ptr, table.shape[1], dl.ptr, max_shared,
            max_own, scale, window, sinks, do.ptr, ldo, ws.ptr, need, stream)
    if q8:
        P.attention_shared_q8_dev(t, *args)
    else:
        P.attention_shared_dev(*args)
    return do.download((B, ldo), D.np_type(t), stream)


# ── adapters ────────────────────────────────────────────────────────────────────────────────────────────────────

def adapter_set(rng, t, count, rank, K, N):
    return (D.rows(rng, t, count, rank, K, scale=K ** -0.5), D.rows(rng, t, count, N, rank, scale=rank ** -0.5),
            rng.uniform(0.5, 2.0, count).astype(np.float32))


def adapters_want(t, x, index, a, b, scale, z):
    """(y, bound) in 64 bits. A sum over K and one over the rank, each addition off by at most one step (2^-23) of the sum of
    sizes, K's over waves and parts too (64 more); the scale and the sum with z one rounding each; one to the type."""
    x, a, b = D.to_f64(t, x), D.to_f64(t, a), D.to_f64(t, b)
    y = np.zeros((x.shape[0], b.shape[1])) if z is None else D.to_f64(t, z).copy()
    bound = np.zeros(y.shape)
    for m, i in enumerate(index):
        if 0 <= i < a.shape[0]:
            h, mag = a[i] @ x[m], np.abs(a[i]) @ np.abs(x[m])
            s = float(scale[i])
            add = s * (b[i] @ h)
            off = s * (np.abs(b[i]) @ ((x.shape[1] + 64) * 2 * D.FP32 * mag + (a.shape[1] + 4) * 2 * D.FP32 * np.abs(h)))
            y[m] += add
            bound[m] = off + 2 * D.FP32 * np.abs(y[m]) + D.HALF[t] * np.abs(y[m]) + D.TINY[t]
    return y, bound


def run_adapters(t, x, index, a, b, scale, z, in_place=False, pads=(0, 0, 0), stream=None, ws=None):
    M, K = x.shape
    count, N, rank = b.shape
    ldx, ldz, ldy = K + pads[0], N + pads[1], N + pads[2]

    def padded(v, ld):
        out = np.full((max(M, 1), ld), 0x7F if t == "bf16" else np.nan, D.np_type(t))
        out[:M, :v.shape[1]] = v
        return out

    dx, di = D.device(padded(x, ldx)), D.device(np.asarray(index, np.int32))
    da, db, ds = D.device(a), D.device(b), D.device(scale)
    dz = None if z is None else D.device(padded(z, ldz))
    dy = dz if in_place else D.preset(t, (max(M, 1), ldy))
    ld = ldz if in_place else ldy
    ad = P.Adapters(t, count, rank, K, N, da.ptr, db.ptr, ds.ptr)
    need = P.adapters_workspace_bytes(ad, M)
    w = P.Workspace(need)
    w.upload(np.full(w.nbytes, 0xFF, np.uint8))
    P.adapters_add_dev(ad, M, dx.ptr, ldx, di.ptr, None if dz is None else dz.ptr, ldz, dy.ptr, ld, w.ptr, need, stream)
    return dy.download((M, ld), D.np_type(t), stream)
