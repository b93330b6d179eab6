"""Plain 64-bit forms of a decoder layer's step (include/p2hip.h: p2h_q4_gemv, p2h_qk_norm_rope, p2h_attention_window,
p2h_attention_paged) and what their tests share: element types on the host, device runs on preset buffers, and error
bounds counted from the roundings a result goes through."""
import numpy as np

import p2gemm as P

TYPES = ("f32", "f16", "bf16")
# half a step of each type, relative to the value
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# a value below the type's smallest normal is off by at most half a step of the subnormals
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -133}
FP32 = 2.0 ** -24


def size(t):
    return 4 if t == "f32" else 2


def to_type(t, a):
    """float array → the bits of type t as the device holds them."""
    a = np.asarray(a, np.float32)
    if t == "f32":
        return np.ascontiguousarray(a)
    if t == "f16":
        with np.errstate(over="ignore"):
            return np.ascontiguousarray(a.astype(np.float16))
    u = a.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.ascontiguousarray(np.where(np.isnan(a), np.uint16(0x7FC0), r))


def to_f64(t, a):
    if t == "bf16":
        return (np.asarray(a, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(a).astype(np.float64)


def np_type(t):
    return {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[t]


def rows(rng, t, *shape, scale=1.0):
    return to_type(t, rng.standard_normal(shape) * scale)


def nibbles(packed, n):
    return np.stack((packed & 15, packed >> 4), 2).reshape(packed.shape[0], -1)[:, :n]


# ── 4-bit weights ───────────────────────────────────────────────────────────────────────────────────────────────

def q4_weight(rng, K, N, group, zeros):
    groups, half = -(-K // group), (N + 1) // 2
    return (rng.integers(0, 256, (K, half), dtype=np.uint8),
            (rng.uniform(0.5, 1.5, (groups, N)) / 64).astype(np.float16),
            rng.integers(0, 256, (groups, half), dtype=np.uint8) if zeros else None)


def q4_values(codes, scales, zeros, K, N, group):
    at = np.arange(K) // group
    z = 8.0 if zeros is None else nibbles(zeros, N).astype(np.float64)[at]
    return (nibbles(codes, N).astype(np.float64) - z) * scales.astype(np.float64)[at]


def q4_bound(t, x, w, out, alpha, K):
    """Products are exact; each is added at most once in its group of <= 128, its wave's units and the 16 waves, each
    addition off by at most one step (2^-23) of a sum no larger than sum |x w|; the group's scale, alpha and beta are one
    rounding each; then one rounding to the type."""
    adds = 128 + K // 128 + 1 + 16 + 4
    return adds * 2 * FP32 * abs(alpha) * (np.abs(x) @ np.abs(w)) + HALF[t] * np.abs(out) + TINY[t]


# ── norm and rotation ───────────────────────────────────────────────────────────────────────────────────────────

def norm_rope(x, gamma, eps, rot, interleaved, freq, pos):
    """x [T][heads][Dh] in 64 bits → (result, bound's scale: the size of the terms each element is made of)."""
    n = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * gamma.astype(np.float64)
    y, size_of = n.copy(), np.abs(n)
    if rot:
        ang = (pos.astype(np.float64)[:, None] * freq.astype(np.float64))[:, None, :]
        c, s = np.cos(ang), np.sin(ang)
        i = np.arange(rot // 2) * (2 if interleaved else 1)
        j = i + (1 if interleaved else rot // 2)
        a, b = n[..., i], n[..., j]
        y[..., i], y[..., j] = a * c - b * s, b * c + a * s
        both = np.abs(a) + np.abs(b)
        size_of[..., i] = size_of[..., j] = both
    return y, size_of


def rope_bound(t, y, size_of, Dh):
    """The mean square is a sum of Dh non-negative terms (Dh / 2 roundings of the norm, as it goes in by its root), root,
    quotient, two products; the turn's sine and cosine are within 2^-22; two products and a sum; one rounding."""
    return (Dh / 2 + 4 + 4 + 3) * FP32 * size_of + HALF[t] * np.abs(y) + TINY[t]


# ── attention ───────────────────────────────────────────────────────────────────────────────────────────────────

def visible(nq, nk, window, ahead, sinks):
    """[nq][nk]: query i stands at i + nk − nq."""
    p = np.arange(nq, dtype=np.int64)[:, None] + nk - nq
    j = np.arange(nk, dtype=np.int64)[None, :]
    return (j <= p + ahead) & ((p - j < window) | (j < sinks))


def attention(t, q, k, v, seen, scale):
    """q [nq][H][Dh], k and v [nk][Hk][Dh] in 64 bits, seen [nq][nk] → (o, bound). The bound: a score is a sum of Dh
    products (each addition off by 2^-23 of sum |q k|), a weight's exponent carries that and 4 roundings of the score,
    the exponential 2^-22; 16-bit rows round each weight to the type; the weighted sum adds at most nk + 8 times (blocks,
    waves and parts rescale by factors of a rounding each); one quotient; one rounding to the type. A weight's error acts
    on its own v and, through the sum of weights, on o."""
    H, Hk, Dh = q.shape[1], k.shape[1], q.shape[2]
    per = H // Hk
    o = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for h in range(H):
        kk, vv = k[:, h // per], v[:, h // per]
        s = (q[:, h] @ kk.T) * scale
        mag = (np.abs(q[:, h]) @ np.abs(kk).T) * scale
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True, initial=-np.inf)
        top = np.where(np.isfinite(top), top, 0.0)
        w = np.exp(s - top)
        den = w.sum(1, keepdims=True)
        w = w / np.where(den == 0, 1.0, den)
        o[:, h] = w @ vv
        gap = np.where(seen, np.abs(s - top) + np.abs(top), 0.0)
        off = np.where(seen, Dh * 2 * FP32 * mag + 4 * FP32 * gap + 4 * FP32, 0.0)
        off = off.max(1, keepdims=True, initial=0.0)   # of any weight of the row
        each = 2 * off + (HALF[t] if t != "f32" else 0.0) + (w.shape[1] + 8) * 2 * FP32
        bound[:, h] = each * (w @ np.abs(vv) + np.abs(o[:, h])) + HALF[t] * np.abs(o[:, h]) + TINY[t]
    return o, bound


# ── device runs ─────────────────────────────────────────────────────────────────────────────────────────────────

def device(a, spare=0):
    """The array on the device, `spare` elements of 0xA5 bytes behind it."""
    a = np.ascontiguousarray(a)
    b = P.DeviceBuffer(a.nbytes + spare * a.itemsize + 16)
    b.upload(np.full(b.nbytes, 0xA5, np.uint8))
    if a.nbytes:
        b.upload(a)
    return b


def preset(t, shape):
    """A buffer of NaN bytes (0xFF) of that many elements."""
    n = int(np.prod(shape)) * size(t)
    return P.DeviceBuffer(max(n, 16)).upload(np.full(max(n, 16), 0xFF, np.uint8))


def check(got, want, bound, what=""):
    assert np.isfinite(got).all(), f"{what}: not finite at {np.argwhere(~np.isfinite(got))[:4].tolist()}"
    off = np.abs(got - want)
    bad = off > bound
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {got.size} off, worst {float((off / bound).max()):.3g} bounds at "
                           f"{np.unravel_index(int((off / bound).argmax()), got.shape)}")


def run_q4(t, x, weight, K, N, group, alpha=1.0, beta=0.0, y0=None, ldx=None, ldy=None, stream=None):
    M = x.shape[0]
    ldx, ldy = ldx or K, ldy or N
    xs = np.full((max(M, 1), ldx), 0x7F, np_type(t)) if t == "bf16" else np.full((max(M, 1), ldx), np.nan, np_type(t))
    xs[:M, :K] = x
    w = P.Q4Weight(*weight, K, N, group)
    dx = device(xs)
    ys = np.zeros((max(M, 1), ldy), np_type(t)) if y0 is None else y0
    dy = device(ys) if y0 is not None else preset(t, (max(M, 1), ldy))
    P.q4_gemv_dev(t, M, N, K, alpha, dx.ptr, ldx, w, beta, dy.ptr, ldy, stream)
    return dy.download(ys.shape, np_type(t), stream)


def run_window(t, q, k, v, H, Hk, Dh, scale, window, ahead, sinks, qs=None, ks=None, pad=0, stream=None, o0=None):
    """q [nq][H·Dh (+ pad)] and so on; starts as int32 arrays or None."""
    nq, nk = q.shape[0], k.shape[0]
    dq, dk, dv = device(q), device(k), device(v)
    dqs = device(np.asarray(qs, np.int32)) if qs is not None else None
    dks = device(np.asarray(ks, np.int32)) if ks is not None else None
    ldo = H * Dh + pad
    do = preset(t, (max(nq, 1), ldo)) if o0 is None else device(o0)
    P.attention_window_dev(t, nq, nk, 1 if qs is None else len(qs) - 1, dqs.ptr if dqs else None, dks.ptr if dks else None,
                           H, Hk, Dh, dq.ptr, q.shape[1], dk.ptr, k.shape[1], dv.ptr, v.shape[1], scale, window, ahead,
                           sinks, do.ptr, ldo, stream)
    return do.download((nq, ldo), np_type(t), stream)


def run_paged(t, q, kc, vc, table, lens, H, scale, window, sinks, split=True, max_len=None, stream=None):
    """q [B][H·Dh]; kc, vc [pages][Hk][page][Dh]; table [B][ld] → o [B][H·Dh]."""
    pages, Hk, page, Dh = kc.shape
    B = q.shape[0]
    dq, dk, dv = device(q), device(kc), device(vc)
    dt, dl = device(np.asarray(table, np.int32)), device(np.asarray(lens, np.int32))
    do = preset(t, (max(B, 1), H * Dh))
    cache = P.KvCache(t, Hk, Dh, page, pages, dk.ptr, dv.ptr)
    most = int(max(lens)) if max_len is None else max_len
    n = P.attention_paged_workspace_bytes(cache, B, H, most, window, sinks) if split else 0
    ws = P.Workspace(n)
    ws.upload(np.full(ws.nbytes, 0xFF, np.uint8))
    P.attention_paged_dev(cache, B, H, dq.ptr, H * Dh, dt.ptr, table.shape[1], dl.ptr, most, scale, window, sinks, do.ptr,
                          H * Dh, ws.ptr if split else None, n, stream)
    return do.download((B, H * Dh), np_type(t), stream)


def gather(t, cache, row, n, page, pages):
    """Tokens 0 .. n − 1 of a sequence as [n][Hk][Dh] in 64 bits, and which of them a page holds."""
    j = np.arange(n)
    p = np.asarray(row)[j // page] if n else np.zeros(0, int)
    held = (p >= 0) & (p < pages)
    vals = to_f64(t, cache)[np.where(held, p, 0), :, j % page]
    return np.where(held[:, None, None], vals, 0.0), held


# ── how far 32-bit results may be off on the whole ──────────────────────────────────────────────────────────────

# Relative 2-norms of the error of fp32 results, beside the elementwise bounds, which count every rounding at its worst and
# would let a loss of half the bits pass.
#
# q4: a matrix product drops what lies below the last place of its sum, up to a step of 2^-23 (products of 2^-26 beside one
# of 1 lose 7/8 of it together), rms 0.58 · 2 · 2^-24 of a sum that grows to its full size as a random walk does: n products
# make 1.15 · sqrt(n / 2) · 2^-24 of the result. A group of 128 takes three pieces by four products, 12 (2.8), of x · code;
# codes have an rms of 8.8, code − zero one of 6.5 (any zero point) or 4.6 (all 8), so that this is up to 1.9 times as much
# of the result (5.4). x · zero the same by 1.7 (4.8), but it is one sum for all outputs of a row: twice that may come for a
# single row (9.6). Then 33 groups' sums in a wave at most (2.4), the waves' 8 and the scales (1.5), to nearest:
# sqrt(5.4² + 9.6² + 2.4² + 1.5²) = 11.4, against 16 allowed.
Q4_NORM = 16 * FP32
# Attention at scores of about 1: a score of 64 or 128 products, 5; its exponent less the reference and the exponential, 3;
# a weighted sum of up to 1100 keys, two or four at a time, 0.58 · sqrt(550 / 2) = 9.6, or less where waves share them; the
# sum of weights and the quotient 1: sqrt(5² + 3² + 9.6² + 1) = 11.3, against 16 allowed.
ATTENTION_NORM = 16 * FP32


def norm_off(got, want):
    return float(np.sqrt(((got - want) ** 2).sum() / (want ** 2).sum()))


def pieces(x, n):
    """The first n of the bf16 pieces (upper 16 bits of what is left) that an fp32 value is cut into, summed."""
    left, out = np.asarray(x, np.float32).copy(), np.zeros(np.shape(x))
    for _ in range(n):
        p = (left.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out += p
        left -= p
    return out


def short(x, bits):
    """fp32 values with `bits` significant bits, the rest cut off."""
    return (np.asarray(x, np.float32).view(np.uint32) & np.uint32(0xFFFFFFFF << (24 - bits) & 0xFFFFFFFF)).view(np.float32)
