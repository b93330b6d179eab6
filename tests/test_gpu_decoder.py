"""A decoder layer's step on the GPU against plain 64-bit forms: 4-bit linears, head norms with rotation, windowed and paged
attention, alone and together. Bounds are counted in tests/_decoder.py."""
import numpy as np
import pytest

import _decoder as D
import p2gemm as P

pytestmark = pytest.mark.gpu

EVERY = P.EVERY_KEY


def rng_of(*key):
    return np.random.default_rng([sum(str(k).encode()) for k in key])


# ── 4-bit weights ───────────────────────────────────────────────────────────────────────────────────────────────

Q4 = [(1, 1, 1, 32, False), (1, 31, 17, 32, True), (2, 33, 16, 64, True), (3, 128, 16, 128, False),
      (16, 130, 33, 64, True), (17, 1000, 48, 32, True), (5, 4096, 250, 128, False), (1, 1024, 1024, 128, False),
      (33, 257, 100, 128, True), (4, 2049, 31, 32, False)]


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M,K,N,group,zeros", Q4)
def test_q4(t, M, K, N, group, zeros):
    rng = rng_of(t, M, K, N, group)
    x, wt = D.rows(rng, t, M, K), D.q4_weight(rng, K, N, group, zeros)
    got = D.to_f64(t, D.run_q4(t, x, wt, K, N, group))
    w, x64 = D.q4_values(*wt, K, N, group), D.to_f64(t, x)
    D.check(got, x64 @ w, D.q4_bound(t, x64, w, x64 @ w, 1.0, K), f"{t} {M}x{K}x{N}")


@pytest.mark.parametrize("t", D.TYPES)
def test_q4_pitches_alpha_beta(t):
    M, K, N, group = 6, 300, 37, 64
    rng = rng_of(t, "pitch")
    x, wt, y0 = D.rows(rng, t, M, K), D.q4_weight(rng, K, N, group, True), D.rows(rng, t, M, N + 5)
    got = D.to_f64(t, D.run_q4(t, x, wt, K, N, group, 0.75, -1.5, y0, K + 3, N + 5))
    w, x64, old = D.q4_values(*wt, K, N, group), D.to_f64(t, x), D.to_f64(t, y0)
    want = 0.75 * (x64 @ w) - 1.5 * old[:, :N]
    D.check(got[:, :N], want, D.q4_bound(t, x64, w, want, 0.75, K) + 4 * D.FP32 * np.abs(old[:, :N]), t)
    assert np.array_equal(got[:, N:], old[:, N:])


@pytest.mark.parametrize("t", D.TYPES)
def test_q4_rows_do_not_depend_on_their_number(t):
    K, N, group = 1500, 80, 32
    rng = rng_of(t, "rows")
    x, wt = D.rows(rng, t, 19, K), D.q4_weight(rng, K, N, group, True)
    many = D.run_q4(t, x, wt, K, N, group)
    for m in (0, 3, 16, 18):
        assert np.array_equal(D.run_q4(t, x[m:m + 1], wt, K, N, group)[0], many[m])


@pytest.mark.parametrize("t", D.TYPES)
def test_q4_every_code_and_zero(t):
    """One row picked by a unit vector gives w itself: (code − zero)·scale, rounded once."""
    K, N, group = 256, 16, 32
    codes = np.tile(np.arange(256, dtype=np.uint8)[:, None], (1, 8))
    zeros = np.tile(np.array([[0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE]], np.uint8), (8, 1))
    scales = np.full((8, N), 2.0 ** -3, np.float16)
    x = D.to_type(t, np.eye(256)[:, :K])
    got = D.to_f64(t, D.run_q4(t, x, (codes, scales, zeros), K, N, group))
    assert np.array_equal(got, D.q4_values(codes, scales, zeros, K, N, group))


@pytest.mark.parametrize("t", D.TYPES)
def test_q4_wide_range_and_non_finite(t):
    K, N, group = 200, 32, 64
    rng = rng_of(t, "inf")
    big = 6e4 if t == "f16" else 1e30
    wt = D.q4_weight(rng, K, N, group, False)
    w = D.q4_values(*wt, K, N, group)
    x = rng.standard_normal((5, K))
    x[0, 3] = np.inf
    x[1, 5] = np.nan
    x[2] = 0.0
    x[3, ::7] *= big / 100
    x[4, 11] = -np.inf
    xt = D.to_type(t, x)
    got = D.to_f64(t, D.run_q4(t, xt, wt, K, N, group))
    with np.errstate(invalid="ignore"):
        want = D.to_f64(t, xt) @ w
    assert np.isnan(got[1]).all() and (got[2] == 0).all()
    for r in (0, 4):   # ±inf by the sign of its weight, NaN where that is 0
        assert np.array_equal(np.isnan(got[r]), np.isnan(want[r]))
        ok = ~np.isnan(want[r])
        assert np.array_equal(got[r][ok], want[r][ok])
    with np.errstate(over="ignore"):
        lim = D.to_f64(t, D.to_type(t, want[3]))
    fin = np.isfinite(lim)
    x3 = D.to_f64(t, xt[3:4])
    D.check(got[3:4, fin], want[3:4, fin], D.q4_bound(t, x3, w, want[3:4], 1.0, K)[:, fin], t)


# wide, wider, long and narrow: the forms with one to four column tiles a wave and with 4, 8 and 16 waves
Q4_FORMS = [(1, 300, 8201, 32, True), (5, 300, 8201, 64, False), (1, 200, 16325, 128, True), (18, 200, 16325, 32, False),
            (1, 4000, 40, 64, True), (3, 4097, 1030, 128, False), (16, 8200, 24, 32, True),
            (2, 400, 5000, 64, True), (1, 600, 16500, 32, False), (9, 1100, 16500, 128, True), (17, 200, 32773, 128, True)]


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("M,K,N,group,zeros", Q4_FORMS)
def test_q4_forms(t, M, K, N, group, zeros):
    rng = rng_of(t, M, K, N, group, "forms")
    x, wt = D.rows(rng, t, M, K), D.q4_weight(rng, K, N, group, zeros)
    w, x64 = D.q4_values(*wt, K, N, group), D.to_f64(t, x)
    for ldx in (K, K + 1):   # the second: rows of no alignment
        got = D.to_f64(t, D.run_q4(t, x, wt, K, N, group, ldx=ldx))
        D.check(got, x64 @ w, D.q4_bound(t, x64, w, x64 @ w, 1.0, K), f"{t} {M}x{K}x{N} pitch {ldx}")


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("K,N", ((4200, 48), (300, 8201), (200, 16325), (700, 31), (8500, 20), (1300, 16500)))
def test_q4_rows_do_not_depend_on_each_other(t, K, N):
    """A row alone, among others and beside rows with infinities and NaN: the same bits."""
    rng = rng_of(t, K, N, "apart")
    x, wt = D.rows(rng, t, 18, K), D.q4_weight(rng, K, N, 64, True)
    many = D.run_q4(t, x, wt, K, N, 64)
    odd = x.copy()
    odd[2, K // 2] = D.to_type(t, [np.inf])[0]
    odd[9, K - 1] = D.to_type(t, [np.nan])[0]
    beside = D.run_q4(t, odd, wt, K, N, 64)
    for m in (0, 3, 15, 17):
        assert np.array_equal(D.run_q4(t, x[m:m + 1], wt, K, N, 64)[0], many[m]), m
    for m in set(range(18)) - {2, 9}:
        assert np.array_equal(beside[m], many[m]), m


@pytest.mark.parametrize("M", (1, 5))
@pytest.mark.parametrize("scale", (2.0 ** -100, 2.0 ** -115, 2.0 ** -125))
def test_q4_tiny_fp32_rows(M, scale):
    """Three bf16 pieces hold a value down to 2^-133: less than that is lost of each, times its code and its zero point."""
    K, N, group = 300, 40, 64
    rng = rng_of("tiny", M)
    x, wt = D.rows(rng, "f32", M, K, scale=scale), D.q4_weight(rng, K, N, group, True)
    w, x64 = D.q4_values(*wt, K, N, group), D.to_f64("f32", x)
    lost = 2.0 ** -133 * 30 * np.repeat(wt[1].astype(np.float64), group, 0)[:K].sum(0)
    got = D.run_q4("f32", x, wt, K, N, group).astype(np.float64)
    D.check(got, x64 @ w, D.q4_bound("f32", x64, w, x64 @ w, 1.0, K) + lost, str(scale))


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("K", (1019, 4100, 130))
def test_q4_one_row_has_no_pitch(t, K):
    """Whatever pitch a single row is given with: the same bits."""
    rng = rng_of(t, K, "one row")
    x, wt = D.rows(rng, t, 1, K), D.q4_weight(rng, K, 70, 64, True)
    want = D.run_q4(t, x, wt, K, 70, 64, ldx=-(-K // 8) * 8)
    for ldx in (K, K + 1, 1 << 25):
        assert np.array_equal(D.run_q4(t, x, wt, K, 70, 64, ldx=ldx), want), ldx


def test_q4_rows_far_apart():
    M, K, N, group = 2, 300, 40, 64
    rng = rng_of("far apart")
    x, wt = D.rows(rng, "f16", M, K), D.q4_weight(rng, K, N, group, True)
    assert np.array_equal(D.run_q4("f16", x, wt, K, N, group, ldx=1 << 25), D.run_q4("f16", x, wt, K, N, group))


@pytest.mark.parametrize("t", D.TYPES)
def test_q4_codes_at_their_zero_point(t):
    """Weights of 0: bf16 and fp32 rows sum code and zero point apart, each off by what q4_bound counts of its own size."""
    K, N, group = 700, 32, 128
    rng = rng_of(t, "zero point")
    codes, scales, _ = D.q4_weight(rng, K, N, group, False)
    x = D.rows(rng, t, 4, K)
    zeros = np.full((6, N // 2), 0x33, np.uint8)
    got = D.to_f64(t, D.run_q4(t, x, (np.full_like(codes, 0x33), scales, zeros), K, N, group))
    both = 2 * 3 * np.repeat(scales.astype(np.float64), group, 0)[:K]
    D.check(got, np.zeros((4, N)), D.q4_bound(t, D.to_f64(t, x), both, np.zeros((4, N)), 1.0, K) + D.HALF[t] * np.abs(got), t)


def test_q4_scales_as_bits():
    """fp16 scales given as uint16 are their bits, as in the C header, not numbers."""
    K, N, group = 100, 24, 32
    rng = rng_of("bits")
    codes, scales, zeros = D.q4_weight(rng, K, N, group, True)
    x = D.rows(rng, "f32", 2, K)
    want = D.run_q4("f32", x, (codes, scales, zeros), K, N, group)
    assert np.array_equal(D.run_q4("f32", x, (codes, scales.view(np.uint16), zeros), K, N, group), want)


def test_q4_bytes_and_wrap():
    K, N, group = 1024, 256, 128
    rng = rng_of("wrap")
    wt = D.q4_weight(rng, K, N, group, True)
    d = [D.device(a) for a in wt]
    w = P.Q4Weight.wrap(d[0].ptr, d[1].ptr, d[2].ptr, K, N, group)
    assert w.device_bytes() == K * N // 2 + 4 * (K // group) * N
    for b in d:
        b.upload(np.zeros(b.nbytes, np.uint8))   # the codes are not read after the call
    x = D.rows(rng, "f32", 2, K)
    dx, dy = D.device(x), D.preset("f32", (2, N))
    P.q4_gemv_dev("f32", 2, N, K, 1.0, dx.ptr, K, w, 0.0, dy.ptr, N)
    assert np.array_equal(dy.download((2, N), np.float32), D.run_q4("f32", x, wt, K, N, group))


# ── norm, rotation and the cache ────────────────────────────────────────────────────────────────────────────────

def run_rope(t, qkv, H, Hk, Dh, gq, gk, eps, rot, inter, freq, pos, page=0, pages=0, slots=None, keys=True, pad=0,
             in_place=False, stream=None):
    T, W = qkv.shape
    dx, dgq, dgk = D.device(qkv), D.device(gq), D.device(gk)
    df, dp = D.device(np.asarray(freq, np.float32)), D.device(np.asarray(pos, np.int32))
    ldq, ldk = (W, W) if in_place else (H * Dh + pad, Hk * Dh + pad)
    dq = dx if in_place else D.preset(t, (max(T, 1), ldq))
    dk = (dx if in_place else D.preset(t, (max(T, 1), ldk))) if keys else None
    cache, ds, kc, vc = None, None, None, None
    if pages:
        fill = np.full((pages, Hk, page, Dh), 3.0)
        kc, vc = D.device(D.to_type(t, fill)), D.device(D.to_type(t, -fill))
        cache = P.KvCache(t, Hk, Dh, page, pages, kc.ptr, vc.ptr)
        ds = D.device(np.asarray(slots, np.int32))
    P.qk_norm_rope_dev(t, T, H, Hk, Dh, dx.ptr, W, dgq.ptr, dgk.ptr, eps, rot, inter, df.ptr, dp.ptr, dq.ptr, ldq,
                       None if dk is None else dk.ptr + (H * Dh * D.size(t) if in_place else 0), ldk, cache,
                       ds.ptr if ds else None, stream)
    out = [dq.download((T, ldq), D.np_type(t), stream)]
    out.append(dk.download((T, ldk), D.np_type(t), stream) if keys and not in_place else None)
    if pages:
        out += [b.download((pages, Hk, page, Dh), D.np_type(t), stream) for b in (kc, vc)]
    return out


ROPE = [(1, 1, 1, 64, 64, False), (3, 4, 2, 128, 128, True), (5, 8, 8, 128, 64, False), (2, 6, 3, 64, 16, True),
        (7, 32, 8, 128, 128, False), (4, 5, 1, 128, 0, False), (130, 3, 1, 64, 48, False), (2, 40, 8, 64, 32, False)]


def rope_inputs(t, T, H, Hk, Dh, rot, key, far=100000):
    rng = rng_of(t, T, H, Dh, rot, key)
    qkv = D.rows(rng, t, T, (H + 2 * Hk) * Dh, scale=3.0)
    gq, gk = (rng.uniform(-1.5, 1.5, Dh).astype(np.float32) for _ in range(2))
    freq = (10000.0 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 1))).astype(np.float32)
    return rng, qkv, gq, gk, freq, rng.integers(0, far, T).astype(np.int32)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("T,H,Hk,Dh,rot,inter", ROPE)
def test_rope(t, T, H, Hk, Dh, rot, inter):
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "plain")
    q, k = run_rope(t, qkv, H, Hk, Dh, gq, gk, 1e-6, rot, inter, freq, pos, pad=16)
    x = D.to_f64(t, qkv).reshape(T, H + 2 * Hk, Dh)
    for got, part, g, n in ((q, x[:, :H], gq, H), (k, x[:, H:H + Hk], gk, Hk)):
        want, size_of = D.norm_rope(part, g, 1e-6, rot, inter, freq, pos)
        D.check(D.to_f64(t, got[:, :n * Dh]).reshape(T, n, Dh), want, D.rope_bound(t, want, size_of, Dh), t)
        assert (got[:, n * Dh:].view(np.uint16) == 0xFFFF).all()   # the pitch's pad is left as it was
    inq = run_rope(t, qkv, H, Hk, Dh, gq, gk, 1e-6, rot, inter, freq, pos, in_place=True)[0]
    assert np.array_equal(inq[:, :H * Dh], q[:, :H * Dh])
    assert np.array_equal(inq[:, H * Dh:(H + Hk) * Dh], k[:, :Hk * Dh])
    assert np.array_equal(inq[:, (H + Hk) * Dh:], qkv[:, (H + Hk) * Dh:])


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("page", (16, 64))
def test_rope_into_the_cache(t, page):
    T, H, Hk, Dh, rot, pages = 21, 6, 3, 128, 128, 5
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, page)
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    slots[4], slots[9], slots[13] = -1, pages * page, 2 ** 31 - 1   # rows that stay out of it
    q, k, kc, vc = run_rope(t, qkv, H, Hk, Dh, gq, gk, 0.0, rot, False, freq, pos, page, pages, slots)
    q2, _, kc2, _ = run_rope(t, qkv, H, Hk, Dh, gq, gk, 0.0, rot, False, freq, pos, page, pages, slots, keys=False)
    assert np.array_equal(q, q2) and np.array_equal(kc, kc2)
    want_k, want_v = D.to_type(t, np.full(kc.shape, 3.0)), D.to_type(t, np.full(kc.shape, -3.0))
    v = qkv[:, (H + Hk) * Dh:].reshape(T, Hk, Dh)
    for i in range(T):
        if 0 <= slots[i] < pages * page:
            want_k[slots[i] // page, :, slots[i] % page] = k[i].reshape(Hk, Dh)
            want_v[slots[i] // page, :, slots[i] % page] = v[i]
    assert np.array_equal(kc, want_k) and np.array_equal(vc, want_v)
    plain = run_rope(t, qkv, H, Hk, Dh, gq, gk, 0.0, rot, False, freq, pos)
    assert np.array_equal(plain[0], q) and np.array_equal(plain[1], k)


@pytest.mark.parametrize("t", D.TYPES)
def test_rope_many_rows_as_few(t):
    """More rows than the form with 1024 threads takes, with a cache: the bits of the same rows in small calls."""
    T, H, Hk, Dh, rot, page = 300, 6, 2, 64, 32, 32
    rng, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "many")
    slots = rng.permutation(10 * page)[:T].astype(np.int32)
    q, k, kc, vc = run_rope(t, qkv, H, Hk, Dh, gq, gk, 1e-5, rot, True, freq, pos, page, 10, slots)
    for a in range(0, T, 100):
        b = a + 100
        r = run_rope(t, qkv[a:b], H, Hk, Dh, gq, gk, 1e-5, rot, True, freq, pos[a:b], page, 10, slots[a:b])
        assert np.array_equal(q[a:b], r[0]) and np.array_equal(k[a:b], r[1])
        at = (slots[a:b] // page, slice(None), slots[a:b] % page)
        assert np.array_equal(kc[at], r[2][at]) and np.array_equal(vc[at], r[3][at])
    x = D.to_f64(t, qkv).reshape(T, H + 2 * Hk, Dh)
    want, size_of = D.norm_rope(x[:, :H], gq, 1e-5, rot, True, freq, pos)
    D.check(D.to_f64(t, q).reshape(T, H, Dh), want, D.rope_bound(t, want, size_of, Dh), t)


@pytest.mark.parametrize("pos", (0, 1, 131071, 2 ** 31 - 1, -5))
def test_rope_far_positions(pos):
    """The angle is the product in 64 bits: 2^31 radians and more are reduced without loss."""
    T, H, Hk, Dh, rot = 2, 1, 1, 64, 64
    _, qkv, gq, gk, freq, _ = rope_inputs("f32", T, H, Hk, Dh, rot, "far")
    at = np.full(T, pos, np.int32)
    q, _ = run_rope("f32", qkv, H, Hk, Dh, gq, gk, 1e-5, rot, True, freq, at)
    want, size_of = D.norm_rope(D.to_f64("f32", qkv).reshape(T, 3, Dh)[:, :1], gq, 1e-5, rot, True, freq, at)
    # 2^31 radians in 64 bits: a product's rounding there is 2^-22, numpy's and the kernel's alike
    extra = abs(pos) * 2.0 ** -51 * size_of
    D.check(q.astype(np.float64).reshape(T, 1, Dh), want, D.rope_bound("f32", want, size_of, Dh) + extra, str(pos))


@pytest.mark.parametrize("t", ("f32", "bf16"))
@pytest.mark.parametrize("scale,eps", ((1e19, 1e-6), (3e20, 0.0), (1e37, 1e-6), (1e-16, 0.0), (1e-22, 0.0), (1e-37, 0.0),
                                       (1e-22, 1e-30), (1e-14, 1e-28), (1e-20, 1e-6)))
def test_rope_heads_of_any_size(t, scale, eps):
    """Squares may leave the range of 32 bits, the norm does not."""
    T, H, Hk, Dh, rot = 3, 4, 2, 128, 64
    _, qkv, gq, gk, freq, pos = rope_inputs(t, T, H, Hk, Dh, rot, "size")
    qkv = D.to_type(t, D.to_f64(t, qkv) / 3 * scale)
    qkv[1, :Dh] = D.to_type(t, D.to_f64(t, qkv[1, :Dh]) / scale)   # an ordinary head beside them
    q, k = run_rope(t, qkv, H, Hk, Dh, gq, gk, eps, rot, False, freq, pos)
    x = D.to_f64(t, qkv).reshape(T, H + 2 * Hk, Dh)
    eps = float(np.float32(eps))
    for got, part, g, n in ((q, x[:, :H], gq, H), (k, x[:, H:H + Hk], gk, Hk)):
        want, size_of = D.norm_rope(part, g, eps, rot, False, freq, pos)
        D.check(D.to_f64(t, got).reshape(T, n, Dh), want, D.rope_bound(t, want, size_of, Dh), f"{t} {scale} {eps}")


@pytest.mark.parametrize("t", D.TYPES)
def test_rope_one_row_in_place(t):
    """A single row has no pitch: in place with the heads' width as pitch."""
    H, Hk, Dh = 4, 2, 64
    _, qkv, gq, gk, freq, pos = rope_inputs(t, 1, H, Hk, Dh, Dh, "one")
    q, k = run_rope(t, qkv, H, Hk, Dh, gq, gk, 1e-6, Dh, False, freq, pos)
    dx, dgq, dgk, df, dp = (D.device(a) for a in (qkv, gq, gk, freq, pos))
    P.qk_norm_rope_dev(t, 1, H, Hk, Dh, dx.ptr, qkv.shape[1], dgq.ptr, dgk.ptr, 1e-6, Dh, False, df.ptr, dp.ptr, dx.ptr, H * Dh,
                       dx.ptr + H * Dh * D.size(t), Hk * Dh)
    got = dx.download(qkv.shape, D.np_type(t))
    assert np.array_equal(got, np.concatenate((q, k, qkv[:, (H + Hk) * Dh:]), 1))


def test_rope_zero_row_and_empty_call():
    T, H, Hk, Dh = 2, 2, 1, 64
    _, qkv, gq, gk, freq, pos = rope_inputs("bf16", T, H, Hk, Dh, 64, "zero")
    qkv[:] = 0
    q, k = run_rope("bf16", qkv, H, Hk, Dh, gq, gk, 1e-6, 64, False, freq, pos)
    assert not (q & 0x7FFF).any() and not (k & 0x7FFF).any()
    run_rope("bf16", qkv[:0], H, Hk, Dh, gq, gk, 1e-6, 64, False, freq, pos[:0])


# ── windowed attention ──────────────────────────────────────────────────────────────────────────────────────────

WIN = [  # query lengths, keys more than queries, heads, key heads, window, ahead, sinks
    ((1,), 0, 1, 1, 1, 0, 0), ((5,), 0, 2, 1, EVERY, 0, 0), ((33,), 7, 3, 3, 4, 0, 2), ((64,), 0, 4, 2, 16, 5, 1),
    ((130,), 0, 2, 2, EVERY, EVERY, 0), ((129,), 300, 4, 1, 100, 0, 33), ((0, 3, 0, 40, 1), 12, 2, 1, 20, 3, 4),
    ((17,), -9, 2, 1, 6, 0, 3), ((300, 2, 77), 0, 8, 2, 64, 0, 70), ((50,), -50, 1, 1, 8, 2, 2),
    ((1,) * 70, 5, 1, 1, EVERY, 0, 0)]


def window_case(t, lens, past, H, Hk, Dh, key="w", scale=1.0):
    rng = rng_of(t, lens, past, H, Dh, key)
    kl = [max(n + past, 0) if n else 0 for n in lens]
    nq, nk = sum(lens), sum(kl)
    q, k, v = (D.rows(rng, t, n, h * Dh, scale=scale) for n, h in ((nq, H), (nk, Hk), (nk, Hk)))
    return q, k, v, np.concatenate(([0], np.cumsum(lens))), np.concatenate(([0], np.cumsum(kl)))


def window_want(t, q, k, v, qs, ks, H, Hk, Dh, scale, window, ahead, sinks):
    want, bound = np.zeros((q.shape[0], H * Dh)), np.zeros((q.shape[0], H * Dh))
    for s in range(len(qs) - 1):
        a, b, c, d = qs[s], qs[s + 1], ks[s], ks[s + 1]
        o, e = D.attention(t, D.to_f64(t, q[a:b]).reshape(b - a, H, Dh), D.to_f64(t, k[c:d]).reshape(d - c, Hk, Dh),
                           D.to_f64(t, v[c:d]).reshape(d - c, Hk, Dh), D.visible(b - a, d - c, window, ahead, sinks), scale)
        want[a:b], bound[a:b] = o.reshape(b - a, H * Dh), e.reshape(b - a, H * Dh)
    return want, bound


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,past,H,Hk,window,ahead,sinks", WIN)
def test_window(t, Dh, lens, past, H, Hk, window, ahead, sinks):
    q, k, v, qs, ks = window_case(t, lens, past, H, Hk, Dh)
    scale = Dh ** -0.5
    got = D.run_window(t, q, k, v, H, Hk, Dh, scale, window, ahead, sinks, qs, ks)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, scale, window, ahead, sinks)
    D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens}")
    if len(lens) == 1:
        alone = D.run_window(t, q, k, v, H, Hk, Dh, scale, window, ahead, sinks)
        assert np.array_equal(alone, got)


@pytest.mark.parametrize("t", D.TYPES)
def test_window_many_rows(t):
    """Enough tiles for the form with 128 queries a workgroup, ragged, with pitches wider than the heads."""
    H, Hk, Dh, lens, window, ahead, sinks = 32, 4, 64, (700, 1, 333), 150, 0, 5
    q, k, v, qs, ks = window_case(t, lens, 40, H, Hk, Dh)
    pad = 16
    wide = [np.concatenate((a, np.full((a.shape[0], pad), np.nan if t != "bf16" else 0x7FC0, a.dtype)), 1) for a in (q, k, v)]
    got = D.run_window(t, *wide, H, Hk, Dh, 0.2, window, ahead, sinks, qs, ks, pad)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, 0.2, window, ahead, sinks)
    D.check(D.to_f64(t, got[:, :H * Dh]), want, bound, t)
    assert (got[:, H * Dh:].view(np.uint16) == 0xFFFF).all()


BIG = [  # rows for the form with 128 of them a workgroup, of 1, 2 and 4 query heads
    ((513,), 0, 32, 32, 300, 7, 0), ((450, 0, 70), 25, 32, 16, 200, 0, 40), ((600,), -37, 32, 8, 256, 64, 3),
    ((520, 3), 130, 32, 4, EVERY, 0, 0), ((1100,), 0, 32, 8, EVERY, EVERY, 0), ((65, 513), 0, 36, 6, 1, 0, 1),
    ((700, 5, 400), 9, 32, 8, 300, 0, 2)]


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,past,H,Hk,window,ahead,sinks", BIG)
def test_window_forms(t, Dh, lens, past, H, Hk, window, ahead, sinks):
    q, k, v, qs, ks = window_case(t, lens, past, H, Hk, Dh, "big")
    got = D.run_window(t, q, k, v, H, Hk, Dh, Dh ** -0.5, window, ahead, sinks, qs, ks)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, Dh ** -0.5, window, ahead, sinks)
    D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens}")


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh", (64, 128))
def test_window_forms_large_scores(t, Dh):
    """Scores in the hundreds over many blocks: the reference is raised again and again."""
    H, Hk = 32, 8
    q, k, v, qs, ks = window_case(t, (530,), 60, H, Hk, Dh, "raise", scale=6.0)
    k[::50] = D.to_type(t, 0.25 * D.to_f64(t, k[::50]))
    got = D.run_window(t, q, k, v, H, Hk, Dh, 1.0, 400, 0, 3, qs, ks)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, 1.0, 400, 0, 3)
    D.check(D.to_f64(t, got), want, bound, t)


@pytest.mark.parametrize("t", D.TYPES)
def test_window_forms_ignore_what_they_mask(t):
    H, Hk, Dh, n, window = 32, 16, 128, 600, 64
    q, k, v, qs, ks = window_case(t, (n,), 0, H, Hk, Dh, "hide")
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, 0.09, window, 0, 0)
    for what in (np.inf, -np.inf, np.nan):
        k2, v2 = k.copy(), v.copy()
        k2[200] = v2[200] = D.to_type(t, np.full(Hk * Dh, what))
        f = D.to_f64(t, D.run_window(t, q, k2, v2, H, Hk, Dh, 0.09, window, 0, 0, qs, ks))
        sees = (np.arange(n) >= 200) & (np.arange(n) < 200 + window)
        D.check(f[~sees], want[~sees], bound[~sees], f"{t} {what}")
        if what != what:
            assert np.isnan(f[sees]).all()


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("lens,H", (((90,), 2), ((1200,), 32)))
def test_window_ignores_what_it_masks(t, lens, H):
    """Infinities and NaN in keys and values that a query must not see do not reach it; those it sees do."""
    Hk, Dh, window, sinks = 1, 64, 10, 2
    q, k, v, qs, ks = window_case(t, lens, 0, H, Hk, Dh, "mask")
    clean = D.run_window(t, q, k, v, H, Hk, Dh, 0.125, window, 0, sinks, qs, ks)
    at = 40
    k2, v2 = k.copy(), v.copy()
    v2[at, :] = D.to_type(t, np.full(Dh, np.inf))
    v2[at + 1, ::2] = D.to_type(t, np.full(Dh // 2, np.nan))
    got = D.run_window(t, q, k2, v2, H, Hk, Dh, 0.125, window, 0, sinks, qs, ks)
    sees = np.arange(lens[0])[(np.arange(lens[0]) >= at) & (np.arange(lens[0]) < at + 1 + window)]
    out = np.setdiff1d(np.arange(lens[0]), sees)
    f = D.to_f64(t, got)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, 0.125, window, 0, sinks)
    D.check(f[out], want[out], bound[out], t)
    assert not np.isfinite(f[sees]).all(1).any()
    k2[at] = D.to_type(t, np.full(Dh, np.nan))
    got = D.to_f64(t, D.run_window(t, q, k2, v, H, Hk, Dh, 0.125, window, 0, sinks, qs, ks))
    seesk = np.arange(at, at + window)
    assert np.isnan(got[seesk]).all()
    rest = np.setdiff1d(np.arange(lens[0]), seesk)
    D.check(got[rest], D.to_f64(t, clean)[rest], 2 * bound[rest], t)


@pytest.mark.parametrize("t", D.TYPES)
def test_window_large_scores(t):
    """Scores in the hundreds: the running maximum keeps every exponential in range."""
    H, Hk, Dh = 2, 1, 64
    q, k, v, qs, ks = window_case(t, (70,), 30, H, Hk, Dh, "large", scale=8.0)
    got = D.run_window(t, q, k, v, H, Hk, Dh, 1.0, EVERY, 0, 0)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, 1.0, EVERY, 0, 0)
    D.check(D.to_f64(t, got), want, bound, t)


@pytest.mark.parametrize("t,H", (("f32", 1), ("f16", 1), ("bf16", 16)))
@pytest.mark.parametrize("n", (64, 65, 200, 4200))
def test_window_many_sequences(t, H, n):
    """More sequences than are looked up at once, empty ones among them, in both forms."""
    Dh = 64
    rng = rng_of(t, n, "many sequences")
    lens = rng.integers(0, 6 if n > 1000 else 30, n)
    qs = np.concatenate(([0], np.cumsum(lens)))
    q, k, v = (D.rows(rng, t, int(qs[-1]), H * Dh) for _ in range(3))
    got = D.run_window(t, q, k, v, H, H, Dh, 0.125, EVERY, 0, 0, qs, qs)
    want, bound = window_want(t, q, k, v, qs, qs, H, H, Dh, 0.125, EVERY, 0, 0)
    D.check(D.to_f64(t, got), want, bound, f"{t} {n}")


def test_window_leaves_rows_outside_the_sequences():
    H, Hk, Dh = 2, 2, 64
    q, k, v, _, _ = window_case("f32", (40,), 0, H, Hk, Dh, "rest")
    o0 = np.full((40, H * Dh), 7.5, np.float32)
    got = D.run_window("f32", q, k, v, H, Hk, Dh, 0.1, EVERY, 0, 0, [3, 10, 10, 21], [0, 7, 9, 30], o0=o0)
    assert (got[:3] == 7.5).all() and (got[21:] == 7.5).all() and (got[3:21] != 7.5).any(1).all()
    # starts outside the rows or descending are held to the rows: nothing outside is touched
    D.run_window("f32", q, k, v, H, Hk, Dh, 0.1, EVERY, 0, 0, [-5, 90, 12, 2 ** 31 - 1], [8, -3, 2 ** 31 - 1, 4], o0=o0)


# ── paged attention ─────────────────────────────────────────────────────────────────────────────────────────────

PAGED = [  # lengths, heads, key heads, page, window, sinks
    ((1,), 1, 1, 16, EVERY, 0), ((0, 5, 16, 17), 4, 2, 16, EVERY, 0), ((33, 100), 8, 8, 64, 20, 3),
    ((1000, 3, 257), 6, 1, 32, 64, 40), ((2500,), 8, 2, 256, EVERY, 0), ((700, 650), 40, 2, 16, 500, 16),
    ((3000, 1, 0, 1024), 2, 1, 1024, 1, 1), ((90,), 3, 3, 16, 32, 200)]


def paged_case(t, lens, H, Hk, page, Dh, key="p", spare=3):
    rng = rng_of(t, lens, H, page, Dh, key)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    order = rng.permutation(pages)
    ld = max(max(per), 1) + 1
    table = np.full((len(lens), ld), -7, np.int32)   # entries past a sequence's pages are not pages
    at = 0
    for s, n in enumerate(per):
        table[s, :n] = order[at:at + n]
        at += n
    q = D.rows(rng, t, len(lens), H * Dh)
    kc, vc = (D.rows(rng, t, pages, Hk, page, Dh) for _ in range(2))
    nan = np.uint16(0x7FC0) if t == "bf16" else np.nan
    for s, n in enumerate(lens):   # what no token was written to holds anything
        for p in range(n, per[s] * page):
            kc[table[s, p // page], :, p % page] = nan
            vc[table[s, p // page], :, p % page] = nan
    return q, kc, vc, table


def paged_want(t, q, kc, vc, table, lens, H, scale, window, sinks):
    pages, Hk, page, Dh = kc.shape
    want, bound = np.zeros((len(lens), H * Dh)), np.zeros((len(lens), H * Dh))
    for s, n in enumerate(lens):
        k, held = D.gather(t, kc, table[s], n, page, pages)
        v, _ = D.gather(t, vc, table[s], n, page, pages)
        seen = D.visible(1, n, window, 0, sinks) & held[None, :]
        o, e = D.attention(t, D.to_f64(t, q[s]).reshape(1, H, Dh), k, v, seen, scale)
        want[s], bound[s] = o.reshape(-1), e.reshape(-1)
    return want, bound


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,H,Hk,page,window,sinks", PAGED)
def test_paged(t, Dh, lens, H, Hk, page, window, sinks):
    q, kc, vc, table = paged_case(t, lens, H, Hk, page, Dh)
    want, bound = paged_want(t, q, kc, vc, table, lens, H, 0.1, window, sinks)
    for split in (False, True):
        got = D.run_paged(t, q, kc, vc, table, lens, H, 0.1, window, sinks, split)
        D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens} split {split}")
    # planned for other lengths than those that come
    for most in (1, 40000):
        got = D.run_paged(t, q, kc, vc, table, lens, H, 0.1, window, sinks, True, most)
        D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {lens} planned for {most}")


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_pages_that_are_not_there(t):
    lens, H, Hk, page, Dh = (200, 64, 130), 4, 1, 16, 64
    q, kc, vc, table = paged_case(t, lens, H, Hk, page, Dh, "holes")
    table[0, 2], table[0, 11], table[1, :] = -1, kc.shape[0], 2 ** 31 - 1
    want, bound = paged_want(t, q, kc, vc, table, lens, H, 0.1, EVERY, 0)
    got = D.to_f64(t, D.run_paged(t, q, kc, vc, table, lens, H, 0.1, EVERY, 0))
    D.check(got, want, bound, t)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_lengths_outside_the_table(t):
    lens, H, Hk, page, Dh = (48, 20), 2, 1, 16, 64
    q, kc, vc, table = paged_case(t, lens, H, Hk, page, Dh, "long")
    table = np.ascontiguousarray(table[:, :3])
    table[1] = table[0]
    got = D.run_paged(t, q, kc, vc, table, (1 << 30, -4), H, 0.1, EVERY, 0, True, 100)
    want = D.run_paged(t, q, kc, vc, table, (48, 0), H, 0.1, EVERY, 0, True, 100)
    assert np.array_equal(got, want)


def test_paged_equals_window():
    """One new token over pages and the last query of a sequence in rows are the same attention."""
    H, Hk, Dh, page, n, t = 4, 2, 128, 16, 333, "f32"
    q, kc, vc, table = paged_case(t, (n,), H, Hk, page, Dh, "same")
    k, v = (np.ascontiguousarray(D.gather(t, c, table[0], n, page, kc.shape[0])[0].reshape(n, -1).astype(np.float32))
            for c in (kc, vc))
    a = D.run_paged(t, q, kc, vc, table, (n,), H, 0.1, 100, 4)
    b = D.run_window(t, q, k, v, H, Hk, Dh, 0.1, 100, 0, 4)
    _, bound = paged_want(t, q, kc, vc, table, (n,), H, 0.1, 100, 4)
    assert (np.abs(a.astype(np.float64) - b) <= 2 * bound).all()


# ── offsets beyond 32 bits ──────────────────────────────────────────────────────────────────────────────────────

def test_cache_beyond_32_bits():
    """A cache of more than 2^32 elements whose last pages are used: written by the rotation, read by the attention."""
    t, H, Hk, Dh, page, pages, n = "bf16", 8, 8, 128, 1024, 4110, 1500
    dk, dv = (P.DeviceBuffer(pages * Hk * page * Dh * 2) for _ in range(2))
    assert pages * Hk * page * Dh > 1 << 32
    small_k, small_v = (P.DeviceBuffer(2 * Hk * page * Dh * 2) for _ in range(2))
    big, small = P.KvCache(t, Hk, Dh, page, pages, dk.ptr, dv.ptr), P.KvCache(t, Hk, Dh, page, 2, small_k.ptr, small_v.ptr)
    _, qkv, gq, gk, freq, pos = rope_inputs(t, n, H, Hk, Dh, Dh, "far pages")
    dx, dgq, dgk, df, dp = (D.device(a) for a in (qkv, gq, gk, freq, pos))
    dq, outs = D.preset(t, (n, H * Dh)), []
    for cache, order in ((big, (pages - 1, pages - 3)), (small, (1, 0))):
        at = np.arange(n)
        slots = (np.array(order)[at // page] * page + at % page).astype(np.int32)
        ds, dt, dl = D.device(slots), D.device(np.array([order], np.int32)), D.device(np.array([n], np.int32))
        do = D.preset(t, (1, H * Dh))
        P.qk_norm_rope_dev(t, n, H, Hk, Dh, dx.ptr, 3 * H * Dh, dgq.ptr, dgk.ptr, 1e-6, Dh, False, df.ptr, dp.ptr, dq.ptr,
                           H * Dh, None, 0, cache, ds.ptr)
        P.attention_paged_dev(cache, 1, H, dq.ptr, H * Dh, dt.ptr, 2, dl.ptr, n, 0.1, EVERY, 0, do.ptr, H * Dh)
        outs.append(do.download((1, H * Dh), np.uint16))
    assert np.isfinite(D.to_f64(t, outs[1])).all() and np.array_equal(*outs)


@pytest.mark.parametrize("t,H", (("f16", 1), ("f32", 1), ("f16", 64), ("f32", 64)))
def test_window_rows_beyond_32_bits(t, H):
    """Rows so far apart that the last ones lie past 2^31 elements (in both forms): the bits of rows side by side."""
    n, Dh, ld = 150, 64, (1 << 23) - 64
    ld = ld if H == 1 else 1 << 22
    n = n if H == 1 else 530
    q, k, v, _, _ = window_case(t, (n,), 0, H, H, Dh, "far rows")
    want = D.run_window(t, q, k, v, H, H, Dh, 0.125, 100, 0, 3)
    es, first = D.size(t), 400 if H == 1 else 0   # H 1: rows 400 .. of a larger buffer are the sequence
    bufs = [P.DeviceBuffer(((n + first - 1) * ld + H * Dh) * es) for _ in range(4)]
    assert (n + first - 1) * ld > 1 << 31
    for b, a in zip(bufs, (q, k, v)):
        for r in range(n):
            b.upload(a[r], offset=(r + first) * ld * es)
    starts = D.device(np.array([first, first + n], np.int32))
    P.attention_window_dev(t, n + first, n + first, 1, starts.ptr, starts.ptr, H, H, Dh, bufs[0].ptr, ld, bufs[1].ptr, ld,
                           bufs[2].ptr, ld, 0.125, 100, 0, 3, bufs[3].ptr, ld)
    got = np.stack([bufs[3].download((H * Dh,), D.np_type(t), offset=(r + first) * ld * es) for r in range(n)])
    assert np.array_equal(got, want)


# ── together, streams and graphs ────────────────────────────────────────────────────────────────────────────────

class Layer:
    """A decoder layer's attention step on the device: qkv by a 4-bit weight, norm and rotation into the cache, attention
    over it, the output projection onto the residual rows."""
    H, Hk, DH, C, PAGE, WINDOW, SINKS = 4, 2, 64, 256, 16, 40, 3

    def __init__(self, t, B, per, seed):
        rng = rng_of(t, B, seed)
        W = (self.H + 2 * self.Hk) * self.DH
        self.t, self.B, self.W = t, B, W
        self.wq, self.wo = D.q4_weight(rng, self.C, W, 64, True), D.q4_weight(rng, self.H * self.DH, self.C, 32, False)
        self.q4q, self.q4o = P.Q4Weight(*self.wq, self.C, W, 64), P.Q4Weight(*self.wo, self.H * self.DH, self.C, 32)
        self.gq, self.gk = (rng.uniform(0.5, 1.5, self.DH).astype(np.float32) for _ in range(2))
        self.freq = (100.0 ** (-np.arange(0, self.DH, 2) / self.DH)).astype(np.float32)
        self.pages = B * per
        self.table = rng.permutation(self.pages).reshape(B, per).astype(np.int32)
        z = D.to_type(t, np.full((self.pages, self.Hk, self.PAGE, self.DH), np.nan))
        self.dk, self.dv, self.dt = D.device(z), D.device(z), D.device(self.table)
        self.cache = P.KvCache(t, self.Hk, self.DH, self.PAGE, self.pages, self.dk.ptr, self.dv.ptr)
        self.dgq, self.dgk, self.df = D.device(self.gq), D.device(self.gk), D.device(self.freq)
        self.dx, self.dqkv = D.preset(t, (B, self.C)), D.preset(t, (B, W))
        self.dq, self.do = D.preset(t, (B, self.H * self.DH)), D.preset(t, (B, self.H * self.DH))
        self.dpos, self.dslot, self.dlen = (D.device(np.zeros(B, np.int32)) for _ in range(3))
        self.most = per * self.PAGE
        self.ws = P.Workspace(P.attention_paged_workspace_bytes(self.cache, B, self.H, self.most, self.WINDOW, self.SINKS))

    def place(self, x, at):
        """The step's inputs: rows x and every sequence's new token at place at[s]."""
        at = np.asarray(at, np.int32)
        self.dx.upload(x)
        self.dpos.upload(at)
        self.dslot.upload((self.table[np.arange(self.B), at // self.PAGE] * self.PAGE + at % self.PAGE).astype(np.int32))
        self.dlen.upload(at + 1)

    def step(self, stream=None):
        t, B, H, Hk, DH = self.t, self.B, self.H, self.Hk, self.DH
        P.q4_gemv_dev(t, B, self.W, self.C, 0.05, self.dx.ptr, self.C, self.q4q, 0.0, self.dqkv.ptr, self.W, stream)
        P.qk_norm_rope_dev(t, B, H, Hk, DH, self.dqkv.ptr, self.W, self.dgq.ptr, self.dgk.ptr, 1e-6, DH, False,
                           self.df.ptr, self.dpos.ptr, self.dq.ptr, H * DH, None, 0, self.cache, self.dslot.ptr, stream)
        P.attention_paged_dev(self.cache, B, H, self.dq.ptr, H * DH, self.dt.ptr, self.table.shape[1], self.dlen.ptr,
                              self.most, DH ** -0.5, self.WINDOW, self.SINKS, self.do.ptr, H * DH, self.ws.ptr,
                              self.ws.nbytes, stream)
        P.q4_gemv_dev(t, B, self.C, H * DH, 0.05, self.do.ptr, H * DH, self.q4o, 1.0, self.dx.ptr, self.C, stream)

    def out(self, stream=None):
        return self.dx.download((self.B, self.C), D.np_type(self.t), stream)

    def plain(self, xs):
        """xs [steps][B][C] in 64 bits, tokens 0, 1, …: the layer's outputs, nothing rounded in between."""
        wq = D.q4_values(*self.wq, self.C, self.W, 64) * 0.05
        wo = D.q4_values(*self.wo, self.H * self.DH, self.C, 32) * 0.05
        S, H, Hk, DH = xs.shape[0], self.H, self.Hk, self.DH
        out = np.zeros(xs.shape)
        for s in range(self.B):
            qkv = (xs[:, s] @ wq).reshape(S, H + 2 * Hk, DH)
            pos = np.arange(S)
            q, _ = D.norm_rope(qkv[:, :H], self.gq, 1e-6, DH, False, self.freq, pos)
            k, _ = D.norm_rope(qkv[:, H:H + Hk], self.gk, 1e-6, DH, False, self.freq, pos)
            o, _ = D.attention("f32", q, k, qkv[:, H + Hk:], D.visible(S, S, self.WINDOW, 0, self.SINKS), DH ** -0.5)
            out[:, s] = xs[:, s] + o.reshape(S, -1) @ wo
        return out


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_token_by_token(t):
    """Sixty tokens of three sequences, one step each. Four roundings to the type lie between the rows and the result (qkv,
    the heads, the attention, the sum): relative to the size of what they round, against a layer that changes its rows by
    its own size, 8 half steps of the root mean square cover them with the 32-bit sums' own errors (2^-16)."""
    B, S = 3, 60
    L = Layer(t, B, 4, "tokens")
    xs = D.rows(rng_of(t, "xs"), t, S, B, L.C)
    want = L.plain(D.to_f64(t, xs))
    for n in range(S):
        L.place(xs[n], np.full(B, n))
        L.step()
        got = D.to_f64(t, L.out())
        rms = np.sqrt((want[n] ** 2).mean())
        assert np.abs(got - want[n]).max() <= 6 * (8 * D.HALF[t] + 2.0 ** -16) * rms, (n, np.abs(got - want[n]).max() / rms)


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_prompt_then_tokens(t):
    """A prompt through p2h_attention_window and its keys put into the cache give the token-by-token bits of the cache."""
    B, S = 2, 25
    L, M = Layer(t, B, 4, "prompt"), Layer(t, B, 4, "prompt")
    xs = D.rows(rng_of(t, "prompt"), t, S, B, L.C)
    for n in range(S):
        L.place(xs[n], np.full(B, n))
        L.step()
    flat = np.ascontiguousarray(xs.transpose(1, 0, 2).reshape(B * S, -1))   # sequence after sequence
    H, Hk, DH, W = L.H, L.Hk, L.DH, L.W
    dx, dqkv = D.device(flat), D.preset(t, (B * S, W))
    P.q4_gemv_dev(t, B * S, W, L.C, 0.05, dx.ptr, L.C, M.q4q, 0.0, dqkv.ptr, W)
    at = np.tile(np.arange(S, dtype=np.int32), B)
    seq = np.repeat(np.arange(B), S)
    slots = (M.table[seq, at // L.PAGE] * L.PAGE + at % L.PAGE).astype(np.int32)
    dpos, dslot = D.device(at), D.device(slots)
    es = D.size(t)
    P.qk_norm_rope_dev(t, B * S, H, Hk, DH, dqkv.ptr, W, M.dgq.ptr, M.dgk.ptr, 1e-6, DH, False, M.df.ptr, dpos.ptr,
                       dqkv.ptr, W, dqkv.ptr + H * DH * es, W, M.cache, dslot.ptr)
    shape = (L.pages, Hk, L.PAGE, DH)
    for a, b in ((L.dk, M.dk), (L.dv, M.dv)):
        assert np.array_equal(a.download(shape, D.np_type(t)).view(np.uint16), b.download(shape, D.np_type(t)).view(np.uint16))
    do, starts = D.preset(t, (B * S, H * DH)), D.device(np.array([0, S, 2 * S], np.int32))
    P.attention_window_dev(t, B * S, B * S, B, starts.ptr, starts.ptr, H, Hk, DH, dqkv.ptr, W, dqkv.ptr + H * DH * es, W,
                           dqkv.ptr + (H + Hk) * DH * es, W, DH ** -0.5, L.WINDOW, 0, L.SINKS, do.ptr, H * DH)
    P.q4_gemv_dev(t, B * S, L.C, H * DH, 0.05, do.ptr, H * DH, M.q4o, 1.0, dx.ptr, L.C)
    got = D.to_f64(t, dx.download((B, S, L.C), D.np_type(t)))
    want = L.plain(D.to_f64(t, xs)).transpose(1, 0, 2)
    rms = np.sqrt((want ** 2).mean())
    assert np.abs(got - want).max() <= 6 * (8 * D.HALF[t] + 2.0 ** -16) * rms


@pytest.mark.parametrize("t", D.TYPES)
def test_layer_in_a_graph(t):
    """A captured step replayed for token after token (the places come from device arrays), with eager work between."""
    B, S = 3, 12
    L, E = Layer(t, B, 3, "graph"), Layer(t, B, 3, "graph")
    s = P.Stream()
    xs = D.rows(rng_of(t, "graph"), t, S, B, L.C)
    with P.Graph(s) as g:
        L.step(s.ptr)
    for n in range(S):
        L.place(xs[n], np.full(B, n))
        E.place(xs[n], np.full(B, n))
        P.sync()
        g.launch()
        s.sync()
        E.step()
        P.sync()
        assert np.array_equal(L.out(s.ptr).view(np.uint16), E.out().view(np.uint16)), n


def test_two_streams_at_once():
    """The same step on two streams with buffers of their own gives each its own result."""
    t, B, S = "f16", 2, 8
    layers = [Layer(t, B, 2, k) for k in ("one", "two")]
    streams = [P.Stream(), P.Stream()]
    alone = [Layer(t, B, 2, k) for k in ("one", "two")]
    xs = D.rows(rng_of("two"), t, S, B, Layer.C)
    for n in range(S):
        for L in (*layers, *alone):
            L.place(xs[n], np.full(B, n))
        P.sync()
        for L, s in zip(layers, streams):
            L.step(s.ptr)
        for s in streams:
            s.sync()
        for L, A, s in zip(layers, alone, streams):
            A.step()
            P.sync()
            assert np.array_equal(L.out(s.ptr), A.out())


@pytest.mark.parametrize("t", D.TYPES)
def test_two_graphs_share_a_workspace(t):
    """Two captured steps with one workspace, replayed in turn on one stream: each as it is alone."""
    rng = rng_of(t, "shared")
    H, Hk, Dh, page = 4, 1, 64, 16
    s, made = P.Stream(), []
    ws = None
    for lens in ((900, 40), (1, 1500)):
        q, kc, vc, table = paged_case(t, lens, H, Hk, page, Dh, "shared")
        bufs = [D.device(a) for a in (q, kc, vc, table, np.asarray(lens, np.int32))]
        cache = P.KvCache(t, Hk, Dh, page, kc.shape[0], bufs[1].ptr, bufs[2].ptr)
        if ws is None:
            ws = P.Workspace(P.attention_paged_workspace_bytes(cache, 2, H, 1500))
            assert ws.nbytes > 0
        do = D.preset(t, (2, H * Dh))
        with P.Graph(s) as g:
            P.attention_paged_dev(cache, 2, H, bufs[0].ptr, H * Dh, bufs[3].ptr, table.shape[1], bufs[4].ptr, 1500, 0.1,
                                  EVERY, 0, do.ptr, H * Dh, ws.ptr, ws.nbytes, s.ptr)
        alone = D.run_paged(t, q, kc, vc, table, lens, H, 0.1, EVERY, 0, True, 1500)
        made.append((g, do, alone, bufs))
    for _ in range(3):
        for g, do, _, _ in made:
            do.upload(np.full(do.nbytes, 0xFF, np.uint8))
        P.sync()
        for g, _, _, _ in made:
            g.launch()
        s.sync()
        for _, do, alone, _ in made:
            assert np.array_equal(do.download((2, H * Dh), D.np_type(t)).view(np.uint16), alone.view(np.uint16))


# ── weights far below the largest ───────────────────────────────────────────────────────────────────────────────

def dominated(n, nq, H, Hk, Dh, key):
    """fp16 rows whose first key takes nearly all of the weight, with a value of 0; the others' weights are about 2^-26 of
    its, so that all of the result is theirs."""
    rng = rng_of(n, H, Dh, key, "dominated")
    q, k = np.zeros((nq, H, Dh)), np.zeros((n, Hk, Dh))
    q[..., 0], k[0, :, 0] = 1.0, 18.0
    k[1:, :, 0] = rng.uniform(-0.5, 0.5, (n - 1, Hk))
    v = rng.uniform(0.5, 1.5, (n, Hk, Dh)) * rng.choice((-30, 30), (1, Hk, Dh))
    v[0] = 0.0
    return D.to_type("f16", q), D.to_type("f16", k), D.to_type("f16", v)


@pytest.mark.parametrize("n,nq,H,Hk,Dh", (
    (20000, 16, 128, 16, 128), (20000, 16, 136, 17, 64), (20000, 1, 2, 1, 64), (20000, 20, 1, 1, 128),
    (3000, 80, 128, 16, 128), (900, 100, 136, 17, 64), (20000, 600, 16, 2, 128)))   # the last three in tiles of 128 rows
def test_window_small_fp16_weights(n, nq, H, Hk, Dh):
    """Weights are rounded to fp16 for their product with V: to half a step, and down to 2^-31 of the largest one."""
    q, k, v = dominated(n, nq, H, Hk, Dh, "window")
    flat = [a.reshape(a.shape[0], -1) for a in (q, k, v)]
    got = D.to_f64("f16", D.run_window("f16", *flat, H, Hk, Dh, 1.0, EVERY, EVERY, 0))
    s = np.array([0, nq]), np.array([0, n])
    want, bound = window_want("f16", *flat, *s, H, Hk, Dh, 1.0, EVERY, EVERY, 0)
    lost = 2.0 ** -31 * np.abs(D.to_f64("f16", v)).sum(0)
    D.check(got, want, bound + np.repeat(lost, H // Hk, 0).reshape(1, -1), f"{nq} {H} {Dh}")


@pytest.mark.parametrize("n,split", ((20000, False), (20000, True), (700, True)))
@pytest.mark.parametrize("Dh", (64, 128))
def test_paged_small_fp16_weights(n, split, Dh):
    """As above; here a weight is taken relative to the largest one of its wave's keys and held down to 2^-40 of it."""
    H, Hk, page = 4, 2, 16
    q, k, v = dominated(n, 1, H, Hk, Dh, "paged")
    per = -(-n // page)
    table = rng_of("dominated pages").permutation(per).astype(np.int32)[None]
    kc, vc = (np.zeros((per, Hk, page, Dh), np.float16) for _ in range(2))
    j = np.arange(n)
    kc[table[0, j // page], :, j % page], vc[table[0, j // page], :, j % page] = k, v
    got = D.to_f64("f16", D.run_paged("f16", q.reshape(1, -1), kc, vc, table, (n,), H, 1.0, EVERY, 0, split))
    want, bound = paged_want("f16", q.reshape(1, -1), kc, vc, table, (n,), H, 1.0, EVERY, 0)
    lost = 2.0 ** -40 * np.abs(D.to_f64("f16", v)).sum(0)
    D.check(got, want, bound + np.repeat(lost, H // Hk, 0).reshape(1, -1), f"{n} {split} {Dh}")


# ── errors ──────────────────────────────────────────────────────────────────────────────────────────────────────

def test_a_refused_allocation_is_reported_once():
    """What follows it on the thread works: an upload, a linear, a five-value weight."""
    K, N, group = 128, 32, 32
    rng = rng_of("refused")
    x, wt = D.rows(rng, "f32", 2, K), D.q4_weight(rng, K, N, group, True)
    want = D.run_q4("f32", x, wt, K, N, group)
    planes = P.gen_fv_weight(1, 1, 128, 64)
    w, dx, dy = P.Q4Weight(*wt, K, N, group), D.device(x), D.preset("f32", (2, N))

    def refuse():
        with pytest.raises(P.P2Error, match="hipMalloc"):
            P.DeviceBuffer(1 << 50)

    refuse()
    P.Q4Weight(*wt, K, N, group)
    refuse()
    P.q4_gemv_dev("f32", 2, N, K, 1.0, dx.ptr, K, w, 0.0, dy.ptr, N)
    assert np.array_equal(dy.download((2, N), np.float32), want)
    refuse()
    P.FvWeight(*planes, 128, 64)
    with pytest.raises(P.P2Error):
        P.Event().elapsed_ms(P.Event())   # never recorded
    P.q4_gemv_dev("f32", 2, N, K, 1.0, dx.ptr, K, w, 0.0, dy.ptr, N)


@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("H,Dh,starts", ((2, 64, True), (32, 128, False), (48, 64, True)))
def test_window_without_keys(t, H, Dh, starts):
    """No key rows at all, and then no pointers to any: zeros in both forms."""
    n = 700 if H > 2 else 40
    q = D.rows(rng_of(t, H, "no keys"), t, n, H * Dh)
    dq, do = D.device(q), D.preset(t, (n, H * Dh))
    qs, ks = D.device(np.array([0, 0, n], np.int32)), D.device(np.zeros(3, np.int32))
    P.attention_window_dev(t, n, 0, 2 if starts else 1, qs.ptr if starts else None, ks.ptr if starts else None, H, H, Dh, dq.ptr,
                           H * Dh, None, 0, None, 0, 0.1, EVERY, EVERY, 5, do.ptr, H * Dh)
    assert not D.to_f64(t, do.download((n, H * Dh), D.np_type(t))).any()


# ── many sequences of few queries ───────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("lens,past,H,Hk,Dh", (((1,) * 64, 40, 32, 8, 128), ((3, 1, 0, 8) * 20, 70, 24, 4, 64),
                                               ((17,) * 30, 0, 24, 4, 128), ((2,) * 5, 1100, 32, 8, 64)))
def test_window_batches_of_few_queries(t, lens, past, H, Hk, Dh):
    q, k, v, qs, ks = window_case(t, lens, past, H, Hk, Dh, "batch")
    got = D.run_window(t, q, k, v, H, Hk, Dh, Dh ** -0.5, EVERY, 0, 0, qs, ks)
    want, bound = window_want(t, q, k, v, qs, ks, H, Hk, Dh, Dh ** -0.5, EVERY, 0, 0)
    D.check(D.to_f64(t, got), want, bound, f"{t} {Dh} {H}")


# ── fp32 results on the whole ───────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("M", (1, 5, 18))
@pytest.mark.parametrize("group,zeros", ((32, False), (32, True), (64, True), (128, False), (128, True)))
@pytest.mark.parametrize("K,N", ((1024, 48), (4096, 40), (8200, 24), (1000, 8201), (1024, 16400)))
def test_q4_fp32_on_the_whole(M, K, N, group, zeros):
    rng = rng_of(M, K, N, group, zeros, "whole")
    x, wt = D.rows(rng, "f32", M, K), D.q4_weight(rng, K, N, group, zeros)
    want = x.astype(np.float64) @ D.q4_values(*wt, K, N, group)
    off = D.norm_off(D.run_q4("f32", x, wt, K, N, group).astype(np.float64), want)
    assert off <= D.Q4_NORM, off / D.FP32


@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,past,H,Hk,window,ahead,sinks", WIN + BIG)
def test_window_fp32_on_the_whole(Dh, lens, past, H, Hk, window, ahead, sinks):
    q, k, v, qs, ks = window_case("f32", lens, past, H, Hk, Dh, "whole")
    got = D.run_window("f32", q, k, v, H, Hk, Dh, Dh ** -0.5, window, ahead, sinks, qs, ks)
    want, _ = window_want("f32", q, k, v, qs, ks, H, Hk, Dh, Dh ** -0.5, window, ahead, sinks)
    if want.any():
        off = D.norm_off(got.astype(np.float64), want)
        assert off <= D.ATTENTION_NORM, off / D.FP32
    else:
        assert not got.any()


@pytest.mark.parametrize("split", (False, True))
@pytest.mark.parametrize("Dh", (64, 128))
@pytest.mark.parametrize("lens,H,Hk,page,window,sinks", PAGED)
def test_paged_fp32_on_the_whole(split, Dh, lens, H, Hk, page, window, sinks):
    q, kc, vc, table = paged_case("f32", lens, H, Hk, page, Dh, "whole")
    want, _ = paged_want("f32", q, kc, vc, table, lens, H, Dh ** -0.5, window, sinks)
    got = D.run_paged("f32", q, kc, vc, table, lens, H, Dh ** -0.5, window, sinks, split, 40000 if split else None)
    off = D.norm_off(got.astype(np.float64), want)
    assert off <= D.ATTENTION_NORM, off / D.FP32


# ── calls that the documentation allows ─────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("t", D.TYPES)
@pytest.mark.parametrize("H,Hk,Dh", ((2, 1, 64), (32, 8, 128)))
def test_window_in_a_graph_sees_new_starts(t, H, Hk, Dh):
    """A captured call reads its sequences' starts when it is replayed, in both forms; eager work lies between replays."""
    n = 600
    q, k, v, _, _ = window_case(t, (n,), 0, H, Hk, Dh, "graph")
    dq, dk, dv = D.device(q), D.device(k), D.device(v)
    dqs, dks = D.device(np.zeros(4, np.int32)), D.device(np.zeros(4, np.int32))
    do, s = D.preset(t, (n, H * Dh)), P.Stream()
    with P.Graph(s) as g:
        P.attention_window_dev(t, n, n, 3, dqs.ptr, dks.ptr, H, Hk, Dh, dq.ptr, H * Dh, dk.ptr, Hk * Dh, dv.ptr, Hk * Dh, 0.1,
                               90, 2, 3, do.ptr, H * Dh, s.ptr)
    for qs, ks in (([0, 200, 200, 600], [0, 150, 300, 600]), ([5, 6, 300, 333], [0, 0, 600, 600]), ([0, 0, 0, 600], [1, 2, 3, 599])):
        dqs.upload(np.array(qs, np.int32))
        dks.upload(np.array(ks, np.int32))
        do.upload(np.full(do.nbytes, 0xFF, np.uint8))
        P.sync()
        g.launch()
        s.sync()
        eager = D.run_window(t, q, k, v, H, Hk, Dh, 0.1, 90, 2, 3, qs, ks)
        assert np.array_equal(do.download((n, H * Dh), D.np_type(t)).view(np.uint16), eager.view(np.uint16)), (qs, ks)


@pytest.mark.parametrize("t", D.TYPES)
def test_paged_sequences_share_pages(t):
    """A page may stand in several sequences' rows, and more than once in one: the bits of pages of their own."""
    H, Hk, Dh, page, lens = 8, 2, 64, 16, (150, 150, 70)
    q, kc, vc, table = paged_case(t, lens, H, Hk, page, Dh, "share")
    table[1, :6] = table[0, :6]
    table[2, 1] = table[2, 2] = table[0, 3]
    own, k2, v2 = table.copy(), [kc], [vc]
    at = kc.shape[0]
    for s in range(3):
        for p in range(-(-lens[s] // page)):
            k2.append(kc[table[s, p]:table[s, p] + 1])
            v2.append(vc[table[s, p]:table[s, p] + 1])
            own[s, p] = at
            at += 1
    k2, v2 = np.concatenate(k2), np.concatenate(v2)
    for split in (False, True):
        a = D.run_paged(t, q, kc, vc, table, lens, H, 0.1, EVERY, 0, split, 40000)
        b = D.run_paged(t, q, k2, v2, own, lens, H, 0.1, EVERY, 0, split, 40000)
        assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_layers_on_two_threads():
    """Two host threads, each with its stream and its buffers, at once: the results of one after the other."""
    import threading
    t, B, S = "bf16", 2, 10
    xs = D.rows(rng_of("threads"), t, S, B, Layer.C)

    def run(seed, out):
        L, s = Layer(t, B, 2, seed), P.Stream()
        got = []
        for n in range(S):
            L.place(xs[n], np.full(B, n))
            P.sync()
            L.step(s.ptr)
            got.append(L.out(s.ptr))
        out.append(np.stack(got))

    alone, both = [[], []], [[], []]
    for i, seed in enumerate(("one", "two")):
        run(seed, alone[i])
    threads = [threading.Thread(target=run, args=(seed, both[i])) for i, seed in enumerate(("one", "two"))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for a, b in zip(alone, both):
        assert len(b) == 1 and np.array_equal(a[0], b[0])


@pytest.mark.parametrize("t,M", (("bf16", 1), ("f32", 1), ("f16", 3)))
def test_q4_weight_beyond_32_bits(t, M):
    """A weight of nearly 2^35 codes, its records past 2^32 bytes: the rows and columns at its ends."""
    K, N, group = 1 << 18, 131056, 128
    half, groups = N // 2, K // group
    dc, ds = P.DeviceBuffer(K * half), P.DeviceBuffer(groups * N * 2)
    for b, byte in ((dc, 0x99), (ds, 0x3C)):   # code 9, less 8, by the fp16 of bits 0x3C3C
        assert P.hip().p2h_memset(b.ptr, byte, b.nbytes, None) == 0
    P.sync()
    scale = float(np.array([0x3C3C], np.uint16).view(np.float16)[0])
    rows, rng = (0, 1, K // 2 + 5, K - 1), rng_of("beyond")
    w = np.full((len(rows), N), 1.0)
    for i, r in enumerate(rows):   # these rows have codes of their own in the last and the first 64 columns
        for c0 in (0, half - 32):
            codes = rng.integers(0, 256, 32, dtype=np.uint8)
            dc.upload(codes, offset=r * half + c0)
            w[i, 2 * c0:2 * c0 + 64] = D.nibbles(codes[None], 64)[0] - 8.0
    weight = P.Q4Weight.wrap(dc.ptr, ds.ptr, None, K, N, group)
    del dc, ds
    x = np.zeros((M, K))
    x[:, rows] = rng.integers(1, 4, (M, len(rows)))
    dx, dy = D.device(D.to_type(t, x)), D.preset(t, (M, N))
    P.q4_gemv_dev(t, M, N, K, 1.0, dx.ptr, K, weight, 0.0, dy.ptr, N)
    got = D.to_f64(t, dy.download((M, N), D.np_type(t)))
    want = x[:, rows] @ w * scale
    assert np.array_equal(got, D.to_f64(t, D.to_type(t, want)))   # sums of small whole numbers, one scale each group: exact
    weight.free()
