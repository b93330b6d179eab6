/*  p2hip_decoder.hip – the device-pointer C ABI of a decoder layer's step (include/p2hip.h) over the kernels in
 *  p2hip_decoder.h.
 *
 *  As in p2hip.hip every shape, stride and alignment that a kernel assumes is checked before its launch, the arguments
 *  before the device, so that a call is refused the same way with or without one.
 */
#include "p2hip_host.h"

#include <climits>
#include <cmath>
#include <cstring>
#include <new>

#include "p2hip_decoder.h"

using p2host::align_up;
using p2host::aligned;
using p2host::cu_count;
using p2host::ensure_init;
using p2host::fail;
using p2host::stream_of;

struct P2hQ4Weight {
    int K, N, group, tiles, units;
    bool zeros;
    uint8_t *base;   /* the one device allocation: records, then scales */
    size_t sc_off, bytes;
};

namespace {

constexpr size_t kGridThreads = (size_t)1 << 32;   /* a launch has fewer threads */

inline size_t elem_size(int dtype) { return dtype == P2H_F32 ? 4 : 2; }
inline bool is_type(int dtype) { return dtype == P2H_F32 || dtype == P2H_F16 || dtype == P2H_BF16; }

template <int V> using ic = std::integral_constant<int, V>;

/* f(type, …) with the element type as a constant */
template <class F> void by_type(int dtype, F f)
{
    if (dtype == P2H_F32) f(ic<p2k::T_F32>{});
    else if (dtype == P2H_F16) f(ic<p2k::T_F16>{});
    else f(ic<p2k::T_BF16>{});
}

/* f(type, head_dim) */
template <class F> void by_type_dim(int dtype, int head_dim, F f)
{
    by_type(dtype, [&](auto t) {
        if (head_dim == 64) f(t, ic<64>{});
        else f(t, ic<128>{});
    });
}

/* M rows of `w` bytes at pitch `ld` bytes, as a range */
struct Rows {
    const char *p;
    size_t ld, w;
    int M;
    const char *end() const { return p + (M ? (size_t)(M - 1) * ld + w : 0); }
};

/* whether two sets of rows share a byte: apart as ranges, or of one pitch with their columns apart */
bool overlap(const Rows &a, const Rows &b)
{
    if (a.M <= 0 || b.M <= 0 || a.end() <= b.p || b.end() <= a.p) return false;
    if (a.ld != b.ld) return true;
    const size_t d = a.p <= b.p ? (size_t)(b.p - a.p) % a.ld : (a.ld - (size_t)(a.p - b.p) % a.ld) % a.ld;
    return !(d >= a.w && d + b.w <= a.ld);
}

int check_heads(const char *name, int dtype, int heads, int kv_heads, int head_dim)
{
    if (!is_type(dtype)) return fail(P2H_E_ARG, "%s: element type %d", name, dtype);
    if (head_dim != 64 && head_dim != 128) return fail(P2H_E_ARG, "%s: head_dim = %d (64 or 128)", name, head_dim);
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || heads > 65536)
        return fail(P2H_E_ARG, "%s: %d heads over %d key heads", name, heads, kv_heads);
    return P2H_OK;
}

int check_rows(const char *name, const char *what, int dtype, const void *p, int ld, int width)
{
    if (!p || !aligned(p, 16)) return fail(P2H_E_ARG, "%s: %s is NULL or not 16-byte aligned", name, what);
    if (ld < width || (size_t)ld * elem_size(dtype) % 16 != 0)
        return fail(P2H_E_ARG, "%s: pitch %d of %s must be >= %d and a multiple of 16 bytes", name, ld, what, width);
    /* a block's rows are addressed by 32-bit offsets from its first */
    if (ld >= 1 << 23) return fail(P2H_E_ARG, "%s: pitch %d of %s must be below 2^23", name, ld, what);
    return P2H_OK;
}

int check_cache(const char *name, const P2hKvCache *c)
{
    if (!c) return fail(P2H_E_ARG, "%s: NULL cache", name);
    if (!is_type(c->dtype) || c->heads < 1 || c->heads > 65536 || (c->head_dim != 64 && c->head_dim != 128))
        return fail(P2H_E_ARG, "%s: cache of type %d with %d heads of %d", name, c->dtype, c->heads, c->head_dim);
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)) != 0 || c->pages < 0)
        return fail(P2H_E_ARG, "%s: %d pages of %d tokens (a power of two, 16 .. 1024)", name, c->pages, c->page);
    if (c->pages > 0 && (!c->K || !c->V || !aligned(c->K, 16) || !aligned(c->V, 16)))
        return fail(P2H_E_ARG, "%s: cache memory is NULL or not 16-byte aligned", name);
    return P2H_OK;
}

/* a cache's keys or values as one row, and whether rows share a byte with either */
Rows cache_row(const P2hKvCache *c, const void *p)
{
    const size_t bytes = (size_t)c->pages * c->heads * c->page * c->head_dim * elem_size(c->dtype);
    return Rows{(const char *)p, bytes, bytes, bytes ? 1 : 0};
}
bool overlap(const Rows &a, const P2hKvCache *c)
{
    return overlap(a, cache_row(c, c->K)) || overlap(a, cache_row(c, c->V));
}

int log2_of(int page)
{
    int s = 0;
    while ((1 << s) < page) s++;
    return s;
}

}  // namespace

extern "C" {

/* ── 4-bit weights ─────────────────────────────────────────────────────────────────────────────────────────── */

static P2hQ4Weight *q4_make(const char *name, const void *d_codes, const void *d_scales, const void *d_zeros, int K, int N,
                            int group)
{
    const int tiles = (N - 1) / 16 + 1, units = (K - 1) / 128 + 1, gpu = 128 / group;
    const size_t n_rec = (size_t)tiles * units * 256, n_sc = (size_t)tiles * units * 16 * gpu;
    P2hQ4Weight *w = new (std::nothrow) P2hQ4Weight();
    if (!w) {
        fail(P2H_E_NOMEM, "%s: no host memory", name);
        return nullptr;
    }
    w->K = K; w->N = N; w->group = group; w->tiles = tiles; w->units = units;
    w->zeros = d_zeros != nullptr;
    w->sc_off = align_up(n_rec * 4, 256);
    w->bytes = w->sc_off + n_sc * (w->zeros ? 4 : 2);
    void *p = nullptr;
    if (hipMalloc(&p, w->bytes) != hipSuccess) {
        fail(P2H_E_NOMEM, "%s: hipMalloc(%zu) failed", name, w->bytes);
        delete w;
        return nullptr;
    }
    w->base = (uint8_t *)p;
    hipStream_t s = stream_of(nullptr);
    const size_t n = n_rec > n_sc ? n_rec : n_sc;
    hipLaunchKernelGGL(p2k::q4_records, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, K, N, group, tiles, units,
                       (const uint8_t *)d_codes, (const uint16_t *)d_scales, (const uint8_t *)d_zeros, (uint32_t *)p,
                       (uint16_t *)(w->base + w->sc_off));
    const hipError_t launched = hipGetLastError(), done = hipStreamSynchronize(s);
    if (launched != hipSuccess || done != hipSuccess) {
        fail(P2H_E_DEVICE, "%s: %s", name, hipGetErrorString(launched != hipSuccess ? launched : done));
        p2h_q4_weight_free(w);
        return nullptr;
    }
    return w;
}

static int q4_check(const char *name, const void *codes, const void *scales, int K, int N, int group)
{
    if (!codes || !scales || !aligned(scales, 2)) return fail(P2H_E_ARG, "%s: NULL codes or scales, or scales not aligned", name);
    if (K < 1 || N < 1 || K > (1 << 28) || N > (1 << 28)) return fail(P2H_E_ARG, "%s: K = %d, N = %d", name, K, N);
    if (group != 32 && group != 64 && group != 128) return fail(P2H_E_ARG, "%s: group = %d (32, 64 or 128)", name, group);
    /* one thread per record word, and at most 512 per two column tiles: a grid has fewer than 2^32 threads */
    if (N > 1 << 27 || (size_t)((N - 1) / 16 + 1) * ((K - 1) / 128 + 1) * 256 >= kGridThreads)
        return fail(P2H_E_ARG, "%s: K = %d by N = %d is too large", name, K, N);
    return P2H_OK;
}

P2hQ4Weight *p2h_q4_weight_wrap(const void *d_codes, const void *d_scales, const void *d_zeros, int K, int N, int group)
{
    const char *name = "p2h_q4_weight_wrap";
    if (q4_check(name, d_codes, d_scales, K, N, group) || ensure_init()) return nullptr;
    return q4_make(name, d_codes, d_scales, d_zeros, K, N, group);
}

P2hQ4Weight *p2h_q4_weight_upload(const unsigned char *codes, const uint16_t *scales, const unsigned char *zeros, int K,
                                  int N, int group)
{
    const char *name = "p2h_q4_weight_upload";
    if (q4_check(name, codes, scales, K, N, group) || ensure_init()) return nullptr;
    const size_t half = ((size_t)N + 1) / 2, groups = ((size_t)K - 1) / group + 1;
    const size_t cb = align_up(half * K, 256), sb = align_up(groups * N * 2, 256), zb = zeros ? groups * half : 0;
    void *stage = nullptr;
    if (hipMalloc(&stage, cb + sb + zb) != hipSuccess) {
        fail(P2H_E_NOMEM, "%s: hipMalloc(%zu) for the codes failed", name, cb + sb + zb);
        return nullptr;
    }
    uint8_t *d = (uint8_t *)stage;
    hipStream_t s = stream_of(nullptr);
    const bool ok = hipMemcpyAsync(d, codes, half * K, hipMemcpyHostToDevice, s) == hipSuccess &&
                    hipMemcpyAsync(d + cb, scales, groups * N * 2, hipMemcpyHostToDevice, s) == hipSuccess &&
                    (!zeros || hipMemcpyAsync(d + cb + sb, zeros, zb, hipMemcpyHostToDevice, s) == hipSuccess);
    P2hQ4Weight *w = nullptr;
    if (ok) w = q4_make(name, d, d + cb, zeros ? d + cb + sb : nullptr, K, N, group);
    else fail(P2H_E_DEVICE, "%s: copy failed", name);
    (void)hipStreamSynchronize(s);   /* nothing reads host memory or the staging buffer any more */
    (void)hipFree(stage);
    return w;
}

void p2h_q4_weight_free(P2hQ4Weight *w)
{
    if (!w) return;
    if (w->base) (void)hipFree(w->base);
    delete w;
}

int p2h_q4_weight_shape(const P2hQ4Weight *w, int *K, int *N, int *group)
{
    if (!w) return fail(P2H_E_ARG, "p2h_q4_weight_shape: NULL weight");
    if (K) *K = w->K;
    if (N) *N = w->N;
    if (group) *group = w->group;
    return P2H_OK;
}

size_t p2h_q4_weight_device_bytes(const P2hQ4Weight *w) { return w ? w->bytes : 0; }

int p2h_q4_gemv(int dtype, int M, int N, int K, float alpha, const void *dX, int ldx, const P2hQ4Weight *w, float beta,
                void *dY, int ldy, void *stream)
{
    const char *name = "p2h_q4_gemv";
    if (!is_type(dtype)) return fail(P2H_E_ARG, "%s: element type %d", name, dtype);
    if (!w) return fail(P2H_E_ARG, "%s: NULL weight", name);
    if (M < 0 || N != w->N || K != w->K)
        return fail(P2H_E_ARG, "%s: M = %d, K = %d, N = %d for a weight [%d, %d]", name, M, K, N, w->K, w->N);
    if (M > 16 * 65535) return fail(P2H_E_ARG, "%s: M = %d (at most %d rows)", name, M, 16 * 65535);
    if (M == 0) return P2H_OK;
    const size_t es = elem_size(dtype);
    if (!dX || !dY || ldx < K || ldy < N || !aligned(dX, es) || !aligned(dY, es))
        return fail(P2H_E_ARG, "%s: NULL or unaligned rows, or ldx = %d < K = %d, ldy = %d < N = %d", name, ldx, K, ldy, N);
    if (overlap(Rows{(const char *)dX, ldx * es, K * es, M}, Rows{(const char *)dY, ldy * es, N * es, M}))
        return fail(P2H_E_ARG, "%s: X and Y overlap", name);
    if (int rc = ensure_init()) return rc;
    p2k::Q4Args a{};
    a.M = M; a.N = N; a.K = K; a.units = w->units; a.ldx = ldx; a.ldy = ldy;
    a.vec = p2k::rows_by_16((uintptr_t)dX, ldx, (int)es, M);
    a.alpha = alpha; a.beta = beta; a.x = dX; a.y = dY;
    a.rec = (const p2k::u4 *)w->base;
    a.sc = w->base + w->sc_off;
    const unsigned row_blocks = (unsigned)((M + 15) / 16);
    hipStream_t s = stream_of(stream);
    by_type(dtype, [&](auto t) {
        auto launch = [&](auto group, auto zp) {
            constexpr int DT = decltype(t)::value, G = decltype(group)::value;
            constexpr bool Z = decltype(zp)::value != 0;
            auto go = [&](auto wv, auto nt) {
                constexpr int WV = decltype(wv)::value, NT = decltype(nt)::value;
                const dim3 grid((unsigned)((w->tiles + NT - 1) / NT), row_blocks);
                if constexpr (DT == p2k::T_F32) {
                    if (M == 1) {
                        hipLaunchKernelGGL((p2k::q4_gemv<DT, G, Z, WV, NT, true>), grid, dim3(64 * WV), 0, s, a);
                        return;
                    }
                }
                hipLaunchKernelGGL((p2k::q4_gemv<DT, G, Z, WV, NT, false>), grid, dim3(64 * WV), 0, s, a);
            };
            /* How many column tiles a wave takes with its rows' values, NT, and the waves that share a tile's K, WV. NT so
             * that one workgroup a CU takes them all (fp16 13 x 4096: 768 tiles 8.1 us by threes, 9.9 by twos, 10.6 one by
             * one; 1024 tiles 9.8 by fours, 12.5 by threes), fp32 rows at most three, for their registers. Of more tiles
             * two (1025: 12.1 us, 12.5 by threes, 14.8 by fours), several fp32 rows three (9 x 4096, 1025 tiles: 23.0
             * against 25.7); from eight a CU on four, in workgroups of four waves, as with a short K eight have one unit
             * each (bf16 16 x 1024, 8000 tiles: 18.3 us against 25.8; fp16 13 x 4096, 2048 tiles: 18.0, 18.4). Sixteen waves
             * where a long K has few tiles (bf16 1 x 14336, 256 tiles: 10.2 us against 11.7; K of 4096: 4.7, 4.8), but not
             * for fp32 rows, whose values would not fit. WV, which sets the order of a row's sums, goes by the weight and
             * the type alone. */
            const int tiles = w->tiles, cus = cu_count();
            if constexpr (DT == p2k::T_F32) {
                if (tiles <= cus) go(ic<8>{}, ic<1>{});
                else if (tiles <= 2 * cus || (tiles > 3 * cus && M == 1)) go(ic<8>{}, ic<2>{});
                else go(ic<8>{}, ic<3>{});
            } else {
                if (tiles <= cus && w->units >= 64) go(ic<16>{}, ic<1>{});
                else if (tiles <= cus) go(ic<8>{}, ic<1>{});
                else if (tiles >= 8 * cus) go(ic<4>{}, ic<4>{});
                else if (tiles <= 2 * cus || tiles > 4 * cus) go(ic<8>{}, ic<2>{});
                else if (tiles <= 3 * cus) go(ic<8>{}, ic<3>{});
                else go(ic<8>{}, ic<4>{});
            }
        };
        auto by_zero = [&](auto group) {
            if (w->zeros) launch(group, ic<1>{});
            else launch(group, ic<0>{});
        };
        if (w->group == 32) by_zero(ic<32>{});
        else if (w->group == 64) by_zero(ic<64>{});
        else by_zero(ic<128>{});
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

/* ── head norms, rotation and the cache ────────────────────────────────────────────────────────────────────── */

int p2h_qk_norm_rope(int dtype, int T, int heads, int kv_heads, int head_dim, const void *dQKV, int ldqkv,
                     const float *dGammaQ, const float *dGammaK, float eps, int rot, int interleaved, const float *dFreq,
                     const int *dPos, void *dQ, int ldq, void *dK, int ldk, const P2hKvCache *cache, const int *dSlots,
                     void *stream)
{
    const char *name = "p2h_qk_norm_rope";
    if (int rc = check_heads(name, dtype, heads, kv_heads, head_dim)) return rc;
    if (T < 0 || (size_t)T * 256 >= kGridThreads) return fail(P2H_E_ARG, "%s: T = %d (below 2^24)", name, T);
    if (rot < 0 || rot > head_dim || rot % 16 != 0)
        return fail(P2H_E_ARG, "%s: rot = %d (a multiple of 16 up to head_dim = %d)", name, rot, head_dim);
    if (!(eps >= 0.0f)) return fail(P2H_E_ARG, "%s: eps = %g", name, (double)eps);
    if (cache) {
        if (int rc = check_cache(name, cache)) return rc;
        if (overlap(cache_row(cache, cache->K), cache_row(cache, cache->V)))
            return fail(P2H_E_ARG, "%s: the cache's keys and values overlap", name);
        if (cache->dtype != dtype || cache->heads != kv_heads || cache->head_dim != head_dim)
            return fail(P2H_E_ARG, "%s: the cache holds %d heads of %d, type %d", name, cache->heads, cache->head_dim,
                        cache->dtype);
    }
    if (!cache && !dK) return fail(P2H_E_ARG, "%s: neither dK nor a cache takes the keys", name);
    if (T == 0) return P2H_OK;
    const int in_w = (heads + (cache ? 2 : 1) * kv_heads) * head_dim, q_w = heads * head_dim, k_w = kv_heads * head_dim;
    if (int rc = check_rows(name, "dQKV", dtype, dQKV, ldqkv, in_w)) return rc;
    if (int rc = check_rows(name, "dQ", dtype, dQ, ldq, q_w)) return rc;
    if (dK)
        if (int rc = check_rows(name, "dK", dtype, dK, ldk, k_w)) return rc;
    if (!dGammaQ || !dGammaK || !aligned(dGammaQ, 4) || !aligned(dGammaK, 4) || (rot > 0 && (!dFreq || !dPos)) ||
        (cache && !dSlots))
        return fail(P2H_E_ARG, "%s: NULL or unaligned norm weights, or NULL frequencies, positions or slots", name);
    const size_t es = elem_size(dtype);
    const Rows x{(const char *)dQKV, ldqkv * es, in_w * es, T}, q{(const char *)dQ, ldq * es, q_w * es, T};
    const Rows xk{x.p + q_w * es, x.ld, in_w * es - q_w * es, T};   /* the rows from their keys on */
    /* in place: exactly the q columns, apart from everything else (a single row has no pitch) */
    const bool q_in = dQ == dQKV && (ldq == ldqkv || T == 1);
    if (q_in ? overlap(q, xk) : overlap(q, x)) return fail(P2H_E_ARG, "%s: dQ overlaps dQKV other than in place", name);
    if (dK) {
        const Rows k{(const char *)dK, ldk * es, k_w * es, T};
        const Rows xq{x.p, x.ld, q_w * es, T}, xv{xk.p + k_w * es, x.ld, xk.w - k_w * es, xk.w > k_w * es ? T : 0};
        const bool k_in = k.p == xk.p && (ldk == ldqkv || T == 1);
        if (k_in ? overlap(k, xq) || overlap(k, xv) : overlap(k, x))
            return fail(P2H_E_ARG, "%s: dK overlaps dQKV other than in place", name);
        if (overlap(q, k)) return fail(P2H_E_ARG, "%s: dQ and dK overlap", name);
        if (cache && overlap(k, cache)) return fail(P2H_E_ARG, "%s: dK overlaps the cache", name);
    }
    if (cache && (overlap(x, cache) || overlap(q, cache))) return fail(P2H_E_ARG, "%s: dQKV or dQ overlaps the cache", name);
    if (int rc = ensure_init()) return rc;
    p2k::RopeArgs a{};
    a.T = T; a.heads = heads; a.kv = kv_heads; a.rot = rot; a.interleaved = interleaved != 0;
    a.ldx = ldqkv; a.ldq = ldq; a.ldk = ldk; a.eps = eps;
    a.x = dQKV; a.q = dQ; a.k = dK; a.gq = dGammaQ; a.gk = dGammaK; a.freq = dFreq; a.pos = dPos;
    if (cache) {
        a.kc = cache->K; a.vc = cache->V; a.slots = dSlots;
        a.page_shift = log2_of(cache->page);
        a.slots_in_cache = (long long)cache->pages * cache->page;
    }
    hipStream_t s = stream_of(stream);
    by_type_dim(dtype, head_dim, [&](auto t, auto d) {
        constexpr int DT = decltype(t)::value, DH = decltype(d)::value;
        if (T <= 256) hipLaunchKernelGGL((p2k::qk_norm_rope<DT, DH, 1024>), dim3((unsigned)T), dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((p2k::qk_norm_rope<DT, DH, 256>), dim3((unsigned)T), dim3(256), 0, s, a);
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

/* ── attention ─────────────────────────────────────────────────────────────────────────────────────────────── */

static int check_scale(const char *name, float scale, int window, int ahead, int sinks)
{
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(P2H_E_ARG, "%s: scale = %g must be positive", name, (double)scale);
    if (window < 1 || window > (1 << 30) || ahead < 0 || ahead > (1 << 30) || sinks < 0 || sinks > (1 << 30))
        return fail(P2H_E_ARG, "%s: window = %d (1 .. 2^30), ahead = %d, sinks = %d (0 .. 2^30)", name, window, ahead, sinks);
    return P2H_OK;
}

int p2h_attention_window(int dtype, int q_rows, int k_rows, int n_seqs, const int *dQStart, const int *dKStart, int heads,
                         int kv_heads, int head_dim, const void *dQ, int ldq, const void *dK, int ldk, const void *dV,
                         int ldv, float scale, int window, int ahead, int sinks, void *dO, int ldo, void *stream)
{
    const char *name = "p2h_attention_window";
    if (int rc = check_heads(name, dtype, heads, kv_heads, head_dim)) return rc;
    if (int rc = check_scale(name, scale, window, ahead, sinks)) return rc;
    if (q_rows < 0 || k_rows < 0 || q_rows >= (1 << 30) || k_rows >= (1 << 30) || n_seqs < 0)
        return fail(P2H_E_ARG, "%s: %d sequences of %d query and %d key rows (below 2^30)", name, n_seqs, q_rows, k_rows);
    if (!dQStart != !dKStart || (!dQStart && n_seqs != 1))
        return fail(P2H_E_ARG, "%s: %d sequences need their starts, of queries and of keys", name, n_seqs);
    if (q_rows == 0 || n_seqs == 0) return P2H_OK;
    if (int rc = check_rows(name, "dQ", dtype, dQ, ldq, heads * head_dim)) return rc;
    if (int rc = check_rows(name, "dO", dtype, dO, ldo, heads * head_dim)) return rc;
    const size_t es = elem_size(dtype), q_w = (size_t)heads * head_dim * es, k_w = (size_t)kv_heads * head_dim * es;
    const Rows o{(const char *)dO, ldo * es, q_w, q_rows};
    if (k_rows > 0) {
        if (int rc = check_rows(name, "dK", dtype, dK, ldk, kv_heads * head_dim)) return rc;
        if (int rc = check_rows(name, "dV", dtype, dV, ldv, kv_heads * head_dim)) return rc;
        if (overlap(o, Rows{(const char *)dK, ldk * es, k_w, k_rows}) ||
            overlap(o, Rows{(const char *)dV, ldv * es, k_w, k_rows}))
            return fail(P2H_E_ARG, "%s: dO overlaps dK or dV", name);
    }
    if (overlap(o, Rows{(const char *)dQ, ldq * es, q_w, q_rows})) return fail(P2H_E_ARG, "%s: dO overlaps dQ", name);
    /* at most 256 threads for 128 rows of one head and for one tile more of each sequence; 512 where they go by 16 queries,
     * which is looked at there */
    if (((size_t)(q_rows / 128 + 1) + n_seqs) * heads + 2048 >= kGridThreads / 512)
        return fail(P2H_E_ARG, "%s: %d rows of %d heads in %d sequences are too many for one call", name, q_rows, heads, n_seqs);
    if (int rc = ensure_init()) return rc;
    /* The queries of a tile and the query heads a workgroup takes (its kernel says why); one tile more per sequence than
     * the rows fill (tile_start). */
    const int G = heads / kv_heads, hpw = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    const size_t few_wgs = ((size_t)q_rows / 16 + n_seqs) * heads;
    const bool few = few_wgs < kGridThreads / 512 && p2k::few_queries(dtype == P2H_F32, head_dim, q_rows, k_rows, n_seqs, heads,
                                                                      window, ahead, cu_count());
    const int qb = few ? 16 : dtype == P2H_F32 ? 128 : 128 / hpw, per = few || dtype == P2H_F32 ? 1 : hpw;
    const long long tiles = (long long)(dQStart ? q_rows / qb + n_seqs : (q_rows + qb - 1) / qb);
    p2k::WinArgs a{};
    a.q_rows = q_rows; a.k_rows = k_rows; a.n_seqs = n_seqs; a.heads = heads; a.kv = kv_heads;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo; a.window = window; a.ahead = ahead; a.sinks = sinks;
    a.tiles = (int)tiles; a.hpw = per; a.c = scale * p2k::kLog2e;
    a.qs = dQStart; a.ks = dKStart; a.q = dQ; a.k = dK; a.v = dV; a.o = dO;
    hipStream_t s = stream_of(stream);
    const int sets = heads / per, wgs = (int)tiles * sets, cus = cu_count();
    a.turn = !few && wgs > cus && wgs <= 2 * cus && sets <= cus ? cus / sets * sets : wgs;
    const dim3 grid((unsigned)wgs);
    by_type_dim(dtype, head_dim, [&](auto t, auto d) {
        constexpr int DT = decltype(t)::value, DH = decltype(d)::value;
        if (few) hipLaunchKernelGGL((p2k::attention_win_few<DT, DH, 8>), grid, dim3(512), 0, s, a);
        else if constexpr (DT == p2k::T_F32) hipLaunchKernelGGL((p2k::attention_win_f32<DH>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((p2k::attention_win<DT, DH>), grid, dim3(256), 0, s, a);
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

/* How many workgroups share the keys of one sequence and key head. Up to 192 KB of keys and values one: what a CU reads in
 * about the time that the second kernel costs (one bf16 sequence over 8 key heads of 128: 375 tokens 6.9 us against 8.5
 * split, 750 9.5 against 8.3, 2000 17.2 against 8.7; 16 fp16 heads of 64: 750 tokens 6.7 us, 1000 7.7 against 7.0).
 * Above that one for every 4 blocks, a block for each wave (2000 tokens in parts of 11 blocks a wave: 12.3), as long as all
 * together are at most 512, two for each of 256 CUs (2 sequences of 131072: 100 us with 32 to 64 parts, 113 with 256; 32 of
 * 8192, 256 groups: 188 us in 2 parts or unsplit, 199 in 16); a number, as the workspace's size is asked for where there may
 * be no device. */
static int page_splits(const P2hKvCache *c, int n_seqs, int heads, int max_len, int window, int sinks)
{
    const int G = heads / c->heads, kb = c->dtype == P2H_F32 ? 16 : 32;
    const long long groups = (long long)n_seqs * c->heads * ((G + 15) / 16);
    const long long keys = p2k::imin(max_len, window) + (long long)p2k::imin(sinks, p2k::imax(max_len - window, 0));
    if (groups == 0 || 2 * keys * c->head_dim * (long long)elem_size(c->dtype) <= 192 << 10) return 1;
    const int n = p2k::imin((int)(512 / groups), (int)(keys / (4 * kb)));
    return n < 1 ? 1 : n;
}

static int check_paged(const char *name, const P2hKvCache *cache, int n_seqs, int heads, int max_len)
{
    if (int rc = check_cache(name, cache)) return rc;
    if (int rc = check_heads(name, cache->dtype, heads, cache->heads, cache->head_dim)) return rc;
    if (n_seqs < 0 || n_seqs > 65536 || max_len < 0 || max_len > (1 << 30))
        return fail(P2H_E_ARG, "%s: %d sequences (at most 65536) of up to %d tokens", name, n_seqs, max_len);
    return P2H_OK;
}

size_t p2h_attention_paged_workspace_bytes(const P2hKvCache *cache, int n_seqs, int heads, int max_len, int window,
                                           int sinks)
{
    const char *name = "p2h_attention_paged_workspace_bytes";
    if (check_paged(name, cache, n_seqs, heads, max_len) || check_scale(name, 1.0f, window, 0, sinks)) return 0;
    const int splits = page_splits(cache, n_seqs, heads, max_len, window, sinks);
    return splits > 1 ? (size_t)n_seqs * heads * splits * (cache->head_dim + 2) * 4 : 0;
}

int p2h_attention_paged(const P2hKvCache *cache, int n_seqs, int heads, const void *dQ, int ldq, const int *dTable,
                        int table_ld, const int *dLen, int max_len, float scale, int window, int sinks, void *dO, int ldo,
                        void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "p2h_attention_paged";
    if (int rc = check_paged(name, cache, n_seqs, heads, max_len)) return rc;
    if (int rc = check_scale(name, scale, window, 0, sinks)) return rc;
    if (table_ld < 0 || (long long)table_ld * cache->page > (1 << 30))
        return fail(P2H_E_ARG, "%s: table rows of %d pages of %d (at most 2^30 tokens)", name, table_ld, cache->page);
    if (n_seqs == 0) return P2H_OK;
    const int dtype = cache->dtype;
    if (int rc = check_rows(name, "dQ", dtype, dQ, ldq, heads * cache->head_dim)) return rc;
    if (int rc = check_rows(name, "dO", dtype, dO, ldo, heads * cache->head_dim)) return rc;
    if (!dLen || (table_ld > 0 && !dTable)) return fail(P2H_E_ARG, "%s: NULL lengths or page table", name);
    const size_t es = elem_size(dtype), w = (size_t)heads * cache->head_dim * es;
    if (overlap(Rows{(const char *)dO, ldo * es, w, n_seqs}, Rows{(const char *)dQ, ldq * es, w, n_seqs}))
        return fail(P2H_E_ARG, "%s: dO overlaps dQ", name);
    const Rows o{(const char *)dO, ldo * es, w, n_seqs};
    int splits = workspace ? page_splits(cache, n_seqs, heads, max_len, window, sinks) : 1;
    if (splits > 1) {
        const size_t need = (size_t)n_seqs * heads * splits * (cache->head_dim + 2) * 4;
        if (workspace_bytes < need || !aligned(workspace, 16))
            return fail(P2H_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", name, workspace_bytes,
                        need);
        const Rows ws{(const char *)workspace, need, need, 1};
        if (overlap(o, ws)) return fail(P2H_E_ARG, "%s: dO overlaps the workspace", name);
        /* it is written while other workgroups still read */
        if (overlap(ws, Rows{(const char *)dQ, ldq * es, w, n_seqs}) || overlap(ws, cache) ||
            overlap(ws, Rows{(const char *)dLen, 4, 4, n_seqs}) ||
            overlap(ws, Rows{(const char *)dTable, (size_t)table_ld * 4, (size_t)table_ld * 4, table_ld ? n_seqs : 0}))
            return fail(P2H_E_ARG, "%s: the workspace overlaps dQ, the cache, the lengths or the page table", name);
    }
    if (overlap(o, cache)) return fail(P2H_E_ARG, "%s: dO overlaps the cache", name);
    const int G = heads / cache->heads, q_groups = (G + 15) / 16;
    const long long grid = (long long)splits * cache->heads * q_groups * n_seqs;
    if ((size_t)grid * 512 >= kGridThreads || (size_t)n_seqs * heads * 512 >= kGridThreads)
        return fail(P2H_E_ARG, "%s: %d sequences of %d heads are too many for one call", name, n_seqs, heads);
    if (int rc = ensure_init()) return rc;
    p2k::PageArgs a{};
    a.n_seqs = n_seqs; a.heads = heads; a.kv = cache->heads; a.q_groups = q_groups; a.splits = splits;
    a.page_shift = log2_of(cache->page); a.pages = cache->pages; a.table_ld = table_ld; a.ldq = ldq; a.ldo = ldo;
    a.window = window; a.sinks = sinks; a.c = scale * p2k::kLog2e;
    a.q = dQ; a.kc = cache->K; a.vc = cache->V; a.table = dTable; a.len = dLen; a.o = dO; a.part = (float *)workspace;
    hipStream_t s = stream_of(stream);
    by_type_dim(dtype, cache->head_dim, [&](auto t, auto d) {
        constexpr int DT = decltype(t)::value, DH = decltype(d)::value;
        /* unsplit long sequences in 8 waves (64 of 4096 tokens: 184 us against 187; 16 of 1000: 20.4 against 21.9) */
        if (splits > 1 || max_len <= 128)
            hipLaunchKernelGGL((p2k::attention_page<DT, DH, 4>), dim3((unsigned)grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((p2k::attention_page<DT, DH, 8>), dim3((unsigned)grid), dim3(512), 0, s, a);
        if (splits > 1)
            hipLaunchKernelGGL((p2k::attention_join<DT, DH>), dim3((unsigned)(n_seqs * heads)),
                               dim3(64 * p2k::kJoinWaves), 0, s, a);
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

}  /* extern "C" */
