/*  p2hip_batch.hip – the device-pointer C ABI of a served batch's step (include/p2hip.h) over the kernels in
 *  p2hip_batch.h: an 8-bit cache read back and attended, prefixes shared by groups of sequences, adapters.
 *
 *  As in p2hip.hip every shape, stride and alignment that a kernel assumes is checked before its launch, the arguments
 *  before the device, so that a call is refused the same way with or without one.
 */
#include "p2hip_args.h"

#include "p2hip_batch.h"

using namespace p2host;

namespace {

constexpr int kWaves = 4;   /* of a workgroup of attend */

/* How the queries and keys of a call go over workgroups. */
struct Plan {
    int p_tiles = 0, p_parts = 0, q_groups = 1, o_parts = 1;
    bool tiled = false;   /* prefixes by tiles of p2k::kTileRows rows */
    int nq = 1;           /* else by 16 · nq */
    int parts() const { return p_parts + o_parts; }
    size_t prefix_workgroups(int kv) const { return (size_t)p_tiles * p_parts * kv; }
    size_t workgroups(int n_seqs, int kv) const { return prefix_workgroups(kv) + (size_t)n_seqs * q_groups * o_parts * kv; }
    size_t bytes(int n_seqs, int heads, int head_dim) const
    {
        return (size_t)n_seqs * heads * parts() * (head_dim + 2) * 4;   /* sums, reference, sum of weights */
    }
};

/* Keys over workgroups: one for every 4 blocks a wave, as long as all together are at most `workgroups`, two for each of 256
 * CUs (three groups of 8 sequences behind 30001 tokens, heads of 64, 8 bits: 36 us, 384 workgroups 43, 1024 40); a number, as the
 * workspace's size is asked for where there may be no device. */
int parts_of(long long groups, long long keys, int block, int workgroups = 512)
{
    const long long most = groups ? workgroups / groups : 1, n = keys / (4ll * block);
    return (int)(n < 1 || most < 1 ? 1 : n < most ? n : most);
}

int block_of(bool q8, int dtype) { return !q8 && dtype == P2H_F32 ? 16 : 32; }

/* the tokens of at most `n` that a window and first keys leave */
long long left_of(int n, int window, int sinks)
{
    return p2k::imin(n, window) + (long long)p2k::imin(sinks, p2k::imax(n - window, 0));
}

Plan paged_plan(const CacheView &c, int n_seqs, int heads, int max_len, int window, int sinks)
{
    Plan p;
    p.q_groups = (heads / c.heads + 15) / 16;
    const long long keys = left_of(max_len, window, sinks);
    /* below 5 · 128 tokens a wave's few blocks cost no more than joining parts (one sequence, 8 heads of 128, fp32: 375 tokens
     * 7.9 us against 9.8 and the second launch, 700 11.7 against 10.5); a block of heads of 64 is little to wait for: four workgroups a CU (8 sequences of 32768: 41 us
     * against 45) */
    if (keys >= 5 * 4 * 32)
        p.o_parts = parts_of((long long)n_seqs * c.heads * p.q_groups, keys, 32, c.head_dim == 64 ? 1024 : 512);
    return p;
}

Plan shared_plan(const CacheView &c, bool q8, int dtype, int n_seqs, int n_groups, int heads, int max_shared, int max_own,
                 int window, int sinks)
{
    Plan p;
    const int G = heads / c.heads, kb = block_of(q8, dtype);
    p.q_groups = (G + 15) / 16;
    const int rows = n_groups ? (n_seqs * G + n_groups - 1) / n_groups : 0;   /* of a group, as the host knows them */
    /* bf16 behind 32768 tokens, with the join: 40 rows 51 us by tiles, 53 by 16 rows, 64 rows 55 and 63, 32 rows 50 and 49. 8 bits,
     * three groups behind 30001: 20 rows 35 us by 32, 36 by 16, 32 rows 36 and 42, 16 rows 35 and 26. */
    p.tiled = !q8 && dtype != P2H_F32 && rows > 32;
    p.nq = q8 && rows > 16 ? 2 : 1;
    const int tr = p.tiled ? p2k::kTileRows : 16 * p.nq;
    p.p_tiles = n_seqs * G / tr + n_groups;
    p.p_parts = parts_of((long long)n_groups * ((rows + tr - 1) / tr) * c.heads, left_of(max_shared, window, sinks), kb);
    /* 512 workgroups for own keys of heads of 64 too, beside those of prefixes, where paged_plan takes 1024: three groups of 8 behind
     * 30001 tokens with up to 1000 of their own each 42.1 us, 1024 41.2; behind 3000 with up to 20000 123.6, 1024 98.7. The workspace grows
     * with the parts. */
    p.o_parts = parts_of((long long)n_seqs * c.heads * p.q_groups, left_of(max_own, window, sinks), kb);
    return p;
}

int check_seqs(const char *name, int dtype, const CacheView &c, int n_seqs, int heads, int table_ld)
{
    if (int rc = check_heads(name, dtype, heads, c.heads, c.head_dim)) return rc;
    if (n_seqs < 0 || n_seqs > 65536) return fail(P2H_E_ARG, "%s: %d sequences (at most 65536)", name, n_seqs);
    if (table_ld < 0 || (long long)table_ld * c.page > (1 << 30))
        return fail(P2H_E_ARG, "%s: table rows of %d pages of %d (at most 2^30 tokens)", name, table_ld, c.page);
    return P2H_OK;
}

/* before a plan is made: what its numbers of rows and workgroups stay within 32 bits for */
int check_batch(const char *name, int n_seqs, int heads)
{
    return (size_t)n_seqs * heads >= 1u << 23
               ? fail(P2H_E_ARG, "%s: %d sequences of %d heads are too many for one call", name, n_seqs, heads)
               : P2H_OK;
}

int check_plan(const char *name, const Plan &plan, const CacheView &c, int n_seqs, int n_groups, int heads)
{
    return plan.workgroups(n_seqs, c.heads) * 64 * kWaves >= kGridThreads
               ? fail(P2H_E_ARG, "%s: %d sequences of %d heads in %d groups are too many for one call", name, n_seqs, heads, n_groups)
               : P2H_OK;
}

int check_tokens(const char *name, int n)
{
    return n < 0 || n > (1 << 30) ? fail(P2H_E_ARG, "%s: up to %d tokens (0 .. 2^30)", name, n) : P2H_OK;
}

Rows ints(const int *p, int ld, int n) { return Rows{(const char *)p, (size_t)ld * 4, (size_t)ld * 4, ld > 0 && p ? n : 0}; }

/* Attention over a cache of either kind, its plan checked; `group` NULL without prefixes. */
int attention(const char *name, int dtype, const CacheView &c, bool q8, const Plan &plan, int n_seqs, int n_groups, int heads,
              const void *dQ, int ldq, const int *dGroup, const int *dShared, const int *dTable, int table_ld,
              const int *dLen, float scale, int window, int sinks, void *dO, int ldo, void *workspace,
              size_t workspace_bytes, void *stream)
{
    if (int rc = check_rows(name, "dQ", dtype, dQ, ldq, heads * c.head_dim)) return rc;
    if (int rc = check_rows(name, "dO", dtype, dO, ldo, heads * c.head_dim)) return rc;
    if (!dLen || (table_ld > 0 && !dTable)) return fail(P2H_E_ARG, "%s: NULL lengths or page table", name);
    if (!words(dLen, dTable, dGroup, dShared))
        return fail(P2H_E_ARG, "%s: lengths, pages or groups are not 4-byte aligned", name);
    const size_t es = elem_size(dtype), width = (size_t)heads * c.head_dim * es;
    const Rows q{(const char *)dQ, ldq * es, width, n_seqs}, o{(const char *)dO, ldo * es, width, n_seqs};
    if (overlap(o, q)) return fail(P2H_E_ARG, "%s: dO overlaps dQ", name);
    const bool parted = dGroup || plan.parts() > 1;
    if (parted) {
        const size_t need = plan.bytes(n_seqs, heads, c.head_dim);
        if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
            return fail(P2H_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", name, workspace_bytes,
                        need);
        const Rows ws{(const char *)workspace, need, need, 1};
        if (overlap(o, ws)) return fail(P2H_E_ARG, "%s: dO overlaps the workspace", name);
        /* it is written while other workgroups still read */
        if (overlap(ws, q) || overlap(ws, c) || overlap(ws, ints(dLen, 1, n_seqs)) ||
            overlap(ws, ints(dTable, table_ld, n_seqs)) || overlap(ws, ints(dGroup, 1, n_groups + 1)) ||
            overlap(ws, ints(dShared, 1, n_groups)))
            return fail(P2H_E_ARG, "%s: the workspace overlaps what the call reads", name);
    }
    if (overlap(o, c)) return fail(P2H_E_ARG, "%s: dO overlaps the cache", name);
    if (overlap(o, ints(dLen, 1, n_seqs)) || overlap(o, ints(dTable, table_ld, n_seqs)) ||
        overlap(o, ints(dGroup, 1, n_groups + 1)) || overlap(o, ints(dShared, 1, n_groups)))
        return fail(P2H_E_ARG, "%s: dO overlaps lengths, pages or groups", name);
    if (int rc = ensure_init()) return rc;
    p2k::BatchArgs a{};
    a.n_seqs = n_seqs; a.n_groups = n_groups; a.heads = heads; a.kv = c.heads; a.page_shift = log2_of(c.page);
    a.pages = c.pages; a.table_ld = table_ld; a.ldq = ldq; a.ldo = ldo; a.window = window; a.sinks = sinks;
    a.p_tiles = plan.p_tiles; a.p_parts = plan.p_parts; a.p_wgs = (int)plan.prefix_workgroups(c.heads);
    a.q_groups = plan.q_groups; a.o_parts = plan.o_parts; a.c = scale * p2k::kLog2e;
    a.q = dQ; a.kc = c.K; a.vc = c.V; a.ks = c.ks; a.vs = c.vs;
    a.table = dTable; a.len = dLen; a.group = dGroup; a.shared = dShared; a.o = dO;
    a.part = parted ? (float *)workspace : nullptr;
    a.stat = parted ? (float2 *)(a.part + (size_t)n_seqs * heads * plan.parts() * c.head_dim) : nullptr;
    hipStream_t s = stream_of(stream);
    by_type_dim(dtype, c.head_dim, [&](auto t, auto d) {
        constexpr int DT = decltype(t)::value, DH = decltype(d)::value;
        const dim3 grid((unsigned)plan.workgroups(n_seqs, c.heads)), threads(64 * kWaves);
        if (q8) {
            if (plan.nq == 2) hipLaunchKernelGGL((p2k::attend<p2k::C_Q8, DT, DH, 2, kWaves>), grid, threads, 0, s, a);
            else hipLaunchKernelGGL((p2k::attend<p2k::C_Q8, DT, DH, 1, kWaves>), grid, threads, 0, s, a);
        } else if (!plan.tiled) {
            hipLaunchKernelGGL((p2k::attend<p2k::C_ROWS, DT, DH, 1, kWaves>), grid, threads, 0, s, a);
        } else {
            if constexpr (DT != p2k::T_F32) hipLaunchKernelGGL((p2k::attend_tiles<DT, DH>), grid, threads, 0, s, a);
        }
        if (parted)
            hipLaunchKernelGGL((p2k::attend_join<DT, DH>), dim3((unsigned)(((size_t)n_seqs * heads + 3) / 4)), dim3(256), 0, s, a);
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

size_t shared_bytes(const char *name, const P2hKvCache *rows, const P2hKvCacheQ8 *q8, int n_seqs, int n_groups, int heads,
                    int max_shared, int max_own, int window, int sinks)
{
    if (rows ? check_cache(name, rows) : check_cache(name, q8)) return 0;
    const CacheView c(rows, q8);
    const int dtype = rows ? rows->dtype : P2H_BF16;
    if (check_seqs(name, dtype, c, n_seqs, heads, 0) || check_batch(name, n_seqs, heads) ||
        check_scale(name, 1.0f, window, 0, sinks) || check_tokens(name, max_shared) || check_tokens(name, max_own))
        return 0;
    if (n_groups < 0 || n_groups > 65536) {
        fail(P2H_E_ARG, "%s: %d groups (at most 65536)", name, n_groups);
        return 0;
    }
    const Plan plan = shared_plan(c, q8 != nullptr, dtype, n_seqs, n_groups, heads, max_shared, max_own, window, sinks);
    return check_plan(name, plan, c, n_seqs, n_groups, heads) ? 0 : plan.bytes(n_seqs, heads, c.head_dim);
}

int shared(const char *name, int dtype, const P2hKvCache *rows, const P2hKvCacheQ8 *q8, int n_seqs, int n_groups, int heads,
           const void *dQ, int ldq, const int *dGroup, const int *dShared, const int *dTable, int table_ld, const int *dLen,
           int max_shared, int max_own, float scale, int window, int sinks, void *dO, int ldo, void *workspace,
           size_t workspace_bytes, void *stream)
{
    if (int rc = rows ? check_cache(name, rows) : check_cache(name, q8)) return rc;
    const CacheView c(rows, q8);
    if (int rc = check_seqs(name, dtype, c, n_seqs, heads, table_ld)) return rc;
    if (int rc = check_batch(name, n_seqs, heads)) return rc;
    if (int rc = check_scale(name, scale, window, 0, sinks)) return rc;
    if (int rc = check_tokens(name, max_shared)) return rc;
    if (int rc = check_tokens(name, max_own)) return rc;
    if (n_groups < 0 || n_groups > 65536) return fail(P2H_E_ARG, "%s: %d groups (at most 65536)", name, n_groups);
    if (n_seqs == 0 || n_groups == 0) return P2H_OK;
    if (!dGroup || !dShared) return fail(P2H_E_ARG, "%s: NULL groups or prefixes", name);
    const Plan plan = shared_plan(c, q8 != nullptr, dtype, n_seqs, n_groups, heads, max_shared, max_own, window, sinks);
    if (int rc = check_plan(name, plan, c, n_seqs, n_groups, heads)) return rc;
    return attention(name, dtype, c, q8 != nullptr, plan, n_seqs, n_groups, heads, dQ, ldq, dGroup, dShared, dTable, table_ld,
                     dLen, scale, window, sinks, dO, ldo, workspace, workspace_bytes, stream);
}

}  // namespace

extern "C" {

/* ── the 8-bit cache ───────────────────────────────────────────────────────────────────────────────────────── */

int p2h_kv_rows_q8(int dtype, const P2hKvCacheQ8 *cache, int rows, int n_seqs, const int *dStart, const int *dTable,
                   int table_ld, void *dK, int ldk, void *dV, int ldv, void *stream)
{
    const char *name = "p2h_kv_rows_q8";
    if (int rc = check_cache(name, cache)) return rc;
    const CacheView c(nullptr, cache);
    if (int rc = check_seqs(name, dtype, c, n_seqs, c.heads, table_ld)) return rc;
    if (rows < 0 || rows >= 1 << 30) return fail(P2H_E_ARG, "%s: %d rows (below 2^30)", name, rows);
    if (rows == 0 || n_seqs == 0) return P2H_OK;
    const int width = c.heads * c.head_dim;
    if (int rc = check_rows(name, "dK", dtype, dK, ldk, width)) return rc;
    if (int rc = check_rows(name, "dV", dtype, dV, ldv, width)) return rc;
    if (!dStart || (table_ld > 0 && !dTable)) return fail(P2H_E_ARG, "%s: NULL starts or page table", name);
    if (!words(dStart, dTable)) return fail(P2H_E_ARG, "%s: starts or pages are not 4-byte aligned", name);
    const size_t es = elem_size(dtype);
    const Rows k{(const char *)dK, ldk * es, width * es, rows}, v{(const char *)dV, ldv * es, width * es, rows};
    if (overlap(k, v)) return fail(P2H_E_ARG, "%s: dK and dV overlap", name);
    if (overlap(k, c) || overlap(v, c)) return fail(P2H_E_ARG, "%s: dK or dV overlaps the cache", name);
    for (const Rows &r : {ints(dStart, 1, n_seqs + 1), ints(dTable, table_ld, n_seqs)})
        if (overlap(k, r) || overlap(v, r)) return fail(P2H_E_ARG, "%s: dK or dV overlaps starts or pages", name);
    if (int rc = ensure_init()) return rc;
    p2k::KvRowsArgs a{};
    a.rows = rows; a.n_seqs = n_seqs; a.kv = c.heads; a.page_shift = log2_of(c.page); a.pages = c.pages;
    a.table_ld = table_ld; a.ldk = ldk; a.ldv = ldv;
    a.start = dStart; a.table = dTable; a.kc = (const int8_t *)c.K; a.vc = (const int8_t *)c.V; a.ks = c.ks; a.vs = c.vs;
    a.k = dK; a.v = dV;
    /* Rows a workgroup: what a lane writes in one go (13 ragged sequences of up to 8191 tokens, 8 heads of 128, bf16: 84 us;
     * twice that 90, four times 93), fewer for fewer rows, so that each CU has some. */
    const int units = width * 2 / (int)(16 / es);
    a.per = p2k::imax(p2k::imin(p2k::imin(256 * p2k::kRowUnits / units, rows / 1024), p2k::kRowsMost), 1);
    const unsigned wgs = (unsigned)((rows - 1) / a.per + 1), across = wgs < 1u << 23 ? wgs : 1u << 23;
    const dim3 grid(across, (wgs - 1) / across + 1);
    hipStream_t s = stream_of(stream);
    by_type_dim(dtype, c.head_dim, [&](auto t, auto d) {
        hipLaunchKernelGGL((p2k::kv_rows_q8<decltype(t)::value, decltype(d)::value>), grid, dim3(256), 0, s, a);
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

size_t p2h_attention_paged_q8_workspace_bytes(const P2hKvCacheQ8 *cache, int n_seqs, int heads, int max_len, int window,
                                              int sinks)
{
    const char *name = "p2h_attention_paged_q8_workspace_bytes";
    if (check_cache(name, cache)) return 0;
    const CacheView c(nullptr, cache);
    if (check_seqs(name, P2H_BF16, c, n_seqs, heads, 0) || check_batch(name, n_seqs, heads) ||
        check_scale(name, 1.0f, window, 0, sinks) || check_tokens(name, max_len))
        return 0;
    const Plan p = paged_plan(c, n_seqs, heads, max_len, window, sinks);
    return p.parts() > 1 && !check_plan(name, p, c, n_seqs, 0, heads) ? p.bytes(n_seqs, heads, c.head_dim) : 0;
}

int p2h_attention_paged_q8(int dtype, const P2hKvCacheQ8 *cache, int n_seqs, int heads, const void *dQ, int ldq,
                           const int *dTable, int table_ld, const int *dLen, int max_len, float scale, int window,
                           int sinks, void *dO, int ldo, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "p2h_attention_paged_q8";
    if (int rc = check_cache(name, cache)) return rc;
    const CacheView c(nullptr, cache);
    if (int rc = check_seqs(name, dtype, c, n_seqs, heads, table_ld)) return rc;
    if (int rc = check_batch(name, n_seqs, heads)) return rc;
    if (int rc = check_scale(name, scale, window, 0, sinks)) return rc;
    if (int rc = check_tokens(name, max_len)) return rc;
    if (n_seqs == 0) return P2H_OK;
    Plan plan = paged_plan(c, n_seqs, heads, max_len, window, sinks);
    if (!workspace) plan.o_parts = 1;
    if (int rc = check_plan(name, plan, c, n_seqs, 0, heads)) return rc;
    return attention(name, dtype, c, true, plan, n_seqs, 0, heads, dQ, ldq, nullptr, nullptr, dTable, table_ld, dLen, scale,
                     window, sinks, dO, ldo, workspace, workspace_bytes, stream);
}

/* ── shared prefixes ───────────────────────────────────────────────────────────────────────────────────────── */

size_t p2h_attention_shared_workspace_bytes(const P2hKvCache *cache, int n_seqs, int n_groups, int heads, int max_shared,
                                            int max_own, int window, int sinks)
{
    const char *name = "p2h_attention_shared_workspace_bytes";
    if (!cache) return fail(P2H_E_ARG, "%s: NULL cache", name), 0;
    return shared_bytes(name, cache, nullptr, n_seqs, n_groups, heads, max_shared, max_own, window, sinks);
}

int p2h_attention_shared(const P2hKvCache *cache, int n_seqs, int n_groups, int heads, const void *dQ, int ldq,
                         const int *dGroup, const int *dShared, const int *dTable, int table_ld, const int *dLen,
                         int max_shared, int max_own, float scale, int window, int sinks, void *dO, int ldo,
                         void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "p2h_attention_shared";
    if (!cache) return fail(P2H_E_ARG, "%s: NULL cache", name);
    return shared(name, cache->dtype, cache, nullptr, n_seqs, n_groups, heads, dQ, ldq, dGroup, dShared, dTable, table_ld,
                  dLen, max_shared, max_own, scale, window, sinks, dO, ldo, workspace, workspace_bytes, stream);
}

size_t p2h_attention_shared_q8_workspace_bytes(const P2hKvCacheQ8 *cache, int n_seqs, int n_groups, int heads,
                                               int max_shared, int max_own, int window, int sinks)
{
    return shared_bytes("p2h_attention_shared_q8_workspace_bytes", nullptr, cache, n_seqs, n_groups, heads, max_shared,
                        max_own, window, sinks);
}

int p2h_attention_shared_q8(int dtype, const P2hKvCacheQ8 *cache, int n_seqs, int n_groups, int heads, const void *dQ,
                            int ldq, const int *dGroup, const int *dShared, const int *dTable, int table_ld,
                            const int *dLen, int max_shared, int max_own, float scale, int window, int sinks, void *dO,
                            int ldo, void *workspace, size_t workspace_bytes, void *stream)
{
    return shared("p2h_attention_shared_q8", dtype, nullptr, cache, n_seqs, n_groups, heads, dQ, ldq, dGroup, dShared, dTable,
                  table_ld, dLen, max_shared, max_own, scale, window, sinks, dO, ldo, workspace, workspace_bytes, stream);
}

/* ── adapters ──────────────────────────────────────────────────────────────────────────────────────────────── */

static int check_adapters(const char *name, const P2hAdapters *ad, int M)
{
    if (!ad) return fail(P2H_E_ARG, "%s: NULL adapters", name);
    if (!is_type(ad->dtype)) return fail(P2H_E_ARG, "%s: element type %d", name, ad->dtype);
    if (ad->rank != 8 && ad->rank != 16 && ad->rank != 32 && ad->rank != 64 && ad->rank != 128)
        return fail(P2H_E_ARG, "%s: rank = %d (8, 16, 32, 64 or 128)", name, ad->rank);
    if (ad->count < 0 || ad->K < 1 || ad->N < 1 || ad->K > (1 << 23) || ad->N > (1 << 23))
        return fail(P2H_E_ARG, "%s: %d adapters of [%d, %d]", name, ad->count, ad->K, ad->N);
    if (M < 0 || M > 16 * 65535) return fail(P2H_E_ARG, "%s: M = %d (at most %d rows)", name, M, 16 * 65535);
    return P2H_OK;
}

/* Adapters that 16 rows may have between them, as the host knows it */
static int adapters_of_16(const P2hAdapters *ad, int M) { return p2k::imin(p2k::imin(M, 16), p2k::imax(ad->count, 1)); }

/* Above kManyRows rows a workgroup of the second product takes 64 rows, not 16 (bf16, K = 4096, rank 16, shrink and expand:
 * 300 rows of 20 an adapter with N = 16384 30 -> 22 us, N = 16389 37 -> 27, 400 rows of one 96 -> 78; but 200 of 20 21 -> 17 too; 128
 * rows of as many adapters 35 -> 42), above kManyShrink one of the first too (both, N = 4096: 6000 fp32 rows, K = 1024, rank 32 65 ->
 * 63 us, 3000 of 375 an adapter, bf16, K = 4096, 30 -> 27.5, 1200 of 20 26.9 either way; but 600 18.8 -> 20.3, fp32 600 17.8 -> 19.1, 1200
 * 22 -> 24.6; 400 15.7 -> 17.8). */
constexpr int kManyRows = 256, kManyShrink = 512;

/* K over workgroups, 0: everything in one launch, each workgroup making H for itself, while that is little to read (one row,
 * 16-bit, rank 8, K = 1024, 16 KB: 4.2 us against 2.6 + 3.4; 128 KB: 7.8 against 3.0 + 3.7, N = 16389 12.4 against 8). A part has
 * at least 128 dimensions, 256 where a wave has few rows' adapters: the second product adds the parts (one row, rank 64, K =
 * 2048: 3.2 + 9.1 us with 128, 4.0 + 6.9 with 256), and there are at most 16 (bf16, rank 16, N = 16389, both products: 32 rows, K =
 * 4096 20.5 us, with 8 23.3, with 32 21.0; 64 rows 29.2, 31.8, 31.8; 17 rows, K = 8192 20.1, 27.2, 17.9; one row of rank 64, K = 8192 13.4, 12.8,
 * 17.5). Above kManyShrink all together are at most 768, three a CU (6000 bf16 rows, K = 4096 48.7 us, 384 49.6, 1536 52.7; 600 and
 * 1200 rows and K = 1024 the same with each). A number, as the workspace's size is asked for where there may be no device. */
static int adapter_parts(const P2hAdapters *ad, int M)
{
    const int n = adapters_of_16(ad, M), tiles = (M - 1) / (M > kManyShrink ? 64 : 16) + 1;
    if (M <= 16 && (size_t)n * ad->rank * ad->K * elem_size(ad->dtype) <= 64 << 10) return 0;
    const int least = n <= 2 && M <= kManyShrink ? 256 : 128, want = M > kManyShrink ? 768 / tiles : (256 + tiles - 1) / tiles;
    return p2k::imax(p2k::imin(p2k::imin(want, 16), ad->K / least), 1);
}

size_t p2h_adapters_workspace_bytes(const P2hAdapters *ad, int M)
{
    if (check_adapters("p2h_adapters_workspace_bytes", ad, M) || M == 0) return 0;
    return (size_t)adapter_parts(ad, M) * M * ad->rank * 4;
}

int p2h_adapters_add(const P2hAdapters *ad, int M, const void *dX, int ldx, const int *dIndex, const void *dZ, int ldz,
                     void *dY, int ldy, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *name = "p2h_adapters_add";
    if (int rc = check_adapters(name, ad, M)) return rc;
    if (M == 0) return P2H_OK;
    const int K = ad->K, N = ad->N;
    const size_t es = elem_size(ad->dtype);
    if (!dX || !dY || ldx < K || ldy < N || (dZ && ldz < N) || !aligned(dX, es) || !aligned(dY, es) || !aligned(dZ, es))
        return fail(P2H_E_ARG, "%s: NULL or unaligned rows, or ldx = %d < K = %d, ldz = %d or ldy = %d < N = %d", name, ldx, K,
                    ldz, ldy, N);
    if (!dIndex || !words(dIndex)) return fail(P2H_E_ARG, "%s: NULL index, or not 4-byte aligned", name);
    if (ad->count > 0 && (!ad->A || !ad->B || !ad->scale || !aligned(ad->A, 16) || !aligned(ad->B, 16) || !words(ad->scale)))
        return fail(P2H_E_ARG, "%s: adapters are NULL or not 16-byte aligned (scales 4-byte)", name);
    const size_t need = p2h_adapters_workspace_bytes(ad, M);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(P2H_E_WORKSPACE, "%s: workspace of %zu bytes, %zu needed, 16-byte aligned", name, workspace_bytes, need);
    const Rows x{(const char *)dX, ldx * es, K * es, M}, y{(const char *)dY, ldy * es, N * es, M};
    const Rows z{(const char *)dZ, ldz * es, N * es, dZ ? M : 0}, ws{(const char *)workspace, need, need, need ? 1 : 0};
    const size_t a_bytes = (size_t)ad->count * ad->rank * K * es, b_bytes = (size_t)ad->count * ad->rank * N * es;
    const Rows am{(const char *)ad->A, a_bytes, a_bytes, a_bytes ? 1 : 0}, bm{(const char *)ad->B, b_bytes, b_bytes, b_bytes ? 1 : 0};
    const Rows sc{(const char *)ad->scale, (size_t)ad->count * 4, (size_t)ad->count * 4, ad->count ? 1 : 0};
    const bool in_place = dZ == dY && (ldz == ldy || M == 1);
    if (!in_place && overlap(y, z)) return fail(P2H_E_ARG, "%s: dY overlaps dZ other than in place", name);
    for (const Rows &r : {x, am, bm, sc, ints(dIndex, 1, M)})
        if (overlap(y, r) || overlap(ws, r)) return fail(P2H_E_ARG, "%s: dY or the workspace overlaps what the call reads", name);
    if (overlap(ws, y) || overlap(ws, z)) return fail(P2H_E_ARG, "%s: the workspace overlaps dY or dZ", name);
    if (int rc = ensure_init()) return rc;
    p2k::AdapterArgs a{};
    a.M = M; a.N = N; a.K = K; a.count = ad->count; a.ldx = ldx; a.ldz = ldz; a.ldy = ldy;
    a.parts = adapter_parts(ad, M);
    if (a.parts) a.chunk = ((K - 1) / a.parts / 128 + 1) * 128;
    a.x = dX; a.z = dZ; a.a = ad->A; a.b = ad->B; a.scale = ad->scale; a.index = dIndex; a.y = dY; a.h = (float *)workspace;
    const bool vec = aligned(dX, 16) && (M == 1 || ldx * es % 16 == 0) && K * es % 16 == 0;
    a.vec = aligned(dY, 16) && (M == 1 || ldy * es % 16 == 0) && (!dZ || (aligned(dZ, 16) && (M == 1 || ldz * es % 16 == 0)));
    const unsigned tiles = (unsigned)((M + 15) / 16), columns = (unsigned)((N - 1) / 64 + 1);
    /* of many rows, columns a workgroup: as many workgroups as three a CU (16-bit rows: four), so that they begin and end
     * together (both products, half as many, as many, twice as many: 6000 fp32 rows, K = 1024, N = 4096 77, 63, 64.5 us, 600 18.4, 19.2,
     * 19.3; bf16, K = 4096, 300 rows, N = 16384 24.7, 21.7, 20.9, 1200 57.6, 48.3, 48.9, 6000, N = 4096 53.3, 48.7, 45.8) */
    const unsigned slots = es == 4 ? 768 : 1024, groups = (tiles + 3) / 4 < slots ? slots / ((tiles + 3) / 4) : 1;
    a.units = (int)((columns + groups - 1) / groups);
    hipStream_t s = stream_of(stream);
    by_type(ad->dtype, [&](auto t) {
        auto go = [&](auto rank) {
            constexpr int DT = decltype(t)::value, R = decltype(rank)::value, NS = R <= 32 ? 16 : 8,   /* waves that registers allow */
                          NF = R == 128 && DT == P2H_F32 ? 4 : 8;
            auto aligned_x = [&](auto v) {
                constexpr bool V = decltype(v)::value != 0;
                if (!a.parts)
                    hipLaunchKernelGGL((p2k::adapter_expand<DT, R, NF, true, V>), dim3(columns, tiles), dim3(64 * NF), 0, s, a);
                else if (V && M > kManyShrink)
                    hipLaunchKernelGGL((p2k::adapter_shrink_rows<DT, R>), dim3((tiles + 3) / 4, (unsigned)a.parts), dim3(256), 0, s, a);
                else
                    hipLaunchKernelGGL((p2k::adapter_shrink<DT, R, NS, V>), dim3(tiles, (unsigned)a.parts), dim3(64 * NS), 0, s, a);
            };
            if (vec) aligned_x(ic<1>{});
            else aligned_x(ic<0>{});
            if (!a.parts) return;
            const dim3 many((columns + a.units - 1) / a.units, (tiles + 3) / 4);
            if (M > kManyRows && ad->count > 0 && a.vec && N >= 64 && p2k::sixteen_rows_in_32_bits(ldy, (int)es))   /* its stores' offsets */
                hipLaunchKernelGGL((p2k::adapter_expand_rows<DT, R, true>), many, dim3(256), 0, s, a);
            else if (M > kManyRows && ad->count > 0)
                hipLaunchKernelGGL((p2k::adapter_expand_rows<DT, R, false>), many, dim3(256), 0, s, a);
            else
                hipLaunchKernelGGL((p2k::adapter_expand<DT, R, 8, false, true>), dim3(columns, tiles), dim3(512), 0, s, a);
        };
        switch (ad->rank) {
        case 8: go(ic<8>{}); break;
        case 16: go(ic<16>{}); break;
        case 32: go(ic<32>{}); break;
        case 64: go(ic<64>{}); break;
        default: go(ic<128>{}); break;
        }
    });
    HIPCHK(hipGetLastError());
    return P2H_OK;
}

}  /* extern "C" */
