/*  p2hip_batch.h – gfx950 kernels of a served batch's step (included once, by p2hip_batch.hip).
 *
 *  Kernels:
 *    kv_rows_q8           kept 8-bit keys and values back as rows
 *    attend               one query per sequence over pages: prefixes of groups of sequences, read once for 16 query rows (8-bit
 *                         codes: 16 or 32), and what each sequence has alone
 *    attend_tiles         the same of 16-bit rows, prefixes read once for 128 query rows
 *    attend_join          adds the parts of each query
 *    adapter_shrink       rows times the first matrix of their adapters, 16 rows a workgroup
 *    adapter_shrink_rows  the same of many aligned rows, 64 a workgroup
 *    adapter_expand       that times the second, added to the rows of the projection beside it, 16 rows a workgroup; of few rows of
 *                         small adapters with the first product too
 *    adapter_expand_rows  the same of many rows, 64 a workgroup
 */
#pragma once

#include "p2hip_async.h"
#include "p2hip_elem.h"
#include "p2hip_few.h"
#include "p2hip_index.h"

namespace p2k {

/* a word that is the same for all lanes, read through the scalar cache: vector loads would be waited for together with the
 * direct loads into LDS that are on their way */
__device__ __forceinline__ int scalar_int(const int *p)
{
    typedef __attribute__((address_space(4))) const int *c4;
    return *(c4)(uintptr_t)p;
}

/* The last s of [0, n) with le(s), which holds up to some s and not behind it; −1 where it holds for none. 64 lanes look at
 * once, so that up to 64 take one wait for memory and 4096 two. */
template <class F> __device__ __forceinline__ int wave_last(int n, F le)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n;
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) / 64, s = lo + lane * step;
        const int k = __popcll(__ballot(s < hi && le(s)));
        lo += imax(k - 1, 0) * step;
        hi = imin(lo + step, hi);
    }
    return lo + __popcll(__ballot(lo + lane < hi && le(lo + lane))) - 1;
}

/* ── an 8-bit cache read back ──────────────────────────────────────────────────────────────────────────────── */

struct KvRowsArgs {
    int rows, n_seqs, kv, page_shift, pages, table_ld, ldk, ldv, per;   /* per: rows a workgroup */
    const int *start, *table;
    const int8_t *kc, *vc;
    const float *ks, *vs;
    void *k, *v;
};

constexpr int kRowsMost = 32;   /* rows a workgroup at most */
constexpr int kRowUnits = 4;    /* units of 16 output bytes of a lane, all read before the first is written */

/* k = code · scale, rounded once. Rows `per` times the workgroup's number ..: where each row's token lies is looked up first, one thread a row;
 * then 16 bytes of output a lane along the rows, K's heads and V's. A unit's row and its place there are carried on: a division
 * for each cost as much as the rest. Bound by memory: 13 ragged sequences of up to 8191 tokens, 8 heads of 128, to bf16, 458 MB:
 * 84 us, 5.4 TB/s (ordinary stores 93; a grid of 2048 with its rows in loops 113). */
template <int DT, int DH>
__global__ __launch_bounds__(256) void kv_rows_q8(KvRowsArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int VE = kPer16<DT>, LPH = DH / VE;
    __shared__ long long at[kRowsMost];   /* (page · kv << page_shift) + place; −1: no such token; −2: no sequence's row */
    const int r0 = (int)(blockIdx.y * gridDim.x + blockIdx.x) * a.per, n = imin(a.per, a.rows - r0);
    if (n <= 0) return;   /* of the last of several rows of workgroups */
    if (threadIdx.x < 64) {
        auto begins = [&](int s) { return imin(imax(a.start[s], 0), a.rows); };
        const int first = wave_last(a.n_seqs, [&](int s) { return begins(s) <= r0; });
        const int last = wave_last(a.n_seqs, [&](int s) { return begins(s) <= r0 + n - 1; });
        const int r = r0 + (int)threadIdx.x;
        if (r < r0 + n) {
            int s = first, end = last + 1;   /* the last sequence that begins at or before r is one of these */
            while (end - s > 1) {
                const int mid = (s + end) / 2;
                if (begins(mid) <= r) s = mid;
                else end = mid;
            }
            int qa = 0, qb = 0;
            if (s >= 0) seq_rows(a.start, s, a.rows, &qa, &qb);
            long long to = -2;
            if (r < qb) {
                const int t = r - qa;
                const int page = page_in(page_entry(a.table + (size_t)s * a.table_ld, a.table_ld, t, a.page_shift), a.pages);
                to = page < 0 ? -1 : (((long long)page * a.kv) << a.page_shift) + (t & ((1 << a.page_shift) - 1));
            }
            at[threadIdx.x] = to;
        }
    }
    __syncthreads();
    constexpr int U = kRowUnits;
    const int per_row = 2 * a.kv * LPH, step_i = 256 / per_row, step_p = 256 - step_i * per_row;
    int i = (int)threadIdx.x / per_row, p = (int)threadIdx.x - i * per_row;
    while (i < n) {
        uint32_t w[U][VE / 4];
        float s[U];
        E *row[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const long long token = i < n ? at[i] : -2;
            const int is_v = p >= a.kv * LPH, q = is_v ? p - a.kv * LPH : p, h = q / LPH, l = q % LPH;
            row[k] = token < -1 ? nullptr
                                : static_cast<E *>(is_v ? a.v : a.k) + (size_t)(r0 + i) * (is_v ? a.ldv : a.ldk) + (size_t)h * DH + VE * l;
            s[k] = 0.0f;
#pragma unroll
            for (int j = 0; j < VE / 4; j++) w[k][j] = 0;
            if (token >= 0) {
                const size_t head = (size_t)token + ((size_t)h << a.page_shift);
                s[k] = (is_v ? a.vs : a.ks)[head];
                __builtin_memcpy(w[k], (is_v ? a.vc : a.kc) + head * DH + VE * l, VE);
            }
            p += step_p, i += step_i;
            if (p >= per_row) p -= per_row, i++;
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            float v[VE];
#pragma unroll
            for (int j = 0; j < VE; j++) v[j] = (float)(int8_t)(w[k][j / 4] >> (8 * (j % 4))) * s[k];
            if (row[k]) __builtin_nontemporal_store(pack<DT>(v), reinterpret_cast<u4 *>(row[k]));
        }
    }
}

/* ── one query per sequence over pages ─────────────────────────────────────────────────────────────────────── */

enum { C_ROWS = 0, C_Q8 = 1 };   /* a cache of rows, of codes */

struct BatchArgs {
    int n_seqs, n_groups, heads, kv, page_shift, pages, table_ld, ldq, ldo, window, sinks;
    int p_tiles, p_parts, p_wgs;   /* of prefixes: tiles of query rows, parts of the keys, workgroups, first in the grid */
    int q_groups, o_parts;         /* of what each sequence has alone: tiles of a key head's queries, parts */
    float c;                       /* scale · log2 e */
    const void *q, *kc, *vc;
    const float *ks, *vs;
    const int *table, *len, *group, *shared;   /* group: NULL without prefixes */
    void *o;
    /* of each part the weighted sums, [sequence][head][p_parts + o_parts][DH], and their reference and the sum of weights; NULL:
     * one part, straight to o */
    float *part;
    float2 *stat;
};

/* A block of 32 keys' codes as it lies in a wave's LDS: rows of CH pieces of 16 bytes, brought by LD direct loads of RPL rows
 * each, and their scales. Pieces are moved within a row so that operand reads fall into different banks: k_place for one piece
 * of 16 keys, v_place for 64 bytes of 4 keys. */
template <int DH> struct CodeBlock {
    static constexpr int KB = 32, CH = DH / 16, RPL = 64 / CH, LD = KB / RPL, BYTES = KB * DH, STAGE = 2 * BYTES + 256,
                         LOADS = 2 * LD + 1,
                         STAGES = 2;   /* in a wave's LDS; three bring nothing (heads of 128: one workgroup a CU, 77 -> 105 us) */
    static __device__ __forceinline__ constexpr int k_place(int r, int p) { return p ^ ((r / (16 / CH)) & (CH - 1)); }
    static __device__ __forceinline__ constexpr int v_place(int r, int p) { return CH == 8 ? p ^ (4 * ((r >> 1) & 1)) : p; }
    /* the key of a block that product t has in row m: a lane's results are rows 4g + i, its four groups of lanes having
     * neighbouring keys */
    static __device__ __forceinline__ constexpr int key_of(int t, int m) { return 16 * t + 4 * (m & 3) + (m >> 2); }
};

/* the upper halves of two floats, of a in the lower half */
__device__ __forceinline__ uint32_t upper_halves(float a, float b)
{
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

/* byte j of w, a code, as a float */
template <int J> __device__ __forceinline__ float code_at(uint32_t w) { return (float)(int8_t)(w >> (8 * J)); }

/* eight codes as an operand of the 16-bit type; whole numbers up to 127 are exact in both */
template <int DT> __device__ __forceinline__ u4 code_operand(uint32_t w0, uint32_t w1)
{
    u4 v;
    auto two = [](float a, float b) {
        if constexpr (DT == T_F16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
        else return upper_halves(a, b);
    };
    v[0] = two(code_at<0>(w0), code_at<1>(w0));
    v[1] = two(code_at<2>(w0), code_at<3>(w0));
    v[2] = two(code_at<0>(w1), code_at<1>(w1));
    v[3] = two(code_at<2>(w1), code_at<3>(w1));
    return v;
}

/* Eight floats as NP bf16 operands that sum to them: the upper 16 bits of what is left after the ones before; of one or two
 * the last is rounded. */
template <int NP> __device__ __forceinline__ void bf16_pieces(const float (&x)[8], u4 (&p)[NP])
{
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = x[i];
#pragma unroll
    for (int n = 0; n < NP; n++) {
        if (n == NP - 1 && NP < 3) {
            p[n] = pack<T_BF16>(v);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) p[n][i] = upper_halves(v[2 * i], v[2 * i + 1]);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] -= __uint_as_float(__float_as_uint(v[i]) & 0xffff0000u);
        }
    }
}

/* What one workgroup takes: `rows` query rows from number r0 on, of the sequences from seq0 on, row r being query head kvh · G
 * + r % G of sequence seq0 + r / G; of the keys [t0, t1) that the table row `pages` names, part `split` of `splits`. Its
 * result is part `slot` of `parts`. */
struct BatchItem {
    int seq0, r0, rows, kvh, t0, t1, split, splits, slot, parts;
    const int *pages;
};

/* its rows' lengths: this lane's (row lane % 16 of every 16), and of all of them the least and the largest */
template <int NQ> struct RowLengths {
    int of[NQ], least, most;
    __device__ __forceinline__ RowLengths(const BatchArgs &a, const BatchItem &w)
    {
        const int G = a.heads / a.kv;
        least = 1 << 30;
        most = 0;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const int r = w.r0 + imin(16 * n + (int)(threadIdx.x & 15), w.rows - 1);
            of[n] = a.pages ? kept_length(a.len[w.seq0 + r / G], a.table_ld, 1 << a.page_shift) : 0;
            least = imin(least, of[n]);
            most = imax(most, of[n]);
        }
        if (w.r0 / G != (w.r0 + w.rows - 1) / G) {   /* more than one sequence */
#pragma unroll
            for (int o = 1; o < 16; o *= 2) {
                least = imin(least, __shfl_xor(least, o));
                most = imax(most, __shfl_xor(most, o));
            }
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
    }
};

/* The item's blocks of KB keys: those that a row of lengths least .. most sees something of, counted from the block that t0
 * lies in, and the part [b0, b1) of them. */
struct ItemBlocks {
    int tb, end_key, b0, b1;
    KeyBlocks blocks;
    __device__ __forceinline__ ItemBlocks(const BatchArgs &a, const BatchItem &w, int least, int most, int kb)
    {
        tb = w.t0 & ~(kb - 1);
        end_key = imin(most, w.t1);
        blocks = key_blocks(imax(least - a.window, w.t0) - tb, end_key - tb, imax(a.sinks - tb, 0), kb);
        split_range(blocks.total, w.splits, w.split, &b0, &b1);
    }
    __device__ __forceinline__ int key(int b, int kb) const { return tb + blocks.at(b) * kb; }
};

/* whether a row of that length sees a key, if a page holds it */
__device__ __forceinline__ bool item_sees(const BatchArgs &a, const BatchItem &w, int key, int len)
{
    return (key >= w.t0) & (key < imin(len, w.t1)) & ((key >= len - a.window) | (key < a.sinks));
}
/* whether rows of lengths least .. most see all n keys from k0 on */
__device__ __forceinline__ bool item_sees_all(const BatchArgs &a, const BatchItem &w, int k0, int n, int least, int most)
{
    return k0 >= w.t0 && k0 + n <= imin(least, w.t1) && (k0 >= most - a.window || k0 + n <= a.sinks);
}

/* the place of a token of this item's key head among all heads' tokens, in a page that is there */
__device__ __forceinline__ size_t token_at(const BatchArgs &a, const BatchItem &w, int page, int key)
{
    return (((size_t)page * a.kv + w.kvh) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
}

/* The sum of the values of dimension d that are not finite, among the keys of the blocks that a row of that length sees. Such
 * values enter products as zeros where some row must not see them; what they do to those that do is added afterwards: any
 * positive weight of an infinity or a NaN is that. Rare, so simple. */
template <int DT, int DH>
__device__ __forceinline__ float odd_values_of(const BatchArgs &a, const BatchItem &w, const ItemBlocks &in, int kb, int len, int d)
{
    typedef typename Elem<DT>::type E;
    float more = 0.0f;
    for (int b = in.b0; b < in.b1; b++)
        for (int key = in.key(b, kb); key < in.key(b, kb) + kb; key++) {
            const int page = page_in(page_entry(w.pages, a.table_ld, key, a.page_shift), a.pages);
            if (page < 0 || !item_sees(a, w, key, len)) continue;
            const float x = Elem<DT>::get(static_cast<const E *>(a.vc)[token_at(a, w, page, key) * DH + d]);
            if (!(__builtin_fabsf(x) < INFINITY)) more += x;
        }
    return __builtin_fabsf(more) < INFINITY ? 0.0f : more;
}

/* one output of the item: straight to o, or as part of it */
template <int DT, int DH>
__device__ __forceinline__ void put_part(const BatchArgs &a, const BatchItem &w, int r, int d, float top, float num, float den)
{
    typedef typename Elem<DT>::type E;
    const int G = a.heads / a.kv, seq = w.seq0 + (w.r0 + r) / G, head = w.kvh * G + (w.r0 + r) % G;
    if (!a.part) {
        static_cast<E *>(a.o)[(size_t)seq * a.ldo + (size_t)head * DH + d] = Elem<DT>::put(den == 0.0f ? 0.0f : num / den);
    } else {
        const size_t to = ((size_t)seq * a.heads + head) * w.parts + w.slot;
        a.part[to * DH + d] = num;
        if (d == 0) a.stat[to] = float2{top, den};
    }
}

/* An item of up to 16 rows over a cache of rows: each wave takes blocks of 32 keys (fp32 16) in turn and has its own running
 * reference, sum and outputs, joined at the end. Bound by waits in turn where there are few keys (4 sequences behind 375, 8 fp32
 * heads of 128: 8.5 us), by memory where each sequence has many (64 sequences of up to 2000 tokens, 32 heads on 8 of 128, bf16, 357 MB:
 * 80 us, 4.5 TB/s). */
template <int DT, int DH, int NW>
__device__ __forceinline__ void attend_rows(const BatchArgs &a, const BatchItem &w, unsigned char *lds)
{
    typedef typename Elem<DT>::type E;
    constexpr int NB = FewPlace<DT>::NB, KB = FewPlace<DT>::KB, EPC = kPer16<DT>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int G = a.heads / a.kv;
    const RowLengths<1> len(a, w);
    const ItemBlocks in(a, w, len.least, len.most, KB);
    u4 q[DH / (4 * EPC)];
    {
        const int r = w.r0 + imin(lane & 15, w.rows - 1);
        const E *p = static_cast<const E *>(a.q) + (size_t)(w.seq0 + r / G) * a.ldq + (size_t)(w.kvh * G + r % G) * DH;
#pragma unroll
        for (int s = 0; s < DH / (4 * EPC); s++) q[s] = *reinterpret_cast<const u4 *>(p + EPC * (4 * s + g));
    }
    FewState<DH> st;
    bool odd = false;
    struct Entries {
        int e[NB];
    };
    auto there = [](const FewPlace<DT> &b, int k) __attribute__((always_inline)) { return b.there[NB == 2 ? k >> 4 : 0]; };
    few_blocks<DT, DH, true>(
        st, q, a.c, in.b0 + wave, in.b1, NW, DH, DH,
        [&](int b) __attribute__((always_inline)) {
            Entries n;   /* pages hold a multiple of 16 tokens */
#pragma unroll
            for (int t = 0; t < NB; t++) {
                const int key = in.key(b, KB) + 16 * t;
                n.e[t] = key < in.end_key ? page_entry(w.pages, a.table_ld, key, a.page_shift) : -1;
            }
            return n;
        },
        [&](int b, Entries n) __attribute__((always_inline)) {
            FewPlace<DT> p;
            p.k0 = in.key(b, KB);
            p.whole = item_sees_all(a, w, p.k0, KB, len.least, len.most);
#pragma unroll
            for (int t = 0; t < NB; t++) {
                const int page = page_in(n.e[t], a.pages);
                const size_t at = token_at(a, w, imax(page, 0), p.k0 + 16 * t) * DH;
                p.have[t] = 16;
                p.there[t] = page >= 0;
                p.k[t] = static_cast<const E *>(a.kc) + at;
                p.v[t] = static_cast<const E *>(a.vc) + at;
                p.whole &= page >= 0;
            }
            return p;
        },
        [&](const FewPlace<DT> &b, int k) __attribute__((always_inline)) {
            return there(b, k) && item_sees(a, w, b.k0 + k, len.of[0]);
        },
        [&](const FewPlace<DT> &b, int k) __attribute__((always_inline)) {   /* seen by some row */
            const int key = b.k0 + k;
            return there(b, k) && key >= w.t0 && key < in.end_key && (key >= len.least - a.window || key < a.sinks);
        },
        odd, lds + wave * few_own_bytes<DT, DH>());
    odd = __syncthreads_or(odd);
    float *J = reinterpret_cast<float *>(lds);
    few_store<DT, DH>(st, J);
    for (int e = threadIdx.x; e < w.rows * DH; e += 64 * NW) {
        const int r = e / DH, d = e % DH;
        float top, num, den;
        few_join<DH, NW>(J, r, d, &top, &num, &den);
        if (odd) {
            const int n = kept_length(a.len[w.seq0 + (w.r0 + r) / G], a.table_ld, 1 << a.page_shift);
            num += odd_values_of<DT, DH>(a, w, in, KB, n, d);
        }
        put_part<DT, DH>(a, w, r, d, top, num, den);
    }
}

constexpr float kCodeSlack = 1024.0f;   /* the largest sum of a lane's eight weights */

template <int DH, int NQ, int NW> constexpr int codes_lds()
{
    constexpr int V = NW * CodeBlock<DH>::STAGES * CodeBlock<DH>::STAGE, J = NW * 16 * NQ * (DH + 2) * 4;
    return V > J ? V : J;
}

/* An item of up to 16 · NQ rows over a cache of codes. Each wave takes blocks of 32 keys in turn, its next block on its way into
 * its own LDS while it multiplies one: S^T = K · Q^T and O^T += V^T · P^T by 16 × 16 × 32 products, codes as 16-bit operands (whole
 * numbers up to 127 are exact), which one conversion and half a permutation make of each. The scales of K multiply the
 * scores, those of V the weights.
 *
 * Nothing is lost but what is said here: fp32 queries and weights go in as three bf16 pieces that sum to them (queries down
 * to 2^-110), 16-bit queries as they are and their weights as two pieces, 16 bits (as one of fp16, a weight times its scale would
 * leave the type's range; as one of bf16, weights cost as much as the rounding of the output: off by 0.00235 of a bf16 output's
 * norm, as two by 0.00166, that rounding alone, for 1 to 8 % of the time).
 *
 * 32 sequences of up to 8192 tokens, 32 heads on 8 of 128, bf16 and fp16, 375 MB: 81 us with the join, 4.6 TB/s, bound by memory
 * (fp32 85; the maximum of every block taken and masks as branches cost 8 more). Three groups of 8 sequences behind 30001 tokens
 * each, heads of 64, fp16 and bf16: 36 us, of which the floor of 104 MB is 20.6: a workgroup's 2 · 16 rows take products of 16 rows
 * twice, the rest is the start and end of 512 workgroups. 64 sequences behind 32768 tokens, 32 heads on 8 of 128: 95 us (fp32 120),
 * vector unit 59 %: codes become operands anew for every 32 rows. One sequence of 375, fp32: 7.9 us, waits in turn (length, page,
 * codes, join). */
template <int DT, int DH, int NQ, int NW>
__device__ __forceinline__ void attend_codes(const BatchArgs &a, const BatchItem &w, unsigned char *lds)
{
    typedef typename Elem<DT>::type E;
    typedef CodeBlock<DH> B;
    constexpr int KB = B::KB, CH = B::CH, RPL = B::RPL, LD = B::LD, NT = DH / 16, KT = DT == T_F16 ? T_F16 : T_BF16;
    constexpr int NP = DT == T_F32 ? 3 : 1, WP = DT == T_F32 ? 3 : 2;   /* pieces of a query, of a weight */
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, x16 = lane & 15;
    const int G = a.heads / a.kv;

    const RowLengths<NQ> len(a, w);
    const ItemBlocks in(a, w, len.least, len.most, KB);
    u4 q[NQ][DH / 32][NP];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r = w.r0 + imin(16 * n + x16, w.rows - 1);
        const E *row = static_cast<const E *>(a.q) + (size_t)(w.seq0 + r / G) * a.ldq + (size_t)(w.kvh * G + r % G) * DH;
#pragma unroll
        for (int s = 0; s < DH / 32; s++) {
            const E *p = row + 64 * (s / 2) + 16 * g + 8 * (s % 2);   /* in the order of the codes' pieces */
            if constexpr (DT == T_F32) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = p[i];
                bf16_pieces<3>(v, q[n][s]);
            } else {
                q[n][s][0] = *reinterpret_cast<const u4 *>(p);
            }
        }
    }

    struct Place {
        int k0;
        bool there[2], whole;
    };
    struct Entries {
        int e[2];
    };
    auto hint = [&](int b) __attribute__((always_inline)) {
        Entries n;   /* pages hold a multiple of 16 tokens */
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int i = (in.key(b, KB) + 16 * t) >> a.page_shift;
            n.e[t] = i < a.table_ld ? scalar_int(w.pages + i) : -1;
        }
        return n;
    };

    constexpr int NS = B::STAGES;
    unsigned char *const own = lds + wave * NS * B::STAGE;
    uint32_t koff[LD], voff[LD];   /* of this lane's 16 bytes from the first row of 16 */
#pragma unroll
    for (int x = 0; x < LD; x++) {
        const int r = RPL * x + lane / CH;
        koff[x] = (r & 15) * DH + 16 * B::k_place(r, lane % CH);
        voff[x] = (r & 15) * DH + 16 * B::v_place(r, lane % CH);
    }
    auto fetch = [&](int b, const Entries &n, unsigned char *to) __attribute__((always_inline)) {
        Place p;
        p.k0 = in.key(b, KB);
        p.whole = item_sees_all(a, w, p.k0, KB, len.least, len.most);
        size_t token[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int page = page_in(n.e[t], a.pages);
            p.there[t] = page >= 0;
            p.whole &= page >= 0;
            token[t] = token_at(a, w, imax(page, 0), p.k0 + 16 * t);
        }
        const unsigned char *kc = static_cast<const unsigned char *>(a.kc), *vc = static_cast<const unsigned char *>(a.vc);
#pragma unroll
        for (int x = 0; x < LD; x++) dma_16(kc + token[RPL * x / 16] * DH, koff[x], to + 1024 * x);
        /* K's 32 scales and V's, in the order of a lane's results */
        dma_4((lane < 32 ? a.ks : a.vs) + (lane & 16 ? token[1] : token[0]) + B::key_of(0, lane & 15), to + 2 * B::BYTES);
#pragma unroll
        for (int x = 0; x < LD; x++) dma_16(vc + token[RPL * x / 16] * DH, voff[x], to + B::BYTES + 1024 * x);
        return p;
    };

    f4 o[NQ][NT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int d = 0; d < NT; d++) o[n][d] = f4{0, 0, 0, 0};
    }

    const int first = in.b0 + wave;
    if (first < in.b1) {
        /* Blocks on their way: NS − 1 while one is multiplied. Those past the wave's last are that one again, so that there are
         * always as many loads to wait for. */
        const int final = first + (in.b1 - 1 - first) / NW * NW;
        Place place[NS];
#pragma unroll
        for (int n = 0; n < NS - 1; n++) {
            const int b = imin(first + n * NW, final);
            place[n] = fetch(b, hint(b), own + n * B::STAGE);
        }
        Entries ahead = hint(imin(first + (NS - 1) * NW, final));
        int stage = 0;
        for (int b = first; b < in.b1; b += NW) {
            const unsigned char *Ks = own + stage * B::STAGE, *Vs = Ks + B::BYTES;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   /* what reads of the stage before brought */
            place[NS - 1] = fetch(imin(b + (NS - 1) * NW, final), ahead, own + (stage == 0 ? NS - 1 : stage - 1) * B::STAGE);
            ahead = hint(imin(b + NS * NW, final));
            const Place now = place[0];
            wait_vm<(NS - 1) * B::LOADS + LD>();   /* all but V's, and the blocks behind */
            f4 s[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; n++) s[n][0] = s[n][1] = f4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int row = B::key_of(t, x16);
#pragma unroll
                for (int x = 0; x < DH / 64; x++) {
                    const u4 k = *reinterpret_cast<const u4 *>(Ks + row * DH + 16 * B::k_place(row, 4 * x + g));
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const u4 kf = code_operand<KT>(k[2 * e], k[2 * e + 1]);
#pragma unroll
                        for (int n = 0; n < NQ; n++)
#pragma unroll
                            for (int p = 0; p < NP; p++) s[n][t] = mfma16<KT>(kf, q[n][2 * x + e][p], s[n][t]);
                    }
                }
            }
            const f4 *sc = reinterpret_cast<const f4 *>(Ks + 2 * B::BYTES);
            f4 vs[2];
            u4 pw[NQ][WP];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f4 ks = sc[4 * t + g];
                vs[t] = sc[8 + 4 * t + g];
#pragma unroll
                for (int n = 0; n < NQ; n++) s[n][t] *= ks;
            }
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                f4 v[2] = {vs[0], vs[1]};
                if (!now.whole) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {   /* whatever the scales of what is not seen */
                        const bool seen = now.there[i / 4] & item_sees(a, w, now.k0 + B::key_of(i / 4, 4 * g + i % 4), len.of[n]);
                        s[n][i / 4][i % 4] = seen ? s[n][i / 4][i % 4] : -INFINITY;
                        v[i / 4][i % 4] = seen ? v[i / 4][i % 4] : 0.0f;
                    }
                }
                float x[8];
                auto weights = [&]() __attribute__((always_inline)) {   /* from the reference on; their sum */
                    const float mu = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = exp2_fast(__builtin_fmaf(s[n][i / 4][i % 4], a.c, -mu));
                    return ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
                };
                float sum = weights();
                /* the reference is raised, to the largest score so far, only where weights have become large or there is none
                 * yet: most blocks need no maximum and leave O as it is */
                if (__any(!(sum <= kCodeSlack) || m[n] == -INFINITY)) {
                    float top = s[n][0][0];
#pragma unroll
                    for (int i = 1; i < 8; i++) top = fmaxf(top, s[n][i / 4][i % 4]);
                    const float mn = fmaxf(m[n], max_quarters(top) * a.c);
                    const float fade = exp2_fast(m[n] - (mn == -INFINITY ? 0.0f : mn));
                    m[n] = mn;
                    l[n] *= fade;
#pragma unroll
                    for (int d = 0; d < NT; d++) o[n][d] *= fade;
                    sum = weights();
                }
                l[n] += sum;
                float wv[8];
#pragma unroll
                for (int i = 0; i < 8; i++) wv[i] = x[i] * v[i / 4][i % 4];
                bf16_pieces<WP>(wv, pw[n]);
            }
            wait_vm<(NS - 1) * B::LOADS>();
#pragma unroll
            for (int h = 0; h < DH / 64; h++) {
                uint32_t dw[8];   /* four neighbouring dimensions of each of the lane's keys, one for each of four products */
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int row = B::key_of(j / 4, 4 * g + j % 4);
                    dw[j] = *reinterpret_cast<const uint32_t *>(Vs + row * DH + 16 * B::v_place(row, 4 * h + x16 / 4) + 4 * (x16 % 4));
                }
                auto product = [&](auto jj) __attribute__((always_inline)) {
                    constexpr int J = decltype(jj)::value;
                    u4 vf;
#pragma unroll
                    for (int i = 0; i < 4; i++) vf[i] = upper_halves(code_at<J>(dw[2 * i]), code_at<J>(dw[2 * i + 1]));
#pragma unroll
                    for (int n = 0; n < NQ; n++)
#pragma unroll
                        for (int p = 0; p < WP; p++) o[n][4 * h + J] = mfma16<T_BF16>(vf, pw[n][p], o[n][4 * h + J]);
                };
                product(std::integral_constant<int, 0>{});
                product(std::integral_constant<int, 1>{});
                product(std::integral_constant<int, 2>{});
                product(std::integral_constant<int, 3>{});
            }
#pragma unroll
            for (int n = 0; n < NS - 1; n++) place[n] = place[n + 1];
            stage = stage == NS - 1 ? 0 : stage + 1;
        }
        wait_vm<0>();   /* nothing comes into the LDS any more */
    }

    __syncthreads();   /* the waves' own parts are done with */
    float *J = reinterpret_cast<float *>(lds);   /* [wave][16 · NQ rows][DH + 2] */
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const float sum = sum_quarters(l[n]);
        float *mine = J + ((wave * NQ + n) * 16 + x16) * (DH + 2);
#pragma unroll
        for (int d = 0; d < NT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) mine[64 * (d / 4) + 4 * (4 * g + i) + d % 4] = o[n][d][i];
        if (g == 0) {
            mine[DH] = m[n];
            mine[DH + 1] = sum;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < w.rows * DH; e += 64 * NW) {
        const int r = e / DH, d = e % DH;
        float top, num, den;
        few_join<DH, NW, 16 * NQ>(J, r, d, &top, &num, &den);
        put_part<DT, DH>(a, w, r, d, top, num, den);
    }
}

/* An item over a cache of either kind: 16 · NQ rows of codes, 16 of rows. */
template <int CK, int DT, int DH, int NQ, int NW> constexpr int attend_lds()
{
    return CK == C_Q8 ? codes_lds<DH, NQ, NW>() : few_lds_bytes<DT, DH, NW>();
}
template <int CK, int DT, int DH, int NQ, int NW>
__device__ __forceinline__ void attend_item(const BatchArgs &a, const BatchItem &w, unsigned char *lds)
{
    if constexpr (CK == C_Q8) attend_codes<DT, DH, NQ, NW>(a, w, lds);
    else attend_rows<DT, DH, NW>(a, w, lds);
}

/* group g's sequences [sa, sb) */
__device__ __forceinline__ int group_start(const BatchArgs &a, int g) { return imin(imax(a.group[g], 0), a.n_seqs); }

/* The prefix that a group shares for 128 of its query rows, 32 for each of four waves; 16-bit rows. Keys come in blocks of 64
 * through LDS, K and V in two buffers each, each wave bringing 16 keys of both, which lie in one page.
 *
 * As in windowed attention, S^T = K · Q^T by 32 × 32 products, so that a lane holds 32 keys of one row and its weights are laid
 * out as the operand of O^T += V^T · P^T; the scores of block b run together with the output product of block b − 1, in
 * stages of equal length, each stage's operands read from LDS two stages ahead and one of the next loads issued in each; the
 * reference of the exponentials is raised only where a block's sum of weights leaves the type's range. One barrier a block.
 *
 * 64 sequences behind 32768 tokens, 32 heads on 8 of 128, bf16: 55 us without their own keys, 0.62 PFLOP/s; 72 with 512 of their
 * own each, which start when tiles end. Eight waves a workgroup with four buffers, one a CU, took 83; tiles and own parts in
 * turn 74, as a SIMD's two waves of tiles fill each other's gaps.
 *
 * Weights are rounded to the type for their product with V, not for their sum, as everywhere where rows are kept in 16 bits: of the
 * same case 0.0023 of the outputs' norm off against 64 bits, where the rounding of the outputs is 0.0017. A second product with
 * what the first lost leaves that alone and costs 12 to 20 % (with the join 78.5 -> 88.3 us, with 20 keys of their own 60.6 -> 72.2; fp16
 * 78 -> 90). An fp16 weight under 2^-31 of the largest that its part of the prefix has had so far is lost (one of 2^-25 under a
 * reference that stands 2^6 below): it takes 2^20 keys of one part, all just under that, to lose half a step of the sum. kLift would lose
 * less, but its sums of 32 weights would leave the type. */
constexpr int kTileRows = 128;
template <int DT> constexpr float kTileLift = DT == T_F16 ? 6.0f : 0.0f;          /* fp16 weights up to 2^6 below … */
template <int DT> constexpr float kTileSlack = DT == T_F16 ? 65504.0f : 1024.0f;  /* … a sum that every type holds */

template <int DT, int DH> constexpr int tile_lds() { return 4 * 64 * DH * 2; }

template <int DT, int DH>
__device__ __forceinline__ void attend_tile(const BatchArgs &a, const BatchItem &w, unsigned char *lds)
{
    typedef typename Elem<DT>::type E;
    constexpr int KB = 64, CH = DH / 8, RPL = 64 / CH, LD = 16 / RPL, QR = DH / 16, NT = DH / 32, RB = 2 * DH;
    constexpr uint32_t BUF = KB * RB;
    static_assert(2 * LD == QR, "one load a stage");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5, col = lane & 31;
    const int G = a.heads / a.kv;
    auto k_place = [](int r, int p) { return p ^ (CH == 16 ? r & 15 : (r >> 1) & 7); };
    auto v_place = [](int r, int p) { return p ^ (CH == 16 ? 4 * (r & 3) : 4 * ((r >> 1) & 1)); };

    const int r = imin(32 * wave + col, w.rows - 1), seq = w.seq0 + (w.r0 + r) / G, head = w.kvh * G + (w.r0 + r) % G;
    const int len = a.pages ? kept_length(a.len[seq], a.table_ld, 1 << a.page_shift) : 0;
    u4 q[QR];
    {
        const E *row = static_cast<const E *>(a.q) + (size_t)seq * a.ldq + (size_t)head * DH;
#pragma unroll
        for (int x = 0; x < QR; x++) q[x] = *reinterpret_cast<const u4 *>(row + 8 * (2 * x + h));
    }
    /* of the wave's rows, and of all rows (the first one's sequence to the last one's) */
    int wave_least = len, wave_most = len, least = 1 << 30, most = 0;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        wave_least = imin(wave_least, __shfl_xor(wave_least, o));
        wave_most = imax(wave_most, __shfl_xor(wave_most, o));
    }
    for (int s = w.seq0 + w.r0 / G + lane; s <= w.seq0 + (w.r0 + w.rows - 1) / G; s += 64) {
        const int n = a.pages ? kept_length(a.len[s], a.table_ld, 1 << a.page_shift) : 0;
        least = imin(least, n);
        most = imax(most, n);
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        least = imin(least, __shfl_xor(least, o));
        most = imax(most, __shfl_xor(most, o));
    }
    wave_least = __builtin_amdgcn_readfirstlane(wave_least);
    wave_most = __builtin_amdgcn_readfirstlane(wave_most);
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
    const ItemBlocks in(a, w, least, most, KB);
    const int b0 = in.b0, b1 = in.b1;

    /* where 16 keys lie: of block b those that this wave brings, and which of the block's four sixteens are in a page */
    struct Entries {
        int mine, e[4];
    };
    auto entry = [&](int key) __attribute__((always_inline)) {
        const int i = key >> a.page_shift;
        return i < a.table_ld ? scalar_int(w.pages + i) : -1;
    };
    auto hint = [&](int b) __attribute__((always_inline)) {
        const int k0 = in.key(b, KB);
        return Entries{entry(k0 + 16 * wave), {entry(k0), entry(k0 + 16), entry(k0 + 32), entry(k0 + 48)}};
    };
    auto token_of = [&](int b, const Entries &n) __attribute__((always_inline)) {
        const int key = in.key(b, KB) + 16 * wave, page = imax(page_in(n.mine, a.pages), 0);
        return token_at(a, w, page, key) * RB;
    };
    auto there = [&](const Entries &n) __attribute__((always_inline)) {
        unsigned long long bits = 0;
#pragma unroll
        for (int t = 0; t < 4; t++)
            if (page_in(n.e[t], a.pages) >= 0) bits |= 0xffffull << (16 * t);
        return bits;
    };
    uint32_t koff[LD], voff[LD];
#pragma unroll
    for (int x = 0; x < LD; x++) {
        const int rr = RPL * x + lane / CH;
        koff[x] = rr * RB + 16 * k_place(rr, lane % CH);
        voff[x] = rr * RB + 16 * v_place(rr, lane % CH);
    }
    auto fetch = [&](int x, const unsigned char *from, const uint32_t (&off)[LD], uint32_t buffer) __attribute__((always_inline)) {
        dma_16(from, off[x], lds + buffer * BUF + 16 * wave * RB + 1024 * x);
    };
    const unsigned char *kc = static_cast<const unsigned char *>(a.kc), *vc = static_cast<const unsigned char *>(a.vc);

    f16v o[NT], s[2];
    u4 pw[4];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) pw[k] = u4{0, 0, 0, 0};
    bool odd = false;

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)lds;
    const int vr = 4 * h + ((lane & 15) >> 2);
    const uint32_t k_at = lds0 + col * RB + 16 * k_place(col, h);
    const uint32_t v_at = lds0 + 2 * BUF + vr * RB + 16 * v_place(vr, 0) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto read_k = [&](uint32_t at, int n, int x) __attribute__((always_inline)) {
        typedef __attribute__((address_space(3))) const u4 *lds16;
        return *(lds16)(uintptr_t)((at ^ (32 * x)) + 32 * n * RB);
    };
    auto read_v = [&](uint32_t at, int k2, int d) __attribute__((always_inline)) {
        const uint32_t x = (at ^ (64 * d)) + 16 * k2 * RB;
        const u2 va = lds_tr(x), vb = lds_tr(x + 8 * RB);
        return u4{va[0], va[1], vb[0], vb[1]};
    };
    /* this wave's loads have come; of V of block b, where some row must not see a key, what no row sees and what is not finite
     * becomes zeros, which `odd` notes of the latter: a weight of 0 times them would be a NaN */
    auto come = [&](int b, unsigned long long held) __attribute__((always_inline)) {
        wait_vm<0>();
        if (b >= b0) {
            const int k0 = in.key(b, KB);
            if (held != ~0ull || !item_sees_all(a, w, k0, KB, least, most)) {
                u4 *v = reinterpret_cast<u4 *>(lds + (2 + ((b - b0) & 1)) * BUF + 16 * wave * RB) + lane;
#pragma unroll
                for (int x = 0; x < LD; x++) {
                    const int e = 16 * wave + RPL * x + lane / CH, key = k0 + e;
                    const bool keep = ((held >> e) & 1) && key < in.end_key && (key >= least - a.window || key < a.sinks);
                    if (!keep) {
                        v[64 * x] = u4{0, 0, 0, 0};
                    } else if (odd_values<DT>(v[64 * x])) {
                        odd = true;
                        v[64 * x] = only_finite<DT>(v[64 * x]);
                    }
                }
            }
        }
        lds_barrier();
    };
    /* what a row must not see: key e of the block is bit e of 64; this lane has keys 8j + 4h .. + 3 of every eight */
    auto mask = [&](int k0, unsigned long long held) __attribute__((always_inline)) {
        if (held == ~0ull && item_sees_all(a, w, k0, KB, wave_least, wave_most)) return;
        auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
        const unsigned long long bits = (below(imin(len, w.t1) - k0) & (~below(len - a.window - k0) | below(a.sinks - k0)) & held) >> (4 * h);
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t seen = (uint32_t)__builtin_amdgcn_sbfe((int)(bits >> (32 * n)), 8 * (i / 4) + i % 4, 1);
                s[n][i] = __uint_as_float((__float_as_uint(s[n][i]) & seen) | (0xff800000u & ~seen));
            }
    };
    auto weights = [&](int k, float mu, float &sum) __attribute__((always_inline)) {
        float pv[8];
#pragma unroll
        for (int i = 0; i < 8; i++) pv[i] = exp2_fast(__builtin_fmaf(s[k / 2][8 * (k & 1) + i], a.c, -mu));
        sum += ((pv[0] + pv[1]) + (pv[2] + pv[3])) + ((pv[4] + pv[5]) + (pv[6] + pv[7]));
        pw[k] = pack<DT>(pv);
    };
    auto settle = [&](float sum) __attribute__((always_inline)) {
        if (__any(sum > kTileSlack<DT> || m == -INFINITY)) {
            float top = s[0][0];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) top = fmaxf(top, s[n][i]);
            const float mn = fmaxf(m, lifted(max_halves(top), a.c, kTileLift<DT>)), mu = mn == -INFINITY ? 0.0f : mn;
            const float fade = exp2_fast(m - mu);
            m = mn;
            l *= fade;
#pragma unroll
            for (int d = 0; d < NT; d++) o[d] *= fade;
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) weights(k, mu, sum);
        }
        l += sum;
    };
    if (b0 < b1) {
        Entries now = hint(b0);
        {
            const unsigned char *from = kc + token_of(b0, now);
#pragma unroll
            for (int x = 0; x < LD; x++) fetch(x, from, koff, 0);
        }
        Entries next = hint(imin(b0 + 1, b1 - 1));
        unsigned long long held = there(now), held_before = 0;
        /* the first block has no weights before it: zeros, with zeros for V */
        for (int x = threadIdx.x; x < KB * CH; x += 256) reinterpret_cast<u4 *>(lds + 3 * BUF)[x] = u4{0, 0, 0, 0};
        for (int b = b0; b < b1; b++) {
            const int k0 = in.key(b, KB), odd_block = (b - b0) & 1;
            /* past the last block that one's K again, which nothing reads */
            const unsigned char *next_k = kc + token_of(imin(b + 1, b1 - 1), next), *this_v = vc + token_of(b, now);
            const uint32_t ka = k_at + odd_block * BUF, va = v_at + (odd_block ^ 1) * BUF;
            u4 kf[3][2], vf[3][2];
            auto read = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    kf[t % 3][j] = read_k(ka, j, t);
                    vf[t % 3][j] = read_v(va, (2 * t + j) / NT, (2 * t + j) % NT);
                }
            };
#pragma unroll
            for (int i = 0; i < 16; i++) s[0][i] = s[1][i] = 0.0f;
            come(b - 1, held_before);
            __builtin_amdgcn_s_setprio(1);   /* products first: the other wave's exponentials fill what they leave */
            read(0);
            read(1);
#pragma unroll
            for (int t = 0; t < QR; t++) {   /* the barriers to the scheduler keep this order */
                if (t + 2 < QR) read(t + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int z = 2 * t + j;
                    s[j] = mfma32<DT>(kf[t % 3][j], q[t], s[j]);
                    o[z % NT] = mfma32<DT>(vf[t % 3][j], pw[z / NT], o[z % NT]);
                }
                if (t < LD) fetch(t, next_k, koff, odd_block ^ 1);
                else fetch(t - LD, this_v, voff, 2 + odd_block);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            const Entries after = hint(imin(b + 2, b1 - 1));   /* not among the LDS reads, which it would be waited for with */
            mask(k0, held);
            const float mu = m == -INFINITY ? 0.0f : m;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) weights(k, mu, sum);
            settle(sum);
            held_before = held;
            now = next;
            next = after;
            held = there(now);
        }
        come(b1 - 1, held_before);
        const uint32_t va = v_at + ((b1 - 1 - b0) & 1) * BUF;
#pragma unroll
        for (int k2 = 0; k2 < 4; k2++)
#pragma unroll
            for (int d = 0; d < NT; d++) o[d] = mfma32<DT>(read_v(va, k2, d), pw[k2], o[d]);
    }
    odd = __syncthreads_or(odd);
    const float sum = sum_halves(l);
    if (32 * wave + col >= w.rows) return;
    const size_t to = ((size_t)seq * a.heads + head) * w.parts + w.slot;
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<f4 *>(a.part + to * DH + 32 * d + 8 * i + 4 * h) = f4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    if (h == 0) a.stat[to] = float2{m, sum};
    if (odd)
        for (int i = 0; i < DH / 2; i++) {   /* those that this lane has just stored */
            const int d = 8 * (i / 4) + 4 * h + i % 4;
            a.part[to * DH + d] += odd_values_of<DT, DH>(a, w, in, KB, len, d);
        }
}

/* this workgroup's tile of TR rows of a group's prefix; false where there is none */
template <int TR> __device__ __forceinline__ bool prefix_item(const BatchArgs &a, int at, BatchItem *w)
{
    /* All parts of a tile next to each other: numbers without a tile would otherwise fall on the same shader engines, to which
     * workgroups go in turn, and leave the work to the others (a tile, none, a tile, …: 86 us in place of 55). */
    const int G = a.heads / a.kv, id = at / a.kv, tile = id / a.p_parts;
    w->kvh = at % a.kv;
    w->split = id % a.p_parts;
    /* tiles are numbered as tile_start does, rows being G for each sequence */
    const int gr = wave_last(a.n_groups, [&](int s) { return group_start(a, s) * G / TR + s <= tile; });
    if (gr < 0) return false;
    const int sa = group_start(a, gr), sb = imax(group_start(a, gr + 1), sa);
    w->r0 = (tile - (sa * G / TR + gr)) * TR;
    if (w->r0 < 0 || w->r0 >= (sb - sa) * G) return false;   /* below 0 where starts descend */
    w->seq0 = sa;
    w->rows = imin(TR, (sb - sa) * G - w->r0);
    w->t0 = 0;
    w->t1 = imax(a.shared[gr], 0);
    w->pages = a.table + (size_t)sa * a.table_ld;
    w->splits = a.p_parts;
    w->slot = w->split;
    w->parts = a.p_parts + a.o_parts;
    return true;
}

/* this workgroup's part of what a sequence has alone, 16 of a key head's queries; false where it has none */
__device__ __forceinline__ bool own_item(const BatchArgs &a, int id, BatchItem *w)
{
    const int G = a.heads / a.kv;
    w->kvh = id % a.kv;
    id /= a.kv;
    w->split = id % a.o_parts;
    id /= a.o_parts;
    w->r0 = 16 * (id % a.q_groups);
    w->seq0 = id / a.q_groups;
    w->rows = imin(16, G - w->r0);
    w->t0 = 0;
    w->t1 = 1 << 30;
    w->pages = a.table + (size_t)w->seq0 * a.table_ld;
    w->splits = a.o_parts;
    w->slot = a.p_parts + w->split;
    w->parts = a.p_parts + a.o_parts;
    if (!a.group) return true;
    const int gr = wave_last(a.n_groups, [&](int s) { return group_start(a, s) <= w->seq0; });
    if (gr < 0 || w->seq0 >= group_start(a, gr + 1)) {   /* in no group: attend_join leaves its rows as they are */
        if (w->split == 0 && (int)threadIdx.x < w->rows)
            a.stat[((size_t)w->seq0 * a.heads + w->kvh * G + w->r0 + threadIdx.x) * w->parts + w->slot] = float2{0.0f, -1.0f};
        return false;
    }
    w->t0 = imax(a.shared[gr], 0);
    return true;
}

/* Prefixes by 16 · NQ rows of a group, then what each sequence has alone. */
template <int CK, int DT, int DH, int NQ, int NW>
__global__ __launch_bounds__(64 * NW, CK == C_ROWS ? (DH == 64 ? 4 : DT == T_F32 ? 3 : 2) : 2) void attend(BatchArgs a)
{
    constexpr int L = attend_lds<CK, DT, DH, NQ, NW>(), L1 = attend_lds<CK, DT, DH, 1, NW>();
    __shared__ __align__(16) unsigned char lds[L > L1 ? L : L1];
    BatchItem w;
    const bool prefix = (int)blockIdx.x < a.p_wgs;
    if (!(prefix ? prefix_item<16 * NQ>(a, blockIdx.x, &w) : own_item(a, blockIdx.x - a.p_wgs, &w))) return;
    if constexpr (NQ > 1) {
        if (prefix) {
            attend_item<CK, DT, DH, NQ, NW>(a, w, lds);
            return;
        }
    }
    attend_item<CK, DT, DH, 1, NW>(a, w, lds);
}

/* Prefixes by tiles of 128 rows, then what each sequence has alone. */
template <int DT, int DH>
__global__ __launch_bounds__(256, 2) void attend_tiles(BatchArgs a)
{
    __shared__ __align__(16) unsigned char lds[tile_lds<DT, DH>()];
    static_assert(tile_lds<DT, DH>() >= few_lds_bytes<DT, DH, 4>(), "what both need");
    BatchItem w;
    if ((int)blockIdx.x < a.p_wgs) {
        if (prefix_item<kTileRows>(a, blockIdx.x, &w)) attend_tile<DT, DH>(a, w, lds);
    } else {
        if (own_item(a, blockIdx.x - a.p_wgs, &w)) attend_rows<DT, DH, 4>(a, w, lds);
    }
}

/* The parts of one query added up by one wave, DH / 64 outputs a lane: o = Σ 2^(top_i − top) num_i / Σ 2^(top_i − top) den_i. Bound by
 * waits (2.6 us for 8 queries, 2 parts; one query of 1024 parts, which a wave reads eight at a time, 44, where what made them took 10)
 * or reading the parts, which the memory-side cache holds (64 · 32 queries of 33 parts, 35 MB: 8 us). */
template <int DT, int DH>
__global__ __launch_bounds__(256) void attend_join(BatchArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int PER = DH / 64;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, parts = a.p_parts + a.o_parts;
    if (row >= a.n_seqs * a.heads) return;
    const float *p = a.part + (size_t)row * parts * DH + PER * lane;
    const float2 *st = a.stat + (size_t)row * parts;
    if (st[a.p_parts].y < 0.0f) return;   /* a sequence of no group */
    float top = -INFINITY;
    for (int s = lane; s < parts; s += 64) top = fmaxf(top, st[s].x);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float mu = top == -INFINITY ? 0.0f : top;
    float num[PER], den = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) num[i] = 0.0f;
#pragma unroll 8
    for (int s = 0; s < parts; s++) {
        const float2 of = st[s];
        const float f = exp2_fast(of.x - mu);
#pragma unroll
        for (int i = 0; i < PER; i++) num[i] = __builtin_fmaf(f, p[(size_t)s * DH + i], num[i]);
        den = __builtin_fmaf(f, of.y, den);
    }
    E *o = static_cast<E *>(a.o) + (size_t)(row / a.heads) * a.ldo + (size_t)(row % a.heads) * DH + PER * lane;
#pragma unroll
    for (int i = 0; i < PER; i++) o[i] = Elem<DT>::put(den == 0.0f ? 0.0f : num[i] / den);
}

/* ── adapters ──────────────────────────────────────────────────────────────────────────────────────────────── */

struct AdapterArgs {
    int M, N, K, count, ldx, ldz, ldy, parts, chunk, vec, units;   /* parts of `chunk` dimensions of K; vec: rows of Z and Y by 16 bytes; 64 columns a unit */
    const void *x, *z, *a, *b;
    const float *scale;
    const int *index;
    void *y;
    float *h;   /* [parts][M][rank] */
};

/* Y = Z + scale · (X · Aᵀ) · Bᵀ in two kernels, the sums of the first, H, in fp32 between them, or in one where all of A that a
 * tile of rows needs is little. fp32 throughout where the type is; 16-bit rows multiply A in 16-bit products with fp32 sums,
 * and H in fp32 products with B's values, which are exact in fp32, so that nothing is rounded before Y. Rows of one adapter among
 * 16 (64) share what is read of it. */

/* The adapters of a workgroup's rows (up to 64), each once, with its rows as bits, in the order of their first rows; rows
 * without one come as adapter −1. */
struct AdapterList {
    int n, of[64];
    unsigned long long rows[64];
};

__device__ __forceinline__ void list_adapters(const AdapterArgs &a, int m0, int rows, AdapterList *list)
{
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        const int id = lane < rows ? a.index[m0 + lane] : -1, mine = (unsigned)id < (unsigned)a.count ? id : -1;
        unsigned long long left = __ballot(lane < rows);
        int n = 0;
        while (left) {
            const int ad = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
            const unsigned long long those = __ballot(mine == ad) & left;
            if (lane == 0) {
                list->of[n] = ad;
                list->rows[n] = those;
            }
            n++;
            left &= ~those;
        }
        if (lane == 0) list->n = n;
    }
    __syncthreads();
}

/* Four steps of 4 dimensions of 16 × 16 fp32 products, or one of 32 16-bit ones */
template <int DT> __device__ __forceinline__ f4 mfma_piece(u4 a, u4 b, f4 c)
{
    if constexpr (DT == T_F32) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    } else {
        return mfma16<DT>(a, b, c);
    }
}

/* 16 bytes of a row from element k on, zeros behind element `end`; VEC: all there and aligned. Otherwise by the element, inside
 * a row too: the first product of bf16, rank 16, K = 4095 against 4096: one row 4.4 us (3.1), 32 rows of as many requests 21 (7.6), 300 rows
 * 9.3 (4.5); 6000 rows, K = 1023 against 1024, 20 (7.8, by 64 rows), fp32 of rank 32 26 (15). */
template <int DT, bool VEC> __device__ __forceinline__ u4 row_piece(const typename Elem<DT>::type *row, int k, int end)
{
    typedef typename Elem<DT>::type E;
    if constexpr (VEC) {
        return *reinterpret_cast<const u4 *>(row + k);
    } else {
        E v[kPer16<DT>];
#pragma unroll
        for (int j = 0; j < kPer16<DT>; j++) v[j] = k + j < end ? row[k + j] : Elem<DT>::put(0.0f);
        u4 r;
        __builtin_memcpy(&r, v, sizeof v);
        return r;
    }
}

/* The sums over dimensions [k0, k1) of 16 rows of X from m0 on times their adapters' A, each adapter by a wave or, where there
 * are fewer adapters than waves, by several that share the dimensions: sum[part][row][r], as many parts as returned. */
template <int DT, int RANK, int NW, bool VEC>
__device__ __forceinline__ int shrink_rows(const AdapterArgs &a, const AdapterList &list, int m0, int rows, int k0, int k1,
                                           float (*sum)[16][RANK + 1])
{
    typedef typename Elem<DT>::type E;
    constexpr int VE = kPer16<DT>, STEP = 4 * VE, RT = (RANK + 15) / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int n = __builtin_amdgcn_readfirstlane(list.n);
    int sets = 1;   /* adapters at a time */
    while (sets < n && sets < NW) sets *= 2;
    const int parts = NW / sets, part = wave / sets;
    const E *x = static_cast<const E *>(a.x) + (size_t)(m0 + imin(c, rows - 1)) * a.ldx;
    for (int j = wave % sets; j < n; j += sets) {
        const int ad = __builtin_amdgcn_readfirstlane(list.of[j]);
        if (ad < 0) continue;
        const uint32_t those = (uint32_t)list.rows[j];
        f4 acc[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t] = f4{0, 0, 0, 0};
        const E *am = static_cast<const E *>(a.a) + (size_t)ad * RANK * a.K;
        int k = k0 + STEP * part;
        if constexpr (VEC) {
#pragma unroll(RT <= 2 ? 8 : 4)
            for (; k + STEP <= k1; k += STEP * parts) {
                const u4 xv = row_piece<DT, true>(x, k + VE * g, k1);
#pragma unroll
                for (int t = 0; t < RT; t++)
                    acc[t] = mfma_piece<DT>(xv, row_piece<DT, true>(am + (size_t)imin(16 * t + c, RANK - 1) * a.K, k + VE * g, k1),
                                            acc[t]);
            }
        }
        for (; k < k1; k += STEP * parts) {
            const u4 xv = row_piece<DT, false>(x, k + VE * g, k1);
#pragma unroll
            for (int t = 0; t < RT; t++)
                acc[t] = mfma_piece<DT>(xv, row_piece<DT, false>(am + (size_t)imin(16 * t + c, RANK - 1) * a.K, k + VE * g, k1),
                                        acc[t]);
        }
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (((those >> (4 * g + i)) & 1) && 16 * t + c < RANK) sum[part][4 * g + i][16 * t + c] = acc[t][i];
    }
    __syncthreads();
    return parts;
}

/* H[part][m][r] = the sum over the part's dimensions k of X[m][k] · A[adapter of m][r][k], 16 rows a workgroup. Bound by the
 * waits for A, which each adapter's wave has alone: 32 rows of 16 adapters, K = 4096, rank 16, bf16: 7.4 us. */
template <int DT, int RANK, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW) void adapter_shrink(AdapterArgs a)
{
    __shared__ float sum[NW][16][RANK + 1];
    __shared__ AdapterList list;
    const int m0 = 16 * blockIdx.x, rows = imin(16, a.M - m0), k0 = blockIdx.y * a.chunk;
    list_adapters(a, m0, rows, &list);
    const int parts = shrink_rows<DT, RANK, NW, VEC>(a, list, m0, rows, k0, imin(k0 + a.chunk, a.K), sum);
    for (int e = threadIdx.x; e < rows * RANK; e += 64 * NW) {   /* rows without an adapter hold anything */
        float s = 0.0f;
        for (int p = 0; p < parts; p++) s += sum[p][e / RANK][e % RANK];
        a.h[((size_t)blockIdx.y * a.M + m0) * RANK + e] = s;
    }
}

/* The same for many rows, 64 a workgroup, 16 a wave, whose X and A come through LDS 256 bytes of a row at a time, read along the
 * rows: read as operands, neighbouring lanes would be in different rows. Two stages in turn. Rows of X and A are 16-byte
 * aligned. fp32, 6000 rows of 375 an adapter, K = 1024, rank 32: 15 us, X at 1.6 TB/s: a workgroup's rows take the two
 * stages' waits in turn. */
template <int RANK> constexpr int shrink_stage() { return (64 + RANK) * 256; }

template <int DT, int RANK>
__global__ __launch_bounds__(256) void adapter_shrink_rows(AdapterArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int VE = kPer16<DT>, KC = 16 * VE, RT = (RANK + 15) / 16, ALD = RANK < 16 ? 1 : RANK / 16;   /* loads of A a wave */
    __shared__ __align__(16) unsigned char lds[2 * shrink_stage<RANK>()];
    __shared__ AdapterList list;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int m0 = 64 * blockIdx.x, rows = imin(64, a.M - m0), k0 = blockIdx.y * a.chunk, k1 = imin(k0 + a.chunk, a.K);
    const int stages = k1 > k0 ? (k1 - k0 + KC - 1) / KC : 0;
    const E *const x = static_cast<const E *>(a.x);
    /* row r has its piece p at place p ^ (r mod 16); a load brings 4 rows */
    auto place = [](int r, int p) { return p ^ (r & 15); };
    auto piece = [&](int st, int r) { return imin(k0 + KC * st + VE * place(r, lane & 15), k1 - VE); };   /* past the end: the last one */
    auto fetch_x = [&](int st, unsigned char *to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 16 * wave + 4 * i + (lane >> 4);
            dma_16(x + (size_t)(m0 + imin(r, rows - 1)) * a.ldx + piece(st, r), to + 1024 * (4 * wave + i));
        }
    };
    auto fetch_a = [&](int ad, int st, unsigned char *to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < ALD; i++) {
            const int load = RANK < 16 ? wave % (RANK / 4) : ALD * wave + i, r = 4 * load + (lane >> 4);
            dma_16(static_cast<const E *>(a.a) + ((size_t)ad * RANK + r) * a.K + piece(st, r), to + 64 * 256 + 1024 * load);
        }
    };
    if (stages > 0) fetch_x(0, lds);   /* on its way while the adapters are looked up */
    list_adapters(a, m0, rows, &list);
    const int n = __builtin_amdgcn_readfirstlane(list.n);
    bool fetched = true;
    for (int j = 0; j < n; j++) {
        const int ad = __builtin_amdgcn_readfirstlane(list.of[j]);
        if (ad < 0) continue;
        const uint32_t those = (uint32_t)__builtin_amdgcn_readfirstlane((int)(list.rows[j] >> (16 * wave))) & 0xffffu;
        f4 acc[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t] = f4{0, 0, 0, 0};
        if (stages > 0) {
            if (!fetched) fetch_x(0, lds);
            fetch_a(ad, 0, lds);
        }
        fetched = false;
        for (int st = 0; st < stages; st++) {
            unsigned char *const now = lds + (st & 1) * shrink_stage<RANK>();
            /* the last stage's loads again, which nothing reads, so that there are always as many to wait for */
            unsigned char *const then = lds + ((st & 1) ^ 1) * shrink_stage<RANK>();
            fetch_x(imin(st + 1, stages - 1), then);
            fetch_a(ad, imin(st + 1, stages - 1), then);
            wait_vm<4 + ALD>();
            lds_barrier();
            if (those) {
                const int have = (k1 - k0 - KC * st) / VE;   /* pieces of this stage */
#pragma unroll
                for (int s = 0; s < 4; s++) {
                    const int p = 4 * s + g;
                    auto read = [&](const unsigned char *base, int r) __attribute__((always_inline)) {
                        u4 v = *reinterpret_cast<const u4 *>(base + 256 * r + 16 * place(r, p));
                        return p < have ? v : u4{0, 0, 0, 0};
                    };
                    const u4 xv = read(now, 16 * wave + c);
#pragma unroll
                    for (int t = 0; t < RT; t++) acc[t] = mfma_piece<DT>(xv, read(now + 64 * 256, imin(16 * t + c, RANK - 1)), acc[t]);
                }
            }
            lds_barrier();   /* everyone is done with what the next loads overwrite */
        }
        wait_vm<0>();
        lds_barrier();
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (((those >> (4 * g + i)) & 1) && 16 * t + c < RANK)
                    a.h[((size_t)blockIdx.y * a.M + m0 + 16 * wave + 4 * g + i) * RANK + 16 * t + c] = acc[t][i];
    }
    wait_vm<0>();   /* nothing comes into the LDS any more, whatever adapters there were */
}

/* Row 4g + i of product t is this column of 64, so that a lane's results are 16 bytes of neighbours (16-bit rows: of two
 * products) and four lanes' 64. */
template <int DT> __device__ __forceinline__ constexpr int expand_column(int t, int r)
{
    return DT == T_F32 ? 16 * t + r : 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
}

/* What 64 columns from n0 on of those of 16 rows from m0 on need from memory, where whole rows are read 16 bytes at a time */
template <int DT> struct ExpandRows {
    static constexpr int VE = kPer16<DT>, NV = 16 / VE;
    u4 z[NV];
    __device__ __forceinline__ void load(const AdapterArgs &a, bool in, int m, int n0, int g)
    {
        typedef typename Elem<DT>::type E;
#pragma unroll
        for (int p = 0; p < NV; p++) {
            z[p] = u4{0, 0, 0, 0};
            if (a.z && in) z[p] = *reinterpret_cast<const u4 *>(static_cast<const E *>(a.z) + (size_t)m * a.ldz + n0 + 4 * VE * p + VE * g);
        }
    }
};

constexpr int kTileRowsLds = 8;

/* … and Y = Z + Σ h · B of them, h this lane's RANK / 4 of row m0 + lane % 16 (times the adapter's scale), b its elements of B's
 * rows, in fp32 products (B's values are exact in fp32), rounded once. Rows that are not read 16 bytes at a time go through
 * the wave's LDS, so that lanes have neighbouring columns of one row. */
template <int DT, int RANK>
__device__ __forceinline__ void expand_rows(const AdapterArgs &a, uint32_t those, int m0, int n0, bool whole,
                                            const ExpandRows<DT> &rows, const float (&h)[RANK / 4],
                                            const typename Elem<DT>::type (&b)[4][RANK / 4], float (*tile)[68])
{
    typedef typename Elem<DT>::type E;
    constexpr int RS = RANK / 4, VE = kPer16<DT>, NV = 16 / VE;
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const E *z = static_cast<const E *>(a.z);
    E *y = static_cast<E *>(a.y);
    E zs[kTileRowsLds];
    auto load_z = [&](uint32_t left) __attribute__((always_inline)) {   /* of the next kTileRowsLds rows */
#pragma unroll
        for (int k = 0; k < kTileRowsLds; k++) {
            zs[k] = Elem<DT>::put(0.0f);
            if (left && z && n0 + lane < a.N) zs[k] = z[(size_t)(m0 + __builtin_ctz(left)) * a.ldz + n0 + lane];
            left &= left - 1;
        }
    };
    if (!whole) load_z(those);
    f4 acc[4];
#pragma unroll
    for (int t = 0; t < 4; t++) acc[t] = f4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < RS; s++)
#pragma unroll
        for (int t = 0; t < 4; t++)
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(Elem<DT>::get(b[t][s]), h[s], acc[t], 0, 0, 0);
    if (whole) {
#pragma unroll
        for (int p = 0; p < NV; p++) {
            float v[VE];
            unpack<DT>(rows.z[p], v);
#pragma unroll
            for (int j = 0; j < VE; j++) v[j] += acc[VE / 4 * p + j / 4][j % 4];
            if ((those >> c) & 1) *reinterpret_cast<u4 *>(y + (size_t)(m0 + c) * a.ldy + n0 + 4 * VE * p + VE * g) = pack<DT>(v);
        }
    } else {
        /* kTileRowsLds of these rows at a time */
        const int place = __popc(those & ((1u << c) - 1)), count = __popc(those);
        uint32_t left = those;
        for (int done = 0; done < count; done += kTileRowsLds) {
            if (((those >> c) & 1) && place >= done && place < done + kTileRowsLds)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) tile[place - done][expand_column<DT>(t, 4 * g + i)] = acc[t][i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < kTileRowsLds; k++)
                if (done + k < count) {
                    const int r = __builtin_ctz(left);
                    left &= left - 1;
                    if (n0 + lane < a.N)
                        y[(size_t)(m0 + r) * a.ldy + n0 + lane] = Elem<DT>::put(Elem<DT>::get(zs[k]) + tile[k][lane]);
                }
            load_z(left);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

/* Y[m][n] = Z[m][n] + scale · the sum over r of H[m][r] · B[adapter of m][n][r]: 16 rows and 64 columns a workgroup, a wave taking
 * one of its adapters at a time. FUSED: H is made here, from all of K. Bound by waits in turn: one row, 1024 × 1024, rank 8,
 * fused 4.2 us; 32 rows of 16 adapters, N = 16384, rank 16, bf16 7.6, N = 16389 12.4, as the 514 workgroups are two more than the
 * CUs hold at once (with 80 registers three would fit a CU, which spills: 15). */
template <int DT, int RANK, int NW, bool FUSED, bool VEC>
__global__ __launch_bounds__(64 * NW) void adapter_expand(AdapterArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int RS = RANK / 4;   /* a lane's elements of a row of rank: RS · g .. */
    __shared__ float tile[NW][kTileRowsLds][68];
    __shared__ AdapterList list;
    __shared__ float sum[FUSED ? NW : 1][16][RANK + 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int m0 = 16 * blockIdx.y, rows = imin(16, a.M - m0), n0 = 64 * blockIdx.x;
    list_adapters(a, m0, rows, &list);
    int parts = a.parts;
    if constexpr (FUSED) parts = shrink_rows<DT, RANK, NW, VEC>(a, list, m0, rows, 0, a.K, sum);
    const int n = __builtin_amdgcn_readfirstlane(list.n);
    for (int j = wave; j < n; j += NW) {
        const int ad = __builtin_amdgcn_readfirstlane(list.of[j]);
        const uint32_t those = (uint32_t)__builtin_amdgcn_readfirstlane((int)list.rows[j]);
        if (ad < 0) {   /* no adapter: Z as it is */
            if (a.z == a.y && a.ldz == a.ldy) continue;
            for (int r = 0; r < rows; r++)
                if (((those >> r) & 1) && n0 + lane < a.N)
                    static_cast<E *>(a.y)[(size_t)(m0 + r) * a.ldy + n0 + lane] =
                        a.z ? static_cast<const E *>(a.z)[(size_t)(m0 + r) * a.ldz + n0 + lane] : Elem<DT>::put(0.0f);
            continue;
        }
        /* everything that the rows need is requested before the first product */
        E b[4][RS];
#pragma unroll
        for (int t = 0; t < 4; t++)
            __builtin_memcpy(b[t], static_cast<const E *>(a.b) +
                                       ((size_t)ad * a.N + imin(n0 + expand_column<DT>(t, c), a.N - 1)) * RANK + RS * g, sizeof b[t]);
        const float scale = a.scale[ad];
        const bool whole = a.vec && n0 + 64 <= a.N, in = (those >> c) & 1;
        ExpandRows<DT> z;
        if (whole) z.load(a, in, m0 + c, n0, g);
        float h[RS];
#pragma unroll
        for (int s = 0; s < RS; s++) h[s] = 0.0f;
        if (in) {
#pragma unroll(RS <= 4 ? 8 : RS <= 8 ? 4 : DT != T_F32 ? 2 : 1)   /* what registers allow */
            for (int p = 0; p < parts; p++) {
                const float *from = FUSED ? &sum[FUSED ? p : 0][c][RS * g] : a.h + ((size_t)p * a.M + m0 + c) * RANK + RS * g;
#pragma unroll
                for (int s = 0; s < RS; s++) h[s] += from[s];
            }
        }
#pragma unroll
        for (int s = 0; s < RS; s++) h[s] *= scale;
        expand_rows<DT, RANK>(a, those, m0, n0, whole, z, h, b, tile[wave]);
    }
}

/* The same for many rows: 64 rows a workgroup, 16 a wave, its columns 64 at a time. Loads and stores go along rows: with lanes in
 * different rows, as the products have them, a CU takes four times as long for each. An adapter's 64 rows of B come through LDS,
 * shared by the waves, and each wave's sums leave through it. VEC: Z and Y are read and written 16 bytes at a time, Z through
 * LDS too; otherwise by the element. fp32, 6000 rows of 375 an adapter, N = 4096, rank 32: 48 us, 4.1 TB/s, bound by memory
 * (201 MB of H, Z, B and Y once, of which the counters see 241; 67 with the compiler's waits and lanes in different rows; both
 * products by 16 rows 246, by 64 66); bf16, 300 rows of 20 an adapter, N = 16384, rank 16: 16 us, N = 16389 27.
 *
 * Everything comes by direct loads, a step (64 columns of one adapter) or a unit (64 columns) ahead, and is waited for by
 * number: the compiler's own waits, which do not know how many stores a path has issued, would wait for all of them. Such a
 * number is that of loads and stores that are sure to have been issued since; `z_since` and `b_since` count them. */
template <int DT, int RANK> struct ExpandLds {
    typedef typename Elem<DT>::type E;
    static constexpr int VE = kPer16<DT>, BCH = RANK / VE, ZCH = 64 / VE;   /* 16-byte pieces of a row of B, of 64 columns */
    static constexpr int NB = BCH < 4 ? 1 : BCH / 4, NZ = ZCH / 4;          /* a wave's loads of 64 rows of B, of 16 of Z */
    E b[2][64 * RANK];
    union {
        E z[2][4][16 * 64];
        float sum[4][16 * 64];   /* VEC false: the sums alone */
    };
    /* where a row's piece lies, so that 16 rows' pieces fall into different banks */
    template <int CH> static __device__ __forceinline__ int place(int r, int p)
    {
        return p ^ (CH >= 16 ? r & 15 : (r / (16 / CH)) & (CH - 1));
    }
};

template <int DT, int RANK, bool VEC>
__global__ __launch_bounds__(256) void adapter_expand_rows(AdapterArgs a)
{
    typedef typename Elem<DT>::type E;
    typedef ExpandLds<DT, RANK> L;
    constexpr int RS = RANK / 4, VE = L::VE, BCH = L::BCH, ZCH = L::ZCH, NB = L::NB, RPL = 64 / ZCH,
                  NZ = VEC ? L::NZ : 0;   /* loads of 16 rows of Z, and stores, that are counted */
    __shared__ __align__(16) L lds;
    __shared__ AdapterList list;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int m0 = 64 * blockIdx.y, rows = imin(64, a.M - m0), mw = m0 + 16 * wave, have = rows - 16 * wave;   /* this wave's rows */
    const int u0 = blockIdx.x * a.units, units = imin(a.units, (a.N + 63) / 64 - u0);
    if (units <= 0) return;
    const E *const zp = static_cast<const E *>(a.z ? a.z : a.y);   /* without Z what is read is not used */
    const int ldz = a.z ? a.ldz : a.ldy, last_piece = a.N / VE - 1;   /* of a row's whole pieces */
    const int zr = lane / ZCH, zc = lane % ZCH;
    auto fetch_z = [&](int u, int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NZ; i++) {
            const int r = RPL * i + zr, row = m0 + imin(16 * wave + r, rows - 1);
            dma_16(zp + (size_t)row * ldz + VE * imin(64 / VE * u + L::template place<ZCH>(r, zc), last_piece), lds.z[buffer][wave] + 512 / (8 / VE) * i);
        }
    };
    if (VEC) fetch_z(u0, 0);   /* on its way while the adapters are looked up */
    list_adapters(a, m0, rows, &list);
    const int n = __builtin_amdgcn_readfirstlane(list.n);
    auto adapter_of = [&](int j) { return __builtin_amdgcn_readfirstlane(list.of[j]); };
    auto rows_of = [&](int j) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(list.rows[j] >> (16 * wave))) & 0xffffu; };
    /* rows of this wave with an adapter; this lane's row times its adapter's scale */
    uint32_t some = 0;
    float h[RS];
#pragma unroll
    for (int s = 0; s < RS; s++) h[s] = 0.0f;
    for (int j = 0; j < n; j++) {
        const int ad = adapter_of(j);
        if (ad < 0) continue;
        const uint32_t those = rows_of(j);
        some |= those;
        if ((those >> c) & 1) {
            const float scale = a.scale[ad];
#pragma unroll(RS <= 8 ? 8 : RS <= 16 ? 4 : 2)
            for (int p = 0; p < a.parts; p++) {
                const float *from = a.h + ((size_t)p * a.M + mw + c) * RANK + RS * g;
#pragma unroll
                for (int s = 0; s < RS; s++) h[s] += from[s];
            }
#pragma unroll
            for (int s = 0; s < RS; s++) h[s] *= scale;
        }
    }
    auto fetch_b = [&](int u, int ad, int buffer) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int load = BCH < 4 ? wave % BCH : NB * wave + i, at = 64 * load + lane, r = at / BCH;
            dma_16(static_cast<const E *>(a.b) + ((size_t)imax(ad, 0) * a.N + imin(64 * u + r, a.N - 1)) * RANK +
                       VE * L::template place<BCH>(r, at % BCH),
                   lds.b[buffer] + 64 * VE * load);
        }
    };
    E *const y = static_cast<E *>(a.y) + (size_t)mw * a.ldy;
    /* VEC false: a lane's column of 16 rows */
    const E *const zrow = static_cast<const E *>(a.z) + (size_t)mw * a.ldz;
    auto load_column = [&](int u, E (&z)[16]) __attribute__((always_inline)) {
        const int col = 64 * u + lane;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            z[r] = Elem<DT>::put(0.0f);
            if (a.z && r < have && col < a.N) z[r] = zrow[(size_t)r * a.ldz + col];
        }
    };
    const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
        y, 0, have > 0 ? (int)((uint32_t)((imin(have, 16) - 1) * a.ldy + a.N) * sizeof(E)) : 0, 0x00020000);

    fetch_b(u0, adapter_of(0), 0);
    int buffer = 0, b_since = 0, z_since = 0;   /* how many are sure to have been issued since the next step's B, the unit's Z */
    for (int k = 0; k < units; k++) {
        const int u = u0 + k;
        E zs[VEC ? 1 : 16];
        if constexpr (!VEC) load_column(u, zs);
        f4 sum[4];
#pragma unroll
        for (int t = 0; t < 4; t++) sum[t] = f4{0, 0, 0, 0};
        for (int j = 0; j < n; j++) {
            const bool end = j + 1 == n;
            const uint32_t those = rows_of(j);
            /* the next step's B and, in a unit's first step, the next unit's Z; past the last the same again, which nothing reads */
            fetch_b(u0 + imin(k + end, units - 1), adapter_of(end ? 0 : j + 1), buffer ^ 1);
            if (VEC && j == 0) fetch_z(u0 + imin(k + 1, units - 1), (k + 1) & 1);
            b_since += NB + (j == 0 ? NZ : 0);
            z_since += NB + (j == 0 ? NZ : 0);
            if (b_since >= NB + 3 * NZ) wait_vm<NB + 3 * NZ>();
            else if (b_since >= NB + 2 * NZ) wait_vm<NB + 2 * NZ>();
            else if (b_since >= NB + NZ) wait_vm<NB + NZ>();
            else wait_vm<NB>();
            lds_barrier();   /* everyone's part of B */
            b_since = j == 0 ? NZ : 0;
            if (those && adapter_of(j) >= 0) {
                const bool in = (those >> c) & 1;
                const E *from = lds.b[buffer];
                f4 acc[4];
                E v[4][RS];
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const int r = expand_column<DT>(t, c);
                    if constexpr (RS >= VE) {
#pragma unroll
                        for (int x = 0; x < RS / VE; x++)
                            __builtin_memcpy(v[t] + VE * x, __builtin_assume_aligned(from + r * RANK + VE * L::template place<BCH>(r, RS / VE * g + x), 16), 16);
                    } else {
                        __builtin_memcpy(v[t], __builtin_assume_aligned(from + r * RANK + VE * L::template place<BCH>(r, RS * g / VE) + RS * g % VE, sizeof v[t]),
                                         sizeof v[t]);
                    }
                    acc[t] = f4{0, 0, 0, 0};
                }
#pragma unroll
                for (int s = 0; s < RS; s++)
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(Elem<DT>::get(v[t][s]), h[s], acc[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) sum[t][i] = in ? acc[t][i] : sum[t][i];
            }
            lds_barrier();   /* everyone is done with this step's B */
            buffer ^= 1;
        }
        if constexpr (!VEC) {
            float *const own = lds.sum[wave];
#pragma unroll
            for (int t = 0; t < 4; t++)   /* columns expand_column(t, 4g) .. + 3: four neighbours */
                *reinterpret_cast<f4 *>(own + 64 * c + 4 * L::template place<16>(c, expand_column<DT>(t, 4 * g) / 4)) = sum[t];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int col = 64 * u + lane;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float add = own[64 * r + 4 * L::template place<16>(r, lane / 4) + lane % 4];
                if (r < have && col < a.N)
                    y[(size_t)r * a.ldy + col] = (some >> r) & 1 ? Elem<DT>::put(Elem<DT>::get(zs[r]) + add) : zs[r];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            continue;
        }
        if (z_since >= NB + 2 * NZ) wait_vm<NB + 2 * NZ>();
        else wait_vm<NB + NZ>();
        /* a lane's results are whole pieces of row c: into their places in LDS, and from there along rows */
        E *const zl = lds.z[k & 1][wave];
#pragma unroll
        for (int p = 0; p < 16 / VE; p++) {
            u4 *at = reinterpret_cast<u4 *>(zl + 64 * c + VE * L::template place<ZCH>(c, 4 * p + g));
            const u4 before = a.z ? *at : u4{0, 0, 0, 0};
            float v[VE];
            unpack<DT>(before, v);
#pragma unroll
            for (int x = 0; x < VE; x++) v[x] += sum[VE / 4 * p + x / 4][x % 4];
            *at = (some >> c) & 1 ? pack<DT>(v) : before;   /* a row without an adapter as it is */
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < NZ; i++) {
            const int r = RPL * i + zr, col = 64 * u + VE * zc;
            const u4 v = *reinterpret_cast<const u4 *>(zl + 64 * r + VE * L::template place<ZCH>(r, zc));
            const bool whole = r < have && col + VE <= a.N;   /* others leave past the end, which writes nothing */
            __builtin_amdgcn_raw_buffer_store_b128(v, out, whole ? (int)((uint32_t)(r * a.ldy + col) * sizeof(E)) : -16, 0, 0);
        }
        if (u == (a.N - 1) / 64 && a.N % VE != 0) {   /* the last columns, fewer than a piece: their Z was not loaded whole either */
            const int col = a.N / VE * VE, t = (col - 64 * u) / VE;
            if (g == t % 4 && c < have) {
                float v[VE];
#pragma unroll
                for (int x = 0; x < VE; x++) v[x] = 0.0f;
#pragma unroll
                for (int p = 0; p < 16 / VE; p++)
                    if (p == t / 4)
#pragma unroll
                        for (int x = 0; x < VE; x++) v[x] = sum[VE / 4 * p + x / 4][x % 4];
#pragma unroll
                for (int x = 0; x < VE; x++)
                    if (col + x < a.N) {
                        const E before = a.z ? static_cast<const E *>(a.z)[(size_t)(mw + c) * a.ldz + col + x] : Elem<DT>::put(0.0f);
                        y[(size_t)c * a.ldy + col + x] = (some >> c) & 1 ? Elem<DT>::put(Elem<DT>::get(before) + v[x]) : before;
                    }
            }
        }
        b_since += NZ;
        z_since = n > 1 ? 0 : NZ;
    }
    wait_vm<0>();   /* nothing comes into the LDS any more */
}

}  // namespace p2k
