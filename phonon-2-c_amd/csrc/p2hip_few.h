/*  p2hip_few.h – attention of up to 16 queries a wave over blocks of rows: the waves of a workgroup take the blocks in turn and
 *  join their sums.
 */
#pragma once

#include "p2hip_elem.h"
#include "p2hip_index.h"

namespace p2k {

/* The softmax state of up to 16 queries (lane % 16) over the blocks that one wave has taken: O^T tiles, the reference (the
 * running maximum less kLift) and this lane's share of the sum of weights. */
template <int DH> struct FewState {
    f4 o[DH / 16];
    float m, l;
    __device__ __forceinline__ FewState() : m(-INFINITY), l(0.0f)
    {
#pragma unroll
        for (int d = 0; d < DH / 16; d++) o[d] = f4{0, 0, 0, 0};
    }
};

/* A block of 32 (fp32: 16) keys from k0 on: each 16 of them, t, have their rows at k[t] and v[t], of which have[t] >= 1 can
 * be read; the rows behind are read as the last of these. `whole`: every query sees every key of the block, and what is
 * read is those. */
template <int DT> struct FewPlace {
    static constexpr int NB = DT == T_F32 ? 1 : 2, KB = 16 * NB;
    const typename Elem<DT>::type *k[NB], *v[NB];
    int have[NB], k0;
    bool whole, there[NB];   /* there: in a page of the cache (in its place page 0 is read) */
};

/* Its rows in registers, 16 bytes a lane along the rows; fp32 V as its operand takes it: a lane's four neighbouring
 * dimensions of a key belong to four products. */
template <int DT, int DH> struct FewRows {
    typedef typename Elem<DT>::type E;
    static constexpr int NB = FewPlace<DT>::NB, EPC = kPer16<DT>, CH = DH / EPC, RPL = 64 / CH, LD = 16 / RPL;
    u4 k[NB * LD], v[DT == T_F32 ? 4 * DH / 64 : NB * LD];
    static __device__ __forceinline__ u4 get(const E *p) { return *reinterpret_cast<const u4 *>(p); }
    static __device__ __forceinline__ u4 row_piece(const E *base, int have, int ld, int r)
    {
        const int lane = threadIdx.x & 63;
        return get(base + (size_t)imin(RPL * r + lane / CH, have - 1) * ld + EPC * (lane % CH));
    }
    __device__ __forceinline__ void keys(const FewPlace<DT> &p, int ld)
    {
#pragma unroll
        for (int x = 0; x < NB * LD; x++) k[x] = row_piece(p.k[x / LD], p.have[x / LD], ld, x % LD);
    }
    __device__ __forceinline__ void values(const FewPlace<DT> &p, int ld)
    {
        if constexpr (DT == T_F32) {
            const int g = (threadIdx.x & 63) >> 4, x16 = threadIdx.x & 15;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int d = 0; d < DH / 64; d++)
                    v[i * (DH / 64) + d] = get(p.v[0] + (size_t)imin(4 * g + i, p.have[0] - 1) * ld + 64 * d + 4 * x16);
        } else {
#pragma unroll
            for (int x = 0; x < NB * LD; x++) v[x] = row_piece(p.v[x / LD], p.have[x / LD], ld, x % LD);
        }
    }
    /* rows as they were read into LDS of that pitch */
    static __device__ __forceinline__ void put(const u4 *from, E *to, int pitch)
    {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int x = 0; x < NB * LD; x++)
            *reinterpret_cast<u4 *>(to + (RPL * x + lane / CH) * pitch + EPC * (lane % CH)) = from[x];
    }
};

/* Blocks b, b + step, … below `end` into the state of 16 queries: S^T = K·Q^T by 16 × 16 products, then O^T += V^T·P^T as in
 * attention_win; K passes through the wave's own LDS, as an operand's neighbouring lanes are in different rows, and a load
 * of such a pattern takes a CU four times as long as one along the rows; 16-bit V for its transposing read.
 *
 * A wave has nothing else to do while it waits for memory, so what the next block of 16-bit rows needs is requested as soon
 * as the registers are free: its keys behind the products with this block's, its values once these lie in LDS. fp32 rows
 * take the matrix unit eight times as long and wait for each block instead: requests ahead did not fit the 168 registers
 * that three waves a SIMD leave (a workgroup of eight waves is two a SIMD, so that heads of 128 could be given 256).
 * place_of(b, hint(b)) says where a block lies, from what hint read (a page table's entries) a block earlier. The last block
 * has code of its own, as the wait for a load that may or may not have been followed by others is a wait for all of them.
 * seen(p, k) says whether this lane's query sees key k of the block at p, and kept(p, k) whether V row k enters the product
 * at all; neither is asked where p.whole. CLEAN: infinities and NaN in V are put aside there, which `odd` notes.
 *
 * 16-bit weights are rounded for their product with V, as attention_win says; a second product with the rest would cost 2 to
 * 9 % (32 sequences of 8192 bf16 tokens 187 -> 190 us, 16 of 1000 18.5 -> 20.2). */
template <int DT, int DH, bool CLEAN, class Hint, class PlaceOf, class Seen, class Kept>
__device__ __forceinline__ void few_blocks(FewState<DH> &st, const u4 (&q)[DH / (4 * kPer16<DT>)], float c, int b, int end,
                                           int step, int ldk, int ldv, Hint hint, PlaceOf place_of, Seen seen, Kept kept,
                                           bool &odd, unsigned char *own)
{
    typedef typename Elem<DT>::type E;
    typedef FewRows<DT, DH> Rows;
    constexpr int NT = DH / 16, VP = DH + 16, KP = DH + kPer16<DT>;   /* pitches that keep a read's rows in different banks */
    const int lane = threadIdx.x & 63, g = lane >> 4, x16 = lane & 15;
    if (b >= end) return;
    auto soften = [&](float top) __attribute__((always_inline)) {
        const float mn = fmaxf(st.m, lifted(max_quarters(top), c, kLift<DT>)), mu = mn == -INFINITY ? 0.0f : mn;
        const float fade = exp2_fast(st.m - mu);
        st.m = mn;
        return float2{mu, fade};
    };
    /* a wave's LDS operations complete in order, and no other wave touches its part; the fences keep the compiler from
     * moving reads and writes across each other */
    auto order = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    E *Ks = reinterpret_cast<E *>(own);
    uint16_t *Vs = reinterpret_cast<uint16_t *>(own);
    auto key = [&](int t, int x) __attribute__((always_inline)) {   /* the operand of keys 16t .., pieces 4x .. */
        return *reinterpret_cast<const u4 *>(Ks + (16 * t + x16) * KP + kPer16<DT> * (4 * x + g));
    };
    Rows rows;
    FewPlace<DT> now, next;
    auto ahead = hint(b);
    auto block = [&](auto last) __attribute__((always_inline)) {
        constexpr bool MORE = !decltype(last)::value;
        if constexpr (MORE) {
            next = place_of(b + step, ahead);
            ahead = hint(imin(b + 2 * step, end - 1));
        }
        Rows::put(rows.k, Ks, KP);
        order();
        if constexpr (DT == T_F32) {
            f4 s = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < NT; x++) {
                const u4 k = key(0, x);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[x][e]), s, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e + 1]), __uint_as_float(q[x][e + 1]), s1, 0,
                                                              0, 0);
                }
            }
            order();
            s += s1;
            if (!now.whole) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (!seen(now, 4 * g + i)) s[i] = -INFINITY;
                    const bool keep = kept(now, 4 * g + i);
#pragma unroll
                    for (int d = 0; d < NT; d++) {
                        uint32_t &v = reinterpret_cast<uint32_t *>(&rows.v[i * (DH / 64) + d / 4])[d % 4];
                        const bool fin = !CLEAN || __builtin_fabsf(__uint_as_float(v)) < INFINITY;
                        odd |= keep && !fin;
                        if (!keep || !fin) v = 0u;
                    }
                }
            }
            const float2 mf = soften(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[i] = exp2_fast(__builtin_fmaf(s[i], c, -mf.x));
                sum += s[i];
            }
            st.l = __builtin_fmaf(st.l, mf.y, sum);
#pragma unroll
            for (int d = 0; d < NT; d++) st.o[d] *= mf.y;
#pragma unroll
            for (int i = 0; i < 4; i++)   /* neighbouring products do not wait for each other */
#pragma unroll
                for (int d = 0; d < NT; d++)
                    st.o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(rows.v[i * (DH / 64) + d / 4][d % 4]), s[i],
                                                                   st.o[d], 0, 0, 0);
        } else {
            constexpr int CH = Rows::CH, RPL = Rows::RPL;   /* pieces of a row, rows per load */
            f4 s[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[t] = f4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < DH / 32; x++) s[t] = mfma16<DT>(key(t, x), q[x], s[t]);
            }
            order();
            if constexpr (MORE) rows.keys(next, ldk);
            if (!now.whole) {
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (!seen(now, 16 * t + 4 * g + i)) s[t][i] = -INFINITY;
#pragma unroll
                for (int r = 0; r < 32 / RPL; r++) {
                    if (!kept(now, RPL * r + lane / CH)) rows.v[r] = u4{0, 0, 0, 0};
                    if (CLEAN && odd_values<DT>(rows.v[r])) {
                        odd = true;
                        rows.v[r] = only_finite<DT>(rows.v[r]);
                    }
                }
            }
            Rows::put(rows.v, Ks, VP);
            if constexpr (MORE) rows.values(next, ldv);
            const float2 mf = soften(fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                           fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))));
            float sum = 0.0f, w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                w[i] = exp2_fast(__builtin_fmaf(s[i / 4][i % 4], c, -mf.x));
                sum += w[i];
            }
            st.l = __builtin_fmaf(st.l, mf.y, sum);
            const u4 pw = pack<DT>(w);
            order();
            const uint16_t *vp = Vs + (4 * g + (x16 >> 2)) * VP + 4 * (x16 & 3);
#pragma unroll
            for (int d = 0; d < NT; d++) {
                const u2 va = lds_tr(vp + 16 * d), vb2 = lds_tr(vp + 16 * VP + 16 * d);
                st.o[d] = mfma16<DT>(u4{va[0], va[1], vb2[0], vb2[1]}, pw, st.o[d] * mf.y);
            }
            order();
        }
    };
    if constexpr (DT == T_F32) {
        for (; b < end; b += step) {
            now = place_of(b, ahead);
            ahead = hint(imin(b + step, end - 1));
            rows.keys(now, ldk);
            rows.values(now, ldv);
            block(std::true_type{});
        }
    } else {
        now = place_of(b, ahead);
        ahead = hint(imin(b + step, end - 1));
        rows.keys(now, ldk);
        rows.values(now, ldv);
        for (; b + step < end; b += step) {
            block(std::false_type{});
            now = next;
        }
        block(std::true_type{});
    }
}

/* the waves' states into LDS as [wave][16 queries][DH + 2], the last two the reference and the sum, and one output of their
 * join: sums relative to the largest reference, which is returned */
template <int DT, int DH> __device__ __forceinline__ void few_store(FewState<DH> &st, float *J)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const float l = sum_quarters(st.l);
    __syncthreads();   /* the waves' own parts are done with */
    float *mine = J + (wave * 16 + (lane & 15)) * (DH + 2);
#pragma unroll
    for (int d = 0; d < DH / 16; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)   /* fp32: product d has every fourth of 64 dimensions */
            mine[DT == T_F32 ? 64 * (d / 4) + 4 * (4 * g + i) + d % 4 : 16 * d + 4 * g + i] = st.o[d][i];
    if (g == 0) {
        mine[DH] = st.m;
        mine[DH + 1] = l;
    }
    __syncthreads();
}
template <int DH, int NW, int ROWS = 16>
__device__ __forceinline__ void few_join(const float *J, int r, int d, float *top, float *num, float *den)
{
    float t = -INFINITY, n = 0.0f, e = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; w++) t = fmaxf(t, J[(w * ROWS + r) * (DH + 2) + DH]);
    const float mu = t == -INFINITY ? 0.0f : t;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        const float *j = J + (w * ROWS + r) * (DH + 2);
        const float f = exp2_fast(j[DH] - mu);
        n = __builtin_fmaf(f, j[d], n);
        e = __builtin_fmaf(f, j[DH + 1], e);
    }
    *top = t;
    *num = n;
    *den = e;
}

/* a wave's own part: 16-bit V, or fp32 K */
template <int DT, int DH> constexpr int few_own_bytes() { return DT == T_F32 ? 16 * (DH + 4) * 4 : 32 * (DH + 16) * 2; }
template <int DT, int DH, int NW> constexpr int few_lds_bytes()
{
    constexpr int V = NW * few_own_bytes<DT, DH>(), J = NW * 16 * (DH + 2) * 4;
    return V > J ? V : J;
}

}  // namespace p2k
