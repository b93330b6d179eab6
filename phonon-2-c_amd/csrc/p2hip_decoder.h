/*  p2hip_decoder.h – gfx950 kernels of a decoder layer's step (included once, by p2hip_decoder.hip).
 *
 *  Kernels:
 *    q4_records      4-bit codes, scales and zero points re-laid per matrix-core operand at upload
 *    q4_gemv         few rows times a 4-bit weight
 *    qk_norm_rope    norm and rotation of query and key heads, keys and values into cache pages
 *    attention_win   attention of ragged sequences over a window and first keys
 *    attention_page  one query per sequence over a paged cache; attention_join adds the parts of a split sequence
 */
#pragma once

#include "p2hip_async.h"
#include "p2hip_elem.h"
#include "p2hip_few.h"
#include "p2hip_index.h"

namespace p2k {

/* ── 4-bit weights ─────────────────────────────────────────────────────────────────────────────────────────── */

/* Records: for each 16 columns and 128 rows 64 lanes × 16 bytes, word b of lane l holding column l % 16's codes of rows
 * 32b + 8(l / 16) + j, j = 0..7: the operand of one 16 × 16 × 32 product. Code j sits in nibble j / 2 + 4·(j & 1), so
 * that one mask takes two neighbouring rows. Scales: [column tile][unit][16 columns][groups in a unit], fp16 (SCALE2:
 * with the zero point's half after each). Rows past K and columns past N have code 0 and scale 0. */
__global__ void q4_records(int K, int N, int group, int tiles, int units, const uint8_t *__restrict__ codes,
                           const uint16_t *__restrict__ scales, const uint8_t *__restrict__ zeros,
                           uint32_t *__restrict__ rec, uint16_t *__restrict__ sc)
{
    const size_t half = ((size_t)N + 1) / 2, n_rec = (size_t)tiles * units * 256;
    const int gpu = 128 / group;
    const size_t n_sc = (size_t)tiles * units * 16 * gpu;
    const size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n_rec) {
        const int b = (int)(i & 3), l = (int)(i >> 2) & 63;
        const size_t tu = i >> 8;
        const int u = (int)(tu % units), t = (int)(tu / units);
        const int n = 16 * t + (l & 15);
        uint32_t r = 0;
        if (n < N)
            for (int j = 0; j < 8; j++) {
                const long long k = 128ll * u + 32 * b + 8 * (l >> 4) + j;
                if (k < K) r |= ((codes[(size_t)k * half + (n >> 1)] >> (4 * (n & 1))) & 15u) << (4 * (j / 2 + 4 * (j & 1)));
            }
        rec[i] = r;
    }
    if (i < n_sc) {
        const int g = (int)(i % gpu), c = (int)(i / gpu) & 15;
        const size_t tu = i / gpu / 16;
        const int u = (int)(tu % units), t = (int)(tu / units);
        const long long gr = (long long)u * gpu + g;
        const int n = 16 * t + c;
        const bool in = n < N && gr * group < K;
        const uint16_t s = in ? scales[(size_t)gr * N + n] : 0;
        if (zeros) {
            const int z = in ? (zeros[(size_t)gr * half + (n >> 1)] >> (4 * (n & 1))) & 15 : 8;
            sc[2 * i] = s;
            sc[2 * i + 1] = (uint16_t)(0xe400 | z);   /* −(1024 + z) as fp16 */
        } else {
            sc[i] = s;
        }
    }
}

struct Q4Args {
    int M, N, K, units, ldx, ldy, vec;
    float alpha, beta;
    const void *x;
    void *y;
    const u4 *rec;
    const void *sc;
};

/* A record word's eight codes as matrix-core operand. fp16: code − zero; 1024 + code has the code in its low bits, 1024 + 16
 * code where it lies four bits up, and adding −(1024 + zero), or a sixteenth and −(64 + zero), is exact: 9 instructions
 * for 8 weights. bf16: the same by way of fp32, of which the upper halves are all there is: 25; or (CODES) the code, as
 * fp8 (e4m3) has 0 .. 15 times 2^-9 in the bits 0 .. 15, which one conversion turns into two bf16 values: 8. */
template <int DT, bool CODES = false>
__device__ __forceinline__ u4 q4_operand(uint32_t w, _Float16 bias, uint32_t low, uint32_t magic)
{
    u4 v;
    if constexpr (CODES) {
        typedef __bf16 bb __attribute__((ext_vector_type(2)));
        w = __builtin_amdgcn_perm(w, w, 0x03010200u);   /* nibbles i and i + 4 into neighbouring bytes */
        const uint32_t a = w & 0x0f0f0f0fu, b = (w >> 4) & 0x0f0f0f0fu;
        v[0] = __builtin_bit_cast(uint32_t, (bb)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, false));
        v[1] = __builtin_bit_cast(uint32_t, (bb)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, false));
        v[2] = __builtin_bit_cast(uint32_t, (bb)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, true));
        v[3] = __builtin_bit_cast(uint32_t, (bb)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, true));
    } else {
        const h2 one = {bias, bias}, up = {(_Float16)0.0625f, (_Float16)0.0625f};
        const h2 six = one + h2{(_Float16)960.0f, (_Float16)960.0f};   /* −(64 + zero) */
        const uint32_t w8 = w >> 8;
        h2 d[4];
        d[0] = __builtin_bit_cast(h2, (w & low) | magic) + one;
        d[1] = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & (low << 4)) | magic), up, six);
        d[2] = __builtin_bit_cast(h2, (w8 & low) | magic) + one;
        d[3] = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w8 & (low << 4)) | magic), up, six);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == T_F16) v[i] = __builtin_bit_cast(uint32_t, d[i]);
            else v[i] = __builtin_amdgcn_perm(__float_as_uint((float)d[i][1]), __float_as_uint((float)d[i][0]), 0x07060302u);
        }
    }
    return v;
}

/* Eight fp32 values as three bf16 pieces each, the upper 16 bits of what is left after the pieces before: exact, as 8 + 8
 * + 8 bits hold the 24 of a float (down to 2^-110: bf16 ends at 2^-133). Nothing is left of an infinity
 * where they are looked for (INF), a NaN otherwise. */
template <bool INF> __device__ __forceinline__ void cut3(u4 lo, u4 hi, u4 (&xp)[3])
{
    uint32_t v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
    for (int p = 0; p < 3; p++) {
#pragma unroll
        for (int i = 0; i < 4; i++) xp[p][i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302u);
        if (p == 2) break;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float left = __uint_as_float(v[j]) - __uint_as_float(v[j] & 0xffff0000u);
            v[j] = INF && p == 0 && (v[j] & 0x7fffffffu) == 0x7f800000u ? 0u : __float_as_uint(left);
        }
    }
}

/* Y rows 16·blockIdx.y .. of 16·NT columns: each of the WV waves sums its 128-row units of K, unit after unit, and the
 * waves' sums are added in order in LDS. A group's products are summed as whole (code − zero) times x, exact factors in
 * both operands, and scaled once per group in 32 bits.
 *
 * fp16 rows multiply as fp16, with code − zero. bf16 rows multiply as bf16 (whole numbers up to 15 are exact there too),
 * with the codes themselves; the zero point times the sum of the group's x, a product with ones, goes off the group's sum.
 * fp32 rows are cut into three bf16 pieces, which sum to the row exactly: three products into the same sums. Sums of codes
 * are up to twice as large as sums of code − zero, which costs a bit of the 32-bit sums: fp32 rows come within 1.2e-7 to
 * 3.6e-7 of the exact result (relative, 2-norm; a single row by groups of 128 without zero points 5.9e-7), where a
 * host library's fp32 product comes within 1.8e-7 to 1.5e-6. A row whose sum of x in a unit is
 * not finite takes that unit's products with code − zero, as an infinity would meet itself; the rows beside it do not
 * change. Operand rows past M repeat the last row and are not stored.
 *
 * ONE: a single fp32 row, which each wave cuts through its part of the LDS, two values a lane; otherwise all 16 lanes of
 * an operand column group would cut the same values.
 *
 * What a unit needs from memory (a record of 1 KB per 16 columns, its scales, 128 values of each row) is requested while
 * the unit before is multiplied. The rows' values are read along the rows and turned into operands through the wave's LDS:
 * read as operands, neighbouring lanes would be in different rows, and such a load takes a CU four times as long (fp16 13 x
 * 8192 x 16389: 28 us, with the waits for the next unit's loads that conditional loads bring; now 21.6). Rows that end
 * inside a unit or are not 16-byte aligned are read by the element.
 *
 * Bound by memory where the weight is large: those 73 MB at 3.4 TB/s from HBM (a copy reaches 4.8), 17.6 us where the
 * memory-side cache holds part of it; 1 x 1024 x 1024 takes 2.5 us, a launch and a few waits. */
template <int DT, int GROUP, bool ZP, int WV, int NT, bool ONE>
__global__ __launch_bounds__(64 * WV) void q4_gemv(Q4Args a)
{
    typedef typename Elem<DT>::type E;
    constexpr int GPU = 128 / GROUP, NP = DT == T_F32 ? 3 : 1;
    constexpr int VE = kPer16<DT>, PR = 128 / VE, XL = ONE ? 1 : 16 * PR / 64;   /* 16-byte pieces of a row; a lane's loads */
    __shared__ float part[WV][256 * NT];
    /* by wave, a unit's 128 values: of 16 rows, a row's pieces followed by an empty one, so that 16 rows' pieces lie in
     * different banks; ONE: of each of the row's three bf16 parts */
    __shared__ __align__(16) u4 stage[WV][ONE ? 3 * 16 : 16 * (PR + 1)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int m0 = 16 * blockIdx.y, rows = imin(16, a.M - m0), tile0 = blockIdx.x * NT;
    const int tiles = (a.N + 15) / 16;
    const E *x = static_cast<const E *>(a.x) + (size_t)m0 * a.ldx;
    uint32_t at[XL];   /* this lane's pieces: 64 lanes read 64 / PR rows' 256 (fp32: 512) bytes */
#pragma unroll
    for (int i = 0; i < XL; i++)
        at[i] = (uint32_t)imin(64 / PR * i + lane / PR, rows - 1) * (uint32_t)a.ldx + VE * (lane % PR);
    uint32_t low = 0x000f000fu, magic = 0x64006400u;   /* kept in registers: an instruction takes one constant */
    asm("" : "+v"(low), "+s"(magic));

    struct Unit {
        u4 rec[NT], x[XL];   /* ONE: this lane's two of the row's 128 values, in x[0] */
        uint32_t sc[NT][GPU];   /* ZP: scale and bias; else the scale's bits */
    };
    const int whole = ONE || a.vec ? a.K / 128 : 0;   /* units whose rows are read 16 bytes (ONE: 8) at a time */
    auto load = [&](Unit &n, int u, auto all) __attribute__((always_inline)) {   /* all: a whole unit */
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const size_t tu = (size_t)imin(tile0 + t, tiles - 1) * a.units + u;
            n.rec[t] = a.rec[tu * 64 + lane];
#pragma unroll
            for (int q = 0; q < GPU; q++)
                n.sc[t][q] = ZP ? static_cast<const uint32_t *>(a.sc)[(tu * 16 + c) * GPU + q]
                                : (uint32_t) static_cast<const uint16_t *>(a.sc)[(tu * 16 + c) * GPU + q];
        }
        if constexpr (ONE) {
            const long long k = 128ll * u + 2 * lane;
            const float *xf = static_cast<const float *>(a.x);
            n.x[0][0] = decltype(all)::value || k < a.K ? __float_as_uint(xf[k]) : 0u;
            n.x[0][1] = decltype(all)::value || k + 1 < a.K ? __float_as_uint(xf[k + 1]) : 0u;
        } else if constexpr (decltype(all)::value) {
#pragma unroll
            for (int i = 0; i < XL; i++) n.x[i] = *reinterpret_cast<const u4 *>(x + 128 * u + at[i]);
        } else {
#pragma unroll
            for (int i = 0; i < XL; i++) {
                const E *row = x + (size_t)imin(64 / PR * i + lane / PR, rows - 1) * a.ldx;
                E v[VE];
#pragma unroll
                for (int j = 0; j < VE; j++) {
                    const long long k = 128ll * u + VE * (lane % PR) + j;
                    v[j] = k < a.K ? row[k] : Elem<DT>::put(0.0f);
                }
                __builtin_memcpy(&n.x[i], v, sizeof v);
            }
        }
    };
    /* a wave's LDS operations complete in order, and no other wave touches its part; the fences keep the compiler from
     * moving reads and writes across each other */
    auto settle = [] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    auto put = [&](const Unit &n) __attribute__((always_inline)) {
        if constexpr (!ONE) {
            settle();
#pragma unroll
            for (int i = 0; i < XL; i++) stage[wave][(64 / PR * i + lane / PR) * (PR + 1) + lane % PR] = n.x[i];
            settle();
        }
    };
    f4 total[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) total[t] = f4{0, 0, 0, 0};
    /* one unit into total; CODES: the sums of x that go with it, of this lane's rows 4g + i */
    auto add = [&](const Unit &n, auto codes) __attribute__((always_inline)) {
        constexpr bool CODES = decltype(codes)::value;
        const u4 one = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
        if constexpr (ONE) {
            /* this lane's two values cut as cut3 does, into the wave's LDS: 128 of each piece */
            uint32_t v[2] = {n.x[0][0], n.x[0][1]};
#pragma unroll
            for (int p = 0; p < 3; p++) {
                reinterpret_cast<uint32_t *>(stage[wave])[64 * p + lane] = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float left = __uint_as_float(v[j]) - __uint_as_float(v[j] & 0xffff0000u);
                    v[j] = !CODES && p == 0 && (v[j] & 0x7fffffffu) == 0x7f800000u ? 0u : __float_as_uint(left);
                }
            }
            settle();
        }
        f4 acc[NT], ones = {0, 0, 0, 0}, every = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = f4{0, 0, 0, 0};
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const bool last = (b + 1) % (GROUP / 32) == 0;   /* of its group */
            u4 xp[NP];
            const u4 *mine = stage[wave] + c * (PR + 1) + PR / 4 * b + PR / 16 * g;
            if constexpr (ONE)
#pragma unroll
                for (int p = 0; p < NP; p++) xp[p] = stage[wave][16 * p + 4 * b + g];
            else if constexpr (DT == T_F32) cut3<!CODES>(mine[0], mine[1], xp);
            else xp[0] = mine[0];
            if constexpr (CODES)
#pragma unroll
                for (int p = 0; p < NP; p++) ones = mfma16<T_BF16>(xp[p], one, ones);
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const uint32_t s = n.sc[t][b * GPU / 4];
                const h2 sb = __builtin_bit_cast(h2, s);
                const _Float16 bias = ZP ? sb[1] : (_Float16)-1032.0f;
                const u4 wv = q4_operand<DT, CODES>(n.rec[t][b], bias, low, magic);
#pragma unroll
                for (int p = 0; p < NP; p++) acc[t] = mfma16<DT == T_F16 ? T_F16 : T_BF16>(xp[p], wv, acc[t]);
                if (last) {
                    if constexpr (CODES) acc[t] += ((float)bias + 1024.0f) * ones;
                    total[t] += (float)sb[0] * acc[t];
                    acc[t] = f4{0, 0, 0, 0};
                }
            }
            if (CODES && last) {
                every += ones;
                ones = f4{0, 0, 0, 0};
            }
        }
        return every;
    };
    auto multiply = [&](const Unit &n) __attribute__((always_inline)) {
        if constexpr (DT == T_F16) {
            add(n, std::false_type{});
        } else {
            f4 before[NT];
#pragma unroll
            for (int t = 0; t < NT; t++) before[t] = total[t];
            const f4 every = add(n, std::true_type{});
            const float all = (every[0] + every[1]) + (every[2] + every[3]);
            if (__any(!(__builtin_fabsf(all) < INFINITY))) {
                f4 by_codes[NT];
                Unit again = n;   /* as if loaded anew, or the compiler keeps what both have in common in registers */
                if constexpr (ONE) asm volatile("" : "+v"(again.x[0]));
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    asm volatile("" : "+v"(again.rec[t]));
                    by_codes[t] = total[t];
                    total[t] = before[t];
                }
                add(again, std::false_type{});
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (__builtin_fabsf(every[i]) < INFINITY) total[t][i] = by_codes[t][i];
            }
        }
    };
    Unit n, now;
    int u = wave;
    if (u < whole) load(n, u, std::true_type{});
    for (; u < whole; u += WV) {
        put(n);
        now = n;
        __builtin_amdgcn_sched_barrier(0);   /* the next unit's loads leave before this one's products */
        if (u + WV < whole) load(n, u + WV, std::true_type{});
        __builtin_amdgcn_sched_barrier(0);
        multiply(now);
    }
    for (; u < a.units; u += WV) {
        load(n, u, std::false_type{});
        put(n);
        multiply(n);
    }
    /* row 4g + i, column c of this wave's sums */
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[wave][(4 * g + i) * 16 * NT + 16 * t + c] = total[t][i];
    __syncthreads();
    for (int t = threadIdx.x; t < 16 * NT * rows; t += 64 * WV) {
        const int n = 16 * tile0 + t % (16 * NT);
        float s = part[0][t];
#pragma unroll
        for (int w = 1; w < WV; w++) s += part[w][t];
        if (n < a.N) {
            E *y = static_cast<E *>(a.y) + (size_t)(m0 + t / (16 * NT)) * a.ldy + n;
            s *= a.alpha;
            if (a.beta != 0.0f) s = __builtin_fmaf(a.beta, Elem<DT>::get(*y), s);
            *y = Elem<DT>::put(s);
        }
    }
}

/* ── head norms, rotation and the cache ────────────────────────────────────────────────────────────────────── */

struct RopeArgs {
    int T, heads, kv, rot, interleaved;
    int ldx, ldq, ldk, page_shift;
    long long slots_in_cache;   /* pages · page, 0 without a cache */
    float eps;
    const void *x;
    void *q, *k, *kc, *vc;
    const float *gq, *gk, *freq;
    const int *pos, *slots;
    float *ks, *vs;   /* Q8: the scales of kc's and vc's codes */
};

/* A head's values v (LPH lanes of VE each, x = lane of the head) as 8-bit codes at `to` and their scale at `s`: scale = largest
 * |value| / 127, code = round-half-even(value · (127 / largest)), so that a value is off by half a step of its head's
 * largest / 127. Below 2^-100 a head is zeros; one with a value that is not finite has a NaN as its scale. */
template <int VE, int LPH> __device__ __forceinline__ void put_codes(const float (&v)[VE], int x, int8_t *to, float *s)
{
    uint32_t top = 0;   /* bits of |value|: in the order of the values, infinities and NaN above all */
#pragma unroll
    for (int i = 0; i < VE; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < LPH; o *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, o, LPH));
    const bool finite = top < 0x7f800000u, some = finite && top >= 0x0d800000u;   /* 2^-100 */
    const float most = __uint_as_float(top), by = some ? 127.0f / most : 0.0f;
    uint32_t w[VE / 4];
#pragma unroll
    for (int i = 0; i < VE / 4; i++) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int code = some ? (int)__builtin_rintf(v[4 * i + j] * by) : 0;
            w[i] |= ((uint32_t)code & 0xffu) << (8 * j);
        }
    }
    __builtin_memcpy(__builtin_assume_aligned(to + VE * x, VE), w, VE);
    if (x == 0) *s = some ? most / 127.0f : finite ? 0.0f : __builtin_nanf("");
}

/* One workgroup of NTHR threads per row: 16 bytes of a head per lane, a head's lanes side by side, so that the mean square
 * is a reduction inside a row of lanes. The row's angles are made once, in 64 bits, as turns reduced to an eighth of a
 * circle (float then holds them to 2^-27 of a radian), and their sines and cosines are shared by all heads through LDS,
 * while the row's first values are on their way. Bound by memory: 6000 rows of 32 + 8 + 8 bf16 heads, 147 MB, in 33.5 us
 * (4.4 TB/s, a copy reaches 4.8); loading 4 heads a thread ahead took 35.9, making the angles before the first load 34.6.
 * Few rows take 1024 threads, all of a row's heads at once (16 rows 3.9 us, 5.7 with 256 threads). Heads whose squares
 * leave the range of 32 bits (values from 2^60 up; without an eps to speak of, below 2^-48) are moved into it first. */
template <int DT, int DH, int NTHR, bool Q8>
__global__ __launch_bounds__(NTHR) void qk_norm_rope(RopeArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int VE = kPer16<DT>, LPH = DH / VE, HPP = NTHR / LPH;
    __shared__ float2 turn[DH / 2];   /* (cos, sin) */
    const int t = blockIdx.x, hl = threadIdx.x / LPH, l = threadIdx.x % LPH, half = a.rot / 2;
    const E *row = static_cast<const E *>(a.x) + (size_t)t * a.ldx;
    const int n_heads = a.heads + a.kv * (a.slots_in_cache ? 2 : 1);
    long long slot = -1;
    if (a.slots_in_cache) {
        slot = a.slots[t];
        if (slot >= a.slots_in_cache) slot = -1;
    }
    for (int h0 = 0; h0 < n_heads; h0 += HPP) {
        const int h = h0 + hl;
        u4 raw = {0, 0, 0, 0};
        if (h < n_heads) raw = *reinterpret_cast<const u4 *>(row + (size_t)h * DH + VE * l);
        if (h0 == 0) {
            if ((int)threadIdx.x < half) {
                const double turns = (double)a.pos[t] * (double)a.freq[threadIdx.x] * 0.15915494309189533577;
                const double f = turns - __builtin_rint(turns), qd = __builtin_rint(4.0 * f);
                const float r = (float)(f - 0.25 * qd);   /* |r| <= 1/8 turn */
                float s, c;
                sincospif(2.0f * r, &s, &c);
                const int q = (int)qd & 3;
                const float cs = (q & 1) ? s : c, sn = (q & 1) ? c : s;
                turn[threadIdx.x] = float2{(q == 1 || q == 2) ? -cs : cs, (q & 2) ? -sn : sn};
            }
            __syncthreads();
        }
        if (h >= n_heads) break;
        u4 res = raw;
        float v[VE];
        const bool is_q = h < a.heads, is_v = h >= a.heads + a.kv;
        if (!is_v) {   /* the same for all lanes of a head */
            float gm[VE];
#pragma unroll
            for (int i = 0; i < VE; i++) gm[i] = (is_q ? a.gq : a.gk)[VE * l + i];   /* on their way during the sum */
            unpack<DT>(raw, v);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; i++) ss = __builtin_fmaf(v[i], v[i], ss);
#pragma unroll
            for (int o = 1; o < LPH; o *= 2) ss += __shfl_xor(ss, o, LPH);
            float eps = a.eps;
            if (DT != T_F16 && __builtin_expect(!(ss < INFINITY) || (ss < 0x1p-90f && eps < 0x1p-60f), false)) {
                /* squares that leave the range of 32 bits, the same for all lanes of a head: of the head times a power of two */
                const float by = ss < 1.0f ? 0x1p90f : 0x1p-68f;
                eps = eps * by * by;
                ss = 0.0f;
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    v[i] *= by;
                    ss = __builtin_fmaf(v[i], v[i], ss);
                }
#pragma unroll
                for (int o = 1; o < LPH; o *= 2) ss += __shfl_xor(ss, o, LPH);
            }
            const float inv = 1.0f / sqrtf(ss * (1.0f / DH) + eps);
#pragma unroll
            for (int i = 0; i < VE; i++) v[i] = v[i] * inv * gm[i];
            if (a.interleaved) {
                if (VE * l < a.rot) {
#pragma unroll
                    for (int i = 0; i < VE; i += 2) {
                        const float2 cs = turn[(VE * l + i) / 2];
                        const float x = v[i], y = v[i + 1];
                        v[i] = x * cs.x - y * cs.y;
                        v[i + 1] = y * cs.x + x * cs.y;
                    }
                }
            } else if (a.rot) {
                /* elements i and i + rot / 2 are rot / 2 / VE lanes apart: rot is a multiple of 16 */
                const int d = half / VE;
                const bool lo = l < d, in = l < 2 * d;
                const int from = lo ? l + d : in ? l - d : l;
#pragma unroll
                for (int i = 0; i < VE; i++) {
                    const float o = __shfl(v[i], from, LPH);
                    const float2 cs = turn[(VE * (lo ? l : in ? l - d : 0) + i) & (DH / 2 - 1)];
                    if (in) v[i] = lo ? v[i] * cs.x - o * cs.y : v[i] * cs.x + o * cs.y;
                }
            }
            res = pack<DT>(v);
        }
        const int hk = is_q ? 0 : (h - a.heads) % a.kv;
        if (is_q)
            *reinterpret_cast<u4 *>(static_cast<E *>(a.q) + (size_t)t * a.ldq + (size_t)h * DH + VE * l) = res;
        else if (!is_v && a.k)
            *reinterpret_cast<u4 *>(static_cast<E *>(a.k) + (size_t)t * a.ldk + (size_t)hk * DH + VE * l) = res;
        if (!is_q && slot >= 0) {
            const size_t page = (size_t)(slot >> a.page_shift), off = (size_t)slot & ((1u << a.page_shift) - 1);
            const size_t head = ((page * a.kv + hk) << a.page_shift) + off;
            if constexpr (Q8) {   /* keys from their 32-bit values; values have not been through the norm */
                if (is_v) unpack<DT>(raw, v);
                put_codes<VE, LPH>(v, l, static_cast<int8_t *>(is_v ? a.vc : a.kc) + head * DH, (is_v ? a.vs : a.ks) + head);
            } else {
                E *to = static_cast<E *>(is_v ? a.vc : a.kc) + head * DH + VE * l;
                *reinterpret_cast<u4 *>(to) = res;
            }
        }
    }
}

/* ── attention over a window ───────────────────────────────────────────────────────────────────────────────── */

struct WinArgs {
    int q_rows, k_rows, n_seqs, heads, kv, ldq, ldk, ldv, ldo, window, ahead, sinks, tiles, hpw;
    int turn;   /* workgroups from this one on take the tiles from the first on (win_tile_of) */
    float c;   /* scale · log2 e */
    const int *qs, *ks;
    const void *q, *k, *v;
    void *o;
};

/* A sequence's query rows [qa, qb) and key rows [ka, kb), and one of its tiles. */
struct WinSeq {
    int qa, qb, ka, kb, tile;
};

/* The sequence that tile number `id` of `rows` queries falls to and which of its tiles it is: the last sequence whose first
 * number (tile_start) is not above it, looked for by 64 lanes at once, so that up to 64 sequences take one wait for memory
 * and 4096 two. False where the sequence has no such tile. */
__device__ __forceinline__ bool find_tile(const WinArgs &a, int rows, int id, WinSeq *seq)
{
    if (!a.qs) {
        *seq = WinSeq{0, a.q_rows, 0, a.k_rows, id};
        return (long long)id * rows < a.q_rows;
    }
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = a.n_seqs;   /* it is one of these */
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) / 64, s = lo + lane * step;
        const int k = __popcll(__ballot(s < hi && tile_start(a.qs, s, a.q_rows, rows) <= id));
        lo += imax(k - 1, 0) * step;
        hi = imin(lo + step, hi);
    }
    int qa = 0, qb = 0, ka = 0, kb = 0, first = id + 1;
    if (lo + lane < hi) {
        seq_rows(a.qs, lo + lane, a.q_rows, &qa, &qb);
        seq_rows(a.ks, lo + lane, a.k_rows, &ka, &kb);
        first = tile_start(a.qs, lo + lane, a.q_rows, rows);
    }
    const int at = __popcll(__ballot(first <= id)) - 1;
    if (at < 0) return false;
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, at); };   /* the same in every lane: scalar registers */
    *seq = WinSeq{of(qa), of(qb), of(ka), of(kb), id - of(first)};
    return seq->tile >= 0 && seq->tile < (seq->qb - seq->qa + rows - 1) / rows;
}

/* One sequence's tile of queries: its rows, places and the key blocks that any of its queries sees. */
struct WinTile {
    int i0, Lq, Lk, off, p0, p1, qa, ka;
    KeyBlocks blocks;
    __device__ __forceinline__ WinTile(const WinArgs &a, const WinSeq &s, int qb, int kb)
    {
        qa = s.qa;
        ka = s.ka;
        Lq = s.qb - qa;
        Lk = s.kb - ka;
        i0 = s.tile * qb;
        off = Lk - Lq;
        p0 = i0 + off;
        p1 = imin(i0 + qb, Lq) - 1 + off;
        blocks = key_blocks(p0 - a.window + 1, imin(Lk, p1 + a.ahead + 1), a.sinks, kb);
    }
    /* whether every query of places pa .. pb sees all n keys from k0 on */
    __device__ __forceinline__ bool all_seen(const WinArgs &a, int k0, int n, int pa, int pb) const
    {
        const int k1 = k0 + n - 1;
        return k1 < Lk && k1 - pa <= a.ahead && (pb - k0 < a.window || k1 < a.sinks);
    }
};

/* A value that is not finite, in a block where some query must not see it, would reach that query as 0 · inf, so such
 * values enter the products as zeros (`odd` notes that there were some), and what they do to the queries that see them
 * is added to the stored outputs here: any positive weight of an infinity or a NaN is that. Rare, so simple: one thread
 * per output, over every key of the blocks concerned. */
template <int DT, int DH>
__device__ __forceinline__ void add_odd_values(const WinArgs &a, const WinTile &w, int kvh, int head0, int n_heads, int qb,
                                               int kb)
{
    typedef typename Elem<DT>::type E;
    const E *vh = static_cast<const E *>(a.v) + (size_t)w.ka * a.ldv + (size_t)kvh * DH;
    const int n = imin(qb, w.Lq - w.i0);
    for (int e = threadIdx.x; e < n * DH * n_heads; e += blockDim.x) {
        const int head = head0 + e % (n_heads * DH) / DH, d = e % DH, i = w.i0 + e / (n_heads * DH), p = i + w.off;
        float more = 0.0f;
        for (int b = 0; b < w.blocks.total; b++) {
            const int k0 = w.blocks.at(b) * kb;
            if (w.all_seen(a, k0, kb, w.p0, w.p1)) continue;
            for (int key = k0; key < imin(k0 + kb, w.Lk); key++) {
                const float x = Elem<DT>::get(vh[(size_t)key * a.ldv + d]);
                if (!(__builtin_fabsf(x) < INFINITY) && key_visible(key, p, a.window, a.ahead, a.sinks)) more += x;
            }
        }
        if (!(__builtin_fabsf(more) < INFINITY)) {
            E *o = static_cast<E *>(a.o) + (size_t)(w.qa + i) * a.ldo + (size_t)head * DH + d;
            *o = Elem<DT>::put(Elem<DT>::get(*o) + more);
        }
    }
}

/* The window kernels' workgroups: a tile of queries of `hpw` query heads that read one key head, the first of them
 * returned. Those of different key heads are next to each other, so that with 8 key heads (or a multiple) each XCD, which
 * takes every eighth workgroup, reads the keys of its own. Later tiles, which see more keys where the window is long,
 * come first; the second workgroups of the CUs, where there are no third ones, take the tiles from the other end, so that
 * each CU has one with many keys and one with few (2000 causal queries of 32 heads of 128: fp32 292 us, 364 in one order;
 * bf16 49.8, 52.6). */
__device__ __forceinline__ bool win_tile_of(const WinArgs &a, int hpw, int qb, int *head, int *kvh, WinSeq *seq)
{
    const int sets = a.heads / hpw, id = blockIdx.x % sets;
    *kvh = id % a.kv;
    *head = *kvh * (a.heads / a.kv) + id / a.kv * hpw;
    const int b = blockIdx.x;
    return find_tile(a, qb, b < a.turn ? a.tiles - 1 - b / sets : (b - a.turn) / sets, seq);
}

/* Where a 16-byte piece cc of row r lies in V's part of the LDS, 16-bit rows of CH pieces: its 64-byte group is moved
 * so that a transposing read (8 rows, one group) falls into different banks. */
template <int CH> __device__ __forceinline__ constexpr int v_place(int r, int cc)
{
    return cc ^ (CH == 16 ? 4 * (r & 3) : 4 * ((r >> 1) & 1));
}

/* The loads of a block of KB rows of one matrix by the NW waves of a workgroup, straight into LDS: per lane and load
 * an offset from the block's first row, the 16-byte piece chosen so that it lands where `place` wants it. Rows past the
 * last are not read: what lies in their place is kept from the result by the masks. */
template <class E, int DH, int KB, int NW> struct BlockLoads {
    static constexpr int EPC = 16 / sizeof(E), CH = DH / EPC, LD = KB * CH / (64 * NW), RPL = 64 / CH;
    uint32_t off[LD];
    int ld;
    const E *base;
    template <class P> __device__ __forceinline__ BlockLoads(const E *b, int pitch, int lane, int wave, P place)
        : ld(pitch), base(b)
    {
#pragma unroll
        for (int x = 0; x < LD; x++) {
            const int r = RPL * (LD * wave + x) + lane / CH;
            off[x] = (uint32_t)(r * ld + EPC * place(r, lane % CH)) * sizeof(E);
        }
    }
    /* the block of rows k0 .. of `rows` */
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t from(int k0, int rows) const
    {
        const int last = imin(rows - k0, KB) - 1;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<E *>(base + (size_t)k0 * ld), 0,
                                                 (int)((uint32_t)(last * ld + DH) * sizeof(E)), 0x00020000);
    }
    __device__ __forceinline__ void fetch(int x, __amdgpu_buffer_rsrc_t r, E *to, int wave) const
    {
        dma_16(r, off[x], to + 64 * EPC * (LD * wave + x));
    }
    __device__ __forceinline__ void fetch(int k0, int rows, E *to, int wave) const
    {
        const __amdgpu_buffer_rsrc_t r = from(k0, rows);
#pragma unroll
        for (int x = 0; x < LD; x++) fetch(x, r, to, wave);
    }
    /* what this lane's loads brought, once they have come: infinities and NaN become zeros; whether there were some */
    template <int DT> static __device__ __forceinline__ bool clean(E *to, int lane, int wave)
    {
        u4 *at = reinterpret_cast<u4 *>(to) + 64 * LD * wave + lane;
        float z = 0.0f;
#pragma unroll
        for (int x = 0; x < LD; x++) z = odd_sum<DT>(at[64 * x], z);
        if (z == z) return false;
#pragma unroll
        for (int x = 0; x < LD; x++) at[64 * x] = only_finite<DT>(at[64 * x]);
        return true;
    }
};

/* attention_win raises its reference only where the exponentials of a block have a sum above kWinSlack in some lane: then
 * to the largest score so far, and they are taken again. It is not raised otherwise, so that most blocks need no maximum
 * and leave O as it is: a weight stays below the slack, which every type holds, and relative to their sum nothing changes.
 * fp16 ends at 65504, so that lift and slack share what is there: a lift of 2^6 loses what is under 2^-31 of the largest
 * and leaves the slack what it is in bf16. Higher lifts raise the reference more often (6000 rows of 32 heads of 128, scores
 * of deviation 2: 2^5 110 us, 2^8 112, 2^10 115; rising scores 108, 112, 118). */
template <int DT> constexpr float kWinLift = DT == T_F16 ? 6.0f : 0.0f;
template <int DT> constexpr float kWinSlack = DT == T_F16 ? 65504.0f : 1024.0f;

/* 32 queries of one head in a wave: lane % 32 is the query, 16-bit rows. */
template <int DH> struct WinSub {
    f16v o[DH / 32], s[2];   /* O^T so far; the scores of a block */
    u4 q[DH / 16], pw[4];    /* the query, elements 8(2x + lane / 32) .. of every 16; a block's weights, 16 keys each */
    float m, l;              /* the reference, in powers of two, and this lane's sum of weights */
    int p, full0, full1;     /* this lane's query's place; blocks from full0 to full1 on are seen whole by all queries */
};

/* O for 128 rows, 32 for each of four waves; 16-bit rows. The rows are 128 / hpw queries of each of hpw (1, 2 or 4) query
 * heads that read the same key head: the fewer queries, the fewer keys that some of them must not see. The keys come in
 * blocks of 64 through LDS, K and V in two buffers each; blocks without a visible key are not touched.
 *
 * Per block and 32 queries S^T = K·Q^T by 32 × 32 products (keys in rows, queries in columns), so that a lane holds 32
 * keys of one query: the sum of its weights needs one exchange with the lane 32 away, at the end, and the weights are
 * already laid out as the operand of O^T += V^T·P^T, whatever order that product takes the keys in, as V's operand reads
 * the same order out of LDS. The exponentials are rounded to the rows' type for that product and summed unrounded in 32
 * bits: against 64 bits the output is off by 0.0021 (bf16, relative 2-norm; fp16 2.6e-4), of which rounding it makes 0.0016
 * (2.0e-4). A second product with what the rounding left brings it down to that, at 148 us instead of 116 (6000 rows as
 * below) and 166 instead of 110 (ragged prompts, heads of 64), so one product it is.
 *
 * A block's exponentials take the vector unit about as long as its products take the matrix unit: two workgroups a CU (heads
 * of 64, whose registers are fewer: three) put two waves on each SIMD, of which one can multiply while the other takes exponentials. For that a wave's products are
 * one stretch without waits: the scores of block b together with the output product of block b − 1, in QR equal stages,
 * each stage's operands read from LDS two stages ahead, and one of the loads of K of block b + 1 and V of block b issued
 * in each (all at once they would wait for each other: a CU takes 64 bytes a cycle). One barrier a block: there the loads
 * of the block before have come, and everyone is done with what the next ones overwrite.
 *
 * 6000 bf16 rows of 32 heads of 128 (8 key heads), window 1024: 113 us, 0.82 PFLOP/s of visible pairs (a large product
 * reaches 1.2). For 85 % of that the SIMDs have a wave; of this the matrix unit is busy 51 %, the vector unit 49 %, together
 * the whole: the two waves hardly overlap. The LDS is busy 26 %. Heads of 64 (ragged prompts): 81 %, of which 48, 73 and 36 %
 * (a third of that conflicts: their K rows of 128 bytes are placed as rows of 256). */
template <int DT, int DH>
__global__ __launch_bounds__(256, 2) void attention_win(WinArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int KB = 64, CH = DH / 8, QR = DH / 16, NT = DH / 32;
    typedef BlockLoads<E, DH, KB, 4> Loads;
    static_assert(2 * Loads::LD == QR, "one load a stage");
    __shared__ __align__(16) E lds[4][KB * DH];   /* K of even and odd blocks, V of even and odd blocks */

    int head0, kvh;
    WinSeq seq;
    if (!win_tile_of(a, a.hpw, 128 / a.hpw, &head0, &kvh, &seq)) return;
    const WinTile w(a, seq, 128 / a.hpw, KB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5,
              col = lane & 31;
    const int head = head0 + wave % a.hpw, sub = 32 * (wave / a.hpw);   /* this wave's head and its first query */

    /* K's row r has its piece cc at place cc ^ (r mod CH): the operand reads (32 rows, one piece) fall into different
     * banks */
    const Loads kl(static_cast<const E *>(a.k) + (size_t)w.ka * a.ldk + (size_t)kvh * DH, a.ldk, lane, wave,
                   [](int r, int cc) { return cc ^ (r & (CH - 1)); });
    const Loads vl(static_cast<const E *>(a.v) + (size_t)w.ka * a.ldv + (size_t)kvh * DH, a.ldv, lane, wave,
                   [](int r, int cc) { return v_place<CH>(r, cc); });
    const int n_blocks = w.blocks.total;
    if (n_blocks > 0) kl.fetch(w.blocks.at(0) * KB, w.Lk, lds[0], wave);

    WinSub<DH> u;
    const int iq = w.i0 + sub + col;
    {
        const E *row = static_cast<const E *>(a.q) + (size_t)(w.qa + imin(iq, w.Lq - 1)) * a.ldq + (size_t)head * DH;
#pragma unroll
        for (int x = 0; x < QR; x++) u.q[x] = *reinterpret_cast<const u4 *>(row + 8 * (2 * x + h));
    }
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) u.o[d][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) u.pw[k] = u4{0, 0, 0, 0};
    u.m = -INFINITY;
    u.l = 0.0f;
    u.p = imin(iq, w.Lq - 1) + w.off;
    u.full0 = imin(w.p0 + sub + 31, w.Lq - 1 + w.off) - a.window + 1;
    u.full1 = last_seen_by_all(w.p0 + sub, w.Lk, a.ahead) - (KB - 1);
    bool odd = false;

    /* LDS byte addresses. K's operand x of 32 keys: row col, piece 2x + h, so that the pieces of a row are an exclusive or
     * apart; V's operand for dimensions 32d .. and 16 keys, of each eight of which this half of the lanes has four: the
     * 64-byte groups of a row are. */
    constexpr uint32_t BUF = KB * DH * 2;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)lds;
    const int vr = 4 * h + ((lane & 15) >> 2);
    const uint32_t k_at = lds0 + col * DH * 2 + 16 * (h ^ (col & (CH - 1)));
    const uint32_t v_at = lds0 + 2 * BUF + vr * DH * 2 + 16 * v_place<CH>(vr, 0) + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
    auto read_k = [&](uint32_t at, int n, int x) __attribute__((always_inline)) {
        typedef __attribute__((address_space(3))) const u4 *lds16;
        return *(lds16)(uintptr_t)((at ^ (32 * x)) + 32 * n * DH * 2);
    };
    auto read_v = [&](uint32_t at, int k2, int d) __attribute__((always_inline)) {
        const uint32_t x = (at ^ (64 * d)) + 16 * k2 * DH * 2;
        const u2 va = lds_tr(x), vb = lds_tr(x + 8 * DH * 2);
        return u4{va[0], va[1], vb[0], vb[1]};
    };
    /* this wave's loads have come; of V of block b, where some query must not see a key, what is not finite is put aside */
    auto come = [&](int b) __attribute__((always_inline)) {
        wait_vm<0>();
        if (b >= 0 && !w.all_seen(a, w.blocks.at(b) * KB, KB, w.p0, w.p1))
            odd |= Loads::template clean<DT>(lds[2 + (b & 1)], lane, wave);
        lds_barrier();
    };
    /* What a query must not see of the block at k0, where its 32 queries do not all see all of it. Key e of the block is
     * bit e of 64; this lane has keys 8j + 4h .. + 3 of every eight. */
    auto mask = [&](int k0) __attribute__((always_inline)) {
        if (k0 <= u.full1 && (k0 >= u.full0 || k0 < a.sinks - (KB - 1))) return;
        const KeySpan span = key_span(k0, u.p, w.Lk, a.window, a.ahead, a.sinks);
        auto below = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
        const unsigned long long bits = (below(span.last + 1) & (~below(span.first) | below(span.sink))) >> (4 * h);
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t seen = (uint32_t)__builtin_amdgcn_sbfe((int)(bits >> (32 * n)), 8 * (i / 4) + i % 4, 1);
                u.s[n][i] = __uint_as_float((__float_as_uint(u.s[n][i]) & seen) | (0xff800000u & ~seen));
            }
    };
    /* weights 8·k .. 8·k + 7 of u's scores from the reference mu on, added to sum */
    auto weights = [&](int k, float mu, float &sum) __attribute__((always_inline)) {
        float pv[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            pv[i] = exp2_fast(__builtin_fmaf(u.s[k / 2][8 * (k & 1) + i], a.c, -mu));
        }
        sum += ((pv[0] + pv[1]) + (pv[2] + pv[3])) + ((pv[4] + pv[5]) + (pv[6] + pv[7]));
        u.pw[k] = pack<DT>(pv);
    };
    /* the weights' sum goes into l; before, where it is too large or there is no reference yet, they are taken again from
     * the largest score */
    auto settle = [&](float sum) __attribute__((always_inline)) {
        if (__any(sum > kWinSlack<DT> || u.m == -INFINITY)) {
            float top = u.s[0][0];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 16; i++) top = fmaxf(top, u.s[n][i]);
            const float mn = fmaxf(u.m, lifted(max_halves(top), a.c, kWinLift<DT>)), mu = mn == -INFINITY ? 0.0f : mn;
            const float fade = exp2_fast(u.m - mu);
            u.m = mn;
            u.l *= fade;
#pragma unroll
            for (int d = 0; d < NT; d++) u.o[d] *= fade;
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) weights(k, mu, sum);
        }
        u.l += sum;
    };
    if (n_blocks > 0) {
        /* the first block has no weights before it: zeros, with zeros for V */
        for (int x = threadIdx.x; x < KB * CH; x += 256) reinterpret_cast<u4 *>(lds[3])[x] = u4{0, 0, 0, 0};
        for (int b = 0; b < n_blocks; b++) {
            const int k0 = w.blocks.at(b) * KB;
            /* past the last block that one's K again, which nothing reads */
            const __amdgpu_buffer_rsrc_t next_k = kl.from(w.blocks.at(imin(b + 1, n_blocks - 1)) * KB, w.Lk),
                                         this_v = vl.from(k0, w.Lk);
            const uint32_t ka = k_at + (b & 1) * BUF, va = v_at + ((b & 1) ^ 1) * BUF;
            u4 kf[3][2], vf[3][2];
            auto read = [&](int t) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    kf[t % 3][j] = read_k(ka, j, t);
                    vf[t % 3][j] = read_v(va, (2 * t + j) / NT, (2 * t + j) % NT);
                }
            };
#pragma unroll
            for (int i = 0; i < 16; i++) u.s[0][i] = u.s[1][i] = 0.0f;
            come(b - 1);
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
                    u.s[j] = mfma32<DT>(kf[t % 3][j], u.q[t], u.s[j]);
                    u.o[z % NT] = mfma32<DT>(vf[t % 3][j], u.pw[z / NT], u.o[z % NT]);
                }
                if (t < Loads::LD) kl.fetch(t, next_k, lds[(b & 1) ^ 1], wave);
                else vl.fetch(t - Loads::LD, this_v, lds[2 + (b & 1)], wave);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            mask(k0);
            const float mu = u.m == -INFINITY ? 0.0f : u.m;
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) weights(k, mu, sum);
            settle(sum);
        }
        come(n_blocks - 1);
        const uint32_t va = v_at + ((n_blocks - 1) & 1) * BUF;
#pragma unroll
        for (int k2 = 0; k2 < 4; k2++)
#pragma unroll
            for (int d = 0; d < NT; d++) u.o[d] = mfma32<DT>(read_v(va, k2, d), u.pw[k2], u.o[d]);
    }
    odd = __syncthreads_or(odd);   /* before the stores, as a barrier behind them would wait for them */
    const float l = sum_halves(u.l), inv = l == 0.0f ? 0.0f : 1.0f / l;
    E *row = static_cast<E *>(a.o) + (size_t)(w.qa + imin(iq, w.Lq - 1)) * a.ldo + (size_t)head * DH + 8 * h;
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            /* of 16 elements this lane has 4 of the first eight and 4 of the second; the lane 32 away the others */
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = u.o[d][4 * k + j] * inv;
            const u4 x = pack<DT>(v);
            const auto e0 = __builtin_amdgcn_permlane32_swap(x[0], x[2], false, false);
            const auto e1 = __builtin_amdgcn_permlane32_swap(x[1], x[3], false, false);
            if (iq < w.Lq) *reinterpret_cast<u4 *>(row + 32 * d + 8 * k) = u4{e0[0], e1[0], e0[1], e1[1]};
        }
    if (odd) {
        __syncthreads();   /* the stores above are there */
        add_odd_values<DT, DH>(a, w, kvh, head0, a.hpw, 128 / a.hpw, KB);
    }
}

/* attention_win for fp32 rows, multiplied in fp32 throughout: its products take the matrix unit several times as long as
 * everything else takes, so nothing is gained by running them together with the exponentials. Blocks of 32 keys, two
 * buffers in turn: while one is multiplied the next is on its way. 2000 causal queries of 32 heads of 128: 292 us, 112
 * TFLOP/s (a large fp32 product reaches 153). */
template <int DH>
__global__ __launch_bounds__(256, 2) void attention_win_f32(WinArgs a)
{
    constexpr int DT = T_F32, KB = 32, CH = DH / 4, QR = DH / 8;
    __shared__ __align__(16) float lds[2][2 * KB * DH];

    int head, kvh;
    WinSeq seq;
    if (!win_tile_of(a, 1, 128, &head, &kvh, &seq)) return;
    const WinTile w(a, seq, 128, KB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5,
              col = lane & 31;
    const int iq = w.i0 + 32 * wave + col, p = imin(iq, w.Lq - 1) + w.off;
    const int pw0 = w.p0 + 32 * wave, pw1 = imin(pw0 + 31, w.Lq - 1 + w.off);   /* this wave's places */

    u4 q[QR];   /* this lane's query: elements 4(2x + h) .. of every 8 */
    {
        const float *row = static_cast<const float *>(a.q) + (size_t)(w.qa + imin(iq, w.Lq - 1)) * a.ldq +
                           (size_t)head * DH;
#pragma unroll
        for (int x = 0; x < QR; x++) q[x] = *reinterpret_cast<const u4 *>(row + 4 * (2 * x + h));
    }
    f16v o[DH / 32];
#pragma unroll
    for (int d = 0; d < DH / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;   /* the reference, in powers of two, and this lane's sum of weights */
    bool odd = false;

    const BlockLoads<float, DH, KB, 4> kl(static_cast<const float *>(a.k) + (size_t)w.ka * a.ldk + (size_t)kvh * DH, a.ldk,
                                       lane, wave, [](int r, int cc) { return cc ^ (r & (CH - 1)); });
    const BlockLoads<float, DH, KB, 4> vl(static_cast<const float *>(a.v) + (size_t)w.ka * a.ldv + (size_t)kvh * DH, a.ldv,
                                       lane, wave, [](int, int cc) { return cc; });
    auto fetch = [&](int k0, float *to) __attribute__((always_inline)) {
        kl.fetch(k0, w.Lk, to, wave);
        vl.fetch(k0, w.Lk, to + KB * DH, wave);
    };

    if (w.blocks.total > 0) fetch(w.blocks.at(0) * KB, lds[0]);
    for (int b = 0; b < w.blocks.total; b++) {
        const int k0 = w.blocks.at(b) * KB;
        float *K = lds[b & 1], *V = K + KB * DH;
        /* this wave's loads have come, and of V, where some query must not see a key, what is not finite is put aside; then
         * everyone's, and every wave is done with the other buffer */
        wait_vm<0>();
        if (!w.all_seen(a, k0, KB, w.p0, w.p1)) odd |= BlockLoads<float, DH, KB, 4>::template clean<DT>(V, lane, wave);
        __syncthreads();
        if (b + 1 < w.blocks.total) fetch(w.blocks.at(b + 1) * KB, lds[(b + 1) & 1]);
        /* no query of this wave sees any of the block, or it has no query */
        if (pw1 < pw0 || k0 - pw1 > a.ahead || (pw0 - (k0 + KB - 1) >= a.window && k0 >= a.sinks)) continue;
        f16v s;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < QR; x++) {
            const u4 k = *reinterpret_cast<const u4 *>(K + col * DH + 4 * ((2 * x + h) ^ (col & (CH - 1))));
#pragma unroll
            for (int e = 0; e < 4; e++)
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q[x][e]), s, 0, 0, 0);
        }
        if (!w.all_seen(a, k0, KB, pw0, pw1)) {
            const KeySpan span = key_span(k0 + 4 * h, p, w.Lk, a.window, a.ahead, a.sinks);   /* from this lane's first key */
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int e = 8 * (i / 4) + i % 4;
                if ((e > span.last) | ((e < span.first) & (e >= span.sink))) s[i] = -INFINITY;
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top, s[i]);
        top = max_halves(top) * a.c;
        if (__any(top > m + 8.0f)) {   /* the reference is raised where a maximum is 2^8 above it, and in the first block */
            const float mn = fmaxf(m, top), fade = exp2_fast(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= fade;
#pragma unroll
            for (int d = 0; d < DH / 32; d++) o[d] *= fade;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            s[i] = exp2_fast(__builtin_fmaf(s[i], a.c, -mu));
            sum += s[i];
        }
        l += sum;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float *row = V + (8 * (i / 4) + 4 * h + i % 4) * DH + col;
#pragma unroll
            for (int d = 0; d < DH / 32; d++)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(row[32 * d], s[i], o[d], 0, 0, 0);
        }
    }
    odd = __syncthreads_or(odd);   /* before the stores, as a barrier behind them would wait for them */
    l = sum_halves(l);
    if (iq < w.Lq) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float *row = static_cast<float *>(a.o) + (size_t)(w.qa + iq) * a.ldo + (size_t)head * DH + 4 * h;
#pragma unroll
        for (int d = 0; d < DH / 32; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) row[32 * d + 8 * (i / 4) + i % 4] = o[d][i] * inv;
    }
    if (odd) {
        __syncthreads();   /* the stores above are there */
        add_odd_values<DT, DH>(a, w, kvh, head, 1, 128, KB);
    }
}

/* ── attention of few queries ──────────────────────────────────────────────────────────────────────────────── */

struct PageArgs {
    int n_seqs, heads, kv, q_groups, splits, page_shift, pages, table_ld, ldq, ldo, window, sinks;
    float c;
    const void *q, *kc, *vc;
    const int *table, *len;
    void *o;
    float *part;   /* [sequence][head][split][DH + 2] where splits > 1: sums, reference, sum of weights */
};

/* attention_win for calls with too few tiles of 128 queries to fill the device: 16 queries of one head a workgroup, whose
 * NW waves take the key blocks in turn, nothing shared between them until their sums are joined. 438 fp32 queries of 8 heads
 * of 128, 128 places back and 32 on: 10.1 us, of which the fp32 products of a CU's 12 blocks take 3. */
template <int DT, int DH, int NW>
__global__ __launch_bounds__(64 * NW, DH == 64 ? 4 : 3) void attention_win_few(WinArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int NB = FewPlace<DT>::NB, KB = FewPlace<DT>::KB, EPC = kPer16<DT>;
    __shared__ __align__(16) unsigned char lds[few_lds_bytes<DT, DH, NW>()];
    int head, kvh;
    WinSeq seq;
    if (!win_tile_of(a, 1, 16, &head, &kvh, &seq)) return;
    const WinTile w(a, seq, 16, KB);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    const int i = imin(w.i0 + (lane & 15), w.Lq - 1), p = i + w.off;
    u4 q[DH / (4 * EPC)];
    {
        const E *row = static_cast<const E *>(a.q) + (size_t)(w.qa + i) * a.ldq + (size_t)head * DH;
#pragma unroll
        for (int s = 0; s < DH / (4 * EPC); s++) q[s] = *reinterpret_cast<const u4 *>(row + EPC * (4 * s + g));
    }
    const E *kh = static_cast<const E *>(a.k) + (size_t)w.ka * a.ldk + (size_t)kvh * DH;
    const E *vh = static_cast<const E *>(a.v) + (size_t)w.ka * a.ldv + (size_t)kvh * DH;
    FewState<DH> st;
    bool odd = false;
    few_blocks<DT, DH, true>(
        st, q, a.c, wave, w.blocks.total, NW, a.ldk, a.ldv, [](int) { return 0; },
        [&](int b, int) __attribute__((always_inline)) {
            FewPlace<DT> p;
            p.k0 = w.blocks.at(b) * KB;
#pragma unroll
            for (int t = 0; t < NB; t++) {
                const int row = imin(p.k0 + 16 * t, w.Lk - 1);
                p.have[t] = imin(16, w.Lk - row);
                p.k[t] = kh + (size_t)row * a.ldk;
                p.v[t] = vh + (size_t)row * a.ldv;
            }
            p.whole = w.all_seen(a, p.k0, KB, w.p0, w.p1);
            return p;
        },
        [&](const FewPlace<DT> &b, int k) __attribute__((always_inline)) {
            return b.k0 + k < w.Lk && key_visible(b.k0 + k, p, a.window, a.ahead, a.sinks);
        },
        [&](const FewPlace<DT> &b, int k) __attribute__((always_inline)) { return b.k0 + k < w.Lk; }, odd,
        lds + wave * few_own_bytes<DT, DH>());
    odd = __syncthreads_or(odd);   /* before the stores, as a barrier behind them would wait for them */
    float *J = reinterpret_cast<float *>(lds);
    few_store<DT, DH>(st, J);
    for (int e = threadIdx.x; e < imin(16, w.Lq - w.i0) * DH; e += 64 * NW) {
        float top, num, den;
        few_join<DH, NW>(J, e / DH, e % DH, &top, &num, &den);
        static_cast<E *>(a.o)[(size_t)(w.qa + w.i0 + e / DH) * a.ldo + (size_t)head * DH + e % DH] =
            Elem<DT>::put(den == 0.0f ? 0.0f : num / den);
    }
    if (odd) {
        __syncthreads();   /* the stores above are there */
        add_odd_values<DT, DH>(a, w, kvh, head, 1, 16, KB);
    }
}

/* One workgroup: one sequence, one key head, up to 16 of the query heads that read it, one part of its key blocks, which
 * its NW waves take in turn. Keys that are not seen (past the end, outside the window, in a page that is not there) have
 * no weight and their V is zeros, whatever lies in the page: all queries here stand at one place. Bound by memory: 32 bf16
 * sequences of up to 8192 tokens over 8 key heads of 128, 713 MB in 134 us (5.3 TB/s; a copy, half of it writes, 4.8). A
 * single sequence of 375 fp32 tokens takes 6.5 us, a chain of waits: length, page, keys. */
template <int DT, int DH, int NW>
__global__ __launch_bounds__(64 * NW, DH == 64 ? 4 : 3) void attention_page(PageArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int NB = FewPlace<DT>::NB, KB = FewPlace<DT>::KB, EPC = kPer16<DT>;
    __shared__ __align__(16) unsigned char lds[few_lds_bytes<DT, DH, NW>()];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int split = blockIdx.x % a.splits, kvh = (blockIdx.x / a.splits) % a.kv;
    const int qg = (blockIdx.x / a.splits / a.kv) % a.q_groups, seq = blockIdx.x / a.splits / a.kv / a.q_groups;
    const int G = a.heads / a.kv, nq = imin(16, G - 16 * qg), head0 = kvh * G + 16 * qg;

    const int *row = a.table + (size_t)seq * a.table_ld;
    const int len = a.pages ? kept_length(a.len[seq], a.table_ld, 1 << a.page_shift) : 0;
    const int w0 = imax(len - a.window, 0);
    const KeyBlocks blocks = key_blocks(w0, len, a.sinks, KB);
    int b0, b1;
    split_range(blocks.total, a.splits, split, &b0, &b1);

    u4 q[DH / (4 * EPC)];
    {
        const E *p = static_cast<const E *>(a.q) + (size_t)seq * a.ldq + (size_t)(head0 + imin(c, nq - 1)) * DH;
#pragma unroll
        for (int s = 0; s < DH / (4 * EPC); s++) q[s] = *reinterpret_cast<const u4 *>(p + EPC * (4 * s + g));
    }
    const size_t page_elems = (size_t)DH << a.page_shift;   /* of one head */
    const E *kc = static_cast<const E *>(a.kc) + kvh * page_elems, *vc = static_cast<const E *>(a.vc) + kvh * page_elems;
    const int in_page = (1 << a.page_shift) - 1;
    FewState<DH> st;
    bool odd = false;
    struct Entries {
        int e[NB];
    };
    auto seen = [&](const FewPlace<DT> &b, int k) __attribute__((always_inline)) {
        const int key = b.k0 + k;
        return b.there[NB == 2 ? k >> 4 : 0] && key < len && (key >= w0 || key < a.sinks);
    };
    few_blocks<DT, DH, false>(
        st, q, a.c, b0 + wave, b1, NW, DH, DH,
        [&](int b) __attribute__((always_inline)) {
            Entries n;   /* pages hold a multiple of 16 tokens */
#pragma unroll
            for (int t = 0; t < NB; t++) {
                const int key = blocks.at(b) * KB + 16 * t;
                n.e[t] = key < len ? page_entry(row, a.table_ld, key, a.page_shift) : -1;
            }
            return n;
        },
        [&](int b, Entries n) __attribute__((always_inline)) {
            FewPlace<DT> p;
            p.k0 = blocks.at(b) * KB;
            p.whole = true;
#pragma unroll
            for (int t = 0; t < NB; t++) {
                const int key = p.k0 + 16 * t, page = page_in(n.e[t], a.pages);
                const size_t at = (size_t)imax(page, 0) * a.kv * page_elems + (size_t)(key & in_page) * DH;
                p.have[t] = 16;
                p.there[t] = page >= 0;
                p.k[t] = kc + at;
                p.v[t] = vc + at;
                p.whole &= page >= 0 && key + 15 < len && (key >= w0 || key + 15 < a.sinks);
            }
            return p;
        },
        seen, seen, odd, lds + wave * few_own_bytes<DT, DH>());
    float *J = reinterpret_cast<float *>(lds);
    few_store<DT, DH>(st, J);
    for (int e = threadIdx.x; e < nq * DH; e += 64 * NW) {
        const int r = e / DH, d = e % DH;
        float top, num, den;
        few_join<DH, NW>(J, r, d, &top, &num, &den);
        if (a.splits == 1) {
            static_cast<E *>(a.o)[(size_t)seq * a.ldo + (size_t)(head0 + r) * DH + d] =
                Elem<DT>::put(den == 0.0f ? 0.0f : num / den);
        } else {
            float *to = a.part + (((size_t)seq * a.heads + head0 + r) * a.splits + split) * (DH + 2);
            to[d] = num;
            if (d == 0) {
                to[DH] = top;
                to[DH + 1] = den;
            }
        }
    }
}

/* The parts of one sequence's head added up by one workgroup: each wave takes every NW-th part, DH / 64 outputs a lane,
 * all its loads independent of each other; the waves' sums are added in LDS. 3 to 5 us, most of it the launch. */
constexpr int kJoinWaves = 8;
template <int DT, int DH>
__global__ __launch_bounds__(64 * kJoinWaves) void attention_join(PageArgs a)
{
    typedef typename Elem<DT>::type E;
    constexpr int PER = DH / 64;
    __shared__ float J[kJoinWaves][DH + 2];
    const int seq = blockIdx.x / a.heads, head = blockIdx.x % a.heads, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float *p = a.part + ((size_t)seq * a.heads + head) * a.splits * (DH + 2);
    float top = -INFINITY;   /* of all parts: 64 at a time */
    for (int s = lane; s < a.splits; s += 64) top = fmaxf(top, p[(size_t)s * (DH + 2) + DH]);
#pragma unroll
    for (int o = 1; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    const float mu = top == -INFINITY ? 0.0f : top;
    float num[PER], den = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) num[i] = 0.0f;
#pragma unroll 8
    for (int s = wave; s < a.splits; s += kJoinWaves) {
        const float *j = p + (size_t)s * (DH + 2);
        const float f = exp2_fast(j[DH] - mu);
#pragma unroll
        for (int i = 0; i < PER; i++) num[i] = __builtin_fmaf(f, j[PER * lane + i], num[i]);
        den = __builtin_fmaf(f, j[DH + 1], den);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) J[wave][PER * lane + i] = num[i];
    if (lane == 0) J[wave][DH] = den;
    __syncthreads();
    if (threadIdx.x < DH) {
        float n = 0.0f, e = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWaves; w++) {
            n += J[w][threadIdx.x];
            e += J[w][DH];
        }
        static_cast<E *>(a.o)[(size_t)seq * a.ldo + (size_t)head * DH + threadIdx.x] =
            Elem<DT>::put(e == 0.0f ? 0.0f : n / e);
    }
}

}  // namespace p2k
