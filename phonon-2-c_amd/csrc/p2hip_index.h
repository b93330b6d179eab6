/*  p2hip_index.h – which keys an attention kernel reads and where they lie: the arithmetic on positions, windows and
 *  pages, apart from the kernels so that a host program can go over it (plain C++, no HIP types).
 */
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define P2_HD __host__ __device__ __forceinline__
#else
#define P2_HD inline
#endif

namespace p2k {

P2_HD int imin(int a, int b) { return a < b ? a : b; }
P2_HD int imax(int a, int b) { return a > b ? a : b; }

/* The aligned blocks of `bs` keys that hold a visible key, in order: blocks 0 .. sink − 1, then first, first + 1, …;
 * `total` of them. Visible are keys [lo, hi) and the keys below `sinks` among [0, hi). */
struct KeyBlocks {
    int sink, first, total;
    P2_HD int at(int b) const { return b < sink ? b : first + (b - sink); }
};

P2_HD KeyBlocks key_blocks(int lo, int hi, int sinks, int bs)
{
    KeyBlocks k{0, 0, 0};
    if (hi <= 0) return k;
    lo = imin(imax(lo, 0), hi);
    const int s1 = imin(sinks, lo);
    k.first = lo / bs;
    const int end = lo < hi ? (hi - 1) / bs + 1 : k.first;
    k.sink = s1 > 0 ? (s1 - 1) / bs + 1 : 0;
    if (end > k.first) k.sink = imin(k.sink, k.first);   /* block `first` comes once */
    k.total = k.sink + end - k.first;
    return k;
}

/* Whether key j is visible to the query at place p. */
P2_HD bool key_visible(int j, int p, int window, int ahead, int sinks)
{
    return j - p <= ahead && (p - j < window || j < sinks);
}

/* The same for the keys from k0 on: k0 + e, below Lk, is visible iff e <= last and (e >= first or e < sink). No key stands
 * before place 0, so that neither does the window's first: with blocks of a tile (k0 <= p + 127 + ahead) nothing here leaves
 * 32 bits. */
struct KeySpan {
    int last, first, sink;
};

P2_HD KeySpan key_span(int k0, int p, int Lk, int window, int ahead, int sinks)
{
    return KeySpan{imin(p + ahead, Lk - 1) - k0, imax(p - window + 1, 0) - k0, sinks - k0};
}

/* The last key that the queries at places p and on all see (apart from where their windows begin); p may lie behind the
 * last place. */
P2_HD int last_seen_by_all(int p, int Lk, int ahead) { return imin(Lk - 1, imin(p, Lk - 1) + ahead); }

/* Part s of `splits` of `total` blocks: [begin, end). */
P2_HD void split_range(int total, int splits, int s, int *begin, int *end)
{
    const int per = (total + splits - 1) / splits;
    *begin = imin(per * s, total);
    *end = imin(*begin + per, total);
}

/* The entry for key t in a sequence's table row of table_ld entries, −1 where it has none; reads only inside the row. */
P2_HD int page_entry(const int32_t *row, int table_ld, int t, int page_shift)
{
    const int i = t >> page_shift;
    return t < 0 || i >= table_ld ? -1 : row[i];
}

/* The page that an entry names, −1 where that lies outside the cache. */
P2_HD int page_in(int entry, int pages) { return (uint32_t)entry < (uint32_t)pages ? entry : -1; }

/* A sequence's length as the kernels take it. */
P2_HD int kept_length(int len, int table_ld, int page)
{
    const long long most = (long long)table_ld * page;
    return len < 0 ? 0 : len > most ? (int)most : len;
}

/* Sequence s's rows as the kernels take them: [a, b) inside [0, rows]. */
P2_HD void seq_rows(const int32_t *start, int s, int rows, int *a, int *b)
{
    if (!start) {
        *a = 0;
        *b = rows;
        return;
    }
    *a = imin(imax(start[s], 0), rows);
    *b = imin(imax(start[s + 1], *a), rows);
}

/* The number of sequence s's first tile of `rows` queries, its others following: floors of the rows before it, and one for
 * every sequence before it, which is never too few. Numbers from tile_start(n) on belong to no sequence. */
P2_HD int tile_start(const int32_t *start, int s, int rows_in_all, int rows)
{
    return imin(imax(start[s], 0), rows_in_all) / rows + s;
}

/* Whether the rows of a 4-bit linear are read 16 bytes at a time: each of them aligned (a single row has no pitch) and 16 of
 * them within 32-bit offsets. Read by the element they cost 2 to 5 times as much, the loads as many instructions and none
 * of them ahead (bf16 1 x 4095 x 4096 17.5 us against 5.1, 13 x 8191 x 16389 91 against 20). */
P2_HD bool rows_by_16(uintptr_t p, int pitch, int elem_size, int rows)
{
    return p % 16 == 0 && (rows == 1 || ((long long)pitch * elem_size % 16 == 0 && pitch < 1 << 25));
}

/* Whether a windowed call goes by 16 queries a workgroup, whose waves share the keys, or by tiles of 128 rows (16-bit rows:
 * of up to four query heads that read one key head). What counts is workgroups: those of 16 queries, by the mean length of
 * the sequences, which with their number is all that the host knows of them.
 *
 * 16-bit rows: 16 queries while they make fewer than 512 workgroups (8 heads of 128, all keys: 375 queries 9.4 us against
 * 13.0, 750 15.3 against 19.4, 1500 both 31.7; 64 heads, 16 queries behind 8000 keys 56 against 135), with heads of 64 and
 * long keys, whose blocks a tile takes one after the other, up to 1024 (2000 queries of 8 heads 21.6 us against 30.0, 8000
 * of 2 57 against 99; 4000 of 8 58 against 54). Sequences of one query are that many workgroups in either form, fewer where
 * tiles share key heads (64 sequences of 1000 keys, 32 heads over 8: 84 us, in tiles 44; 256 of 1000, heads of 64: 214, 117).
 *
 * fp32 rows, whose products take ten times as long: while 128-row tiles do not fill the device (1500 queries 73 us against
 * 203, 4000 362 against 525, 32 heads of 2000 396 against 292), but for short windows only below 128 of them (window 256,
 * 3000 queries: 69 against 65); and where sequences have at most 16 queries, since a tile multiplies 128 all the same (256
 * sequences of 8 queries and 100 keys, 32 heads: 0.53 of the tiles' time; of 17 queries 1.02). */
P2_HD bool few_queries(bool f32, int head_dim, int q_rows, int k_rows, int n_seqs, int heads, int window, int ahead, int cus)
{
    const int seqs = imin(n_seqs, q_rows), mean = (q_rows - 1) / seqs + 1;
    const long long wgs = (long long)heads * seqs * ((mean - 1) / 16 + 1);
    if (!f32) {
        const bool long_keys = imin(k_rows / n_seqs, window + imin(ahead, k_rows)) >= 1000;
        return wgs < 512 || (head_dim == 64 && wgs <= 1024 && long_keys);
    }
    const long long full = (long long)((q_rows - 1) / 128 + 1) * heads;
    return mean <= 16 || (full <= cus && (full < 128 || (long long)window + ahead >= 512));
}

}  // namespace p2k
