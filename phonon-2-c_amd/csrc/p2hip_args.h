/*  p2hip_args.h – what the entries of a decoder's step share on the host: element types as constants, rows in memory, and
 *  the checks of heads, rows and caches.
 */
#pragma once

#include "p2hip_host.h"

#include <cmath>
#include <type_traits>

#include "p2hip_elem.h"

namespace p2host {

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

/* whether arrays of words are aligned: the scalar cache reads the aligned word that an address lies in */
template <class... P> bool words(const P *...p) { return (aligned(p, 4) && ...); }

/* M rows of `w` bytes at pitch `ld` bytes, as a range */
struct Rows {
    const char *p;
    size_t ld, w;
    int M;
    const char *end() const { return p + (M ? (size_t)(M - 1) * ld + w : 0); }
};

/* whether two sets of rows share a byte: apart as ranges, or of one pitch with their columns apart */
inline bool overlap(const Rows &a, const Rows &b)
{
    if (a.M <= 0 || b.M <= 0 || a.end() <= b.p || b.end() <= a.p) return false;
    if (a.ld != b.ld) return true;
    const size_t d = a.p <= b.p ? (size_t)(b.p - a.p) % a.ld : (a.ld - (size_t)(a.p - b.p) % a.ld) % a.ld;
    return !(d >= a.w && d + b.w <= a.ld);
}

inline int check_heads(const char *name, int dtype, int heads, int kv_heads, int head_dim)
{
    if (!is_type(dtype)) return fail(P2H_E_ARG, "%s: element type %d", name, dtype);
    if (head_dim != 64 && head_dim != 128) return fail(P2H_E_ARG, "%s: head_dim = %d (64 or 128)", name, head_dim);
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads != 0 || heads > 65536)
        return fail(P2H_E_ARG, "%s: %d heads over %d key heads", name, heads, kv_heads);
    return P2H_OK;
}

inline int check_rows(const char *name, const char *what, int dtype, const void *p, int ld, int width)
{
    if (!p || !aligned(p, 16)) return fail(P2H_E_ARG, "%s: %s is NULL or not 16-byte aligned", name, what);
    if (ld < width || (size_t)ld * elem_size(dtype) % 16 != 0)
        return fail(P2H_E_ARG, "%s: pitch %d of %s must be >= %d and a multiple of 16 bytes", name, ld, what, width);
    /* a block's rows are addressed by 32-bit offsets from its first */
    if (ld >= 1 << 23) return fail(P2H_E_ARG, "%s: pitch %d of %s must be below 2^23", name, ld, what);
    return P2H_OK;
}

inline int check_cache(const char *name, const P2hKvCache *c)
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

inline int check_cache(const char *name, const P2hKvCacheQ8 *c)
{
    if (!c) return fail(P2H_E_ARG, "%s: NULL cache", name);
    if (c->heads < 1 || c->heads > 65536 || (c->head_dim != 64 && c->head_dim != 128))
        return fail(P2H_E_ARG, "%s: cache with %d heads of %d", name, c->heads, c->head_dim);
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)) != 0 || c->pages < 0)
        return fail(P2H_E_ARG, "%s: %d pages of %d tokens (a power of two, 16 .. 1024)", name, c->pages, c->page);
    if (c->pages > 0 && (!c->K || !c->V || !aligned(c->K, 16) || !aligned(c->V, 16) || !c->KScale || !c->VScale ||
                         !aligned(c->KScale, 4) || !aligned(c->VScale, 4)))
        return fail(P2H_E_ARG, "%s: cache memory is NULL, or codes not 16-byte or scales not 4-byte aligned", name);
    return P2H_OK;
}

/* a cache's keys or values as one row, and whether rows share a byte with either */
inline Rows cache_row(const P2hKvCache *c, const void *p)
{
    const size_t bytes = (size_t)c->pages * c->heads * c->page * c->head_dim * elem_size(c->dtype);
    return Rows{(const char *)p, bytes, bytes, bytes ? 1 : 0};
}
inline bool overlap(const Rows &a, const P2hKvCache *c)
{
    return overlap(a, cache_row(c, c->K)) || overlap(a, cache_row(c, c->V));
}

inline int check_scale(const char *name, float scale, int window, int ahead, int sinks)
{
    if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(P2H_E_ARG, "%s: scale = %g must be positive", name, (double)scale);
    if (window < 1 || window > (1 << 30) || ahead < 0 || ahead > (1 << 30) || sinks < 0 || sinks > (1 << 30))
        return fail(P2H_E_ARG, "%s: window = %d (1 .. 2^30), ahead = %d, sinks = %d (0 .. 2^30)", name, window, ahead, sinks);
    return P2H_OK;
}

/* a cache of either kind: what it holds and where */
struct CacheView {
    int heads = 0, head_dim = 0, page = 0, pages = 0;
    void *K = nullptr, *V = nullptr;
    float *ks = nullptr, *vs = nullptr;
    size_t bytes = 0, scale_bytes = 0;   /* of keys or values; of the scales of either */
    CacheView(const P2hKvCache *rows, const P2hKvCacheQ8 *q8)
    {
        if (rows) set(*rows, elem_size(rows->dtype));
        if (q8) {
            set(*q8, 1);
            ks = q8->KScale;
            vs = q8->VScale;
            scale_bytes = (size_t)pages * heads * page * 4;
        }
    }
    /* its arrays, as rows, into f until that returns true */
    template <class F> bool any(F f) const
    {
        const Rows r[4] = {row(K, bytes), row(V, bytes), row(ks, scale_bytes), row(vs, scale_bytes)};
        for (int i = 0; i < 4; i++)
            if (f(r[i], i)) return true;
        return false;
    }

private:
    static Rows row(const void *p, size_t n) { return Rows{(const char *)p, n, n, n ? 1 : 0}; }
    template <class C> void set(const C &c, size_t es)
    {
        heads = c.heads; head_dim = c.head_dim; page = c.page; pages = c.pages;
        K = c.K; V = c.V;
        bytes = (size_t)pages * heads * page * head_dim * es;
    }
};
/* whether rows share a byte with a cache; whether a cache's own arrays do */
inline bool overlap(const Rows &a, const CacheView &c)
{
    return c.any([&](const Rows &r, int) { return overlap(a, r); });
}
inline bool overlap(const CacheView &c)
{
    return c.any([&](const Rows &a, int i) { return c.any([&](const Rows &b, int j) { return i < j && overlap(a, b); }); });
}

inline int log2_of(int page)
{
    int s = 0;
    while ((1 << s) < page) s++;
    return s;
}

}  // namespace p2host
