"""What a served batch's entries (include/p2hip.h) refuse: the arguments are checked before the device, so every refusal here
is the same with and without one. Addresses are never followed."""
import ctypes as C

import pytest

import p2gemm as P

E_ARG, E_WORKSPACE = -1, -4
A = 1 << 20   # an aligned address that nothing reads
FAR = 1 << 30


def refused(rc, part):
    assert rc == E_ARG, (rc, P.last_error())
    assert part in P.last_error(), P.last_error()


def q8(**kw):
    a = dict(heads=2, head_dim=64, page=16, pages=4, dK=8 * A, dV=9 * A, dKScale=10 * A, dVScale=11 * A)
    a.update(kw)
    return P.KvCacheQ8(**a)


CODES, SCALES = 4 * 2 * 16 * 64, 4 * 2 * 16 * 4   # bytes of such a cache's arrays

BAD_CACHES = [(dict(heads=0), "0 heads"), (dict(head_dim=80), "80"), (dict(page=24), "24"), (dict(page=8), "8"),
              (dict(page=2048), "2048"), (dict(pages=-1), "-1"), (dict(dK=None), "cache memory"),
              (dict(dV=9 * A + 8), "cache memory"), (dict(dKScale=None), "cache memory"), (dict(dVScale=11 * A + 2), "cache memory")]


def rope(**kw):
    a = dict(dtype=1, T=4, heads=4, kv=2, dim=64, x=A, ldx=512, gq=A, gk=A, eps=1e-6, rot=64, inter=0, freq=A, pos=A,
             q=2 * A, ldq=256, k=3 * A, ldk=128, cache=q8(), slots=A)
    a.update(kw)
    c = a["cache"]
    return P.hip().p2h_qk_norm_rope_q8(a["dtype"], a["T"], a["heads"], a["kv"], a["dim"], a["x"], a["ldx"], a["gq"], a["gk"],
                                       a["eps"], a["rot"], a["inter"], a["freq"], a["pos"], a["q"], a["ldq"], a["k"],
                                       a["ldk"], C.byref(c) if c is not None else None, a["slots"], None)


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=3), "element type"), (dict(T=-1), "T = -1"), (dict(dim=96), "head_dim"), (dict(heads=3), "3 heads"),
    (dict(rot=8), "rot"), (dict(eps=-1.0), "eps"), (dict(cache=None), "NULL cache"), (dict(slots=None), "slots"),
    (dict(cache=q8(heads=3)), "3 heads"), (dict(cache=q8(head_dim=128)), "heads of 128"), (dict(ldx=380), "pitch"),
    (dict(q=A + 16, ldq=512), "dQ overlaps"), (dict(cache=q8(dV=8 * A + CODES - 16)), "keys and values overlap"),
    (dict(cache=q8(dKScale=11 * A + SCALES - 4)), "keys and values overlap"),
    (dict(cache=q8(dKScale=9 * A)), "keys and values overlap"),
    (dict(cache=q8(dK=A + 1024)), "dQKV or dQ overlaps the cache"),
    (dict(cache=q8(dVScale=A + 512)), "dQKV or dQ overlaps the cache"),
    (dict(cache=q8(dKScale=2 * A)), "dQKV or dQ overlaps the cache"),
    (dict(cache=q8(dKScale=3 * A)), "dK overlaps the cache")] + [(dict(cache=q8(**kw)), part) for kw, part in BAD_CACHES])
def test_rope(kw, part):
    refused(rope(**kw), part)


def rows(c=None, **kw):
    a = dict(dtype=2, rows=40, n=3, start=A, table=A + 4096, ld=3, k=2 * A, ldk=128, v=3 * A, ldv=128)
    a.update(kw)
    c = q8() if c is None else c
    return P.hip().p2h_kv_rows_q8(a["dtype"], C.byref(c), *(a[n] for n in ("rows", "n", "start", "table", "ld", "k", "ldk", "v",
                                                                         "ldv")), None)


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=-1), "element type"), (dict(rows=-1), "rows"), (dict(rows=1 << 30), "rows"), (dict(n=-1), "-1 seq"),
    (dict(n=65537), "65537"), (dict(ld=-1), "table rows"), (dict(ld=1 << 27), "table rows"), (dict(start=None), "starts"),
    (dict(table=None), "page table"), (dict(k=None), "dK"), (dict(v=3 * A + 8), "dV"), (dict(ldk=120), "pitch"),
    (dict(ldv=132), "pitch"), (dict(v=2 * A + 128), "dK and dV overlap"), (dict(k=8 * A), "overlaps the cache"),
    (dict(v=11 * A), "overlaps the cache"), (dict(k=A), "starts or pages"), (dict(v=A + 4096), "starts or pages")]
    + [(dict(c=q8(**kw)), part) for kw, part in BAD_CACHES])
def test_rows(kw, part):
    refused(rows(**kw), part)


def test_rows_null_cache():
    refused(P.hip().p2h_kv_rows_q8(0, None, 1, 1, A, A, 1, A, 128, A, 128, None), "NULL cache")


def paged(c=None, **kw):
    a = dict(dtype=1, n=2, heads=4, q=A, ldq=256, table=30 * A, ld=3, lens=31 * A, most=48, scale=0.1, window=8, sinks=0,
             o=2 * A, ldo=256, ws=None, wsb=0)
    a.update(kw)
    c = q8() if c is None else c
    return P.hip().p2h_attention_paged_q8(a["dtype"], C.byref(c), *(a[n] for n in (
        "n", "heads", "q", "ldq", "table", "ld", "lens", "most", "scale", "window", "sinks", "o", "ldo", "ws", "wsb")), None)


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=5), "element type"), (dict(n=-1), "-1 seq"), (dict(n=70000), "70000"), (dict(heads=3), "3 heads"),
    (dict(most=-1), "-1 tokens"), (dict(most=FAR + 1), "tokens"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(window=0), "window"), (dict(sinks=-2), "sinks"), (dict(ld=-1), "table rows"), (dict(ld=1 << 27), "table rows"),
    (dict(q=None), "dQ"), (dict(o=2 * A + 4), "dO"), (dict(ldq=252), "pitch"), (dict(ldo=1 << 23), "pitch"),
    (dict(lens=None), "lengths"), (dict(table=None), "page table"), (dict(o=A), "dO overlaps dQ"),
    (dict(o=8 * A), "dO overlaps the cache"), (dict(o=11 * A + SCALES - 16), "dO overlaps the cache"),
    (dict(o=31 * A), "dO overlaps lengths")] + [(dict(c=q8(**kw)), part) for kw, part in BAD_CACHES])
def test_paged(kw, part):
    refused(paged(**kw), part)


def test_paged_workspace():
    c = q8()
    need = P.attention_paged_q8_workspace_bytes(c, 1, 4, 100000)
    assert need > 0
    big = dict(n=1, most=100000, window=FAR)
    assert paged(ws=50 * A, wsb=need - 1, **big) == E_WORKSPACE and "workspace" in P.last_error()
    assert paged(ws=50 * A + 4, wsb=need, **big) == E_WORKSPACE
    for ws in (A, A - need + 16, 8 * A, 9 * A + CODES - 16, 10 * A, 11 * A + SCALES - 16, 30 * A, 31 * A):
        refused(paged(ws=ws, wsb=need, **dict(big, o=60 * A)), "workspace overlaps")
    refused(paged(ws=60 * A + 16, wsb=need, **dict(big, o=60 * A)), "dO overlaps the workspace")
    assert P.attention_paged_q8_workspace_bytes(c, 1, 4, 20) == 0          # nothing to split
    assert P.attention_paged_q8_workspace_bytes(c, 1, 4, 100000, 64) == 0  # a short window
    assert P.attention_paged_q8_workspace_bytes(c, 1, 3, 100000) == 0 and "3 heads" in P.last_error()
    assert P.attention_paged_q8_workspace_bytes(q8(page=5), 1, 4, 100000) == 0
    assert P.hip().p2h_attention_paged_q8_workspace_bytes(None, 1, 4, 100000, 1, 0) == 0


def row_cache(**kw):
    a = dict(dtype="f16", heads=2, head_dim=64, page=16, pages=4, dK=8 * A, dV=9 * A)
    a.update(kw)
    return P.KvCache(**a)


def shared(kind, c=None, **kw):
    a = dict(dtype=1, n=4, g=2, heads=4, q=A, ldq=256, group=32 * A, shared=33 * A, table=30 * A, ld=3, lens=31 * A, ms=40,
             mo=20, scale=0.1, window=FAR, sinks=0, o=2 * A, ldo=256, ws=50 * A, wsb=1 << 19)
    a.update(kw)
    names = ("n", "g", "heads", "q", "ldq", "group", "shared", "table", "ld", "lens", "ms", "mo", "scale", "window", "sinks", "o",
             "ldo", "ws", "wsb")
    if kind == "q8":
        c = q8() if c is None else c
        return P.hip().p2h_attention_shared_q8(a["dtype"], C.byref(c), *(a[n] for n in names), None)
    c = row_cache() if c is None else c
    return P.hip().p2h_attention_shared(C.byref(c), *(a[n] for n in names), None)


@pytest.mark.parametrize("kind", ("rows", "q8"))
@pytest.mark.parametrize("kw,part", [
    (dict(n=-1), "-1 seq"), (dict(n=65537), "65537"), (dict(g=-1), "-1 groups"), (dict(g=65537), "65537 groups"),
    (dict(heads=5), "5 heads"), (dict(ms=-1), "tokens"), (dict(mo=FAR + 1), "tokens"), (dict(scale=-0.1), "scale"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks"), (dict(ld=-1), "table rows"), (dict(group=None), "groups"),
    (dict(shared=None), "prefixes"), (dict(lens=None), "lengths"), (dict(table=None), "page table"), (dict(q=A + 4), "dQ"),
    (dict(ldo=255), "pitch"), (dict(o=A), "dO overlaps dQ"), (dict(o=9 * A), "dO overlaps the cache"),
    (dict(o=30 * A), "dO overlaps lengths"), (dict(o=32 * A), "groups"), (dict(o=33 * A), "groups"),
    (dict(o=50 * A), "dO overlaps the workspace"), (dict(ws=8 * A), "workspace overlaps"), (dict(ws=A), "workspace overlaps"),
    (dict(ws=32 * A), "workspace overlaps"), (dict(ws=33 * A), "workspace overlaps"), (dict(ws=31 * A), "workspace overlaps")])
def test_shared(kind, kw, part):
    refused(shared(kind, **kw), part)


@pytest.mark.parametrize("kw,part", BAD_CACHES)
def test_shared_q8_caches(kw, part):
    refused(shared("q8", q8(**kw)), part)
    assert P.attention_shared_q8_workspace_bytes(q8(**kw), 4, 2, 4, 40, 20) == 0


def test_shared_caches_and_workspaces():
    refused(shared("rows", row_cache(dtype=5)), "type 5")
    refused(shared("rows", row_cache(page=5)), "5 tokens")
    refused(P.hip().p2h_attention_shared(None, 1, 1, 4, A, 256, A, A, A, 1, A, 1, 1, 0.1, 1, 0, A, 256, A, 1, None), "NULL cache")
    assert P.hip().p2h_attention_shared_workspace_bytes(None, 1, 1, 4, 1, 1, 1, 0) == 0
    for kind, c, size in (("rows", row_cache(), P.attention_shared_workspace_bytes),
                          ("q8", q8(), P.attention_shared_q8_workspace_bytes)):
        need = size(c, 4, 2, 4, 40, 20)
        assert 0 < need <= 1 << 19
        assert size(c, 4, 2, 3, 40, 20) == 0 and "3 heads" in P.last_error()
        assert size(c, 4, -2, 4, 40, 20) == 0 and size(c, 4, 2, 4, -1, 20) == 0 and size(c, 4, 2, 4, 40, 20, 0) == 0
        for kw in (dict(ws=None), dict(wsb=need - 1), dict(ws=50 * A + 8)):
            assert shared(kind, c, **kw) == E_WORKSPACE and "workspace" in P.last_error()


def adapters(**kw):
    a = dict(dtype="bf16", count=3, rank=16, K=64, N=40, dA=40 * A, dB=41 * A, dScale=42 * A)
    a.update(kw)
    return P.Adapters(**a)


def add(ad=None, **kw):
    a = dict(M=40, x=A, ldx=64, index=43 * A, z=2 * A, ldz=40, y=3 * A, ldy=40, ws=50 * A, wsb=1 << 19)
    a.update(kw)
    ad = adapters() if ad is None else ad
    return P.hip().p2h_adapters_add(C.byref(ad), *(a[n] for n in ("M", "x", "ldx", "index", "z", "ldz", "y", "ldy", "ws", "wsb")),
                                    None)


@pytest.mark.parametrize("kw,part", [
    (dict(ad=adapters(dtype=3)), "element type"), (dict(ad=adapters(rank=12)), "rank"), (dict(ad=adapters(rank=256)), "rank"),
    (dict(ad=adapters(rank=0)), "rank"), (dict(ad=adapters(count=-1)), "-1 adapters"), (dict(ad=adapters(K=0)), "[0, 40]"),
    (dict(ad=adapters(N=0)), "[64, 0]"), (dict(ad=adapters(K=(1 << 23) + 1), ldx=1 << 24), "adapters of"),
    (dict(ad=adapters(dA=None)), "adapters are NULL"), (dict(ad=adapters(dB=41 * A + 8)), "adapters are NULL"),
    (dict(ad=adapters(dScale=None)), "adapters are NULL"), (dict(M=-1), "M = -1"), (dict(M=1 << 20), "M ="),
    (dict(x=None), "NULL"), (dict(x=A + 1), "unaligned"), (dict(ldx=63), "ldx"), (dict(ldz=39), "ldz"), (dict(ldy=39), "ldy"),
    (dict(y=None), "NULL"), (dict(index=None), "NULL index"), (dict(y=2 * A + 2), "dZ other than in place"),
    (dict(y=2 * A, ldy=48), "dZ other than in place"), (dict(y=A + 64), "overlaps what"), (dict(y=40 * A), "overlaps what"),
    (dict(y=41 * A), "overlaps what"), (dict(y=42 * A), "overlaps what"), (dict(y=43 * A), "overlaps what"),
    (dict(ws=A), "overlaps what"), (dict(ws=41 * A), "overlaps what"), (dict(ws=43 * A), "overlaps what"),
    (dict(ws=3 * A), "workspace overlaps"), (dict(ws=2 * A), "workspace overlaps")])
def test_adapters(kw, part):
    refused(add(**kw), part)


def test_adapters_workspace():
    need = P.adapters_workspace_bytes(adapters(), 40)
    assert need >= 40 * 16 * 4 and P.adapters_workspace_bytes(adapters(), 5) == 0
    for kw in (dict(ws=None), dict(wsb=need - 1), dict(ws=50 * A + 8)):
        assert add(**kw) == E_WORKSPACE and "workspace" in P.last_error()
    assert P.adapters_workspace_bytes(adapters(rank=3), 5) == 0 and "rank" in P.last_error()
    refused(P.hip().p2h_adapters_add(None, 1, A, 64, A, A, 40, A, 40, A, 1, None), "NULL adapters")


def test_empty_calls():
    """Nothing to do is no error, whatever the pointers, and needs no device."""
    assert rope(T=0, x=None, q=None) == 0
    assert rows(rows=0, k=None) == 0 and rows(n=0, start=None) == 0
    assert paged(n=0, q=None, o=None) == 0
    for kind in ("rows", "q8"):
        assert shared(kind, n=0, q=None, ws=None) == 0 and shared(kind, g=0, group=None, ws=None) == 0
    assert add(M=0, x=None, ws=None) == 0


def test_too_many_for_one_launch():
    refused(rope(T=1 << 24), "below 2^24")
    far = q8(dK=1 << 50, dV=1 << 51, dKScale=1 << 52, dVScale=1 << 53)
    refused(paged(far, n=65536, heads=256, q=1 << 45, ldq=16384, o=1 << 47, ldo=16384), "too many")
    refused(shared("q8", far, n=65536, heads=128, q=1 << 45, ldq=8192, o=1 << 47, ldo=8192, ws=1 << 48, wsb=1 << 47), "too many")


@pytest.mark.parametrize("n,heads,kv,groups", ((65536, 65536, 1, 1), (65536, 65536, 65536, 1), (32768, 65536, 1, 7), (65536, 128, 2, 1),
                                               (1, 256, 256, 65536)))
def test_too_many_for_a_workspace_too(n, heads, kv, groups):
    """What a call refuses has no workspace, also where the products of its numbers pass 32 bits."""
    far = q8(heads=kv, dK=1 << 50, dV=1 << 51, dKScale=1 << 52, dVScale=1 << 53)
    apart = row_cache(heads=kv, dK=1 << 50, dV=1 << 51)
    assert P.attention_shared_q8_workspace_bytes(far, n, groups, heads, 100, 100) == 0 and "too many" in P.last_error()
    assert P.attention_shared_workspace_bytes(apart, n, groups, heads, 100, 100) == 0 and "too many" in P.last_error()
    ld = heads * 64
    for kind, c in (("q8", far), ("rows", apart)):
        refused(shared(kind, c, n=n, g=groups, heads=heads, q=1 << 45, ldq=ld, o=1 << 47, ldo=ld, ws=1 << 48, wsb=1 << 47), "too many")
    if groups == 1:
        assert P.attention_paged_q8_workspace_bytes(far, n, heads, 100000) == 0 and "too many" in P.last_error()


def test_as_many_as_there_may_be():
    """The most that is never too many: 2^23 - 1 rows of queries, and groups times key heads below 2^23 - 2^19."""
    one = q8(heads=1, dK=1 << 50, dV=1 << 51, dKScale=1 << 52, dVScale=1 << 53)
    many = q8(heads=120, dK=1 << 50, dV=1 << 51, dKScale=1 << 52, dVScale=1 << 53)
    assert 65535 * 120 < (1 << 23) - (1 << 19) < 65535 * 121
    assert P.attention_shared_q8_workspace_bytes(many, 65535, 65535, 120, 100, 100) > 0
    assert P.attention_shared_q8_workspace_bytes(one, 65535, 65535, 128, 100, 100) > 0
    assert P.attention_shared_q8_workspace_bytes(one, 65535, 1, 128, FAR, FAR) > 0
    assert P.attention_shared_workspace_bytes(row_cache(heads=120, dK=1 << 50, dV=1 << 51), 65535, 65535, 120, 100, 100) > 0


@pytest.mark.parametrize("off", (1, 2, 3))
def test_arrays_of_words_that_are_not_aligned(off):
    for name in ("start", "table"):
        refused(rows(**{name: 5 * A + off}), "4-byte")
    for name in ("lens", "table"):
        refused(paged(**{name: 30 * A + off}), "4-byte")
    for kind in ("rows", "q8"):
        for name in ("lens", "table", "group", "shared"):
            refused(shared(kind, **{name: 34 * A + off}), "4-byte")
    refused(add(index=43 * A + off), "4-byte")
    refused(add(adapters(dScale=42 * A + off)), "4-byte")


@pytest.mark.parametrize("off", (1, 2, 3))
def test_rope_arrays_of_words_that_are_not_aligned(off):
    for name in ("freq", "pos", "slots"):
        refused(rope(**{name: A + off}), "4-byte")
