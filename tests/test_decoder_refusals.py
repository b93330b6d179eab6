"""What a decoder layer's entries (include/p2hip.h) refuse: the arguments are checked before the device, so every refusal
here is the same with and without one. Addresses are never followed."""
import ctypes as C

import pytest

import p2gemm as P

E_ARG, E_WORKSPACE = -1, -4
A = 1 << 20   # an aligned address that nothing reads


def refused(rc, part):
    assert rc == E_ARG, (rc, P.last_error())
    assert part in P.last_error(), P.last_error()


def cache(**kw):
    a = dict(dtype="f16", heads=2, head_dim=64, page=16, pages=4, dK=A, dV=A + (1 << 20))
    a.update(kw)
    return P.KvCache(**a)


@pytest.mark.parametrize("kw,part", [
    (dict(codes=None), "NULL"), (dict(scales=None), "NULL"), (dict(K=0), "K = 0"), (dict(N=0), "N = 0"),
    (dict(K=-3), "K = -3"), (dict(group=16), "group"), (dict(group=256), "group"), (dict(N=(1 << 28) + 1), "N ="),
    (dict(K=1 << 28, N=1 << 28), "too large")])
@pytest.mark.parametrize("entry", ("p2h_q4_weight_upload", "p2h_q4_weight_wrap"))
def test_q4_weight(entry, kw, part):
    a = dict(codes=A, scales=A, zeros=None, K=128, N=16, group=32)
    a.update(kw)
    assert not getattr(P.hip(), entry)(a["codes"], a["scales"], a["zeros"], a["K"], a["N"], a["group"])
    assert part in P.last_error(), P.last_error()


def test_q4_null_weight():
    refused(P.hip().p2h_q4_gemv(0, 1, 16, 128, 1.0, A, 128, None, 0.0, A, 16, None), "NULL weight")
    refused(P.hip().p2h_q4_gemv(7, 1, 16, 128, 1.0, A, 128, None, 0.0, A, 16, None), "element type")
    assert P.hip().p2h_q4_weight_shape(None, None, None, None) == E_ARG
    assert P.hip().p2h_q4_weight_device_bytes(None) == 0
    P.hip().p2h_q4_weight_free(None)


def rope(**kw):
    a = dict(dtype=1, T=4, heads=4, kv=2, dim=64, x=A, ldx=512, gq=A, gk=A, eps=1e-6, rot=64, inter=0, freq=A, pos=A,
             q=2 * A, ldq=256, k=3 * A, ldk=128, cache=None, slots=None)
    a.update(kw)
    c = a["cache"]
    return P.hip().p2h_qk_norm_rope(a["dtype"], a["T"], a["heads"], a["kv"], a["dim"], a["x"], a["ldx"], a["gq"], a["gk"],
                                    a["eps"], a["rot"], a["inter"], a["freq"], a["pos"], a["q"], a["ldq"], a["k"], a["ldk"],
                                    C.byref(c) if c is not None else None, a["slots"], None)


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=3), "element type"), (dict(T=-1), "T = -1"), (dict(dim=96), "head_dim"), (dict(heads=3), "3 heads"),
    (dict(kv=0), "key heads"), (dict(rot=8), "rot"), (dict(rot=80), "rot"), (dict(rot=-16), "rot"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(k=None), "neither"), (dict(x=None), "dQKV"), (dict(x=A + 8), "dQKV"),
    (dict(ldx=380), "pitch"), (dict(ldx=516), "pitch"), (dict(q=None), "dQ"), (dict(ldq=255), "pitch"),
    (dict(ldk=120), "pitch"), (dict(gq=None), "norm weights"), (dict(pos=None), "positions"), (dict(freq=None), "frequencies"),
    (dict(cache=cache()), "slots"), (dict(cache=cache(heads=3), slots=A), "3 heads"),
    (dict(cache=cache(dtype="f32"), slots=A), "type 0"), (dict(cache=cache(page=24), slots=A), "24"),
    (dict(cache=cache(page=8), slots=A), "8"), (dict(cache=cache(pages=-1), slots=A), "-1"),
    (dict(cache=cache(dK=None), slots=A), "cache memory"), (dict(cache=cache(dV=A + 4), slots=A), "cache memory"),
    (dict(q=A + 16, ldq=512), "dQ overlaps"), (dict(q=A, ldq=256), "dQ overlaps"), (dict(k=A, ldk=512), "dK overlaps"),
    (dict(k=2 * A + 256, ldk=256), "dQ and dK overlap"), (dict(q=A + 768, ldq=512, cache=cache(), slots=A), "dQ overlaps")])
def test_rope(kw, part):
    refused(rope(**kw), part)


def win(**kw):
    a = dict(dtype=2, qr=40, kr=50, n=1, qs=None, ks=None, heads=4, kv=2, dim=128, q=A, ldq=512, k=2 * A, ldk=256, v=3 * A,
             ldv=256, scale=0.1, window=8, ahead=0, sinks=0, o=4 * A, ldo=512)
    a.update(kw)
    return P.hip().p2h_attention_window(*(a[n] for n in ("dtype", "qr", "kr", "n", "qs", "ks", "heads", "kv", "dim", "q",
                                                         "ldq", "k", "ldk", "v", "ldv", "scale", "window", "ahead", "sinks",
                                                         "o", "ldo")), None)


@pytest.mark.parametrize("kw,part", [
    (dict(dtype=-1), "element type"), (dict(dim=32), "head_dim"), (dict(heads=5), "5 heads"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(window=0), "window"), (dict(window=(1 << 30) + 1), "window"), (dict(ahead=-1), "ahead"), (dict(sinks=-1), "sinks"),
    (dict(qr=-1), "rows"), (dict(kr=1 << 30), "rows"), (dict(n=2), "starts"), (dict(qs=A), "starts"), (dict(n=-1), "-1 seq"),
    (dict(q=None), "dQ"), (dict(k=A + 2), "dK"), (dict(v=None), "dV"), (dict(o=A + 8), "dO"), (dict(ldq=508), "pitch"),
    (dict(ldk=260), "pitch"), (dict(ldv=255), "pitch"), (dict(ldo=0), "pitch"), (dict(o=A), "dO overlaps dQ"),
    (dict(o=2 * A), "overlaps dK or dV"), (dict(o=3 * A + 512 * 49), "overlaps dK or dV")])
def test_window(kw, part):
    refused(win(**kw), part)


def paged(c=None, **kw):
    a = dict(n=2, heads=4, q=A, ldq=256, table=A, ld=3, lens=A, most=48, scale=0.1, window=8, sinks=0, o=2 * A, ldo=256,
             ws=None, wsb=0)
    a.update(kw)
    c = cache() if c is None else c
    return P.hip().p2h_attention_paged(C.byref(c), *(a[n] for n in ("n", "heads", "q", "ldq", "table", "ld", "lens", "most",
                                                                    "scale", "window", "sinks", "o", "ldo", "ws", "wsb")), None)


@pytest.mark.parametrize("kw,part", [
    (dict(c=cache(dtype=5)), "type 5"), (dict(c=cache(page=0)), "0 tokens"), (dict(c=cache(page=2048)), "2048"),
    (dict(c=cache(head_dim=80)), "80"), (dict(c=cache(heads=0)), "0 heads"), (dict(n=-1), "-1 seq"), (dict(n=70000), "70000"),
    (dict(heads=3), "3 heads"), (dict(most=-1), "-1 tokens"), (dict(scale=0.0), "scale"), (dict(window=0), "window"),
    (dict(sinks=-2), "sinks"), (dict(ld=-1), "table rows"), (dict(ld=1 << 27), "table rows"), (dict(q=None), "dQ"),
    (dict(o=2 * A + 4), "dO"), (dict(ldq=252), "pitch"), (dict(lens=None), "lengths"), (dict(table=None), "page table"),
    (dict(o=A), "overlaps")])
def test_paged(kw, part):
    refused(paged(**kw), part)


def test_paged_workspace():
    c = cache()
    need = P.attention_paged_workspace_bytes(c, 1, 4, 100000)
    assert need > 0
    big = dict(n=1, most=100000, window=1 << 30)
    assert paged(ws=A, wsb=need - 1, **big) == E_WORKSPACE and "workspace" in P.last_error()
    assert paged(ws=A + 4, wsb=need, **big) == E_WORKSPACE
    assert P.attention_paged_workspace_bytes(c, 1, 4, 20) == 0          # nothing to split
    assert P.attention_paged_workspace_bytes(c, 1, 4, 100000, 64) == 0  # a short window
    assert P.attention_paged_workspace_bytes(c, 1, 3, 100000) == 0      # refused
    assert "3 heads" in P.last_error()
    assert P.attention_paged_workspace_bytes(cache(page=5), 1, 4, 100000) == 0


def test_empty_calls():
    """Nothing to do is no error, whatever the pointers, and needs no device."""
    assert rope(T=0, x=None, q=None) == 0
    assert win(qr=0, q=None, o=None) == 0
    assert win(n=0, qs=A, ks=A) == 0
    assert paged(n=0, q=None, o=None) == 0


@pytest.mark.parametrize("kw,part", [
    (dict(x=A + (1 << 20), cache=cache(dK=8 * A, dV=2 * A + 1024), slots=A, q=20 * A), "dQKV or dQ overlaps the cache"),
    (dict(cache=cache(dK=8 * A, dV=2 * A + 1024), slots=A), "dQKV or dQ overlaps the cache"),
    (dict(cache=cache(dK=3 * A - 16, dV=8 * A), slots=A), "dK overlaps the cache"),
    (dict(cache=cache(dK=8 * A, dV=8 * A + 4 * 2 * 16 * 64 * 2 - 16), slots=A), "keys and values overlap")])
def test_rope_and_its_cache(kw, part):
    refused(rope(**kw), part)


@pytest.mark.parametrize("kw,part", [(dict(K=(1 << 28) + 1), "K ="), (dict(N=(1 << 27) + 1, K=1), "too large"),
                                     (dict(K=1 << 28, N=16 * 8), "too large"), (dict(K=128 << 12, N=16 << 12), "too large")])
def test_q4_weight_limits(kw, part):
    """K to 2^28, N to 2^27, ceil(K / 128) · ceil(N / 16) below 2^24."""
    test_q4_weight("p2h_q4_weight_wrap", kw, part)


def test_launch_limits():
    """As the header states them: (q_rows / 128 + 1 + n_seqs) · heads below 2^23 − 2^11; n_seqs · heads below 2^23."""
    far = dict(q=1 << 45, k=1 << 46, v=1 << 47, o=1 << 48)
    refused(win(n=(1 << 21) - 512 - 1, qs=A, ks=A, **far), "too many")
    refused(paged(cache(dK=1 << 50, dV=1 << 51), n=65536, heads=128, q=1 << 45, ldq=8192, o=1 << 47, ldo=8192), "too many")


def test_rope_of_one_row_in_place():
    """A single row has no pitch: in place whatever pitches are given. That it passes is seen by what is refused next."""
    last = dict(cache=cache(dK=8 * A, dV=A + 1024 - 16), slots=A)   # the cache's values on the row's end
    for kw in (dict(q=A, ldq=256), dict(q=A, ldq=512), dict(q=A, ldq=256, k=A + 512, ldk=128),
               dict(q=A, ldq=1024, k=A + 512, ldk=256)):
        refused(rope(T=1, **dict(dict(k=3 * A), **kw), **last), "dQKV or dQ overlaps the cache")
        if kw["ldq"] != 512:
            refused(rope(T=2, **dict(dict(k=3 * A), **kw), **last), "dQ overlaps dQKV")
    refused(rope(T=1, q=A + 16, ldq=256), "dQ overlaps dQKV")
    refused(rope(T=1, q=A, ldq=256, k=A + 528, ldk=128), "dK overlaps dQKV")


def test_paged_output_apart_from_what_it_reads():
    c = cache(dK=8 * A, dV=9 * A)
    size = 4 * 2 * 16 * 64 * 2
    refused(paged(c, o=8 * A + size - 16), "dO overlaps the cache")
    refused(paged(c, o=9 * A - 256 * 2 - 16), "dO overlaps the cache")
    need = P.attention_paged_workspace_bytes(c, 1, 4, 100000)
    refused(paged(c, n=1, most=100000, window=1 << 30, ws=2 * A - need + 16, wsb=need), "dO overlaps the workspace")


def test_paged_workspace_apart_from_what_it_reads():
    """The parts are written while other workgroups still read queries, keys, lengths and pages."""
    c = cache(dK=8 * A, dV=9 * A)
    size = 4 * 2 * 16 * 64 * 2
    need = P.attention_paged_workspace_bytes(c, 1, 4, 100000)
    big = dict(n=1, most=100000, window=1 << 30, wsb=need, q=20 * A, lens=30 * A, table=40 * A, ld=7, o=50 * A)
    for ws in (8 * A, 8 * A + size - 16, 9 * A - need + 16, 9 * A,   # the cache
               20 * A, 20 * A - need + 16, 20 * A + 496,             # one row of 256 queries
               30 * A, 30 * A - need + 16, 40 * A + 16, 40 * A - need + 16):
        refused(paged(c, ws=ws, **big), "workspace overlaps")
    for ws in (8 * A + size, 9 * A - need, 20 * A + 512, 30 * A + 16, 40 * A + 32):   # side by side: refused only for dO
        refused(paged(c, ws=ws, **dict(big, o=8 * A + 16)), "dO overlaps the cache")


def test_too_many_for_one_launch():
    refused(rope(T=1 << 24), "below 2^24")
    refused(win(qr=1 << 29, kr=1 << 29, heads=8, o=1 << 50, k=1 << 51, v=1 << 52, ldk=256, ldq=1024, ldo=1024), "too many")
    refused(paged(cache(dK=1 << 50, dV=1 << 51), n=65536, heads=256, q=1 << 45, ldq=16384, o=1 << 47, ldo=16384), "too many")
    assert not P.hip().p2h_q4_weight_wrap(A, A, None, 1 << 20, 1 << 16, 32) and "too large" in P.last_error()
