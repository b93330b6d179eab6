"""A served batch of a decoder next to the encoder: what it costs, as cases that can be timed and compared.

Six entries are called the way such a program calls them:

  put8      p2h_qk_norm_rope_q8, then p2h_kv_rows_q8: head norms and rotation of new q | k | v rows, their keys and values
            into a paged cache of 8 bits, and the kept keys and values read back as rows, as a prompt's chunk does before
            its windowed attention
  rows8     p2h_kv_rows_q8 alone: what ragged sequences have kept, as rows
  paged8    p2h_attention_paged_q8: one new token per sequence over the 8-bit cache
  shared    p2h_attention_shared (cache "rows", of the rows' type) and p2h_attention_shared_q8 (cache "q8"): the same where
            groups of sequences share a long prefix
  adapters  p2h_adapters_add: low-rank adapters of many requests at once beside a projection that all of them share

Widths are the encoder's (1024 channels, 8 heads of 128, feed-forward 4096; 375 frames a 30 s window, 6000 sixteen of them)
and generic decoder ones (32 query heads over 8 key heads, heads of 64).

`own` False computes the plain form: elementary torch operations in 32 bits (angles in 64), rounded once at the end.
"""
import itertools
import math
import os
import sys

import torch   # before the binding, so that the process holds one HIP runtime

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FAR = 1 << 30   # a window that reaches every key


def listed():
    return [
        # one new token of each of 16 sequences, put into pages of their own and read back: launches and latency
        {"name": "put8_bf16_t16", "op": "put8", "type": "bf16", "T": 16, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": "half", "page": 16, "far": 131072},
        # sixteen windows as one prompt
        {"name": "put8_f16_t6000", "op": "put8", "type": "f16", "T": 6000, "heads": 32, "kv": 8, "dim": 128, "rot": 64,
         "pairs": "next", "page": 64, "far": 6000},
        # one 30 s window's kept keys and values as fp32 rows
        {"name": "rows8_f32_t375", "op": "rows8", "type": "f32", "seqs": 1, "longest": 375, "kv": 8, "dim": 128, "page": 16},
        # thirteen ragged prompts before their next chunks
        {"name": "rows8_bf16_ragged", "op": "rows8", "type": "bf16", "seqs": 13, "longest": 8191, "kv": 8, "dim": 128,
         "page": 64},
        # one sequence's next token after a 30 s window: latency
        {"name": "paged8_f32_b1_375", "op": "paged8", "type": "f32", "seqs": 1, "longest": 375, "heads": 8, "kv": 8,
         "dim": 128, "page": 16, "window": FAR, "sinks": 0},
        # a served batch of ragged lengths
        {"name": "paged8_bf16_b32_8192", "op": "paged8", "type": "bf16", "seqs": 32, "longest": 8192, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "window": FAR, "sinks": 0},
        # four hypotheses behind one 30 s window
        {"name": "shared_f32_b4_p375", "op": "shared", "cache": "rows", "type": "f32", "groups": 1, "per": 4, "prefix": 375,
         "own": 38, "heads": 8, "kv": 8, "dim": 128, "page": 16, "window": FAR, "sinks": 0},
        # 64 requests with one long instruction before their own short ones: the largest shared prefix
        {"name": "shared_bf16_b64_p32768", "op": "shared", "cache": "rows", "type": "bf16", "groups": 1, "per": 64,
         "prefix": 32768, "own": 512, "heads": 32, "kv": 8, "dim": 128, "page": 64, "window": FAR, "sinks": 0},
        # three documents with eight questions each, heads of 64, an 8-bit cache
        {"name": "shared8_f16_g3_p30001", "op": "shared", "cache": "q8", "type": "f16", "groups": 3, "per": 8,
         "prefix": 30001, "own": 1000, "heads": 32, "kv": 8, "dim": 64, "page": 32, "window": FAR, "sinks": 0},
        # one token through a square projection with its request's adapter: latency
        {"name": "adapters_f16_m1_1024", "op": "adapters", "type": "f16", "M": 1, "K": 1024, "N": 1024, "rank": 8,
         "count": 4, "rows": 1},
        # 32 requests' tokens through a feed-forward's up-projection of an odd width, sixteen adapters
        {"name": "adapters_bf16_m32_odd", "op": "adapters", "type": "bf16", "M": 32, "K": 4096, "N": 16389, "rank": 16,
         "count": 16, "rows": 1},
        # sixteen windows' fp32 rows (the encoder's own type) through its up-projection, each window with its adapter
        {"name": "adapters_f32_t6000", "op": "adapters", "type": "f32", "M": 6000, "K": 1024, "N": 4096, "rank": 32,
         "count": 8, "rows": 375},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, t = rng.choice(("put8", "rows8", "paged8", "shared", "shared", "adapters", "adapters")), \
        rng.choice(("f32", "f16", "bf16"))
    if op == "adapters":
        rows = rng.choice((1, 1, _log_int(rng, 2, 500)))
        M = _log_int(rng, 1, 128) if rows == 1 else min(6000, rows * _log_int(rng, 1, 32))
        return {"op": op, "type": t, "M": M, "K": _log_int(rng, 64, 8192), "N": _log_int(rng, 64, 16384),
                "rank": rng.choice((8, 16, 32, 64)), "count": _log_int(rng, 1, 32), "rows": rows}
    dim, kv = rng.choice((64, 128)), rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 2, 4) if kv == 8 else (1, 3, 4, 8))
    page = rng.choice((16, 32, 64, 256))
    if op == "put8":
        # 16-bit rows: an fp32 key's code may lie on a border that the last bit of its norm decides
        return {"op": op, "type": rng.choice(("f16", "bf16")), "T": _log_int(rng, 1, 6000), "heads": heads, "kv": kv,
                "dim": dim, "rot": rng.choice((dim, dim // 2)), "pairs": rng.choice(("half", "next")), "page": page,
                "far": _log_int(rng, 8000, 1000000)}
    if op == "rows8":
        seqs = _log_int(rng, 1, 64)
        return {"op": op, "type": t, "seqs": seqs, "longest": _log_int(rng, 1, 131072 // seqs), "kv": kv, "dim": dim,
                "page": page}
    window = FAR if rng.random() < 0.5 else _log_int(rng, 16, 16384)
    base = {"op": op, "type": t, "heads": heads, "kv": kv, "dim": dim, "page": page, "window": window,
            "sinks": rng.choice((0, 0, 1, 4, 16))}
    if op == "paged8":
        seqs = _log_int(rng, 1, 64)
        return dict(base, seqs=seqs, longest=_log_int(rng, 1, 262144 // seqs))
    groups, per = rng.choice((1, 1, 2, 3, 5)), _log_int(rng, 1, 48)
    return dict(base, cache=rng.choice(("rows", "q8")), groups=groups, per=per,
                prefix=_log_int(rng, 256, 65536 // groups), own=_log_int(rng, 1, 32768 // (groups * per)))


# ── inputs, from the seed alone ─────────────────────────────────────────────────────────────────────────────────

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _whole(g, lo, hi, *shape):
    """Whole numbers of [lo, hi)."""
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _kept(g, pages, kv, page, dim):
    """Codes and scales of heads of normal values of about 1: the largest of a head about 2.7 times as large."""
    codes = [torch.randn(pages, kv, page, dim, generator=g, device="cuda").mul_(45.0).round_().clamp_(-127, 127)
             .to(torch.int8) for _ in range(2)]
    scales = [(0.5 + torch.rand(pages, kv, page, generator=g, device="cuda")) / 45.0 for _ in range(2)]
    return {"kc": codes[0], "vc": codes[1], "ks": scales[0], "vs": scales[1]}


def _inputs(case, seed):
    """What a case's computation is a function of."""
    c, g, dt = case, _gen(seed), TYPES[case["type"]]
    if c["op"] == "adapters":
        M, K, N, r, n = c["M"], c["K"], c["N"], c["rank"], c["count"]
        # activations with one value in a thousand twenty times as large
        x = torch.randn(M, K, generator=g, device="cuda")
        x = (x * torch.where(torch.rand(M, K, generator=g, device="cuda") < 0.001, 20.0, 1.0)).to(dt)
        requests = -(-M // c["rows"])
        of = _whole(g, 0, n, requests)
        of = torch.where(torch.rand(requests, generator=g, device="cuda") < 0.1, torch.full_like(of, -1), of)
        of[0] = 0   # one request in ten has no adapter, but not the only one
        return {"x": x, "z": _normal(g, M, N, dtype=dt), "index": of.repeat_interleave(c["rows"])[:M].contiguous(),
                "a": _normal(g, n, r, K, dtype=dt, scale=K ** -0.5), "b": _normal(g, n, N, r, dtype=dt, scale=r ** -0.5),
                "scale": 0.5 + torch.rand(n, generator=g, device="cuda")}
    Hk, Dh, page = c["kv"], c["dim"], c["page"]
    if c["op"] == "put8":
        T, H = c["T"], c["heads"]
        i = {"qkv": _normal(g, T, (H + 2 * Hk) * Dh, dtype=dt, scale=2.0),
             "gq": 0.5 + torch.rand(Dh, generator=g, device="cuda"),
             "gk": 0.5 + torch.rand(Dh, generator=g, device="cuda"),
             "freq": torch.pow(10000.0, -torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64)
                               / c["rot"]).float(),
             # a prompt's consecutive positions, or (few tokens) each sequence's own
             "pos": (torch.arange(T, device="cuda", dtype=torch.int32) + c["far"] - T if T > 64
                     else _whole(g, 0, c["far"], T))}
        pages = -(-T // page) + 3 if T > 64 else T + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(T, device="cuda")
        # a prompt fills page after page from the middle of one; single tokens land in pages of their own
        slots = order[(t + page // 2) // page] * page + (t + page // 2) % page if T > 64 else \
            order[t] * page + _whole(g, 0, page, T).long()
        i.update(_kept(g, pages, Hk, page, Dh), slots=slots.to(torch.int32), table=order.to(torch.int32).view(1, -1),
                 starts=torch.tensor([0, pages * page], dtype=torch.int32, device="cuda"), rows=pages * page)
        return i
    if c["op"] == "rows8":
        n, longest = c["seqs"], c["longest"]
        per = -(-longest // page)
        lens = [longest] + [1 + longest // 3 + k * (longest - longest // 3) // n for k in range(1, n)]
        starts = torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device="cuda")
        return dict(_kept(g, n * per, Hk, page, Dh), starts=starts, rows=sum(lens),
                    table=torch.randperm(n * per, generator=g, device="cuda").view(n, per).to(torch.int32))
    H = c["heads"]
    if c["op"] == "paged8":
        B, longest = c["seqs"], c["longest"]
        per = -(-longest // page)
        lens = _whole(g, 1 + longest // 3, longest + 1, B)
        lens[0] = longest
        return dict(_kept(g, B * per, Hk, page, Dh), q=_normal(g, B, H * Dh, dtype=dt), lens=lens,
                    table=torch.randperm(B * per, generator=g, device="cuda").view(B, per).to(torch.int32))
    # groups of as many sequences each; a group's prefix pages come first in the tables of all of its sequences, and the page
    # that a prefix ends in is each one's own from there on
    ng, per, P, O = c["groups"], c["per"], c["prefix"], c["own"]
    B = ng * per
    held, tail = -(-P // page), -(-O // page) + 1
    shared = _whole(g, 1 + P * 2 // 3, P + 1, ng)
    shared[0] = P
    behind = _whole(g, 1 + O // 3, O + 1, B)
    behind[0] = O
    order = torch.randperm(ng * held + B * tail, generator=g, device="cuda")
    first, rest = order[:ng * held].view(ng, held), order[ng * held:].view(B, tail)
    at = torch.arange(held + tail, device="cuda").expand(B, -1)
    whole = (shared.long() // page).repeat_interleave(per)[:, None]   # pages that the prefix fills
    table = torch.where(at < whole, first.repeat_interleave(per, 0).gather(1, at.clamp(max=held - 1)),
                        rest.gather(1, (at - whole).clamp(0, tail - 1)))
    lead = torch.arange(ng, device="cuda") * per   # its first sequence has the prefix's last page too
    table[lead[:, None], at[:ng, :held]] = torch.where(at[:ng, :held] < whole[lead], table[lead, :held], first)
    last = (shared.long() - 1) // page             # and goes on in that
    more = at[:ng] - last[:, None] - 1
    table[lead] = torch.where(more >= 0, rest[lead].gather(1, more.clamp(0, tail - 1)), table[lead])
    i = {"q": _normal(g, B, H * Dh, dtype=dt), "lens": shared.repeat_interleave(per) + behind, "shared": shared,
         "starts": (torch.arange(ng + 1, device="cuda") * per).to(torch.int32), "table": table.to(torch.int32)}
    pages = ng * held + B * tail
    if c["cache"] == "q8":
        i.update(_kept(g, pages, Hk, page, Dh))
    else:
        i.update(kc=_normal(g, pages, Hk, page, Dh, dtype=dt), vc=_normal(g, pages, Hk, page, Dh, dtype=dt))
    return i


# ── what a program holds ────────────────────────────────────────────────────────────────────────────────────────

_held = {}


def _binding():
    """The framework's binding and the stream this program works on."""
    if not _held:
        sys.path.insert(0, os.path.join(ROOT, "phonon-2-c_amd"))
        import p2gemm
        p2gemm.init()
        _held.update(P=p2gemm, stream=p2gemm.Stream())
    return _held["P"], _held["stream"]


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=dict(case))
    torch.cuda.synchronize()   # the framework works on streams of its own
    if not own:
        return st
    P, stream = _binding()
    c, dt = case, TYPES[case["type"]]
    st["P"], st["stream"] = P, stream.ptr
    if c["op"] == "adapters":
        st["set"] = P.Adapters(c["type"], c["count"], c["rank"], c["K"], c["N"], st["a"].data_ptr(), st["b"].data_ptr(),
                               st["scale"].data_ptr())
        st["ws"] = P.Workspace(P.adapters_workspace_bytes(st["set"], c["M"]))
        st["y"] = torch.empty_like(st["z"])
        return st
    if "ks" in st:
        st["cache"] = P.KvCacheQ8(c["kv"], c["dim"], c["page"], st["kc"].shape[0], st["kc"].data_ptr(),
                                  st["vc"].data_ptr(), st["ks"].data_ptr(), st["vs"].data_ptr())
    else:
        st["cache"] = P.KvCache(c["type"], c["kv"], c["dim"], c["page"], st["kc"].shape[0], st["kc"].data_ptr(),
                                st["vc"].data_ptr())
    if c["op"] in ("put8", "rows8"):
        st["ok"] = torch.empty(st["rows"], c["kv"] * c["dim"], device="cuda", dtype=dt)
        st["ov"] = torch.empty_like(st["ok"])
    if c["op"] == "put8":
        st["oq"] = torch.empty(c["T"], c["heads"] * c["dim"], device="cuda", dtype=dt)
    if c["op"] == "paged8":
        st["o"] = torch.empty_like(st["q"])
        st["ws"] = P.Workspace(P.attention_paged_q8_workspace_bytes(st["cache"], c["seqs"], c["heads"], c["longest"],
                                                                    c["window"], c["sinks"]))
    if c["op"] == "shared":
        st["o"] = torch.empty_like(st["q"])
        bytes_of = P.attention_shared_q8_workspace_bytes if "ks" in st else P.attention_shared_workspace_bytes
        st["ws"] = P.Workspace(bytes_of(st["cache"], c["groups"] * c["per"], c["groups"], c["heads"], c["prefix"], c["own"],
                                        c["window"], c["sinks"]))
    return st


def run(st):
    return _run_own(st) if own else _PLAIN[st["case"]["op"]](st)


def _run_own(st):
    c, P, s = st["case"], st["P"], st["stream"]
    if c["op"] == "adapters":
        P.adapters_add_dev(st["set"], c["M"], st["x"].data_ptr(), c["K"], st["index"].data_ptr(), st["z"].data_ptr(), c["N"],
                           st["y"].data_ptr(), c["N"], st["ws"].ptr, st["ws"].nbytes, s)
        return st["y"]
    Hk, Dh = c["kv"], c["dim"]
    if c["op"] in ("put8", "rows8"):
        if c["op"] == "put8":
            H = c["heads"]
            P.qk_norm_rope_q8_dev(c["type"], c["T"], H, Hk, Dh, st["qkv"].data_ptr(), (H + 2 * Hk) * Dh,
                                  st["gq"].data_ptr(), st["gk"].data_ptr(), 1e-6, c["rot"], c["pairs"] == "next",
                                  st["freq"].data_ptr(), st["pos"].data_ptr(), st["oq"].data_ptr(), H * Dh, None, 0,
                                  st["cache"], st["slots"].data_ptr(), s)
        P.kv_rows_q8_dev(c["type"], st["cache"], st["rows"], st["starts"].numel() - 1, st["starts"].data_ptr(),
                         st["table"].data_ptr(), st["table"].shape[1], st["ok"].data_ptr(), Hk * Dh, st["ov"].data_ptr(),
                         Hk * Dh, s)
        return (st["oq"], st["ok"], st["ov"]) if c["op"] == "put8" else (st["ok"], st["ov"])
    H = c["heads"]
    if c["op"] == "paged8":
        P.attention_paged_q8_dev(c["type"], st["cache"], c["seqs"], H, st["q"].data_ptr(), H * Dh, st["table"].data_ptr(),
                                 st["table"].shape[1], st["lens"].data_ptr(), c["longest"], Dh ** -0.5, c["window"],
                                 c["sinks"], st["o"].data_ptr(), H * Dh, st["ws"].ptr, st["ws"].nbytes, s)
        return st["o"]
    args = (st["cache"], c["groups"] * c["per"], c["groups"], H, st["q"].data_ptr(), H * Dh, st["starts"].data_ptr(),
            st["shared"].data_ptr(), st["table"].data_ptr(), st["table"].shape[1], st["lens"].data_ptr(), c["prefix"],
            c["own"], Dh ** -0.5, c["window"], c["sinks"], st["o"].data_ptr(), H * Dh, st["ws"].ptr, st["ws"].nbytes, s)
    if "ks" in st:
        P.attention_shared_q8_dev(c["type"], *args)
    else:
        P.attention_shared_dev(*args)
    return st["o"]


# ── the plain forms ─────────────────────────────────────────────────────────────────────────────────────────────

def _plain_adapters(st):
    c = st["case"]
    M, r, n = c["M"], c["rank"], c["count"]
    # the rows times every adapter at once, each row's own taken, the others' places zeros
    h = (st["x"].float() @ st["a"].float().view(n * r, -1).t()).view(M, n, r)
    mine = (st["index"][:, None] == torch.arange(n, device=h.device)).float() * st["scale"]
    d = (h * mine[:, :, None]).view(M, n * r) @ st["b"].float().transpose(1, 2).reshape(n * r, -1)
    return (st["z"].float() + d).to(st["z"].dtype)


def _quantised(x):
    """[..., Dh] in 32 bits → codes and the scale of each head."""
    top = x.abs().amax(-1)
    some = top > 0
    by = torch.where(some, 127.0 / torch.where(some, top, torch.ones_like(top)), torch.zeros_like(top))
    return torch.round(x * by[..., None]).to(torch.int8), top / 127.0


def _plain_rows8(st):
    c = st["case"]
    page, rows = c["page"], torch.arange(st["rows"], device=st["starts"].device)
    seq = torch.searchsorted(st["starts"].long(), rows, right=True) - 1
    t = rows - st["starts"].long()[seq]
    at = st["table"].long()[seq, t // page]
    return tuple((st[x + "c"][at, :, t % page].float() * st[x + "s"][at, :, t % page][..., None])
                 .reshape(rows.numel(), -1).to(TYPES[c["type"]]) for x in "kv")


def _plain_put8(st):
    c = st["case"]
    T, H, Hk, Dh, R = c["T"], c["heads"], c["kv"], c["dim"], c["rot"]
    x = st["qkv"].float().view(T, H + 2 * Hk, Dh)
    qk, v = x[:, :H + Hk], x[:, H + Hk:]
    gain = torch.cat((st["gq"].expand(H, Dh), st["gk"].expand(Hk, Dh)))
    y = qk / torch.sqrt((qk * qk).mean(2, keepdim=True) + 1e-6) * gain
    angle = st["pos"].double()[:, None, None] * st["freq"].double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = (y[..., :R // 2], y[..., R // 2:R]) if c["pairs"] == "half" else (y[..., 0:R:2], y[..., 1:R:2])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.cat(turned, 2) if c["pairs"] == "half" else torch.stack(turned, 3).flatten(2)
    y = torch.cat((turned, y[..., R:]), 2)
    at, off = st["slots"].long() // c["page"], st["slots"].long() % c["page"]
    st["kc"][at, :, off], st["ks"][at, :, off] = _quantised(y[:, H:])
    st["vc"][at, :, off], st["vs"][at, :, off] = _quantised(v)
    return (y[:, :H].reshape(T, H * Dh).to(st["qkv"].dtype), *_plain_rows8(st))


def _scores(q, k, seen, scale):
    """q [.., H, n, Dh], k [.., H, m, Dh], seen [.., n, m] with H's axis: minus infinity where it is not seen."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    return torch.where(seen, s, torch.full_like(s[..., :1, :1], -math.inf))


def _plain_paged8(st):
    c = st["case"]
    B, H, Hk, Dh = c["seqs"], c["heads"], c["kv"], c["dim"]
    # the pages in order: [B][pages][Hk][page][Dh] → [B][Hk][keys][Dh]
    k, v = ((st[t + "c"][st["table"].long()].float() * st[t + "s"][st["table"].long()][..., None])
            .transpose(1, 2).reshape(B, Hk, -1, Dh) for t in "kv")
    at = torch.arange(k.shape[2], device=k.device)
    last = st["lens"].long()[:, None] - 1
    seen = (at <= last) & ((last - at < c["window"]) | (at < c["sinks"]))
    s = _scores(st["q"].float().view(B, Hk, H // Hk, Dh), k, seen[:, None, None, :], Dh ** -0.5)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.reshape(B, H * Dh).to(st["q"].dtype)


def _plain_shared(st):
    c = st["case"]
    ng, per, H, Hk, Dh, page = c["groups"], c["per"], c["heads"], c["kv"], c["dim"], c["page"]
    B, G = ng * per, H // Hk
    table, shared, dev = st["table"].long(), st["shared"].long(), st["q"].device
    last = st["lens"].long()[:, None] - 1
    visible = lambda t: (t <= last) & ((last - t < c["window"]) | (t < c["sinks"]))   # noqa: E731

    def tokens(seqs, t, x):
        """Keys or values of tokens t [n][m] of sequences [n]: [n][Hk][m][Dh]."""
        at = table[seqs[:, None], (t // page).clamp(max=table.shape[1] - 1)]
        y = st[x + "c"][at, :, t % page].float()
        return (y * st[x + "s"][at, :, t % page][..., None] if x + "s" in st else y).transpose(1, 2).contiguous()

    q = st["q"].float().view(ng, per, Hk, G, Dh).transpose(1, 2).reshape(ng, Hk, per * G, Dh)
    # every group's prefix, from the table of its first sequence
    t = torch.arange(c["prefix"], device=dev).expand(ng, -1)
    k, v = (tokens(torch.arange(ng, device=dev) * per, t, x) for x in "kv")
    seen = (t < shared[:, None]).repeat_interleave(per, 0) & visible(t[:1])
    s1 = _scores(q, k, seen.view(ng, 1, per, 1, -1).expand(-1, -1, -1, G, -1).reshape(ng, 1, per * G, -1), Dh ** -0.5)
    # what each sequence has behind it
    t = shared.repeat_interleave(per)[:, None] + torch.arange(c["own"], device=dev)
    k2, v2 = (tokens(torch.arange(B, device=dev), t, x) for x in "kv")
    s2 = _scores(st["q"].float().view(B, Hk, G, Dh), k2, visible(t)[:, None, None, :], Dh ** -0.5)
    top2 = s2.amax(-1, keepdim=True)
    top = torch.maximum(s1.amax(-1, keepdim=True).view(ng, Hk, per, G, 1).transpose(1, 2).reshape(B, Hk, G, 1), top2)
    p1 = torch.exp(s1 - top.view(ng, per, Hk, G, 1).transpose(1, 2).reshape(ng, Hk, per * G, 1))
    p2 = torch.exp(s2 - top)
    back = lambda x: x.view(ng, Hk, per, G, -1).transpose(1, 2).reshape(B, Hk, G, -1)   # noqa: E731
    o = (back(torch.matmul(p1, v)) + torch.matmul(p2, v2)) / (back(p1.sum(-1, keepdim=True)) + p2.sum(-1, keepdim=True))
    return o.reshape(B, H * Dh).to(st["q"].dtype)


_PLAIN = {"put8": _plain_put8, "rows8": _plain_rows8, "paged8": _plain_paged8, "shared": _plain_shared,
          "adapters": _plain_adapters}


# ── what a pass cannot do without ───────────────────────────────────────────────────────────────────────────────

def work(case):
    c = case
    e = 4 if c["type"] == "f32" else 2
    if c["op"] == "adapters":
        M, K, N, r = c["M"], c["K"], c["N"], c["rank"]
        used = min(c["count"], -(-M // c["rows"]))
        return {"bytes": e * (M * (K + 2 * N) + used * r * (K + N)) + 4 * M, "flops": 2 * M * r * (K + N)}
    Hk, Dh, page = c["kv"], c["dim"], c["page"]
    token = 2 * Hk * (Dh + 4)   # a token's codes and scales
    if c["op"] == "put8":
        T, H = c["T"], c["heads"]
        back = (-(-T // page) + 3 if T > 64 else T + 3) * page
        return {"bytes": T * (2 * H * Dh * e + 2 * Hk * Dh * e + token + 8) + 8 * Dh + 2 * c["rot"]
                + back * (token + 2 * Hk * Dh * e),
                "flops": T * ((H + Hk) * (4 * Dh + 3 * c["rot"]) + 4 * Hk * Dh) + back * 2 * Hk * Dh}
    if c["op"] == "rows8":
        n = c["longest"] + (c["seqs"] - 1) * (c["longest"] * 2 // 3 + 1)
        return {"bytes": n * (token + 2 * Hk * Dh * e), "flops": n * 2 * Hk * Dh}
    H = c["heads"]
    if "cache" in c and c["cache"] == "rows":
        token = 2 * Hk * Dh * e
    if c["op"] == "paged8":
        # lengths are spread evenly from a third of the longest to all of it
        B, L = c["seqs"], c["longest"]
        lens = [L] + [L * 2 // 3 + 1] * (B - 1)
        keys = sum(min(x, c["window"]) + min(max(x - c["window"], 0), c["sinks"]) for x in lens)
        return {"bytes": keys * token + 2 * B * H * Dh * e, "flops": 4 * keys * H * Dh}
    # prefixes from two thirds of the longest to all of it, what is behind them from a third
    ng, B = c["groups"], c["groups"] * c["per"]
    P, O = [c["prefix"]] + [c["prefix"] * 5 // 6 + 1] * (ng - 1), c["own"] * 2 // 3 + 1
    of_prefix = [max(min(p, c["window"] - O), 0) for p in P]
    of_prefix = [n + min(c["sinks"], p - n) for n, p in zip(of_prefix, P)]
    own_keys = B * min(O, c["window"])
    return {"bytes": (sum(of_prefix) + own_keys) * token + 2 * B * H * Dh * e,
            "flops": 4 * (sum(of_prefix) * c["per"] + own_keys) * H * Dh}


# ── the same in 64 bits, from the definitions ───────────────────────────────────────────────────────────────────

def _exact_kept(i, x, page, off):
    """Codes times scales (or the rows kept) of tokens at pages and places [n]: [n][Hk][Dh] in 64 bits."""
    v = i[x + "c"][page, :, off].double()
    return v * i[x + "s"][page, :, off].double().unsqueeze(-1) if x + "s" in i else v


def _exact_attend(q, k, v):
    """q [H][Dh]; k and v [n][Hk][Dh]: query head h reads key head h // (H / Hk)."""
    H, Dh = q.shape
    k, v = (t.permute(1, 0, 2).contiguous() for t in (k, v))
    s = torch.matmul(q.view(k.shape[0], -1, Dh), k.transpose(1, 2).contiguous()) / math.sqrt(Dh)
    return torch.matmul(torch.softmax(s, 2), v).reshape(-1)


def exact(case, seed):
    c, i = case, _inputs(case, seed)
    if c["op"] == "adapters":
        y = i["z"].double()
        for a in range(c["count"]):
            rows = (i["index"] == a).nonzero().flatten()
            if rows.numel():
                h = i["x"][rows].double() @ i["a"][a].double().t()
                y[rows] += i["scale"][a].double() * (h @ i["b"][a].double().t())
        return y
    Hk, Dh, page = c["kv"], c["dim"], c["page"]
    if c["op"] in ("put8", "rows8"):
        starts = i["starts"].tolist()
        back = {}
        for x in "kv":
            parts = []
            for s in range(len(starts) - 1):
                t = torch.arange(starts[s + 1] - starts[s], device="cuda")
                parts.append((i["table"][s].long()[t // page], t % page))
            at, off = (torch.cat(p) for p in zip(*parts))
            back[x] = _exact_kept(i, x, at, off)
        if c["op"] == "rows8":
            return tuple(back[x].reshape(starts[-1], -1) for x in "kv")
        T, R, H = c["T"], c["rot"], c["heads"]
        heads = i["qkv"].double().view(T, H + 2 * Hk, Dh).clone()
        norm = heads[:, :H + Hk] * torch.rsqrt(heads[:, :H + Hk].pow(2).sum(2, keepdim=True) / Dh + 1e-6)
        norm[:, :H] *= i["gq"].double()
        norm[:, H:] *= i["gk"].double()
        turn = torch.polar(torch.ones(T, 1, R // 2, dtype=torch.float64, device="cuda"),
                           (i["pos"].double()[:, None] * i["freq"].double())[:, None])
        even = torch.arange(R // 2, device="cuda") * (2 if c["pairs"] == "next" else 1)
        odd = even + (1 if c["pairs"] == "next" else R // 2)
        z = torch.complex(norm[..., even], norm[..., odd]) * turn
        norm[..., even], norm[..., odd] = z.real, z.imag
        # where each slot comes among the rows read back
        place = torch.empty_like(i["table"][0].long())
        place[i["table"][0].long()] = torch.arange(place.numel(), device="cuda")
        row = place[i["slots"].long() // page] * page + i["slots"].long() % page
        for x, new in (("k", norm[:, H:]), ("v", heads[:, H + Hk:])):
            step = new.abs().amax(2, keepdim=True) / 127
            back[x][row] = torch.round(new / step) * step
        return (norm[:, :H].reshape(T, -1), *(back[x].reshape(starts[-1], -1) for x in "kv"))
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(i["lens"].tolist()):
        j = torch.arange(n, device="cuda")
        j = j[(j >= n - c["window"]) | (j < c["sinks"])]
        table = i["table"][b].long()
        at = table[j // page]
        if c["op"] == "shared":
            group = b // c["per"]
            at = torch.where(j < i["shared"][group], i["table"][group * c["per"]].long()[j // page], at)
        k, v = (_exact_kept(i, x, at, j % page) for x in "kv")
        out[b] = _exact_attend(i["q"][b].double().view(-1, Dh), k, v)
    return out
