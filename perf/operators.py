"""A decoder layer's attention step next to the encoder: what it costs, as cases that can be timed and compared.

Four operators are called the way such a program calls them:

  q4       p2h_q4_gemv: a linear with 4-bit weights and one scale (and zero point) per group of rows, on few rows
  rope     p2h_qk_norm_rope: RMS norm of every query and key head and the position rotation, in one pass over the
           fused q | k | v rows, with the keys and values put into a paged cache
  window   p2h_attention_window: attention of ragged sequences over a sliding window and a few first tokens
  paged    p2h_attention_paged: one new token per sequence over the paged cache

Widths are the encoder's (1024 channels, 8 heads of 128, feed-forward 4096; 375 frames a 30 s window, 438 the longest
one, 6000 sixteen of them) and generic decoder ones (32 query heads over 8 key heads, heads of 64).

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
        # one token through a square projection: launch and latency are all there is
        {"name": "q4_bf16_m1_1024", "op": "q4", "type": "bf16", "M": 1, "K": 1024, "N": 1024, "group": 128,
         "zeros": False},
        # one token's fp32 row (the framework's own activations) through the up-projection, fine groups, zero points
        {"name": "q4_f32_m1_up", "op": "q4", "type": "f32", "M": 1, "K": 1024, "N": 4096, "group": 32, "zeros": True},
        # thirteen sequences' tokens through a wide output layer of odd size: the largest weight
        {"name": "q4_f16_m13_odd", "op": "q4", "type": "f16", "M": 13, "K": 8192, "N": 16389, "group": 64,
         "zeros": True},
        # one new token of each of 16 sequences, its key and value appended to the cache
        {"name": "rope_bf16_t16_append", "op": "rope", "type": "bf16", "T": 16, "heads": 32, "kv": 8, "dim": 128,
         "rot": 128, "pairs": "half", "cache": True, "page": 16, "far": 131072},
        # one 30 s window's fp32 rows with half of each head rotated in neighbouring pairs, no cache
        {"name": "rope_f32_t375", "op": "rope", "type": "f32", "T": 375, "heads": 8, "kv": 8, "dim": 128, "rot": 64,
         "pairs": "next", "cache": False, "page": 16, "far": 375},
        # sixteen windows as one prompt, appended to the cache
        {"name": "rope_bf16_t6000_append", "op": "rope", "type": "bf16", "T": 6000, "heads": 32, "kv": 8, "dim": 128,
         "rot": 128, "pairs": "half", "cache": True, "page": 64, "far": 6000},
        # the longest window's fp32 rows with a limited context to both sides
        {"name": "window_f32_t438", "op": "window", "type": "f32", "lens": "438", "past": 0, "heads": 8, "kv": 8,
         "dim": 128, "window": 128, "ahead": 32, "sinks": 4},
        # sixteen windows as one long sequence, bounded context with a few first tokens kept
        {"name": "window_bf16_t6000", "op": "window", "type": "bf16", "lens": "6000", "past": 0, "heads": 32, "kv": 8,
         "dim": 128, "window": 1024, "ahead": 0, "sinks": 4},
        # a ragged batch of prompts behind kept keys, every earlier key visible, heads of 64
        {"name": "window_f16_ragged_causal", "op": "window", "type": "f16", "lens": "4001,1,0,1875,375,38", "past": 77,
         "heads": 32, "kv": 8, "dim": 64, "window": FAR, "ahead": 0, "sinks": 0},
        # one sequence's next token after a 30 s window: latency
        {"name": "paged_f32_b1_375", "op": "paged", "type": "f32", "seqs": 1, "longest": 375, "heads": 8, "kv": 8,
         "dim": 128, "page": 16, "window": FAR, "sinks": 0},
        # a served batch of ragged lengths
        {"name": "paged_bf16_b32_8192", "op": "paged", "type": "bf16", "seqs": 32, "longest": 8192, "heads": 32,
         "kv": 8, "dim": 128, "page": 64, "window": FAR, "sinks": 0},
        # two very long sequences: the cache is split over its length
        {"name": "paged_f16_b2_200001", "op": "paged", "type": "f16", "seqs": 2, "longest": 200001, "heads": 16,
         "kv": 4, "dim": 128, "page": 256, "window": 131072, "sinks": 5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, t = rng.choice(("q4", "rope", "window", "paged")), rng.choice(("f32", "f16", "bf16"))
    if op == "q4":
        return {"op": op, "type": t, "M": _log_int(rng, 1, 16), "K": _log_int(rng, 64, 8192),
                "N": _log_int(rng, 64, 16384), "group": rng.choice((32, 64, 128)), "zeros": rng.random() < 0.5}
    dim = rng.choice((64, 128))
    kv = rng.choice((1, 2, 4, 8))
    heads = kv * rng.choice((1, 2, 4) if kv == 8 else (1, 3, 4, 8))
    base = {"op": op, "type": t, "heads": heads, "kv": kv, "dim": dim}
    if op == "rope":
        return dict(base, T=_log_int(rng, 1, 6000), rot=rng.choice((dim, dim // 2)), pairs=rng.choice(("half", "next")),
                    cache=rng.random() < 0.6, page=rng.choice((16, 64, 256)), far=_log_int(rng, 8000, 1000000))
    window = FAR if rng.random() < 0.4 else _log_int(rng, 16, 4096)
    sinks = rng.choice((0, 0, 1, 4, 16))
    if op == "window":
        n = rng.choice((1, 1, 2, 3, 7))
        lens = [_log_int(rng, 1, (2000 if t == "f32" else 4000) // n) for _ in range(n)]
        return dict(base, lens=",".join(str(x) for x in lens), past=rng.choice((0, 0, 130)), window=window,
                    ahead=rng.choice((0, 0, 16, FAR)), sinks=sinks)
    seqs = _log_int(rng, 1, 64)
    longest = _log_int(rng, 1, 262144 // seqs)
    return dict(base, seqs=seqs, longest=longest, page=rng.choice((16, 32, 64, 256)), window=window, sinks=sinks)


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


def _group_starts(lens):
    return torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    """What a case's computation is a function of."""
    g, dt = _gen(seed), TYPES[case["type"]]
    if case["op"] == "q4":
        M, K, N, G = case["M"], case["K"], case["N"], case["group"]
        groups, half = -(-K // G), (N + 1) // 2
        # activations with one value in a thousand twenty times as large; weights of about 1/sqrt(K)
        x = torch.randn(M, K, generator=g, device="cuda")
        x = (x * torch.where(torch.rand(M, K, generator=g, device="cuda") < 0.001, 20.0, 1.0)).to(dt)
        scales = ((0.5 + torch.rand(groups, N, generator=g, device="cuda")) / (4.6 * math.sqrt(K))).half()
        return {"x": x, "codes": _whole(g, 0, 256, K, half).to(torch.uint8), "scales": scales,
                "zeros": _whole(g, 0, 256, groups, half).to(torch.uint8) if case["zeros"] else None}
    H, Hk, Dh = case["heads"], case["kv"], case["dim"]
    if case["op"] == "rope":
        T, page = case["T"], case["page"]
        i = {"qkv": _normal(g, T, (H + 2 * Hk) * Dh, dtype=dt, scale=2.0),
             "gq": 0.5 + torch.rand(Dh, generator=g, device="cuda"),
             "gk": 0.5 + torch.rand(Dh, generator=g, device="cuda"),
             "freq": torch.pow(10000.0, -torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
                               / case["rot"]).float(),
             # a prompt's consecutive positions, or (few tokens) each sequence's own
             "pos": (torch.arange(T, device="cuda", dtype=torch.int32) + case["far"] - T if T > 64
                     else _whole(g, 0, case["far"], T))}
        if case["cache"]:
            pages = -(-T // page) + 3 if T > 64 else T + 3
            order = torch.randperm(pages, generator=g, device="cuda")
            t = torch.arange(T, device="cuda")
            # a prompt fills page after page from the middle of one; single tokens land in pages of their own
            slots = order[(t + page // 2) // page] * page + (t + page // 2) % page if T > 64 else \
                order[t] * page + _whole(g, 0, page, T).long()
            i["slots"] = slots.to(torch.int32)
            i["kc"] = _normal(g, pages, Hk, page, Dh, dtype=dt)
            i["vc"] = _normal(g, pages, Hk, page, Dh, dtype=dt)
        return i
    if case["op"] == "window":
        lens = [int(x) for x in case["lens"].split(",")]
        kl = [n + case["past"] for n in lens]
        return {"q": _normal(g, sum(lens), H * Dh, dtype=dt), "k": _normal(g, sum(kl), Hk * Dh, dtype=dt),
                "v": _normal(g, sum(kl), Hk * Dh, dtype=dt), "qs": _group_starts(lens), "ks": _group_starts(kl)}
    B, page, longest = case["seqs"], case["page"], case["longest"]
    per = -(-longest // page)
    lens = _whole(g, 1 + longest // 3, longest + 1, B)
    lens[0] = longest
    return {"q": _normal(g, B, H * Dh, dtype=dt), "lens": lens,
            "table": torch.randperm(B * per, generator=g, device="cuda").view(B, per).to(torch.int32),
            "kc": _normal(g, B * per, Hk, page, Dh, dtype=dt), "vc": _normal(g, B * per, Hk, page, Dh, dtype=dt)}


# ── what a program holds ────────────────────────────────────────────────────────────────────────────────────────

_kept = {}


def _binding():
    """The framework's binding and the stream this program works on."""
    if not _kept:
        sys.path.insert(0, os.path.join(ROOT, "phonon-2-c_amd"))
        import p2gemm
        p2gemm.init()
        _kept.update(P=p2gemm, stream=p2gemm.Stream())
    return _kept["P"], _kept["stream"]


def prepare(case, seed):
    st = dict(_inputs(case, seed), case=dict(case))
    torch.cuda.synchronize()   # the framework works on streams of its own
    if not own:
        return st
    P, stream = _binding()
    c, dt = case, TYPES[case["type"]]
    st["P"], st["stream"] = P, stream.ptr
    if c["op"] == "q4":
        st["w"] = P.Q4Weight.wrap(st["codes"].data_ptr(), st["scales"].data_ptr(),
                                  st["zeros"].data_ptr() if c["zeros"] else None, c["K"], c["N"], c["group"])
        st["y"] = torch.empty(c["M"], c["N"], device="cuda", dtype=dt)
    elif c["op"] == "rope":
        st["oq"] = torch.empty(c["T"], c["heads"] * c["dim"], device="cuda", dtype=dt)
        st["ok"] = torch.empty(c["T"], c["kv"] * c["dim"], device="cuda", dtype=dt) if not c["cache"] else None
    else:
        st["o"] = torch.empty_like(st["q"])
    if "kc" in st:
        st["cache"] = P.KvCache(c["type"], c["kv"], c["dim"], c["page"], st["kc"].shape[0], st["kc"].data_ptr(),
                                st["vc"].data_ptr())
    if c["op"] == "paged":
        st["ws"] = P.Workspace(P.attention_paged_workspace_bytes(st["cache"], c["seqs"], c["heads"], c["longest"],
                                                                 c["window"], c["sinks"]))
    return st


def run(st):
    return _run_own(st) if own else _PLAIN[st["case"]["op"]](st)


def _run_own(st):
    c, P, s = st["case"], st["P"], st["stream"]
    if c["op"] == "q4":
        P.q4_gemv_dev(c["type"], c["M"], c["N"], c["K"], 1.0, st["x"].data_ptr(), c["K"], st["w"], 0.0,
                      st["y"].data_ptr(), c["N"], s)
        return st["y"]
    H, Hk, Dh = c["heads"], c["kv"], c["dim"]
    if c["op"] == "rope":
        P.qk_norm_rope_dev(c["type"], c["T"], H, Hk, Dh, st["qkv"].data_ptr(), (H + 2 * Hk) * Dh, st["gq"].data_ptr(),
                           st["gk"].data_ptr(), 1e-6, c["rot"], c["pairs"] == "next", st["freq"].data_ptr(),
                           st["pos"].data_ptr(), st["oq"].data_ptr(), H * Dh,
                           st["ok"].data_ptr() if st["ok"] is not None else None, Hk * Dh, st.get("cache"),
                           st["slots"].data_ptr() if c["cache"] else None, s)
        return (st["oq"], st["kc"], st["vc"]) if c["cache"] else (st["oq"], st["ok"])
    if c["op"] == "window":
        P.attention_window_dev(c["type"], st["q"].shape[0], st["k"].shape[0], st["qs"].numel() - 1,
                               st["qs"].data_ptr(), st["ks"].data_ptr(), H, Hk, Dh, st["q"].data_ptr(), H * Dh,
                               st["k"].data_ptr(), Hk * Dh, st["v"].data_ptr(), Hk * Dh, Dh ** -0.5, c["window"],
                               c["ahead"], c["sinks"], st["o"].data_ptr(), H * Dh, s)
    else:
        P.attention_paged_dev(st["cache"], c["seqs"], H, st["q"].data_ptr(), H * Dh, st["table"].data_ptr(),
                              st["table"].shape[1], st["lens"].data_ptr(), c["longest"], Dh ** -0.5, c["window"],
                              c["sinks"], st["o"].data_ptr(), H * Dh, st["ws"].ptr, st["ws"].nbytes, s)
    return st["o"]


# ── the plain forms ─────────────────────────────────────────────────────────────────────────────────────────────

def _nibbles(packed, n):
    """[rows][ceil(n/2)] bytes → [rows][n] codes, the even column in the low half."""
    return torch.stack((packed & 15, packed >> 4), 2).view(packed.shape[0], -1)[:, :n]


def _plain_q4(st):
    c = st["case"]
    code = _nibbles(st["codes"], c["N"]).float()
    zero = _nibbles(st["zeros"], c["N"]).float() if c["zeros"] else torch.full_like(st["scales"], 8.0).float()
    group = torch.arange(c["K"], device=code.device) // c["group"]
    w = (code - zero[group]) * st["scales"].float()[group]
    return (st["x"].float() @ w).to(st["x"].dtype)


def _plain_rope(st):
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
    y = torch.cat((turned, y[..., R:]), 2).to(st["qkv"].dtype)
    q, k = y[:, :H].reshape(T, H * Dh), y[:, H:]
    if not c["cache"]:
        return q, k.reshape(T, Hk * Dh)
    at, off = st["slots"].long() // c["page"], st["slots"].long() % c["page"]
    st["kc"][at, :, off] = k
    st["vc"][at, :, off] = v.to(k.dtype)
    return q, st["kc"], st["vc"]


def _attend(q, k, v, seen, scale):
    """q [.., H, n, Dh], k and v [.., H, m, Dh], seen [.., n, m] → softmax over the seen keys; zero where none is."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = torch.where(seen.unsqueeze(-3), s, torch.full_like(s[..., :1, :1], -math.inf))
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(s - top)
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-37)


def _plain_window(st):
    c = st["case"]
    H, Hk, Dh = c["heads"], c["kv"], c["dim"]
    n, m, dev = st["q"].shape[0], st["k"].shape[0], st["q"].device
    i, j = torch.arange(n, device=dev), torch.arange(m, device=dev)
    # the sequence of each row, each key's place in its sequence, and each query's place among its keys
    si = torch.searchsorted(st["qs"].long(), i, right=True) - 1
    sj = torch.searchsorted(st["ks"].long(), j, right=True) - 1
    at = j - st["ks"].long()[sj]
    p = i - st["qs"].long()[si + 1] + (st["ks"].long()[si + 1] - st["ks"].long()[si])
    back = p[:, None] - at[None, :]
    seen = (si[:, None] == sj[None, :]) & (back >= -c["ahead"]) & ((back < c["window"]) | (at < c["sinks"])[None, :])
    q = st["q"].float().view(n, H, Dh).transpose(0, 1)
    k, v = (st[t].float().view(m, Hk, Dh).transpose(0, 1).repeat_interleave(H // Hk, 0) for t in "kv")
    o = _attend(q, k, v, seen, Dh ** -0.5)
    return o.transpose(0, 1).reshape(n, H * Dh).to(st["q"].dtype)


def _plain_paged(st):
    c = st["case"]
    B, H, Hk, Dh = c["seqs"], c["heads"], c["kv"], c["dim"]
    # the pages in order: [B][pages][Hk][page][Dh] → [B][Hk][keys][Dh]
    k, v = (st[t][st["table"].long()].float().transpose(1, 2).reshape(B, Hk, -1, Dh) for t in ("kc", "vc"))
    at = torch.arange(k.shape[2], device=k.device)
    last = st["lens"].long()[:, None] - 1
    seen = (at <= last) & ((last - at < c["window"]) | (at < c["sinks"]))
    o = _attend(st["q"].float().view(B, Hk, H // Hk, Dh), k, v, seen[:, None, :], Dh ** -0.5)
    return o.reshape(B, H * Dh).to(st["q"].dtype)


_PLAIN = {"q4": _plain_q4, "rope": _plain_rope, "window": _plain_window, "paged": _plain_paged}


# ── what a pass cannot do without ───────────────────────────────────────────────────────────────────────────────

def _pairs(n, past, window, ahead, sinks):
    """Visible (query, key) pairs of one sequence of n queries over n + past keys."""
    p = torch.arange(n, dtype=torch.float64) + past
    m = n + past
    hi = torch.clamp(p + ahead + 1, max=m)                  # keys up to here
    lo = torch.clamp(p - window + 1, min=0)                 # the window's first key
    return int((torch.clamp(hi - lo, min=0) + torch.clamp(torch.minimum(lo, hi), max=sinks)).sum())


def work(case):
    c = case
    e = 4 if c["type"] == "f32" else 2
    if c["op"] == "q4":
        M, K, N = c["M"], c["K"], c["N"]
        groups, half = -(-K // c["group"]), (N + 1) // 2
        return {"bytes": K * half + 2 * groups * N + groups * half * c["zeros"] + e * M * (K + N), "flops": 2 * M * N * K}
    H, Hk, Dh = c["heads"], c["kv"], c["dim"]
    if c["op"] == "rope":
        T = c["T"]
        moved = 2 * (H + Hk + (Hk if c["cache"] else 0)) * Dh * e
        return {"bytes": T * (moved + 8) + 8 * Dh + 2 * c["rot"], "flops": T * (H + Hk) * (4 * Dh + 3 * c["rot"])}
    if c["op"] == "window":
        lens = [int(x) for x in c["lens"].split(",")]
        n, m = sum(lens), sum(lens) + c["past"] * len(lens)
        pairs = sum(_pairs(x, c["past"], c["window"], c["ahead"], c["sinks"]) for x in lens)
        return {"bytes": e * Dh * (2 * n * H + 2 * m * Hk), "flops": 4 * pairs * H * Dh}
    # lengths are spread evenly from a third of the longest to all of it
    B, L = c["seqs"], c["longest"]
    lens = [L] + [L * 2 // 3 + 1] * (B - 1)
    keys = sum(min(x, c["window"]) + min(max(x - c["window"], 0), c["sinks"]) for x in lens)
    return {"bytes": 2 * keys * Hk * Dh * e + 2 * B * H * Dh * e, "flops": 4 * keys * H * Dh}


# ── the same in 64 bits, from the definitions ───────────────────────────────────────────────────────────────────

def _exact_heads(q, k, v, seen, scale):
    """q [H][n][Dh], k and v [Hk][m][Dh] in 64 bits: query head h reads key head h // (H / Hk)."""
    Hk, n = k.shape[0], q.shape[1]
    s = torch.matmul(q.view(Hk, -1, q.shape[2]), k.transpose(1, 2).contiguous()).view(Hk, -1, n, k.shape[1]) * scale
    w = torch.softmax(s.masked_fill_(~seen, -math.inf), 3)
    w = torch.where(seen.any(1, keepdim=True), w, torch.zeros_like(w))
    return torch.matmul(w.view(Hk, -1, k.shape[1]), v).view(q.shape)


def exact(case, seed):
    c, i = case, _inputs(case, seed)
    if c["op"] == "q4":
        N = c["N"]
        cols = torch.arange(N, device="cuda")
        pick = lambda packed: (packed[:, cols // 2].int() >> (4 * (cols % 2))) & 15   # noqa: E731
        zero = pick(i["zeros"]).double() if c["zeros"] else torch.tensor(8.0, dtype=torch.float64, device="cuda")
        code = torch.nn.functional.pad(pick(i["codes"]).double(), (0, 0, 0, -c["K"] % c["group"]))
        w = (code.view(-1, c["group"], N) - (zero[:, None] if c["zeros"] else zero)) * i["scales"].double()[:, None]
        return i["x"].double() @ w.reshape(-1, N)[:c["K"]]
    H, Hk, Dh = c["heads"], c["kv"], c["dim"]
    if c["op"] == "rope":
        T, R = c["T"], c["rot"]
        rows = i["qkv"].double()
        heads = rows[:, :(H + Hk) * Dh].reshape(T, H + Hk, Dh)
        heads = heads * torch.rsqrt(heads.pow(2).sum(2, keepdim=True) / Dh + 1e-6)
        heads[:, :H] *= i["gq"].double()
        heads[:, H:] *= i["gk"].double()
        turn = torch.polar(torch.ones(T, 1, R // 2, dtype=torch.float64, device="cuda"),
                           (i["pos"].double()[:, None] * i["freq"].double())[:, None])
        even = torch.arange(R // 2, device="cuda") * (2 if c["pairs"] == "next" else 1)
        odd = even + (1 if c["pairs"] == "next" else R // 2)
        z = torch.complex(heads[..., even], heads[..., odd]) * turn
        heads[..., even], heads[..., odd] = z.real, z.imag
        q, k = heads[:, :H].reshape(T, -1), heads[:, H:]
        if not c["cache"]:
            return q, k.reshape(T, -1)
        kc, vc = i["kc"].double(), i["vc"].double()
        at, off = i["slots"].long() // c["page"], i["slots"].long() % c["page"]
        kc[at, :, off] = k
        vc[at, :, off] = rows[:, (H + Hk) * Dh:].reshape(T, Hk, Dh)
        return q, kc, vc
    if c["op"] == "window":
        out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
        qs, ks = i["qs"].tolist(), i["ks"].tolist()
        for s in range(len(qs) - 1):
            n, m = qs[s + 1] - qs[s], ks[s + 1] - ks[s]
            if n == 0:
                continue
            d = torch.arange(n, device="cuda")[:, None] + (m - n) - torch.arange(m, device="cuda")[None, :]
            seen = (d >= -c["ahead"]) & ((d < c["window"]) | (torch.arange(m, device="cuda") < c["sinks"]))
            q, k, v = (i[t][a:b].double().view(b - a, -1, Dh).transpose(0, 1).contiguous()
                       for t, a, b in (("q", qs[s], qs[s + 1]), ("k", ks[s], ks[s + 1]), ("v", ks[s], ks[s + 1])))
            out[qs[s]:qs[s + 1]] = _exact_heads(q, k, v, seen, 1.0 / math.sqrt(Dh)).transpose(0, 1).reshape(n, -1)
        return out
    out = torch.zeros(i["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(i["lens"].tolist()):
        j = torch.arange(n, device="cuda")
        j = j[(j >= n - c["window"]) | (j < c["sinks"])]
        page = i["table"][b].long()[j // c["page"]]
        k, v = (i[t][page, :, j % c["page"]].double().transpose(0, 1).contiguous() for t in ("kc", "vc"))
        q = i["q"][b].double().view(H, 1, Dh)
        out[b] = _exact_heads(q, k, v, torch.ones(1, j.numel(), dtype=torch.bool, device="cuda"),
                              1.0 / math.sqrt(Dh)).reshape(-1)
    return out
