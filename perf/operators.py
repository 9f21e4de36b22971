"""The serving operators' cases: what one pass of each reads, its plain form, and its definition in 64 bits.

Four operators of one decode or prefill step over a paged key/value cache:

  qk_norm_rope   RMS norm of every query and key head, then the rotation of its position
  append         rotate (and optionally norm) new keys, store keys and values in their cache slots
  attention      attention of a batch whose sequences share a prefix, held in the cache once
  sample         one token per row of logits: temperature, top-k, top-p, min-p, a given random number

`run` computes them in elementary torch operations; with `own` set it calls the library.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f16": torch.float16, "f32": torch.float32}
_SIZE = {"f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------- cases
def _rope_case(name, tokens, hq, hkv, d, rot, dtype, interleaved, far=0):
    """far: the first token's position (the cached length of a decode step, 0 for a prompt)."""
    return {"name": name, "op": "qk_norm_rope", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "rot": rot,
            "dtype": dtype, "interleaved": interleaved, "far": far}


def _append_case(name, tokens, hkv, d, rot, page, dtype, interleaved, norm, pad, far=0):
    """pad: tokens of a padded batch that have no slot (their slot is -1)."""
    return {"name": name, "op": "append", "tokens": tokens, "hkv": hkv, "d": d, "rot": rot, "page": page, "dtype": dtype,
            "interleaved": interleaved, "norm": norm, "pad": pad, "far": far}


def _attn_case(name, batch, queries, hq, hkv, d, prefix, longest, page):
    """queries: new tokens of a sequence, 1 in a decode step (else lengths from half of it to all of it);
    longest: the longest own length of a sequence, its new tokens among them (ragged below that)."""
    return {"name": name, "op": "attention", "batch": batch, "queries": queries, "hq": hq, "hkv": hkv, "d": d,
            "prefix": prefix, "longest": longest, "page": page}


def _sample_case(name, rows, vocab, dtype, mode):
    """mode: which filters the rows use ("greedy", "top_k", "top_p", "mixed": each row its own)."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode}


def listed():
    return [
        # one new token of one conversation, 16 query heads of 128 as in the benchmark's decoder block: latency
        _rope_case("norm_rope_1", 1, 16, 4, 128, 128, "f16", True, far=70001),
        # a prompt batch of the benchmark's decoder block (8 x 1024 tokens), grouped key heads
        _rope_case("norm_rope_8192", 8192, 16, 4, 128, 128, "f16", False),
        # an odd prompt length in fp32, half of each head rotated
        _rope_case("norm_rope_4097_f32", 4097, 32, 8, 64, 32, "f32", True, far=130000),
        # a decode step of 64 sequences writes one slot each
        _append_case("append_64", 64, 8, 128, 128, 16, "f16", False, False, 0, far=9000),
        # a prompt of 16381 tokens with 19 tokens of padding behind it
        _append_case("append_16400", 16400, 8, 128, 128, 16, "f16", True, True, 19),
        # two answers sampled for one short prompt: latency
        _attn_case("attn_b2", 2, 1, 16, 4, 128, 500, 40, 16),
        # the common decode step: 64 sequences behind one long system prompt
        _attn_case("attn_b64_p8192", 64, 1, 32, 8, 128, 8192, 1023, 16),
        # GPT-2 head layout (12 heads of 64, no grouping), a short prefix with an odd length
        _attn_case("attn_b32_d64", 32, 1, 12, 12, 64, 333, 690, 16),
        # chunks of prompts that follow the shared prefix: many queries a sequence, causal among themselves
        _attn_case("attn_chunks", 8, 251, 32, 8, 128, 4096, 509, 64),
        # the largest decode step: 128 sequences, a prefix of 16385 tokens
        _attn_case("attn_b128_p16385", 128, 1, 32, 4, 128, 16385, 2047, 32),
        # one row of GPT-2 logits: latency
        _sample_case("sample_1", 1, 50257, "f32", "top_p"),
        # a serving batch, every row with its own parameters
        _sample_case("sample_256", 256, 128000, "f16", "mixed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "append", "attention", "attention", "sample"])
    cap = {"qk_norm_rope": "norm_rope_8192", "append": "append_16400", "attention": "attn_b128_p16385",
           "sample": "sample_256"}[op]
    largest = {c["name"]: work(c) for c in listed()}
    while True:
        if op == "qk_norm_rope":
            d = rng.choice([64, 96, 128, 256])
            hkv = rng.choice([1, 2, 4, 8])
            case = _rope_case("", _log_int(rng, 1, 16384), hkv * rng.choice([1, 2, 3, 4, 8]), hkv, d,
                              rng.choice([d, d, d // 2]), rng.choice(["f16", "f16", "f32"]), rng.random() < 0.5,
                              rng.choice([0, 5000, 131072]))
        elif op == "append":
            d = rng.choice([64, 96, 128, 256])
            tokens = _log_int(rng, 1, 16384)
            case = _append_case("", tokens, rng.choice([1, 2, 4, 8, 12]), d, rng.choice([0, d, d, d // 2]),
                                rng.choice([1, 16, 24, 32, 64, 128]), rng.choice(["f16", "f16", "f32"]),
                                rng.random() < 0.5, rng.random() < 0.5, rng.choice([0, tokens // 9]),
                                rng.choice([0, 5000, 131072]))
        elif op == "attention":
            hkv = rng.choice([1, 2, 4, 8])
            queries = rng.choice([1, 1, 1, _log_int(rng, 2, 300)])
            case = _attn_case("", _log_int(rng, 1, 128), queries, hkv * rng.choice([1, 2, 3, 4, 6, 8]), hkv,
                              rng.choice([64, 128]), rng.choice([0, _log_int(rng, 1, 20000), _log_int(rng, 100, 20000)]),
                              queries + _log_int(rng, 1, 3000), rng.choice([16, 16, 32, 64, 24]))
        else:
            case = _sample_case("", _log_int(rng, 1, 256), _log_int(rng, 1000, 150000), rng.choice(["f16", "f32"]),
                                rng.choice(["greedy", "top_k", "top_p", "mixed"]))
        w, top = work(case), largest[cap]
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            case.pop("name")
            return case


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Query counts and own lengths of the sequences (host integers, fixed by the case)."""
    r = np.random.default_rng(case["batch"] * 7919 + case["longest"])
    b, nq, top = case["batch"], case["queries"], case["longest"]
    counts = [nq] * b if nq == 1 else [int(x) for x in r.integers(max(1, nq // 2), nq + 1, b)]
    counts[0] = nq
    lens = [int(x) for x in r.integers(max(1, top // 4), top + 1, b)]
    lens[b // 2] = top
    return counts, [max(n, c) for n, c in zip(lens, counts)]


def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def _heads(g, tokens, heads, d, dtype):
    return torch.randn(tokens, heads, d, generator=g, device="cuda").to(dtype)


def _positions(case):
    """Positions of the tokens: a prompt counts up; tokens of a decode batch sit near their cached lengths."""
    t, far = case["tokens"], case["far"]
    p = torch.arange(t, device="cuda", dtype=torch.int64)
    return p + far if t > 512 or t == 1 else (p * 37) % 911 + far


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case)
    if op == "qk_norm_rope":
        dt = _DT[case["dtype"]]
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        qkv = _heads(g, t, hq + 2 * hkv, d, dt)            # the fused projection's rows: q | k | v
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        s["wq"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
        s["wk"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
        s["pos"] = _positions(case)
        s["q_out"] = torch.empty(t, hq, d, dtype=dt, device="cuda")
        s["k_out"] = torch.empty(t, hkv, d, dtype=dt, device="cuda")
    elif op == "append":
        dt = _DT[case["dtype"]]
        t, hkv, d, page = case["tokens"], case["hkv"], case["d"], case["page"]
        qkv = _heads(g, t, 3 * hkv, d, dt)
        s["k"], s["v"] = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:]
        s["wk"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if case["norm"] else None
        s["pos"] = _positions(case) if case["rot"] else None
        pages = -(-t // page) + 3
        s["k_cache"] = torch.zeros(pages, page, hkv, d, dtype=dt, device="cuda")
        s["v_cache"] = torch.zeros(pages, page, hkv, d, dtype=dt, device="cuda")
        if t > 512:   # a prompt fills whole pages that lie anywhere in the pool
            order = torch.randperm(pages, generator=g, device="cuda")
            at = torch.arange(t, device="cuda")
            slots = order[at // page] * page + at % page
        else:         # a decode step: one slot anywhere for each sequence
            slots = torch.randperm(pages * page, generator=g, device="cuda")[:t].clone()
        if case["pad"]:
            slots[t - case["pad"]:] = -1
        s["slots"] = slots.to(torch.int64)
    elif op == "attention":
        counts, lens = _lengths(case)
        hq, hkv, d, page, prefix = case["hq"], case["hkv"], case["d"], case["page"], case["prefix"]
        npre = -(-prefix // page)
        width = max(-(-n // page) for n in lens)
        used = npre + sum(-(-n // page) for n in lens)
        pages = used + 5
        order = torch.randperm(pages, generator=_gen(seed + 1, "cpu"))
        table = torch.zeros(len(lens), width, dtype=torch.int32)
        at = npre
        for b, n in enumerate(lens):
            c = -(-n // page)
            table[b, :c] = order[at:at + c]
            at += c
        s["q"] = _heads(g, sum(counts), hq, d, torch.float16)
        s["k_cache"] = torch.randn(pages, page, hkv, d, generator=g, device="cuda", dtype=torch.float16)
        s["v_cache"] = torch.randn(pages, page, hkv, d, generator=g, device="cuda", dtype=torch.float16)
        s["prefix_pages"] = order[:npre].to(torch.int32).cuda()
        s["table"] = table.cuda()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["offsets"] = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
        s["max_q"], s["max_len"] = max(counts), max(lens)
        s["out"] = torch.empty_like(s["q"])
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=g, device="cuda") * 2.0
        x += torch.rand(rows, vocab, generator=g, device="cuda").pow_(400) * 9.0     # the few likely tokens of a row
        s["logits"] = x.to(_DT[case["dtype"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        r = np.random.default_rng(seed)
        mode = case["mode"]
        if mode == "greedy":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.0, 0, 1.0, 0.0
        elif mode == "top_k":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.8, 50, 1.0, 0.0
        elif mode == "top_p":
            s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.9, 0, 0.95, 0.0
        else:
            f = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda")
            s["temperature"] = f(r.choice([0.0, 0.6, 0.8, 1.0, 1.3], rows), torch.float32)
            s["top_k"] = f(r.choice([0, 0, 1, 20, 50, 1000, 40000], rows), torch.int32)
            s["top_p"] = f(r.choice([1.0, 0.5, 0.9, 0.95, 0.99], rows), torch.float32)
            s["min_p"] = f(r.choice([0.0, 0.0, 0.02, 0.1], rows), torch.float32)
        s["out"] = torch.empty(rows, dtype=torch.int64, device="cuda")
    return s


# -------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "qk_norm_rope":
        n = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * n * _SIZE[case["dtype"]] + 8 * case["tokens"] + 2 * case["d"] * _SIZE[case["dtype"]],
                "flops": 7 * n}
    if op == "append":
        n = (case["tokens"] - case["pad"]) * case["hkv"] * case["d"]
        return {"bytes": 4 * n * _SIZE[case["dtype"]] + 16 * case["tokens"],
                "flops": (3 * n if case["rot"] else 0) + (4 * n if case["norm"] else 0)}
    if op == "attention":
        counts, lens = _lengths(case)
        hq, hkv, d, prefix = case["hq"], case["hkv"], case["d"], case["prefix"]
        keys = sum(c * prefix + c * n - c * (c - 1) // 2 for c, n in zip(counts, lens))     # visible (query, key) pairs
        return {"bytes": 2 * 2 * sum(counts) * hq * d + 2 * 2 * (prefix + sum(lens)) * hkv * d,
                "flops": 4 * keys * hq * d}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _SIZE[case["dtype"]] + 12 * case["rows"], "flops": 3 * n}


# --------------------------------------------------------------------------------------- plain forms
def _plain_rotate(x, pos, rot, interleaved, theta=10000.0):
    """x: float32 [T, H, D]; angles in 64 bits: a far position times a frequency loses the angle in 32."""
    half = rot // 2
    freq = torch.pow(torch.tensor(theta, dtype=torch.float64, device=x.device),
                     -torch.arange(half, dtype=torch.float64, device=x.device) * 2 / rot)
    ang = pos.to(torch.float64)[:, None] * freq[None, :]
    cs, sn = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cs - b * sn, a * sn + b * cs
    else:
        a, b = x[..., :half], x[..., half:rot]
        out[..., :half], out[..., half:rot] = a * cs - b * sn, a * sn + b * cs
    return out


def _plain_norm(x, w, eps=1e-6):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()


def _plain_attention(s):
    hq, hkv, d, page, prefix = s["hq"], s["hkv"], s["d"], s["page"], s["prefix"]
    grp, b = hq // hkv, s["batch"]
    off, lens = s["offsets"].long(), s["lens"].long()
    nq = off[1:] - off[:-1]
    mq, ml = s["max_q"], s["max_len"]
    at = torch.arange(mq, device="cuda")
    real = at[None, :] < nq[:, None]                                            # [B, mq]
    idx = (off[:-1, None] + at[None, :]).clamp_(max=s["q"].shape[0] - 1)
    q = s["q"][idx].float().view(b, mq, hkv, grp, d).permute(0, 2, 3, 1, 4)     # [B, Hkv, G, mq, D]
    q = q.reshape(b, hkv, grp * mq, d) * (1.0 / math.sqrt(d))
    key = torch.arange(ml, device="cuda")
    rows = s["table"].long()[:, key // page] * page + key % page                # [B, ml] slots
    ks = s["k_cache"].view(-1, hkv, d)[rows].float().permute(0, 2, 1, 3)        # [B, Hkv, ml, D]
    vs = s["v_cache"].view(-1, hkv, d)[rows].float().permute(0, 2, 1, 3)
    seen = key[None, None, :] <= (lens - nq)[:, None, None] + at[None, :, None]  # [B, mq, ml]
    sc = torch.matmul(q, ks.transpose(2, 3)).view(b, hkv, grp, mq, ml)
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    if prefix:
        kp = s["k_cache"][s["prefix_pages"].long()].reshape(-1, hkv, d)[:prefix].float().permute(1, 0, 2)
        vp = s["v_cache"][s["prefix_pages"].long()].reshape(-1, hkv, d)[:prefix].float().permute(1, 0, 2)
        flat = q.permute(1, 0, 2, 3).reshape(hkv, b * grp * mq, d)
        sp = torch.matmul(flat, kp.transpose(1, 2)).view(hkv, b, grp, mq, prefix).permute(1, 0, 2, 3, 4)
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
        ep = torch.exp(sp - top)
        acc = torch.matmul(ep.permute(1, 0, 2, 3, 4).reshape(hkv, b * grp * mq, prefix), vp)
        acc = acc.view(hkv, b, grp, mq, d).permute(1, 0, 2, 3, 4)
        total = ep.sum(-1, keepdim=True)
    else:
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        acc, total = 0.0, 0.0
    es = torch.exp(sc - top)
    acc = acc + torch.matmul(es.view(b, hkv, grp * mq, ml), vs).view(b, hkv, grp, mq, d)
    total = total + es.sum(-1, keepdim=True)
    o = torch.where(total > 0, acc / total, torch.zeros_like(acc)).to(torch.float16)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, mq, hq, d)
    return o[real]                                                              # [T, Hq, D]: the real rows, in order


def _plain_sample(s):
    x = s["logits"].double()
    rows, vocab = x.shape
    per_row = lambda v: (v.double() if torch.is_tensor(v) else torch.full((rows,), v, dtype=torch.float64, device="cuda"))[:, None]
    # the library takes its parameters in 32 bits
    f32 = lambda v: v.float() if torch.is_tensor(v) else float(np.float32(v))
    temp, top_k = per_row(f32(s["temperature"])), per_row(s["top_k"])
    top_p, min_p = per_row(f32(s["top_p"])), per_row(f32(s["min_p"]))
    v, order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(vocab, device="cuda")[None, :]
    z = (v - v[:, :1]) / torch.where(temp > 0, temp, torch.ones_like(temp))
    w = torch.exp(z)
    keep = (top_k <= 0) | (rank < top_k)
    w = w * keep
    cum = torch.cumsum(w, -1)
    nucleus = (top_p >= 1) | (cum - w < top_p * cum[:, -1:]) | (rank == 0)
    keep = keep & nucleus & (w >= min_p)
    keep = torch.where(temp > 0, keep, rank == 0)
    back = torch.zeros_like(w).scatter_(1, order, w * keep)
    cum = torch.cumsum(back, -1)
    target = s["u"].double()[:, None] * cum[:, -1:]
    return (cum <= target).sum(-1).clamp_(max=vocab - 1)


def run(state):
    s = state
    op = s["op"]
    if own:
        import hexb200

        ops = hexb200.ops
        if op == "qk_norm_rope":
            ops.qk_norm_rope(s["q"], s["k"], s["q_out"], s["k_out"], s["pos"], s["wq"], s["wk"], rotary_dim=s["rot"],
                             interleaved=s["interleaved"])
            return s["q_out"], s["k_out"]
        if op == "append":
            ops.kv_cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], positions=s["pos"],
                                k_weight=s["wk"], rotary_dim=s["rot"] or None, interleaved=s["interleaved"])
            return s["k_cache"], s["v_cache"]
        if op == "attention":
            ops.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["out"], s["prefix_pages"], s["prefix"],
                                        s["table"], s["lens"], q_offsets=s["offsets"], max_q=s["max_q"])
            return s["out"]
        ops.sample_tokens(s["logits"], s["u"], s["out"], temperature=s["temperature"], top_k=s["top_k"],
                          top_p=s["top_p"], min_p=s["min_p"])
        return s["out"]
    if op == "qk_norm_rope":
        dt = s["q"].dtype
        return tuple(_plain_rotate(_plain_norm(x.float(), w), s["pos"], s["rot"], s["interleaved"]).to(dt)
                     for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])))
    if op == "append":
        dt = s["k"].dtype
        k = s["k"].float()
        if s["wk"] is not None:
            k = _plain_norm(k, s["wk"])
        if s["pos"] is not None:
            k = _plain_rotate(k, s["pos"], s["rot"], s["interleaved"])
        n = s["tokens"] - s["pad"]                         # the padding sits behind the real tokens
        hkv, d = s["hkv"], s["d"]
        s["k_cache"].view(-1, hkv, d)[s["slots"][:n]] = k[:n].to(dt)
        s["v_cache"].view(-1, hkv, d)[s["slots"][:n]] = s["v"][:n]
        return s["k_cache"], s["v_cache"]
    if op == "attention":
        return _plain_attention(s)
    return _plain_sample(s)


# ---------------------------------------------------------------------------- the definition in 64 bits
def _exact_head(x, w, pos, rot, interleaved):
    """x [T, H, D] in 64 bits; the rotation as a complex product."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
    if pos is None:
        return x
    i = torch.arange(rot // 2, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None, None] * torch.exp(-(2 * i / rot) * math.log(10000.0))
    turn = torch.polar(torch.ones_like(ang), ang)
    head, tail = x[..., :rot], x[..., rot:]
    if interleaved:
        pair = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous())
        head = torch.view_as_real(pair * turn).flatten(-2)
    else:
        pair = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous()) * turn
        head = torch.cat([pair.real, pair.imag], -1)
    return torch.cat([head, tail], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "qk_norm_rope":
        return (_exact_head(s["q"], s["wq"], s["pos"], case["rot"], case["interleaved"]),
                _exact_head(s["k"], s["wk"], s["pos"], case["rot"], case["interleaved"]))
    if op == "append":
        k = _exact_head(s["k"], s["wk"], s["pos"], case["rot"], case["interleaved"])
        kc, vc = s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
        use = s["slots"] >= 0
        kc[s["slots"][use]] = k[use]
        vc[s["slots"][use]] = s["v"].double()[use]
        return kc.view(s["k_cache"].shape), vc.view(s["v_cache"].shape)
    if op == "attention":
        counts, lens = _lengths(case)
        hq, hkv, d, page, prefix = case["hq"], case["hkv"], case["d"], case["page"], case["prefix"]
        outs, t = [], 0
        grow = lambda cache, pages, n: cache[pages.long()].flatten(0, 1)[:n].double()
        pre_k, pre_v = grow(s["k_cache"], s["prefix_pages"], prefix), grow(s["v_cache"], s["prefix_pages"], prefix)
        for b, (c, n) in enumerate(zip(counts, lens)):
            pages = s["table"][b, :-(-n // page)]
            k = torch.cat([pre_k, grow(s["k_cache"], pages, n)]).transpose(0, 1)      # [Hkv, P + n, D]
            v = torch.cat([pre_v, grow(s["v_cache"], pages, n)]).transpose(0, 1)
            o = torch.empty(c, hq, d, dtype=torch.float64, device="cuda")
            hidden = torch.ones(c, n, dtype=torch.bool, device="cuda").triu(n - c + 1)
            hidden = torch.cat([torch.zeros(c, prefix, dtype=torch.bool, device="cuda"), hidden], 1)
            for h in range(hkv):
                for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    a = (s["q"][t:t + c, j].double() @ k[h].T) / math.sqrt(d)
                    o[:, j] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v[h]
            outs.append(o)
            t += c
        return torch.cat(outs)
    x = s["logits"].cpu().numpy().astype(np.float64)
    u = s["u"].cpu().numpy().astype(np.float64)
    host = lambda v, i: float(v[i]) if torch.is_tensor(v) else float(np.float32(v))
    picked = []
    for r in range(case["rows"]):
        temp, k, p, m = (host(s[n], r) for n in ("temperature", "top_k", "top_p", "min_p"))
        if temp <= 0:
            picked.append(int(np.argmax(x[r])))
            continue
        order = np.argsort(-x[r], kind="stable")
        if k >= 1:
            order = order[:int(k)]
        weight = np.exp((x[r][order] - x[r][order[0]]) / temp)
        if p < 1:
            before = np.concatenate([[0.0], np.cumsum(weight)[:-1]])
            order = order[:max(1, int(np.searchsorted(before, p * weight.sum(), side="left")))]
        chosen = np.sort(order)
        weight = np.exp((x[r][chosen] - x[r].max()) / temp)
        chosen, weight = chosen[weight >= m], weight[weight >= m]
        up = np.cumsum(weight)
        picked.append(int(chosen[min(len(chosen) - 1, int(np.searchsorted(up, u[r] * up[-1], side="right")))]))
    return torch.tensor(picked, dtype=torch.int64)
