"""GPU: the serving operators together, as a server runs them -- a prompt shared by all sequences goes into the paged cache once,
then every step embeds the last tokens, projects, norms and rotates, appends, attends, projects to the vocabulary and
samples, captured as one CUDA graph whose lengths, slots and positions advance on the device.

Each step's attention is compared with the formulas over the whole history in 64 bits, fed with the same fp16 weights and
rounded to fp16 where the step stores fp16 (projections, normed and rotated heads).  A value there may round to the
neighbour: one step of 2^-10 relative.  So scores differ by at most 2 * 2^-10 * sum |q k| * scale = e, weights by the factor
exp(2 e), and the output by (exp(2 e) - 1 + 2^-10 (value) + 2 * 2^-11 (weights and output)) * sum(p |v|) / l.  The token
of a step has to be the one that its logits and random number define."""
import math

import numpy as np
import pytest
import torch

import hexb200
from hexb200 import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda:0")

V, DM, HQ, HKV, D, PAGE = 1000, 256, 8, 2, 64, 16


def weights(seed):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, k: (torch.randn(*s, generator=g) * k).half().to(dev)
    return {"emb": n(V, DM, k=1.0), "wqkv": n(DM, (HQ + 2 * HKV) * D, k=DM ** -0.5), "wo": n(HQ * D, DM, k=(HQ * D) ** -0.5),
            "gq": 1 + n(D, k=0.1), "gk": 1 + n(D, k=0.1)}


def heads64(w, tokens):
    """q, k, v of a history in 64 bits, rounded to fp16 where the step stores fp16."""
    T = len(tokens)
    qkv = (w["emb"][tokens].double() @ w["wqkv"].double()).half().double().view(T, HQ + 2 * HKV, D)
    ang = torch.arange(T, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    turn = torch.polar(torch.ones_like(ang), ang)[:, None]

    def rotate(x, gain):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * gain.double()
        return torch.view_as_real(torch.view_as_complex(x.view(T, -1, D // 2, 2).contiguous()) * turn).flatten(-2).half().double()

    return rotate(qkv[:, :HQ], w["gq"]), rotate(qkv[:, HQ:HQ + HKV], w["gk"]), qkv[:, HQ + HKV:]


def check_attention(w, history, got):
    q, k, v = heads64(w, history)
    q = q[-1].view(HKV, HQ // HKV, D)
    scale = 1 / math.sqrt(D)
    s = torch.einsum("hgd,nhd->hgn", q, k) * scale
    p = torch.softmax(s, -1)
    want = torch.einsum("hgn,nhd->hgd", p, v)
    spread = torch.einsum("hgn,nhd->hgd", p, v.abs())
    e = 2 * 2.0 ** -10 * float(torch.einsum("hgd,nhd->hgn", q.abs(), k.abs()).max()) * scale
    bound = (math.expm1(2 * e) + 2.0 ** -10 + 2 * 2.0 ** -11) * spread + 2.0 ** -20
    err = (got.double().view_as(want) - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def draw64(x, u, temp, top_k, top_p):
    order = np.argsort(-x, kind="stable")[:top_k]
    wt = np.exp((x[order] - x[order[0]]) / temp)
    before = np.concatenate([[0.0], np.cumsum(wt)[:-1]])
    order = np.sort(order[:max(1, int(np.searchsorted(before, top_p * wt.sum(), side="left")))])
    up = np.cumsum(np.exp((x[order] - x.max()) / temp))
    return int(order[min(len(order) - 1, int(np.searchsorted(up, u * up[-1], side="right")))])


@pytest.mark.parametrize("B,prompt", [(3, 37), (70, 130)])
def test_decode_steps_behind_a_shared_prompt(B, prompt):
    w = weights(11)
    steps, per_seq = 6, 3                                    # three pages of own keys a sequence
    g = torch.Generator().manual_seed(B)
    prompt_ids = torch.randint(0, V, (prompt,), generator=g).to(dev)
    npre = -(-prompt // PAGE)
    order = torch.randperm(npre + B * per_seq + 2, generator=g).to(torch.int32)
    prefix_pages, table = order[:npre].to(dev), order[npre:npre + B * per_seq].view(B, per_seq).to(dev)
    kc = torch.full((len(order), PAGE, HKV, D), float("nan"), dtype=torch.float16, device=dev)
    vc = kc.clone()

    # the prompt, once for all: keys normed and rotated on the way into the cache
    x = w["emb"][prompt_ids]
    qkv = torch.empty(prompt, (HQ + 2 * HKV) * D, dtype=torch.float16, device=dev)
    ops.matmul(x, w["wqkv"], qkv)
    h = qkv.view(prompt, HQ + 2 * HKV, D)
    pos = torch.arange(prompt, device=dev)
    slots = prefix_pages.long()[pos // PAGE] * PAGE + pos % PAGE
    ops.kv_cache_append(h[:, HQ:HQ + HKV], h[:, HQ + HKV:], kc, vc, slots, pos, k_weight=w["gk"], check_slots=True)

    tokens = torch.randint(0, V, (B,), generator=g).to(dev)  # every sequence continues with its own token
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    u = torch.zeros(B, device=dev)
    f16 = lambda *s: torch.empty(*s, dtype=torch.float16, device=dev)
    x, qkv, att, y = f16(B, DM), f16(B, (HQ + 2 * HKV) * D), f16(B, HQ, D), f16(B, DM)
    logits = torch.empty(B, V, dtype=torch.float32, device=dev)

    def step():
        x.copy_(w["emb"][tokens])
        ops.matmul(x, w["wqkv"], qkv)
        h = qkv.view(B, HQ + 2 * HKV, D)
        at = lens.long()
        ops.qk_norm_rope(h[:, :HQ], h[:, HQ:HQ + HKV], h[:, :HQ], h[:, HQ:HQ + HKV], at + prompt, w["gq"], w["gk"])
        slot = table.long().gather(1, (at // PAGE)[:, None])[:, 0] * PAGE + at % PAGE
        ops.kv_cache_append(h[:, HQ:HQ + HKV], h[:, HQ + HKV:], kc, vc, slot)
        lens.add_(1)
        ops.shared_prefix_attention(h[:, :HQ], kc, vc, att, prefix_pages, prompt, table, lens)
        ops.linear(att.view(B, HQ * D), w["wo"], y, residual=x)
        ops.matmul_nt(y, w["emb"], logits)
        ops.sample_tokens(logits, u, tokens, temperature=0.9, top_k=50, top_p=0.95)

    history = [prompt_ids.tolist() + [t] for t in tokens.tolist()]
    r = np.random.default_rng(3)
    graph = None
    for i in range(steps):
        u.copy_(torch.from_numpy(r.random(B, dtype=np.float32)))
        if i == 0:
            step()
        else:
            if graph is None:
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            graph.replay()
        for b in range(0, B, max(1, B // 5)):
            check_attention(w, torch.tensor(history[b], device=dev), att[b])
        xs, us = logits.double().cpu().numpy(), u.double().cpu().numpy()
        new = tokens.tolist()
        assert new == [draw64(xs[b], us[b], float(np.float32(0.9)), 50, float(np.float32(0.95))) for b in range(B)]
        for b in range(B):
            history[b].append(new[b])
    assert hexb200.device_status() == 0
    assert lens.tolist() == [steps] * B
    # slots that no key was written to are as they were
    written = torch.zeros(kc.shape[:2], dtype=torch.bool, device=dev)
    written.view(-1)[slots] = True
    for b in range(B):
        for j in range(steps):
            written[int(table[b, j // PAGE]), j % PAGE] = True
    assert bool(kc[~written].isnan().all()) and bool(torch.isfinite(kc[written]).all())
