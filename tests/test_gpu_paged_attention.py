"""GPU: attention over a paged cache with a shared prefix, against softmax attention in 64 bits.

Tolerance, element by element: the output's rounding (half a step, 2^-11 of the value), the rounding of the weights
to fp16 for the second product (2^-11 of sum(p |v|) / l, and half of the smallest subnormal, 2^-25, for each
weight), and the error of the scores: fp32 accumulation of D products, D * 2^-23 of sum |q k| * scale (one step
per addition, allowing truncation), which enters numerator and denominator."""
import math

import pytest
import torch

import hexb200
from hexb200 import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda:0")


def pool(pages, page, Hkv, D, seed, heads_first=False):
    g = torch.Generator(device=dev).manual_seed(seed)
    shape = (pages, Hkv, page, D) if heads_first else (pages, page, Hkv, D)
    kc = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    vc = torch.randn(shape, generator=g, device=dev, dtype=torch.float16)
    return (kc.transpose(1, 2), vc.transpose(1, 2)) if heads_first else (kc, vc)


def layout(prefix, lens, page, seed, spare=3):
    """Pages anywhere in the pool: prefix pages, block table, number of pages."""
    npre, need = -(-prefix // page), [-(-n // page) for n in lens]
    total = npre + sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(need + [0])), 1 << 30, dtype=torch.int32)     # unused entries are never read
    at = npre
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return order[:npre].to(dev), table.to(dev), total


def spoil_unused(kc, vc, prefix, prefix_pages, lens, table, page):
    """NaN and inf in every slot that no visible key occupies."""
    keep = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for j in range(prefix):
        keep[int(prefix_pages[j // page]), j % page] = True
    tab = table.cpu()
    for b, n in enumerate(lens):
        for j in range(n):
            keep[int(tab[b, j // page]), j % page] = True
    keep = keep.to(dev)
    kc[~keep] = float("nan")
    vc[~keep] = float("inf")


def gather(cache, pages, n):
    return cache[pages.long()].reshape(-1, *cache.shape[2:])[:n].double()


def check(out, q, kc, vc, prefix_pages, prefix, table, lens, counts, scale=None):
    T, Hq, D = q.shape
    Hkv, page = kc.shape[2], kc.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    t = 0
    for b, (c, n) in enumerate(zip(counts, lens)):
        if c == 0:
            continue
        own = table[b, :-(-n // page)] if table is not None else torch.zeros(0, dtype=torch.int32, device=dev)
        k = torch.cat([gather(kc, prefix_pages, prefix), gather(kc, own, n)]) if prefix else gather(kc, own, n)
        v = torch.cat([gather(vc, prefix_pages, prefix), gather(vc, own, n)]) if prefix else gather(vc, own, n)
        x = q[t:t + c].double().view(c, Hkv, Hq // Hkv, D)
        s = torch.einsum("chgd,nhd->chgn", x, k) * scale
        i, j = torch.arange(c, device=dev)[:, None], torch.arange(prefix + n, device=dev)[None, :]
        seen = j < prefix + n - c + i + 1
        seen = seen | (j < prefix)
        s = s.masked_fill(~seen[:, None, None, :], -math.inf)
        top = s.amax(-1, keepdim=True) if prefix + n else torch.full((c, Hkv, Hq // Hkv, 1), -math.inf, device=dev, dtype=torch.float64)
        p = torch.exp(s - torch.where(top.isinf(), torch.zeros_like(top), top))
        l = p.sum(-1, keepdim=True)
        safe = torch.where(l > 0, l, torch.ones_like(l))
        want = torch.einsum("chgn,nhd->chgd", p, v) / safe
        wabs = torch.einsum("chgn,nhd->chgd", p, v.abs()) / safe
        vsum = torch.einsum("chgn,nhd->chgd", (p > 0).double(), v.abs()) / safe
        err_s = 0.0
        if prefix + n:
            err_s = D * 2.0 ** -23 * float(torch.einsum("chgd,nhd->chgn", x.abs(), k.abs()).max()) * abs(scale)
        bound = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * err_s) * wabs + 2.0 ** -25 * vsum + 2.0 ** -25
        err = (out[t:t + c].double().view_as(want) - want).abs()
        assert bool((err <= bound).all()), (b, float((err / bound).max()))
        assert bool((out[t:t + c].view_as(want)[(l == 0).expand_as(want)] == 0).all())
        t += c


CASES = [
    # Hq, Hkv, D, page, prefix, query counts, own lengths
    (8, 2, 128, 16, 500, [1] * 3, [1, 17, 64]),
    (8, 2, 128, 16, 0, [1] * 4, [0, 1, 63, 200]),                 # no prefix; a sequence without keys: zeros
    (4, 4, 64, 16, 1, [1], [0]),                                  # one visible key in all
    (4, 1, 64, 1, 65, [1] * 2, [3, 129]),                         # pages of one slot
    (6, 2, 128, 24, 130, [1] * 5, [24, 25, 23, 1, 700]),          # pages that end inside a block
    (10, 2, 64, 16, 64, [1] * 7, [1] * 7),                        # five heads a group
    (32, 2, 128, 32, 2049, [1] * 9, [33] * 9),                    # sixteen heads a group
    (40, 1, 128, 16, 300, [1, 1], [5, 600]),                      # forty heads a group
    (8, 8, 72, 16, 100, [1] * 3, [9, 90, 900]),                   # head sizes between the tiled ones
    (8, 2, 8, 16, 100, [1] * 3, [9, 90, 300]),
    (4, 2, 256, 16, 333, [1] * 3, [1, 65, 400]),
    (8, 2, 128, 16, 200, [5, 1, 0, 17], [5, 3, 9, 40]),           # ragged new tokens, one sequence without
    (8, 2, 64, 16, 0, [5, 3], [2, 3]),                            # more new tokens than keys: rows that see nothing
    (8, 2, 128, 64, 129, [70, 200], [70, 333]),                   # chunks, causal among themselves
    (4, 4, 64, 128, 1000, [129], [129]),
    (12, 12, 64, 16, 64, [33, 64, 1], [40, 64, 500]),
    (16, 2, 128, 16, 4096, [1] * 40, [100] * 40),                 # many rows against a long prefix
    (24, 8, 128, 64, 777, [1] * 64, list(range(64))),             # three heads a group, many rows
    (8, 2, 128, 8, 300, [1] * 40, [100] * 40),                    # the smallest page that TMA pieces fit
    (8, 2, 64, 40, 300, [30, 41], [100, 90]),                     # pages of five pieces
    (200, 1, 64, 16, 100, [1, 3], [30, 31]),                      # more heads a group than a tile has rows
    (128, 1, 128, 16, 100, [2, 3], [30, 31]),
    (2, 2, 128, 512, 700, [100, 90], [1500, 90]),                 # pages longer than a block
    (6, 6, 64, 16, 90, [40], [40]),
    (2, 1, 128, 16, 20000, [1], [5]),
    (2, 1, 64, 16, 0, [1], [20000]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("heads_first", [False, True])
def test_vs_softmax_in_64_bits(case, heads_first):
    Hq, Hkv, D, page, prefix, counts, lens = CASES[case]
    prefix_pages, table, pages = layout(prefix, lens, page, case)
    kc, vc = pool(pages, page, Hkv, D, case, heads_first)
    spoil_unused(kc, vc, prefix, prefix_pages, lens, table, page)
    g = torch.Generator(device=dev).manual_seed(100 + case)
    T = sum(counts)
    q = torch.randn(T + 3, Hq, D, generator=g, device=dev, dtype=torch.float16)
    out = torch.full_like(q, 5.0)
    off = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    ln = torch.tensor(lens, dtype=torch.int32, device=dev)
    for max_q in (0, max(counts), 1):                             # shapes the launch, never the result
        out.fill_(5.0)
        ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, prefix, table, ln, off, max_q=max_q)
        assert hexb200.device_status() == 0
        assert bool((out[T:] == 5.0).all())                       # rows behind the last sequence
        check(out[:T], q[:T], kc, vc, prefix_pages, prefix, table, lens, counts)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix,B,G", [(63, 1, 1), (64, 100, 4), (65, 37, 8), (1025, 64, 5), (5000, 33, 4), (128, 300, 12)])
def test_prefix_only(D, prefix, B, G):
    Hkv, page = 2, 16
    prefix_pages, _, pages = layout(prefix, [], page, 1)
    kc, vc = pool(pages, page, Hkv, D, 2)
    spoil_unused(kc, vc, prefix, prefix_pages, [], torch.zeros(0, 0), page)
    q = torch.randn(B, Hkv * G, D, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).half()
    out = torch.empty_like(q)
    ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, prefix)
    check(out, q, kc, vc, prefix_pages, prefix, None, [0] * B, [1] * B)


@pytest.mark.parametrize("case", [0, 5, 11, 13, 16])
def test_without_overlapping_launches(case):
    """Option "pdl" 0: the launches of a call run one after the other."""
    hexb200.set_option("pdl", 0)
    try:
        test_vs_softmax_in_64_bits(case, False)
    finally:
        hexb200.set_option("pdl", 1)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales_and_large_scores(scale):
    prefix_pages, table, pages = layout(700, [50, 60], 16, 4)
    kc, vc = pool(pages, 16, 2, 64, 5)
    q = torch.randn(2, 64, 64, device=dev, generator=torch.Generator(device=dev).manual_seed(6)).half()
    out = torch.empty_like(q)
    ln = torch.tensor([50, 60], dtype=torch.int32, device=dev)
    ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, 700, table, ln, sm_scale=scale)
    check(out, q, kc, vc, prefix_pages, 700, table, [50, 60], [1, 1], scale=scale)


def test_rising_scores_over_a_long_prefix():
    """Every block of keys raises the running maximum: the accumulators are rescaled again and again."""
    P, D = 4096, 64
    prefix_pages, _, pages = layout(P, [], 64, 4)
    kc, vc = pool(pages, 64, 1, D, 5)
    ramp = torch.linspace(0, 30, P, device=dev).half()
    flat = torch.zeros(P, 1, D, dtype=torch.float16, device=dev)
    flat[:, 0, 0] = ramp
    kc[prefix_pages.long()] = flat.view(-1, 64, 1, D)
    q = torch.zeros(200, 1, D, dtype=torch.float16, device=dev)
    q[:, 0, 0] = torch.linspace(-8, 8, 200, device=dev).half()
    out = torch.empty_like(q)
    ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, P)
    check(out, q, kc, vc, prefix_pages, P, None, [0] * 200, [1] * 200)


@pytest.mark.parametrize("D,G", [(64, 4), (128, 4), (80, 4), (128, 1)])
def test_keys_of_infinite_scores(D, G):
    """Keys at -inf in a column where every query is positive weigh nothing, whole key ranges of them too."""
    P, B, Hkv = 1500, 24, 2
    prefix_pages, table, pages = layout(P, [70] * B, 16, 4)
    kc, vc = pool(pages, 16, Hkv, D, 5)
    rows = kc.view(-1, Hkv, D)
    slots = (prefix_pages.long()[:, None] * 16 + torch.arange(16, device=dev)).flatten()
    rows[slots[:900], :, 0] = -float("inf")
    rows[slots[1400:1440], :, 0] = -float("inf")
    kc[table[:, :2].long().flatten(), :, :, 0] = -float("inf")
    q = torch.randn(B, Hkv * G, D, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).half()
    q[..., 0] = 0.5
    out = torch.empty_like(q)

    def same_as_without_them(own):
        # the keys that count, as sequences of their own in pages of one slot
        for b in range(B if own else 1):
            k = torch.cat([gather(kc, prefix_pages, P)] + ([gather(kc, table[b], 70)] if own else []))
            v = torch.cat([gather(vc, prefix_pages, P)] + ([gather(vc, table[b], 70)] if own else []))
            left = ~k[:, 0, 0].isinf()
            k, v = k[left].half()[:, None], v[left].half()[:, None]
            n = k.shape[0]
            assert n == (P - 940 + 38 if own else P - 940)
            some = slice(b, b + 1) if own else slice(0, B)
            check(out[some], q[some], k, v, torch.arange(n, device=dev), n, None, [0] * (1 if own else B), [1] * (1 if own else B))

    ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, P)
    same_as_without_them(False)
    ln = torch.full((B,), 70, dtype=torch.int32, device=dev)
    ops.shared_prefix_attention(q, kc, vc, out, prefix_pages, P, table, ln)
    same_as_without_them(True)


def test_in_place_views_and_a_second_stream():
    Hq, Hkv, D = 8, 2, 128
    prefix_pages, table, pages = layout(300, [20, 30, 70], 16, 9)
    kc, vc = pool(pages, 16, Hkv, D, 9)
    buf = torch.randn(3, Hq + 2 * Hkv, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).half()
    q, keep = buf[:, :Hq], buf.clone()
    wide = torch.full((3, 50), -7, dtype=torch.int32, device=dev)            # a table with a row stride
    wide[:, :table.shape[1]] = table
    ln = torch.tensor([20, 30, 70], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.shared_prefix_attention(q, kc, vc, q, prefix_pages, 300, wide[:, :table.shape[1]], ln)
    torch.cuda.current_stream().wait_stream(side)
    check(q, keep[:, :Hq], kc, vc, prefix_pages, 300, table, [20, 30, 70], [1] * 3)
    assert torch.equal(buf[:, Hq:], keep[:, Hq:])


def test_a_captured_step_follows_lengths_and_tables():
    Hq, Hkv, D, page = 8, 2, 64, 16
    prefix_pages, table, pages = layout(100, [64, 64, 64], page, 2)
    kc, vc = pool(pages, page, Hkv, D, 2)
    q = torch.randn(3, Hq, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).half()
    q2 = torch.randn(3, Hq, D, device=dev, generator=torch.Generator(device=dev).manual_seed(9)).half()
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    ln = torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)
    call = lambda a, o: ops.shared_prefix_attention(a, kc, vc, o, prefix_pages, 100, table, ln)
    call(q, out)
    graphs = []
    for a, o in ((q, out), (q2, out2)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(a, o)
        graphs.append(gr)
    for lens in ([64, 0, 17], [5, 33, 64]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        table.copy_(table[[1, 2, 0]])
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        for s in (s1, s2):
            s.wait_stream(torch.cuda.current_stream())
        for s, gr in ((s1, graphs[0]), (s2, graphs[1])):                     # two graphs at once
            with torch.cuda.stream(s):
                gr.replay()
        for s in (s1, s2):
            torch.cuda.current_stream().wait_stream(s)
        check(out, q, kc, vc, prefix_pages, 100, table, lens, [1] * 3)
        check(out2, q2, kc, vc, prefix_pages, 100, table, lens, [1] * 3)


def test_bad_pages_and_lengths_are_recorded():
    Hq, Hkv, D, page = 4, 2, 64, 16
    kc, vc = pool(6, page, Hkv, D, 2)
    q = torch.randn(2, Hq, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).half()
    out = torch.empty_like(q)
    table = torch.tensor([[0, 6], [-1, 2]], dtype=torch.int32, device=dev)   # pages 6 and -1 do not exist
    ln = torch.tensor([32, 32], dtype=torch.int32, device=dev)
    ops.shared_prefix_attention(q, kc, vc, out, None, 0, table, ln)
    assert hexb200.device_status() == -1 and hexb200.device_status() == 0
    pad = lambda c: torch.cat([c, torch.zeros(1, page, Hkv, D, dtype=c.dtype, device=dev)])
    good = torch.tensor([[0, 6], [6, 2]], dtype=torch.int32, device=dev)     # reads as a page of zeros
    check(out, q, pad(kc), pad(vc), None, 0, good, [32, 32], [1, 1])
    ln.fill_(33)                                                             # one more than the table holds
    table = torch.tensor([[0, 1], [4, 2]], dtype=torch.int32, device=dev)
    ops.shared_prefix_attention(q, kc, vc, out, None, 0, table, ln)
    assert hexb200.device_status() == -1
    check(out, q, kc, vc, None, 0, table, [32, 32], [1, 1])
    bad = torch.tensor([1, 99], dtype=torch.int32, device=dev)
    qq = torch.randn(200, Hq, D, device=dev, generator=torch.Generator(device=dev).manual_seed(8)).half()
    oo = torch.empty_like(qq)
    ops.shared_prefix_attention(qq, kc, vc, oo, bad, 32)
    assert hexb200.device_status() == -1
    check(oo, qq, pad(kc), pad(vc), torch.tensor([1, 6], device=dev), 32, None, [0] * 200, [1] * 200)


def test_no_keys_at_all_and_empty_calls():
    kc, vc = pool(2, 16, 2, 64, 2)
    q = torch.randn(3, 4, 64, device=dev).half()
    out = torch.full_like(q, 3.0)
    ops.shared_prefix_attention(q, kc, vc, out)
    assert bool((out == 0).all())
    e = q[:0]
    ops.shared_prefix_attention(e, kc, vc, e.clone())
    off = torch.zeros(1, dtype=torch.int32, device=dev)
    out.fill_(3.0)
    ops.shared_prefix_attention(q, kc, vc, out, q_offsets=off)               # a batch of none
    assert bool((out == 3.0).all())


def test_cache_offsets_past_32_bits():
    D, Hkv, page = 64, 1, 16
    store = torch.zeros((1 << 31) + (1 << 23), dtype=torch.float16, device=dev)
    kc = store.as_strided((513, page, Hkv, D), (1 << 22, D, D, 1))
    vc = store.as_strided((513, page, Hkv, D), (1 << 22, D, D, 1), 2048)
    kc[510:] = torch.randn(3, page, Hkv, D, device=dev).half()
    vc[510:] = torch.randn(3, page, Hkv, D, device=dev).half()
    q = torch.randn(70, 2, D, device=dev).half()
    out = torch.empty_like(q)
    pre = torch.tensor([512, 511], dtype=torch.int32, device=dev)
    table = torch.full((70, 1), 510, dtype=torch.int32, device=dev)
    ln = torch.full((70,), 11, dtype=torch.int32, device=dev)
    ops.shared_prefix_attention(q, kc, vc, out, pre, 32, table, ln)
    check(out, q, kc, vc, pre, 32, table, [11] * 70, [1] * 70)


def test_host_tensors_are_staged():
    prefix_pages, table, pages = layout(40, [9], 16, 4)
    kc, vc = pool(pages, 16, 2, 64, 5)
    q = torch.randn(1, 4, 64, device=dev).half()
    out = torch.empty_like(q).cpu()
    ln = torch.tensor([9], dtype=torch.int32)
    ops.shared_prefix_attention(q.cpu(), kc.cpu(), vc.cpu(), out, prefix_pages.cpu(), 40, table.cpu(), ln)
    check(out.to(dev), q, kc, vc, prefix_pages, 40, table, [9], [1])


@pytest.mark.parametrize("D", [64, 128, 80])
def test_inputs_written_right_before_the_call(D):
    """Queries, lengths, tables and own keys that the kernels before it in the stream wrote, step after step."""
    B, Hq, Hkv, page, P = 70, 8, 2, 16, 700
    prefix_pages, table, pages = layout(P, [64] * B, page, 3)
    kc, vc = pool(pages, page, Hkv, D, 3)
    g = torch.Generator(device=dev).manual_seed(4)
    own_pages = table.flatten().long()
    sources, outs = [], []
    for i in range(6):
        lens = torch.randint(0, 65, (B,), generator=g, device=dev, dtype=torch.int32)
        q = torch.randn(B, Hq, D, generator=g, device=dev).half()
        keys = torch.randn(2, B * 4, page, Hkv, D, generator=g, device=dev).half()
        sources.append((q, lens, table[torch.randperm(B, generator=g, device=dev)], keys))
        outs.append(torch.empty_like(q))
    q, lens, tab = torch.empty_like(sources[0][0]), torch.empty_like(sources[0][1]), torch.empty_like(table)

    def step(i):
        kc.index_copy_(0, own_pages, sources[i][3][0])
        vc.index_copy_(0, own_pages, sources[i][3][1])
        for dst, src in zip((tab, lens, q), (sources[i][2], sources[i][1], sources[i][0])):
            dst.copy_(src)
        ops.shared_prefix_attention(q, kc, vc, outs[i], prefix_pages, P, tab, lens)

    for _ in range(20):
        for i in range(6):
            step(i)
    torch.cuda.synchronize()
    for i in range(6):
        got = outs[i].clone()
        step(i)
        assert torch.equal(outs[i], got)                         # the same, whatever ran before
        check(got, sources[i][0], kc, vc, prefix_pages, P, sources[i][2], sources[i][1].tolist(), [1] * B)
