"""GPU: token sampling against the definition in 64 bits (a sort, exact filters, the draw in index order).

Tokens are whole numbers and have to be equal.  The library's sums are good to about 2^-36 of the mass, so where a
random row's u (or top_p) lies within 1e-9 of the mass of a border, it is moved by 2^-20 before the call.  Rows
on a border by design (ties, u = 0) are exact in both."""
import numpy as np
import pytest
import torch

import hexb200
from hexb200 import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda:0")


def define(x, u, temp, top_k, top_p, min_p):
    """(token, distance of the closest border in mass) of one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    real = np.flatnonzero(x > -np.inf)
    if len(real) == 0:
        return -1, 1.0
    if temp <= 0:
        return int(np.argmax(x)), 1.0
    order = real[np.argsort(-x[real], kind="stable")]
    top = x[order[0]]
    if top_k > 0:
        order = order[:top_k]
    weigh = lambda v: np.where(v == top, 1.0, np.exp((np.where(v == top, 0.0, v) - (0.0 if np.isinf(top) else top)) / temp)
                               * (0.0 if np.isinf(top) else 1.0))
    w = weigh(x[order])
    near = 1.0
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        near = float(np.abs(before[1:] - top_p * w.sum()).min() / w.sum()) if len(w) > 1 else 1.0
        order = order[:max(1, int(np.searchsorted(before, top_p * w.sum(), side="left")))]
    chosen = np.sort(order)
    w = weigh(x[chosen])
    chosen, w = chosen[w >= min_p], w[w >= min_p]
    up = np.cumsum(w)
    i = min(len(chosen) - 1, int(np.searchsorted(up, u * up[-1], side="right")))
    return int(chosen[i]), min(near, float(np.abs(up[:-1] - u * up[-1]).min() / up[-1]) if len(up) > 1 else 1.0)


def settle(x, u, temp, top_k, top_p, min_p):
    """The arguments with u (and top_p) moved off close borders, and the tokens."""
    x64 = x.double().cpu().numpy()
    f = lambda v: float(np.float32(v))
    tokens = []
    for r in range(x.shape[0]):
        for _ in range(50):
            token, near = define(x64[r], f(u[r]), f(temp[r]), int(top_k[r]), f(top_p[r]), f(min_p[r]))
            if near > 1e-9:
                break
            u[r] = min(max(0.0, u[r] + 2.0 ** -20), 1 - 2.0 ** -24) if u[r] < 0.5 else u[r] - 2.0 ** -20
            if top_p[r] < 1:
                top_p[r] -= 2.0 ** -20
        tokens.append(token)
    return u, top_p, tokens


def call(x, u, temp, top_k, top_p, min_p):
    out = torch.full((x.shape[0],), -9, dtype=torch.int64, device=dev)
    t = lambda v, dt: torch.tensor(np.asarray(v), dtype=dt, device=dev)
    ops.sample_tokens(x, t(u, torch.float32), out, t(temp, torch.float32), t(top_k, torch.int32), t(top_p, torch.float32),
                      t(min_p, torch.float32))
    return out.cpu().tolist()


def compare(x, u, temp, top_k, top_p, min_p):
    u, top_p, want = settle(x, list(u), list(temp), list(top_k), list(top_p), list(min_p))
    assert call(x, u, temp, top_k, top_p, min_p) == want


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 33), (40, 1000), (17, 16384), (13, 16385), (24, 50257), (9, 100003),
                                        (6, 151936)])
@pytest.mark.parametrize("spread", [0.5, 3.0])
def test_random_rows(rows, vocab, dtype, spread):
    g = torch.Generator().manual_seed(rows * 7 + vocab)
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype).to(dev)
    r = np.random.default_rng(vocab)
    u = r.random(rows, dtype=np.float32)
    temp = r.choice([0.0, 0.3, 0.7, 1.0, 1.5], rows)
    top_k = r.choice([0, 0, 1, 2, 50, 1000, 30000], rows)
    top_p = r.choice([1.0, 1.0, 0.1, 0.9, 0.95, 0.999], rows)
    min_p = r.choice([0.0, 0.0, 0.05, 0.3], rows)
    compare(x, u, temp, top_k, top_p, min_p)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_ties_go_to_the_lowest_index(dtype):
    V = 20000
    x = torch.full((8, V), 2.0, dtype=dtype, device=dev)
    x[4:] = -1.0
    x[4:, ::7] = 3.0                                                # 2858 equal logits on top
    u = np.array([0.0, 0.5, 0.999, 0.25] * 2, dtype=np.float32)
    # k of equal logits: the first k indexes, equally likely
    assert call(x, u, [1.0] * 8, [10] * 8, [1.0] * 8, [0.0] * 8) == [0, 5, 9, 2, 0, 35, 63, 14]
    # half of the mass of V equal logits: V/2 of them; an eighth of 2858 is 357.25: the 358th still begins below it
    assert call(x, u, [1.0] * 4 + [0.1] * 4, [0] * 8, [0.5] * 4 + [0.125] * 4, [0.0] * 8) == \
        [0, 5000, 9990, 2500, 0, 7 * 179, 7 * 357, 7 * 89]
    assert call(x, u, [0.0] * 8, [0] * 8, [1.0] * 8, [0.0] * 8) == [0] * 8
    assert call(x, u, [1.0] * 8, [1] * 8, [1.0] * 8, [0.0] * 8) == [0] * 8


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_masked_infinite_and_nan_logits(dtype):
    V = 40001
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, V, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = -float("inf")                                            # nothing to choose from
    x[1] = float("nan")
    x[2, :] = -float("inf")
    x[2, 777] = -3.0                                                # one logit
    x[3, 100:] = -float("inf")
    x[4, 50:] = low                                                 # masked with the lowest value
    x[5, ::2] = float("nan")
    x[6, 30] = x[6, 40000] = float("inf")                           # only these have weight
    x[7, :] = low                                                   # equal, however low
    x[8, 5], x[8, 6] = -0.0, 0.0
    x[8, 7:] = -1.0
    x[9, 1::3] = -float("inf")
    x[10] = 0.0
    x[11, 0] = torch.finfo(dtype).max
    x = x.to(dev)
    r = np.random.default_rng(1)
    for temp, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 20, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 2000, 0.8, 0.01), (0.0, 0, 1.0, 0.0),
                          (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0)):
        compare(x, r.random(12, dtype=np.float32), [temp] * 12, [k] * 12, [p] * 12, [m] * 12)


def test_border_random_numbers_and_scalar_parameters():
    x = torch.zeros(6, 8, device=dev)
    x[:, 0] = -float("inf")
    out = torch.empty(6, dtype=torch.int64, device=dev)
    u = torch.tensor([0.0, 1 / 7 + 1e-6, 1 - 2.0 ** -24, 1.0, -3.0, float("nan")], device=dev)   # the last three are clamped
    ops.sample_tokens(x, u, out)
    assert out.tolist()[:5] == [1, 2, 7, 7, 1] and 1 <= out[5] <= 7
    ops.sample_tokens(x, u, out, temperature=0)
    assert out.tolist() == [1] * 6
    ops.sample_tokens(x, u, out, top_k=3, top_p=0.5, min_p=0.5)
    assert out.tolist()[:5] == [1, 1, 2, 2, 1]
    ops.sample_tokens(x, u, out, top_k=1 << 40)
    assert out.tolist()[:5] == [1, 2, 7, 7, 1]


@pytest.mark.parametrize("rows", [2, 160])
def test_rows_masked_but_for_few(rows):
    """Constrained decoding: all but a few logits are -inf (or the lowest value), wherever they lie."""
    V = 60000
    g = torch.Generator().manual_seed(rows)
    x = torch.full((rows, V), -float("inf"))
    x[1::2] = torch.finfo(torch.float16).min
    for r in range(rows):
        at = torch.randperm(V, generator=g)[:100]
        x[r, at] = torch.randn(100, generator=g) * 3
    x = x.half().to(dev)
    r = np.random.default_rng(4)
    compare(x, r.random(rows, dtype=np.float32), r.choice([0.5, 1.0], rows), r.choice([0, 7, 200], rows),
            r.choice([1.0, 0.9], rows), r.choice([0.0, 0.01], rows))


@pytest.mark.parametrize("temp", [1e-40, 1e-3, 50.0, 1e30])
def test_extreme_temperatures(temp):
    """The definition's weights in 64 bits: near 0 the largest logits alone, far above 1 all alike."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 30000, generator=g).to(dev)
    x[1, 7] = x[1, 20000] = 9.0
    compare(x, [0.1, 0.6, 0.5, 0.99], [temp] * 4, [0, 0, 500, 0], [1.0, 0.9, 0.9, 0.3], [0.0, 0.0, 0.0, 0.2])


@pytest.mark.parametrize("temp", [1e36, 3e38, float("inf")])
@pytest.mark.parametrize("rows", [2, 160])
def test_temperatures_that_level_every_logit(rows, temp):
    # the weights of all finite logits are 1 to 64 bits; masked places stay out
    V = 4099
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, V, generator=g)
    x[:, ::3] = -float("inf")
    x[:, 1::7] = float("nan")
    x = x.to(dev)
    for top_k, top_p, min_p in ((0, 1.0, 0.0), (0, 0.5, 0.0), (100, 1.0, 0.0), (2000, 0.25, 0.5), (0, 1.0, 1.0), (0, 0.5, 1.0),
                                 (100, 1.0, 1.0), (2000, 1.0, 1.0)):
        u = np.random.default_rng(7).random(rows, dtype=np.float32)
        compare(x, u, [temp] * rows, [top_k] * rows, [top_p] * rows, [min_p] * rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strided_rows_of_any_alignment(dtype):
    g = torch.Generator().manual_seed(5)
    wide = (torch.randn(9, 20011, generator=g) * 2).to(dtype).to(dev)
    r = np.random.default_rng(2)
    for a, b in ((0, 20011), (1, 20010), (3, 17000), (7, 12), (2, 5)):
        x = wide[:, a:b] if b > a else wide[:, b:a]
        compare(x, r.random(9, dtype=np.float32), [0.9] * 9, [0, 5, 100] * 3, [0.9, 1.0, 0.5] * 3, [0.0] * 9)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_row_larger_than_shared_memory(dtype):
    V = 900001
    g = torch.Generator(device=dev).manual_seed(5)
    x = (torch.randn(2, V, generator=g, device=dev) * 2).to(dtype)
    compare(x, [0.37, 0.81], [1.0, 0.8], [0, 300], [0.9, 1.0], [0.0, 0.0])


def test_same_result_every_time_and_frequencies():
    """Bit-equal runs (the atomics' order has no say), and the empirical distribution: 2^16 rows of 64 logits; each
    frequency within 5 standard deviations of its probability (a chance of 4e-5 over 64 classes for random u;
    u is a low-discrepancy sequence here, which stays far inside)."""
    n, V = 1 << 16, 64
    g = torch.Generator(device=dev).manual_seed(5)
    base = torch.randn(V, generator=g, device=dev)
    x = base.expand(n, V).contiguous()
    u = (torch.arange(n, device=dev, dtype=torch.float64) * 0.6180339887498949 % 1.0).float().clamp_(max=1 - 2.0 ** -24)
    a, b = torch.empty(n, dtype=torch.int64, device=dev), torch.empty(n, dtype=torch.int64, device=dev)
    ops.sample_tokens(x, u, a, top_p=0.99)
    ops.sample_tokens(x, u, b, top_p=0.99)
    assert torch.equal(a, b)
    p = torch.softmax(base.double(), 0)
    v, i = torch.sort(p, descending=True)
    keep = (v.cumsum(0) - v) < float(np.float32(0.99))
    q = torch.zeros_like(p).scatter_(0, i, v * keep)
    q /= q.sum()
    freq = torch.bincount(a, minlength=V).double() / n
    assert bool(((freq - q).abs() <= 5 * torch.sqrt(q * (1 - q) / n) + 1e-12).all())


def test_another_stream_graph_and_empty():
    x = torch.randn(4, 5000, device=dev)
    u = torch.full((4,), 0.3, device=dev)
    out = torch.full((4,), -5, dtype=torch.int64, device=dev)
    ops.sample_tokens(x[:0], u[:0], out[:0])
    ops.sample_tokens(x, u, out, top_k=40)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_tokens(x, u, out, top_k=40)
    x.copy_(torch.randn(4, 5000, device=dev))
    u.fill_(0.9)
    graph.replay()
    got = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_tokens(x, u, out, top_k=40)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, out)
    assert got.tolist() == [define(r, 0.9, 1.0, 40, 1.0, 0.0)[0] for r in x.double().cpu().numpy()]
    host = torch.empty(4, dtype=torch.int64)
    ops.sample_tokens(x.cpu(), u.cpu(), host, top_k=torch.full((4,), 40, dtype=torch.int32))
    assert torch.equal(host, got.cpu())
    assert hexb200.device_status() == 0


def test_min_p_keeps_logits_behind_the_histograms_range():
    """A constrained vocabulary: the first places of a row do not show how far its few logits reach."""
    V, at = 60000, [0, 1, 1000, 2000, 3000]
    row = torch.full((V,), -float("inf"), dtype=torch.float16)
    row[at] = torch.tensor([5.0, 4.5, 4.0, 3.5, 3.0], dtype=torch.float16)
    for rows in (1, 80):
        x = row.to(dev).expand(rows, V)
        for top_k, top_p in ((50, 1.0), (0, 0.99), (50, 0.99)):
            for u in np.linspace(0.01, 0.99, 80, dtype=np.float32).reshape(-1, rows)[::8 if rows == 1 else 1]:
                compare(x, u, [1.0] * rows, [top_k] * rows, [top_p] * rows, [0.05] * rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [50257, 128000])
@pytest.mark.parametrize("rows", [1, 160])
def test_min_p_with_few_allowed_tokens(rows, vocab, dtype):
    g = torch.Generator().manual_seed(vocab + rows)
    r = np.random.default_rng(vocab)
    for trial in range(16 if rows == 1 else 1):
        x = torch.full((rows, vocab), -float("inf"))
        for i in range(rows):
            at = torch.randperm(vocab, generator=g)[:(2, 5, 10, 20)[(i + trial) % 4]]
            x[i, at] = torch.randn(len(at), generator=g) * 2
        x = x.to(dtype).to(dev)
        for top_k, top_p in ((50, 1.0), (0, 0.99), (8, 0.9), (0, 1.0)):
            compare(x, r.random(rows, dtype=np.float32), r.choice([0.7, 1.0], rows), [top_k] * rows, [top_p] * rows,
                    r.choice([0.02, 0.05, 0.1], rows))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [2, 160])
def test_filters_among_thousands_of_infinite_logits(rows, dtype):
    """+inf logits are equals: the filters keep the lowest indexes of them, finite ones weigh nothing."""
    V = 20000
    x = torch.full((rows, V), 3.0, dtype=dtype)
    x[:, ::5] = -7.0
    x[:, 1::3] = float("inf")                                       # 6667
    x = x.to(dev)
    u = np.resize(np.array([0.0, 0.21, 0.52, 0.999], dtype=np.float32), rows)
    # 5 by top-k; before the 3334th lie 3333 of 6667, less than half; 1500 of 6000; all with min-p alone
    for top_k, top_p, min_p, kept in ((5, 1.0, 0.0, 5), (0, 0.5, 0.0, 3334), (6000, 0.25, 0.0, 1500), (6000, 1.0, 0.5, 6000),
                                      (0, 1.0, 1.0, 6667)):
        assert call(x, u, [0.8] * rows, [top_k] * rows, [top_p] * rows, [min_p] * rows) == [1 + 3 * int(float(v) * kept) for v in u]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1000003), (80, 1000003), (1, 12000001)])
@pytest.mark.parametrize("with_top_k", [False, True])
def test_top_p_among_millions_of_equal_logits(rows, vocab, with_top_k, dtype):
    """Logits 0 at even places and -1 at odd ones: sums of the definition are whole numbers of two weights."""
    row = torch.zeros(vocab, dtype=dtype)
    row[1::2] = -1.0
    n0, n1, w = (vocab + 1) // 2, vocab // 2, float(np.exp(-1.0))
    top_k, top_p = 0, float(np.float32(0.9))
    if with_top_k:
        n1 = n1 * 3 // 4
        top_k = n0 + n1
    last = (top_p * (n0 + n1 * w) - n0) / w                          # of the odd places, how many are kept
    assert 0.05 < last % 1 < 0.95
    odd = np.arange(vocab) % 2 == 1
    c1 = np.minimum(np.cumsum(odd), int(np.ceil(last)))
    cum = np.cumsum(~odd) + c1 * w
    r = np.random.default_rng(5)
    u = np.concatenate([[np.float32(1 - 2.0 ** -24), np.float32(0.9999)], r.random(200, dtype=np.float32)]).astype(np.float32)
    t = u.astype(np.float64) * cum[-1]
    want = np.searchsorted(cum, t, side="right")
    far = np.minimum(np.abs(cum[np.minimum(want, vocab - 1)] - t), np.abs(t - cum[want - 1])) > 1e-9 * cum[-1]
    u, want = u[far], want[far].tolist()
    x = row.to(dev).expand(rows, vocab)
    for i in range(0, 8 if rows == 1 else 1):
        assert call(x, u[i:i + rows], [1.0] * rows, [top_k] * rows, [top_p] * rows, [0.0] * rows) == want[i:i + rows]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows", [2, 160])
def test_top_p_of_what_top_k_leaves_of_equal_logits(rows, dtype):
    """Top-k cuts through thousands of equal logits, and top-p (0.9 of 5) may leave all that top-k did."""
    V = 12000
    x = torch.full((rows, V), -1.0, dtype=dtype)
    x[:, ::2] = 2.0                                                  # 6000
    x = x.to(dev)
    u = np.resize(np.array([0.0, 0.21, 0.53, 0.999], dtype=np.float32), rows)
    for top_k, top_p, min_p, kept in ((5, 0.9, 0.0, 5), (50, 0.99, 0.5, 50), (5000, 0.9999, 0.0, 5000), (5000, 0.5, 0.9, 2500)):
        assert call(x, u, [0.7] * rows, [top_k] * rows, [top_p] * rows, [min_p] * rows) == [2 * int(float(v) * kept) for v in u]
