"""GPU: per-head norm with rotation, and the append to a paged cache, against the formulas in 64 bits.

Tolerance of a computed row: half a step of the output type relative to the value, and fp32 round-off relative to
the row's largest element.  The latter counts, in steps of 2^-24: the sum of squares (one rounding per
element a lane adds, D / 32 for a warp's lanes, halved by the root: D / 64; 21 -> 11 in the vector form), rsqrtf (4),
the two products of the gain (2), the angle as a fraction of a turn in 32 bits (pi * 2^-24) with sincospif (2), and
the rotation itself (3): 24 + D / 64 steps."""
import math

import pytest
import torch

import hexb200
from hexb200 import ops

pytestmark = pytest.mark.gpu
dev = torch.device("cuda:0")


def exact_rows(x, w, norm, pos, rot, interleaved, theta=10000.0, eps=1e-6):
    x = x.double()
    D = x.shape[-1]
    if norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            x = x * w.double()
    if not rot:
        return x
    y = x.clone()
    for p in range(rot // 2):
        ang = pos.double() * theta ** (-2.0 * p / rot)
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


def assert_rows(got, want):
    D = want.shape[-1]
    step = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * step      # half a step among the subnormal numbers
    bound = step * want.abs() + (24 + D / 64) * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) * math.sqrt(2) + tiny
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), float((err / bound).max())


def make(T, heads, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, heads, D, generator=g) * 1.5).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", [
    (1, 16, 4, 128, 128), (3, 5, 1, 64, 64), (777, 12, 12, 64, 32), (65, 8, 2, 256, 256), (2049, 6, 2, 96, 96),
    (33, 4, 4, 128, 0), (9, 3, 1, 80, 20), (7, 2, 1, 10, 6), (5, 1, 1, 2, 2), (4, 2, 1, 513, 512), (130, 40, 8, 128, 64), (70, 3, 2, 8, 8), (41, 2, 1, 16, 16), (12, 2, 2, 32, 32),
    (6, 64, 8, 128, 128), (5, 2, 1, 1024, 1024), (2000, 1, 0, 64, 64), (300, 0, 3, 64, 64)])
def test_qk_norm_rope_vs_formula(T, Hq, Hkv, D, rot, interleaved, dtype):
    q, k = make(T, Hq, D, dtype, 1), make(T, Hkv, D, dtype, 2)
    wq, wk = make(1, 1, D, dtype, 3).view(D), make(1, 1, D, dtype, 4).view(D)
    pos = (torch.arange(T, device=dev) * 977) % 200003
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(q, k, qo, ko, pos if rot else None, wq, wk, rotary_dim=rot or None, interleaved=interleaved)
    assert_rows(qo, exact_rows(q, wq, True, pos, rot, interleaved))
    assert_rows(ko, exact_rows(k, wk, True, pos, rot, interleaved))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,off", [(128, 0), (128, 1), (72, 0)])
def test_qk_norm_rope_in_place_on_views_of_a_fused_buffer(D, off, interleaved):
    T, Hq, Hkv = 37, 6, 2
    buf = make(T, Hq + 2 * Hkv, D + off, torch.float16, 7)          # off = 1: rows that no 16-byte vector reads
    keep = buf.clone()
    q, k = buf[:, :Hq, off:], buf[:, Hq:Hq + Hkv, off:]
    pos = torch.arange(T, device=dev) + 100000
    ops.qk_norm_rope(q, k, q, k, pos, interleaved=interleaved)
    assert_rows(q, exact_rows(keep[:, :Hq, off:], None, True, pos, D, interleaved))
    assert_rows(k, exact_rows(keep[:, Hq:Hq + Hkv, off:], None, True, pos, D, interleaved))
    assert torch.equal(buf[:, Hq + Hkv:], keep[:, Hq + Hkv:]) and torch.equal(buf[..., :off], keep[..., :off])


def test_zero_row_inf_and_empty_calls():
    q, k = make(4, 2, 64, torch.float16, 1), make(4, 1, 64, torch.float16, 2)
    q[1, 0] = 0
    q[2, 1, 3] = float("nan")
    pos = torch.arange(4, device=dev)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ops.qk_norm_rope(q, k, qo, ko, pos)
    assert bool((qo[1, 0] == 0).all()) and bool(qo[2, 1].isnan().all())
    assert bool(torch.isfinite(qo[2, 0]).all()) and bool(torch.isfinite(ko).all())
    e = torch.empty(0, 2, 64, dtype=torch.float16, device=dev)
    ops.qk_norm_rope(e, e, e, e, pos[:0])
    cache = torch.ones(2, 4, 2, 64, dtype=torch.float16, device=dev)
    ops.kv_cache_append(e, e, cache, cache.clone(), pos[:0])
    assert bool((cache == 1).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,H,D,page,rot,norm,interleaved", [
    (1, 8, 128, 16, 128, False, True), (64, 2, 64, 1, 64, True, False), (777, 3, 96, 24, 96, True, True),
    (1030, 1, 256, 64, 128, False, False), (19, 4, 128, 16, 0, False, True), (21, 2, 20, 7, 12, True, False),
    (3000, 8, 64, 128, 64, False, False)])
@pytest.mark.parametrize("heads_first", [False, True])
def test_append_vs_formula(T, H, D, page, rot, norm, interleaved, heads_first, dtype):
    k, v = make(T, H, D, dtype, 1), make(T, H, D, dtype, 2)
    v[0, 0, 0] = float("inf")
    w = make(1, 1, D, dtype, 3).view(D) if norm else None
    pages = T // page + 3
    shape = (pages, H, page, D) if heads_first else (pages, page, H, D)
    kc, vc = torch.full(shape, 7.0, dtype=dtype, device=dev), torch.full(shape, 8.0, dtype=dtype, device=dev)
    kv, vv = (c.transpose(1, 2) if heads_first else c for c in (kc, vc))        # [pages, page, H, D] views
    g = torch.Generator().manual_seed(5)
    slots = torch.randperm(pages * page, generator=g)[:T].to(dev)
    slots[T // 2] = -1
    pos = (torch.arange(T, device=dev) * 31) % 150001
    ops.kv_cache_append(k, v, kv, vv, slots, pos if rot else None, k_weight=w, rotary_dim=rot or None,
                        interleaved=interleaved, check_slots=True)
    used = slots >= 0
    rows = lambda c: c.reshape(pages * page, H, D)
    assert_rows(rows(kv)[slots[used]], exact_rows(k, w, norm, pos, rot, interleaved)[used])
    assert torch.equal(rows(vv)[slots[used]], v[used])
    rest = torch.ones(pages * page, dtype=torch.bool, device=dev)
    rest[slots[used]] = False
    assert bool((rows(kv)[rest] == 7).all()) and bool((rows(vv)[rest] == 8).all())
    assert hexb200.device_status() == 0


def test_append_outside_the_cache_stores_nothing_and_is_recorded():
    k = make(3, 2, 64, torch.float16, 1)
    kc, vc = torch.zeros(2, 4, 2, 64, dtype=torch.float16, device=dev), torch.zeros(2, 4, 2, 64, dtype=torch.float16, device=dev)
    slots = torch.tensor([8, 3, 1 << 40], device=dev)
    ops.kv_cache_append(k, k, kc, vc, slots)
    assert hexb200.device_status() == -1 and hexb200.device_status() == 0
    assert torch.equal(vc.view(8, 2, 64)[3], k[1]) and int((vc.view(8, -1) != 0).any(1).sum()) == 1
    with pytest.raises(IndexError):
        ops.kv_cache_append(k, k, kc, vc, slots, check_slots=True)
    with pytest.raises(ValueError):
        ops.kv_cache_append(k, k, kc, vc, torch.tensor([1, 2, 1], device=dev), check_slots=True)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements (views of one page spread 2^22 elements apart)."""
    D, H = 64, 1
    pool = torch.zeros((1 << 31) + (1 << 23), dtype=torch.float16, device=dev)
    kc = pool.as_strided((513, 2, H, D), (1 << 22, 4096, D, 1))
    vc = pool.as_strided((513, 2, H, D), (1 << 22, 4096, D, 1), 1024)
    k, v = make(2, H, D, torch.float16, 1), make(2, H, D, torch.float16, 2)
    ops.kv_cache_append(k, v, kc, vc, torch.tensor([1024, 1025], device=dev))
    assert torch.equal(kc[512], k) and torch.equal(vc[512], v)
    assert int((pool != 0).sum()) == int((k != 0).sum() + (v != 0).sum())


def test_another_stream_and_graph_replay():
    T, H, D = 5, 2, 128
    k, v = make(T, H, D, torch.float16, 1), make(T, H, D, torch.float16, 2)
    kc, vc = torch.zeros(4, 4, H, D, dtype=torch.float16, device=dev), torch.zeros(4, 4, H, D, dtype=torch.float16, device=dev)
    slots, pos = torch.arange(T, device=dev), torch.arange(T, device=dev)
    qo, ko = torch.empty_like(k), torch.empty_like(k)

    def step():
        ops.qk_norm_rope(k, k, qo, ko, pos)
        ops.kv_cache_append(ko, v, kc, vc, slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    kc.zero_()
    slots += 6
    pos += 1000
    graph.replay()
    rows = kc.view(-1, H, D)
    assert_rows(rows[6:6 + T], exact_rows(k, None, True, pos, D, True))
    assert bool((rows[:6] == 0).all())


def test_host_tensors_are_staged():
    k, v = make(3, 2, 64, torch.float32, 1).cpu(), make(3, 2, 64, torch.float32, 2).cpu()
    kc, vc = torch.zeros(1, 4, 2, 64), torch.zeros(1, 4, 2, 64)
    pos = torch.arange(3)
    ops.kv_cache_append(k, v, kc, vc, torch.tensor([0, 2, 3]), pos)
    assert_rows(kc.view(4, 2, 64)[[0, 2, 3]], exact_rows(k, None, False, pos, 64, True))
    qo, ko = torch.empty_like(k), torch.empty_like(v)
    ops.qk_norm_rope(k, v, qo, ko, pos)
    assert_rows(qo, exact_rows(k, None, True, pos, 64, True))
