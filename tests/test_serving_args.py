"""CPU: the serving operators refuse what they do not compute, before anything touches a device."""
import ctypes as C

import pytest
import torch

import hexb200
from hexb200 import _lib, ops

i64 = C.c_int64


def test_qk_norm_rope_status_codes():
    lib = hexb200.load()
    st = (i64 * 8)(*([64] * 8))
    call = lambda dt=1, ptr=64, pos=64, T=4, Hq=2, Hkv=1, D=64, rot=64, theta=1e4: lib.hexb_qk_norm_rope(
        dt, ptr, ptr, ptr, ptr, pos, None, None, T, Hq, Hkv, D, st, rot, 1, theta, 1e-6, None)
    assert call(dt=6) == -2 and call(T=-1) == -1 and call(rot=66) == -1 and call(rot=3) == -1
    assert call(T=0) == 0 and call(D=0, rot=0) == 0 and call(Hq=0, Hkv=0) == 0
    assert call(ptr=None) == -1 and call(pos=None) == -1 and call(theta=0.0) == -1 and call(theta=float("nan")) == -1
    assert call(D=5000, rot=0) == -2 and call(Hq=65000, Hkv=1000) == -2


def test_kv_cache_append_status_codes():
    lib = hexb200.load()
    st = (i64 * 10)(*([64] * 10))
    call = lambda dt=1, ptr=64, slots=64, pos=64, T=4, H=2, D=64, pages=4, page=16, rot=64: lib.hexb_kv_cache_append(
        dt, ptr, ptr, ptr, ptr, slots, pos, None, T, H, D, pages, page, st, 0, rot, 1, 1e4, 1e-6, None)
    assert call(dt=0) == -2 and call(pages=-1) == -1 and call(rot=-2) == -1 and call(page=0) == -1
    assert call(T=0) == 0 and call(H=0) == 0
    assert call(ptr=None) == -1 and call(slots=None) == -1 and call(pos=None) == -1
    assert call(page=1 << 31) == -2 and call(pages=1 << 62) == -2


def desc(**kw):
    d = _lib.PagedAttentionDesc()
    for n in ("Q", "K_cache", "V_cache", "Out", "prefix_pages", "block_table", "seq_lens"):
        setattr(d, n, 4096)
    d.T, d.B, d.Hq, d.Hkv, d.D, d.num_pages, d.page_size, d.prefix_len = 4, 4, 8, 2, 64, 10, 16, 100
    d.table_width = d.table_stride = 5
    d.strides = (i64 * 10)(*([512] * 10))
    d.sm_scale = 0.125
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_paged_attention_status_codes():
    lib = hexb200.load()
    call = lambda **kw: lib.hexb_paged_attention_f16(C.byref(desc(**kw)), None, 0, None)
    assert lib.hexb_paged_attention_f16(None, None, 0, None) == -1
    for bad in (dict(T=-1), dict(Hkv=3), dict(Hkv=0), dict(page_size=0), dict(prefix_len=-1), dict(T=5), dict(Q=None),
                dict(Out=None), dict(K_cache=None), dict(prefix_pages=None), dict(block_table=None), dict(seq_lens=None),
                dict(max_q=-1), dict(table_width=-1)):
        assert call(**bad) == -1, bad
    for bad in (dict(D=60), dict(D=264), dict(prefix_len=1 << 31), dict(table_width=1 << 28), dict(T=1 << 25, B=1 << 25)):
        assert call(**bad) == -2, bad
    assert call(Q=4104) == -3 and call(V_cache=4098) == -3 and call(strides=(i64 * 10)(*([4] * 10))) == -3
    assert call(T=0, B=0) == 0 and call(Hq=0) == 0
    # the prefix and the own keys are computed apart and joined: a workspace is needed, the query says so
    assert lib.hexb_paged_attention_workspace_bytes(C.byref(desc())) >= 4 * 8 * (64 * 4 + 8)
    assert lib.hexb_paged_attention_workspace_bytes(C.byref(desc(T=0, B=0))) == 0
    assert lib.hexb_paged_attention_workspace_bytes(C.byref(desc(D=60))) == 0


def test_sizes_past_32_bits_are_refused_or_cut():
    lib, call = hexb200.load(), lambda **k: hexb200.load().hexb_paged_attention_f16(C.byref(desc(**k)), None, 0, None)
    assert call(T=1 << 24, B=1 << 20, q_offsets=64, Hq=1 << 15, Hkv=1 << 15) == -2       # rows
    assert call(Hq=1 << 40, Hkv=1 << 12) == -2 and call(T=1 << 40, B=1 << 40) == -2
    # a hint of any size means no more than all tokens of the call
    need = lambda **k: lib.hexb_paged_attention_workspace_bytes(C.byref(desc(**k)))
    t = desc().T
    assert need(max_q=(1 << 63) - 1) == need(max_q=t) == need(max_q=1 << 40)


def meta(*shape, dtype=torch.float16):
    """A tensor that is refused before its data or device matter."""
    class Fake:
        def __init__(self, t):
            self.t, self.device, self.is_cuda, self.get_device = t, torch.device("cuda:0"), True, lambda: 0

        def __getattr__(self, n):
            return getattr(self.t, n)
    return Fake(torch.empty(*shape, dtype=dtype))


def test_python_checks_of_the_head_operators():
    x, pos = lambda *s, **k: meta(*s, **k), meta(4, dtype=torch.int64)
    q, k = x(4, 8, 64), x(4, 2, 64)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, x(5, 2, 64), q, x(5, 2, 64), pos)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, q, x(4, 2, 64, dtype=torch.float32), pos)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, q, k, meta(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, q, k, pos, rotary_dim=63)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, q, k, rotary_dim=64)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(q, k, q, k, pos, q_weight=meta(32))
    with pytest.raises(TypeError):
        b = lambda *s: meta(*s, dtype=torch.bfloat16)
        ops.qk_norm_rope(b(4, 8, 64), b(4, 2, 64), b(4, 8, 64), b(4, 2, 64), pos)
    cache, slots = x(3, 16, 2, 64), meta(4, dtype=torch.int64)
    with pytest.raises(ValueError):
        ops.kv_cache_append(k, k, x(3, 16, 4, 64), x(3, 16, 4, 64), slots)
    with pytest.raises(TypeError):
        ops.kv_cache_append(k, k, x(3, 16, 2, 64, dtype=torch.float32), x(3, 16, 2, 64, dtype=torch.float32), slots)
    with pytest.raises(ValueError):
        ops.kv_cache_append(k, k, cache, cache, meta(4, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.kv_cache_append(k, k, cache, cache, slots, k_weight=meta(64), k_norm=False)
    with pytest.raises(ValueError):
        ops.kv_cache_append(k, k, x(3, 0, 2, 64), x(3, 0, 2, 64), slots)


def test_python_checks_of_the_attention():
    q, cache = meta(4, 8, 64), meta(10, 16, 2, 64)
    pages, table, lens = (meta(*s, dtype=torch.int32) for s in ((7,), (4, 5), (4,)))
    call = lambda q=q, kc=cache, vc=cache, out=q, pp=pages, n=100, t=table, ln=lens, off=None, **k: \
        ops.shared_prefix_attention(q, kc, vc, out, pp, n, t, ln, off, **k)
    for bad in (dict(out=meta(4, 8, 32)), dict(kc=meta(10, 16, 3, 64), vc=meta(10, 16, 3, 64)), dict(vc=meta(9, 16, 2, 64)),
                dict(n=113), dict(n=-1), dict(pp=None), dict(pp=meta(7, dtype=torch.int64)), dict(t=None), dict(ln=None),
                dict(t=meta(3, 5, dtype=torch.int32)), dict(ln=meta(5, dtype=torch.int32)),
                dict(off=meta(4, dtype=torch.int32)), dict(off=meta(5, dtype=torch.int64)), dict(max_q=-2),
                dict(kc=meta(10, 0, 2, 64), vc=meta(10, 0, 2, 64))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(TypeError):
        call(q=meta(4, 8, 64, dtype=torch.float32), out=meta(4, 8, 64, dtype=torch.float32))


def test_sample_tokens_refusals():
    lib = hexb200.load()
    call = lambda dt=2, ptr=64, rows=4, V=100, st=100, u=64: lib.hexb_sample_tokens(
        dt, ptr, u, 64, rows, V, st, None, None, None, None, 1.0, 0, 1.0, 0.0, None)
    assert call(dt=6) == -2 and call(rows=-1) == -1 and call(V=0) == -1 and call(st=-1) == -1 and call(rows=0) == 0
    assert call(ptr=None) == -1 and call(u=None) == -1 and call(ptr=66) == -3 and call(V=1 << 29) == -2
    x, u, out = meta(4, 100), meta(4, dtype=torch.float32), meta(4, dtype=torch.int64)
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1),
                dict(min_p=2.0)):
        with pytest.raises(ValueError):
            ops.sample_tokens(x, u, out, **bad)
    with pytest.raises(ValueError):
        ops.sample_tokens(x, meta(5, dtype=torch.float32), out)
    with pytest.raises(ValueError):
        ops.sample_tokens(meta(4, 0), u, out)
    with pytest.raises(ValueError):
        ops.sample_tokens(meta(400), u, out)
    with pytest.raises(TypeError):
        ops.sample_tokens(x, u, meta(4, dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.sample_tokens(meta(4, 100, dtype=torch.bfloat16), u, out)
