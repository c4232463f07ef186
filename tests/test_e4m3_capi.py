"""The 8-bit operators without a GPU: the entry points refuse bad arguments before they touch the
device, zero-sized work is a no-op, and the torch front end checks devices, types and shapes."""
import ctypes as C

import pytest
import torch

from fastembed_b200.capi import DTYPE, EPI

buf = C.c_void_p(4096)   # never dereferenced: every call below is refused, or has nothing to do
odd = C.c_void_p(4096 + 4)
F32, BF16 = DTYPE["f32"], DTYPE["bf16"]


def test_row_quantisers_refuse(fe_lib):
    q, n = fe_lib.fe_quantize_rows_e4m3, fe_lib.fe_add_rmsnorm_e4m3
    assert q(buf, F32, -1, 8, buf, buf, None) == 1
    assert q(buf, F32, 4, 0, buf, buf, None) == 1
    assert q(buf, 7, 4, 8, buf, buf, None) == 1
    assert q(buf, F32, 1 << 31, 8, buf, buf, None) == 4
    assert b"fe_quantize_rows_e4m3" in fe_lib.fe_last_error_message()
    for missing in range(3):
        p = [buf, buf, buf]
        p[missing] = None
        assert q(p[0], F32, 4, 8, p[1], p[2], None) == 1
    assert q(None, F32, 0, 8, None, None, None) == 0
    assert n(buf, BF16, buf, buf, 0, -1.0, 4, 8, buf, buf, None) == 1
    assert n(buf, BF16, buf, buf, 0, float("nan"), 4, 8, buf, buf, None) == 1
    assert n(buf, 3, buf, buf, 0, 1e-6, 4, 8, buf, buf, None) == 1
    assert n(buf, F32, None, buf, 0, 1e-6, 4, 8, buf, buf, None) == 1
    assert n(None, F32, None, None, 0, 1e-6, 0, 8, None, None, None) == 0


def test_linear_refuses(fe_lib):
    f = fe_lib.fe_linear_e4m3

    def call(x=buf, xs=buf, w=buf, ws=buf, b=buf, r=buf, y=buf, m=4, n=128, k=64, epi="bias", dt=BF16):
        return f(x, xs, w, ws, b, r, y, m, n, k, EPI.get(epi, epi), dt, None)

    assert call(k=24) == 1 and call(n=12) == 1 and call(m=-1) == 1 and call(k=0) == 1
    assert call(epi=9) == 1 and call(dt=2) == 1
    assert call(epi="bias_gelu", dt=F32) == 1 and call(epi="swiglu", dt=F32) == 1
    assert call(epi="bias_residual") == 1 and call(epi="bias_residual", dt=F32, r=None) == 1
    assert call(epi="swiglu", n=192) == 1
    assert call(b=None) == 1 and call(xs=None) == 1 and call(ws=None) == 1 and call(y=None) == 1
    assert call(x=odd) == 1 and call(ws=odd) == 1 and call(b=odd) == 1
    assert call(m=1 << 31) == 4
    assert call(m=0, x=None, xs=None, w=None, ws=None, b=None, y=None) == 0


def _cache_call(f, tail, **kw):
    a = dict(qkv=buf, cu=buf, batch=2, max_len=3, total=5, hq=4, hkv=2, hd=64, past=buf, table=buf, width=2, k=buf, v=buf,
             ks=buf, vs=buf, pages=4, page=32)
    a.update(kw)
    return f(a, tail)


def _append(fe_lib, **kw):
    return _cache_call(lambda a, _: fe_lib.fe_kv_cache_append_e4m3(
        a["qkv"], a["cu"], a["batch"], a["max_len"], a["total"], a["hq"], a["hkv"], a["hd"], a["past"], a["table"],
        a["width"], a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["page"], None), None, **kw)


def _attend(fe_lib, max_kv=100, scale=0.1, out=buf, ws=None, ws_bytes=0, **kw):
    return _cache_call(lambda a, _: fe_lib.fe_attention_cache_e4m3(
        a["qkv"], a["cu"], a["batch"], a["max_len"], a["total"], a["hq"], a["hkv"], a["hd"], a["past"], max_kv, a["table"],
        a["width"], a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["page"], 1, scale, out, ws, ws_bytes, None), None, **kw)


@pytest.mark.parametrize("call", [_append, _attend])
def test_cache_operators_refuse(fe_lib, call):
    assert call(fe_lib, hd=96) == 4 and call(fe_lib, page=48) == 4 and call(fe_lib, page=8) == 4
    assert call(fe_lib, hq=3) == 1 and call(fe_lib, hkv=0) == 1 and call(fe_lib, batch=-1) == 1
    assert call(fe_lib, width=-1) == 1 and call(fe_lib, pages=-1) == 1 and call(fe_lib, total=-1) == 1
    assert call(fe_lib, batch=70000) == 4 and call(fe_lib, max_len=1 << 21) == 4
    assert call(fe_lib, batch=60000, max_len=1 << 20) == 4
    for name in ("qkv", "cu", "past", "table", "k", "v", "ks", "vs"):
        assert call(fe_lib, **{name: None}) == 1, name
    for name in ("qkv", "k", "v"):
        assert call(fe_lib, **{name: odd}) == 1, name
    assert call(fe_lib, batch=0) == 0 and call(fe_lib, total=0, qkv=None) == 0 and call(fe_lib, max_len=0) == 0


def test_attention_cache_workspace(fe_lib):
    size = C.c_size_t(99)
    ask = lambda batch, max_len, total, kv, hq, hkv, hd: (
        fe_lib.fe_attention_cache_workspace_bytes(batch, max_len, total, kv, hq, hkv, hd, C.byref(size)), size.value)
    assert ask(1, 1, 1, 100, 16, 8, 128) == (0, 0)          # too short to split
    assert ask(1, 1, 1, 4000, 16, 8, 128) == (0, 0)         # eight parts or fewer meet in a cluster
    status, need = ask(1, 1, 1, 64000, 16, 8, 128)          # one token over a very long cache
    assert status == 0 and need >= 16 * 9 * 130 * 4
    assert ask(8, 2000, 16000, 3000, 16, 8, 128) == (0, 0)  # enough CTAs without
    assert ask(0, 0, 0, 0, 16, 8, 128) == (0, 0)
    assert ask(1, 1, 1, -1, 16, 8, 128)[0] == 1 and ask(1, 1, 1, 10, 16, 8, 80)[0] == 4
    assert fe_lib.fe_attention_cache_workspace_bytes(1, 1, 1, 1, 1, 1, 64, None) == 1
    assert _attend(fe_lib, max_kv=64000, batch=1, total=1, max_len=1, hd=128, hq=16, hkv=8) == 1
    assert b"workspace" in fe_lib.fe_last_error_message()
    assert _attend(fe_lib, max_kv=64000, batch=1, total=1, max_len=1, hd=128, hq=16, hkv=8, ws=buf, ws_bytes=need - 1) == 1
    assert _attend(fe_lib, max_kv=64000, batch=1, total=1, max_len=1, hd=128, hq=16, hkv=8, ws=odd, ws_bytes=need) == 1
    assert _attend(fe_lib, scale=float("inf")) == 1 and _attend(fe_lib, max_kv=-1) == 1 and _attend(fe_lib, out=None) == 1


def test_front_end_refuses_host_tensors(fe_lib):
    from fastembed_b200 import ops
    f8 = torch.zeros(4, 32, dtype=torch.uint8).view(ops.F8)
    one = torch.ones(4)
    with pytest.raises(ValueError):
        ops.quantize_rows_e4m3(torch.zeros(4, 32))
    with pytest.raises(ValueError):
        ops.quantize_rows_e4m3(torch.zeros(4, 32, dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.add_rmsnorm_e4m3(None, torch.zeros(4, 32), torch.ones(32), 1e-6)
    with pytest.raises(ValueError):
        ops.linear_e4m3(f8, one, f8, one)
    cache = ops.kv_cache_e4m3(3, 16, 2, 64, "cpu")
    assert cache.k.shape == (3, 2, 16, 64) and cache.v_scale.shape == (3, 2) and cache.k.dtype == ops.F8
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv_cache_append_e4m3(torch.zeros(1, 8 * 64, dtype=torch.bfloat16), i, 1, i[:1], i[None], cache, 4)


def test_attention_cache_rows_past_a_grid_are_refused(fe_lib):
    kw = dict(batch=1, total=5, hd=128, hkv=1)
    assert _attend(fe_lib, max_len=1 << 20, hq=9, **kw) == 4 and b"max_len" in fe_lib.fe_last_error_message()
    size = C.c_size_t(99)
    assert fe_lib.fe_attention_cache_workspace_bytes(1, 1 << 20, 5, 100, 9, 1, 128, C.byref(size)) == 4
    assert fe_lib.fe_attention_cache_workspace_bytes(1, 65535, 5, 100, 128, 1, 128, C.byref(size)) == 0


def test_row_quantisers_refuse_rows_past_their_counters(fe_lib):
    big = (1 << 30) + 8
    assert fe_lib.fe_quantize_rows_e4m3(buf, F32, 1, big, buf, buf, None) == 4
    assert fe_lib.fe_add_rmsnorm_e4m3(None, F32, buf, buf, 0, 1e-6, 1, big, buf, buf, None) == 4
    assert fe_lib.fe_quantize_rows_e4m3(None, F32, 0, 1 << 30, None, None, None) == 0
