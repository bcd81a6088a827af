"""What the decoder operators' C entry points refuse, before any device work (no GPU here)."""
import ctypes

import pytest

from iconnx_amd import _lib

BUF = ctypes.create_string_buffer(4096)
PTR = (ctypes.addressof(BUF) + 255) & ~255
BAD, SHAPE, DTYPE, WORKSPACE, UNSUPPORTED = 1, 2, 3, 4, 6
F32, F16, BF16, I8, I32, I64 = _lib.ICX_F32, _lib.ICX_F16, _lib.ICX_BF16, _lib.ICX_I8, _lib.ICX_I32, _lib.ICX_I64


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def cache(data=PTR, pages=4, page=16, heads=2, D=64, bits=4):
    return _lib.KvCacheDesc(data, pages, page, heads, D, bits)


@pytest.mark.parametrize("kw,status", [(dict(bits=3), UNSUPPORTED), (dict(D=0), UNSUPPORTED), (dict(D=48), UNSUPPORTED),
                                       (dict(D=288), UNSUPPORTED), (dict(page=0), UNSUPPORTED), (dict(page=24), UNSUPPORTED),
                                       (dict(page=1040), UNSUPPORTED), (dict(heads=0), SHAPE), (dict(pages=0), SHAPE),
                                       (dict(pages=1 << 31), SHAPE), (dict(data=PTR + 8), BAD), (dict(data=None), BAD)])
def test_caches_that_are_refused(L, kw, status):
    c = ctypes.byref(cache(**kw))
    if kw.get("data", PTR) == PTR:
        assert L.icx_kv_cache_bytes(c) == 0
    assert L.icx_kv_cache_write(None, c, ctypes.byref(_lib.KvWrite(PTR, PTR, PTR, 128, 64, 128, 64, 1, F32, I32))) == status
    assert L.icx_last_error()
    assert L.icx_kv_cache_read(None, c, PTR, I32, 1, PTR, PTR, F32) == status
    assert L.icx_kv_cache_attention(None, c, ctypes.byref(attention()), None, 0) == status


def test_cache_bytes(L):
    """A block of 32 values: its codes and a byte of scale."""
    for bits in (4, 8):
        for D in (32, 96, 256):
            assert L.icx_kv_cache_bytes(ctypes.byref(cache(None, 7, 48, 3, D, bits))) == 7 * 48 * 3 * 2 * (D * bits // 8 + D // 32)
    assert L.icx_kv_cache_bytes(None) == 0


def attention(**kw):
    a = dict(q=PTR, out=PTR, q_row_stride=256, q_head_stride=64, out_row_stride=256, out_head_stride=64, page_table=PTR, table_stride=4,
             lengths=PTR, q_starts=None, slopes=None, dtype=F32, rows=3, batch=3, q_heads=4, max_rows=1, table_width=4, scale=1.0, softcap=0.0,
             window=0, causal=1)
    a.update(kw)
    return _lib.KvAttention(**a)


@pytest.mark.parametrize("kw,status", [(dict(dtype=I8), DTYPE), (dict(q_heads=3), SHAPE), (dict(q_heads=0), SHAPE), (dict(rows=-1), SHAPE),
                                       (dict(batch=4), SHAPE), (dict(max_rows=-2), SHAPE), (dict(table_width=-1), SHAPE),
                                       (dict(table_width=1 << 27), SHAPE), (dict(softcap=-1.0), BAD), (dict(softcap=float("nan")), BAD),
                                       (dict(softcap=1e20), UNSUPPORTED), (dict(softcap=1025.0, dtype=BF16), UNSUPPORTED),
                                       (dict(softcap=1025.0, dtype=F16), UNSUPPORTED), (dict(rows=1 << 20, batch=1, q_starts=PTR, q_heads=4096), SHAPE),
                                       (dict(window=-1), BAD), (dict(q=None), BAD), (dict(out=None), BAD), (dict(lengths=None), BAD),
                                       (dict(page_table=None), BAD), (dict(table_width=1 << 20), WORKSPACE)])
def test_attention_that_is_refused(L, kw, status):
    assert L.icx_kv_cache_attention(None, ctypes.byref(cache()), ctypes.byref(attention(**kw)), None, 0) == status
    assert b"KvCacheAttention" in L.icx_last_error()


def test_attention_of_nothing_is_done_at_once(L):
    for kw in (dict(rows=0, batch=0), dict(rows=0, q_starts=PTR), dict(max_rows=0)):
        assert L.icx_kv_cache_attention(None, ctypes.byref(cache()), ctypes.byref(attention(**kw)), None, 0) == 0
    assert L.icx_kv_cache_attention(None, ctypes.byref(cache()), None, None, 0) == BAD


def test_cache_writes_and_reads_that_are_refused(L):
    c = ctypes.byref(cache())

    def write(k=PTR, v=PTR, dtype=F32, tokens=1, slots=PTR, st=I64):
        return L.icx_kv_cache_write(None, c, ctypes.byref(_lib.KvWrite(k, v, slots, 128, 64, 128, 64, tokens, dtype, st)))

    assert L.icx_kv_cache_write(None, c, None) == BAD
    assert write(dtype=I8) == DTYPE and write(st=F32) == DTYPE
    assert write(k=None) == BAD and write(v=None) == BAD and write(slots=None) == BAD
    assert write(tokens=1 << 40) == UNSUPPORTED and write(tokens=(1 << 64) - 1) == SHAPE
    assert write(tokens=0) == 0
    assert L.icx_kv_cache_read(None, c, PTR, I64, 1, PTR, PTR, I32) == DTYPE
    assert L.icx_kv_cache_read(None, c, None, I64, 1, PTR, PTR, F16) == BAD
    assert L.icx_kv_cache_read(None, c, PTR, I64, 1, None, None, F16) == 0


def test_products_that_are_refused(L):
    def run(x=PTR, xt=BF16, xs=None, M=2, K=64, N=32, w=PTR, ws=PTR, y=PTR, yt=F32, work=None, n=0, ld=None):
        args = _lib.TokenLinear(x, xs, K if ld is None else ld, M, K, N, w, ws, None, y, N, xt, yt, 0, 0)
        return L.icx_token_qlinear(None, ctypes.byref(args), work, n)

    assert L.icx_token_qlinear(None, None, None, 0) == BAD
    assert run(xt=I8, xs=PTR, K=128, x=PTR + 1) == BAD and run(xt=I8, xs=PTR, K=128, ld=130) == BAD
    assert run(xt=I8, xs=PTR, K=128, ld=(1 << 23) + 16) == SHAPE and run(xt=I8, xs=PTR, K=128, ld=-128) == SHAPE
    assert run(xt=I8, xs=PTR, K=100) == WORKSPACE  # (rows that have to be padded)

    assert run(xt=I32) == DTYPE and run(yt=I8) == DTYPE
    assert run(xs=PTR) == BAD and run(xt=I8) == BAD
    assert run(x=None) == BAD and run(w=None) == BAD and run(ws=None) == BAD and run(y=None) == BAD and run(w=PTR + 4) == BAD
    assert run(K=0) == SHAPE and run(K=131072) == SHAPE and run(M=1 << 30) == SHAPE and run(N=1 << 30) == SHAPE
    assert run(M=0) == 0 and run(N=0) == 0
    need = L.icx_token_qlinear_workspace_size(2000, 64, 32, BF16)
    assert need >= 2000 * 128 + 4 * 2000
    assert run(M=2000, work=PTR, n=need - 1) == WORKSPACE and run(M=2000, n=need) == WORKSPACE
    assert L.icx_token_weight_bytes(100, 7) == 128 * 7
    assert L.icx_pack_token_weight(None, None, 64, 32, PTR) == BAD and L.icx_pack_token_weight(None, PTR, 0, 32, PTR) == SHAPE
    assert L.icx_quantize_tokens(None, PTR, I8, 1, 64, 64, PTR, 64, PTR) == DTYPE
    assert L.icx_quantize_tokens(None, PTR, F32, 1, 0, 64, PTR, 64, PTR) == SHAPE
    assert L.icx_quantize_tokens(None, None, F32, 1, 64, 64, PTR, 64, PTR) == BAD
    assert L.icx_quantize_tokens(None, PTR, F32, 1, 64, 64, PTR, 63, PTR) == SHAPE
    assert L.icx_quantize_tokens(None, PTR, F32, 1 << 24, 2048, 2048, PTR, 2048, PTR) == UNSUPPORTED
    assert L.icx_quantize_tokens(None, PTR, F32, 1 << 26, 64, 64, PTR, 64, PTR) == UNSUPPORTED
    assert run(xt=I8, xs=PTR, K=100, M=1 << 24, work=PTR, n=1 << 40) == UNSUPPORTED
    assert L.icx_quantize_tokens(None, None, F32, 0, 64, 64, None, 64, None) == 0
