"""What the entry points of a bounded cache (windows with sinks, accumulated weights, eviction) refuse, before anything
touches a GPU."""
import ctypes

import pytest

from hyprstream_amd import bindings as hb

P, Q = ctypes.c_void_p(0x100000), ctypes.c_void_p(0x900000)
F = ctypes.c_float(0.1)
BIG = ctypes.c_size_t(1 << 40)


def i64(x):
    return ctypes.c_int64(x)


def test_windows_and_sinks_are_not_negative():
    L = hb.lib()
    for field in ("decode_window", "attn_sinks"):
        lay = hb.contiguous_layout(2, 512, 128)
        setattr(lay, field, -1)
        assert L.hs_decode_attn_int8(P, P, P, P, P, ctypes.byref(lay), P, P, P, BIG, 1, 8, 2, 128, 512, F, None) == hb.HS_ERR_INVALID_ARGUMENT
        assert b"negative" in L.hs_attn_last_error()
    for field in ("prefill_window", "attn_sinks"):
        lay = hb.contiguous_layout(2, 512, 128)
        setattr(lay, field, -1)
        assert L.hs_prefill_attn_int8(P, P, P, P, P, P, P, ctypes.byref(lay), 0, Q, 1, 8, 8, 2, 128, F, 0, None) == hb.HS_ERR_INVALID_ARGUMENT
        assert L.hs_attn_weights(0, P, P, P, ctypes.byref(lay), None, 0, None, P, i64(512), P, BIG, 1, 8, 8, 2, 128, 512, F, None) == hb.HS_ERR_INVALID_ARGUMENT


def _step(lay=None, w_in=None, w=P, stride=512, ws=P, nbytes=None, B=1, Hq=8, Hkv=2, D=128, T=512, k_new=None, v_new=None, q=P):
    L = hb.lib()
    lay = lay or hb.contiguous_layout(Hkv, 512, D)
    n = L.hs_decode_weights_workspace_bytes(B, Hq, Hkv, D, T) if nbytes is None else nbytes
    return L.hs_decode_step_weights(0, q, k_new, v_new, hb.HS_BF16, P, P, P, P, ctypes.byref(lay), P, P, w_in, w, i64(stride), ws,
                                    ctypes.c_size_t(n), B, Hq, Hkv, D, T, F, None)


def test_decode_step_weights_refusals():
    assert _step(w=None) == hb.HS_ERR_INVALID_ARGUMENT
    assert _step(w=ctypes.c_void_p(0x100008)) == hb.HS_ERR_INVALID_ARGUMENT     # alignment
    assert _step(w_in=ctypes.c_void_p(0x100004)) == hb.HS_ERR_INVALID_ARGUMENT
    assert _step(stride=514) == hb.HS_ERR_INVALID_ARGUMENT                      # not a multiple of four
    assert _step(stride=508) == hb.HS_ERR_OVERFLOW
    assert _step(T=513, stride=516) == hb.HS_ERR_OVERFLOW                       # past the cache
    assert _step(k_new=P) == hb.HS_ERR_INVALID_ARGUMENT                         # K without V
    assert _step(Hq=7) == hb.HS_ERR_INVALID_ARGUMENT
    assert _step(D=96) == hb.HS_ERR_INVALID_ARGUMENT
    assert _step(q=None) == hb.HS_ERR_INVALID_ARGUMENT
    assert _step(ws=None) == hb.HS_ERR_WORKSPACE
    assert _step(ws=ctypes.c_void_p(0x100080)) == hb.HS_ERR_INVALID_ARGUMENT    # 256-byte alignment
    # the plain step's workspace is not enough: the scores pass through this one
    assert _step(nbytes=hb.decode_workspace_bytes(1, 8, 2, 128, 512)) == hb.HS_ERR_WORKSPACE
    assert _step(B=0, w=None, ws=None) == hb.HS_OK                              # an empty problem


def _weights(lay=None, q=P, w=P, stride=512, ws=P, nbytes=None, B=1, S=8, Hq=8, Hkv=2, D=128, T=512, at=0, pos=None):
    L = hb.lib()
    lay = lay or hb.contiguous_layout(Hkv, 512, D)
    n = L.hs_attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T) if nbytes is None else nbytes
    return L.hs_attn_weights(0, q, P, P, ctypes.byref(lay), pos, at, None, w, i64(stride), ws, ctypes.c_size_t(n), B, S, Hq, Hkv, D, T, F, None)


def test_attn_weights_refusals():
    assert _weights(w=None) == hb.HS_ERR_INVALID_ARGUMENT
    assert _weights(q=None) == hb.HS_ERR_INVALID_ARGUMENT
    assert _weights(q=ctypes.c_void_p(0x100002)) == hb.HS_ERR_INVALID_ARGUMENT  # alignment
    assert _weights(at=505) == hb.HS_ERR_OVERFLOW                               # 505 + 8 > 512
    assert _weights(at=-1) == hb.HS_ERR_INVALID_ARGUMENT
    assert _weights(T=513, stride=516) == hb.HS_ERR_OVERFLOW
    assert _weights(stride=256) == hb.HS_ERR_OVERFLOW
    assert _weights(Hq=9) == hb.HS_ERR_INVALID_ARGUMENT
    assert _weights(D=32) == hb.HS_ERR_INVALID_ARGUMENT
    assert _weights(ws=None) == hb.HS_ERR_WORKSPACE
    assert _weights(nbytes=16) == hb.HS_ERR_WORKSPACE
    assert _weights(ws=ctypes.c_void_p(0x100040)) == hb.HS_ERR_INVALID_ARGUMENT
    lay = hb.contiguous_layout(2, 96, 128)
    lay.k_block_table = lay.v_block_table = 0x5000000
    lay.block_table_stride = 8
    assert _weights(lay=lay) == hb.HS_ERR_INVALID_ARGUMENT                      # blocks of 96 tokens
    assert _weights(B=0) == hb.HS_OK and _weights(S=0, q=None, w=None) == hb.HS_OK


def _evict(B=1, Hkv=2, D=128, T=512, budget=64, sinks=4, recent=16, w=P, stride=512, wo=None, wo_stride=512, lay=None, lay_out=None,
           out=(0x10000000, 0x20000000, 0x30000000, 0x40000000), ws=P, nbytes=None, lens=P, src=(0x1000000, 0x2000000, 0x3000000, 0x4000000)):
    L = hb.lib()
    lay = lay or hb.contiguous_layout(Hkv, 512, D)
    lay_out = lay_out or hb.contiguous_layout(Hkv, 128, D)
    n = L.hs_kv_evict_workspace_bytes(B, Hkv, budget, T) if nbytes is None else nbytes
    return L.hs_kv_evict(0, *[ctypes.c_void_p(x) for x in src], ctypes.byref(lay), lens, w, i64(stride), *[ctypes.c_void_p(x) for x in out],
                         ctypes.byref(lay_out), P, wo, i64(wo_stride), None, budget, sinks, recent, ws, ctypes.c_size_t(n), B, Hkv, D, T, None)


def test_evict_refusals():
    assert _evict(budget=0) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(sinks=-1) == hb.HS_ERR_INVALID_ARGUMENT and _evict(recent=-1) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(sinks=50, recent=15) == hb.HS_ERR_INVALID_ARGUMENT            # more than the budget
    assert _evict(budget=2**31 - 1, sinks=2**31 - 1, recent=1) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(T=513, stride=516) == hb.HS_ERR_OVERFLOW
    assert _evict(T=0) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(budget=129) == hb.HS_ERR_OVERFLOW                             # the destination holds 128
    assert _evict(stride=256) == hb.HS_ERR_OVERFLOW
    assert _evict(stride=513) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(wo=P, wo_stride=60) == hb.HS_ERR_OVERFLOW
    assert _evict(wo=Q, wo_stride=66) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(w=P, wo=P, stride=512, wo_stride=516) == hb.HS_ERR_INVALID_ARGUMENT  # in place with two strides
    assert _evict(w=ctypes.c_void_p(0x100004)) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(ws=None) == hb.HS_ERR_WORKSPACE and _evict(nbytes=100) == hb.HS_ERR_WORKSPACE
    assert _evict(ws=ctypes.c_void_p(0x100010)) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(lens=None) == hb.HS_ERR_INVALID_ARGUMENT
    assert _evict(out=(0x10000008, 0x20000000, 0x30000000, 0x40000000)) == hb.HS_ERR_INVALID_ARGUMENT
    src = (0x1000000, 0x2000000, 0x3000000, 0x4000000)
    assert _evict(out=src) == hb.HS_ERR_INVALID_ARGUMENT                        # its own buffers with other strides
    same = hb.contiguous_layout(2, 512, 128)
    assert _evict(out=(src[0], 0x20000000, src[2], src[3]), lay_out=same) == hb.HS_ERR_INVALID_ARGUMENT  # half of it
    assert _evict(out=(src[1], src[0], src[3], src[2]), lay_out=same) == hb.HS_ERR_INVALID_ARGUMENT      # K where V was
    assert _evict(out=(0x10000000, 0x20000000, src[2], src[3])) == hb.HS_ERR_INVALID_ARGUMENT            # codes move, scales do not
    assert _evict(B=0, lens=None) == hb.HS_OK
    assert _evict(D=96) == hb.HS_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("n", [1, 63, 64, 65, 8192])
def test_workspace_sizes(n):
    L = hb.lib()
    base = hb.decode_workspace_bytes(2, 8, 2, 128, n)
    assert hb.decode_weights_workspace_bytes(2, 8, 2, 128, n) == base + 2 * 8 * ((n + 63) // 64 * 64) * 4
    assert hb.attn_weights_workspace_bytes(2, 4, 8, 2, 128, n) >= 2 * 2 * 16 * 4
    assert hb.attn_weights_workspace_bytes(2, 4, 9, 2, 128, n) == 0 and hb.attn_weights_workspace_bytes(0, 4, 8, 2, 128, n) == 0
    assert hb.kv_evict_workspace_bytes(2, 2, 10, n) >= 2 * 2 * 12 * 4 and hb.kv_evict_workspace_bytes(2, 2, 0, n) == 0
    for f, a in ((L.hs_decode_weights_workspace_bytes, (2, 8, 2, 128, n)), (L.hs_attn_weights_workspace_bytes, (1, 7, 8, 2, 64, n)),
                 (L.hs_kv_evict_workspace_bytes, (1, 3, 5, n))):
        assert f(*a) % 256 == 0
