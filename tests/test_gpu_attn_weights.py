"""Accumulated attention weights (hs_decode_step_weights, hs_attn_weights) against a plain 64-bit form."""
import numpy as np
import pytest
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import workloads as wl
from bounded_util import Cache, DEV, HALF_F32, attention, bf16_randn, decode_tolerance, f64

pytestmark = pytest.mark.gpu


def weight_tolerance(add, start, bound, D, terms):
    """fp32 all the way: a score is a sum of D exact products (each addition half a step of the partial sums, at most the
    sum of absolute terms `bound`) and three more roundings; a weight moves by twice its score's relative to itself, and
    sums of `terms` weights add half a step each.  exp2 and log2 of the hardware: within two steps."""
    score = (D + 8) * HALF_F32 * max(1.0, bound.max())
    return add * (2 * score + (terms + 16) * HALF_F32) + 2 * HALF_F32 * np.abs(start) + 1e-30


def _rows(stream, B, Hkv, T):
    stride = (T + 3) // 4 * 4 + 8
    r = wl.philox(stream)
    return torch.from_numpy(np.abs(r.standard_normal((B, Hkv, stride))).astype(np.float32)).to(DEV)


DECODE = [  # B, Hq, Hkv, D, T, lens, window, sinks, fp8, paged
    (2, 8, 2, 128, 700, (700, 351), 0, 0, False, 0),
    (3, 4, 4, 64, 900, (900, 1, 0), 0, 0, False, 0),
    (2, 16, 1, 256, 400, (400, 399), 0, 0, True, 0),
    (2, 6, 2, 128, 700, (650, 130), 129, 1, True, 64),
    (1, 32, 8, 128, 5003, (5003,), 1024, 4, False, 0),
    (64, 8, 8, 128, 300, tuple(range(237, 301)), 0, 0, False, 0),
    (2, 8, 2, 64, 600, (600, 555), 200, 5, False, 64),
]
_id = lambda c: "B%d-%d/%d-D%d-T%d-w%d-s%d-%s%s" % (c[0], c[1], c[2], c[3], c[4], c[6], c[7], "fp8" if c[8] else "int8", "-p%d" % c[9] if c[9] else "")


@pytest.mark.parametrize("case", DECODE, ids=_id)
def test_decode_weights(case):
    B, Hq, Hkv, D, T, lens, window, sinks, fp8, paged = case
    c = Cache(4000 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    q = bf16_randn(4001, B, Hq, D)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = torch.full((hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T),), 0xFF, dtype=torch.uint8, device=DEV)
    out = torch.full((B, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    w = _rows(4002, B, Hkv, T)
    start = f64(w)
    wo = torch.full_like(w, -7.0)
    call = lambda wi, wout: hb.decode_step_weights(q, None, None, *c.tensors, c.layout, seq, out, wi, wout, ws, Hkv, T, D ** -0.5,
                                                   fp8=fp8, window=window, sinks=sinks)
    call(w, wo)
    got = f64(wo)
    for b in range(B):
        n = lens[b]
        assert (got[b, :, n:] == -7.0).all()  # entries behind the sequence are left alone
        if n == 0:
            assert not out[b].float().abs().any()
            continue
        ref, add, mag, bound = attention(f64(q[b])[None], c.K[b, :n], c.V[b, :n], [n - 1], window, sinks, D ** -0.5)
        err = np.abs(got[b, :, :n] - start[b, :, :n] - add)
        assert (err <= weight_tolerance(add, start[b, :, :n] + add, bound, D, Hq // Hkv)).all(), (b, err.max())
        assert (np.abs(f64(out[b]) - ref[0]) <= decode_tolerance(ref, mag, bound)[0]).all()
    first = wo.clone()
    call(w, w)  # in place: the same bits, nothing else touched
    assert torch.equal(torch.where(first == -7.0, w, first), w)
    call(None, wo)  # from nothing
    for b in range(B):
        n = lens[b]
        total = f64(wo)[b, :, :n].sum(axis=1)
        assert np.allclose(total, Hq // Hkv if n else 0.0, rtol=1e-4)


def test_decode_weights_step_writes_its_token():
    B, Hq, Hkv, D, T = 2, 8, 2, 128, 300
    c = Cache(4100, B, Hkv, T, D)
    q, kn, vn = bf16_randn(4101, B, Hq, D), bf16_randn(4102, B, 1, Hkv, D), bf16_randn(4103, B, 1, Hkv, D)
    seq = torch.tensor([300, 129], dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    out = [torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    w = [torch.zeros(B, Hkv, T, device=DEV) for _ in range(2)]
    hb.decode_step_weights(q, kn, vn, *c.tensors, c.layout, seq, out[0], None, w[0], ws, Hkv, T, D ** -0.5)
    after = [t.clone() for t in c.tensors]
    hb.kv_quantize_int8(kn, vn, *c.tensors, c.layout, seq, -1)
    assert all(torch.equal(x, t) for x, t in zip(after, c.tensors))
    hb.decode_step_weights(q, None, None, *c.tensors, c.layout, seq, out[1], None, w[1], ws, Hkv, T, D ** -0.5)
    assert torch.equal(out[0], out[1]) and torch.equal(w[0], w[1])


PROMPT = [  # B, S, start, Hq, Hkv, D, window, sinks, fp8, paged
    (2, 300, 0, 8, 2, 128, 0, 0, False, 0),
    (1, 1, 0, 4, 4, 128, 0, 0, False, 0),
    (1, 1, 700, 6, 2, 64, 0, 0, True, 0),
    (2, 33, 1000, 8, 1, 128, 0, 0, False, 64),
    (1, 700, 100, 16, 2, 64, 0, 0, False, 0),     # columns in several segments
    (1, 257, 64, 4, 2, 256, 0, 0, True, 64),
    (1, 300, 600, 8, 2, 128, 100, 4, False, 0),
    (2, 200, 0, 8, 2, 128, 64, 70, True, 0),
    (1, 32, 4000, 32, 8, 128, 0, 0, True, 0),     # an observation window: keys in chunks
    (1, 32, 4000, 32, 8, 128, 900, 65, False, 0),
    (1, 600, 30, 10, 2, 256, 129, 1, False, 64),
]
_pid = lambda c: "B%d-S%d-at%d-%d/%d-D%d-w%d-s%d-%s%s" % (c[:8] + ("fp8" if c[8] else "int8", "-p%d" % c[9] if c[9] else ""))


@pytest.mark.parametrize("case", PROMPT, ids=_pid)
def test_prompt_weights(case):
    B, S, at, Hq, Hkv, D, window, sinks, fp8, paged = case
    T = at + S
    c = Cache(4200 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    q = bf16_randn(4201, B, S, Hq, D)
    ws = torch.full((max(256, hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T)),), 0xFF, dtype=torch.uint8, device=DEV)
    w = _rows(4202, B, Hkv, T)
    start, wo = f64(w), torch.full_like(w, -7.0)
    call = lambda wi, wout: hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, wi, wout, ws, Hkv, T, D ** -0.5, start_pos=at,
                                            fp8=fp8, window=window, sinks=sinks)
    call(w, wo)
    got = f64(wo)
    assert (got[:, :, T:] == -7.0).all()
    for b in range(B):
        _, add, _, bound = attention(f64(q[b]), c.K[b], None, at + np.arange(S), window, sinks, D ** -0.5)
        err = np.abs(got[b, :, :T] - start[b, :, :T] - add)
        assert (err <= weight_tolerance(add, start[b, :, :T] + add, bound, D, S * Hq // Hkv)).all(), (b, err.max())
    first = wo.clone()
    call(w, w)
    assert torch.equal(torch.where(first == -7.0, w, first), w)


FEW = [  # B, S, start, Hq, Hkv, D, window, sinks, fp8, paged: columns that fit one wavefront
    (2, 1, 2000, 4, 2, 64, 0, 0, False, 64),
    (1, 9, 700, 12, 2, 128, 0, 0, True, 64),
    (3, 16, 1300, 12, 3, 256, 0, 0, False, 0),
    (1, 16, 999, 8, 2, 256, 333, 70, True, 64),
    (2, 40, 900, 9, 3, 128, 65, 0, False, 0),
    (1, 64, 0, 4, 2, 64, 17, 2, False, 0),
    (1, 21, 3001, 18, 3, 128, 1000, 130, False, 64),
]


@pytest.mark.parametrize("case", FEW, ids=lambda c: "B%d-S%d-at%d-%d/%d-D%d-w%d-s%d-%s%s" % (c[:8] + ("fp8" if c[8] else "int8", "-p%d" % c[9] if c[9] else "")))
def test_prompt_weights_of_few_queries(case):
    """From nothing, from other rows and in place; the last token of the cache is never the last position."""
    B, S, at, Hq, Hkv, D, window, sinks, fp8, paged = case
    n, T = at + S, at + S + 77
    c = Cache(4250 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    q, w = bf16_randn(4251, B, S, Hq, D), _rows(4252, B, Hkv, T)
    ws = torch.full((hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T),), 0xFF, dtype=torch.uint8, device=DEV)
    ref = [attention(f64(q[b]), c.K[b, :n], None, at + np.arange(S), window, sinks, D ** -0.5)[1::2] for b in range(B)]
    inplace = w.clone()
    for win, wout in ((None, torch.full_like(w, -7.0)), (w, torch.full_like(w, -7.0)), (inplace, inplace)):
        hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, win, wout, ws, Hkv, T, D ** -0.5, start_pos=at, fp8=fp8, window=window, sinks=sinks)
        start, got = np.zeros(w.shape) if win is None else f64(w), f64(wout)
        assert (got[:, :, n:] == (start[:, :, n:] if wout is inplace else -7.0)).all()
        for b, (add, bound) in enumerate(ref):
            err = np.abs(got[b, :, :n] - start[b, :, :n] - add)
            assert (err <= weight_tolerance(add, start[b, :, :n] + add, bound, D, S * Hq // Hkv)).all(), (b, err.max())


@pytest.mark.parametrize("S,at,Hq,Hkv,D,T", [(1, 100, 4, 1, 128, 400), (7, 0, 8, 1, 64, 500), (16, 30, 8, 2, 128, 512), (3, 5, 4, 4, 256, 2000),
                                             (20, 60, 6, 1, 128, 1500)])
def test_prompt_weights_of_a_cache_with_room(S, at, Hq, Hkv, D, T):
    """Few queries, max_seq_len far behind the last one."""
    c = Cache(4350 + T, 1, Hkv, T, D)
    q = bf16_randn(4351, 1, S, Hq, D)
    n = at + S
    ws = torch.full((hb.attn_weights_workspace_bytes(1, S, Hq, Hkv, D, T),), 0xFF, dtype=torch.uint8, device=DEV)
    _, add, _, bound = attention(f64(q[0]), c.K[0, :n], None, at + np.arange(S), 0, 0, D ** -0.5)
    for fill in (0xFF, 0):  # whatever the workspace held
        ws.fill_(fill)
        wo = torch.full((1, Hkv, T), -7.0, device=DEV)
        hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, None, wo, ws, Hkv, T, D ** -0.5, start_pos=at)
        got = f64(wo)[0]
        assert (got[:, n:] == -7.0).all()
        assert (np.abs(got[:, :n] - add) <= weight_tolerance(add, add, bound, D, S * Hq // Hkv)).all()


@pytest.mark.parametrize("D,fp8", [(128, False), (64, True)])
def test_prompt_weights_at_positions(D, fp8):
    """Rows at positions of their own; queries outside [0, max_seq_len) count nothing, NaN in their place or in tokens
    nobody sees included."""
    B, S, Hq, Hkv, T = 5, 70, 8, 2, 400
    c = Cache(4300 + D, B, Hkv, T, D, fp8=fp8)
    at = np.array([330, 0, -20, 360, -100], np.int32)  # within; from the start; 20 queries early; 30 too late; all early
    q = bf16_randn(4301, B, S, Hq, D)
    pos = at[:, None] + np.arange(S)[None]
    q[torch.from_numpy((pos < 0) | (pos >= T)).to(DEV)] = float("nan")
    if not fp8:
        c.tensors[2][1, :, 70:] = float("nan")  # scales of tokens behind the second row's last query
    ws = torch.empty(hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    wo = torch.full((B, Hkv, T), -7.0, device=DEV)
    hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, None, wo, ws, Hkv, T, D ** -0.5,
                    positions=torch.from_numpy(at).to(DEV), fp8=fp8)
    got = f64(wo)
    for b in range(B):
        ok = (pos[b] >= 0) & (pos[b] < T)
        n = max(0, min(T, at[b] + S))
        assert (got[b, :, n:] == -7.0).all()
        if n == 0:
            continue
        _, add, _, bound = attention(f64(q[b])[ok], c.K[b, :n], None, pos[b][ok], 0, 0, D ** -0.5)
        err = np.abs(got[b, :, :n] - add)
        assert (err <= weight_tolerance(add, add, bound, D, S * Hq // Hkv)).all(), (b, err.max())


def test_prompt_weights_equal_decode_weights():
    """One query at the last position is a decode step."""
    B, Hq, Hkv, D, T = 2, 8, 2, 128, 900
    c = Cache(4400, B, Hkv, T, D)
    q = bf16_randn(4401, B, 1, Hq, D)
    seq = torch.full((B,), T, dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T) + hb.attn_weights_workspace_bytes(B, 1, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    w = [torch.zeros(B, Hkv, T, device=DEV) for _ in range(2)]
    out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV)
    hb.decode_step_weights(q[:, 0], None, None, *c.tensors, c.layout, seq, out, None, w[0], ws, Hkv, T, D ** -0.5, window=300, sinks=2)
    hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, None, w[1], ws, Hkv, T, D ** -0.5, start_pos=T - 1, window=300, sinks=2)
    assert torch.allclose(w[0], w[1], rtol=1e-4, atol=1e-9)
