"""Sliding windows with sinks in decode and prefill (hs_kv_layout.decode_window, prefill_window, attn_sinks) against a
plain 64-bit form.  Hidden tokens carry values a thousand times the visible ones, so one that leaks shows."""
import numpy as np
import pytest
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import workloads as wl
from bounded_util import Cache, DEV, HALF_BF16, HALF_F16, attention, bf16_randn, decode_tolerance, f64, visible

pytestmark = pytest.mark.gpu

CASES = [  # B, Hq, Hkv, D, T, lens, window, sinks, fp8, paged
    (2, 8, 2, 128, 700, (700, 351), 100, 4, False, 0),
    (2, 8, 2, 128, 700, (700, 1), 1, 0, False, 0),
    (3, 4, 4, 64, 900, (900, 64, 0), 64, 64, False, 0),
    (2, 16, 1, 256, 400, (400, 399), 33, 17, False, 0),
    (2, 6, 2, 128, 700, (650, 130), 129, 1, True, 64),
    (1, 8, 8, 64, 1500, (1500,), 512, 4, True, 64),
    (2, 8, 2, 256, 600, (600, 555), 200, 5, False, 32),
    (1, 32, 8, 128, 5000, (4999,), 1024, 4, False, 0),
    (2, 8, 2, 128, 700, (700, 200), 300, 1000, False, 0),   # more sinks than tokens: nothing is hidden
    (2, 8, 2, 128, 700, (700, 200), 5000, 3, False, 0),     # a window nobody fills
    (64, 8, 8, 128, 300, tuple(range(237, 301)), 70, 9, False, 0),  # one workgroup per (sequence, head)
]


def _outlier_cache(stream, B, Hkv, T, D, lens, window, sinks, fp8, paged):
    r = wl.philox(stream)
    k = torch.from_numpy(r.standard_normal((B, T, Hkv, D)).astype(np.float32))
    v = torch.from_numpy(r.standard_normal((B, T, Hkv, D)).astype(np.float32))
    if not fp8:  # (one scale per head: an outlier would take the visible tokens' bits)
        for b in range(B):
            hidden = ~visible([lens[b] - 1], T, window, sinks)[0]
            v[b, torch.from_numpy(hidden)] *= 1000.0
    return Cache(stream + 1, B, Hkv, T, D, fp8=fp8, paged=paged, k=k.to(torch.bfloat16).to(DEV), v=v.to(torch.bfloat16).to(DEV))


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B%d-%d/%d-D%d-T%d-w%d-s%d-%s%s" % (c[0], c[1], c[2], c[3], c[4], c[6], c[7], "fp8" if c[8] else "int8", "-p%d" % c[9] if c[9] else ""))
def test_decode_window(case):
    B, Hq, Hkv, D, T, lens, window, sinks, fp8, paged = case
    c = _outlier_cache(3000 + T + D, B, Hkv, T, D, lens, window, sinks, fp8, paged)
    q = bf16_randn(3100 + T, B, Hq, D)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = torch.full((hb.decode_workspace_bytes(B, Hq, Hkv, D, T),), 0xFF, dtype=torch.uint8, device=DEV)
    out = torch.full((B, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    hb.decode_attn(q, *c.tensors, c.layout, seq, out, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=sinks)
    torch.cuda.synchronize()
    for b in range(B):
        n = lens[b]
        if n == 0:
            assert not out[b].float().abs().any()
            continue
        ref, _, mag, bound = attention(f64(q[b])[None], c.K[b, :n], c.V[b, :n], [n - 1], window, sinks, D ** -0.5)
        err = np.abs(f64(out[b]) - ref[0])
        assert (err <= decode_tolerance(ref, mag, bound)[0]).all(), (b, err.max())


@pytest.mark.parametrize("case", [CASES[0], CASES[4], CASES[7], CASES[10]], ids=["split", "fp8-paged", "long", "direct"])
def test_decode_step_window_equals_write_then_window(case):
    """The step forms (plain, with the prologue, static) with a window give what the write and the window give."""
    B, Hq, Hkv, D, T, lens, window, sinks, fp8, paged = case
    c = Cache(3200 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    q, kn, vn = bf16_randn(3201, B, Hq, D), bf16_randn(3202, B, 1, Hkv, D), bf16_randn(3203, B, 1, Hkv, D)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.decode_workspace_bytes(B, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    new = lambda: torch.full((B, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    before = [t.clone() for t in c.tensors]
    step = new()
    hb.decode_step(q, kn, vn, *c.tensors, c.layout, seq, step, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=sinks)
    after = [t.clone() for t in c.tensors]
    for t, x in zip(c.tensors, before):
        t.copy_(x)
    (hb.kv_quantize_fp8 if fp8 else hb.kv_quantize_int8)(kn, vn, *c.tensors, c.layout, seq, -1)
    assert all(torch.equal(x, t) for x, t in zip(after, c.tensors))
    want = new()
    hb.decode_attn(q, *c.tensors, c.layout, seq, want, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=sinks)
    assert torch.equal(step, want)
    if not fp8:
        got = new()
        hb.decode_attn_static(q, *c.tensors, c.layout, seq, got, Hkv, T, D ** -0.5, window=window, sinks=sinks)
        assert torch.equal(got, want)
    rope = [torch.randn(T, D // 2, device=DEV).to(torch.bfloat16) for _ in range(2)]
    pro = hb.qk_prologue(rope_sin=rope[0], rope_cos=rope[1])
    got = new()
    hb.decode_step_prologue(q, kn, vn, pro, *c.tensors, c.layout, seq, got, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=sinks)
    qr, kr, pos = torch.empty(B, 1, Hq, D, dtype=torch.bfloat16, device=DEV), torch.empty_like(kn), seq - 1
    hb.qk_prologue_apply(q.view(B, 1, Hq, D), kn, pro, qr, kr, positions=pos)
    hb.decode_step(qr.view(B, Hq, D), kr, vn, *c.tensors, c.layout, seq, want, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=sinks)
    assert torch.equal(got, want)


def test_decode_window_two_phases_and_hint():
    """The two phases on their own, and a ragged batch's hint, which a window overrides."""
    B, Hq, Hkv, D, T = 4, 8, 2, 128, 2000
    c = Cache(3300, B, Hkv, T, D)
    q = bf16_randn(3301, B, Hq, D)
    seq = torch.tensor([2000, 17, 900, 300], dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.decode_workspace_bytes(B, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    out = [torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    args = lambda o: (q, *c.tensors, c.layout, seq, o, ws, Hkv, T, D ** -0.5)
    hb.decode_attn(*args(out[0]), window=500, sinks=7)
    c.layout.total_tokens_hint = 3217
    hb.decode_attn(*args(out[1]), window=500, sinks=7)
    hb.decode_attn(*args(out[2]), phases=1, window=500, sinks=7)
    hb.decode_attn(*args(out[2]), phases=2, window=500, sinks=7)
    assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[2])


PREFILL = [  # B, S, H, Hq, Hkv, D, window, sinks, fp8, paged
    (2, 64, 300, 8, 2, 128, 100, 4, False, 0),
    (1, 1, 500, 8, 2, 128, 70, 4, False, 0),
    (1, 200, 0, 8, 2, 128, 60, 4, False, 0),      # a prompt: the sinks are among the call's own tokens
    (2, 333, 3, 4, 4, 64, 64, 10, False, 0),      # sinks on both sides of the history's end
    (1, 100, 1000, 16, 4, 256, 150, 70, True, 64),
    (2, 130, 257, 6, 2, 128, 1, 1, True, 64),
    (1, 512, 1500, 32, 8, 128, 200, 129, False, 0),
    (1, 90, 640, 8, 1, 64, 128, 64, False, 64),
    (1, 300, 200, 8, 2, 128, 100, 5000, False, 0),  # everything is a sink
]


@pytest.mark.parametrize("case", PREFILL, ids=lambda c: "B%d-S%d-H%d-%d/%d-D%d-w%d-s%d-%s" % (c[:8] + ("fp8" if c[8] else "int8",)))
@pytest.mark.parametrize("ragged", [False, True])
def test_prefill_window(case, ragged):
    B, S, H, Hq, Hkv, D, window, sinks, fp8, paged = case
    T = H + S
    c = Cache(3400 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    q, kn, vn = bf16_randn(3401, B, S, Hq, D), bf16_randn(3402, B, S, Hkv, D), bf16_randn(3403, B, S, Hkv, D)
    hist = [H] * B
    lens = None
    if ragged:
        hist = [max(0, H - 37 * b - (H > 40) * 5) for b in range(B)]
        lens = torch.tensor(hist, dtype=torch.int32, device=DEV)
    out = torch.full((B, S, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    before = [t.clone() for t in c.tensors]
    hb.prefill_attn(q, kn, vn, *c.tensors, c.layout, H, out, D ** -0.5, quantize_on_write=False, fp8=fp8, hist_lens=lens,
                    window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert all(torch.equal(x, t) for x, t in zip(before, c.tensors))
    for b in range(B):
        K = np.concatenate([c.K[b, :hist[b]], f64(kn[b])])
        V = np.concatenate([c.V[b, :hist[b]], f64(vn[b])])
        pos = hist[b] + np.arange(S)
        ref, _, mag, bound = attention(f64(q[b]), K, V, pos, window, sinks, D ** -0.5)
        # q * scale is rounded once (bf16 in the new tokens' half, half a step) and the history's K operands once (fp16):
        # a score moves by at most (2^-8 + 2^-11) of its absolute terms, a weight by the exponential of twice that; the
        # weights themselves are rounded to bf16, the history's V operands to fp16, the output to bf16
        move = np.expm1(2 * (HALF_BF16 + HALF_F16) * bound)[..., None]
        tol = HALF_BF16 * np.abs(ref) + (HALF_BF16 + 2 * HALF_F16 + move) * mag + 1e-5
        err = np.abs(f64(out[b]) - ref)
        assert (err <= tol).all(), (b, err.max())
        # worst cases add up as above; on average roundings cancel: the mean error stays within a step of the output
        assert err.mean() <= 2 * HALF_BF16 * np.abs(ref).mean() + 1e-5, (b, err.mean())
        # the visible set itself, row by row: one-hot values would show a token that is wrongly seen or missed, so would
        # the uniform weights of equal keys, checked in test_prefill_window_counts_its_keys


@pytest.mark.parametrize("S,H,D,window,sinks", [(130, 300, 128, 100, 4), (130, 0, 128, 50, 70), (64, 129, 64, 64, 1), (70, 200, 256, 33, 65)])
def test_prefill_window_counts_its_keys(S, H, D, window, sinks):
    """Equal keys make every visible token weigh 1/n; values that are powers of two by position sum to a number that names
    the visible set (positions modulo 7, scaled by 8^-(p % 7) so that counts below 8 of any class would be exact; here the
    counts themselves are compared through seven one-hot value columns)."""
    T = H + S
    k = torch.ones(1, T, 1, D).to(torch.bfloat16).to(DEV)
    v = torch.zeros(1, T, 1, D)
    v[0, torch.arange(T), 0, torch.arange(T) % D] = 1.0  # token t lights column t % D
    v = v.to(torch.bfloat16).to(DEV)
    c = Cache(3500, 1, 1, T, D, k=k, v=v)
    q = torch.zeros(1, S, 2, D, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(1, S, 2, D, dtype=torch.bfloat16, device=DEV)
    hb.prefill_attn(q, k[:, H:].contiguous(), v[:, H:].contiguous(), *c.tensors, c.layout, H, out, 1.0, quantize_on_write=False,
                    window=window, sinks=sinks)
    see = visible(H + np.arange(S), T, window, sinks)
    n = see.sum(axis=1)
    for s in range(S):
        want = np.bincount(np.arange(T)[see[s]] % D, minlength=D)
        got = f64(out[0, s, 0]) * n[s]
        assert (np.rint(got) == want).all(), s


def test_window_off_and_sinks_change_nothing():
    """Sinks without a window are ignored, bit for bit, in both directions."""
    B, Hq, Hkv, D, T = 2, 8, 2, 128, 500
    c = Cache(3600, B, Hkv, T, D)
    q, kn, vn = bf16_randn(3601, B, 40, Hq, D), bf16_randn(3602, B, 40, Hkv, D), bf16_randn(3603, B, 40, Hkv, D)
    seq = torch.full((B,), T, dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.decode_workspace_bytes(B, Hq, Hkv, D, T), dtype=torch.uint8, device=DEV)
    o = [torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    p = [torch.empty_like(q) for _ in range(2)]
    q0 = q[:, 0].contiguous()
    for i, sinks in enumerate((0, 9)):
        hb.decode_attn(q0, *c.tensors, c.layout, seq, o[i], ws, Hkv, T, D ** -0.5, sinks=sinks)
        hb.prefill_attn(q, kn, vn, *c.tensors, c.layout, T - 40, p[i], D ** -0.5, quantize_on_write=False, sinks=sinks)
    assert torch.equal(o[0], o[1]) and torch.equal(p[0], p[1])
