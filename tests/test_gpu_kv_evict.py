"""Eviction (hs_kv_evict) against a plain selection, bit for bit."""
import numpy as np
import pytest
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import workloads as wl
from bounded_util import Cache, DEV, bf16_randn, keep

pytestmark = pytest.mark.gpu

CASES = [  # B, Hkv, D, T, lens, budget, sinks, recent, fp8, paged
    (2, 2, 128, 700, (700, 650), 100, 4, 30, False, 0),
    (3, 1, 64, 900, (900, 100, 0), 128, 0, 0, False, 0),
    (2, 3, 256, 333, (333, 332), 332, 16, 100, True, 0),
    (2, 2, 128, 600, (600, 64), 64, 4, 60, False, 64),      # nothing to choose: sinks + recent fill the budget
    (1, 8, 128, 9000, (9000,), 1000, 4, 100, False, 0),     # several tiles
    (2, 2, 64, 500, (499, 30), 77, 1, 3, True, 64),
    (1, 1, 128, 5, (5,), 1, 0, 0, False, 0),
    (1, 2, 128, 4200, (4200,), 4199, 1, 1, False, 0),       # one token leaves
]


def _weights(stream, B, Hkv, T, kind):
    r = wl.philox(stream)
    stride = (T + 3) // 4 * 4 + 4
    w = np.exp(2 * r.standard_normal((B, Hkv, stride))).astype(np.float32)
    if kind == "ties":
        w = np.rint(w).astype(np.float32)
    if kind == "odd":  # NaN, infinities, both zeros, negative and subnormal numbers
        pick = r.integers(0, 9, w.shape)
        for i, x in enumerate([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-42]):
            w[pick == i] = x
    if kind == "sparse":  # most tokens never seen
        w[r.random(w.shape) > 0.02] = 0
    if kind == "equal":
        w[:] = 0.25
    return w


def _check(c, c_out, w, lens, budget, sinks, recent, w_out, lens_out, kept, src):
    for b in range(c.B):
        for h in range(c.Hkv):
            want = keep(None if w is None else w[b, h], lens[b], budget, sinks, recent)
            n = len(want)
            got = kept[b, h].cpu().numpy()
            assert (got[:n] == want).all() and (got[n:] == -1).all(), (b, h)
            idx = torch.from_numpy(want).to(DEV)
            for j in range(2 if c.fp8 else 4):
                assert torch.equal(c_out.dense(j, n)[b, h], src[j][b, h][idx]), (b, h, j)
            if w_out is not None:
                row = w_out[b, h].cpu().numpy()
                assert np.array_equal(row[:n], np.zeros(n, np.float32) if w is None else w[b, h][want], equal_nan=True)
                assert not row[n:min(len(row), c.T)].any()
        assert lens_out[b].item() == min(lens[b], budget)
    if c.fp8:
        assert torch.equal(c_out.tensors[2], src[2]) and torch.equal(c_out.tensors[3], src[3])


@pytest.mark.parametrize("case", CASES, ids=lambda c: "B%d-H%d-D%d-T%d-to%d-s%d-r%d-%s%s" % (c[:4] + c[5:8] + ("fp8" if c[8] else "int8", "-p%d" % c[9] if c[9] else "")))
@pytest.mark.parametrize("kind", ["smooth", "ties", "odd", "equal", "sparse", None])
@pytest.mark.parametrize("where", ["out", "in"])
def test_evict(case, kind, where):
    B, Hkv, D, T, lens, budget, sinks, recent, fp8, paged = case
    c = Cache(5000 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    w = None if kind is None else _weights(5001, B, Hkv, T, kind)
    wd = None if kind is None else torch.from_numpy(w).to(DEV)
    src = [c.dense(j).clone() for j in range(4)]
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = torch.full((hb.kv_evict_workspace_bytes(B, Hkv, budget, T),), 0xFF, dtype=torch.uint8, device=DEV)
    kept = torch.full((B, Hkv, budget), -9, dtype=torch.int32, device=DEV)
    if where == "out":
        z = torch.zeros(B, budget, Hkv, D, dtype=torch.bfloat16, device=DEV)
        o = Cache(5002, B, Hkv, budget, D, fp8=fp8, paged=paged, k=z, v=z)
        lo, wo = torch.full((B,), -9, dtype=torch.int32, device=DEV), torch.full((B, Hkv, (budget + 3) // 4 * 4), 7.0, device=DEV)
    else:
        o, lo, wo = c, seq, (wd if wd is not None else torch.full((B, Hkv, (T + 3) // 4 * 4), 7.0, device=DEV))
    hb.kv_evict(c.tensors, c.layout, seq, wd, o.tensors, o.layout, lo, wo, ws, budget, sinks, recent, T, kept=kept, fp8=fp8)
    torch.cuda.synchronize()
    _check(c, o, w, lens, budget, sinks, recent, wo, lo, kept, src)
    if where == "out":
        assert all(torch.equal(c.dense(j), src[j]) for j in range(4))


def test_evict_within_a_pool_through_another_table():
    """Source and destination blocks of one pool."""
    B, Hkv, D, T, blk, budget = 2, 2, 128, 512, 64, 128
    c = Cache(5100, B, Hkv, T, D, paged=blk)
    src = [c.dense(j).clone() for j in range(4)]
    nb = T // blk
    for j in range(4):  # room behind the pool for the kept tokens
        t = c.tensors[j]
        c.tensors[j] = torch.cat([t, torch.zeros((B * budget // blk,) + tuple(t.shape[1:]), dtype=t.dtype, device=DEV)])
    table = (B * nb + torch.arange(B * budget // blk, device=DEV)).to(torch.int32).view(B, -1)
    o = object.__new__(Cache)
    o.__dict__.update(c.__dict__)
    o.tables, o.layout = [table, table.clone()], None
    o.layout = hb.paged_layout(Hkv, blk, D, *o.tables)
    w = _weights(5101, B, Hkv, T, "smooth")
    seq, lo = torch.tensor([512, 300], dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    ws = torch.empty(hb.kv_evict_workspace_bytes(B, Hkv, budget, T), dtype=torch.uint8, device=DEV)
    kept = torch.zeros(B, Hkv, budget, dtype=torch.int32, device=DEV)
    hb.kv_evict(c.tensors, c.layout, seq, torch.from_numpy(w).to(DEV), c.tensors, o.layout, lo, None, ws, budget, 4, 20, T, kept=kept)
    _check(c, o, w, [512, 300], budget, 4, 20, None, lo, kept, src)


def test_prompt_weights_evict_decode():
    """The operators together, as a session uses them: a prompt with its weights, an eviction, steps that keep counting,
    another eviction in place; against the same over float64 rows kept on the host."""
    from bounded_util import attention, decode_tolerance, f64
    B, Hq, Hkv, D, S, cap, budget, sinks, recent = 2, 8, 2, 128, 500, 640, 160, 4, 64
    G = Hq // Hkv
    q, k, v = bf16_randn(5200, B, S, Hq, D), bf16_randn(5201, B, S, Hkv, D), bf16_randn(5202, B, S, Hkv, D)
    z = torch.zeros(B, cap, Hkv, D, dtype=torch.bfloat16, device=DEV)
    c = Cache(5203, B, Hkv, cap, D, k=z, v=z)
    out = torch.empty_like(q)
    hb.prefill_attn(q, k, v, *c.tensors, c.layout, 0, out, D ** -0.5, window=300, sinks=sinks)
    w = torch.zeros(B, Hkv, cap, device=DEV)
    ws = torch.empty(max(hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, cap), hb.kv_evict_workspace_bytes(B, Hkv, budget, cap),
                         hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, cap)), dtype=torch.uint8, device=DEV)
    hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, None, w, ws, Hkv, cap, D ** -0.5, window=300, sinks=sinks)
    seq = torch.full((B,), S, dtype=torch.int32, device=DEV)
    for turn in range(2):
        before, wb, lens = [c.dense(j).clone() for j in range(4)], w.cpu().numpy(), seq.tolist()
        kept = torch.zeros(B, Hkv, budget, dtype=torch.int32, device=DEV)
        hb.kv_evict(c.tensors, c.layout, seq, w, c.tensors, c.layout, seq, w, ws, budget, sinks, recent, cap, kept=kept)
        _check(c, c, wb, lens, budget, sinks, recent, w, seq, kept, before)
        for step in range(20):
            seq += 1
            qn, kn, vn = (bf16_randn(5300 + 100 * turn + step, B, *s) for s in ((Hq, D), (1, Hkv, D), (1, Hkv, D)))
            o = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV)
            before_w = f64(w)
            hb.decode_step_weights(qn, kn, vn, *c.tensors, c.layout, seq, o, w, w, ws, Hkv, cap, D ** -0.5)
            n = budget + step + 1
            K, V = c.values()
            for b in range(B):
                ref, add, mag, bound = attention(f64(qn[b])[None], K[b, :n], V[b, :n], [n - 1], 0, 0, D ** -0.5)
                assert (np.abs(f64(o[b]) - ref[0]) <= decode_tolerance(ref, mag, bound)[0]).all()
                assert np.allclose(f64(w)[b, :, :n], before_w[b, :, :n] + add, rtol=1e-4, atol=1e-7)
