"""What a bounded cache needs, as a program around it calls it: in HIP graphs, on streams of its own, over long rows and
strides, and through the LayerKVCache mirror."""
import numpy as np
import pytest
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import kv_cache as kc
from hyprstream_amd import workloads as wl
from bounded_util import Cache, DEV, attention, bf16_randn, decode_tolerance, f64, keep
from test_gpu_attn_weights import weight_tolerance
from test_gpu_graph import _capture
from test_gpu_kv_evict import _check, _weights

pytestmark = pytest.mark.gpu


def _space(n):
    return torch.full((max(256, n),), 0xFF, dtype=torch.uint8, device=DEV)


class Op:
    """One call over inputs of its own: run() enqueues it, outputs() are the tensors it writes, poison() spoils them and the
    workspace, restore() puts back what an in-place call consumed."""

    def __init__(self, name, seed=6000):
        self.saved = []
        name, _, variant = name.partition("-")
        getattr(self, name)(variant, seed)
        self.saved = [(t, t.clone()) for t in self.inout]

    def restore(self):
        for t, s in self.saved:
            t.copy_(s)

    def poison(self):
        for t in self.outs:
            t.fill_(float("nan") if t.is_floating_point() else 77)
        self.ws.fill_(0xFF)
        self.restore()

    def window(self, variant, seed):
        B, Hq, Hkv, D, T = (1, 8, 2, 128, 9000) if variant == "split" else (64, 8, 8, 64, 600)
        c = Cache(seed, B, Hkv, T, D, fp8=variant != "split", paged=0 if variant == "split" else 64)
        q, seq = bf16_randn(seed + 1, B, Hq, D), torch.arange(T - B + 1, T + 1, dtype=torch.int32, device=DEV)
        out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV)
        self.ws, self.outs, self.inout = _space(hb.decode_workspace_bytes(B, Hq, Hkv, D, T)), [out], []
        w = 4096 if variant == "split" else 300
        self.run = lambda: hb.decode_attn(q, *c.tensors, c.layout, seq, out, self.ws, Hkv, T, 0.09, fp8=c.fp8, window=w, sinks=4)

    def prefill(self, variant, seed):
        B, S, Hq, Hkv, D, H = 2, 200, 8, 2, 128, 300
        c = Cache(seed, B, Hkv, H + S, D)
        q, k, v = bf16_randn(seed + 1, B, S, Hq, D), bf16_randn(seed + 2, B, S, Hkv, D), bf16_randn(seed + 3, B, S, Hkv, D)
        out = torch.empty(B, S, Hq, D, dtype=torch.bfloat16, device=DEV)
        self.ws, self.outs, self.inout = _space(0), [out], list(c.tensors)
        self.run = lambda: hb.prefill_attn(q, k, v, *c.tensors, c.layout, H, out, 0.09, window=130, sinks=70)

    def decode(self, variant, seed):
        B, Hq, Hkv, D, T = (1, 8, 2, 128, 5000) if variant == "split" else (64, 8, 8, 64, 400)
        c = Cache(seed, B, Hkv, T, D)
        q, kn, vn = bf16_randn(seed + 1, B, Hq, D), bf16_randn(seed + 2, B, 1, Hkv, D), bf16_randn(seed + 3, B, 1, Hkv, D)
        seq = torch.arange(T - B + 1, T + 1, dtype=torch.int32, device=DEV)
        out, w = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV), torch.from_numpy(_weights(seed, B, Hkv, T, "smooth")).to(DEV)
        self.ws, self.outs, self.inout = _space(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T)), [out], [w] + c.tensors
        self.run = lambda: hb.decode_step_weights(q, kn, vn, *c.tensors, c.layout, seq, out, w, w, self.ws, Hkv, T, 0.09)

    def prompt(self, variant, seed):
        B, S, Hq, Hkv, D, at = (1, 16, 16, 2, 128, 3000) if variant == "chunks" else (1, 600, 8, 2, 64, 40)
        T = at + S
        c = Cache(seed, B, Hkv, T, D, fp8=variant == "chunks")
        q, w = bf16_randn(seed + 1, B, S, Hq, D), torch.from_numpy(_weights(seed, B, Hkv, T, "smooth")).to(DEV)
        self.ws, self.outs, self.inout = _space(hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T)), [], [w]
        self.run = lambda: hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, w, w, self.ws, Hkv, T, 0.09, start_pos=at, fp8=c.fp8)

    def evict(self, variant, seed):
        B, Hkv, D, T = 2, 2, 128, 3000
        budget = 200 if variant == "small" else 2000
        c = Cache(seed, B, Hkv, T, D)
        w, seq = torch.from_numpy(_weights(seed + 1, B, Hkv, T, "ties")).to(DEV), torch.tensor([T, 2500], dtype=torch.int32, device=DEV)
        self.ws = _space(hb.kv_evict_workspace_bytes(B, Hkv, budget, T))
        kept = torch.zeros(B, Hkv, budget, dtype=torch.int32, device=DEV)
        if variant == "inplace":
            self.outs, self.inout = [kept], [w, seq] + c.tensors
            self.run = lambda: hb.kv_evict(c.tensors, c.layout, seq, w, c.tensors, c.layout, seq, w, self.ws, budget, 4, 100, T, kept=kept)
        else:
            z = torch.zeros(B, budget, Hkv, D, dtype=torch.bfloat16, device=DEV)
            o, lo, wo = Cache(seed, B, Hkv, budget, D, k=z, v=z), torch.zeros_like(seq), torch.zeros(B, Hkv, budget, device=DEV)
            self.outs, self.inout = [kept, lo, wo] + o.tensors, []
            self.run = lambda: hb.kv_evict(c.tensors, c.layout, seq, w, o.tensors, o.layout, lo, wo, self.ws, budget, 4, 100, T, kept=kept)


OPS = ["window-split", "window-direct", "prefill", "decode-split", "decode-direct", "prompt-chunks", "prompt-shares", "evict-small",
       "evict-large", "evict-inplace"]


@pytest.mark.parametrize("name", OPS)
def test_in_a_graph(name):
    op = Op(name)
    op.run()
    torch.cuda.synchronize()
    want = [t.clone() for t in op.outs + op.inout]
    g = _capture(op.run)
    x = torch.randn(256, 256, device=DEV)
    for i in range(4):
        op.poison()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(op.outs + op.inout, want)), "replay %d" % i
        (x @ x).sum().item()  # unrelated eager work between replays


def test_two_streams_at_once():
    """The calls on two streams, each with inputs and a workspace of its own."""
    ops = [[Op(n, 6100 + 50 * i) for n in OPS] for i in range(2)]
    wants = []
    for row in ops:
        wants.append([])
        for op in row:
            op.run()
            torch.cuda.synchronize()
            wants[-1].append([t.clone() for t in op.outs + op.inout])
            op.poison()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for pair in zip(*ops):
        for s, op in zip(streams, pair):
            with torch.cuda.stream(s):
                op.run()
    torch.cuda.synchronize()
    for row, want in zip(ops, wants):
        for op, w, name in zip(row, want, OPS):
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(op.outs + op.inout, w)), name


LONG = [  # B, Hkv, D, T, lens, budget, sinks, recent, fp8, paged
    (1, 1, 64, 70000, (70000,), 20000, 4, 128, False, 0),      # rows of several selection tiles
    (1, 2, 64, 33000, (32999,), 32900, 0, 0, True, 64),
    (2, 1, 128, 40000, (40000, 5), 64, 0, 64, False, 0),
    (300, 1, 64, 40, tuple(i % 41 for i in range(300)), 16, 1, 4, False, 0),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "B%d-T%d-to%d" % (c[0], c[3], c[5]))
@pytest.mark.parametrize("kind", ["smooth", "ties", "equal", "sparse", None])
@pytest.mark.parametrize("where", ["out", "out-lens", "in"])
def test_evict_long_rows(case, kind, where):
    B, Hkv, D, T, lens, budget, sinks, recent, fp8, paged = case
    c = Cache(6200 + T, B, Hkv, T, D, fp8=fp8, paged=paged)
    w = None if kind is None else _weights(6201, B, Hkv, T, kind)
    wd = None if kind is None else torch.from_numpy(w).to(DEV)
    src = [c.dense(j).clone() for j in range(4)]
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ws = _space(hb.kv_evict_workspace_bytes(B, Hkv, budget, T))
    kept = torch.full((B, Hkv, budget), -9, dtype=torch.int32, device=DEV)
    o, lo, wo = c, seq, wd
    if where != "in":
        z = torch.zeros(B, budget, Hkv, D, dtype=torch.bfloat16, device=DEV)
        o = Cache(6202, B, Hkv, budget, D, fp8=fp8, paged=paged, k=z, v=z)
        lo, wo = seq if where == "out-lens" else torch.zeros_like(seq), torch.full((B, Hkv, (budget + 3) // 4 * 4), 7.0, device=DEV)
    hb.kv_evict(c.tensors, c.layout, seq, wd, o.tensors, o.layout, lo, wo, ws, budget, sinks, recent, T, kept=kept, fp8=fp8)
    _check(c, o, w, lens, budget, sinks, recent, wo, lo, kept, src)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("src,dst", [(0, 64), (128, 0), (64, 128)])
@pytest.mark.parametrize("budget", [50, 700])
def test_evict_from_one_layout_to_another(fp8, src, dst, budget):
    B, Hkv, D, T, lens = 3, 2, 128, 1000, (1000, 701, 33)
    c = Cache(6250, B, Hkv, T, D, fp8=fp8, paged=src)
    w = _weights(6251, B, Hkv, T, "smooth")
    before = [c.dense(j).clone() for j in range(4)]
    z = torch.zeros(B, budget, Hkv, D, dtype=torch.bfloat16, device=DEV)
    o = Cache(6252, B, Hkv, budget, D, fp8=fp8, paged=dst, k=z, v=z)
    seq, lo = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    kept, wo = torch.zeros(B, Hkv, budget, dtype=torch.int32, device=DEV), torch.full((B, Hkv, (budget + 3) // 4 * 4), 7.0, device=DEV)
    hb.kv_evict(c.tensors, c.layout, seq, torch.from_numpy(w).to(DEV), o.tensors, o.layout, lo, wo, _space(hb.kv_evict_workspace_bytes(B, Hkv, budget, T)),
                budget, 3, 20, T, kept=kept, fp8=fp8)
    _check(c, o, w, lens, budget, 3, 20, wo, lo, kept, before)


def test_evict_of_sequences_that_share_blocks():
    """Two sequences with the same blocks in front, as after a common prompt, into blocks of their own; what lies behind
    the kept tokens there stays."""
    B, Hkv, D, T, blk, budget = 2, 2, 128, 512, 64, 100
    c = Cache(6260, B, Hkv, T, D, paged=blk)
    for t in c.tables:
        t[1, :4] = t[0, :4]
    before = [c.dense(j).clone() for j in range(4)]
    w = _weights(6261, B, Hkv, T, "smooth")
    z = torch.zeros(B, 128, Hkv, D, dtype=torch.bfloat16, device=DEV)
    o = Cache(6262, B, Hkv, 128, D, paged=blk, k=z, v=z)
    for t in o.tensors:
        t.fill_(9)
    seq, lo = torch.tensor([512, 400], dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    kept = torch.zeros(B, Hkv, budget, dtype=torch.int32, device=DEV)
    hb.kv_evict(c.tensors, c.layout, seq, torch.from_numpy(w).to(DEV), o.tensors, o.layout, lo, None, _space(hb.kv_evict_workspace_bytes(B, Hkv, budget, T)),
                budget, 4, 20, T, kept=kept)
    _check(c, o, w, [512, 400], budget, 4, 20, None, lo, kept, before)
    assert all((o.dense(j, 128)[:, :, budget:] == 9).all() for j in range(4))


@pytest.mark.parametrize("fp8", [False, True])
def test_strides_past_32_bits(fp8):
    """Sequences more than 2^31 bytes apart, weights rows more than 2^32: the same bits as over compact buffers."""
    B, Hq, Hkv, D, T, S = 2, 8, 2, 64, 500, 40
    c = Cache(6300, B, Hkv, T, D, fp8=fp8)
    gap, wgap = (1 << 31) + 4096, (1 << 30) + 64
    far = []
    for i in range(2):
        buf = torch.empty(gap + Hkv * T * D, dtype=c.tensors[i].dtype, device=DEV)
        view = torch.as_strided(buf, (B, Hkv, T, D), (gap, T * D, D, 1))
        view.copy_(c.tensors[i])
        far.append(view)
    lay = hb.contiguous_layout(Hkv, T, D)
    lay.code_stride_seq = gap
    rows = torch.empty(B, Hkv, wgap, device=DEV)
    start = torch.from_numpy(_weights(6301, B, Hkv, T, "smooth")).to(DEV)
    near = start[:, :, :T].contiguous()
    rows[:, :, :T] = near
    seq = torch.tensor([T, T - 7], dtype=torch.int32, device=DEV)
    q, qs = bf16_randn(6302, B, Hq, D), bf16_randn(6303, B, S, Hq, D)
    kn, vn = bf16_randn(6304, B, 1, Hkv, D), bf16_randn(6305, B, 1, Hkv, D)
    ws = _space(max(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T), hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T),
                    hb.kv_evict_workspace_bytes(B, Hkv, 100, T)))
    outs = [torch.empty(3, B, Hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for tensors, layout, w, out, lens in ((c.tensors, c.layout, near, outs[0], seq.clone()), (far + c.tensors[2:], lay, rows, outs[1], seq.clone())):
        if tensors is not c.tensors:
            tensors = far + [t.clone() for t in scales]
        else:
            scales = [t.clone() for t in c.tensors[2:]]
        hb.decode_attn(q, *tensors, layout, lens, out[0], ws, Hkv, T, 0.1, fp8=fp8, window=100, sinks=3)
        hb.decode_step_weights(q, kn, vn, *tensors, layout, lens, out[1], w, w, ws, Hkv, T, 0.1, fp8=fp8, window=300, sinks=70)
        hb.attn_weights(qs, tensors[0], tensors[2], layout, w, w, ws, Hkv, T, 0.1, start_pos=T - S, fp8=fp8)
        hb.kv_evict(tensors, layout, lens, w, tensors, layout, lens, w, ws, 100, 4, 10, T, fp8=fp8)
        hb.decode_attn(q, *tensors, layout, lens, out[2], ws, Hkv, T, 0.1, fp8=fp8)
        assert lens.tolist() == [100, 100]
    assert torch.equal(outs[0], outs[1]) and torch.equal(near[:, :, :100], rows[:, :, :100])
    assert all(torch.equal(c.tensors[i][:, :, :100], far[i][:, :, :100]) for i in range(2))


def test_heads_outside_sequences():
    """Buffers laid out [Hkv, B, T, D]."""
    B, Hq, Hkv, D, T, S = 3, 6, 2, 128, 300, 50
    c = Cache(6400, B, Hkv, T, D)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in c.tensors]
    lay = hb.contiguous_layout(Hkv, T, D)
    lay.code_stride_head, lay.code_stride_seq = B * T * D, T * D
    lay.scale_stride_head, lay.scale_stride_seq = turned[2].stride(1), turned[2].stride(0)
    q, qs = bf16_randn(6401, B, Hq, D), bf16_randn(6402, B, S, Hq, D)
    seq = torch.tensor([300, 222, 90], dtype=torch.int32, device=DEV)
    ws = _space(max(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T), hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T),
                    hb.kv_evict_workspace_bytes(B, Hkv, 64, T)))
    got = []
    for tensors, layout in ((c.tensors, c.layout), (turned, lay)):
        w, out, lens = torch.zeros(B, Hkv, T, device=DEV), torch.empty(2, B, Hq, D, dtype=torch.bfloat16, device=DEV), seq.clone()
        hb.decode_step_weights(q, None, None, *tensors, layout, lens, out[0], w, w, ws, Hkv, T, 0.1)
        hb.attn_weights(qs, tensors[0], tensors[2], layout, w, w, ws, Hkv, T, 0.1, positions=seq - S, window=64, sinks=5)
        hb.kv_evict(tensors, layout, lens, w, tensors, layout, lens, w, ws, 64, 4, 10, T)
        hb.decode_attn(q, *tensors, layout, lens, out[1], ws, Hkv, T, 0.1, window=20, sinks=4)
        got.append([w, out, lens] + [t[:, :, :64].contiguous() for t in tensors])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("D,Hq,Hkv,S,at", [(128, 6, 2, 130, 0), (64, 10, 2, 40, 700), (256, 5, 1, 65, 64), (128, 8, 8, 400, 10)])
def test_prompt_weights_of_uneven_queries(D, Hq, Hkv, S, at):
    """Queries of very different sizes beside each other and elements of very different sizes in one query: rows that are
    almost uniform next to rows that see a single token."""
    B, T = 1, at + S
    c = Cache(6500 + D, B, Hkv, T, D)
    r = wl.philox(6501)
    q = bf16_randn(6502, B, S, Hq, D).float()
    q *= torch.from_numpy(np.exp2(r.integers(-12, 6, (B, S, Hq, 1))).astype(np.float32)).to(DEV)
    q *= torch.from_numpy(np.exp2(r.integers(-9, 1, (B, S, Hq, D))).astype(np.float32)).to(DEV)
    q[:, ::7, 0] = 0
    q = q.to(torch.bfloat16)
    ws = _space(hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T))
    w = torch.full((B, Hkv, (T + 3) // 4 * 4), -7.0, device=DEV)
    hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, None, w, ws, Hkv, T, D ** -0.5, start_pos=at)
    _, add, _, bound = attention(f64(q[0]), c.K[0], None, at + np.arange(S), 0, 0, D ** -0.5)
    err = np.abs(f64(w)[0, :, :T] - add)
    assert (err <= weight_tolerance(add, add, bound, D, S * Hq // Hkv)).all(), err.max()


@pytest.mark.parametrize("quant", [kc.INT8, kc.FP8])
@pytest.mark.parametrize("window,sinks,scratch", [(0, 0, 0), (96, 3, 0), (96, 3, 512)])
def test_mirror_follows_the_calls(quant, window, sinks, scratch):
    """A session through LayerKVCache against the same calls on buffers of the test's own, bit for bit: prompt, steps,
    eviction, a truncation, a chunk behind it."""
    B, Hq, Hkv, D, cap, fp8 = 2, 8, 2, 128, 512, quant == kc.FP8
    scale = D ** -0.5
    cache = kc.LayerKVCache(cap, quant)
    cache.set_window(window, sinks)
    cache.track_weights()
    if scratch:
        cache.enable_prompt_scratch(scratch)  # (a windowed prompt reads the codes and is not split: the same bits)
    c = Cache(6600, B, Hkv, cap, D, fp8=fp8)
    w = torch.zeros(B, Hkv, cap, device=DEV)
    n = 0
    ws = _space(max(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, cap), hb.attn_weights_workspace_bytes(B, 300, Hq, Hkv, D, cap),
                    hb.kv_evict_workspace_bytes(B, Hkv, 200, cap)))
    seed = [6601]

    def rnd(*s):
        seed[0] += 1
        return bf16_randn(seed[0], *s)

    def lens():
        return torch.full((B,), n, dtype=torch.int32, device=DEV)

    def same(a=None, b=None):
        assert a is None or torch.equal(a, b)
        assert cache.seq_pos == n and torch.equal(cache.weights(), w[:, :, :n])

    def chunk(S, at):
        nonlocal n
        q, k, v = rnd(B, S, Hq, D), rnd(B, S, Hkv, D), rnd(B, S, Hkv, D)
        got, want = cache.prefill(q, k, v, at, scale), torch.empty_like(q)
        if fp8 and at == 0:
            hb.kv_fp8_calibrate(k, v, *c.tensors[2:])
        hb.prefill_attn(q, k, v, *c.tensors, c.layout, at, want, scale, fp8=fp8, window=window, sinks=sinks)
        n = at + S
        w[:, :, at:] = 0
        hb.attn_weights(q, c.tensors[0], c.tensors[2], c.layout, w, w, ws, Hkv, n, scale, start_pos=at, fp8=fp8, window=window, sinks=sinks)
        same(got, want)

    def step(new=True):
        nonlocal n
        q, want = rnd(B, Hq, D), torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV)
        k, v = (rnd(B, 1, Hkv, D), rnd(B, 1, Hkv, D)) if new else (None, None)
        got = cache.decode_step(q, k, v, scale) if new else cache.decode_attention(q, scale)
        n += new
        hb.decode_step_weights(q, k, v, *c.tensors, c.layout, lens(), want, w, w, ws, Hkv, n, scale, fp8=fp8, window=window, sinks=sinks)
        same(got, want)

    def evict(budget, sinks, recent):
        nonlocal n
        cache.evict(budget, sinks, recent)
        if budget < n:
            l = lens()
            hb.kv_evict(c.tensors, c.layout, l, w, c.tensors, c.layout, l, w, ws, budget, sinks, recent, n, fp8=fp8)
            n = budget
            w[:, :, n:] = 0
        same()

    def truncate(to):
        nonlocal n
        cache.truncate_to(to)
        n = to
        w[:, :, n:] = 0
        same()

    chunk(300, 0)
    chunk(70, 300)
    step(), step(False), step()
    evict(200, 4, 50)
    evict(200, 4, 50)  # nothing to leave out
    step(), step()
    truncate(150)
    step()
    chunk(33, 151)
    evict(100, 0, 0)
    step()
    chunk(20, 60)  # again from the middle
    step()
    k, v = cache.get(torch.float32)
    K, V = c.values()
    assert np.array_equal(f64(k), K[:, :n].astype(np.float32)) and np.array_equal(f64(v), V[:, :n].astype(np.float32))
    cache.track_weights(False)
    with pytest.raises(kc.CacheError, match="no weights"):
        cache.weights()
    q = rnd(B, Hq, D)  # without counting: the plain windowed step
    want = torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV)
    dws = _space(hb.decode_workspace_bytes(B, Hq, Hkv, D, cap))
    hb.decode_attn(q, *c.tensors, c.layout, lens(), want, dws, Hkv, n, scale, fp8=fp8, window=window, sinks=sinks)
    assert torch.equal(cache.decode_attention(q, scale), want)
    cache.evict(40, 8, 0)  # nothing counted: the first 8 and the newest
    k2, _ = cache.get(torch.float32)
    assert torch.equal(k2, torch.cat([k[:, :8], k[:, n - 32:]], dim=1))


def test_mirror_bounds_an_endless_session():
    """A cache of 160 tokens serves 500 steps; attention stays the 64-bit one over the tokens that are left."""
    B, Hq, Hkv, D, cap = 1, 4, 2, 64, 160
    cache = kc.LayerKVCache(cap)
    cache.track_weights()
    cache.prefill(bf16_randn(6700, B, 100, Hq, D), bf16_randn(6701, B, 100, Hkv, D), bf16_randn(6702, B, 100, Hkv, D), 0, D ** -0.5)
    qs, ks, vs = bf16_randn(6703, 500, B, Hq, D), bf16_randn(6704, 500, B, 1, Hkv, D), bf16_randn(6705, 500, B, 1, Hkv, D)
    for i in range(500):
        if cache.seq_pos == cap:
            before, w = [t.clone() for t in cache.get(torch.float32)], cache.weights()
            cache.evict(128, 4, 32)
            after = cache.get(torch.float32)
            for h in range(Hkv):
                idx = torch.from_numpy(keep(w[0, h].cpu().numpy(), cap, 128, 4, 32)).to(DEV)
                assert all(torch.equal(a[0, :, h], b[0, idx, h]) for a, b in zip(after, before))
        out = cache.decode_step(qs[i], ks[i], vs[i], D ** -0.5)
        if i % 50 == 49:
            K, V = (f64(t)[0] for t in cache.get(torch.float32))
            ref, _, mag, bound = attention(f64(qs[i][0])[None], K, V, [cache.seq_pos - 1], 0, 0, D ** -0.5)
            assert (np.abs(f64(out[0]) - ref[0]) <= decode_tolerance(ref, mag, bound)[0]).all()


@pytest.mark.parametrize("quant", [kc.INT8, kc.FP8])
@pytest.mark.parametrize("counted", [False, True])
def test_paged_mirror_gives_blocks_back(quant, counted):
    """Eviction through a paged cache: the tokens that stay are the right ones, their blocks too, the others are free, and
    another cache of the pool keeps what it holds."""
    H, D, n = 2, 64, 1100
    pool = kc.BlockPool(24, H, D, quant)
    one, two = kc.PagedLayerKVCache(2048, pool, "one"), kc.PagedLayerKVCache(2048, pool, "two")
    k, v = bf16_randn(6750, 1, n, H, D), bf16_randn(6751, 1, n, H, D)
    two.update(k[:, :300], v[:, :300], 0)
    one.update(k, v, 0)
    other, before = [t.clone() for t in two.get(torch.float32)], [t.clone() for t in one.get(torch.float32)]
    w = _weights(6752, 1, H, n, "smooth")[0] if counted else None
    wd = torch.from_numpy(w).to(DEV) if counted else None
    assert one.num_blocks == 5
    one.evict(300, 4, 100, weights=wd)
    assert one.seq_pos == 300 and one.num_blocks == 2 and pool.used_blocks() == 8
    want = [keep(None if w is None else w[h], n, 300, 4, 100) for h in range(H)]
    after = one.get(torch.float32)
    for h in range(H):
        idx = torch.from_numpy(want[h]).to(DEV)
        assert all(torch.equal(a[0, :, h], b[0, idx, h]) for a, b in zip(after, before))
        assert w is None or np.array_equal(wd[h, :300].cpu().numpy(), w[h][want[h]])
    assert all(torch.equal(a, b) for a, b in zip(two.get(torch.float32), other))
    q = bf16_randn(6753, 1, 4, D)
    out = one.decode_attention(q, D ** -0.5)
    K, V = (f64(t)[0] for t in one.get(torch.float32))
    ref, _, mag, bound = attention(f64(q), K, V, [299], 0, 0, D ** -0.5)
    assert (np.abs(f64(out) - ref) <= decode_tolerance(ref, mag, bound)).all()
    one.update(k[:, :200], v[:, :200], 300)  # into blocks taken anew
    assert one.seq_pos == 500 and all(torch.equal(a[:, :300], b) for a, b in zip(one.get(torch.float32), after))
    one.evict(600)
    assert one.seq_pos == 500
    for bad in ((0, 0, 0), (8, 5, 4), (8, -1, 0)):
        with pytest.raises(kc.CacheError, match="sinks"):
            one.evict(*bad)
    with pytest.raises(kc.CacheError, match="weights_stride"):
        one.evict(8, weights=torch.zeros(H, 400, device=DEV))
    one.clear()
    with pytest.raises(kc.CacheError, match="empty"):
        one.evict(8)


def test_mirror_refusals():
    cache = kc.LayerKVCache(64)
    with pytest.raises(kc.CacheError, match="empty"):
        cache.evict(8)
    for bad in ((-1, 0), (4, -1)):
        with pytest.raises(kc.CacheError, match="negative"):
            cache.set_window(*bad)
    k = bf16_randn(6800, 1, 20, 2, 64)
    cache.update(k, k, 0)
    for bad in ((0, 0, 0), (8, 5, 4), (8, -1, 0), (8, 0, -1)):
        with pytest.raises(kc.CacheError, match="sinks"):
            cache.evict(*bad)
    with pytest.raises(kc.CacheError, match="no weights"):
        cache.weights()
    cache.evict(30)
    assert cache.seq_pos == 20


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_scales_of_hidden_tokens_do_not_matter(D, bad):
    """Scales that are no numbers in tokens that the window hides: every output keeps its bits, but for prefill's.  Its
    operands are fp16 relative to a power of two that the first tokens' scales choose, hidden ones among them: without
    those it may be another power.  Then only q elements that fp16 holds as subnormals round elsewhere, by at most 2^-25
    each; history operands are below 127/4 < 2^5, so a score moves by at most D 2^-20 (log2 units), a weight by twice
    ln 2 times that relative to itself, the output by as much of the largest |v|, and bf16 may round to the neighbour."""
    B, Hq, Hkv, T, S, window, sinks = 2, 8, 2, 500, 40, 101, 5
    q, qs = bf16_randn(6900, B, Hq, D), bf16_randn(6901, B, S, Hq, D)
    kn, vn = bf16_randn(6902, B, S, Hkv, D), bf16_randn(6903, B, S, Hkv, D)
    seq = torch.full((B,), T, dtype=torch.int32, device=DEV)
    ws = _space(max(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T + S), hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T + S)))
    got = []
    for fill in (None, bad):
        c = Cache(6904, B, Hkv, T + S, D)
        outs = [torch.empty(B, Hq, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)] + [torch.empty_like(qs)]
        w = [torch.zeros(B, Hkv, T + S, device=DEV) for _ in range(2)]
        if fill is not None:  # hidden from the query at T - 1 and from every later one
            for t in c.tensors[2:]:
                t[:, :, sinks:T - window] = fill
        hb.decode_attn(q, *c.tensors, c.layout, seq, outs[0], ws, Hkv, T, 0.1, window=window, sinks=sinks)
        hb.decode_step_weights(q, None, None, *c.tensors, c.layout, seq, outs[1], None, w[0], ws, Hkv, T, 0.1, window=window, sinks=sinks)
        hb.prefill_attn(qs, kn, vn, *c.tensors, c.layout, T, outs[2], 0.1, window=window, sinks=sinks)
        hb.attn_weights(qs, c.tensors[0], c.tensors[2], c.layout, None, w[1], ws, Hkv, T + S, 0.1, start_pos=T, window=window, sinks=sinks)
        got.append(outs + w)
    for i, (a, b) in enumerate(zip(*got)):
        assert torch.isfinite(a.float()).all() and torch.isfinite(b.float()).all(), i
        if i == 2:
            x, y, vmax = f64(a), f64(b), vn.abs().max().item() + np.abs(c.V[:, :sinks]).max() + np.abs(c.V[:, T - window:T]).max()
            assert (np.abs(x - y) <= 2.0 ** -7 * np.maximum(np.abs(x), np.abs(y)) + 2 * np.log(2) * D * 2.0 ** -20 * vmax).all()
        else:
            assert torch.equal(a, b), i
