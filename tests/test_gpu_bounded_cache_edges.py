"""Corners of a bounded cache: what the window hides, layouts and buffers that outlive a call, calls that are refused."""
import ctypes

import pytest
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import kv_cache as kc
from bounded_util import Cache, DEV, bf16_randn
from test_gpu_output_gate import _check as _check_gate, _with_gate

pytestmark = pytest.mark.gpu


def _space(n):
    return torch.full((max(256, n),), 0xFF, dtype=torch.uint8, device=DEV)


# ---- windowed prefill: the power of two its operands are relative to
HIDDEN = [  # B, S, T, Hq, Hkv, D, window, sinks, paged
    (2, 40, 500, 8, 2, 64, 101, 5, 0),
    (2, 40, 500, 8, 2, 128, 101, 5, 0),
    (2, 40, 500, 8, 2, 256, 101, 5, 0),
    (1, 40, 500, 8, 2, 128, 101, 0, 0),     # all of the first 64 tokens are hidden
    (1, 300, 700, 8, 2, 64, 70, 0, 64),     # several query tiles, the window starts anywhere in a block
    (1, 200, 333, 8, 2, 128, 129, 70, 64),  # more sinks than the reference looks at
    (1, 1, 449, 8, 2, 256, 2, 0, 64),       # one visible history token, the first of its block
]


@pytest.mark.parametrize("case", HIDDEN, ids=lambda c: "B%d-S%d-T%d-%d/%d-D%d-w%d-s%d-p%d" % c)
def test_finite_scales_of_hidden_tokens_do_not_matter(case):
    """Prefill's history operands are fp16 relative to a power of two chosen from scales: of tokens some query of the tile
    sees, so whatever the hidden ones hold, every bit of the output stays."""
    B, S, T, Hq, Hkv, D, window, sinks, paged = case
    q, kn, vn = bf16_randn(7000, B, S, Hq, D), bf16_randn(7001, B, S, Hkv, D), bf16_randn(7002, B, S, Hkv, D)
    outs = []
    for fill in (None, 1e30, 1e-30, 0.0, 2.0 ** 13, 2.0 ** -13, float("nan"), float("inf")):
        c = Cache(7003, B, Hkv, T, D, paged=paged)
        if fill is not None:  # tokens [sinks, T - window]: hidden from the query at T and from every later one
            relative = 2.0 ** -13 <= fill <= 2.0 ** 13
            for j in (2, 3):
                s = c.tensors[j]
                for b in range(B):
                    for t in range(sinks, T - window + 1):
                        at = (int(c.tables[j & 1][b, t // paged]), slice(None), t % paged) if paged else (b, slice(None), t)
                        s[at] = s[at] * fill if relative else fill
        out = torch.full((B, S, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV)
        hb.prefill_attn(q, kn, vn, *c.tensors, c.layout, T, out, D ** -0.5, quantize_on_write=False, window=window, sinks=sinks)
        outs.append(out)
        assert torch.equal(out, outs[0]), (fill, (out.float() - outs[0].float()).abs().max().item())


# ---- the mirror: its view, its buffers, calls it refuses
def _view(cache):
    """(k_codes, v_codes, k_scales, v_scales) as addresses, and the layout, of a LayerKVCache."""
    lay, p = hb.KvLayout(), [ctypes.c_void_p() for _ in range(4)]
    cache._check(kc.lib().hs_cache_get_view(cache._h, *[ctypes.byref(x) for x in p], ctypes.byref(lay), None, None, None))
    return p, lay


@pytest.mark.parametrize("early", [False, True])
def test_view_carries_the_whole_window(early):
    """The layout that a windowed cache gives out windows the calls it is handed to: prefill and the prompt's weights as
    much as decode."""
    B, S, H, Hq, Hkv, D, window, sinks = 2, 60, 200, 8, 2, 128, 50, 3
    cache = kc.LayerKVCache(H + S)
    if early:
        cache.set_window(window, sinks)
    k, v = bf16_randn(7100, B, H, Hkv, D), bf16_randn(7101, B, H, Hkv, D)
    cache.update(k, v, 0)
    if not early:
        cache.set_window(window, sinks)
    cache.track_weights()
    q, kn, vn = bf16_randn(7102, B, S, Hq, D), bf16_randn(7103, B, S, Hkv, D), bf16_randn(7104, B, S, Hkv, D)
    want = cache.prefill(q, kn, vn, H, D ** -0.5)
    p, lay = _view(cache)
    assert (lay.prefill_window, lay.decode_window, lay.attn_sinks) == (window, window, sinks)
    got, T = torch.empty_like(want), H + S
    L = hb.lib()
    hb.check(L.hs_prefill_attn_int8(q.data_ptr(), kn.data_ptr(), vn.data_ptr(), *p, ctypes.addressof(lay), H, got.data_ptr(), B, S, Hq, Hkv,
                                    D, D ** -0.5, 0, hb._stream()))
    w, ws = torch.zeros(B, Hkv, T, device=DEV), _space(hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T))
    hb.check(L.hs_attn_weights(0, q.data_ptr(), p[0], p[2], ctypes.addressof(lay), None, H, None, w.data_ptr(), T, ws.data_ptr(), ws.numel(),
                               B, S, Hq, Hkv, D, T, D ** -0.5, hb._stream()))
    assert torch.equal(got, want) and torch.equal(w, cache.weights())
    cache.set_window(0)
    _, lay = _view(cache)
    assert (lay.prefill_window, lay.decode_window, lay.attn_sinks) == (0, 0, 0)


def test_counted_prompt_allocates_once():
    """A prompt in chunks: the buffers of a counting cache are those of the first chunk, at whatever position the others
    are, and of the steps behind them.  (An unmeasured session comes first: the runtime's own memory for a kernel's first
    launch shows in the same figure.)"""
    B, S, T, Hq, Hkv, D = 1, 512, 16384, 32, 8, 128
    q, k, v = bf16_randn(7200, B, S, Hq, D), bf16_randn(7201, B, S, Hkv, D), bf16_randn(7202, B, S, Hkv, D)
    out = torch.empty_like(q)

    def session():
        cache, free = kc.LayerKVCache(T), []
        cache.track_weights()
        for at in range(0, 8192, S):
            cache._check(kc.lib().hs_cache_prefill(cache._h, hb._ptr(q), hb._ptr(k), hb._ptr(v), hb._ptr(out), B, S, Hq, Hkv, D,
                                                   ctypes.c_int64(at), ctypes.c_float(D ** -0.5), hb._stream()))
            torch.cuda.synchronize()
            free.append(torch.cuda.mem_get_info()[0])
        for _ in range(2):
            cache._check(kc.lib().hs_cache_decode_step(cache._h, hb._ptr(q), hb._ptr(k), hb._ptr(v), hb.HS_BF16, hb._ptr(out), Hq,
                                                       ctypes.c_float(D ** -0.5), hb._stream()))
            torch.cuda.synchronize()
            free.append(torch.cuda.mem_get_info()[0])
        cache.close()
        return free

    session()
    free = session()
    assert free == [free[0]] * len(free), free


def test_captured_steps_outlive_longer_prompts():
    """A counting step captured right behind a prompt (which has made the buffers) and replayed after a longer one, which
    needs more: the step's buffers are still there, and every replay adds the same weights."""
    Hq, Hkv, D, T, n = 8, 2, 128, 4096, 100
    scale = D ** -0.5
    q, k, v = bf16_randn(7250, 1, 1024, Hq, D), bf16_randn(7251, 1, 1024, Hkv, D), bf16_randn(7252, 1, 1024, Hkv, D)
    qs, ks, vs = bf16_randn(7253, 1, Hq, D), bf16_randn(7254, 1, 1, Hkv, D), bf16_randn(7255, 1, 1, Hkv, D)
    cache, plain = kc.LayerKVCache(T), kc.LayerKVCache(T)
    out = torch.empty_like(qs)
    for c in (cache, plain):
        c.track_weights()
        c.prefill(q[:, :n].contiguous(), k[:, :n], v[:, :n], 0, scale)

    def step():
        cache._check(kc.lib().hs_cache_decode_step(cache._h, hb._ptr(qs), hb._ptr(ks), hb._ptr(vs), hb.HS_BF16, hb._ptr(out), Hq,
                                                   ctypes.c_float(scale), hb._stream()))

    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        step()
    start = plain.weights()
    want = plain.decode_step(qs, ks, vs, scale)
    once = plain.weights()
    for _ in range(3):  # the same step again and again: one more time its weights for every token
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    thrice = cache.weights()
    add = once - torch.nn.functional.pad(start, (0, 1))
    assert torch.allclose(thrice, once + 2 * add, rtol=1e-5, atol=0) and (add > 0).all()
    cache.prefill(q, k, v, n + 1, scale)  # ten times as long
    cache.truncate_to(n + 1)
    before = cache.weights()
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.allclose(cache.weights(), before + add, rtol=1e-5, atol=0)


def test_captured_paged_steps_outlive_an_eviction():
    """Attention over a paged cache, captured, and replayed after an eviction and new tokens have brought the cache back to
    its length: the workspace that the eviction has outgrown is still there."""
    Hq, Hkv, D, n = 4, 2, 64, 700
    pool = kc.BlockPool(16, Hkv, D, kc.INT8)
    cache = kc.PagedLayerKVCache(65536, pool, "s")
    k, v, q = bf16_randn(7260, 1, n, Hkv, D), bf16_randn(7261, 1, n, Hkv, D), bf16_randn(7262, 1, Hq, D)
    cache.update(k, v, 0)
    first, out = cache.decode_attention(q, 0.125), torch.empty_like(q)
    torch.cuda.synchronize()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        cache._check(kc.lib().hs_paged_cache_decode_attention(cache._h, hb._ptr(q), hb._ptr(out), Hq, ctypes.c_float(0.125), hb._stream()))
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    cache.evict(300, 4, 100)
    cache.update(k[:, :400], v[:, :400], 300)
    second = cache.decode_attention(q, 0.125)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, second) and not torch.equal(out, first)


def test_refused_calls_keep_the_weights():
    """A call that is refused leaves the counted weights of the tokens it would have replaced as they are."""
    B, S, Hq, Hkv, D = 1, 100, 4, 2, 64
    cache = kc.LayerKVCache(256)
    cache.track_weights()
    q, k, v = bf16_randn(7300, B, S, Hq, D), bf16_randn(7301, B, S, Hkv, D), bf16_randn(7302, B, S, Hkv, D)
    cache.prefill(q, k, v, 0, 0.125)
    before = cache.weights()
    assert (before > 0).all()
    odd = bf16_randn(7303, B, 10, 3, D)  # three query heads over two kv-heads
    with pytest.raises(kc.CacheError):
        cache.prefill(odd, k[:, :10], v[:, :10], 40, 0.125)
    rc = kc.lib().hs_cache_update(cache._h, hb._ptr(k), hb._ptr(v), 9, B, 10, Hkv, D, ctypes.c_int64(40), hb._stream())  # no such dtype
    assert rc == hb.HS_ERR_INVALID_ARGUMENT
    rc = kc.lib().hs_cache_update(cache._h, None, hb._ptr(v), hb.HS_BF16, B, 10, Hkv, D, ctypes.c_int64(40), hb._stream())
    assert rc == hb.HS_ERR_INVALID_ARGUMENT
    assert cache.seq_pos == S and torch.equal(cache.weights(), before)
    cache.update(k[:, :10], v[:, :10], 40)  # one that is served: its tokens start without weight
    after = cache.weights()
    assert cache.seq_pos == 50 and torch.equal(after[:, :, :40], before[:, :, :40]) and not after[:, :, 40:].any()


@pytest.mark.parametrize("quant", [kc.INT8, kc.FP8])
def test_windowed_prompt_keeps_no_copy(quant):
    """The prompt scratch serves prompts without a window: a windowed one is neither copied nor split, so nothing is
    allocated or written for it."""
    B, S, Hq, Hkv, D, cap = 1, 512, 32, 8, 128, 65536
    q, k, v = bf16_randn(7400, B, S, Hq, D), bf16_randn(7401, B, S, Hkv, D), bf16_randn(7402, B, S, Hkv, D)
    cache, plain = kc.LayerKVCache(cap, quant), kc.LayerKVCache(cap, quant)
    for c in (cache, plain):
        c.set_window(300, 4)
        c.update(k[:, :64], v[:, :64], 0)  # the storage
    cache.enable_prompt_scratch(cap)
    out, ref = cache.prefill(q, k, v, 0, D ** -0.5), plain.prefill(q, k, v, 0, D ** -0.5)
    out = cache.prefill(q, k, v, 0, D ** -0.5)
    assert not cache.prompt_copy_active and torch.equal(out, ref)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    cache.drop_prompt_scratch()
    assert torch.cuda.mem_get_info()[0] == free
    assert torch.equal(cache.prefill(q, k, v, S, D ** -0.5), plain.prefill(q, k, v, S, D ** -0.5))
    cache.set_window(0)  # and without one it is begun by a prompt at position 0
    plain.set_window(0)
    cache.prefill(q, k, v, 0, D ** -0.5)
    assert cache.prompt_copy_active


# ---- the paged mirror
@pytest.mark.parametrize("quant", [kc.INT8, kc.FP8])
def test_counted_session_over_a_paged_cache(quant):
    """A counted session over a paged cache, its weights made through the view, against the contiguous mirror's own
    counting: outputs, weights and the tokens that an eviction leaves, bit for bit."""
    Hq, Hkv, D, cap, fp8 = 8, 2, 128, 1500, quant == kc.FP8
    scale = D ** -0.5
    pool = kc.BlockPool(16, Hkv, D, quant)
    paged, plain, other = kc.PagedLayerKVCache(cap, pool, "a"), kc.LayerKVCache(cap, quant), kc.PagedLayerKVCache(cap, pool, "b")
    with pytest.raises(kc.CacheError, match="empty"):
        paged.view()
    plain.track_weights()
    stride = (cap + 3) // 4 * 4
    w = torch.zeros(1, Hkv, stride, device=DEV)
    ws = _space(max(hb.attn_weights_workspace_bytes(1, 700, Hq, Hkv, D, cap), hb.decode_weights_workspace_bytes(1, Hq, Hkv, D, cap)))
    seed = [7600]

    def rnd(*s):
        seed[0] += 1
        return bf16_randn(seed[0], *s)

    def same():
        n = plain.seq_pos
        assert paged.seq_pos == n and torch.equal(w[:, :, :n], plain.weights())
        assert all(torch.equal(a, b) for a, b in zip(paged.get(torch.float32), plain.get(torch.float32)))

    def chunk(S, at):
        q, k, v = rnd(1, S, Hq, D), rnd(1, S, Hkv, D), rnd(1, S, Hkv, D)
        assert torch.equal(paged.prefill(q, k, v, at, scale), plain.prefill(q, k, v, at, scale))
        buffers, layout = paged.view()
        w[:, :, at:] = 0
        hb.attn_weights(q, buffers[0], buffers[2], layout, w, w, ws, Hkv, at + S, scale, start_pos=at, fp8=fp8)
        same()

    def step(buffers, layout):
        q, k, v = rnd(1, Hq, D), rnd(1, 1, Hkv, D), rnd(1, 1, Hkv, D)
        n, out = paged.seq_pos, torch.empty_like(q)
        paged.update(k, v, n)
        w[:, :, n] = 0
        lens = torch.full((1,), n + 1, dtype=torch.int32, device=DEV)
        hb.decode_step_weights(q, None, None, *buffers, layout, lens, out, w, w, ws, Hkv, n + 1, scale, fp8=fp8)
        assert torch.equal(out, plain.decode_step(q, k, v, scale))
        same()

    other.update(rnd(1, 10, Hkv, D), rnd(1, 10, Hkv, D), 0)  # its blocks lie between the session's
    chunk(700, 0)
    other.update(rnd(1, 300, Hkv, D), rnd(1, 300, Hkv, D), 10)
    chunk(60, 700)
    view = paged.view()
    for _ in range(12):  # over a block's end, through one view
        step(*view)
    for c in (paged, plain):
        c.evict(300, 4, 100, **({"weights": w[0]} if c is paged else {}))
    same()
    for _ in range(3):
        step(*view)
    chunk(500, paged.seq_pos)


@pytest.mark.parametrize("taker", ["update", "prefill", "batch", "pool", "clear"])
def test_blocks_of_a_queued_eviction_wait_for_it(taker):
    """An eviction is still queued behind other work of its stream when another session, on a stream of its own, is given
    the blocks behind the kept tokens: neither reads or overwrites what the other holds."""
    Hq, Hkv, D, n = 4, 2, 128, 1024
    pool = kc.BlockPool(10, Hkv, D, kc.INT8)
    one, two, ref = kc.PagedLayerKVCache(2048, pool, "one"), kc.PagedLayerKVCache(2048, pool, "two"), kc.LayerKVCache(2048)
    k, v = bf16_randn(7700, 1, n, Hkv, D), bf16_randn(7701, 1, n, Hkv, D)
    k2, v2, q2 = bf16_randn(7702, 1, 257, Hkv, D), bf16_randn(7703, 1, 257, Hkv, D), bf16_randn(7704, 1, 257, Hq, D)
    two.update(k2[:, :256], v2[:, :256], 0)
    for c in (one, ref):  # twice: the first time makes the workspaces
        c.update(k, v, 0)
        c.evict(300, 4, 100)
        c.update(k[:, 300:], v[:, 300:], 300)
    assert pool.free_block_count() == 0
    big = torch.randn(8192, 8192, device=DEV)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        for _ in range(10):
            big = big @ big * 1e-4
        one.evict(300, 4, 100)
    busy = not s1.query()
    assert pool.free_block_count() == 4
    third = kc.PagedLayerKVCache(2048, pool, "three")
    with torch.cuda.stream(s2):
        if taker == "update":
            two.update(k2[:, 256:], v2[:, 256:], 256)
        elif taker == "prefill":
            two.prefill(q2[:, 256:], k2[:, 256:], v2[:, 256:], 256, 0.1)
        elif taker == "batch":
            kc.paged_batch_decode_step(pool, [two], q2[:, 256].contiguous(), k2[:, 256:].contiguous(), v2[:, 256:].contiguous(), 0.1)
        elif taker == "pool":
            ids = [pool.allocate("raw") for _ in range(4)]
            assert s1.query() and pool.free_block_count() == 0
            for i in ids:
                pool.free("raw", i)
        else:  # taken, never used and given back: the next owner still waits
            third.update(k2[:, :1], v2[:, :1], 0)
            third.clear()
            two.update(k2[:, 256:], v2[:, 256:], 256)
        if taker not in ("batch", "pool"):
            assert busy and not s1.query()  # the host has not waited
    torch.cuda.synchronize()
    ref.evict(300, 4, 100)
    assert all(torch.equal(a, b) for a, b in zip(one.get(torch.float32), ref.get(torch.float32)))
    if taker != "pool":
        alone = kc.LayerKVCache(2048)
        alone.update(k2, v2, 0)
        assert two.seq_pos == 257 and all(torch.equal(a, b) for a, b in zip(two.get(torch.float32), alone.get(torch.float32)))


def test_capture_over_blocks_of_a_queued_eviction():
    """A step over blocks that an eviction gave back is refused under capture until a plain call has seen the eviction end."""
    Hq, Hkv, D = 4, 2, 64
    pool = kc.BlockPool(8, Hkv, D, kc.INT8)
    one, two = kc.PagedLayerKVCache(1024, pool, "one"), kc.PagedLayerKVCache(1024, pool, "two")
    k, q = bf16_randn(7760, 1, 600, Hkv, D), bf16_randn(7761, 1, Hq, D)
    two.update(k[:, :256], k[:, :256], 0)
    one.update(k, k, 0)
    one.evict(100)
    x = torch.zeros(4, device=DEV)
    torch.cuda.synchronize()

    def capture(body):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            body()
        return g

    def refused():
        with pytest.raises(kc.CacheError, match="eviction") as e:
            two.update(k[:, :1], k[:, :1], 256)
        assert e.value.code == hb.HS_ERR_BUSY
        x.add_(1)

    capture(refused).replay()
    assert two.seq_pos == 256
    two.update(k[:, :1], k[:, :1], 256)
    want, out = two.decode_attention(q, 0.125), torch.empty_like(q)
    torch.cuda.synchronize()
    g = capture(lambda: two._check(kc.lib().hs_paged_cache_decode_attention(two._h, hb._ptr(q), hb._ptr(out), Hq, ctypes.c_float(0.125), hb._stream())))
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and x[0].item() == 1


@pytest.mark.parametrize("paged", [False, True])
def test_eviction_through_the_mirrors_is_refused_under_capture(paged):
    """It moves a position and gives blocks back when it is called, tokens whenever the graph is replayed."""
    pool = kc.BlockPool(8, 2, 64, kc.INT8)
    cache = kc.PagedLayerKVCache(1024, pool, "s") if paged else kc.LayerKVCache(1024)
    k = bf16_randn(7750, 1, 600, 2, 64)
    cache.update(k, k, 0)
    before = [t.clone() for t in cache.get(torch.float32)]
    x = torch.zeros(4, device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        with pytest.raises(kc.CacheError, match="capture"):
            cache.evict(100)
        x += 1
    g.replay()
    torch.cuda.synchronize()
    assert x[0].item() == 1 and cache.seq_pos == 600 and pool.used_blocks() == (6 if paged else 0)
    assert all(torch.equal(a, b) for a, b in zip(cache.get(torch.float32), before))


@pytest.mark.parametrize("B,T,D,fp8,window", [(1, 5000, 128, False, 0), (64, 300, 64, False, 0), (2, 3000, 256, True, 700), (70, 200, 128, True, 90)])
def test_decode_weights_with_an_output_gate(B, T, D, fp8, window):
    """The gate of hs_decode_step_weights: applied once, by the attention kernel (one chunk) or by the merge beside the
    weights (split sequences), and the weights know nothing of it."""
    Hq, Hkv = 8, 8 if B >= 64 else 2
    c = Cache(7500 + T, B, Hkv, T, D, fp8=fp8)
    assert (hb.decode_num_chunks(B, Hkv, min(T, window + 300) if window else T) > 1) == (B < 64)
    q = bf16_randn(7501, B, Hq, D)
    gate = (2 * bf16_randn(7502, B, Hq, D).float()).to(torch.bfloat16)
    seq = torch.randint(1, T + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32).to(DEV)
    ws = _space(hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T))
    outs, ws_out = [], []
    for layout in (c.layout, _with_gate(c.layout, gate)):
        out, w = torch.full((B, Hq, D), float("nan"), dtype=torch.bfloat16, device=DEV), torch.zeros(B, Hkv, (T + 3) // 4 * 4, device=DEV)
        hb.decode_step_weights(q, None, None, *c.tensors, layout, seq, out, None, w, ws, Hkv, T, D ** -0.5, fp8=fp8, window=window, sinks=5)
        outs.append(out)
        ws_out.append(w)
    _check_gate(outs[1], outs[0], gate)
    assert torch.equal(*ws_out) and ws_out[0].any()
