"""What a bounded KV cache needs, case by case: attention with a sliding window and sinks, accumulated attention weights,
eviction.  Every operator in its plain form (elementary torch operations) and, with `own` set, through the framework."""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BLOCK = 256  # tokens per pool block of the paged cases


def _case(op, name, **kw):
    c = dict(op=op, B=1, S=1, Hq=32, Hkv=8, D=128, T=2048, ragged=False, fp8=False, paged=False, window=0, sinks=0, budget=0, recent=0)
    c.update(kw)
    c["name"] = name
    return c


def listed():
    return [
        # one stream with a long context in a layer that sees the last 1024 tokens and four sinks: launch latency
        _case("decode", "decode-window-b1", T=32768, window=1024, sinks=4),
        # a serving batch of ragged conversations
        _case("decode", "decode-window-b64", B=64, T=8192, ragged=True, window=4096, sinks=4),
        # long contexts in a paged FP8 pool, a window that is no multiple of anything
        _case("decode", "decode-window-paged-fp8", B=32, Hq=64, T=32768, fp8=True, paged=True, window=8191, sinks=64),
        # a late chunk of four prompts
        _case("prefill", "prefill-window-b4", B=4, S=512, T=4096, window=1024, sinks=4),
        # a chunk of odd length of one prompt with 256-wide heads over a paged FP8 history
        _case("prefill", "prefill-window-d256", B=1, S=1000, Hq=16, Hkv=4, D=256, T=5999, fp8=True, paged=True, window=2000, sinks=16),
        # tracking the weights while generating: a full batch, and one long stream
        _case("decode_weights", "decode-weights-b64", B=64, T=8192),
        _case("decode_weights", "decode-weights-b1", T=32768),
        # the weights of whole prompts, before their caches are cut down
        _case("prompt_weights", "prompt-weights-b4", B=4, S=4096, T=4096),
        # the weights of the last 32 queries of a long prompt (an observation window), FP8 cache
        _case("prompt_weights", "prompt-weights-tail", S=32, T=32768, fp8=True),
        # cutting caches down: a batch, one long stream, small paged FP8 caches of different lengths
        _case("evict", "evict-b64", B=64, T=8192, budget=1024, sinks=4, recent=256),
        _case("evict", "evict-b1", T=32768, budget=4096, sinks=4, recent=1024),
        _case("evict", "evict-paged-fp8", B=5, Hkv=4, D=64, T=2500, ragged=True, fp8=True, paged=True, budget=512, sinks=4, recent=100),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "prefill", "decode_weights", "prompt_weights", "evict"])
    D = rng.choice([64, 128, 128, 256])
    Hkv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, B=1, S=1, Hq=Hkv * rng.choice([1, 2, 4, 8]), Hkv=Hkv, D=D, T=0, ragged=rng.random() < 0.5,
             fp8=rng.random() < 0.4, paged=rng.random() < 0.4, window=0, sinks=0, budget=0, recent=0)
    if op in ("decode", "decode_weights", "evict"):
        c["B"] = _log(rng, 1, 64)
        c["T"] = _log(rng, 300, 32768 if c["B"] <= 16 else 8192)
    if op in ("decode", "prefill"):
        c["window"], c["sinks"] = _log(rng, 64, 8192), rng.choice([0, 1, 4, 16, 64])
    if op == "decode_weights" and rng.random() < 0.3:
        c["window"], c["sinks"] = _log(rng, 64, 8192), 4
    if op == "prefill":
        c["B"], c["S"], c["ragged"] = _log(rng, 1, 8), _log(rng, 2, 1024), False
        c["T"] = c["S"] + _log(rng, 1, 8192)
    if op == "prompt_weights":
        c["B"], c["S"], c["ragged"] = _log(rng, 1, 4), _log(rng, 1, 2048), False
        c["T"] = c["S"] + _log(rng, 1, 8192 if c["S"] > 256 else 32768)
        if rng.random() < 0.3:
            c["window"], c["sinks"] = _log(rng, 64, 4096), 4
    if op == "evict":
        c["budget"] = max(32, min(_log(rng, 64, 4096), c["T"] - 1, 131072 // c["B"]))
        c["sinks"] = rng.choice([0, 1, 4, 16])
        c["recent"] = rng.randrange(0, c["budget"] - c["sinks"])
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _cap(c):
    return (c["T"] + BLOCK - 1) // BLOCK * BLOCK if c["paged"] else c["T"]


def _quantize(x, fp8):
    """x [B, Hkv, T, D] fp32 -> codes and fp32 scales (int8: [B, Hkv, T]; e4m3fn: [B, Hkv])."""
    if fp8:
        s = x.abs().amax(dim=(2, 3)) / 448.0
        return (x / s[:, :, None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8), s
    s = x.abs().amax(dim=3) / 127.0
    return torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8), s


def _inputs(c, seed):
    """The tensors of a case from its seed: a cache [B, Hkv, T, D] as codes and scales, queries, lengths.  Keys lean
    towards their head's mean query by a different amount each, the first ones most: a few tokens carry much of the
    weight, as they do in trained models."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, S, Hq, Hkv, D, T, fp8 = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "T", "fp8"))
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    st = {}
    lean = rnd(B, Hkv, 1, D)
    cdt = torch.uint8 if fp8 else torch.int8
    for name in ("k", "v"):
        codes = torch.empty(B, Hkv, T, D, dtype=cdt, device=DEV)
        scales = torch.empty((B, Hkv) if fp8 else (B, Hkv, T), device=DEV)
        for b in range(B):  # one sequence at a time: the fp32 source is four times the cache
            x = rnd(1, Hkv, T, D)
            if name == "k":
                pull = torch.rand(1, Hkv, T, 1, generator=g, device=DEV) ** 8
                pull[:, :, :4] = 1.5
                x = x + 0.6 * pull * lean[b:b + 1]
            codes[b:b + 1], scales[b:b + 1] = _quantize(x.to(torch.bfloat16).float(), fp8)
        st[name + "c"], st[name + "s"] = codes, scales
    if c["ragged"]:
        st["lens"] = torch.randint(max(1, T // 16), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
        st["lens"][0] = T
    else:
        st["lens"] = torch.full((B,), T, dtype=torch.int32, device=DEV)
    q = rnd(B, S, Hkv, Hq // Hkv, D) + 0.5 * lean.view(B, 1, Hkv, 1, D)
    st["q"] = q.reshape(B, S, Hq, D).to(torch.bfloat16)
    if c["op"] == "prefill":  # the chunk's own keys and values arrive in bf16
        st["kn"], st["vn"] = rnd(B, S, Hkv, D).to(torch.bfloat16), rnd(B, S, Hkv, D).to(torch.bfloat16)
    if c["op"] in ("decode_weights", "prompt_weights", "evict"):
        w = torch.exp(2.0 * rnd(B, Hkv, T) - 6.0)
        w[torch.rand(B, Hkv, T, generator=g, device=DEV) < 0.2] = 0.0  # tokens nobody has looked at
        st["w"] = w
    return st


def _store(c, st, seed):
    """The cache as the framework stores it: [B, Hkv, cap, D], or a pool of blocks behind a table."""
    B, Hkv, D, T = (c[k] for k in ("B", "Hkv", "D", "T"))
    cap, fp8 = _cap(c), c["fp8"]
    if not c["paged"]:
        pad = (-T) % 4
        for s in ("ks", "vs"):
            if not fp8 and pad:
                st[s] = torch.cat([st[s], torch.zeros(B, Hkv, pad, device=DEV)], dim=2).contiguous()
        return
    nb = cap // BLOCK
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    st["table"] = torch.randperm(B * nb, generator=g, device=DEV).to(torch.int32).view(B, nb)
    where = st["table"].long().view(-1)
    for x in ("kc", "vc") + (() if fp8 else ("ks", "vs")):
        src = st[x]
        full = torch.zeros((B, Hkv, cap) + tuple(src.shape[3:]), dtype=src.dtype, device=DEV)
        full[:, :, :T] = src
        full = full.view((B, Hkv, nb, BLOCK) + tuple(src.shape[3:])).transpose(1, 2).reshape((B * nb, Hkv, BLOCK) + tuple(src.shape[3:])).contiguous()
        pool = torch.empty_like(full)
        pool[where] = full
        st[x] = pool


def prepare(case, seed):
    c = case
    st = _inputs(c, seed)
    _store(c, st, seed)
    st["c"], st["scale"] = c, 1.0 / math.sqrt(c["D"])
    B, S, Hq, Hkv, D, T = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "T"))
    if c["op"] == "evict":
        n = c["budget"]
        for x in ("kc", "vc"):
            st[x + "o"] = torch.zeros(B, Hkv, n, D, dtype=st[x].dtype, device=DEV)
        for x in ("ks", "vs"):
            st[x + "o"] = torch.zeros((B, Hkv) if c["fp8"] else (B, Hkv, (n + 3) // 4 * 4), device=DEV)
        st["wo"] = torch.zeros(B, Hkv, (n + 3) // 4 * 4, device=DEV)
        st["lo"] = torch.zeros(B, dtype=torch.int32, device=DEV)
        st["kept"] = torch.zeros(B, Hkv, n, dtype=torch.int32, device=DEV)
    if c["op"] in ("decode_weights", "prompt_weights", "evict"):  # rows of the tracker: a multiple of four entries
        st["w"] = torch.cat([st["w"], torch.zeros(B, Hkv, (-T) % 4, device=DEV)], dim=2).contiguous()
        if c["op"] != "evict":
            st["wo"] = torch.zeros_like(st["w"])
    if own:
        from hyprstream_amd import bindings as hb
        lay = lambda: hb.paged_layout(Hkv, BLOCK, D, st["table"], st["table"]) if c["paged"] else hb.contiguous_layout(Hkv, T, D)
        st["layout"] = lay()
        size = {"decode": lambda: hb.decode_workspace_bytes(B, Hq, Hkv, D, T),
                "prefill": lambda: 0,
                "decode_weights": lambda: hb.decode_weights_workspace_bytes(B, Hq, Hkv, D, T),
                "prompt_weights": lambda: hb.attn_weights_workspace_bytes(B, S, Hq, Hkv, D, T),
                "evict": lambda: hb.kv_evict_workspace_bytes(B, Hkv, c["budget"], T)}[c["op"]]()
        st["ws"] = torch.empty(max(256, size), dtype=torch.uint8, device=DEV)
        if c["op"] == "evict":
            st["layout_out"] = hb.contiguous_layout(Hkv, c["budget"], D)
        else:
            st["out"] = torch.empty(B, S, Hq, D, dtype=torch.bfloat16, device=DEV)
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _dense(c, st, x, b):
    """codes * scale of one sequence, fp32 [Hkv, T, D]."""
    codes, scales = _rows(c, st, x + "c", b), st[x + "s"][b] if c["fp8"] else _rows(c, st, x + "s", b)
    if c["fp8"]:
        return codes.view(torch.float8_e4m3fn).float() * scales[:, None, None]
    return codes.float() * scales[..., None]


def _rows(c, st, x, b):
    """One sequence's codes [Hkv, T, D] or token scales [Hkv, T]."""
    if c["paged"]:
        t = st[x][st["table"][b].long()].transpose(0, 1)
        return t.reshape((c["Hkv"], -1) + tuple(t.shape[3:]))[:, :c["T"]]
    return st[x][b][:, :c["T"]]


def _visible(c, pos, keys):
    """[queries, keys] truth values: the key is not after the query and inside the window or one of the sinks."""
    ok = keys[None, :] <= pos[:, None]
    if c["window"]:
        ok = ok & ((keys[None, :] > pos[:, None] - c["window"]) | (keys[None, :] < c["sinks"]))
    return ok


def _weights_of(c, st, q, k, pos, keys):
    """q [Hkv, G, S, D], k [Hkv, T, D] -> softmax weights [Hkv, G, S, T]."""
    s = (q.reshape(c["Hkv"], -1, c["D"]) @ k.transpose(1, 2)).view(q.shape[:3] + (k.shape[1],)) * st["scale"]
    s = s.masked_fill(~_visible(c, pos, keys), float("-inf"))
    e = torch.exp(s - s.amax(dim=-1, keepdim=True))
    return e / e.sum(dim=-1, keepdim=True)


def _heads(c, q):
    """[S, Hq, D] -> fp32 [Hkv, G, S, D]"""
    return q.float().view(q.shape[0], c["Hkv"], c["Hq"] // c["Hkv"], c["D"]).permute(1, 2, 0, 3)


def _plain_attention(c, st):
    B, S, T = c["B"], c["S"], c["T"]
    out = torch.empty(B, S, c["Hq"], c["D"], dtype=torch.bfloat16, device=DEV)
    with_weights = c["op"] == "decode_weights"
    w = st["wo"].clone().zero_() if with_weights else None
    keys = torch.arange(T, device=DEV)
    for b in range(B):
        k, v = _dense(c, st, "k", b), _dense(c, st, "v", b)
        if c["op"] == "prefill":
            k[:, T - S:], v[:, T - S:] = st["kn"][b].float().transpose(0, 1), st["vn"][b].float().transpose(0, 1)
        pos = st["lens"][b].long() - S + torch.arange(S, device=DEV)
        p = _weights_of(c, st, _heads(c, st["q"][b]), k, pos, keys)
        out[b] = (p.reshape(c["Hkv"], -1, T) @ v).view(c["Hkv"], -1, S, c["D"]).permute(2, 0, 1, 3).reshape(S, c["Hq"], c["D"]).to(torch.bfloat16)
        if with_weights:
            live = keys < st["lens"][b]
            w[b, :, :T] = torch.where(live, st["w"][b, :, :T] + p.sum(dim=(1, 2)), w[b, :, :T])
    return (out, w) if with_weights else out


def _plain_prompt_weights(c, st):
    B, S, T = c["B"], c["S"], c["T"]
    w = torch.zeros_like(st["wo"])
    keys = torch.arange(T, device=DEV)
    for b in range(B):
        k = _dense(c, st, "k", b)
        add = torch.zeros(c["Hkv"], T, device=DEV)
        for s0 in range(0, S, 256):
            s1 = min(S, s0 + 256)
            pos = T - S + torch.arange(s0, s1, device=DEV)
            add += _weights_of(c, st, _heads(c, st["q"][b, s0:s1]), k, pos, keys).sum(dim=(1, 2))
        w[b, :, :T] = st["w"][b, :, :T] + add
    return w


def _plain_evict(c, st):
    B, T, n = c["B"], c["T"], c["budget"]
    o = {x: torch.zeros_like(st[x]) for x in ("kco", "vco", "kso", "vso", "wo", "lo", "kept")}
    L = st["lens"].long().view(B, 1, 1)
    t = torch.arange(T, device=DEV).view(1, 1, T)
    rank = st["w"][:, :, :T].masked_fill((t < c["sinks"]) | (t >= L - c["recent"]), float("inf")).masked_fill(t >= L, float("-inf"))
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :n]
    best = best.masked_fill(torch.arange(n, device=DEV) >= L, T)  # fewer tokens than the budget: all of them stay
    kept = torch.sort(best, dim=2).values
    live = kept < T
    at = kept.clamp(max=T - 1)
    o["kept"].copy_(torch.where(live, kept, -1))
    o["lo"].copy_(torch.minimum(st["lens"], torch.full_like(st["lens"], n)))
    for x in ("k", "v"):
        rows = torch.stack([_rows(c, st, x + "c", b) for b in range(B)])
        o[x + "co"].copy_(torch.gather(rows, 2, at[..., None].expand(-1, -1, -1, c["D"])) * live[..., None].to(rows.dtype))
        if c["fp8"]:
            o[x + "so"].copy_(st[x + "s"])
        else:
            rows = torch.stack([_rows(c, st, x + "s", b) for b in range(B)])
            o[x + "so"][:, :, :n] = torch.gather(rows, 2, at) * live
    o["wo"][:, :, :n] = torch.gather(st["w"], 2, at) * live
    return _evicted(c, o)


def _evicted(c, o):
    codes = (lambda x: x.view(torch.float8_e4m3fn)) if c["fp8"] else (lambda x: x)
    return codes(o["kco"]), codes(o["vco"]), o["kso"], o["vso"], o["wo"], o["lo"], o["kept"]


def run(state):
    st, c = state, state["c"]
    if not own:
        return {"decode": _plain_attention, "prefill": _plain_attention, "decode_weights": _plain_attention,
                "prompt_weights": _plain_prompt_weights, "evict": _plain_evict}[c["op"]](c, st)
    from hyprstream_amd import bindings as hb
    Hkv, T, S = c["Hkv"], c["T"], c["S"]
    cache = (st["kc"], st["vc"], st["ks"], st["vs"], st["layout"])
    if c["op"] == "decode":
        hb.decode_attn(st["q"][:, 0], *cache, st["lens"], st["out"][:, 0], st["ws"], Hkv, T, st["scale"], fp8=c["fp8"],
                       window=c["window"], sinks=c["sinks"])
        return st["out"]
    if c["op"] == "prefill":
        hb.prefill_attn(st["q"], st["kn"], st["vn"], *cache, T - S, st["out"], st["scale"], quantize_on_write=False,
                        fp8=c["fp8"], window=c["window"], sinks=c["sinks"])
        return st["out"]
    if c["op"] == "decode_weights":
        hb.decode_step_weights(st["q"][:, 0], None, None, *cache, st["lens"], st["out"][:, 0], st["w"], st["wo"], st["ws"], Hkv,
                               T, st["scale"], fp8=c["fp8"], window=c["window"], sinks=c["sinks"])
        return st["out"], st["wo"]
    if c["op"] == "prompt_weights":
        hb.attn_weights(st["q"], st["kc"], st["ks"], st["layout"], st["w"], st["wo"], st["ws"], Hkv, T, st["scale"],
                        start_pos=T - S, fp8=c["fp8"], window=c["window"], sinks=c["sinks"])
        return st["wo"]
    hb.kv_evict((st["kc"], st["vc"], st["ks"], st["vs"]), st["layout"], st["lens"], st["w"],
                (st["kco"], st["vco"], st["kso"], st["vso"]), st["layout_out"], st["lo"], st["wo"], st["ws"], c["budget"],
                c["sinks"], c["recent"], T, kept=st["kept"], fp8=c["fp8"])
    return _evicted(c, st)


# ------------------------------------------------------------------------------------------------ work
def _pairs(c, n):
    """Visible (query, key) pairs of one sequence of n tokens whose last S are queries."""
    total = 0
    for p in range(n - c["S"], n):
        total += p + 1 if not c["window"] else min(p + 1, c["window"] + min(c["sinks"], max(0, p + 1 - c["window"])))
    return total


def work(case):
    c = case
    B, S, Hq, Hkv, D, T = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "T"))
    mean = T if not c["ragged"] or B == 1 else (T + (B - 1) * (T + max(1, T // 16)) // 2) // B  # the lengths are drawn
    row = D + (0 if c["fp8"] else 4)
    if c["op"] == "evict":
        kept = min(c["budget"], mean)
        return {"bytes": B * Hkv * (4 * mean + 2 * kept * (2 * row + 4) + 4 * kept), "flops": B * Hkv * mean}
    pairs = _pairs(c, mean)
    seen = mean if not c["window"] else min(mean, c["window"] + S - 1 + c["sinks"])  # tokens some query sees
    both = 1 if c["op"] == "prompt_weights" else 2  # K alone, or K and V
    out = 0 if c["op"] == "prompt_weights" else 2 * S * Hq * D
    cached = seen if c["op"] != "prefill" else max(0, seen - S)
    n = both * cached * Hkv * row + 2 * S * Hq * D + out
    if c["op"] == "prefill":
        n += 2 * S * Hkv * D * 2
    if c["op"] in ("decode_weights", "prompt_weights"):
        n += 8 * mean * Hkv
    return {"bytes": B * n, "flops": B * (2 if c["op"] == "prompt_weights" else 4) * pairs * Hq * D}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_evict(c, st):
    """Row by row on the host: the middle ordered by weight, then by index."""
    B, Hkv, D, n, T = c["B"], c["Hkv"], c["D"], c["budget"], c["T"]
    w, lens = st["w"].double().cpu().numpy(), st["lens"].tolist()
    kept = np.full((B, Hkv, n), -1, np.int32)
    for b in range(B):
        L = lens[b]
        lo, hi = c["sinks"], L - c["recent"]
        for h in range(Hkv):
            if L <= n:
                kept[b, h, :L] = np.arange(L)
                continue
            middle = np.arange(lo, hi)
            order = middle[np.lexsort((middle, -w[b, h, lo:hi]))][:n - c["sinks"] - c["recent"]]
            kept[b, h] = np.sort(np.concatenate([np.arange(lo), order, np.arange(hi, L)]))
    kept = torch.from_numpy(kept).to(DEV)
    live, at = kept >= 0, kept.long().clamp(min=0)
    pick = lambda x: torch.take_along_dim(x, at, 2) * live
    rows = lambda x: torch.where(live[..., None], torch.take_along_dim(x, at[..., None], 2), torch.zeros((), dtype=x.dtype, device=DEV))
    padded = lambda x: torch.cat([x, torch.zeros(B, Hkv, (-n) % 4, dtype=x.dtype, device=DEV)], dim=2)
    codes = [rows(st[x]).view(torch.float8_e4m3fn) if c["fp8"] else rows(st[x]) for x in ("kc", "vc")]
    scales = [st[x].double() if c["fp8"] else padded(pick(st[x].double())) for x in ("ks", "vs")]
    count = torch.tensor([min(L, n) for L in lens], dtype=torch.int32, device=DEV)
    return codes[0], codes[1], scales[0], scales[1], padded(pick(st["w"].double())), count, kept


def exact(case, seed):
    """The definitions in 64 bits, one (sequence, kv-head) at a time over the keys that count."""
    c = case
    st = _inputs(c, seed)
    B, S, Hq, Hkv, D, T = (c[k] for k in ("B", "S", "Hq", "Hkv", "D", "T"))
    G, scale = Hq // Hkv, float(D) ** -0.5
    if c["op"] == "evict":
        return _exact_evict(c, st)
    value = lambda x, b, h, idx: (st[x + "c"][b, h, idx].view(torch.float8_e4m3fn).double() * st[x + "s"][b, h].double() if c["fp8"]
                                  else st[x + "c"][b, h, idx].double() * st[x + "s"][b, h, idx].double()[:, None])
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=DEV)
    total = torch.zeros(B, Hkv, T + (-T) % 4, dtype=torch.float64, device=DEV)
    lens = st["lens"].tolist()
    for b in range(B):
        n = lens[b]
        first = 0 if not c["window"] else max(0, n - S - c["window"] + 1)
        idx = torch.arange(n, device=DEV)
        if c["window"]:
            idx = idx[(idx >= first) | (idx < c["sinks"])]
        for h in range(Hkv):
            K = value("k", b, h, idx)
            if c["op"] == "prefill":
                K = torch.where((idx >= n - S)[:, None], st["kn"][b, (idx - (n - S)).clamp(min=0), h].double(), K)
            V = None
            if c["op"] != "prompt_weights":
                V = value("v", b, h, idx)
                if c["op"] == "prefill":
                    V = torch.where((idx >= n - S)[:, None], st["vn"][b, (idx - (n - S)).clamp(min=0), h].double(), V)
            col = torch.zeros(idx.numel(), dtype=torch.float64, device=DEV)
            for s0 in range(0, S, 1024):
                p = n - S + torch.arange(s0, min(S, s0 + 1024), device=DEV)
                q = st["q"][b, s0:s0 + 1024, h * G:(h + 1) * G].double()  # [s, G, D]
                hidden = idx[None] > p[:, None]
                if c["window"]:
                    hidden |= (idx[None] <= p[:, None] - c["window"]) & (idx[None] >= c["sinks"])
                z = torch.matmul(q.reshape(-1, D), K.t()).view(-1, G, idx.numel()) * scale
                P = torch.softmax(z.masked_fill(hidden[:, None], -math.inf), dim=-1)
                if V is not None:
                    out[b, s0:s0 + 1024, h * G:(h + 1) * G] = torch.matmul(P, V)
                col += P.sum(dim=(0, 1))
            if c["op"] in ("decode_weights", "prompt_weights"):
                total[b, h, :n] = st["w"][b, h, :n].double()
                total[b, h, idx] += col
    if c["op"] == "decode_weights":
        return out, total
    return total if c["op"] == "prompt_weights" else out
