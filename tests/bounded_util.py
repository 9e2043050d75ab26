"""Plain 64-bit forms of what a bounded cache needs (windows with sinks, accumulated weights, eviction) and the caches the
GPU tests run them on."""
import numpy as np
import torch

from hyprstream_amd import bindings as hb
from hyprstream_amd import workloads as wl
from gpu_util import DEV, DeviceCache

HALF_BF16 = 2.0 ** -8   # half a step, relative
HALF_F16 = 2.0 ** -11
HALF_F32 = 2.0 ** -24


def visible(p, n, window, sinks):
    """Truth values [len(p), n]: token t is seen by a query at position p."""
    t = np.arange(n)[None, :]
    p = np.asarray(p)[:, None]
    ok = t <= p
    if window > 0:
        ok &= (t > p - window) | (t < sinks)
    return ok


def attention(q, K, V, pos, window, sinks, scale):
    """q [S, Hq, D], K, V [n, Hkv, D] (float64): (out [S, Hq, D], summed weights [Hkv, n], sum p|v| [S, Hq, D],
    score bound [S, Hq] = largest sum_d |q k| scale over the visible keys)."""
    S, Hq, D = q.shape
    n, Hkv, _ = K.shape
    G = Hq // Hkv
    see = visible(pos, n, window, sinks)
    out, mag = np.zeros((S, Hq, D)), np.zeros((S, Hq, D))
    w, bound = np.zeros((Hkv, n)), np.zeros((S, Hq))
    for h in range(Hkv):
        for g in range(G):
            z = q[:, h * G + g] @ K[:, h].T * scale
            zb = np.abs(q[:, h * G + g]) @ np.abs(K[:, h]).T * scale
            live = see.any(axis=1)
            z = np.where(see, z, -np.inf)
            e = np.exp(z - np.where(live, z.max(axis=1, initial=-np.inf), 0.0)[:, None])
            e[~live] = 0.0
            p = e / np.where(live, e.sum(axis=1), 1.0)[:, None]
            w[h] += p.sum(axis=0)
            bound[:, h * G + g] = np.where(see, zb, 0.0).max(axis=1, initial=0.0)
            if V is not None:
                out[:, h * G + g] = p @ V[:, h]
                mag[:, h * G + g] = p @ np.abs(V[:, h])
    return out, w, mag, bound


def keep(w, L, budget, sinks, recent):
    """Positions that stay of a row of L weights (None: the sinks and the newest)."""
    if L <= budget:
        return np.arange(L)
    if w is None:
        return np.concatenate([np.arange(sinks), np.arange(L - (budget - sinks), L)])
    middle = np.arange(sinks, L - recent)
    x = w[middle].astype(np.float64)
    rank = np.where(np.isnan(x), -np.inf, x)
    # NaN below every number, -inf included; equal weights by position
    order = middle[np.lexsort((middle, -rank, np.isnan(x)))][:budget - sinks - recent]
    return np.sort(np.concatenate([np.arange(sinks), order, np.arange(L - recent, L)]))


class Cache:
    """A filled int8 / fp8 cache, contiguous or paged, with its dequantized values in float64."""

    def __init__(self, stream, B, Hkv, T, D, fp8=False, paged=0, k=None, v=None):
        r = wl.philox(stream)
        rnd = lambda: torch.from_numpy(r.standard_normal((B, T, Hkv, D)).astype(np.float32)).to(torch.bfloat16).to(DEV)
        k, v = (rnd() if k is None else k), (rnd() if v is None else v)
        c = DeviceCache(B, Hkv, T, D, fp8=fp8)
        if fp8:
            hb.kv_fp8_calibrate(k, v, c.k_scales, c.v_scales)
        c.write(k, v)
        self.B, self.Hkv, self.T, self.D, self.fp8, self.paged = B, Hkv, T, D, fp8, 0
        self.layout = c.layout
        self.tensors = [c.k_codes, c.v_codes, c.k_scales, c.v_scales]
        self.K, self.V = self.values()
        if paged:
            nb = (T + paged - 1) // paged
            tables = []
            for i in (0, 1):  # K and V through tables of their own
                table = torch.from_numpy(r.permutation(B * nb).astype(np.int32).reshape(B, nb))
                where = table.long().view(-1).to(DEV)
                for j in (i,) if fp8 else (i, i + 2):
                    src = self.tensors[j][:, :, :T]
                    full = torch.zeros((B, Hkv, nb * paged) + tuple(src.shape[3:]), dtype=src.dtype, device=DEV)
                    full[:, :, :T] = src
                    blocks = full.view((B, Hkv, nb, paged) + tuple(src.shape[3:])).transpose(1, 2).reshape((B * nb, Hkv, paged) + tuple(src.shape[3:])).contiguous()  # (one sequence: reshape is a view)
                    pool = torch.empty_like(blocks)
                    pool[where] = blocks
                    self.tensors[j] = pool
                tables.append(table.to(DEV))
            self.tables, self.paged = tables, paged
            self.layout = hb.paged_layout(Hkv, paged, D, *tables)

    def dense(self, j, n=None):
        """Tensor j as [B, Hkv, T(, D)] whatever the layout (head scales: [B, Hkv])."""
        t = self.tensors[j]
        if self.fp8 and j >= 2:
            return t
        if self.paged:
            g = t[self.tables[j & 1].long()].transpose(1, 2)  # [B, Hkv, nb, block, ...]
            t = g.reshape((self.B, self.Hkv, -1) + tuple(g.shape[4:]))
        return t[:, :, :self.T if n is None else n]

    def values(self):
        out = []
        for i in (0, 1):
            codes, s = self.dense(i), self.dense(i + 2).double()
            x = codes.view(torch.float8_e4m3fn).float().double() * s[:, :, None, None] if self.fp8 else codes.double() * s[..., None]
            out.append(x.permute(0, 2, 1, 3).cpu().numpy())  # [B, T, Hkv, D]
        return out


def bf16_randn(stream, *shape):
    r = wl.philox(stream)
    return torch.from_numpy(r.standard_normal(shape).astype(np.float32)).to(torch.bfloat16).to(DEV)


def f64(t):
    return t.detach().double().cpu().numpy()


def decode_tolerance(ref, mag, bound):
    """bf16 output (half a step); the weights enter the second product as fp16 (half a step each); scores carry fp32
    roundings of sums whose terms reach 1152/127 times the products themselves (the codes' offset), which moves a weight
    by their relative size; fp16 drops weights below 2^-25 / 64 of the largest."""
    score = 512 * HALF_F32 * 10.0 * bound.max()
    return HALF_BF16 * np.abs(ref) + (2 * HALF_F16 + 2 * score) * mag + 1e-6
