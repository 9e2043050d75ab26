// Softmax weights of S queries per sequence over the cached keys, summed over the queries and over the query heads of
// each kv-head: how much attention every cached token received.
//
//   s[c, t] = scale q_c . k_t (c = a (query, head) column of one kv-head, t visible to it),  p = exp(s - lse_c),
//   weights[t] += sum_c p[c, t],   lse_c = log sum_t exp(s[c, t]).
//
// lse_c is needed before the first p and takes all of s, so s is computed twice: weights_stats_kernel walks the keys for
// a block of columns and leaves (m, l) per column, weights_columns_kernel walks the columns for a block of keys and adds
// up.  Storing p in between instead would move S x T values per query head.  Both products run on the matrix cores with
// exact operands (the result is an fp32 tensor, and a rounded operand would show in it): codes are integers (int8) or
// short floats (e4m3fn) that fp16 and bf16 hold exactly, q is bf16.  Each kernel keeps its stationary side in registers
// and converts only there or once per workgroup: columns as fp16 in the first (the streamed codes take one byte permute
// and one subtraction per two), keys as bf16 in the second (the streamed q is used as it lies).
// The keys sit on the M axis, so a lane's four score registers are four keys of one column: row statistics stay in the
// lane until the end of the walk, and so do the column sums.
#include <algorithm>

#include "mfma_common.hpp"

namespace hs {

constexpr float kWLog2e = 1.4426950408889634f;
constexpr int kWStep = 64;       // keys of a step (first kernel), columns of a step (second)
constexpr int kWSegment = 2048;  // columns of a workgroup of the second kernel, at most

struct WeightsArgs {
    const uint16_t *q;   // [B, S, Hq, D] bf16
    const uint8_t *kc;
    const float *ks;
    KvAddr ka;
    const int32_t *positions;
    const float *in;
    float *out;
    int64_t stride;
    float *part_ml;      // [B, Hkv, key chunks, columns, 2]
    float *lse;          // [B, Hkv, columns], log2 units; +inf = the column sees nothing
    float *part_w;       // [segments, B, Hkv, part_stride] when the columns of a key block are split
    int64_t part_stride;
    int32_t start_pos, B, S, Hq, Hkv, G, cols, max_seq_len, window, sinks;
    int32_t key_chunks, chunk_tokens, segments;
    float scale_log2e;
};

// Position of sequence b's first query.
__device__ __forceinline__ int first_pos(const WeightsArgs &a, int b) {
    return (a.positions ? a.positions[b] : 0) + a.start_pos;
}
// Tokens of sequence b that some query may see: positions below min(max_seq_len, last query + 1).
__device__ __forceinline__ int key_count(const WeightsArgs &a, int pos0) {
    return (int)min((int64_t)a.max_seq_len, max((int64_t)0, (int64_t)pos0 + a.S));
}
__device__ __forceinline__ bool sees(const WeightsArgs &a, int p, int t) {  // p already inside [0, max_seq_len)
    return t <= p && (a.window == 0 || t > p - a.window || t < a.sinks);
}

// e4m3fn code -> bf16 bits (exact)
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t c) {
    const half2v h = __builtin_bit_cast(half2v, e4m3_high_bytes_to_f16(c << 8));  // value / 256 in the low half
    return __float_as_uint((float)h[0] * 256.0f) >> 16;
}
__device__ __forceinline__ uint32_t code_to_bf16(uint32_t c, bool fp8) {
    return fp8 ? e4m3_to_bf16(c) : __float_as_uint((float)(int8_t)c) >> 16;
}

template <int D, bool FP8>
__global__ __launch_bounds__(256, 2) void weights_stats_kernel(WeightsArgs a) {
    constexpr int KG = D / 32, TPR = D / 32, RPP = 256 / TPR;  // threads per key row (32 codes each), rows per pass
    constexpr int PASSES = RPP >= kWStep ? 1 : kWStep / RPP;
    constexpr int NB = D == 256 ? 2 : 4;                       // 16-column blocks of a wavefront
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int units = a.B * a.Hkv;
    // units are the fastest index: the workgroups that stream one unit's keys share an XCD and its L2
    const int unit = blockIdx.x % units, chunk = (blockIdx.x / units) % a.key_chunks;
    const int blk = (int)((a.cols + 64 * NB - 1) / (64 * NB)) - 1 - (int)(blockIdx.x / units / a.key_chunks);  // late columns first: they see most
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int pos0 = first_pos(a, b);
    const int wg_c0 = blk * 64 * NB, wg_c1 = min(a.cols, wg_c0 + 64 * NB) - 1;
    const int T = key_count(a, pos0);
    __shared__ __attribute__((aligned(16))) uint8_t sm_k[2][4 * KG][1024];  // block KG u + j: keys 16u .., d 32j ..; operand order
    __shared__ __attribute__((aligned(16))) float sm_s[2][kWStep];

    // ---- columns: lane (li, lq) holds column li of each block, d = 32j + 8 lq + e
    half8 qop[NB][KG];
    float cq[NB], m[NB], l[NB];
    int pos[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int c = wg_c0 + 16 * NB * wave + 16 * nb + li, cc = min(c, a.cols - 1);
        const int s = cc / a.G, g = cc % a.G;
        const uint16_t *qp = a.q + (((int64_t)b * a.S + s) * a.Hq + h * a.G + g) * D + 8 * lq;
        float qf[8 * KG], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < KG; ++j) {
            const u32x4 w = *(const u32x4 *)(qp + 32 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qf[8 * j + 2 * e] = __uint_as_float(w[e] << 16);
                qf[8 * j + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
#pragma unroll
        for (int i = 0; i < 8 * KG; ++i) amax = fmaxf(amax, fabsf(qf[i]));
        amax = quad_max(amax);
        // amax = f 2^ex with f in [0.5, 1): the power of two comes off the operands and goes back into the scale, exactly
        int ex = 0;
        if (amax > 0.0f && amax < 3.0e38f) ex = min(126, max(-125, (int)((__float_as_uint(amax) >> 23) & 0xff) - 126));
        const float down = __uint_as_float((uint32_t)(127 - ex) << 23), up = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
        for (int j = 0; j < KG; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) qop[nb][j][e] = (_Float16)(qf[8 * j + e] * down);
        cq[nb] = a.scale_log2e * up * (FP8 ? 256.0f : 1.0f);  // e4m3fn operands are value / 256
        const int p = pos0 + s;
        pos[nb] = c < a.cols && p < a.max_seq_len ? p : -1;   // a column that sees nothing (p < 0 included)
        m[nb] = -INFINITY;
        l[nb] = 0.0f;
    }
    const float head_scale = FP8 ? a.ks[(int64_t)b * a.Hkv + h] : 0.0f;

    // ---- steps: [s_lo, s_hi) of this chunk, without those between the sinks and the window of the first column
    const int p_first = pos0 + wg_c0 / a.G, p_last = min(pos0 + wg_c1 / a.G, T - 1);
    const int c_lo = chunk * a.chunk_tokens, c_hi = min(c_lo + a.chunk_tokens, p_last + 1);
    const int sink_steps = a.window ? (a.sinks + kWStep - 1) / kWStep : 0;
    const int win_step = a.window ? max(0, p_first - a.window + 1) / kWStep : 0;
    auto next_step = [&](int st) { return a.window && st >= sink_steps && st < win_step ? win_step : st; };
    const int s_hi = c_hi > c_lo ? (c_hi + kWStep - 1) / kWStep : 0;
    int st = next_step(c_lo / kWStep);

    u32x4 raw[PASSES][2];
    float rawsc = 0.0f;
    const int krow = tid / TPR, kq = tid % TPR;
    auto load = [&](int step) {
        const int t0 = step * kWStep;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            int64_t ku;
            int slot;
            const int row = krow + p * RPP;
            if (RPP > kWStep && row >= kWStep) continue;
            resolve(a.ka, b, min(t0 + row, T - 1), ku, slot);
            const u32x4 *src = (const u32x4 *)(a.kc + ku * a.ka.code_stride_seq + (int64_t)h * a.ka.code_stride_head + (int64_t)slot * D + 32 * kq);
            raw[p][0] = src[0];
            raw[p][1] = src[1];
        }
        if (tid < kWStep) {
            if (FP8) rawsc = head_scale;
            else {
                int64_t ku;
                int slot;
                resolve(a.ka, b, min(t0 + tid, T - 1), ku, slot);
                rawsc = a.ks[ku * a.ka.scale_stride_seq + (int64_t)h * a.ka.scale_stride_head + slot];
            }
        }
    };
    auto commit = [&](int buf) {
        const _Float16 bias = (_Float16)1152.0f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = krow + p * RPP;
            if (RPP > kWStep && row >= kWStep) continue;
            uint8_t *dst = sm_k[buf][KG * (row >> 4) + kq] + (row & 15) * 16;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const uint32_t w0 = raw[p][q4 >> 1][2 * (q4 & 1)], w1 = raw[p][q4 >> 1][2 * (q4 & 1) + 1];
                *(half8 *)(dst + 256 * q4) = FP8 ? e4m3x8_to_f16_div256(w0, w1) : int8x8_to_f16_biased(w0, w1) - bias;
            }
        }
        if (tid < kWStep) sm_s[buf][tid] = rawsc;
    };
    const int wave_first = pos0 + (wg_c0 + 16 * NB * wave) / a.G, wave_last = pos0 + min(a.cols - 1, wg_c0 + 16 * NB * wave + 16 * NB - 1) / a.G;
    const bool active = wg_c0 + 16 * NB * wave < a.cols;
    if (st < s_hi) {
        load(st);
        commit(0);
    }
    __syncthreads();
    for (int buf = 0; st < s_hi; buf ^= 1) {
        const int nst = next_step(st + 1);
        if (nst < s_hi) load(nst);
        const int t0 = st * kWStep;
        if (active && t0 <= wave_last) {
            // some (key, column) pair of the step may be hidden: in the future, out of the window, past the chunk or in no sequence
            const bool edge = t0 + kWStep - 1 > wave_first || wave_last >= a.max_seq_len || wave_first < 0 || (a.window && t0 <= wave_last - a.window) ||
                              (wg_c1 + 1 == a.cols && wg_c0 + 16 * NB * (wave + 1) > a.cols);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float sc[16];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < KG; ++j)
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const half8 *)(sm_k[buf][KG * u + j] + lane * 16), qop[nb][j], acc, 0, 0, 0);
                    const float4v sk = *(const float4v *)&sm_s[buf][16 * u + 4 * lq];
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[4 * u + r] = acc[r] * sk[r] * cq[nb];
                }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!sees(a, pos[nb], t0 + 16 * (i >> 2) + 4 * lq + (i & 3))) sc[i] = -INFINITY;
                }
                float mx = sc[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
                if (__builtin_amdgcn_ballot_w64(mx > m[nb]) != 0) {
                    const float m_new = fmaxf(m[nb], mx);
                    if (m_new != -INFINITY) l[nb] *= __builtin_amdgcn_exp2f(m[nb] - m_new);
                    m[nb] = m_new;
                }
                const float ref = m[nb] == -INFINITY ? 0.0f : m[nb];
#pragma unroll
                for (int i = 0; i < 16; ++i) l[nb] += __builtin_amdgcn_exp2f(sc[i] - ref);
            }
        }
        if (nst < s_hi) commit(buf ^ 1);
        __syncthreads();
        st = nst;
    }
    // ---- join the four lanes of a column; one (m, l) per column and chunk, or the finished statistic
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float M = quad_max(m[nb]);
        const float L = quad_sum(m[nb] == -INFINITY ? l[nb] : l[nb] * __builtin_amdgcn_exp2f(m[nb] - M));
        const int c = wg_c0 + 16 * NB * wave + 16 * nb + li;
        if (lq != 0 || c >= a.cols) continue;
        if (a.key_chunks == 1) {
            a.lse[(int64_t)unit * a.cols + c] = L == 0.0f ? INFINITY : M + __builtin_amdgcn_logf(L);
        } else {
            float *ml = a.part_ml + (((int64_t)unit * a.key_chunks + chunk) * a.cols + c) * 2;
            ml[0] = M;
            ml[1] = L;
        }
    }
}

// lse of a column from its key chunks: sixteen columns a workgroup, the chunks of one over sixteen lanes.
__global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15), n = (int64_t)a.B * a.Hkv * a.cols;
    const int part = threadIdx.x >> 4;
    __shared__ float sm_m[16][16], sm_l[16][16];
    float M = -INFINITY, L = 0.0f;
    if (i < n) {
        const int64_t unit = i / a.cols, c = i % a.cols;
        const float *ml = a.part_ml + (unit * a.key_chunks * a.cols + c) * 2;
        for (int k = part; k < a.key_chunks; k += 16) M = fmaxf(M, ml[(int64_t)k * a.cols * 2]);
        for (int k = part; k < a.key_chunks; k += 16) {
            const float m = ml[(int64_t)k * a.cols * 2], l = ml[(int64_t)k * a.cols * 2 + 1];
            L += m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - M);  // (a chunk without a key has l = 0; NaN stays)
        }
    }
    sm_m[part][threadIdx.x & 15] = M;
    sm_l[part][threadIdx.x & 15] = L;
    __syncthreads();
    if (part != 0 || i >= n) return;
    float Mt = M, Lt = 0.0f;
    for (int p = 1; p < 16; ++p) Mt = fmaxf(Mt, sm_m[p][threadIdx.x]);
    for (int p = 0; p < 16; ++p) {
        const float m = sm_m[p][threadIdx.x], l = sm_l[p][threadIdx.x];
        Lt += m == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - Mt);
    }
    a.lse[i] = Lt == 0.0f ? INFINITY : Mt + __builtin_amdgcn_logf(Lt);
}

template <int D, bool FP8>
__global__ __launch_bounds__(256, 2) void weights_columns_kernel(WeightsArgs a) {
    constexpr int KG = D / 32, NU = D == 256 ? 2 : 4;  // 16-key tiles of a wavefront
    constexpr int KEYS = 64 * NU;                      // keys of the workgroup
    constexpr int CPR = D / 8, LOADS = kWStep * CPR / 256;  // 16-byte pieces of a column, pieces per thread and step
    constexpr int SWZ = CPR < 16 ? CPR - 1 : 15;       // pieces are stored at piece ^ (column & SWZ): the sixteen columns a load reads lie in different banks
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int units = a.B * a.Hkv;
    const int unit = blockIdx.x % units, seg = (blockIdx.x / units) % a.segments, kb = blockIdx.x / units / a.segments;
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int pos0 = first_pos(a, b), T = key_count(a, pos0);
    const int k0 = kb * KEYS, wk0 = k0 + 16 * NU * wave;
    if (k0 >= T) return;
    const int per = a.segments == 1 ? (a.cols + kWStep - 1) / kWStep * kWStep : kWSegment;
    int c_lo = seg * per, c_hi = min(a.cols, c_lo + per);
    // columns that can see a key of the block: from the query at its first key on; with a window, to the query that
    // loses its last key (unless the block holds sinks)
    c_lo = max(c_lo, (int)(min((int64_t)a.cols, max((int64_t)0, ((int64_t)k0 - pos0) * a.G)) / kWStep * kWStep));
    if (a.window && k0 >= a.sinks) c_hi = (int)min((int64_t)c_hi, max((int64_t)0, ((int64_t)k0 + KEYS - 1 + a.window - pos0) * a.G));
    __shared__ __attribute__((aligned(16))) uint8_t sm_q[2][kWStep * D * 2];
    __shared__ float sm_lse[2][kWStep];

    float4v sum[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) sum[u] = (float4v){0.f, 0.f, 0.f, 0.f};
    if (c_lo < c_hi) {
        // ---- keys: lane (li, lq) holds key 16u + li, d = 32j + 8 lq + e, as bf16
        bf16x8 kop[NU][KG];
        float4v sk[NU];  // scale of keys 16u + 4 lq + r, times the softmax scale in log2 units
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            int64_t ku;
            int slot;
            resolve(a.ka, b, min(wk0 + 16 * u + li, T - 1), ku, slot);
            const uint8_t *src = a.kc + ku * a.ka.code_stride_seq + (int64_t)h * a.ka.code_stride_head + (int64_t)slot * D + 8 * lq;
#pragma unroll
            for (int j = 0; j < KG; ++j) {
                const u32x2 w = *(const u32x2 *)(src + 32 * j);
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t x = w[e >> 1] >> (16 * (e & 1));
                    o[e] = code_to_bf16(x & 0xffu, FP8) | (code_to_bf16((x >> 8) & 0xffu, FP8) << 16);
                }
                kop[u][j] = pack_bf16x8(o[0], o[1], o[2], o[3]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float s;
                if (FP8) s = a.ks[(int64_t)b * a.Hkv + h];
                else {
                    resolve(a.ka, b, min(wk0 + 16 * u + 4 * lq + r, T - 1), ku, slot);
                    s = a.ks[ku * a.ka.scale_stride_seq + (int64_t)h * a.ka.scale_stride_head + slot];
                }
                sk[u][r] = s * a.scale_log2e;
            }
        }
        u32x4 raw[LOADS];
        float rawl = 0.0f;
        const float *lse = a.lse + (int64_t)unit * a.cols;
        auto load = [&](int c0) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int x = tid + 256 * i, c = min(c0 + x / CPR, a.cols - 1);
                const int s = c / a.G, g = c % a.G;
                raw[i] = *(const u32x4 *)(a.q + (((int64_t)b * a.S + s) * a.Hq + h * a.G + g) * D + 8 * (x % CPR));
            }
            if (tid < kWStep) rawl = c0 + tid < c_hi ? lse[c0 + tid] : INFINITY;  // +inf: no weight
        };
        auto commit = [&](int buf) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int x = tid + 256 * i, c = x / CPR, pc = x % CPR;
                *(u32x4 *)(sm_q[buf] + (c * CPR + (pc ^ (c & SWZ))) * 16) = raw[i];
            }
            if (tid < kWStep) sm_lse[buf][tid] = rawl;
        };
        load(c_lo);
        commit(0);
        __syncthreads();
        int buf = 0;
        for (int c0 = c_lo; c0 < c_hi; c0 += kWStep, buf ^= 1) {
            if (c0 + kWStep < c_hi) load(c0 + kWStep);
            const int p0 = pos0 + c0 / a.G, p1 = pos0 + min(c0 + kWStep - 1, a.cols - 1) / a.G;
            if (wk0 <= p1 && wk0 < T) {
                // some (key, column) pair of the step may be hidden: in the future, out of the window, past the last key or in no sequence
                const bool edge = wk0 + 16 * NU - 1 > p0 || wk0 + 16 * NU > T || p0 < 0 || p1 >= a.max_seq_len || (a.window && wk0 <= p1 - a.window);
#pragma unroll
                for (int nb = 0; nb < 4; ++nb) {
                    const int c = 16 * nb + li;
                    bf16x8 qop[KG];
#pragma unroll
                    for (int j = 0; j < KG; ++j) qop[j] = *(const bf16x8 *)(sm_q[buf] + (c * CPR + ((4 * j + lq) ^ (c & SWZ))) * 16);
                    const float ref = sm_lse[buf][c];
                    int p = -1;
                    if (edge) {
                        p = pos0 + (c0 + c) / a.G;
                        if (p >= a.max_seq_len) p = -1;
                    }
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < KG; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[u][j], qop[j], acc, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float w = __builtin_amdgcn_exp2f(acc[r] * sk[u][r] - ref);
                            if (edge && !(sees(a, p, wk0 + 16 * u + 4 * lq + r) && wk0 + 16 * u + 4 * lq + r < T)) w = 0.0f;
                            sum[u][r] += w;
                        }
                    }
                }
            }
            if (c0 + kWStep < c_hi) commit(buf ^ 1);
            __syncthreads();
        }
    }
    // ---- the sixteen columns of a key's lanes meet; lane li = 0 of each group writes its four keys
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = sum[u][r];
            x += __shfl_xor(x, 1, 64);
            x += __shfl_xor(x, 2, 64);
            x += __shfl_xor(x, 4, 64);
            x += __shfl_xor(x, 8, 64);
            sum[u][r] = x;
        }
        const int t = wk0 + 16 * u + 4 * lq;
        if (li != 0 || t >= T) continue;
        if (a.segments == 1) {
            const int64_t o = (int64_t)unit * a.stride + t;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (t + r < T) a.out[o + r] = (a.in ? a.in[o + r] : 0.0f) + sum[u][r];
        } else {
            *(float4v *)(a.part_w + ((int64_t)seg * units + unit) * a.part_stride + t) = sum[u];
        }
    }
}

// weights = in + the column segments' sums, in their order.
__global__ __launch_bounds__(256) void weights_sum_kernel(WeightsArgs a) {
    const int unit = blockIdx.y, b = unit / a.Hkv;
    const int T = key_count(a, first_pos(a, b)), t = 4 * (blockIdx.x * 256 + threadIdx.x);
    if (t >= T) return;
    const int64_t o = (int64_t)unit * a.stride + t;
    float4v w = a.in ? *(const float4v *)(a.in + o) : (float4v){0.f, 0.f, 0.f, 0.f}, add = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.segments; ++s) add += *(const float4v *)(a.part_w + ((int64_t)s * gridDim.y + unit) * a.part_stride + t);
    w += add;
    if (t + 4 <= T) *(float4v *)(a.out + o) = w;
    else
        for (int r = 0; r < T - t; ++r) a.out[o + r] = w[r];
}

int validate_layout(const hs_kv_layout *l, int B, int S, int Hkv, int D, bool need_scales);
int check_weights(const float *in, const float *out, int64_t stride, int max_seq_len, bool used);

struct WeightsPlan {
    int64_t cols, col_blocks, key_blocks;
    int key_chunks, chunk_tokens, segments;
    int64_t part_stride;
    size_t ml_floats, lse_floats, w_floats;
};

static WeightsPlan plan_weights(int B, int S, int Hq, int Hkv, int D, int max_seq_len) {
    WeightsPlan p;
    const int64_t units = (int64_t)B * Hkv;
    p.cols = (int64_t)S * (Hq / Hkv);
    const int wg_cols = D == 256 ? 128 : 256, wg_keys = D == 256 ? 128 : 256;
    p.col_blocks = (p.cols + wg_cols - 1) / wg_cols;
    p.key_blocks = ((int64_t)max_seq_len + wg_keys - 1) / wg_keys;
    // First kernel: few columns (an observation window) leave most CUs idle unless the keys are split, into chunks of
    // at least 512.
    const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, units * p.col_blocks));
    int64_t ct = ((int64_t)max_seq_len + want - 1) / want;
    ct = std::max<int64_t>(512, (ct + kWStep - 1) / kWStep * kWStep);
    p.chunk_tokens = (int)std::min<int64_t>(ct, ((int64_t)max_seq_len + kWStep - 1) / kWStep * kWStep);
    p.key_chunks = (int)(((int64_t)max_seq_len + p.chunk_tokens - 1) / p.chunk_tokens);
    // Second kernel: the columns of a key block in segments, which also evens out the causal triangle.
    p.segments = (int)((p.cols + kWSegment - 1) / kWSegment);
    p.part_stride = p.key_blocks * wg_keys;
    p.lse_floats = (size_t)(units * p.cols + 3) / 4 * 4;
    p.ml_floats = p.key_chunks > 1 ? (size_t)units * p.key_chunks * p.cols * 2 : 0;
    p.w_floats = p.segments > 1 ? (size_t)p.segments * units * p.part_stride : 0;
    return p;
}

template <int D, bool FP8>
static void launch_weights(const WeightsArgs &a, const WeightsPlan &p, hipStream_t st) {
    const int64_t units = (int64_t)a.B * a.Hkv;
    weights_stats_kernel<D, FP8><<<(unsigned)(units * p.key_chunks * p.col_blocks), 256, 0, st>>>(a);
    if (p.key_chunks > 1) weights_join_kernel<<<(unsigned)((units * p.cols + 15) / 16), 256, 0, st>>>(a);
    weights_columns_kernel<D, FP8><<<(unsigned)(units * p.segments * p.key_blocks), 256, 0, st>>>(a);
    if (p.segments > 1) weights_sum_kernel<<<dim3((unsigned)((a.max_seq_len + 1023) / 1024), (unsigned)units), 256, 0, st>>>(a);
}

}  // namespace hs

extern "C" {

size_t hs_attn_weights_workspace_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_seq_len) {
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128 && D != 256) || max_seq_len <= 0) return 0;
    const hs::WeightsPlan p = hs::plan_weights(B, S, Hq, Hkv, D, max_seq_len);
    return ((p.ml_floats + p.lse_floats + p.w_floats) * sizeof(float) + 255) / 256 * 256;
}

int hs_attn_weights(int fmt_fp8, const void *q, const void *k_codes, const float *k_scales, const hs_kv_layout *layout,
                    const int32_t *positions, int32_t start_pos, const float *weights_in, float *weights_out,
                    int64_t weights_stride, void *workspace, size_t workspace_bytes, int32_t B, int32_t S, int32_t Hq,
                    int32_t Hkv, int32_t D, int32_t max_seq_len, float softmax_scale, hs_stream_t stream) {
    using namespace hs;
    const bool fp8 = fmt_fp8 != 0;
    if (int rc = validate_layout(layout, B, S, Hkv, D, !fp8)) return rc;
    if (Hq <= 0 || Hq % Hkv != 0) return fail(HS_ERR_INVALID_ARGUMENT, "need Hq %% Hkv == 0 (Hq=%d Hkv=%d)", Hq, Hkv);
    if (max_seq_len <= 0) return fail(HS_ERR_INVALID_ARGUMENT, "max_seq_len must be positive");
    if (layout->prefill_window < 0 || layout->attn_sinks < 0)
        return fail(HS_ERR_INVALID_ARGUMENT, "negative prefill_window %d or attn_sinks %d", layout->prefill_window, layout->attn_sinks);
    const int64_t cap = layout->k_block_table ? (int64_t)layout->capacity_tokens * layout->block_table_stride : layout->capacity_tokens;
    if (max_seq_len > cap)
        return fail(HS_ERR_OVERFLOW, "max_seq_len %d exceeds what the cache can hold (%lld tokens)", max_seq_len, (long long)cap);
    if (!positions && start_pos < 0) return fail(HS_ERR_INVALID_ARGUMENT, "negative start_pos");
    if (!positions && (int64_t)start_pos + S > max_seq_len)
        return fail(HS_ERR_OVERFLOW, "queries at positions %d..%lld, but max_seq_len is %d", start_pos, (long long)start_pos + S - 1, max_seq_len);
    const bool used = B > 0 && S > 0;
    if (int rc = check_weights(weights_in, weights_out, weights_stride, max_seq_len, used)) return rc;
    if (!used) return HS_OK;
    if (!q || !k_codes || !k_scales) return fail(HS_ERR_INVALID_ARGUMENT, "null buffer");
    if ((((uintptr_t)q | (uintptr_t)k_codes) & 15) != 0 || (layout->code_stride_seq & 15) != 0)
        return fail(HS_ERR_INVALID_ARGUMENT, "q and the codes must be 16-byte aligned");
    const WeightsPlan p = plan_weights(B, S, Hq, Hkv, D, max_seq_len);
    const int64_t units = (int64_t)B * Hkv;
    if (p.cols > INT32_MAX / 2 || units > 65535 || units * p.key_chunks * p.col_blocks > INT32_MAX || units * p.segments * p.key_blocks > INT32_MAX)
        return fail(HS_ERR_INVALID_ARGUMENT, "too large for one call (B=%d S=%d Hq=%d Hkv=%d)", B, S, Hq, Hkv);
    const size_t need = hs_attn_weights_workspace_bytes(B, S, Hq, Hkv, D, max_seq_len);
    if (!workspace || workspace_bytes < need)
        return fail(HS_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
    if (((uintptr_t)workspace & 255) != 0) return fail(HS_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    WeightsArgs a;
    a.q = (const uint16_t *)q;
    a.kc = (const uint8_t *)k_codes;
    a.ks = k_scales;
    a.ka = make_addr(*layout, 0);
    a.positions = positions;
    a.in = weights_in; a.out = weights_out; a.stride = weights_stride;
    a.lse = (float *)workspace;
    a.part_w = a.lse + p.lse_floats;
    a.part_ml = a.part_w + p.w_floats;
    a.part_stride = p.part_stride;
    a.start_pos = start_pos; a.B = B; a.S = S; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv;
    a.cols = (int)p.cols; a.max_seq_len = max_seq_len;
    a.window = layout->prefill_window; a.sinks = std::min(layout->attn_sinks, max_seq_len);
    a.key_chunks = p.key_chunks; a.chunk_tokens = p.chunk_tokens; a.segments = p.segments;
    a.scale_log2e = softmax_scale * kWLog2e;
    hipStream_t st = (hipStream_t)stream;
    if (D == 64) fp8 ? launch_weights<64, true>(a, p, st) : launch_weights<64, false>(a, p, st);
    else if (D == 128) fp8 ? launch_weights<128, true>(a, p, st) : launch_weights<128, false>(a, p, st);
    else fp8 ? launch_weights<256, true>(a, p, st) : launch_weights<256, false>(a, p, st);
    return check_launch("attn_weights");
}

}  // extern "C"
