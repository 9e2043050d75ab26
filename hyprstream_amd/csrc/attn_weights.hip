// Softmax weights of S queries per sequence over the cached keys, summed over the queries and over the query heads of
// each kv-head: how much attention every cached token received.
//
//   s[c, t] = scale q_c . k_t (c = a (query, head) column of one kv-head, t visible to it),  p = exp(s - lse_c),
//   weights[t] += sum_c p[c, t],   lse_c = log sum_t exp(s[c, t]).
//
// lse_c is needed before the first p and takes all of s, so s is computed twice: weights_stats_kernel walks the keys for
// a block of columns and leaves (m, l) per column, weights_columns_kernel walks the columns for a block of keys and adds
// up.  (weights_narrow_kernel does both where all columns fit a wavefront.)  Storing p in between instead would move S x T
// values per query head.  Both products run on the matrix cores, and the result is an fp32 tensor in which a rounded
// operand would show: codes are integers (int8) or short floats (e4m3fn) that fp16 and bf16 hold exactly, q is bf16.  Each
// kernel keeps its stationary side in registers and converts only there or once per workgroup: columns in the first, keys
// as bf16 in the second (the streamed q is used as it lies; the narrow kernels multiply bf16 by bf16 in both).  The first
// kernel's columns are fp16 relative to a power of two P above their largest element (by 2 at most; by 2^5 where columns
// share it), so that the streamed codes take one byte permute and one subtraction per two: bf16's eight bits fit down to
// 2^-17 P, smaller elements are fp16 subnormals and off by at most 2^-25 P.
// 4 x 4096 queries of 32 heads on their own keys (550 GFLOP in both products): 302 + 267 + 5 us, 575 a call, 956 TFLOP/s; the
// second kernel takes 28 % less without its LDS operand reads, which share the LDS with the tiles' copies.
// The keys sit on the M axis, so a lane's four score registers are four keys of one column: row statistics stay in the
// lane until the end of the walk, and so do the column sums.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "mfma_common.hpp"

namespace hs {

constexpr float kWLog2e = 1.4426950408889634f;
constexpr int kWStep = 64;       // keys of a step of the first kernel
constexpr int kCStepMax = 128;   // columns of a step of the second (64 at head_dim 256)
constexpr int kWThreads = 256;   // both kernels
// Statistics (key chunks x columns) up to which every workgroup of the narrow kernel joins them itself instead of a launch of
// its own (us a call: 8 chunks x 64 columns 12.6 against 15.2, 512 x 8 27 against 33, 64 x 128 40.1 against 40.5, 256 x 128
// 30.6 against 29.3).
constexpr int kJoinMost = 8192;

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
    float *lse;          // [B, Hkv, lse_stride], log2 units; +inf = the column sees nothing, or there is none
    float *part_w;       // [segments, B, Hkv, part_stride] when the columns of a key block are split
    int64_t part_stride;
    int32_t start_pos, B, S, Hq, Hkv, G, cols, max_seq_len, window, sinks;
    int32_t key_chunks, chunk_tokens, segments, lse_stride, joins;
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
// Does a query at p (inside [0, max_seq_len), or negative: no query) see token t?  lo: below which tokens are out of the
// window (INT_MIN without one).  No branches: this runs for every score of a step that is cut by a bound.
__device__ __forceinline__ bool sees(int p, int lo, int sinks, int t) {
    return (t <= p) & ((t > lo) | (t < sinks));
}
__device__ __forceinline__ int window_lo(const WeightsArgs &a, int p) { return a.window == 0 ? INT_MIN : p - a.window; }

// Memory straight to LDS, 16 or 4 bytes a lane: lane i's go to dst + 16 i (4 i), dst uniform over the wavefront.
typedef __attribute__((address_space(3))) void *lds_ptr;
__device__ __forceinline__ void copy16_to_lds(const void *src, void *dst) { __builtin_amdgcn_global_load_lds(src, (lds_ptr)dst, 16, 0, 0); }
__device__ __forceinline__ void copy4_to_lds(const void *src, void *dst) { __builtin_amdgcn_global_load_lds(src, (lds_ptr)dst, 4, 0, 0); }

// Sum over the sixteen lanes of a row, in every one of them (rotations inside the row).
__device__ __forceinline__ float row_sum(float x) {
#define HS_ROR_ADD(n) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + n, 0xf, 0xf, false))
    HS_ROR_ADD(8);
    HS_ROR_ADD(4);
    HS_ROR_ADD(2);
    HS_ROR_ADD(1);
#undef HS_ROR_ADD
    return x;
}

// Eight codes (two dwords) -> eight bf16, exactly.
template <bool FP8>
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t w0, uint32_t w1) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? w0 : w1;
        if constexpr (FP8) {
            o[i] = __builtin_bit_cast(uint32_t, (i & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
        } else {
            const float lo = (float)(int8_t)(w >> (16 * (i & 1))), hi = (float)(int8_t)(w >> (16 * (i & 1) + 8));
            o[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);  // the upper halves
        }
    }
    return pack_bf16x8(o[0], o[1], o[2], o[3]);
}

// Address of token t's codes and scale (uniform over the wavefront; `span` tokens from there lie in one block).
struct KeyBase {
    const uint8_t *codes;
    const float *scales;
};
__device__ __forceinline__ KeyBase key_base(const WeightsArgs &a, int b, int h, int t, int D, bool fp8) {
    int64_t u;
    int slot;
    resolve(a.ka, b, t, u, slot);
    KeyBase k;
    k.codes = a.kc + u * a.ka.code_stride_seq + (int64_t)h * a.ka.code_stride_head + (int64_t)slot * D;
    k.scales = fp8 ? nullptr : a.ks + u * a.ka.scale_stride_seq + (int64_t)h * a.ka.scale_stride_head + slot;
    return k;
}

// NB: 16-column blocks of a wavefront (its columns stay in registers as B operands).  Per 16 keys a wavefront reads the
// K operands once from LDS and multiplies all its columns with them; a lane keeps a running (m, l) of its own keys of
// each column, m a bound that overshoots (as in the prefill kernel) so that most steps only check it.
template <int D, bool FP8, int NB>
__global__ __launch_bounds__(kWThreads, 2) void weights_stats_kernel(WeightsArgs a) {
    constexpr int KG = D / 32, TPR = D / 16, RPP = kWThreads / TPR;  // threads per key row (16 codes each), rows per pass
    constexpr int PASSES = RPP >= kWStep ? 1 : kWStep / RPP, WGC = kWThreads / 4 * NB;  // columns of the workgroup
    constexpr float kOver = 8.0f;  // log2 units by which the bound overshoots a new maximum
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int units = a.B * a.Hkv;
    // units are the fastest index: the workgroups that stream one unit's keys share an XCD and its L2
    const int unit = blockIdx.x % units, chunk = (blockIdx.x / units) % a.key_chunks;
    const int blk = (int)((a.cols + WGC - 1) / WGC) - 1 - (int)(blockIdx.x / units / a.key_chunks);  // late columns first: they see most
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int pos0 = first_pos(a, b);
    const int wg_c0 = blk * WGC, wg_c1 = min(a.cols, wg_c0 + WGC) - 1, wv_c0 = wg_c0 + 16 * NB * wave;
    const int T = key_count(a, pos0);
    // block KG u + j: the operand of keys 16u .. and d 32j ..; its 16-byte piece of lane (li, lq) sits at piece
    // 16 lq + (li ^ (2j + lq / 2)), which spreads the eight pieces a key row writes at once over the banks
    __shared__ __attribute__((aligned(16))) uint8_t sm_k[2][4 * KG][1024];
    const int piece = 16 * lq + (li ^ (lq >> 1));
    __shared__ __attribute__((aligned(16))) float sm_s[2][kWStep];

    // ---- columns: lane (li, lq) holds column li of each block, d = 32j + 8 lq + e, as fp16 times a power of two.  One
    //      power for the blocks of a lane (it then goes into the keys' scales) while their magnitudes are within 2^4 of
    //      each other, else (`own`) one per column.
    half8 qop[NB][KG];
    float cq[NB], m[NB], l[NB];
    int pos[NB], ex[NB], ex_hi = -1000, ex_lo = 1000;
    auto load_q = [&](int nb, float (&qf)[8 * KG]) {
        const int c = min(wv_c0 + 16 * nb + li, a.cols - 1), s = c / a.G, g = c % a.G;
        const uint16_t *qp = a.q + (((int64_t)b * a.S + s) * a.Hq + h * a.G + g) * D + 8 * lq;
#pragma unroll
        for (int j = 0; j < KG; ++j) {
            const u32x4 w = *(const u32x4 *)(qp + 32 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qf[8 * j + 2 * e] = __uint_as_float(w[e] << 16);
                qf[8 * j + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            }
        }
        return pos0 + s;
    };
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        float qf[8 * KG], amax = 0.0f;
        const int p = load_q(nb, qf);
#pragma unroll
        for (int i = 0; i < 8 * KG; ++i) amax = fmaxf(amax, fabsf(qf[i]));
        amax = quad_max(amax);
        // amax = f 2^ex with f in [0.5, 1)
        ex[nb] = 0;
        if (amax > 0.0f && amax < 3.0e38f) ex[nb] = min(126, max(-125, (int)((__float_as_uint(amax) >> 23) & 0xff) - 126));
        ex_hi = max(ex_hi, ex[nb]);
        ex_lo = min(ex_lo, ex[nb]);
        pos[nb] = wv_c0 + 16 * nb + li < a.cols && p < a.max_seq_len ? p : -1;  // a column that sees nothing (p < 0 included)
        m[nb] = 0.0f;
        l[nb] = 0.0f;
    }
    const bool own = NB > 1 && __builtin_amdgcn_ballot_w64(ex_hi - ex_lo > 4) != 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        if (!own) ex[nb] = ex_hi;
        const float down = __uint_as_float((uint32_t)(127 - ex[nb]) << 23), up = __uint_as_float((uint32_t)(127 + ex[nb]) << 23);
        float qf[8 * KG];
        load_q(nb, qf);
#pragma unroll
        for (int j = 0; j < KG; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) qop[nb][j][e] = (_Float16)(qf[8 * j + e] * down);
        cq[nb] = a.scale_log2e * up * (FP8 ? 256.0f : 1.0f);  // e4m3fn operands are value / 256
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

    u32x4 raw[PASSES];
    float rawsc = head_scale;
    const int krow = tid / TPR, kq = tid % TPR;
    auto load = [&](int step) {
        const int t0 = step * kWStep, last = T - 1 - t0;
        const KeyBase k = key_base(a, b, h, t0, D, FP8);
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = krow + p * RPP;
            if (RPP > kWStep && row >= kWStep) continue;
            raw[p] = *(const u32x4 *)(k.codes + (uint32_t)(min(row, last) * D + 16 * kq));
        }
        if (!FP8 && tid < kWStep) rawsc = k.scales[min(tid, last)];
    };
    auto commit = [&](int buf) {
        const _Float16 bias = (_Float16)1152.0f;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
            const int row = krow + p * RPP;
            if (RPP > kWStep && row >= kWStep) continue;
            // codes 16 kq ..: d-group j = kq / 2, lane groups lq = 2 (kq % 2) and the next
            uint8_t *dst = sm_k[buf][KG * (row >> 4) + (kq >> 1)] + (32 * (kq & 1) + ((row & 15) ^ (2 * (kq >> 1) + (kq & 1)))) * 16;
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
                const uint32_t w0 = raw[p][2 * q2], w1 = raw[p][2 * q2 + 1];
                *(half8 *)(dst + 256 * q2) = FP8 ? e4m3x8_to_f16_div256(w0, w1) : int8x8_to_f16_biased(w0, w1) - bias;
            }
        }
        if (tid < kWStep) sm_s[buf][tid] = rawsc;
    };
    const int wave_first = pos0 + wv_c0 / a.G, wave_last = pos0 + min(a.cols - 1, wv_c0 + 16 * NB - 1) / a.G;
    const bool active = wv_c0 < a.cols, ragged = wave_last >= a.max_seq_len || wave_first < 0 || wv_c0 + 16 * NB > a.cols;
    bool force = true;  // some column has no bound yet
    if (st < s_hi) {
        load(st);
        commit(0);
    }
    __syncthreads();
    auto walk = [&](auto own_tag) {
        constexpr bool kOwn = decltype(own_tag)::value;
        for (int buf = 0; st < s_hi; buf ^= 1) {
            const int nst = next_step(st + 1);
            if (nst < s_hi) load(nst);
            const int t0 = st * kWStep;
            if (active && t0 <= wave_last) {
                // some (key, column) pair of the step may be hidden: in the future, out of the window or in no sequence
                const bool edge = t0 + kWStep - 1 > wave_first || ragged || (a.window && t0 <= wave_last - a.window);
                // A step without hidden pairs, once every column has a bound: no score is compared with it.  The bound only
                // keeps the exponentials in range; a score that passes it by less than kFar is as good as any, and a step
                // with one beyond is done again with the comparing form.  Operands are read kAhead blocks ahead through a
                // ring, the exponentials of sixteen keys are made among the products of the next, in a pinned order.
                auto consume_fast = [&]() {
                    constexpr int kAhead = 4, kRing = 8, kBlocks = 4 * KG;
                    constexpr float kFar = 64.0f;
                    float4v acc[2][NB], sk[2];
                    half8 ring[kRing];
                    float l_old[NB], pend = 0.0f;
                    int over = INT_MIN, last_x = INT_MIN;
                    auto read = [&](int k) { return *(const half8 *)(sm_k[buf][k] + (piece ^ (2 * (k % KG))) * 16); };
                    auto weight = [&](int u, int e) {  // e = 4 nb + r
                        if (e > 0) l[(e - 1) >> 2] += pend;
                        const float x = acc[u & 1][e >> 2][e & 3] * sk[u & 1][e & 3] - m[e >> 2];
                        if (e & 1) over = max(over, max(last_x, __float_as_int(x)));  // positive floats order like their bits
                        last_x = __float_as_int(x);
                        pend = __builtin_amdgcn_exp2f(x);
                    };
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) l_old[nb] = l[nb];
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) ring[k] = read(k);
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) {
                        const int u = k / KG, j = k % KG;
                        if (k + kAhead < kBlocks) ring[(k + kAhead) % kRing] = read(k + kAhead);
                        if (j == 0) sk[u & 1] = *(const float4v *)&sm_s[buf][16 * u + 4 * lq] * cq[0];
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            acc[u & 1][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[k % kRing], qop[nb][j], j == 0 ? (float4v){0.f, 0.f, 0.f, 0.f} : acc[u & 1][nb], 0, 0, 0);
                            if (u > 0) {
                                const int i = j * NB + nb;  // product i of KG NB
#pragma unroll
                                for (int e = i * 4 / KG; e < (i + 1) * 4 / KG; ++e) weight(u - 1, e);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        if (u > 0 && j == KG - 1) l[NB - 1] += pend;
                    }
#pragma unroll
                    for (int e = 0; e < 4 * NB; ++e) weight(3, e);
                    l[NB - 1] += pend;
                    if (__builtin_amdgcn_ballot_w64(over > __float_as_int(kFar)) == 0) return true;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) l[nb] = l_old[nb];
                    return false;
                };
                auto consume = [&](auto edge_tag) {
                    constexpr bool kEdge = decltype(edge_tag)::value;
                    float4v acc[NB];
                    auto product = [&](int u) {
#pragma unroll
                        for (int j = 0; j < KG; ++j) {
                            const half8 kop = *(const half8 *)(sm_k[buf][KG * u + j] + (piece ^ (2 * j)) * 16);
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
                                acc[nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kop, qop[nb][j], j == 0 ? (float4v){0.f, 0.f, 0.f, 0.f} : acc[nb], 0, 0, 0);
                        }
                    };
                    product(0);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        float4v sk = *(const float4v *)&sm_s[buf][16 * u + 4 * lq];
                        if (!kOwn) sk *= cq[0];
                        float e[NB][4];
                        int over = force ? INT_MAX : INT_MIN;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                e[nb][r] = (kOwn ? acc[nb][r] * cq[nb] : acc[nb][r]) * sk[r] - m[nb];
                                if (kEdge && !sees(pos[nb], window_lo(a, pos[nb]), a.sinks, t0 + 16 * u + 4 * lq + r)) e[nb][r] = -INFINITY;
                                over = max(over, __float_as_int(e[nb][r]));  // positive floats order like their bits
                            }
                        if (__builtin_amdgcn_ballot_w64(over > 0) != 0) {
                            bool open = false;
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                const float mx = fmaxf(fmaxf(e[nb][0], e[nb][1]), fmaxf(e[nb][2], e[nb][3]));  // relative to m
                                float up = 0.0f;
                                if (l[nb] == 0.0f) up = mx > -INFINITY ? mx + kOver : 0.0f;  // the column's first keys in this lane
                                else if (mx > 0.0f) up = mx + kOver;
                                l[nb] *= __builtin_amdgcn_exp2f(-up);
                                m[nb] += up;
#pragma unroll
                                for (int r = 0; r < 4; ++r) e[nb][r] -= up;
                                open = open || (pos[nb] >= 0 && l[nb] == 0.0f && !(mx > -INFINITY));
                            }
                            force = __builtin_amdgcn_ballot_w64(open) != 0;
                        }
                        if (u < 3) product(u + 1);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
                            l[nb] += (__builtin_amdgcn_exp2f(e[nb][0]) + __builtin_amdgcn_exp2f(e[nb][1])) +
                                     (__builtin_amdgcn_exp2f(e[nb][2]) + __builtin_amdgcn_exp2f(e[nb][3]));
                    }
                };
                if (edge) consume(std::true_type{});
                else if (kOwn || force || !consume_fast()) consume(std::false_type{});
            }
            if (nst < s_hi) commit(buf ^ 1);
            __syncthreads();
            st = nst;
        }
    };
    if (own) walk(std::true_type{});
    else walk(std::false_type{});
    // ---- join the four lanes of a column; one (m, l) per column and chunk, or the finished statistic
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const float mine = l[nb] == 0.0f ? -INFINITY : m[nb];
        const float M = quad_max(mine);
        const float L = quad_sum(l[nb] == 0.0f ? 0.0f : l[nb] * __builtin_amdgcn_exp2f(mine - M));
        const int c = wv_c0 + 16 * nb + li;
        if (lq != 0 || c >= a.lse_stride) continue;
        if (a.key_chunks == 1) {
            a.lse[(int64_t)unit * a.lse_stride + c] = L == 0.0f ? INFINITY : M + __builtin_amdgcn_logf(L);
        } else if (c < a.cols) {
            float *ml = a.part_ml + (((int64_t)unit * a.key_chunks + chunk) * a.cols + c) * 2;
            ml[0] = M;
            ml[1] = L;
        }
    }
}

// Few columns (an observation window of the last queries, or single tokens): a wavefront holds all of them as B operands and
// streams keys from memory straight into A operands, sixteen at a time, two steps ahead; no barrier in the loop.  Against the
// wide kernels (us a call): one query on 64 x 8 rows of 8192 keys 443 -> 224 (1.07 GB of codes read in the two passes: 4.8
// TB/s), one on 8 x 32768 39.6 -> 25, 32 queries (128 columns) there 49 -> 38.  At 128 columns the vector pipe bounds it:
// about 200 instructions, 32 exponentials and 32 products per 16 keys do not overlap further with two wavefronts a SIMD.
// Operand j of a lane is d = (D/4) lq + 8 j ..: a lane's codes of a key lie together, and q is used as it lies (bf16).
// COLUMNS false: (m, l) of the columns over a chunk of keys; true: the weights of a chunk's keys, lse given.
template <int D, bool FP8, int NB, bool COLUMNS>
__global__ __launch_bounds__(kWThreads, 2) void weights_narrow_kernel(WeightsArgs a) {
    constexpr int KG = D / 32, LOADS = D / 64;  // 16-byte loads of a lane per key
    constexpr float kOver = 8.0f, kFar = 64.0f;  // as in weights_stats_kernel
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int units = a.B * a.Hkv, unit = blockIdx.x % units, chunk = blockIdx.x / units;
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int pos0 = first_pos(a, b), T = key_count(a, pos0);
    const int p_first = max(pos0, 0), p_last = T - 1;  // of the queries that see anything
    const int c_lo = chunk * a.chunk_tokens, c_hi = min(c_lo + a.chunk_tokens, T);
    const int s_hi = c_hi > c_lo ? (c_hi + kWStep - 1) / kWStep : 0;
    const int sink_steps = a.window ? (a.sinks + kWStep - 1) / kWStep : 0;
    const int win_step = a.window ? max(0, p_first - a.window + 1) / kWStep : 0;
    auto gap = [&](int st) { return a.window && st >= sink_steps && st < win_step; };  // nobody sees a key of the step
    // without a sum to write (or with the one that is there already) such steps are left out
    const bool skips = !COLUMNS || a.in == a.out;
    auto next_step = [&](int st) { return skips && gap(st) ? win_step : st; };
    int st = next_step(c_lo / kWStep), nst = next_step(st + 1);
    if (COLUMNS && st >= s_hi) return;

    u32x4 raw[2][LOADS];
    float rawsc[2][4];
    float4v before[2];
    // Always as many loads, whatever the step is (behind the end the last one again, in the gap the one behind it): only then
    // is a wait for the older of two loads in flight not a wait for both.
    const float *in = a.in ? a.in : a.out;
    auto load = [&](int step, auto slot_tag) {
        constexpr int kSlot = decltype(slot_tag)::value;
        step = min(step, s_hi - 1);
        if (COLUMNS) {
            const int t = step * kWStep + 16 * wave + 4 * lq;
            before[kSlot] = *(const float4v *)(in + (int64_t)unit * a.stride + min((int64_t)t, a.stride - 4));
            if (gap(step)) step = min(win_step, s_hi - 1);
        }
        const int t0 = step * kWStep, last = T - 1 - t0;
        const KeyBase k = key_base(a, b, h, t0, D, FP8);
        const uint8_t *src = k.codes + (uint32_t)(min(16 * wave + li, last) * D + D / 4 * lq);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) raw[kSlot][i] = *(const u32x4 *)(src + 16 * i);
        if (!FP8) {
#pragma unroll
            for (int r = 0; r < 4; ++r) rawsc[kSlot][r] = k.scales[min(16 * wave + 4 * lq + r, last)];
        }
    };
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const float head_scale = FP8 ? a.ks[(int64_t)b * a.Hkv + h] : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) rawsc[s][r] = head_scale;
    }
    if (s_hi > 0) {
        load(st, std::integral_constant<int, 0>{});
        load(nst, std::integral_constant<int, 1>{});
    }
    // ---- columns: block nb, column li.  One that sees nothing (no query, or none inside [0, max_seq_len)) is zero.  They come
    //      through LDS (16-byte piece pc of column c at piece pc ^ c, modulo 16): read by every wavefront for itself, 64 MB
    //      from L2 at 512 workgroups, the columns took 8 us of a kernel of 24.
    constexpr int CPR = D / 8, SWZ = CPR < 16 ? CPR - 1 : 15;
    __shared__ __attribute__((aligned(16))) uint8_t sm_q[16 * NB * D * 2];
#pragma unroll
    for (int i = 0; i < 16 * NB * CPR / kWThreads; ++i) {
        const int x = tid + kWThreads * i, c = x / CPR, cc = min(c, a.cols - 1), s = cc / a.G;
        copy16_to_lds(a.q + (((int64_t)b * a.S + s) * a.Hq + h * a.G + cc - s * a.G) * D + 8 * ((x % CPR) ^ (c & SWZ)), sm_q + 16 * (kWThreads * i + 64 * wave));
    }
    // the columns' lse: from their key chunks where these are few, else weights_join_kernel has made them
    constexpr int kCols = 16 * NB, kParts = kWThreads / kCols;
    __shared__ float sm_jm[COLUMNS ? kParts : 1][kCols], sm_jl[COLUMNS ? kParts : 1][kCols];
    const bool joins = COLUMNS && a.joins;
    if (joins) {
        const int c = tid % kCols;
        const float *ml = a.part_ml + ((int64_t)unit * a.key_chunks * a.cols + min(c, a.cols - 1)) * 2;
        float M = -3.0e38f, L = 0.0f;
        for (int k0 = tid / kCols; k0 < a.key_chunks; k0 += 8 * kParts) {
            float cm[8], cl[8], top = M;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int k = k0 + i * kParts;
                const float2 x = *(const float2 *)(ml + (int64_t)min(k, a.key_chunks - 1) * a.cols * 2);
                cm[i] = x.x;
                cl[i] = k < a.key_chunks ? x.y : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, cm[i]);
            L *= __builtin_amdgcn_exp2f(M - top);
#pragma unroll
            for (int i = 0; i < 8; ++i) L += cl[i] * __builtin_amdgcn_exp2f(cm[i] - top);
            M = top;
        }
        sm_jm[tid / kCols][c] = M;
        sm_jl[tid / kCols][c] = L;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    bf16x8 qop[NB][KG];
    int pos[NB];
    float m[NB], l[NB], sum[4];  // COLUMNS: m = lse
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int c = 16 * nb + li, p = pos0 + min(c, a.cols - 1) / a.G;
        pos[nb] = c < a.cols && p < a.max_seq_len ? max(p, -1) : -1;
#pragma unroll
        for (int j = 0; j < KG; ++j) {
            const u32x4 w = *(const u32x4 *)(sm_q + (c * CPR + ((KG * lq + j) ^ (c & SWZ))) * 16) & (uint32_t)~(pos[nb] >> 31);
            qop[nb][j] = pack_bf16x8(w[0], w[1], w[2], w[3]);
        }
        m[nb] = 0.0f;
        if (COLUMNS && joins) {
            float M = -3.0e38f, L = 0.0f;
#pragma unroll
            for (int i = 0; i < kParts; ++i) M = fmaxf(M, sm_jm[i][c]);
#pragma unroll
            for (int i = 0; i < kParts; ++i) L += sm_jl[i][c] * __builtin_amdgcn_exp2f(sm_jm[i][c] - M);
            m[nb] = L == 0.0f || c >= a.cols ? INFINITY : M + __builtin_amdgcn_logf(L);
        } else if (COLUMNS) {
            m[nb] = a.lse[(int64_t)unit * a.lse_stride + c];
        }
        l[nb] = 0.0f;
    }
    // the loads above end here: a wait for them inside the loop would be a wait for the keys of the steps ahead as well
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        asm volatile("" : "+v"(m[nb]));
#pragma unroll
        for (int j = 0; j < KG; ++j) asm volatile("" : "+v"(qop[nb][j]));
    }
    bool force = true;  // some column has no bound yet
    auto body = [&](auto slot_tag) {
        constexpr int kSlot = decltype(slot_tag)::value;
        const int t0 = st * kWStep + 16 * wave;  // this wavefront's keys
        bf16x8 kop[KG];
        float sk[4];
        // (the codes are unpacked here: carried through the loop as bytes they take four times the registers)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) asm volatile("" : "+v"(raw[kSlot][i]));
#pragma unroll
        for (int j = 0; j < KG; ++j) kop[j] = codes_to_bf16<FP8>(raw[kSlot][j / 2][2 * (j & 1)], raw[kSlot][j / 2][2 * (j & 1) + 1]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sk[r] = rawsc[kSlot][r] * a.scale_log2e;
            sum[r] = 0.0f;
        }
        const float4v start = before[kSlot];
        const int after = next_step(nst + 1);
        load(after, slot_tag);
        const bool edge = t0 + 15 > p_first || (a.window && t0 <= p_last - a.window);
        // The products of block nb among the weights of block nb - 1, each added up one weight later, in a pinned order.
        float4v acc[2];
        auto products = [&](int nb, int j) { acc[nb & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[j], qop[nb][j], j == 0 ? (float4v){0.f, 0.f, 0.f, 0.f} : acc[nb & 1], 0, 0, 0); };
        auto blocks = [&](auto look, auto add) {
            float pend = 0.0f;
#pragma unroll
            for (int nb = 0; nb <= NB; ++nb) {
#pragma unroll
                for (int j = 0; j < KG; ++j) {
                    if (nb < NB) products(nb, j);
                    if (nb > 0) {
#pragma unroll
                        for (int r = j * 4 / KG; r < (j + 1) * 4 / KG; ++r) {
                            const int i = 4 * (nb - 1) + r;
                            if (i > 0) add((i - 1) / 4, (i - 1) % 4, pend);
                            const float x = acc[(nb - 1) & 1][r] * sk[r] - m[nb - 1];
                            look(x);
                            pend = __builtin_amdgcn_exp2f(x);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            add(NB - 1, 3, pend);
        };
        if (t0 < T && !(COLUMNS && gap(st))) {
            if constexpr (COLUMNS) {
                auto none = [](float) {};
                if (edge) blocks(none, [&](int nb, int r, float w) { sum[r] += sees(pos[nb], window_lo(a, pos[nb]), a.sinks, t0 + 4 * lq + r) ? w : 0.0f; });
                else blocks(none, [&](int, int r, float w) { sum[r] += w; });
            } else {
                bool done = false;
                if (!edge && !force) {  // no comparisons but one: done again with them if a score is far above its bound
                    float l_old[NB];
                    int over = INT_MIN, last_x = INT_MIN;
                    bool second = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) l_old[nb] = l[nb];
                    blocks(
                        [&](float x) {
                            if (second) over = max(over, max(last_x, __float_as_int(x)));  // positive floats order like their bits
                            last_x = __float_as_int(x);
                            second = !second;
                        },
                        [&](int nb, int, float w) { l[nb] += w; });
                    done = __builtin_amdgcn_ballot_w64(over > __float_as_int(kFar)) == 0;
                    if (!done) {
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) l[nb] = l_old[nb];
                    }
                }
                if (!done) {
                    bool open = false;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                        for (int j = 0; j < KG; ++j) products(nb, j);
                        float e[4], mx = -INFINITY;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            e[r] = acc[nb & 1][r] * sk[r] - m[nb];
                            if (edge && !sees(pos[nb], window_lo(a, pos[nb]), a.sinks, t0 + 4 * lq + r)) e[r] = -INFINITY;
                            mx = fmaxf(mx, e[r]);
                        }
                        float up = 0.0f;
                        if (l[nb] == 0.0f) up = mx > -INFINITY ? mx + kOver : 0.0f;  // the column's first keys in this lane
                        else if (mx > 0.0f) up = mx + kOver;
                        l[nb] *= __builtin_amdgcn_exp2f(-up);
                        m[nb] += up;
#pragma unroll
                        for (int r = 0; r < 4; ++r) l[nb] += __builtin_amdgcn_exp2f(e[r] - up);
                        open = open || (pos[nb] >= 0 && l[nb] == 0.0f);
                    }
                    force = __builtin_amdgcn_ballot_w64(open) != 0;
                }
            }
        }
        if constexpr (COLUMNS) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] = (a.in ? start[r] : 0.0f) + row_sum(sum[r]);
            const int t = t0 + 4 * lq;
            if (li == 0 && t < T) {
                float *o = a.out + (int64_t)unit * a.stride + t;
                if (t + 4 <= T) *(float4v *)o = (float4v){sum[0], sum[1], sum[2], sum[3]};
                else
                    for (int r = 0; r < 4; ++r)
                        if (t + r < T) o[r] = sum[r];
            }
        }
        st = nst;
        nst = after;
    };
    while (st < s_hi) {
        body(std::integral_constant<int, 0>{});
        if (st >= s_hi) break;
        body(std::integral_constant<int, 1>{});
    }
    if constexpr (!COLUMNS) {
        // ---- join the four lanes of a column, then the wavefronts
        __shared__ float sm_m[4][16 * NB], sm_l[4][16 * NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const bool none = l[nb] == 0.0f || pos[nb] < 0;
            const float mine = none ? -INFINITY : m[nb], M = quad_max(mine);
            const float L = quad_sum(none ? 0.0f : l[nb] * __builtin_amdgcn_exp2f(mine - M));
            if (lq == 0) {
                sm_m[wave][16 * nb + li] = M;
                sm_l[wave][16 * nb + li] = L;
            }
        }
        __syncthreads();
        if (tid >= 16 * NB) return;
        float M = -INFINITY, L = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w][tid]);
#pragma unroll
        for (int w = 0; w < 4; ++w) L += sm_m[w][tid] == -INFINITY ? sm_l[w][tid] : sm_l[w][tid] * __builtin_amdgcn_exp2f(sm_m[w][tid] - M);
        if (a.key_chunks == 1) {
            a.lse[(int64_t)unit * a.lse_stride + tid] = L == 0.0f ? INFINITY : M + __builtin_amdgcn_logf(L);
        } else if (tid < a.cols) {
            float *ml = a.part_ml + (((int64_t)unit * a.key_chunks + chunk) * a.cols + tid) * 2;
            ml[0] = M;
            ml[1] = L;
        }
    }
}

// lse of a column from its key chunks: sixteen columns a workgroup, the chunks of one over sixteen lanes.
__global__ __launch_bounds__(256) void weights_join_kernel(WeightsArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15), n = (int64_t)a.B * a.Hkv * a.lse_stride;
    const int part = threadIdx.x >> 4;
    __shared__ float sm_m[16][16], sm_l[16][16];
    float M = -INFINITY, L = 0.0f;
    const int64_t unit = i / a.lse_stride, c = i % a.lse_stride;
    if (i < n && c < a.cols) {
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
__global__ __launch_bounds__(kWThreads, 2) void weights_columns_kernel(WeightsArgs a) {
    constexpr int KG = D / 32, NU = D == 256 ? 2 : 4;  // 16-key tiles of a wavefront
    constexpr int KEYS = kWThreads / 4 * NU;                     // keys of the workgroup
    constexpr int kCStep = D == 256 ? 64 : kCStepMax;
    constexpr int CPR = D / 8, LOADS = kCStep * CPR / kWThreads;  // 16-byte pieces of a column, pieces per thread and step
    constexpr int SWZ = CPR < 16 ? CPR - 1 : 15;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lq = lane >> 4;
    const int units = a.B * a.Hkv;
    // key blocks in ascending order: the first ones are seen by the most columns and start first
    const int unit = blockIdx.x % units, seg = (blockIdx.x / units) % a.segments, kb = blockIdx.x / units / a.segments;
    const int b = unit / a.Hkv, h = unit % a.Hkv;
    const int pos0 = first_pos(a, b), T = key_count(a, pos0);
    const int k0 = kb * KEYS, wk0 = k0 + 16 * NU * wave;
    if (k0 >= T) return;
    // steps of kCStep columns; this workgroup takes every a.segments-th of them
    int c_lo = 0, c_hi = (a.cols + kCStep - 1) / kCStep * kCStep;
    const int stride = kCStep * a.segments;
    // columns that can see a key of the block: from the query at its first key on; with a window, to the query that
    // loses its last key (unless the block holds sinks)
    c_lo = max(c_lo, (int)(min((int64_t)a.cols, max((int64_t)0, ((int64_t)k0 - pos0) * a.G)) / kCStep * kCStep));
    c_lo += (seg + a.segments - c_lo / kCStep % a.segments) % a.segments * kCStep;
    if (a.window && k0 >= a.sinks)
        c_hi = (int)min((int64_t)c_hi, (max((int64_t)0, ((int64_t)k0 + KEYS - 1 + a.window - pos0) * a.G) + kCStep - 1) / kCStep * kCStep);
    // two buffers of kCStep columns as they lie in q (16-byte piece pc of a column at piece pc ^ (column & SWZ): the sixteen
    // columns a load of operands reads lie in different banks), and their lse.  The copies go straight from memory to LDS.
    constexpr int kTileBytes = kCStep * D * 2, kTile = kTileBytes + kCStep * 4;
    __shared__ __attribute__((aligned(16))) uint8_t sm[2 * kTile];

    float4v sum[NU], before[NU];  // `before`: what the weights of this lane's keys start from, loaded while there is other work
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        sum[u] = before[u] = (float4v){0.f, 0.f, 0.f, 0.f};
        if (a.segments == 1 && a.in && li == 0) before[u] = *(const float4v *)(a.in + (int64_t)unit * a.stride + min((int64_t)(wk0 + 16 * u + 4 * lq), a.stride - 4));
    }
    if (c_lo < c_hi) {
        // ---- columns, kCStep a step: copy i of this thread is piece (x % CPR) of the tile's column x / CPR, x = tid + kWThreads i.
        //      Where kCStep is a multiple of G the columns' rows move by one constant from step to step.
        const float *lse = a.lse + (int64_t)unit * a.lse_stride;
        const uint8_t *qb = (const uint8_t *)(a.q + ((int64_t)b * a.S * a.Hq + h * a.G) * D);
        const bool regular = kCStep % a.G == 0;
        const int64_t step_bytes = (int64_t)(kCStep / a.G) * a.Hq * D * 2;
        uint32_t off[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int x = tid + kWThreads * i, c = x / CPR;
            off[i] = (uint32_t)((c / a.G) * a.Hq + c % a.G) * (D * 2) + 16 * ((x % CPR) ^ (c & SWZ));
        }
        auto fetch = [&](int c0, int buf) {
            uint8_t *dst = sm + buf * kTile + 1024 * wave;
            if (regular && c0 + kCStep <= a.cols) {
                const uint8_t *src = qb + (int64_t)(c0 / kCStep) * step_bytes;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) copy16_to_lds(src + off[i], dst + 16 * kWThreads * i);
            } else {  // any other group size; the last, partial step repeats the last column
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int x = tid + kWThreads * i, c = x / CPR, cc = min(c0 + c, a.cols - 1);
                    const uint8_t *src = qb + ((int64_t)(cc / a.G) * a.Hq + cc % a.G) * (D * 2) + 16 * ((x % CPR) ^ (c & SWZ));
                    copy16_to_lds(src, dst + 16 * kWThreads * i);
                }
            }
            if (wave < kCStep / 64) copy4_to_lds(lse + c0 + 64 * wave + lane, sm + buf * kTile + kTileBytes + 256 * wave);
        };
        // ---- keys: lane (li, lq) holds key 16u + li, d = 32j + 8 lq + e, as bf16
        bf16x8 kop[NU][KG];
        float4v sk[NU];  // scale of keys 16u + 4 lq + r, times the softmax scale in log2 units
        {
            const KeyBase k = key_base(a, b, h, min(wk0, T - 1), D, FP8);  // (a wavefront behind the last key: any address)
            const int last = max(0, T - 1 - wk0);
            u32x2 w[NU][KG];
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const uint8_t *src = k.codes + (uint32_t)(min(16 * u + li, last) * D + 8 * lq);
#pragma unroll
                for (int j = 0; j < KG; ++j) w[u][j] = *(const u32x2 *)(src + 32 * j);
#pragma unroll
                for (int r = 0; r < 4; ++r) sk[u][r] = a.scale_log2e * (FP8 ? a.ks[(int64_t)b * a.Hkv + h] : k.scales[min(16 * u + 4 * lq + r, last)]);
            }
            fetch(c_lo, 0);
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < KG; ++j) kop[u][j] = codes_to_bf16<FP8>(w[u][j][0], w[u][j][1]);
        }
        // one step of a wavefront; kEdge: some (key, column) pair may be hidden
        uint32_t qoff[KG];  // this lane's piece of the operand of d-group j, column li
#pragma unroll
        for (int j = 0; j < KG; ++j) qoff[j] = (uint32_t)((li * CPR + ((4 * j + lq) ^ (li & SWZ))) * 16);
        auto consume = [&](auto buf_tag, int c0, auto edge_tag) {
            constexpr int kBuf = decltype(buf_tag)::value;
            constexpr bool kEdge = decltype(edge_tag)::value;
            const uint8_t *tile = sm + kBuf * kTile;
            // Operand block k = KG nb + j is read kAhead blocks ahead of its products through a ring of registers; the
            // weights of the previous sixteen columns are made among the products of these, four NU of them spread over
            // KG NU products.  The order is pinned: left to itself the compiler reads each operand right before its use.
            constexpr int kBlocks = kCStep / 16 * KG, kAhead = 4, kRing = 8;
            float4v acc[2][NU];
            bf16x8 ring[kRing];
            float ref[2] = {0.0f, 0.0f}, pend = 0.0f;
            int p = -1, lo = 0;
            auto read = [&](int k) { return *(const bf16x8 *)(tile + (k / KG) * 16 * CPR * 16 + qoff[k % KG]); };
            auto add = [&](int e) {  // weight e of a group of sixteen columns: tile e / 4, key row e % 4
                if constexpr (kEdge) sum[e >> 2][e & 3] += sees(p, lo, a.sinks, wk0 + 16 * (e >> 2) + 4 * lq + (e & 3)) ? pend : 0.0f;
                else sum[e >> 2][e & 3] += pend;
            };
            auto weight = [&](int nb, int e) {
                if (e > 0) add(e - 1);
                pend = __builtin_amdgcn_exp2f(acc[nb & 1][e >> 2][e & 3] * sk[e >> 2][e & 3] - ref[nb & 1]);
            };
            auto bounds = [&](int nb) {
                if constexpr (kEdge) {
                    p = pos0 + (c0 + 16 * nb + li) / a.G;
                    if (p >= a.max_seq_len) p = -1;
                    lo = window_lo(a, p);
                    p = min(p, T - 1);
                }
            };
#pragma unroll
            for (int k = 0; k < kAhead; ++k) ring[k] = read(k);
#pragma unroll
            for (int k = 0; k < kBlocks; ++k) {
                const int nb = k / KG, j = k % KG;
                if (k + kAhead < kBlocks) ring[(k + kAhead) % kRing] = read(k + kAhead);
                if (j == 0) ref[nb & 1] = ((const float *)(tile + kTileBytes))[16 * nb + li];
                if (j == 0 && nb > 0) bounds(nb - 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    acc[nb & 1][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop[u][j], ring[k % kRing], j == 0 ? (float4v){0.f, 0.f, 0.f, 0.f} : acc[nb & 1][u], 0, 0, 0);
                    if (nb > 0) {
                        const int i = j * NU + u;  // product i of KG NU
#pragma unroll
                        for (int e = i * 4 / KG; e < (i + 1) * 4 / KG; ++e) weight(nb - 1, e);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (nb > 0 && j == KG - 1) add(4 * NU - 1);
            }
            bounds(kCStep / 16 - 1);
#pragma unroll
            for (int e = 0; e < 4 * NU; ++e) weight(kCStep / 16 - 1, e);
            add(4 * NU - 1);
        };
        auto step = [&](auto buf_tag, int c0) {
            // this wavefront's copies of the tile have landed, then everybody's; nobody reads the other buffer any more
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (c0 + stride < c_hi) fetch(c0 + stride, 1 - decltype(buf_tag)::value);
            const int p0 = pos0 + c0 / a.G, p1 = pos0 + min(c0 + kCStep - 1, a.cols - 1) / a.G;
            if (wk0 <= p1 && wk0 < T) {
                // hidden: in the future, out of the window, past the last key or in no sequence
                const bool edge = wk0 + 16 * NU - 1 > p0 || wk0 + 16 * NU > T || p0 < 0 || p1 >= a.max_seq_len || (a.window && wk0 <= p1 - a.window);
                if (edge) consume(buf_tag, c0, std::true_type{});
                else consume(buf_tag, c0, std::false_type{});
            }
        };
        for (int c0 = c_lo; c0 < c_hi; c0 += 2 * stride) {
            step(std::integral_constant<int, 0>{}, c0);
            if (c0 + stride < c_hi) step(std::integral_constant<int, 1>{}, c0 + stride);
        }
    }
    // ---- the sixteen columns of a key's lanes meet; lane li = 0 of each group writes its four keys
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            sum[u][r] = row_sum(sum[u][r]);
        }
        const int t = wk0 + 16 * u + 4 * lq;
        if (li != 0 || t >= T) continue;
        if (a.segments == 1) {
            const int64_t o = (int64_t)unit * a.stride + t;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (t + r < T) a.out[o + r] = before[u][r] + sum[u][r];
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
    int64_t cols, col_blocks, key_blocks, lse_stride;
    bool narrow;
    int nb;  // 16-column blocks per wavefront of the first kernel
    int key_chunks, chunk_tokens, segments;
    int64_t part_stride;
    size_t ml_floats, lse_floats, w_floats;
};

static WeightsPlan plan_weights(int B, int S, int Hq, int Hkv, int D, int max_seq_len) {
    WeightsPlan p;
    const int64_t units = (int64_t)B * Hkv;
    p.cols = (int64_t)S * (Hq / Hkv);
    // All columns in the registers of one wavefront (128; 64 at head_dim 256): the narrow kernels.  Else a wavefront of the
    // first kernel holds 64 columns (32).
    const int most = D == 256 ? 64 : 128;
    p.narrow = p.cols <= most;
    p.nb = !p.narrow ? most / 32 : p.cols <= 32 ? 2 : p.cols <= 64 ? 4 : 8;
    const int wg_cols = kWThreads / 4 * p.nb, wg_keys = kWThreads / 4 * (D == 256 ? 2 : 4);
    p.col_blocks = p.narrow ? 1 : (p.cols + wg_cols - 1) / wg_cols;
    p.key_blocks = ((int64_t)max_seq_len + wg_keys - 1) / wg_keys;
    // Few columns leave most CUs idle unless the keys are split.  Narrow: 512 workgroups, one round, of at least 128 keys (32
    // columns x 16 on 8 units, 4096 keys, us a call: 15.0 with 128, 17.5 with 256, 22.7 with 512) and at most 4096 (512 units
    // x 8192 keys, single queries: 223 us, 246 with one chunk).  Wide: at least 512
    // keys (256 columns on 8 units, 32768 keys: 70 us, 77 with 256, 71 with 1024).
    const int64_t want = std::max<int64_t>(1, (p.narrow ? 512 : 1024) / std::max<int64_t>(1, units * p.col_blocks));
    int64_t ct = (((int64_t)max_seq_len + want - 1) / want + kWStep - 1) / kWStep * kWStep;
    ct = p.narrow ? std::min<int64_t>(4096, std::max<int64_t>(128, ct)) : std::max<int64_t>(512, ct);
    p.chunk_tokens = (int)std::min<int64_t>(ct, ((int64_t)max_seq_len + kWStep - 1) / kWStep * kWStep);
    p.key_chunks = (int)(((int64_t)max_seq_len + p.chunk_tokens - 1) / p.chunk_tokens);
    // Second kernel: two workgroups are resident on each of 256 CUs, and each of them should come round twice: started in
    // order of their work, long items then meet short ones and the causal triangle evens out (4 x 4096 tokens, 16 key
    // blocks on 32 units, us: 369 with one share of the columns, 305 with two, 308 with four).
    const int64_t items = units * p.key_blocks, steps = (p.cols + kCStepMax - 1) / kCStepMax;
    p.segments = p.narrow ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(steps, 16), (1024 + items - 1) / items));
    p.part_stride = p.key_blocks * wg_keys;
    p.lse_stride = p.narrow ? 16 * p.nb : (p.cols + 127) / 128 * 128;
    p.lse_floats = (size_t)(units * p.lse_stride);
    p.ml_floats = p.key_chunks > 1 ? (size_t)units * p.key_chunks * p.cols * 2 : 0;
    p.w_floats = p.segments > 1 ? (size_t)p.segments * units * p.part_stride : 0;
    return p;
}

// Most floats that a call with THESE sizes, or with fewer queries or a smaller max_seq_len, takes: a caller sizes its
// workspace once, for its longest chunk and the capacity of its cache.  plan_weights's own sum falls and rises with either
// (chunks are rounded, and the fewer there are of one thing the more another is split), hence a bound of each part.
static size_t most_floats(int B, int S, int Hq, int Hkv, int D, int max_seq_len) {
    const int64_t units = (int64_t)B * Hkv, cols = (int64_t)S * (Hq / Hkv), n = max_seq_len;
    const int64_t most = D == 256 ? 64 : 128, few = std::min(cols, most);  // columns of a narrow call
    const int64_t wg_cols = 2 * most, wg_keys = kWThreads / 4 * (D == 256 ? 2 : 4);
    int64_t lse = few <= 32 ? 32 : few <= 64 ? 64 : 128;
    // narrow: chunks of at least 128 keys, `want` of them at most unless they reach 4096 keys
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, units));
    const int64_t chunks = std::min((n + 127) / 128, std::max(want, (n + 4095) / 4096));
    int64_t ml = chunks > 1 ? units * chunks * few * 2 : 0, w = 0;
    if (cols > most) {
        lse = std::max(lse, (cols + 127) / 128 * 128);
        // wide: chunks of at least 512 keys, and only while units x column blocks x chunks stay within 1024
        if (n > 512) ml = std::max(ml, 2 * std::min(units * ((n + 511) / 512) * cols, 1024 * wg_cols));
        // shares of the columns: at most 16, no more than there are steps, and only up to 1024 + items
        const int64_t items = units * ((n + wg_keys - 1) / wg_keys), steps = (cols + kCStepMax - 1) / kCStepMax;
        if (steps > 1) w = wg_keys * std::min(std::min<int64_t>(steps, 16) * items, 1023 + std::min<int64_t>(items, 1023));
    }
    return (size_t)(units * lse + ml + w);
}

template <int D, bool FP8, int NB>
static void launch_narrow(const WeightsArgs &a, const WeightsPlan &p, hipStream_t st) {
    const int64_t units = (int64_t)a.B * a.Hkv;
    weights_narrow_kernel<D, FP8, NB, false><<<(unsigned)(units * p.key_chunks), kWThreads, 0, st>>>(a);
    if (p.key_chunks > 1 && !a.joins) weights_join_kernel<<<(unsigned)((units * p.lse_stride + 15) / 16), 256, 0, st>>>(a);
    weights_narrow_kernel<D, FP8, NB, true><<<(unsigned)(units * p.key_chunks), kWThreads, 0, st>>>(a);
}

template <int D, bool FP8>
static void launch_weights(const WeightsArgs &a, const WeightsPlan &p, hipStream_t st) {
    const int64_t units = (int64_t)a.B * a.Hkv;
    if (p.narrow) {
        if (p.nb == 2) return launch_narrow<D, FP8, 2>(a, p, st);
        if (p.nb == 4) return launch_narrow<D, FP8, 4>(a, p, st);
        if constexpr (D < 256) return launch_narrow<D, FP8, 8>(a, p, st);
    }
    weights_stats_kernel<D, FP8, D == 256 ? 2 : 4><<<(unsigned)(units * p.key_chunks * p.col_blocks), kWThreads, 0, st>>>(a);
    if (p.key_chunks > 1) weights_join_kernel<<<(unsigned)((units * p.lse_stride + 15) / 16), 256, 0, st>>>(a);
    weights_columns_kernel<D, FP8><<<(unsigned)(units * p.segments * p.key_blocks), kWThreads, 0, st>>>(a);
    if (p.segments > 1) weights_sum_kernel<<<dim3((unsigned)((a.max_seq_len + 1023) / 1024), (unsigned)units), 256, 0, st>>>(a);
}

}  // namespace hs

extern "C" {

size_t hs_attn_weights_workspace_bytes(int32_t B, int32_t S, int32_t Hq, int32_t Hkv, int32_t D, int32_t max_seq_len) {
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128 && D != 256) || max_seq_len <= 0) return 0;
    return (hs::most_floats(B, S, Hq, Hkv, D, max_seq_len) * sizeof(float) + 255) / 256 * 256;
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
    if (layout->k_block_table && (layout->capacity_tokens % kWStep) != 0)  // a step reads 64 tokens of one block
        return fail(HS_ERR_INVALID_ARGUMENT, "paged blocks must hold a multiple of %d tokens", kWStep);
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
    const size_t need = (p.ml_floats + p.lse_floats + p.w_floats) * sizeof(float);  // (of this call; the size function's answer covers smaller ones)
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
    a.cols = (int)p.cols; a.lse_stride = (int)p.lse_stride; a.max_seq_len = max_seq_len;
    a.window = layout->prefill_window; a.sinks = std::min(layout->attn_sinks, max_seq_len);
    a.joins = p.narrow && p.key_chunks > 1 && p.key_chunks * p.cols <= kJoinMost;
    a.key_chunks = p.key_chunks; a.chunk_tokens = p.chunk_tokens; a.segments = p.segments;
    a.scale_log2e = softmax_scale * kWLog2e;
    hipStream_t st = (hipStream_t)stream;
    if (D == 64) fp8 ? launch_weights<64, true>(a, p, st) : launch_weights<64, false>(a, p, st);
    else if (D == 128) fp8 ? launch_weights<128, true>(a, p, st) : launch_weights<128, false>(a, p, st);
    else fp8 ? launch_weights<256, true>(a, p, st) : launch_weights<256, false>(a, p, st);
    return check_launch("attn_weights");
}

}  // extern "C"
