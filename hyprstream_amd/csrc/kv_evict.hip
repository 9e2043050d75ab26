// Eviction from the quantized cache: every (sequence, kv-head) keeps its first tokens, its last ones and the heaviest of
// those between, moved to the front in their order.
//
// Two launches.  evict_select_kernel, one workgroup per (sequence, kv-head), finds the weight of the last token that
// stays (a radix selection: three digits of the weight's bits, most significant first) and lists the tokens that stay in
// order; it also moves their weights.  evict_move_kernel copies the listed code rows and scales, tiles of tokens in
// parallel; evict_inplace_kernel does the same inside one buffer, where a tile may only be overwritten once it has been
// read, with one workgroup per (sequence, kv-head, tensor) that walks its tiles in order.
//
// 64 x 8 rows of 8192 tokens cut to 1024 (D = 128; 300 MB of weights, kept rows read and written): 14 us of selection and 53
// of copy at 5.3 TB/s.  8 rows of 32768 cut to 4096: 23 us, one workgroup's chain of passes over a row, and 4 of copy.
// Caches and weights flushed by other work before every call: 92 us for the first (in place 90), 39 for the second (in place
// 73: two workgroups a row walk its tiles in order), 8 rows of 131072 cut to 16384 153 (in place 300).
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace hs {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

struct EvictArgs {
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    uint8_t *kco, *vco;
    float *kso, *vso;
    KvAddr ka, va, kao, vao;
    const int32_t *seq_lens;
    int32_t *seq_lens_out;
    const float *w;
    float *wo;
    int64_t w_stride, wo_stride;
    int32_t *kept;      // caller's list or nullptr
    int32_t *list;      // workspace [B, Hkv, budget]
    int32_t *info;      // workspace [B, Hkv, 2]: tokens kept, first list entry that moves
    int32_t budget, sinks, recent, Hkv, max_seq_len, fp8;
    int32_t finish;     // entries per row of kept and weights_out that are written
};

// Weights as unsigned integers in the same order: NaN below everything, the two zeros equal.
__device__ __forceinline__ uint32_t weight_key(float f) {
    if (f != f) return 0u;
    const uint32_t u = f == 0.0f ? 0u : __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// What goes with the codes of list entries [i0, i1): the caller's list, the weights and the zeros behind them (weights in
// place have been moved by the selection).  `threads` threads take part.
__device__ __forceinline__ void finish_rows(const EvictArgs &a, int64_t row, int n, int i0, int i1, int tid, int threads) {
    const int32_t *list = a.list + row * a.budget;
    const bool move_weights = a.wo != nullptr && a.w != a.wo;
    if (!move_weights && a.kept == nullptr) return;
    const int64_t w_end = min(a.wo_stride, (int64_t)a.max_seq_len);
    for (int i = i0 + tid; i < i1; i += threads) {
        const int t = i < n ? list[i] : -1;
        if (a.kept && i < a.budget) a.kept[row * a.budget + i] = t;
        if (move_weights && i < w_end) a.wo[row * a.wo_stride + i] = t >= 0 && a.w ? a.w[row * a.w_stride + t] : 0.0f;
    }
}

// Codes and scales of list entries [i0, i0 + TOKENS) of a row, by THREADS threads.
template <int D, int THREADS, int TOKENS>
__device__ __forceinline__ void move_tile(const EvictArgs &a, int64_t row, int b, int h, int n, int i0, int tid) {
    constexpr int LPR = D / 16, RPP = THREADS / LPR, PASSES = TOKENS / RPP;  // lanes per row, rows per pass
    const int32_t *list = a.list + row * a.budget;
    const int sub = tid % LPR, r = tid / LPR;
    u32x4 k[PASSES], v[PASSES];
    bool ok[PASSES];
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int i = i0 + p * RPP + r;
        int64_t ku, vu;
        int kslot, vslot;
        const int t = i < n ? list[i] : -1;
        const bool k_ok = resolve(a.ka, b, t, ku, kslot), v_ok = resolve(a.va, b, t, vu, vslot);
        ok[p] = k_ok && v_ok;
        if (ok[p]) {
            k[p] = *((const u32x4 *)(a.kc + ku * a.ka.code_stride_seq + (int64_t)h * a.ka.code_stride_head + (int64_t)kslot * D + 16 * sub));
            v[p] = *((const u32x4 *)(a.vc + vu * a.va.code_stride_seq + (int64_t)h * a.va.code_stride_head + (int64_t)vslot * D + 16 * sub));
        }
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int i = i0 + p * RPP + r;
        int64_t ku, vu;
        int kslot, vslot;
        const bool k_ok = resolve(a.kao, b, i, ku, kslot), v_ok = resolve(a.vao, b, i, vu, vslot);
        if (ok[p] && k_ok && v_ok) {
            __builtin_nontemporal_store(k[p], (u32x4 *)(a.kco + ku * a.kao.code_stride_seq + (int64_t)h * a.kao.code_stride_head + (int64_t)kslot * D + 16 * sub));
            __builtin_nontemporal_store(v[p], (u32x4 *)(a.vco + vu * a.vao.code_stride_seq + (int64_t)h * a.vao.code_stride_head + (int64_t)vslot * D + 16 * sub));
        }
    }
    if (!a.fp8 && tid < 2 * TOKENS) {  // the K scales of the tile, then its V scales
        const int i = i0 + (tid & (TOKENS - 1)), which = tid / TOKENS;
        const KvAddr &src = which ? a.va : a.ka, &dst = which ? a.vao : a.kao;
        int64_t u;
        int slot;
        if (i < n && resolve(src, b, list[i], u, slot)) {
            const float s = (which ? a.vs : a.ks)[u * src.scale_stride_seq + (int64_t)h * src.scale_stride_head + slot];
            if (resolve(dst, b, i, u, slot)) (which ? a.vso : a.kso)[u * dst.scale_stride_seq + (int64_t)h * dst.scale_stride_head + slot] = s;
        }
    }
}

// Inclusive sum over the wavefront's lanes on the vector pipe (row shifts inside sixteen lanes, then the broadcasts of
// lane 15 and of lane 31): six dependent additions instead of six trips through the LDS crossbar.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
#define HS_DPP_ADD(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false)
    HS_DPP_ADD(0x111, 0xf);  // row_shr:1
    HS_DPP_ADD(0x112, 0xf);  // row_shr:2
    HS_DPP_ADD(0x114, 0xf);  // row_shr:4
    HS_DPP_ADD(0x118, 0xf);  // row_shr:8
    HS_DPP_ADD(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    HS_DPP_ADD(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef HS_DPP_ADD
    return v;
}
// One workgroup per row.  The weights' keys go to LDS once (protected tokens take the largest key, so every pass is one
// comparison per token) and all passes read them there; a row longer than kTile tokens is read again for every pass, a
// tile at a time.  A row is a chain of short steps -- three histograms with a scan each, one scan for the list -- so what
// it costs is latency: the scans run on the vector pipe, a pass counts without branches (what it
// does not count goes to a place of the lane's own), and sixteen wavefronts hide each other's latencies (with four per
// row and 32 weights a thread: 25 us at 64 x 8 rows of 8192 tokens, 14 now).
constexpr uint32_t kProtected = 0xffffffffu, kZeroKey = 0x80000000u;
// Two workgroups share a CU where LDS lets them (64 registers: 14 us at 64 x 8 rows of 8192, 20 with 66).
// MOVE: head_dim of the codes if the workgroup goes on to move its row's tokens itself, 0 if evict_move_kernel does.
template <int TILE, int MOVE>
__global__ __launch_bounds__(1024, TILE == 8192 && MOVE == 0 ? 8 : 4) void evict_select_kernel(EvictArgs a) {
    constexpr int THREADS = 1024;
    constexpr uint32_t kCand = 1024;
    constexpr int kWaves = THREADS / 64, kGroup = 4 * THREADS, kGroups = TILE / kGroup, kCounts = kGroups * kWaves;
    static_assert(kCounts <= 128, "two counts per lane");
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = (int64_t)b * a.Hkv + h;
    const int L = min(max(a.seq_lens[b], 0), a.max_seq_len);
    const float *w = a.w ? a.w + row * a.w_stride : nullptr;
    int32_t *list = a.list + row * a.budget;
    __shared__ __attribute__((aligned(16))) uint32_t sm_key[TILE], sm_hist[2048 + 64];  // bins, and a place per lane for what is not counted
    __shared__ uint32_t sm_list[kCand], sm_wave[4], sm_pick[3], sm_cand, sm_cnt[kCounts], sm_pre[kCounts + 1];
    __shared__ int sm_first;
    const int n = min(L, a.budget);
    if (L <= a.budget || w == nullptr) {
        // nothing to choose: everything, or the sinks and the newest
        const int s = L <= a.budget ? n : a.sinks;
        for (int i = tid; i < n; i += THREADS) list[i] = i < s ? i : L - n + i;
        if (tid == 0) sm_first = s;
    } else {
        const int lo = a.sinks, hi = L - a.recent, K = a.budget - a.sinks - a.recent;
        const int tiles = TILE == 8192 ? 1 : (L + TILE - 1) / TILE;  // (the small tile serves max_seq_len <= 8192)
        // keys of the tile that starts at `base`: every thread reads back only what it wrote.  Tokens behind the row
        // take key 0: the lowest one, and last among its equals.
        auto load = [&](int base) {
            float4v x[kGroups];
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                const int t = base + i * kGroup + 4 * tid;
                x[i] = t < L ? *(const float4v *)(w + t) : (float4v){0.f, 0.f, 0.f, 0.f};  // rows are a multiple of four long
            }
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                u32x4 k;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = base + i * kGroup + 4 * tid + e;
                    k[e] = t >= L ? 0u : t < lo || t >= hi ? kProtected : weight_key(x[i][e]);
                }
                *(u32x4 *)&sm_key[i * kGroup + 4 * tid] = k;
            }
        };
        if (tid == 0) sm_first = n;
        load(0);
        // ---- key of the K-th heaviest token of [lo, hi), three digits of 11, 11 and 10 bits; `need` of those that share
        //      it stay, the lowest positions first.  The keys that share the first digit are few as a rule: they are put
        //      together and the other digits found among them, unless they are more than kCand.
        uint32_t prefix = K > 0 ? 0u : kProtected - 1, need = (uint32_t)K, cand = kCand + 1;
#pragma unroll 1
        for (int shift = 21; K > 0; shift = shift == 21 ? 10 : 0) {
            const uint32_t mask = shift == 0 ? 1023u : 2047u, fixed = shift == 21 ? 0u : shift == 10 ? 0xffe00000u : 0xfffffc00u;
            if (tid < 512) *(u32x4 *)&sm_hist[4 * tid] = (u32x4){0u, 0u, 0u, 0u};
            if (tid == 0) sm_cand = 0;
            __syncthreads();
            if (cand <= kCand) {
                for (uint32_t i = tid; i < cand; i += THREADS) {
                    const uint32_t k = sm_list[i];
                    if (((k ^ prefix) & fixed) == 0u) atomicAdd(&sm_hist[(k >> shift) & mask], 1u);
                }
            } else {
                uint32_t zeros = 0;  // tokens without any weight are many and would queue at one counter
                auto count = [&](auto first_tag) {
                    constexpr bool kFirst = decltype(first_tag)::value;
#pragma unroll 1
                    for (int tile = 0; tile < tiles; ++tile) {
                        if (tiles > 1) load(tile * TILE);
                        const int left = L - tile * TILE - 4 * tid;  // tokens of the row from this thread's first one on
#pragma unroll
                        for (int i = 0; i < kGroups; ++i) {
                            if (i * kGroup >= left) break;
                            const u32x4 k = *(const u32x4 *)&sm_key[i * kGroup + 4 * tid];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t own = 2048u + lane;
                                if constexpr (kFirst) {
                                    const bool none = k[e] == kZeroKey;
                                    zeros += none ? 1u : 0u;
                                    atomicAdd(&sm_hist[k[e] != kProtected && !none && i * kGroup + e < left ? k[e] >> 21 : own], 1u);
                                } else {
                                    // more than kCand keys share the first digit: often they are all equal, so lane 0 (whose
                                    // tokens come first: it is there while any is) counts for every lane that shares its bin
                                    // (8 rows of 32768, 1 % of them with a weight: 77 us without, 31 with; the first pass,
                                    // where weights differ, loses 1 us of 26 to it)
                                    const bool counts = k[e] != kProtected && ((k[e] ^ prefix) & fixed) == 0u && i * kGroup + e < left;
                                    const uint32_t bin = counts ? (k[e] >> shift) & mask : own;
                                    const bool led = bin == (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
                                    const uint32_t many = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(led));
                                    atomicAdd(&sm_hist[led && lane != 0 ? own : bin], lane == 0 ? many : 1u);
                                }
                            }
                        }
                    }
                };
                if (shift == 21) count(std::true_type{});
                else count(std::false_type{});
                if (shift == 21) {
                    zeros = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(zeros), 63);
                    if (lane == 0 && zeros != 0) atomicAdd(&sm_hist[kZeroKey >> 21], zeros);
                }
            }
            __syncthreads();
            // the digit at which the count from the top reaches `need`: eight bins for each thread of the first four
            // wavefronts, thread i those below 2048 - 8 i
            uint32_t bin[8], sum = 0, incl = 0;
            if (wave < 4) {
                const u32x4 b0 = *(const u32x4 *)&sm_hist[2040 - 8 * tid], b1 = *(const u32x4 *)&sm_hist[2044 - 8 * tid];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bin[e] = b0[e];
                    bin[4 + e] = b1[e];
                    sum += b0[e] + b1[e];
                }
                incl = wave_scan(sum);
                if (lane == 63) sm_wave[wave] = incl;
            }
            __syncthreads();
            if (wave < 4) {
                for (int v = 0; v < wave; ++v) incl += sm_wave[v];
                uint32_t excl = incl - sum;
                if (excl < need && need <= incl) {
#pragma unroll
                    for (int e = 7; e >= 0; --e) {
                        if (excl < need && need <= excl + bin[e]) {
                            sm_pick[0] = (uint32_t)(2040 - 8 * tid + e);
                            sm_pick[1] = need - excl;
                            sm_pick[2] = bin[e];
                        }
                        excl += bin[e];
                    }
                }
            }
            __syncthreads();
            prefix |= sm_pick[0] << shift;
            need = sm_pick[1];
            if (shift == 0) break;
            if (shift == 21 && tiles == 1 && sm_pick[2] <= kCand) {
                cand = sm_pick[2];
                const int left = L - 4 * tid;
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    if (i * kGroup >= left) break;
                    const u32x4 k = *(const u32x4 *)&sm_key[i * kGroup + 4 * tid];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if ((k[e] ^ prefix) < (1u << 21) && k[e] != kProtected && i * kGroup + e < left) sm_list[atomicAdd(&sm_cand, 1u)] = k[e];
                }
                __syncthreads();
            }
        }
        // ---- list, in order.  A token stays if its key is larger, or one of the first `need` equal ones.
        //      Counts travel in pairs: larger ones in the low half, ties in the high one (a tile holds at most 32768).
        uint32_t sure = 0, ties = 0;  // of the tiles before this one
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile) {
            if (tiles > 1) load(tile * TILE);
            const int base = tile * TILE, groups = (min(TILE, L - base) + kGroup - 1) / kGroup;
            auto pairs = [&](const u32x4 &k) {
                uint32_t c = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) c += k[e] > prefix ? 1u : k[e] == prefix ? 0x10000u : 0u;
                return c;
            };
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                if (i >= groups) break;
                const uint32_t incl = wave_scan(pairs(*(const u32x4 *)&sm_key[i * kGroup + 4 * tid]));
                if (lane == 63) sm_cnt[i * kWaves + wave] = incl;
            }
            __syncthreads();
            // counts in the order of the tokens: entry i * kWaves + wave; the first wavefront sums them up
            if (wave == 0) {
                const uint32_t c0 = 2 * lane < groups * kWaves ? sm_cnt[2 * lane] : 0u, c1 = 2 * lane + 1 < groups * kWaves ? sm_cnt[2 * lane + 1] : 0u;
                const uint32_t incl = wave_scan(c0 + c1);
                if (2 * lane < kCounts) {
                    sm_pre[2 * lane + 1] = incl - c1;
                    sm_pre[2 * lane + 2] = incl;
                }
                if (lane == 0) sm_pre[0] = 0;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kGroups; ++i) {
                if (i >= groups) break;
                const int g = i * kGroup + 4 * tid;
                const u32x4 k = *(const u32x4 *)&sm_key[g];
                const uint32_t cnt = pairs(k), before = sm_pre[i * kWaves + wave] + wave_scan(cnt) - cnt;
                uint32_t s = sure + (before & 0xffffu), q = ties + (before >> 16);
                bool gap = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool is_sure = k[e] > prefix, is_tie = k[e] == prefix;
                    if (is_sure || (is_tie && q < need)) {
                        list[s + min(q, need)] = base + g + e;
                    } else {
                        gap = true;
                    }
                    s += is_sure ? 1u : 0u;
                    q += is_tie ? 1u : 0u;
                }
                // the first list entry that moves is the first token that leaves; a lower bound at four tokens' grain
                const uint64_t gaps = __builtin_amdgcn_ballot_w64(gap);
                if (gaps != 0 && lane == 0) atomicMin(&sm_first, base + i * kGroup + 256 * wave + 4 * __builtin_ctzll(gaps));
            }
            const uint32_t all = sm_pre[groups * kWaves];
            sure += all & 0xffffu;
            ties += all >> 16;
            __syncthreads();  // sm_cnt and sm_pre may be written again
        }
    }
    // ---- weights in place (otherwise they move with their tokens): list[r] >= r, so a tile of them overwrites nothing that
    //      later ones read; then the tail, and the row's counts
    __syncthreads();
    if (a.w && a.w == a.wo) {
        float *wo = a.wo + row * a.wo_stride;
        for (int r0 = 0; r0 < n; r0 += THREADS) {
            const float x = r0 + tid < n ? w[list[r0 + tid]] : 0.0f;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (r0 + tid < n) wo[r0 + tid] = x;
        }
        __syncthreads();
        for (int64_t i = n + tid; i < min(a.wo_stride, (int64_t)a.max_seq_len); i += THREADS) wo[i] = 0.0f;
    }
    if constexpr (MOVE != 0) {
        __syncthreads();  // the list
        constexpr int kTokens = 2 * (THREADS / (MOVE / 16));
        if (h == 0 && tid == 0) a.seq_lens_out[b] = n;  // (the lengths the other heads read are another array)
        if (a.fp8 && tid < 2) (tid ? a.vso : a.kso)[row] = (tid ? a.vs : a.ks)[row];
        finish_rows(a, row, n, 0, a.finish, tid, THREADS);
        for (int i0 = 0; i0 < n; i0 += kTokens) move_tile<MOVE, THREADS, kTokens>(a, row, b, h, n, i0, tid);
    } else if (tid == 0) {
        a.info[2 * row] = n;
        a.info[2 * row + 1] = min(sm_first, n);
    }
}

// Tokens of a workgroup.  Few registers and many wavefronts beat more loads per thread: 64 x 8 rows of 1024 tokens (D = 128,
// 290 MB moved) take 53-55 us with 64 tokens, 63-66 with 128, 131 with 256.  Loads may hit what the last attention left in
// the caches (one stream of 32k tokens: 4.4 us, 6.1 with the streaming hint); stores stream past them.
constexpr int kMoveTokens = 64;

template <int D>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int64_t row = (int64_t)b * a.Hkv + h;
    const int n = a.info[2 * row], i0 = blockIdx.x * kMoveTokens;
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.seq_lens_out[b] = n;
    if (blockIdx.x == 0 && a.fp8 && tid < 2) (tid ? a.vso : a.kso)[row] = (tid ? a.vs : a.ks)[row];
    finish_rows(a, row, n, i0, (int)min((int64_t)i0 + kMoveTokens, (int64_t)a.finish), tid, 256);
    if (i0 < n) move_tile<D, 256, kMoveTokens>(a, row, b, h, n, i0, tid);
}

// In place: list[i] >= i, so a tile of destinations can only overlap sources of its own tile and of earlier ones.  Every
// tile is in registers (and the loads have returned) before the barrier behind which it is written.
template <int D>
__global__ __launch_bounds__(1024) void evict_inplace_kernel(EvictArgs a) {
    constexpr int LPR = D / 16, RPP = 1024 / LPR, U = 4;
    const int h = blockIdx.y, b = blockIdx.z, which = blockIdx.x, tid = threadIdx.x;
    const int64_t row = (int64_t)b * a.Hkv + h;
    const int n = a.info[2 * row], first = a.info[2 * row + 1];
    if (which == 0 && h == 0 && tid == 0) a.seq_lens_out[b] = n;
    if (which == 0) finish_rows(a, row, n, 0, a.finish, tid, 1024);
    const int32_t *list = a.list + row * a.budget;
    const KvAddr &ad = which ? a.va : a.ka;
    uint8_t *codes = which ? a.vco : a.kco;
    float *scales = which ? a.vso : a.kso;
    const int sub = tid % LPR, r = tid / LPR;
    for (int i0 = first; i0 < n; i0 += U * RPP) {
        u32x4 x[U];
        float s[U];
        bool ok[U];
#pragma unroll
        for (int p = 0; p < U; ++p) {
            const int i = i0 + p * RPP + r;
            int64_t u;
            int slot;
            ok[p] = resolve(ad, b, i < n ? list[i] : -1, u, slot);
            if (ok[p]) {
                x[p] = *(const u32x4 *)(codes + u * ad.code_stride_seq + (int64_t)h * ad.code_stride_head + (int64_t)slot * D + 16 * sub);
                if (!a.fp8 && sub == 0) s[p] = scales[u * ad.scale_stride_seq + (int64_t)h * ad.scale_stride_head + slot];
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int p = 0; p < U; ++p) {
            const int i = i0 + p * RPP + r;
            int64_t u;
            int slot;
            if (ok[p] && resolve(ad, b, i, u, slot)) {
                *(u32x4 *)(codes + u * ad.code_stride_seq + (int64_t)h * ad.code_stride_head + (int64_t)slot * D + 16 * sub) = x[p];
                if (!a.fp8 && sub == 0) scales[u * ad.scale_stride_seq + (int64_t)h * ad.scale_stride_head + slot] = s[p];
            }
        }
        // the next tile reads tokens behind everything written so far: no barrier is needed before its loads
    }
}

int validate_layout(const hs_kv_layout *l, int B, int S, int Hkv, int D, bool need_scales);

static bool same_storage(const hs_kv_layout &x, const hs_kv_layout &y) {
    return x.code_stride_seq == y.code_stride_seq && x.code_stride_head == y.code_stride_head &&
           x.scale_stride_seq == y.scale_stride_seq && x.scale_stride_head == y.scale_stride_head &&
           x.capacity_tokens == y.capacity_tokens && x.block_table_stride == y.block_table_stride &&
           x.k_block_table == y.k_block_table && x.v_block_table == y.v_block_table;
}

static int64_t capacity(const hs_kv_layout &l) {
    return l.k_block_table ? (int64_t)l.capacity_tokens * l.block_table_stride : l.capacity_tokens;
}

}  // namespace hs

extern "C" {

size_t hs_kv_evict_workspace_bytes(int32_t B, int32_t Hkv, int32_t budget, int32_t max_seq_len) {
    if (B <= 0 || Hkv <= 0 || budget <= 0 || max_seq_len <= 0) return 0;
    return ((size_t)B * Hkv * ((size_t)budget + 2) * sizeof(int32_t) + 255) / 256 * 256;
}

int hs_kv_evict(int fmt_fp8, const void *k_codes, const void *v_codes, const float *k_scales, const float *v_scales,
                const hs_kv_layout *layout, const int32_t *seq_lens, const float *weights, int64_t weights_stride,
                void *k_codes_out, void *v_codes_out, float *k_scales_out, float *v_scales_out,
                const hs_kv_layout *layout_out, int32_t *seq_lens_out, float *weights_out, int64_t weights_out_stride,
                int32_t *kept, int32_t budget, int32_t sinks, int32_t recent, void *workspace, size_t workspace_bytes,
                int32_t B, int32_t Hkv, int32_t D, int32_t max_seq_len, hs_stream_t stream) {
    using namespace hs;
    const bool fp8 = fmt_fp8 != 0;
    if (int rc = validate_layout(layout, B, 0, Hkv, D, !fp8)) return rc;
    if (int rc = validate_layout(layout_out, B, 0, Hkv, D, !fp8)) return rc;
    if (max_seq_len <= 0) return fail(HS_ERR_INVALID_ARGUMENT, "max_seq_len must be positive");
    if (budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
        return fail(HS_ERR_INVALID_ARGUMENT, "need budget > 0 and 0 <= sinks + recent <= budget (budget=%d sinks=%d recent=%d)",
                    budget, sinks, recent);
    if (max_seq_len > capacity(*layout))
        return fail(HS_ERR_OVERFLOW, "max_seq_len %d exceeds what the cache can hold (%lld tokens)", max_seq_len,
                    (long long)capacity(*layout));
    if (std::min(budget, max_seq_len) > capacity(*layout_out))
        return fail(HS_ERR_OVERFLOW, "the cache the tokens go to holds %lld tokens, the budget is %d",
                    (long long)capacity(*layout_out), budget);
    if (B == 0) return HS_OK;
    if (B > 65535 || Hkv > 65535) return fail(HS_ERR_INVALID_ARGUMENT, "at most 65535 sequences and kv-heads (B=%d Hkv=%d)", B, Hkv);
    if (!k_codes || !v_codes || !k_scales || !v_scales || !seq_lens || !k_codes_out || !v_codes_out || !k_scales_out ||
        !v_scales_out || !seq_lens_out)
        return fail(HS_ERR_INVALID_ARGUMENT, "null buffer");
    if ((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_codes_out | (uintptr_t)v_codes_out) & 15) != 0 ||
        ((layout->code_stride_seq | layout_out->code_stride_seq) & 15) != 0)
        return fail(HS_ERR_INVALID_ARGUMENT, "code buffers and their strides must be 16-byte aligned");
    if (weights && ((((uintptr_t)weights) & 15) != 0 || (weights_stride & 3) != 0))
        return fail(HS_ERR_INVALID_ARGUMENT, "weights must be 16-byte aligned, with a stride that is a multiple of 4");
    if (weights && weights_stride < max_seq_len)
        return fail(HS_ERR_OVERFLOW, "weights_stride %lld is below max_seq_len %d", (long long)weights_stride, max_seq_len);
    if (weights_out && ((((uintptr_t)weights_out) & 15) != 0 || (weights_out_stride & 3) != 0))
        return fail(HS_ERR_INVALID_ARGUMENT, "weights_out must be 16-byte aligned, with a stride that is a multiple of 4");
    if (weights_out && weights_out_stride < std::min(budget, max_seq_len))
        return fail(HS_ERR_OVERFLOW, "weights_out_stride %lld is below the budget %d", (long long)weights_out_stride, budget);
    if (weights && weights_out == weights && weights_out_stride != weights_stride)
        return fail(HS_ERR_INVALID_ARGUMENT, "weights in place need one stride, got %lld and %lld", (long long)weights_stride,
                    (long long)weights_out_stride);
    const size_t need = hs_kv_evict_workspace_bytes(B, Hkv, budget, max_seq_len);
    if (!workspace || workspace_bytes < need)
        return fail(HS_ERR_WORKSPACE, "workspace of %zu bytes given, %zu needed", workspace_bytes, need);
    if (((uintptr_t)workspace & 255) != 0) return fail(HS_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    // the same buffers through the same tables and strides: in place.  The same buffers in another way is only possible
    // through block tables, whose blocks the caller keeps apart.
    const bool all = k_codes_out == k_codes && v_codes_out == v_codes && k_scales_out == k_scales && v_scales_out == v_scales;
    const bool any = k_codes_out == k_codes || v_codes_out == v_codes || k_codes_out == v_codes || v_codes_out == k_codes;
    const bool in_place = all && same_storage(*layout, *layout_out);
    if (any && !in_place && !(layout->k_block_table && layout_out->k_block_table &&
                              layout->k_block_table != layout_out->k_block_table && layout->v_block_table != layout_out->v_block_table))
        return fail(HS_ERR_INVALID_ARGUMENT,
                    "a cache evicted into its own buffers needs the same buffers, tables and strides on both sides, or "
                    "block tables of its own");
    if (!fp8 && !in_place && !any && (k_scales_out == k_scales || v_scales_out == v_scales || k_scales_out == v_scales || v_scales_out == k_scales))
        return fail(HS_ERR_INVALID_ARGUMENT, "codes and scales must both stay or both move");
    EvictArgs a;
    a.kc = (const uint8_t *)k_codes; a.vc = (const uint8_t *)v_codes;
    a.ks = k_scales; a.vs = v_scales;
    a.kco = (uint8_t *)k_codes_out; a.vco = (uint8_t *)v_codes_out;
    a.kso = k_scales_out; a.vso = v_scales_out;
    a.ka = make_addr(*layout, 0); a.va = make_addr(*layout, 1);
    a.kao = make_addr(*layout_out, 0); a.vao = make_addr(*layout_out, 1);
    a.seq_lens = seq_lens; a.seq_lens_out = seq_lens_out;
    a.w = weights; a.wo = weights_out;
    a.w_stride = weights_stride; a.wo_stride = weights_out_stride;
    a.kept = kept;
    a.list = (int32_t *)workspace;
    a.info = a.list + (size_t)B * Hkv * budget;
    a.budget = budget; a.sinks = sinks; a.recent = recent;
    a.Hkv = Hkv; a.max_seq_len = max_seq_len; a.fp8 = fp8 ? 1 : 0;
    a.finish = std::max(std::min(budget, max_seq_len), kept ? budget : 0);
    if (weights_out) a.finish = std::max<int64_t>(a.finish, std::min<int64_t>(weights_out_stride, max_seq_len));
    hipStream_t st = (hipStream_t)stream;
    // One launch where there is little to move: a workgroup per row then moves its tokens itself.  (5 x 4 rows of 512 tokens
    // of 64 codes: a call every 11.3 us, 15.7 in two launches, whose second one costs the host as much as the GPU; 64 x 8
    // rows of 1024 tokens of 128: 73.6 us of kernel against 68.9; 8 rows of 4096 tokens: 51 against 34.)
    const int64_t row_bytes = (int64_t)a.finish * D;
    const bool one = !in_place && seq_lens_out != seq_lens && row_bytes <= 65536 && (int64_t)B * Hkv * row_bytes <= (8 << 20);
#define HS_EVICT_SELECT(M)                                                                          \
    do {                                                                                            \
        if (max_seq_len <= 8192) evict_select_kernel<8192, M><<<dim3(Hkv, B), 1024, 0, st>>>(a);    \
        else evict_select_kernel<32768, M><<<dim3(Hkv, B), 1024, 0, st>>>(a);                       \
    } while (0)
    if (!one) HS_EVICT_SELECT(0);
    else if (D == 64) HS_EVICT_SELECT(64);
    else if (D == 128) HS_EVICT_SELECT(128);
    else HS_EVICT_SELECT(256);
#undef HS_EVICT_SELECT
    if (int rc = check_launch("kv_evict (selection)")) return rc;
    if (one) return HS_OK;
    if (in_place) {
        const dim3 grid(2, Hkv, B);
        if (D == 64) evict_inplace_kernel<64><<<grid, 1024, 0, st>>>(a);
        else if (D == 128) evict_inplace_kernel<128><<<grid, 1024, 0, st>>>(a);
        else evict_inplace_kernel<256><<<grid, 1024, 0, st>>>(a);
    } else {
        const dim3 grid((unsigned)(((int64_t)a.finish + kMoveTokens - 1) / kMoveTokens), Hkv, B);
        if (D == 64) evict_move_kernel<64><<<grid, 256, 0, st>>>(a);
        else if (D == 128) evict_move_kernel<128><<<grid, 256, 0, st>>>(a);
        else evict_move_kernel<256><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("kv_evict (move)");
}

}  // extern "C"
