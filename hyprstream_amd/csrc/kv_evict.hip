// Eviction from the quantized cache: every (sequence, kv-head) keeps its first tokens, its last ones and the heaviest of
// those between, moved to the front in their order.
//
// Two launches.  evict_select_kernel, one workgroup per (sequence, kv-head), finds the weight of the last token that
// stays (a radix selection: three digits of the weight's bits, most significant first) and lists the tokens that stay in
// order; it also moves their weights.  evict_move_kernel copies the listed code rows and scales, tiles of tokens in
// parallel; evict_inplace_kernel does the same inside one buffer, where a tile may only be overwritten once it has been
// read, with one workgroup per (sequence, kv-head, tensor) that walks its tiles in order.
#include <algorithm>

#include "common.hpp"

namespace hs {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr int kSelectThreads = 1024;

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
    int32_t budget, sinks, recent, Hkv, D, max_seq_len, fp8;
};

// Weights as unsigned integers in the same order: NaN below everything, the two zeros equal.
__device__ __forceinline__ uint32_t weight_key(float f) {
    if (f != f) return 0u;
    const uint32_t u = f == 0.0f ? 0u : __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Inclusive scan over the workgroup of a packed pair of counts (no carry between the halves: tiles hold 4096 tokens).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *sm_wave, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(v, o, 64);
        if (lane >= o) v += up;
    }
    if (lane == 63) sm_wave[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const uint32_t c = sm_wave[w];
        if (w < wave) before += c;
        all += c;
    }
    total = all;
    __syncthreads();  // sm_wave may be written again
    return v + before;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int64_t row = (int64_t)b * a.Hkv + h;
    const int L = min(max(a.seq_lens[b], 0), a.max_seq_len);
    const float *w = a.w ? a.w + row * a.w_stride : nullptr;
    float *wo = a.wo ? a.wo + row * a.wo_stride : nullptr;
    int32_t *list = a.list + row * a.budget, *kept = a.kept ? a.kept + row * a.budget : nullptr;
    __shared__ uint32_t sm_hist[2048], sm_wave[kSelectThreads / 64], sm_pick[3];
    const int n = min(L, a.budget);
    int first_moved = n;
    if (L <= a.budget || w == nullptr) {
        // nothing to choose: everything, or the sinks and the newest
        const int s = L <= a.budget ? n : a.sinks;
        for (int i = tid; i < a.budget; i += kSelectThreads) {
            const int t = i < s ? i : L - n + i;
            if (i < n) list[i] = t;
            if (kept) kept[i] = i < n ? t : -1;
            if (wo && i < n && !(w == wo)) wo[i] = w ? w[t] : 0.0f;
        }
        first_moved = L <= a.budget ? n : a.sinks;
    } else {
        const int lo = a.sinks, hi = L - a.recent, K = a.budget - a.sinks - a.recent;
        // ---- key of the K-th heaviest token of [lo, hi), three digits of 11, 11 and 10 bits; `need` of those that share
        //      it stay, the lowest positions first
        uint32_t prefix = 0, need = (uint32_t)K;
        if (K > 0) {
            const int shift[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                for (int i = tid; i < 2048; i += kSelectThreads) sm_hist[i] = 0;
                __syncthreads();
                const uint32_t mask = (1u << bits[p]) - 1;
                for (int t = lo + tid; t < hi; t += kSelectThreads) {
                    const uint32_t k = weight_key(w[t]);
                    if (p == 0 || (k >> (shift[p] + bits[p])) == (prefix >> (shift[p] + bits[p]))) atomicAdd(&sm_hist[(k >> shift[p]) & mask], 1u);
                }
                __syncthreads();
                // the digit at which the count from the top reaches `need`: thread i owns the two bins below 2048 - 2 i
                const int top = 2047 - 2 * tid;
                const uint32_t c1 = sm_hist[top], c0 = sm_hist[top - 1];
                uint32_t all;
                const uint32_t incl = block_scan(c1 + c0, sm_wave, all), excl = incl - c1 - c0;
                if (excl < need && need <= incl) {
                    const bool upper = excl + c1 >= need;
                    sm_pick[0] = upper ? top : top - 1;
                    sm_pick[1] = need - excl - (upper ? 0u : c1);
                }
                __syncthreads();
                prefix |= sm_pick[0] << shift[p];
                need = sm_pick[1];
                __syncthreads();
            }
        }
        // ---- list, in order.  A token stays if it is protected, heavier than the key, or one of the first `need` at it.
        uint32_t sure = 0, ties = 0;  // of the tiles before this one
        const int tiles = (L + 4 * kSelectThreads - 1) / (4 * kSelectThreads);
        for (int tile = 0; tile < tiles; ++tile) {
            const int t0 = tile * 4 * kSelectThreads + 4 * tid;
            float4v x = {0.f, 0.f, 0.f, 0.f};
            if (t0 < L) x = *(const float4v *)(w + t0);  // rows are a multiple of four long
            uint32_t own[4], cnt = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = t0 + e;
                const uint32_t k = weight_key(x[e]);
                const bool prot = t < L && (t < lo || t >= hi);
                const bool mid = K > 0 && t >= lo && t < hi;
                own[e] = prot || (mid && k > prefix) ? 1u : (mid && k == prefix ? 0x10000u : 0u);
                cnt += own[e];
            }
            uint32_t all;
            uint32_t at = block_scan(cnt, sm_wave, all) - cnt;
            uint32_t s = sure + (at & 0xffffu), q = ties + (at >> 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool stays = own[e] == 1u || (own[e] == 0x10000u && q < need);
                if (stays) {
                    const int r = (int)(s + min(q, need));
                    list[r] = t0 + e;
                    if (kept) kept[r] = t0 + e;
                    if (wo) wo[r] = x[e];  // in place: r <= t0 + e, and this tile has been read
                    if (r != t0 + e) first_moved = min(first_moved, r);
                }
                s += own[e] & 1u;
                q += own[e] >> 16;
            }
            sure += all & 0xffffu;
            ties += all >> 16;
        }
    }
    // ---- the tail of the weights and of the list, the row's counts
    __syncthreads();
    if (wo)
        for (int64_t i = n + tid; i < min(a.wo_stride, (int64_t)a.max_seq_len); i += kSelectThreads) wo[i] = 0.0f;
    if (tid == 0) sm_pick[2] = (uint32_t)n;
    __syncthreads();
    atomicMin(&sm_pick[2], (uint32_t)first_moved);
    __syncthreads();
    if (tid == 0) {
        a.info[2 * row] = n;
        a.info[2 * row + 1] = (int)sm_pick[2];
    }
}

constexpr int kMoveTokens = 128;  // tokens of a workgroup

template <int D>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a) {
    constexpr int LPR = D / 16, RPP = 256 / LPR, PASSES = kMoveTokens / RPP;  // lanes per row, rows per pass
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int64_t row = (int64_t)b * a.Hkv + h;
    const int n = a.info[2 * row];
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.seq_lens_out[b] = n;
    if (blockIdx.x == 0 && a.fp8 && tid < 2) (tid ? a.vso : a.kso)[row] = (tid ? a.vs : a.ks)[row];
    const int i0 = blockIdx.x * kMoveTokens;
    if (i0 >= n) return;
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
            k[p] = __builtin_nontemporal_load((const u32x4 *)(a.kc + ku * a.ka.code_stride_seq + (int64_t)h * a.ka.code_stride_head + (int64_t)kslot * D + 16 * sub));
            v[p] = __builtin_nontemporal_load((const u32x4 *)(a.vc + vu * a.va.code_stride_seq + (int64_t)h * a.va.code_stride_head + (int64_t)vslot * D + 16 * sub));
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
    if (!a.fp8) {  // threads 0..127 the K scales of the tile, 128..255 the V scales
        const int i = i0 + (tid & (kMoveTokens - 1)), which = tid / kMoveTokens;
        const KvAddr &src = which ? a.va : a.ka, &dst = which ? a.vao : a.kao;
        int64_t u;
        int slot;
        if (i < n && resolve(src, b, list[i], u, slot)) {
            const float s = (which ? a.vs : a.ks)[u * src.scale_stride_seq + (int64_t)h * src.scale_stride_head + slot];
            if (resolve(dst, b, i, u, slot)) (which ? a.vso : a.kso)[u * dst.scale_stride_seq + (int64_t)h * dst.scale_stride_head + slot] = s;
        }
    }
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
    a.Hkv = Hkv; a.D = D; a.max_seq_len = max_seq_len; a.fp8 = fp8 ? 1 : 0;
    hipStream_t st = (hipStream_t)stream;
    evict_select_kernel<<<dim3(Hkv, B), kSelectThreads, 0, st>>>(a);
    if (int rc = check_launch("kv_evict (selection)")) return rc;
    if (in_place) {
        const dim3 grid(2, Hkv, B);
        if (D == 64) evict_inplace_kernel<64><<<grid, 1024, 0, st>>>(a);
        else if (D == 128) evict_inplace_kernel<128><<<grid, 1024, 0, st>>>(a);
        else evict_inplace_kernel<256><<<grid, 1024, 0, st>>>(a);
    } else {
        const dim3 grid((std::min(budget, max_seq_len) + kMoveTokens - 1) / kMoveTokens, Hkv, B);
        if (D == 64) evict_move_kernel<64><<<grid, 256, 0, st>>>(a);
        else if (D == 128) evict_move_kernel<128><<<grid, 256, 0, st>>>(a);
        else evict_move_kernel<256><<<grid, 256, 0, st>>>(a);
    }
    return check_launch("kv_evict (move)");
}

}  // extern "C"
