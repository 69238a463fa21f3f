// Launches of the tcgen05 prefill kernel in its packed form (packed.cuh), for the two operators that use it.
#pragma once
#include "prefill_tc.cuh"
#include <cmath>

namespace b200p {

// Rows of a tensor at most: counts of rows are rounded up to tiles, and of tiles to levels of work (packed_walk), in 32 bits.
constexpr int kMostRows = 0x7fffffff - 0xffff;

// Query tiles that all the sequences have at most, over all key heads: each may end inside one.
inline long long packed_tiles(long long rows, int batch, int tokens, int kv_heads) { return (rows / tokens + batch) * kv_heads; }

// Everything of p but the launch's own fields (tokens, sticky; span where it is 0) is set.
template <typename T, int D, bool PARTIAL, bool WALK>
int launch_packed(PackedParams p, int dtype, cudaStream_t st) {
    using Sh = PackedShape<D, PARTIAL, WALK>;
    const CUtensorMapDataType dt = dtype == B200P_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    p.tokens = kBM / p.group;
    const int sms = sm_count();
    const long long tiles = packed_tiles(p.seqQ, p.batch, p.tokens, p.nKVH) * p.splits;
    if (p.span == 0) p.span = tiles <= sms ? 1 : 2;            // a tile alone takes 0.6 of a pair's time (prefill.cu)
    const int block = p.span * p.tokens;
    const long long items = (WALK ? packed_tiles(p.seqQ, p.batch, block, p.nKVH) : (long long)((p.seqQ + block - 1) / block) * p.nKVH) * p.splits;
    if (items > (1 << 29)) return B200P_E_RANGE;
    CUtensorMap mq, mk, mv;
    auto rows_map = [&](CUtensorMap* m, const void* base, long long token, long long head) {      // [head of a group][token][group]
        const uint64_t dims[4] = {uint64_t(D), uint64_t(p.group), uint64_t(p.seqQ), uint64_t(p.nKVH)};
        const uint64_t strides[3] = {uint64_t(head) * 2, uint64_t(token) * 2, uint64_t(head) * p.group * 2};
        const uint32_t box[4] = {64, uint32_t(p.group), uint32_t(p.tokens), 1};
        return make_tensor_map(m, dt, 4, base, dims, strides, box, Swizzle::B128);
    };
    auto keys_map = [&](CUtensorMap* m, const void* base, long long token, long long head) {
        const uint64_t dims[4] = {uint64_t(D), uint64_t(p.seqK > 0 ? p.seqK : 1), uint64_t(p.nKVH), 1};
        const uint64_t strides[3] = {uint64_t(token) * 2, uint64_t(head) * 2, uint64_t(head) * p.nKVH * 2};
        const uint32_t box[4] = {64, 128, 1, 1};
        return make_tensor_map(m, dt, 4, p.seqK > 0 ? base : p.Q, dims, strides, box, Swizzle::B128);
    };
    cudaError_t e = rows_map(&mq, p.Q, p.q_token, p.q_head);
    if (e == cudaSuccess) e = keys_map(&mk, p.K, p.k_token, p.k_head);
    if (e == cudaSuccess) e = keys_map(&mv, p.V, p.v_token, p.v_head);
    if (e != cudaSuccess) return int(e);
    auto kern = prefill_tc_kernel<T, Sh, 1, false>;
    if (int ae = allow_dynamic_smem(reinterpret_cast<const void*>(kern), Sh::SMEM_BYTES)) return ae;
    p.o_wide = aligned(p.O, 32) && p.o_token % 16 == 0 && p.o_head % 16 == 0;
    p.sticky = device_status_ptr();
    if (!p.sticky) return B200P_E_NO_DEVICE;
    p.items = int(items);
    // the items of one sequence are alike: a CTA per SM with a fixed share
    const long long ctas = !WALK && items > sms ? sms : items;
    kern<<<unsigned(ctas), prefill_threads(1), Sh::SMEM_BYTES, st>>>(p, mq, mk, mv, mq, mq, mk);
    return launched();
}

// ---- parts of rows (the splits' results) into the rows' results ------------------------------------------
constexpr int kMostParts = 160;
constexpr int kMergeWarps = 4;
constexpr int kFewParts = 12;

__device__ __forceinline__ float weight_of(float m, float most) { return exp2f(m - (most == -INFINITY ? 0.f : most)); }

// From L2.  Volatile: a load must not move behind the test whether its part counts, or each waits for the one before it.
template <int E> __device__ __forceinline__ void load_part(const float* at, float (&v)[E]) {
    static_assert(E == 2 || E == 4);
    if constexpr (E == 4) asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "l"(at) : "memory");
    else asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "l"(at) : "memory");
}

// The weight of a part with maximum and sum `ml` beside the maximum of all, or kNoKey for a part without keys, whose O is not stored.  Any other part
// counts, with a weight of 0 too: where its keys gave no number its maximum may be -inf, or far below the others', and what is no number
// is none in the row, as it is without splits.
__device__ __forceinline__ float part_weight(float2 ml, float most) { return ml.y == kNoKey ? kNoKey : weight_of(ml.x, most); }

// Row r = token * nQH + head from part_o[s][r][D] and part_ml[s][r].  m = max m_s, O = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s;
// parts without a key do not count, a row without any gives zeros.  first, last: device words with the first row to be written and the one
// behind the last, in tokens, or null.  A warp per row; or, for few rows and for many parts (launch_merge), four that take every fourth part.
template <typename T, int D, bool MANY>
__global__ void __launch_bounds__(kMergeWarps * 32)
merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, int parts, int tokens, int nQH, T* __restrict__ o, long long o_token, long long o_head,
             const int* first, const int* last) {
    constexpr int E = D / 32, P = ((MANY ? kMostParts : kFewParts) + 31) / 32, STEP = MANY ? kMergeWarps : 1;
    __shared__ float s_f[kMergeWarps][32 * P];
    __shared__ float s_x[MANY ? kMergeWarps : 1][MANY ? D : 1];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, row = MANY ? blockIdx.x : blockIdx.x * kMergeWarps + warp, rows = tokens * nQH, token = row / nQH;
    griddep_wait();
    if (row >= rows || (first && (token < *first || token >= *last))) return;
    float2 ml[P];
    float most = -INFINITY;
    bool some = false;
    #pragma unroll
    for (int k = 0; k < P; ++k) {
        const int s = 32 * k + lane;
        ml[k] = s < parts ? __ldcg(reinterpret_cast<const float2*>(&part_ml[2 * (size_t(s) * rows + row)])) : make_float2(-INFINITY, kNoKey);
        most = fmaxf(most, ml[k].x);
        some |= ml[k].y != kNoKey;
    }
    #pragma unroll
    for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    some = __any_sync(0xffffffffu, some);
    float sum = 0.f;
    #pragma unroll
    for (int k = 0; k < P; ++k) {
        const float f = part_weight(ml[k], most);
        if (f != kNoKey) sum += f * ml[k].y;
        s_f[warp][32 * k + lane] = f;
    }
    #pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    __syncwarp();
    float x[E] = {};
    #pragma unroll 8
    for (int s = MANY ? warp : 0; s < parts; s += STEP) {
        float v[E];
        load_part<E>(part_o + (size_t(s) * rows + row) * D + lane * E, v);
        const float f = s_f[warp][s];
        #pragma unroll
        for (int e = 0; e < E; ++e) if (f != kNoKey) x[e] += f * v[e];
    }
    if constexpr (MANY) {
        #pragma unroll
        for (int e = 0; e < E; ++e) s_x[warp][lane * E + e] = x[e];
        __syncthreads();
        if (warp > 0) return;
        #pragma unroll
        for (int k = 1; k < kMergeWarps; ++k)
            #pragma unroll
            for (int e = 0; e < E; ++e) x[e] += s_x[k][lane * E + e];
    }
    const float inv = some ? 1.f / sum : 0.f;               // nothing but scores of -inf: 0 / 0
    T* y = o + token * o_token + (row - token * nQH) * o_head + lane * E;
    if constexpr (E == 4) *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(x[0] * inv, x[1] * inv), pack2<T>(x[2] * inv, x[3] * inv));
    else *reinterpret_cast<uint32_t*>(y) = pack2<T>(x[0] * inv, x[1] * inv);
}

// A launch that may get ready while the stream's last one runs (it calls griddep_wait for its results).
template <typename... P, typename... A>
int launch_after(void (*kern)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(unsigned(threads)); cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr; cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) { cudaGetLastError(); return int(e); }
    return launched();
}

template <typename T, int D>
int launch_merge(const float* part_o, const float* part_ml, int parts, int tokens, int nQH, void* o, long long o_token, long long o_head, const int* first, const int* last,
                 cudaStream_t st) {
    if (parts > kMostParts) return B200P_E_RANGE;
    // A part's load is L2 latency, which few rows have few warps to hide.  Whole calls of decode behind a prefix, a warp and four per row, us: 32 rows
    // of 86 parts 18.8 and 10.4; 102 of 12 11.6 and 9.9; 1536 of 9 19.2 and 18.7; but 948 of 3 10.7 and 11.2; 3360 of 8 22.8 and 25.2; 8192 of 5 140 and 145.
    const long long rows = (long long)tokens * nQH, ctas = (rows + kMergeWarps - 1) / kMergeWarps;
    if (parts <= kFewParts && rows > 220LL * parts)
        return launch_after(merge_kernel<T, D, false>, dim3(unsigned(ctas)), kMergeWarps * 32, st, part_o, part_ml, parts, tokens, nQH, static_cast<T*>(o), o_token, o_head, first, last);
    return launch_after(merge_kernel<T, D, true>, dim3(unsigned(rows)), kMergeWarps * 32, st, part_o, part_ml, parts, tokens, nQH, static_cast<T*>(o), o_token, o_head, first, last);
}

} // namespace b200p
