// Launches of the tcgen05 prefill kernel in its packed form (packed.cuh), for the two operators that use it.
#pragma once
#include "prefill_tc.cuh"
#include <cmath>

namespace b200p {

// Query tiles that all the sequences have at most, over all key heads: each may end inside one.
inline long long packed_tiles(long long rows, int batch, int tokens, int kv_heads) { return (rows / tokens + batch) * kv_heads; }

// Everything of p but the launch's own fields (tokens, sticky; span where it is 0) is set.
template <typename T, int D, bool PARTIAL>
int launch_packed(PackedParams p, int dtype, cudaStream_t st) {
    using Sh = PackedShape<D, PARTIAL>;
    const CUtensorMapDataType dt = dtype == B200P_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    p.tokens = kBM / p.group;
    const int sms = sm_count();
    const long long tiles = packed_tiles(p.seqQ, p.batch, p.tokens, p.nKVH) * p.splits;
    if (p.span == 0) p.span = tiles <= sms ? 1 : 2;            // a tile alone takes 0.6 of a pair's time (prefill.cu)
    const int block = p.span * p.tokens;
    const long long items = PARTIAL ? (long long)((p.seqQ + block - 1) / block) * p.nKVH * p.splits : packed_tiles(p.seqQ, p.batch, block, p.nKVH);
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
    // PARTIAL items are alike, and a launch that waits for this one comes behind them: a CTA per SM with a fixed share
    const long long ctas = PARTIAL && items > sms ? sms : items;
    kern<<<unsigned(ctas), prefill_threads(1), Sh::SMEM_BYTES, st>>>(p, mq, mk, mv, mq, mq, mk);
    return launched();
}

} // namespace b200p
