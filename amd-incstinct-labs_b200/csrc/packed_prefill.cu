// ---------------------------------------------------------------------------
// packed_prefill.cu -- attention of prompts of different lengths that lie one after the other in one tensor.
// ---------------------------------------------------------------------------
#include "packed_launch.cuh"

namespace b200p {
namespace {

template <typename T, int D>
int launch(const void* Q, const void* K, const void* V, const int* qo, const int* ko, void* O, const b200p_packed_args& a, cudaStream_t st) {
    PackedParams p{};
    p.Q = Q; p.K = K; p.V = V; p.O = O; p.q_offsets = qo; p.k_offsets = ko;
    p.seqQ = a.total_q; p.seqK = a.total_k; p.batch = a.batch; p.causal = a.causal != 0;
    p.nQH = a.nQHeads; p.nKVH = a.nKVHeads; p.group = a.nQHeads / a.nKVHeads; p.splits = 1;
    p.scale_log2 = 1.4426950408889634f * (a.scale > 0.f ? a.scale : 1.f / sqrtf(float(D)));
    p.q_token = a.q_token; p.q_head = a.q_head; p.k_token = a.k_token; p.k_head = a.k_head;
    p.v_token = a.v_token; p.v_head = a.v_head; p.o_token = a.o_token; p.o_head = a.o_head;
    return launch_packed<T, D, false>(p, a.dtype, st);
}

// Checks what the entry points share and fills in the dense strides.
int checked(const b200p_packed_args* args, b200p_packed_args* out) {
    if (!args) return B200P_E_NULL;
    b200p_packed_args a = *args;
    if (a.dtype != B200P_F16 && a.dtype != B200P_BF16) return B200P_E_DTYPE;
    if (a.D != 64 && a.D != 128) return B200P_E_DIM;
    if (a.nQHeads <= 0 || a.nKVHeads <= 0 || a.nQHeads % a.nKVHeads != 0) return B200P_E_DIM;
    if (a.batch < 0 || a.total_q < 0 || a.total_k < 0 || !(a.scale >= 0.f) || std::isinf(a.scale)) return B200P_E_LENGTH;
    if (a.nQHeads / a.nKVHeads > 128 || a.nQHeads > 65535 || a.batch > (1 << 24)) return B200P_E_RANGE;
    const long long D = a.D;
    auto fill = [&](long long& token, long long& head, long long heads) { if (token == 0 && head == 0) { token = heads * D; head = D; } };
    fill(a.q_token, a.q_head, a.nQHeads); fill(a.k_token, a.k_head, a.nKVHeads); fill(a.v_token, a.v_head, a.nKVHeads); fill(a.o_token, a.o_head, a.nQHeads);
    // the stride of a dimension of one element says nothing
    if (a.total_q == 1) a.q_token = a.o_token = a.nQHeads * D;
    if (a.total_k == 1) a.k_token = a.v_token = a.nKVHeads * D;
    if (a.nQHeads == 1) a.q_head = a.o_head = D;
    if (a.nKVHeads == 1) a.k_head = a.v_head = D;
    for (long long s : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head, a.o_token, a.o_head}) if (s <= 0 || s % 8 != 0) return B200P_E_ALIGN;
    *out = a;
    return B200P_OK;
}

} // namespace
} // namespace b200p

using namespace b200p;

extern "C" size_t b200p_attn_prefill_packed_workspace_bytes(const b200p_packed_args* args) {
    (void)args;
    return 0;
}

extern "C" int b200p_attn_prefill_packed(const void* Q, const void* K, const void* V, const int* q_offsets, const int* k_offsets, void* O,
                                         const b200p_packed_args* args, void* workspace, size_t workspace_bytes, b200p_stream_t stream) {
    b200p_packed_args a;
    if (int e = checked(args, &a)) return e;
    if (a.batch == 0 || a.total_q == 0) return B200P_OK;
    if (!Q || !O || !q_offsets || !k_offsets || (a.total_k > 0 && (!K || !V))) return B200P_E_NULL;
    if (!aligned(Q, 16) || !aligned(K, 16) || !aligned(V, 16) || !aligned(O, 16) || !aligned(q_offsets, 4) || !aligned(k_offsets, 4)) return B200P_E_ALIGN;
    if (sm_count() <= 0) return B200P_E_NO_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dtype == B200P_F16) return a.D == 128 ? launch<__half, 128>(Q, K, V, q_offsets, k_offsets, O, a, st) : launch<__half, 64>(Q, K, V, q_offsets, k_offsets, O, a, st);
    return a.D == 128 ? launch<__nv_bfloat16, 128>(Q, K, V, q_offsets, k_offsets, O, a, st) : launch<__nv_bfloat16, 64>(Q, K, V, q_offsets, k_offsets, O, a, st);
}
