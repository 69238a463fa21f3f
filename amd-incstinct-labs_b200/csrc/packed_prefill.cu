// ---------------------------------------------------------------------------
// packed_prefill.cu -- attention of prompts of different lengths that lie one after the other in one tensor.
// ---------------------------------------------------------------------------
#include "common.cuh"
#include "attn_rows.cuh"
#include <cmath>

namespace b200p {
namespace {

constexpr int kRowWarps = 4;

// The sequence that row `at` belongs to: the last one whose first row is at or before it (empty sequences share their first row
// with the next one).
__device__ __forceinline__ int sequence_of(const int* offsets, int batch, int at) {
    int lo = 0, hi = batch;                       // offsets[lo] <= at < offsets[hi], or at lies outside all sequences
    while (hi - lo > 1) { const int mid = (lo + hi) / 2; if (offsets[mid] <= at) lo = mid; else hi = mid; }
    return lo;
}

// One warp per row of Q.
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32)
packed_rows_kernel(const b200p_packed_args a, const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                   const int* __restrict__ q_offsets, const int* __restrict__ k_offsets, T* __restrict__ O, float scale_log2) {
    constexpr int E = D / 32;
    const long long id = (long long)blockIdx.x * kRowWarps + threadIdx.x / 32;
    const int lane = threadIdx.x % 32, head = int(id % a.nQHeads), row = int(id / a.nQHeads);
    if (row >= a.total_q || row < q_offsets[0] || row >= q_offsets[a.batch]) return;
    const int b = sequence_of(q_offsets, a.batch, row);
    const int q0 = q_offsets[b], n = q_offsets[b + 1] - q0;
    const int k0 = min(max(k_offsets[b], 0), a.total_k), keys = min(max(k_offsets[b + 1], k0), a.total_k) - k0;
    const int seen = a.causal ? min(keys, keys - n + (row - q0) + 1) : keys;
    const int kvh = head / (a.nQHeads / a.nKVHeads);
    float q[E];
    load_part<T, E>(Q + row * a.q_token + head * a.q_head + lane * E, q);
    RowState<D> st;
    attend_keys<T, D>(st, q, K + k0 * a.k_token + kvh * a.k_head, V + k0 * a.v_token + kvh * a.v_head, a.k_token, a.v_token, seen, scale_log2);
    T* o = O + row * a.o_token + head * a.o_head + lane * E;
    for (int i = 0; i < E; ++i) o[i] = from_float<T>(seen > 0 ? st.o[i] / st.l : 0.f);
}

template <typename T, int D>
int launch_rows(const void* Q, const void* K, const void* V, const int* qo, const int* ko, void* O, const b200p_packed_args& a, float scale_log2, cudaStream_t st) {
    const long long warps = (long long)a.total_q * a.nQHeads, ctas = (warps + kRowWarps - 1) / kRowWarps;
    if (ctas > 0x7fffffffLL) return B200P_E_RANGE;
    packed_rows_kernel<T, D><<<unsigned(ctas), kRowWarps * 32, 0, st>>>(a, static_cast<const T*>(Q), static_cast<const T*>(K), static_cast<const T*>(V), qo, ko,
                                                                      static_cast<T*>(O), scale_log2);
    return launched();
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
    const float scale_log2 = 1.4426950408889634f * (a.scale > 0.f ? a.scale : 1.f / sqrtf(float(a.D)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dtype == B200P_F16)
        return a.D == 128 ? launch_rows<__half, 128>(Q, K, V, q_offsets, k_offsets, O, a, scale_log2, st) : launch_rows<__half, 64>(Q, K, V, q_offsets, k_offsets, O, a, scale_log2, st);
    return a.D == 128 ? launch_rows<__nv_bfloat16, 128>(Q, K, V, q_offsets, k_offsets, O, a, scale_log2, st)
                      : launch_rows<__nv_bfloat16, 64>(Q, K, V, q_offsets, k_offsets, O, a, scale_log2, st);
}
