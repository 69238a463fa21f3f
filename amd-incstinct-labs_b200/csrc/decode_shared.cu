// ---------------------------------------------------------------------------
// decode_shared.cu -- attention of one new token per sequence of a batch whose sequences share a prefix:
// the prefix's keys and values exist once, each sequence has a cache of its own behind them.
// ---------------------------------------------------------------------------
#include "common.cuh"
#include "attn_rows.cuh"
#include <cmath>

namespace b200p {
namespace {

constexpr int kRowWarps = 4;

// One warp per (sequence, query head).
template <typename T, int D>
__global__ void __launch_bounds__(kRowWarps * 32)
shared_rows_kernel(const b200p_shared_args a, const T* __restrict__ q, const T* __restrict__ Kp, const T* __restrict__ Vp, const T* __restrict__ K,
                   const T* __restrict__ V, const int* __restrict__ lengths, T* __restrict__ o, float scale_log2) {
    constexpr int E = D / 32;
    const long long id = (long long)blockIdx.x * kRowWarps + threadIdx.x / 32;
    const int lane = threadIdx.x % 32, head = int(id % a.nQHeads), b = int(id / a.nQHeads);
    if (b >= a.batch) return;
    const int kvh = head / (a.nQHeads / a.nKVHeads), own = a.max_own > 0 ? min(max(lengths[b], 0), a.max_own) : 0;
    float x[E];
    load_part<T, E>(q + b * a.q_batch + head * D + lane * E, x);
    RowState<D> st;
    attend_keys<T, D>(st, x, Kp + kvh * a.prefix_head, Vp + kvh * a.prefix_head, D, D, a.prefix_len, scale_log2);
    const long long at = b * a.own_batch + kvh * a.own_head;
    attend_keys<T, D>(st, x, K + at, V + at, D, D, own, scale_log2);
    T* y = o + b * a.o_batch + head * D + lane * E;
    for (int i = 0; i < E; ++i) y[i] = from_float<T>(a.prefix_len + own > 0 ? st.o[i] / st.l : 0.f);
}

template <typename T, int D>
int launch_rows(const void* q, const void* Kp, const void* Vp, const void* K, const void* V, const int* lengths, void* o, const b200p_shared_args& a,
                float scale_log2, cudaStream_t st) {
    const long long warps = (long long)a.batch * a.nQHeads, ctas = (warps + kRowWarps - 1) / kRowWarps;
    if (ctas > 0x7fffffffLL) return B200P_E_RANGE;
    auto as = [](const void* p) { return static_cast<const T*>(p); };
    shared_rows_kernel<T, D><<<unsigned(ctas), kRowWarps * 32, 0, st>>>(a, as(q), as(Kp), as(Vp), as(K), as(V), lengths, static_cast<T*>(o), scale_log2);
    return launched();
}

int checked(const b200p_shared_args* args, b200p_shared_args* out) {
    if (!args) return B200P_E_NULL;
    b200p_shared_args a = *args;
    if (a.dtype != B200P_F16 && a.dtype != B200P_BF16) return B200P_E_DTYPE;
    if (a.D != 64 && a.D != 128) return B200P_E_DIM;
    if (a.nQHeads <= 0 || a.nKVHeads <= 0 || a.nQHeads % a.nKVHeads != 0) return B200P_E_DIM;
    if (a.batch < 0 || a.prefix_len < 0 || a.max_own < 0 || !(a.scale >= 0.f) || std::isinf(a.scale)) return B200P_E_LENGTH;
    if (a.nQHeads / a.nKVHeads > 128 || a.nQHeads > 65535 || a.batch > 65535) return B200P_E_RANGE;
    const long long D = a.D;
    if (a.prefix_head == 0) a.prefix_head = a.prefix_len * D;
    if (a.own_head == 0) a.own_head = a.max_own * D;
    if (a.own_batch == 0) a.own_batch = a.nKVHeads * a.own_head;
    if (a.q_batch == 0) a.q_batch = a.nQHeads * D;
    if (a.o_batch == 0) a.o_batch = a.nQHeads * D;
    if (a.prefix_head < a.prefix_len * D || a.own_head < a.max_own * D || a.own_batch < 0 || a.q_batch < a.nQHeads * D || a.o_batch < a.nQHeads * D) return B200P_E_LENGTH;
    for (long long s : {a.prefix_head, a.own_head, a.own_batch, a.q_batch, a.o_batch}) if (s % 8 != 0) return B200P_E_ALIGN;
    *out = a;
    return B200P_OK;
}

} // namespace
} // namespace b200p

using namespace b200p;

extern "C" size_t b200p_attn_decode_shared_workspace_bytes(const b200p_shared_args* args) {
    (void)args;
    return 0;
}

extern "C" int b200p_attn_decode_shared(const void* q, const void* K_prefix, const void* V_prefix, const void* K, const void* V, const int* lengths, void* o,
                                        const b200p_shared_args* args, void* workspace, size_t workspace_bytes, b200p_stream_t stream) {
    b200p_shared_args a;
    if (int e = checked(args, &a)) return e;
    if (a.batch == 0) return B200P_OK;
    if (!q || !o || (a.prefix_len > 0 && (!K_prefix || !V_prefix)) || (a.max_own > 0 && (!K || !V || !lengths))) return B200P_E_NULL;
    for (const void* p : {q, K_prefix, V_prefix, K, V, static_cast<const void*>(o)}) if (!aligned(p, 16)) return B200P_E_ALIGN;
    if (!aligned(lengths, 4)) return B200P_E_ALIGN;
    if (sm_count() <= 0) return B200P_E_NO_DEVICE;
    const float scale_log2 = 1.4426950408889634f * (a.scale > 0.f ? a.scale : 1.f / sqrtf(float(a.D)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a.dtype == B200P_F16)
        return a.D == 128 ? launch_rows<__half, 128>(q, K_prefix, V_prefix, K, V, lengths, o, a, scale_log2, st) : launch_rows<__half, 64>(q, K_prefix, V_prefix, K, V, lengths, o, a, scale_log2, st);
    return a.D == 128 ? launch_rows<__nv_bfloat16, 128>(q, K_prefix, V_prefix, K, V, lengths, o, a, scale_log2, st)
                      : launch_rows<__nv_bfloat16, 64>(q, K_prefix, V_prefix, K, V, lengths, o, a, scale_log2, st);
}
