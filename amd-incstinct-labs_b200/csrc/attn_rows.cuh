// ---------------------------------------------------------------------------
// attn_rows.cuh -- one query row of attention by one warp, straight from the formula:
// m = max s_j, l = sum 2^(s_j - m), o = sum 2^(s_j - m) v_j over a run of keys, all in fp32.
// A key that is not in the run is not read, so nothing that lies there can reach the row.
// ---------------------------------------------------------------------------
#pragma once
#include "attn_common.cuh"
#include <cstdint>

namespace b200p {

// A row's state over the keys so far: maximum of the scores in log2 units, sum and (not yet divided) output; lane i holds
// columns i * E .. i * E + E - 1.
template <int D> struct RowState {
    static constexpr int E = D / 32;
    float m = -INFINITY, l = 0.f, o[E] = {};
};

// E = 2 or 4 consecutive 16-bit elements as fp32
template <typename T, int E> __device__ __forceinline__ void load_part(const T* p, float (&f)[E]) {
    uint32_t w[E / 2];
    if constexpr (E == 4) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
    const T* e = reinterpret_cast<const T*>(w);
    #pragma unroll
    for (int i = 0; i < E; ++i) f[i] = to_float(e[i]);
}

// Keys 0 .. n-1 of rows K + j * k_row, V + j * v_row (each D elements) into the state.  q: this lane's columns of the query.
template <typename T, int D>
__device__ __forceinline__ void attend_keys(RowState<D>& st, const float (&q)[D / 32], const T* K, const T* V, long long k_row, long long v_row, int n, float scale_log2) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x % 32;
    #pragma unroll 4
    for (int j = 0; j < n; ++j) {
        float k[E], v[E];
        load_part<T, E>(K + j * k_row + lane * E, k);
        load_part<T, E>(V + j * v_row + lane * E, v);
        float s = 0.f;
        #pragma unroll
        for (int i = 0; i < E; ++i) s += q[i] * k[i];
        #pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= scale_log2;
        const float m = fmaxf(st.m, s);                     // a NaN score is no maximum, it shows in l and o
        const float ref = m == -INFINITY ? 0.f : m;         // every score so far is -inf: their weights are 0
        const float a = exp2f(st.m - ref), p = exp2f(s - ref);
        st.m = m;
        st.l = st.l * a + p;
        #pragma unroll
        for (int i = 0; i < E; ++i) st.o[i] = st.o[i] * a + p * v[i];
    }
}

} // namespace b200p
