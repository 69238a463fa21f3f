// ---------------------------------------------------------------------------
// logits.cu -- the rules that a request puts on its logits before a token is picked:
//   x <- x > 0 ? x / repetition : x * repetition     for tokens of the prompt or generated so far
//   x <- x - frequency * count - presence * [count > 0]   count: how often the token was generated
//   x <- x + the token's biases, in their order
//   x <- -inf                                         for tokens whose bit in the mask is 0
// in fp32, each operation rounded once, the result rounded once to the logits' type.
// ---------------------------------------------------------------------------
#include "common.cuh"
#include "attn_common.cuh"
#include "logits.cuh"

namespace b200p {
namespace {

constexpr int kThreads = 256;
constexpr int kSegment = 32 * kThreads;          // tokens a CTA handles, a word of shared memory for each
// A token's word: how often it was generated, and two flags.
constexpr unsigned kInPrompt = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1;

struct LogitsParams {
    b200p_logits_args a;
    int prompt_ls, token_ls;
};

struct RowRules {
    float repetition, presence, frequency;
    const int* bias_ids; const float* bias_values; int bias_n;
};

// By selection rather than branches: a thread does its touched tokens one after the other, and a warp takes every branch that one of its
// lanes takes (48 rows of 50001, bf16: 7.7 us, so 7.4).
__device__ __forceinline__ float adjusted(float x, unsigned word, int token, const RowRules& r) {
    const float less = __fdiv_rn(x, r.repetition), more = __fmul_rn(x, r.repetition);
    x = word & (kInPrompt | kCount) ? (x > 0.f ? less : more) : x;
    const unsigned count = word & kCount;
    const float taken = __fsub_rn(__fsub_rn(x, __fmul_rn(r.frequency, float(count))), r.presence);
    x = count ? taken : x;
    if (word & kBiased) {
        float b = 0.f;
        for (int i = 0; i < r.bias_n; ++i) if (r.bias_ids[i] == token) b = __fadd_rn(b, r.bias_values[i]);
        x = __fadd_rn(x, b);
    }
    return x;
}

__device__ __forceinline__ uint4 load_logits(const void* p) {        // may be the place that is written: not the read-only path
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
template <typename T> __device__ __forceinline__ T pick(const uint4& v, int e) { return reinterpret_cast<const T*>(&v)[e]; }
template <typename T> __device__ __forceinline__ void put(uint4& v, int e, T x) { reinterpret_cast<T*>(&v)[e] = x; }

// One CTA per (segment of the vocabulary, row).  The logits are read and written once, 16 bytes at a time.  Their loads, the
// mask's and the histories' first ids are issued together and are under way while the segment's part of the histories is counted: every
// CTA of a row reads the row's whole histories (from L2, but for the first), keeps the ids of its segment and counts them in shared
// memory, so that no count leaves the SM and nothing has to be cleared or merged.  Integer atomics: the order does not show.
// Rows may start anywhere: places are counted from the last 16-byte boundary of `out` at or before the row; where a whole vector lies in
// the row it is stored as one, and loaded as one if `in` lies the same way.
// HBM-bound without histories: 256 rows of 128000 fp32 logits 40.8 us = 6.4 TB/s, with masks 42.  Histories (2048 + 512 ids a row on average, biases)
// make it 61: a CTA's two barriers and its trips for ids leave the memory idle, and 16 CTAs of a row look at the same ids.  Segments of 16384 and 32768
// tokens halve and quarter that and take 66 and 74 us: fewer CTAs an SM to fill each other's waits.  Each id
// looked at by one CTA of a cluster of 8, which counts it in its owner's shared memory, 73 (frequent tokens have one owner); ids by 16-byte loads 63.
// One row of 32000: 3.1 us, launch included.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
logits_kernel(const LogitsParams p, const T* in, T* out) {
    constexpr int E = 16 / sizeof(T), VECS = kSegment / E / kThreads;
    static_assert(VECS * E == 32, "a thread's places in one word");
    extern __shared__ __align__(16) unsigned words[];               // [kSegment]
    const b200p_logits_args& a = p.a;
    const int row = blockIdx.y, V = a.vocab;
    const T* const x = in + size_t(row) * a.in_stride;
    T* const y = out + size_t(row) * a.out_stride;
    const int before = int(reinterpret_cast<uintptr_t>(y) % 16 / sizeof(T));
    const bool alike = reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T) == unsigned(before);
    const int i0 = int(blockIdx.x) * kSegment - before;             // the segment's first token (negative: what lies before the row)
    if (i0 >= V) return;                                            // the grid has room for a row that starts behind a boundary
    const bool whole = alike && i0 >= 0 && i0 + kSegment <= V;      // vectors only
    const int which = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    const unsigned* const mask = which >= 0 && which < a.n_masks ? a.mask + size_t(which) * ((V + 31) / 32) : nullptr;
    auto token_of = [&](int k) { return i0 + (k * kThreads + int(threadIdx.x)) * E; };     // the vector's first
    uint4 v[VECS];
    if (whole) {
        #pragma unroll
        for (int k = 0; k < VECS; ++k) v[k] = load_logits(x + token_of(k));
    } else {
        #pragma unroll
        for (int k = 0; k < VECS; ++k) {
            const int t = token_of(k);
            if (alike && t >= 0 && t + E <= V) v[k] = load_logits(x + t);
            else {
                #pragma unroll
                for (int e = 0; e < E; ++e) if (t + e >= 0 && t + e < V) put<T>(v[k], e, x[t + e]);
            }
        }
    }
    unsigned allowed = ~0u;                                         // of this thread's 32 places
    if (mask) {
        allowed = 0;
        if (whole && before == 0) {                                 // a vector's bits in one word
            #pragma unroll
            for (int k = 0; k < VECS; ++k) allowed |= (mask[token_of(k) >> 5] >> (token_of(k) & 31) & ((1u << E) - 1)) << (k * E);
        } else {
            #pragma unroll
            for (int k = 0; k < VECS; ++k) {
                const int t = token_of(k);
                if (t + E <= 0 || t >= V) continue;
                const int f = max(t, 0), l = min(t + E, V) - 1;
                const unsigned lo = mask[f >> 5], hi = (l >> 5) != (f >> 5) ? mask[l >> 5] : 0u;
                allowed |= (__funnelshift_r(lo, hi, f & 31) << (f - t) & ((1u << E) - 1)) << (k * E);
            }
        }
    }
    // The lists' first ids, ahead of their lengths: up to a row's end they are there, whether they count or not.
    const int* const prompt = a.prompt + size_t(row) * a.prompt_max; const int* const tokens = a.tokens + size_t(row) * a.tokens_max;
    const int* const biased = a.bias_ids + size_t(row) * a.bias_n;
    constexpr int P0 = 4, T0 = 2, B0 = 1;
    int id_p[P0], id_t[T0], id_b[B0];
    auto first_ids = [&](auto& id, const int* ids, int n) {
        #pragma unroll
        for (int u = 0; u < int(sizeof(id) / 4); ++u) { const int i = u * kThreads + int(threadIdx.x); id[u] = i < n ? ids[i] : -1; }
    };
    first_ids(id_p, prompt, a.prompt ? a.prompt_max : 0);
    first_ids(id_t, tokens, a.tokens ? a.tokens_max : 0);
    first_ids(id_b, biased, a.bias_n);
    auto length = [&](const int* ids, const int* lengths, int stride, int most) { return !ids ? 0 : lengths ? min(max(lengths[size_t(row) * stride], 0), most) : most; };
    const int n_prompt = length(a.prompt, a.prompt_lengths, p.prompt_ls, a.prompt_max), n_tokens = length(a.tokens, a.token_lengths, p.token_ls, a.tokens_max);
    const RowRules r{a.repetition ? a.repetition[row] : 1.f, a.presence ? a.presence[row] : 0.f, a.frequency ? a.frequency[row] : 0.f,
                     biased, a.bias_values + size_t(row) * a.bias_n, a.bias_n};
    unsigned touched = 0;                                           // of this thread's places
    if (n_prompt + n_tokens + a.bias_n > 0) {                       // the same in all threads
        #pragma unroll
        for (int i = 0; i < kSegment / 4 / kThreads; ++i) reinterpret_cast<uint4*>(words)[i * kThreads + threadIdx.x] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        const int low = max(i0, 0);                                 // the segment's ids: low ... low + range - 1
        const unsigned range = unsigned(min(i0 + kSegment, V) - low);
        auto each = [&](auto& first, const int* ids, int n, auto&& mark) {
            constexpr int F = int(sizeof(first) / 4), U = 4;        // U loads in flight
            #pragma unroll
            for (int u = 0; u < F; ++u) if (u * kThreads + int(threadIdx.x) < n && unsigned(first[u] - low) < range) mark(&words[first[u] - i0]);
            for (int i = F * kThreads + int(threadIdx.x); i < n; i += U * kThreads) {
                int id[U];
                #pragma unroll
                for (int u = 0; u < U; ++u) id[u] = i + u * kThreads < n ? ids[i + u * kThreads] : -1;
                #pragma unroll
                for (int u = 0; u < U; ++u) if (unsigned(id[u] - low) < range) mark(&words[id[u] - i0]);
            }
        };
        each(id_p, prompt, n_prompt, [](unsigned* w) { atomicOr(w, kInPrompt); });
        each(id_t, tokens, n_tokens, [](unsigned* w) { atomicAdd(w, 1u); });
        each(id_b, biased, a.bias_n, [](unsigned* w) { atomicOr(w, kBiased); });
        __syncthreads();
        #pragma unroll
        for (int q = 0; q < 8; ++q) {
            const uint4 w = *reinterpret_cast<const uint4*>(&words[(q * 4 / E * kThreads + int(threadIdx.x)) * E + q * 4 % E]);
            touched |= (w.x ? 1u : 0u) << (4 * q) | (w.y ? 2u : 0u) << (4 * q) | (w.z ? 4u : 0u) << (4 * q) | (w.w ? 8u : 0u) << (4 * q);
        }
        touched &= allowed;                                         // a masked one stays masked
    }
    // All logits out, but for the masked ones as they came in.  Those that the rules touch are done in a loop of its own: the rules
    // inlined at every place are more code than the instruction cache holds (256 rows of 128000: 141 us, so 93).
    const T none = from_float<T>(-INFINITY);
    #pragma unroll
    for (int k = 0; k < VECS; ++k) {
        if (mask) {
            #pragma unroll
            for (int e = 0; e < E; ++e) if (!(allowed >> (k * E + e) & 1u)) put<T>(v[k], e, none);
        }
        const int t = token_of(k);
        if (whole || (t >= 0 && t + E <= V)) *reinterpret_cast<uint4*>(y + t) = v[k];
        else {
            #pragma unroll
            for (int e = 0; e < E; ++e) if (t + e >= 0 && t + e < V) y[t + e] = pick<T>(v[k], e);
        }
    }
    for (; touched; touched &= touched - 1) {
        const int b = __ffs(touched) - 1, place = (b / E * kThreads + int(threadIdx.x)) * E + b % E, t = i0 + place;
        T z = pick<T>(v[0], 0);                                     // the value is still in a register: found by comparisons, not read again
        #pragma unroll
        for (int i = 1; i < 32; ++i) if (i == b) z = pick<T>(v[i / E], i % E);
        y[t] = from_float<T>(adjusted(to_float(z), words[place], t, r));
    }
}

template <typename T>
int launch(const void* in, void* out, const LogitsParams& p, cudaStream_t st) {
    const long long places = (long long)p.a.vocab + 16 / (long long)sizeof(T) - 1;
    constexpr int kBytes = kSegment * int(sizeof(unsigned));
    if (int e = allow_dynamic_smem(reinterpret_cast<const void*>(logits_kernel<T>), kBytes)) return e;
    logits_kernel<T><<<dim3(unsigned((places + kSegment - 1) / kSegment), unsigned(p.a.rows)), kThreads, kBytes, st>>>(p, static_cast<const T*>(in), static_cast<T*>(out));
    return launched();
}

} // namespace

int logits_adjust(const void* in, void* out, const b200p_logits_args* a, int prompt_length_stride, int token_length_stride, cudaStream_t st) {
    const LogitsParams p{*a, prompt_length_stride, token_length_stride};
    switch (a->dtype) {
        case B200P_F32: return launch<float>(in, out, p, st);
        case B200P_F16: return launch<__half>(in, out, p, st);
        case B200P_BF16: return launch<__nv_bfloat16>(in, out, p, st);
    }
    return B200P_E_DTYPE;
}

} // namespace b200p

using namespace b200p;

extern "C" int b200p_logits_adjust(const void* logits, void* out, const b200p_logits_args* args, b200p_stream_t stream) {
    if (!args) return B200P_E_NULL;
    b200p_logits_args a = *args;
    if (a.dtype != B200P_F32 && a.dtype != B200P_F16 && a.dtype != B200P_BF16) return B200P_E_DTYPE;
    if (a.rows < 0 || a.vocab <= 0 || a.prompt_max < 0 || a.tokens_max < 0 || a.bias_n < 0 || a.n_masks < 0) return B200P_E_LENGTH;
    if (a.rows == 0) return B200P_OK;
    if (a.rows > 65535 || a.vocab > (1 << 30) || a.tokens_max >= int(kCount) || a.bias_n > kMostBias) return B200P_E_RANGE;
    if (a.in_stride == 0) a.in_stride = a.vocab;
    if (a.out_stride == 0) a.out_stride = a.vocab;
    if (a.in_stride < a.vocab || a.out_stride < a.vocab || (logits == out && a.in_stride != a.out_stride)) return B200P_E_LENGTH;
    if (!logits || !out) return B200P_E_NULL;
    if ((a.prompt_max > 0 && !a.prompt) || (a.tokens_max > 0 && !a.tokens) || (a.bias_n > 0 && (!a.bias_ids || !a.bias_values)) || (a.n_masks > 0 && !a.mask))
        return B200P_E_NULL;
    if (a.mask && !a.mask_rows && a.n_masks < a.rows) return B200P_E_LENGTH;
    const size_t size = a.dtype == B200P_F32 ? 4 : 2;
    if (!aligned(logits, size) || !aligned(out, size)) return B200P_E_ALIGN;
    if (a.prompt_max == 0) a.prompt = nullptr;
    if (a.tokens_max == 0) a.tokens = nullptr;
    if (sm_count() <= 0) return B200P_E_NO_DEVICE;
    return logits_adjust(logits, out, &a, 1, 1, static_cast<cudaStream_t>(stream));
}
