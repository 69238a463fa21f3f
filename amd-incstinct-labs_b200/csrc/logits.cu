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

constexpr int kSegment = 8192;                   // tokens a CTA handles, a word of shared memory for each
constexpr int kThreads = 256;
constexpr int kMostBias = 1024;
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

__device__ __forceinline__ float adjusted(float x, unsigned word, int token, const RowRules& r) {
    if (word & (kInPrompt | kCount)) x = x > 0.f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    const unsigned count = word & kCount;
    if (count) x = __fsub_rn(__fsub_rn(x, __fmul_rn(r.frequency, float(count))), r.presence);
    if (word & kBiased) {
        float b = 0.f;
        for (int i = 0; i < r.bias_n; ++i) if (r.bias_ids[i] == token) b = __fadd_rn(b, r.bias_values[i]);
        x = __fadd_rn(x, b);
    }
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
logits_kernel(const LogitsParams p, const T* __restrict__ in, T* __restrict__ out) {
    extern __shared__ unsigned words[];          // [kSegment]
    const b200p_logits_args& a = p.a;
    const int row = blockIdx.y, i0 = blockIdx.x * kSegment, n = min(kSegment, a.vocab - i0);
    for (int i = threadIdx.x; i < n; i += kThreads) words[i] = 0;
    __syncthreads();
    auto length = [&](const int* lengths, int stride, int most) { return lengths ? min(max(lengths[size_t(row) * stride], 0), most) : most; };
    if (a.prompt) {
        const int m = length(a.prompt_lengths, p.prompt_ls, a.prompt_max);
        for (int i = threadIdx.x; i < m; i += kThreads) {
            const unsigned t = unsigned(a.prompt[size_t(row) * a.prompt_max + i]) - unsigned(i0);
            if (t < unsigned(n)) atomicOr(&words[t], kInPrompt);
        }
    }
    if (a.tokens) {
        const int m = length(a.token_lengths, p.token_ls, a.tokens_max);
        for (int i = threadIdx.x; i < m; i += kThreads) {
            const unsigned t = unsigned(a.tokens[size_t(row) * a.tokens_max + i]) - unsigned(i0);
            if (t < unsigned(n)) atomicAdd(&words[t], 1u);
        }
    }
    RowRules r{a.repetition ? a.repetition[row] : 1.f, a.presence ? a.presence[row] : 0.f, a.frequency ? a.frequency[row] : 0.f,
               a.bias_ids + size_t(row) * a.bias_n, a.bias_values + size_t(row) * a.bias_n, a.bias_n};
    for (int i = threadIdx.x; i < a.bias_n; i += kThreads) {
        const unsigned t = unsigned(r.bias_ids[i]) - unsigned(i0);
        if (t < unsigned(n)) atomicOr(&words[t], kBiased);
    }
    __syncthreads();
    const int which = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
    const unsigned* mask = which >= 0 && which < a.n_masks ? a.mask + size_t(which) * ((a.vocab + 31) / 32) : nullptr;
    const T* x = in + size_t(row) * a.in_stride;
    T* y = out + size_t(row) * a.out_stride;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int token = i0 + i;
        float v = adjusted(to_float(x[token]), words[i], token, r);
        if (mask && !(mask[token >> 5] >> (token & 31) & 1u)) v = -INFINITY;
        y[token] = from_float<T>(v);
    }
}

template <typename T>
int launch(const void* in, void* out, const LogitsParams& p, cudaStream_t st) {
    const dim3 grid(unsigned((p.a.vocab + kSegment - 1) / kSegment), unsigned(p.a.rows));
    logits_kernel<T><<<grid, kThreads, kSegment * sizeof(unsigned), st>>>(p, static_cast<const T*>(in), static_cast<T*>(out));
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
