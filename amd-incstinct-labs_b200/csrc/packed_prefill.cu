// ---------------------------------------------------------------------------
// packed_prefill.cu -- attention of prompts of different lengths that lie one after the other in one tensor: row i of a
// sequence with n queries and m keys is softmax(scale q_i K^T) V over the keys j <= m - n + i (causal) or all m.
//
// The tcgen05 prefill kernel (prefill_tc.cuh) in its packed form (packed.cuh): one pass over the keys with the running maximum
// and sum, S and O in tensor memory.  Bound by the softmax warps' own instruction stream, as the dense form is: a step of 128 keys
// takes two query tiles 1.7 us whether heads are 64 or 128 wide, and an item 3 us more for its first S and its way out.  Measured, calls replayed
// from a graph: 8 documents of 2000 to 8192 tokens, 32 / 8 heads of 128, bf16, causal, 2.35 ms = 1073 TFLOP/s (0.65 of the GEMM's burst);
// 16 prompts of 100 to 1500 tokens 100 us = 748; 27 texts of 0 to 900, 32 / 4 heads of 64, fp16, not causal, 42 to 46 us = 370; 6 portions of
// 120 to 512 tokens on up to 6500 cached keys 127 us = 904; two questions of 19 and 40 tokens 7.2 us.
// ---------------------------------------------------------------------------
#include "packed_launch.cuh"

namespace b200p {
namespace {

// In how many splits the keys are taken: for few query tiles with many keys (a few new tokens on a long cache), and for a few sequences
// of which some may be much longer than the others.  The lengths are on the device, so the times, in microseconds, go by the means: an
// item takes 3 and 1.35 per 128 keys (2.05 with two query tiles); the last one to end may be of a sequence 1.8 times as long and begins
// when the others are under way; the merge takes 3, and the parts' way through the workspace.  A split has two
// key tiles, by the mean of the sequences' keys, but for what the last one is left with (a mean of 300 keys may take two); a shorter sequence leaves
// splits without keys.
// (One and the number chosen, 8 / 2 heads of 128: 39 tokens each of 11 sequences on 3950 keys 81 and 30; 2 texts of 1000 and 5000 tokens, one head, 72 and 28;
// 32 / 8 heads: 4 times 16 tokens on 1500 keys 32.6 and 18; 300 tokens, 300 keys, 10.3 and, with 2, 11.4: none.  Of 280 drawn calls of 200 keys and
// more the mean is 4 % above the best number of splits tried; the worst, 1.65 times, where one sequence has most of the tokens.)
struct PackedPlan { int splits; size_t off_ml, ws_bytes; };
PackedPlan plan_packed(const b200p_packed_args& a) {
    PackedPlan pl{1, 0, 0};
    if (a.batch == 0 || a.total_q == 0) return pl;
    const int sms = sm_count() > 0 ? sm_count() : 148, group = a.nQHeads / a.nKVHeads;
    const int tokens = kBM / group;
    const long long about = a.total_q / tokens + (a.batch + 1) / 2;            // of a key head: every second sequence fills a tile more than its share
    const long long tiles = (about > a.batch ? about : a.batch) * a.nKVHeads, most_tiles = packed_tiles(a.total_q, a.batch, tokens, a.nKVHeads);
    const int fixed = tuning(KNOB_PACKED_SPLITS, 0);
    const double keys = double(a.total_k) / a.batch, new_keys = double(a.total_q) / a.batch;
    if (fixed > 0) pl.splits = fixed < kMostParts ? fixed : kMostParts;
    else if (keys > 2 * kBN && tiles <= 2 * sms) {
        const double mean = (keys - (a.causal ? new_keys / 2 : 0)) / kBN, longest = (a.batch > 1 && 1.8 * keys < a.total_k ? 1.8 * keys : a.total_k) / kBN;
        double best = 0;
        for (int s = 1; s <= kMostParts && s <= keys / (2 * kBN) + 1; ++s) {
            const bool pairs = most_tiles * s > sms && new_keys >= 1.5 * tokens;
            const double step = pairs ? 2.05 : 1.35, items = double(tiles) * s / (pairs ? 2 : 1);
            const double last = 4.5 + step * std::ceil(longest / s), all = items * (3 + step * (mean > 0.5 * s ? mean / s : 0.5)) / sms + 0.75 * last;
            double t = items > sms && all > last ? all : last;
            if (s > 1) t += 3 + double(s) * a.total_q * a.nQHeads * a.D * 8 / 5e6;
            if (best == 0 || t < best) { best = t; pl.splits = s; }
        }
    }
    if (pl.splits > 1) {
        const size_t all = size_t(pl.splits) * a.total_q * a.nQHeads;
        pl.off_ml = (all * a.D * 4 + 255) / 256 * 256;
        pl.ws_bytes = pl.off_ml + (all * 8 + 255) / 256 * 256;
    }
    return pl;
}

template <typename T, int D>
int launch(const void* Q, const void* K, const void* V, const int* qo, const int* ko, void* O, const b200p_packed_args& a, const PackedPlan& pl, void* workspace, cudaStream_t st) {
    PackedParams p{};
    p.Q = Q; p.K = K; p.V = V; p.O = O; p.q_offsets = qo; p.k_offsets = ko;
    p.seqQ = a.total_q; p.seqK = a.total_k; p.batch = a.batch; p.causal = a.causal != 0;
    p.nQH = a.nQHeads; p.nKVH = a.nKVHeads; p.group = a.nQHeads / a.nKVHeads; p.splits = pl.splits;
    p.scale_log2 = 1.4426950408889634f * (a.scale > 0.f ? a.scale : 1.f / sqrtf(float(D)));
    p.q_token = a.q_token; p.q_head = a.q_head; p.k_token = a.k_token; p.k_head = a.k_head;
    p.v_token = a.v_token; p.v_head = a.v_head; p.o_token = a.o_token; p.o_head = a.o_head;
    if (pl.splits == 1) return launch_packed<T, D, false, true>(p, a.dtype, st);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + pl.off_ml);
    if (int e = launch_packed<T, D, true, true>(p, a.dtype, st)) return e;
    return launch_merge<T, D>(p.part_o, p.part_ml, pl.splits, a.total_q, a.nQHeads, O, a.o_token, a.o_head, qo, qo + a.batch, st);
}

// Checks what the entry points share and fills in the dense strides.
int checked(const b200p_packed_args* args, b200p_packed_args* out) {
    if (!args) return B200P_E_NULL;
    b200p_packed_args a = *args;
    if (a.dtype != B200P_F16 && a.dtype != B200P_BF16) return B200P_E_DTYPE;
    if (a.D != 64 && a.D != 128) return B200P_E_DIM;
    if (a.nQHeads <= 0 || a.nKVHeads <= 0 || a.nQHeads % a.nKVHeads != 0) return B200P_E_DIM;
    if (a.batch < 0 || a.total_q < 0 || a.total_k < 0 || !(a.scale >= 0.f) || std::isinf(a.scale)) return B200P_E_LENGTH;
    if (a.total_q > kMostRows || a.total_k > kMostRows) return B200P_E_RANGE;
    if (a.nQHeads / a.nKVHeads > 128 || a.nQHeads > 65535 || a.batch > (1 << 24) || (long long)a.total_q * a.nQHeads > 0x7fffffffLL) return B200P_E_RANGE;
    const long long D = a.D;
    auto fill = [&](long long& token, long long& head, long long heads) { if (token == 0 && head == 0) { token = heads * D; head = D; } };
    fill(a.q_token, a.q_head, a.nQHeads); fill(a.k_token, a.k_head, a.nKVHeads); fill(a.v_token, a.v_head, a.nKVHeads); fill(a.o_token, a.o_head, a.nQHeads);
    // the stride of a dimension of one element, or none, says nothing
    if (a.total_q <= 1) a.q_token = a.o_token = a.nQHeads * D;
    if (a.total_k <= 1) a.k_token = a.v_token = a.nKVHeads * D;
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
    b200p_packed_args a;
    return checked(args, &a) == B200P_OK ? plan_packed(a).ws_bytes : 0;
}

extern "C" int b200p_attn_prefill_packed(const void* Q, const void* K, const void* V, const int* q_offsets, const int* k_offsets, void* O,
                                         const b200p_packed_args* args, void* workspace, size_t workspace_bytes, b200p_stream_t stream) {
    b200p_packed_args a;
    if (int e = checked(args, &a)) return e;
    if (a.batch == 0 || a.total_q == 0) return B200P_OK;
    if (!Q || !O || !q_offsets || !k_offsets || (a.total_k > 0 && (!K || !V))) return B200P_E_NULL;
    if (!aligned(Q, 16) || !aligned(K, 16) || !aligned(V, 16) || !aligned(O, 16) || !aligned(q_offsets, 4) || !aligned(k_offsets, 4)) return B200P_E_ALIGN;
    if (sm_count() <= 0) return B200P_E_NO_DEVICE;
    const PackedPlan pl = plan_packed(a);
    if (pl.ws_bytes > 0 && (!workspace || workspace_bytes < pl.ws_bytes)) return B200P_E_WORKSPACE;
    if (!aligned(workspace, 256)) return B200P_E_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto tag) -> int {
        using T = decltype(tag);
        return a.D == 128 ? launch<T, 128>(Q, K, V, q_offsets, k_offsets, O, a, pl, workspace, st) : launch<T, 64>(Q, K, V, q_offsets, k_offsets, O, a, pl, workspace, st);
    };
    return a.dtype == B200P_F16 ? run(__half{}) : run(__nv_bfloat16{});
}
