// ---------------------------------------------------------------------------
// decode_shared.cu -- attention of one new token per sequence of a batch whose sequences share a prefix:
// the prefix's keys and values exist once, each sequence has a cache of its own behind them.
//
// Softmax over both parts is the merge of what each part gives (m: maximum, l: sum, O: weighted sum of values):
//   m = max m_i;  l = sum l_i 2^(m_i - m);  O = sum O_i 2^(m_i - m) / l.
// Two launches:
//  1. the prefix, for the whole batch: the query rows of a key head are ONE matrix of batch * group rows, so this is the tcgen05
//     prefill kernel (packed.cuh) over one "sequence" of `batch` tokens without a mask, its keys split so that all SMs have work;
//     (m, l, O) of every split go to the workspace in fp32.  Each tile of the prefix is read once per 256 rows.
//  2. the sequences' own keys, and the merge: HBM-bound, every byte of the caches is read once (own_kernel below).  It is a
//     programmatic dependent of the first launch and waits for it only ahead of the merge.
// A prefix that is small for its batch is cheaper read per sequence (from L2) by the second kernel alone.
// ---------------------------------------------------------------------------
#include "packed_launch.cuh"

namespace b200p {
namespace {

constexpr int kOwnWarps = 4;
constexpr int kOwnThreads = kOwnWarps * 32;
constexpr int kKeyBlock = 16;                    // keys of a warp's step
constexpr int kMostOwnCluster = 8;

struct OwnParams {
    const void *q, *Kp, *Vp, *K, *V;
    void* o;
    const int* lengths;
    int batch, nKVH, group, max_own, row_groups;
    int prefix_here, prefix_len;                 // keys of the prefix that this kernel reads itself; all of the prefix
    long long prefix_head, own_head, own_batch, q_batch, o_batch;
    float scale_log2;
    int splits;                                  // of the prefix, in the workspace
    const float *part_o, *part_ml;               // [splits][batch][nQH][D], [..][2]
};

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float load_cluster_f32(uint32_t smem, uint32_t cta) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float weight_of(float m, float most) { return exp2f(m - (most == -INFINITY ? 0.f : most)); }

// One cluster of `gridDim.x` CTAs per (sequence, key head, 8 * NT query rows); a warp takes every (warps of the cluster)-th block of
// 16 keys.  A step is S^T = K Q^T and O^T += V^T P^T with mma.sync m16n8k16 (keys, then head columns, in the 16 rows; the query
// heads of a group in the 8 columns, so that 8 heads fill an instruction).  Operands come straight from global memory, 16 bytes per
// lane and load: the contraction runs over the head columns in the order in which the lanes hold them, for K and Q alike; V's rows
// are paired up by byte permutes.  No shared memory or barrier stands between the loads and the products, a warp has 8 KB (heads of
// 128) in flight, 16 warps fit an SM.  Rows past the length are not read: their registers are zero.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kOwnThreads, NT == 1 ? 4 : D == 64 ? 3 : 2)
own_kernel(const OwnParams p) {
    constexpr int KC = D / 32, VC = D / 64, R = 8 * NT;
    __shared__ __align__(16) float s_o[kOwnWarps][R][D + 4];
    __shared__ float s_ml[kOwnWarps][R][2];
    __shared__ __align__(16) float s_sum[R][D];           // the CTA's result, for the cluster
    __shared__ float s_sum_ml[R][2];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
    const int ctas = gridDim.x, rank = blockIdx.x, kvh = blockIdx.y / p.row_groups, r0 = (blockIdx.y % p.row_groups) * R, b = blockIdx.z;
    const int own = p.max_own > 0 ? min(max(p.lengths[b], 0), p.max_own) : 0;
    const int rows = min(R, p.group - r0), nQH = p.nKVH * p.group, head0 = kvh * p.group + r0;

    // Q: column n of the B operand is query row r0 + n; lane (g, t4) has row g's columns 32 c + 8 t4 ..
    uint4 qf[NT][KC];
    #pragma unroll
    for (int n = 0; n < NT; ++n) {
        const T* row = static_cast<const T*>(p.q) + b * p.q_batch + (long long)(head0 + n * 8 + g) * D + t4 * 8;
        #pragma unroll
        for (int c = 0; c < KC; ++c) qf[n][c] = n * 8 + g < rows ? *reinterpret_cast<const uint4*>(row + 32 * c) : make_uint4(0, 0, 0, 0);
    }
    float o[NT][D / 16][4] = {};                          // tile (c, i): rows d = 64 c + 8 g + 2 i and + 1, columns 2 t4 and + 1
    float m[NT][2], l[NT][2];
    #pragma unroll
    for (int n = 0; n < NT; ++n) { m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.f; }

    const int prefix_blocks = (p.prefix_here + kKeyBlock - 1) / kKeyBlock, blocks = prefix_blocks + (own + kKeyBlock - 1) / kKeyBlock;
    const long long own_at = b * p.own_batch + kvh * p.own_head, prefix_at = kvh * p.prefix_head;
    for (int j = rank * kOwnWarps + warp; j < blocks; j += ctas * kOwnWarps) {
        const bool shared = j < prefix_blocks;
        const int key0 = (shared ? j : j - prefix_blocks) * kKeyBlock, there = (shared ? p.prefix_here : own) - key0;      // keys of the block
        const long long at = (shared ? prefix_at : own_at) + (long long)key0 * D;
        const T* K = static_cast<const T*>(shared ? p.Kp : p.K) + at;
        const T* V = static_cast<const T*>(shared ? p.Vp : p.V) + at;
        uint4 kf[2][KC], vf[4][VC];
        #pragma unroll
        for (int h = 0; h < 2; ++h)
            #pragma unroll
            for (int c = 0; c < KC; ++c) kf[h][c] = g + 8 * h < there ? load16(K + (g + 8 * h) * D + 32 * c + 8 * t4) : make_uint4(0, 0, 0, 0);
        #pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int key = 2 * t4 + (h & 1) + 8 * (h >> 1);
            #pragma unroll
            for (int c = 0; c < VC; ++c) vf[h][c] = key < there ? load16(V + key * D + 64 * c + 8 * g) : make_uint4(0, 0, 0, 0);
        }
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};            // keys g and g + 8, rows 2 t4 and + 1
            #pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint32_t a0[4] = {kf[0][c].x, kf[1][c].x, kf[0][c].y, kf[1][c].y}, a1[4] = {kf[0][c].z, kf[1][c].z, kf[0][c].w, kf[1][c].w};
                mma_16816<T>(s, a0, qf[n][c].x, qf[n][c].y);
                mma_16816<T>(s, a1, qf[n][c].z, qf[n][c].w);
            }
            if (g >= there) s[0] = s[1] = -INFINITY;
            if (g + 8 >= there) s[2] = s[3] = -INFINITY;
            float alpha[2];
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(s[e], s[2 + e]);
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                const float next = fmaxf(m[n][e], x * p.scale_log2), ref = next == -INFINITY ? 0.f : next;
                alpha[e] = fast_exp2(m[n][e] - ref);
                m[n][e] = next;
                s[e] = fast_exp2(fmaf(s[e], p.scale_log2, -ref));
                s[2 + e] = fast_exp2(fmaf(s[2 + e], p.scale_log2, -ref));
                l[n][e] = l[n][e] * alpha[e] + (s[e] + s[2 + e]);
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) { o[n][i][0] *= alpha[0]; o[n][i][1] *= alpha[1]; o[n][i][2] *= alpha[0]; o[n][i][3] *= alpha[1]; }
            }
            const uint32_t b0 = transposed_8x8(pack2<T>(s[0], s[1])), b1 = transposed_8x8(pack2<T>(s[2], s[3]));
            #pragma unroll
            for (int c = 0; c < VC; ++c) {
                const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0][c]); const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1][c]);
                const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2][c]); const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3][c]);
                #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t a[4] = {__byte_perm(v0[i], v1[i], 0x5410), __byte_perm(v0[i], v1[i], 0x7632), __byte_perm(v2[i], v3[i], 0x5410), __byte_perm(v2[i], v3[i], 0x7632)};
                    mma_16816<T>(o[n][c * 4 + i], a, b0, b1);
                }
            }
        }
    }
    // the warp's result
    #pragma unroll
    for (int n = 0; n < NT; ++n)
        #pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[n][e];
            #pragma unroll
            for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            const int row = n * 8 + 2 * t4 + e;
            if (g == 0) { s_ml[warp][row][0] = m[n][e]; s_ml[warp][row][1] = x; }
            #pragma unroll
            for (int c = 0; c < VC; ++c)
                #pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4*>(&s_o[warp][row][64 * c + 8 * g + 4 * h]) =
                        make_float4(o[n][c * 4 + 2 * h][e], o[n][c * 4 + 2 * h][2 + e], o[n][c * 4 + 2 * h + 1][e], o[n][c * 4 + 2 * h + 1][2 + e]);
        }
    __syncthreads();
    // the CTA's, where a cluster follows
    if (ctas > 1) {
        for (int i = threadIdx.x; i < rows * D; i += kOwnThreads) {
            const int row = i / D, d = i % D;
            float most = -INFINITY, sum = 0.f, x = 0.f;
            for (int w = 0; w < kOwnWarps; ++w) most = fmaxf(most, s_ml[w][row][0]);
            for (int w = 0; w < kOwnWarps; ++w) { const float f = weight_of(s_ml[w][row][0], most); sum += f * s_ml[w][row][1]; x += f * s_o[w][row][d]; }
            s_sum[row][d] = x;
            if (d == 0) { s_sum_ml[row][0] = most; s_sum_ml[row][1] = sum; }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    griddep_wait();                                       // the prefix's splits are there
    const int share = (rows * D + ctas - 1) / ctas, last = min(rows * D, (rank + 1) * share);
    for (int i = rank * share + threadIdx.x; i < last; i += kOwnThreads) {
        const int row = i / D, d = i % D;
        const size_t part = size_t(b) * nQH + head0 + row, next = size_t(p.batch) * nQH;
        float most = -INFINITY;
        float om[kMostOwnCluster], ol[kMostOwnCluster], ox[kMostOwnCluster];
        const int parts = ctas > 1 ? ctas : kOwnWarps;
        #pragma unroll
        for (int w = 0; w < kMostOwnCluster; ++w) {
            if (w >= parts) break;
            if (ctas > 1) {
                om[w] = load_cluster_f32(dme::smem_addr(&s_sum_ml[row][0]), w); ol[w] = load_cluster_f32(dme::smem_addr(&s_sum_ml[row][1]), w);
                ox[w] = load_cluster_f32(dme::smem_addr(&s_sum[row][d]), w);
            } else { om[w] = s_ml[w][row][0]; ol[w] = s_ml[w][row][1]; ox[w] = s_o[w][row][d]; }
            most = fmaxf(most, om[w]);
        }
        for (int s = 0; s < p.splits; ++s) most = fmaxf(most, p.part_ml[2 * (part + s * next)]);
        float sum = 0.f, x = 0.f;
        #pragma unroll
        for (int w = 0; w < kMostOwnCluster; ++w) {
            if (w >= parts) break;
            const float f = weight_of(om[w], most);
            sum += f * ol[w]; x += f * ox[w];
        }
        for (int s = 0; s < p.splits; ++s) {
            const float2 ml = *reinterpret_cast<const float2*>(&p.part_ml[2 * (part + s * next)]);
            if (ml.y == 0.f) continue;                    // no key: nothing was stored
            const float f = weight_of(ml.x, most);
            sum += f * ml.y; x += f * p.part_o[(part + s * next) * D + d];
        }
        static_cast<T*>(p.o)[b * p.o_batch + (long long)(head0 + row) * D + d] = from_float<T>(p.prefix_len + own > 0 ? x / sum : 0.f);
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");       // nobody leaves while a peer reads here
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// How a call is run.
struct SharedPlan {
    bool prefix_apart;           // the prefix in a launch of its own
    int splits, span;            // of that launch
    int cluster, rows;           // CTAs and query rows (8 or 16) of a unit of the second
    size_t off_ml, ws_bytes;
};

SharedPlan plan_shared(const b200p_shared_args& a) {
    SharedPlan pl{};
    const int sms = sm_count() > 0 ? sm_count() : 148, group = a.nQHeads / a.nKVHeads;
    pl.rows = group <= 8 ? 8 : 16;
    const long long units = (long long)a.batch * a.nKVHeads * ((group + pl.rows - 1) / pl.rows);
    pl.prefix_apart = a.prefix_len > 0 && (long long)a.batch * a.prefix_len > 4096;
    if (pl.prefix_apart) {
        const int tokens = kBM / group, tiles = (a.batch + tokens - 1) / tokens, steps = (a.prefix_len + kBN - 1) / kBN;
        double best = 0;
        for (int s = 1; s <= steps && s <= 32; ++s) {
            for (int span = 1; span <= 2; ++span) {
                if (span == 2 && tiles == 1) continue;
                const long long items = (long long)(tiles + span - 1) / span * a.nKVHeads * s;
                const double step = span == 1 ? 1.0 : 1.7;                    // in steps of one tile, 1.2 us
                const double t = double((items + sms - 1) / sms) * ((steps + s - 1) / s * step + 2.0) + double(s) * a.batch * a.nQHeads * a.D * 8 / 7.8e6;
                if (best == 0 || t < best) { best = t; pl.splits = s; pl.span = span; }
            }
        }
        const size_t rows = size_t(pl.splits) * a.batch * a.nQHeads;
        pl.off_ml = (rows * a.D * 4 + 255) / 256 * 256;
        pl.ws_bytes = pl.off_ml + (rows * 8 + 255) / 256 * 256;
    }
    const long long keys = a.max_own + (pl.prefix_apart ? 0 : a.prefix_len);
    pl.cluster = 1;
    while (pl.cluster < kMostOwnCluster && units * pl.cluster < 2 * sms && keys > 2 * kKeyBlock * kOwnWarps * pl.cluster) pl.cluster *= 2;
    return pl;
}

template <typename T, int D, int NT>
int launch_own(const OwnParams& p, int cluster, bool dependent, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(cluster), unsigned(p.nKVH * p.row_groups), unsigned(p.batch)); cfg.blockDim = dim3(kOwnThreads); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = unsigned(cluster); attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr; cfg.numAttrs = unsigned(n);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, own_kernel<T, D, NT>, p);
    if (e != cudaSuccess) { cudaGetLastError(); return int(e); }
    return launched();
}

template <typename T, int D>
int launch(const void* q, const void* Kp, const void* Vp, const void* K, const void* V, const int* lengths, void* o, const b200p_shared_args& a,
           const SharedPlan& pl, void* workspace, cudaStream_t st) {
    const float scale_log2 = 1.4426950408889634f * (a.scale > 0.f ? a.scale : 1.f / sqrtf(float(D)));
    const int group = a.nQHeads / a.nKVHeads;
    float* part_o = static_cast<float*>(workspace);
    float* part_ml = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + pl.off_ml);
    if (pl.prefix_apart) {
        PackedParams p{};
        p.Q = q; p.K = Kp; p.V = Vp;
        p.seqQ = a.batch; p.seqK = a.prefix_len; p.batch = 1;
        p.nQH = a.nQHeads; p.nKVH = a.nKVHeads; p.group = group; p.splits = pl.splits; p.span = pl.span;
        p.scale_log2 = scale_log2;
        p.q_token = a.q_batch; p.q_head = D; p.k_token = p.v_token = D; p.k_head = p.v_head = a.prefix_head;
        p.part_o = part_o; p.part_ml = part_ml;
        if (int e = launch_packed<T, D, true>(p, a.dtype, st)) return e;
    }
    OwnParams w{};
    w.q = q; w.Kp = Kp; w.Vp = Vp; w.K = K; w.V = V; w.o = o; w.lengths = lengths;
    w.batch = a.batch; w.nKVH = a.nKVHeads; w.group = group; w.max_own = a.max_own; w.row_groups = (group + pl.rows - 1) / pl.rows;
    w.prefix_here = pl.prefix_apart ? 0 : a.prefix_len; w.prefix_len = a.prefix_len;
    w.prefix_head = a.prefix_head; w.own_head = a.own_head; w.own_batch = a.own_batch; w.q_batch = a.q_batch; w.o_batch = a.o_batch;
    w.scale_log2 = scale_log2; w.splits = pl.prefix_apart ? pl.splits : 0; w.part_o = part_o; w.part_ml = part_ml;
    return pl.rows == 8 ? launch_own<T, D, 1>(w, pl.cluster, pl.prefix_apart, st) : launch_own<T, D, 2>(w, pl.cluster, pl.prefix_apart, st);
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
    b200p_shared_args a;
    return checked(args, &a) == B200P_OK && a.batch > 0 ? plan_shared(a).ws_bytes : 0;
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
    const SharedPlan pl = plan_shared(a);
    if (pl.ws_bytes > 0 && (!workspace || workspace_bytes < pl.ws_bytes)) return B200P_E_WORKSPACE;
    if (!aligned(workspace, 256)) return B200P_E_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto tag) -> int {
        using T = decltype(tag);
        return a.D == 128 ? launch<T, 128>(q, K_prefix, V_prefix, K, V, lengths, o, a, pl, workspace, st) : launch<T, 64>(q, K_prefix, V_prefix, K, V, lengths, o, a, pl, workspace, st);
    };
    return a.dtype == B200P_F16 ? run(__half{}) : run(__nv_bfloat16{});
}
