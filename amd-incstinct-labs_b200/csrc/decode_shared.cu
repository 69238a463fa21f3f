// ---------------------------------------------------------------------------
// decode_shared.cu -- attention of one new token per sequence of a batch whose sequences share a prefix:
// the prefix's keys and values exist once, each sequence has a cache of its own behind them.
//
// Softmax over both parts is the merge of what each part gives (m: maximum, l: sum, O: weighted sum of values):
//   m = max m_i;  l = sum l_i 2^(m_i - m);  O = sum O_i 2^(m_i - m) / l.
// Two or three launches:
//  1. the prefix, for the whole batch: the query rows of a key head are ONE matrix of batch * group rows, so this is the tcgen05
//     prefill kernel (packed.cuh) over one "sequence" of `batch` tokens without a mask, its keys split so that all SMs have work;
//     (m, l, O) of every split go to the workspace in fp32.  Each tile of the prefix is read once per 256 rows.
//  2. the sequences' own keys (own_kernel): HBM-bound, every byte of the caches is read once.  A programmatic dependent that
//     waits for nothing: its CTAs run wherever the first launch leaves room.
//  3. the merge (merge_kernel, packed_launch.cuh); or the second launch waits for the first and merges itself (plan_shared).
// A prefix that is small for its batch is cheaper read per sequence (from L2), by own_kernel, which then is the only launch.
//
// Measured, calls replayed from a graph, 32 / 8 heads of 128 unless said otherwise: 4 sequences, 512 keys in front, up to 32 of their own 6.5 us (one
// launch); 32, 2000, up to 512, fp16, 16.6; 48 with 32 / 4 heads of 64, 5000, up to 1000, 18.7; 256, 32768, up to 256, 141 to 160 (980 TFLOP/s and
// more, the tiles at the prefill kernel's rate).  What bounds the middle ones is latency: dependent launches, of which the tiles' takes 4.5 us
// for its barriers, Q, first keys and way out and 1.35 a key tile, the own keys' 10 from start to end, the merge 2 to 3.
// (Not kept: the prefix by mma.sync warps that share their keys through L1, 4 warps of 16 rows each, never clearly faster than the tiles, 220 against
// 55 us for 34 sequences behind 25299 keys.)
// ---------------------------------------------------------------------------
#include "packed_launch.cuh"

namespace b200p {
namespace {

constexpr int kOwnWarps = 4;
constexpr int kOwnThreads = kOwnWarps * 32;
constexpr int kKeyBlock = 16;                    // keys of a warp's step
constexpr int kMostOwnCluster = 8;
constexpr int kMostJoined = 32;                  // splits that own_kernel merges itself: a lane each
constexpr int kMostSplits = kMostParts - kMostOwnCluster;        // of the prefix: one for each SM, for a single key head

struct OwnParams {
    const void *q, *Kp, *Vp, *K, *V;
    void* o;
    const int* lengths;
    int batch, nKVH, group, max_own, row_groups;
    int prefix_here;                             // keys of the prefix that this kernel reads itself
    long long prefix_head, own_head, own_batch, q_batch, o_batch;
    float scale_log2;
    int apart;                                   // 1: results go to the workspace, as parts `first_part` + the CTA's place in its unit
    int first_part;
    int joined;                                  // splits of the prefix that this launch waits for and merges itself
    float *part_o, *part_ml;                     // [part][batch][nQH][D], not divided; [..][2]: maximum in log2 units, sum
};

__device__ __forceinline__ uint32_t transposed_8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float load_cluster_f32(uint32_t smem, uint32_t cta) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(cta));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_cluster_f32x4(uint32_t smem, uint32_t cta) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem), "r"(cta));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

// Up to 8 * NT query rows against blocks of 16 keys by one warp.  A step is S^T = K Q^T and O^T += V^T P^T with mma.sync m16n8k16: keys,
// then head columns, in the 16 rows, the query rows in the 8 columns, so that 8 of them fill an instruction.  Operands come straight
// from global memory, 16 bytes per lane and load: the contraction runs over the head columns in the order in which the lanes hold
// them, for K and Q alike; V's rows are paired up by byte permutes.  No shared memory and no barrier stands between the loads and the
// products; a warp has 8 KB (heads of 128) in flight.  Rows past the run's end are not read: their registers are zero.
// Lane (g, t4) = (lane / 4, lane % 4).
template <typename T, int D, int NT> struct KeyWalk {
    static constexpr int KC = D / 32, VC = D / 64;
    uint4 qf[NT][KC];                                     // row n * 8 + g, columns 32 c + 8 t4 ..
    uint4 kf[2][KC], vf[4][VC];                           // keys g, g + 8, the same columns; keys 2 t4, + 1, + 8, + 9, columns 64 c + 8 g ..
    float o[NT][D / 16][4];                               // tile (c, i): columns d = 64 c + 8 g + 2 i and + 1 of rows n * 8 + 2 t4 and + 1
    float m[NT][2], l[NT][2];                             // of those rows; l: over this lane's keys
    int g, t4;

    __device__ __forceinline__ KeyWalk() : g(threadIdx.x % 32 / 4), t4(threadIdx.x % 4) {
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY; l[n][0] = l[n][1] = 0.f;
            #pragma unroll
            for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
        }
    }
    static __device__ __forceinline__ uint4 load16(const T* p) {
        uint4 v;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
        return v;
    }
    // row: this lane's row (n * 8 + g) or null
    __device__ __forceinline__ void load_q(int n, const T* row) {
        #pragma unroll
        for (int c = 0; c < KC; ++c) qf[n][c] = row ? *reinterpret_cast<const uint4*>(row + 32 * c + 8 * t4) : make_uint4(0, 0, 0, 0);
    }
    // the block's first row, and how many rows there are
    __device__ __forceinline__ void load_k(const T* K, int there) {
        #pragma unroll
        for (int h = 0; h < 2; ++h)
            #pragma unroll
            for (int c = 0; c < KC; ++c) kf[h][c] = g + 8 * h < there ? load16(K + (g + 8 * h) * D + 32 * c + 8 * t4) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load_v(const T* V, int there) {
        #pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int key = 2 * t4 + (h & 1) + 8 * (h >> 1);
            #pragma unroll
            for (int c = 0; c < VC; ++c) vf[h][c] = key < there ? load16(V + key * D + 64 * c + 8 * g) : make_uint4(0, 0, 0, 0);
        }
    }
    // values that were loaded ahead of knowing the end
    __device__ __forceinline__ void drop_v(int there) {
        #pragma unroll
        for (int h = 0; h < 4; ++h)
            #pragma unroll
            for (int c = 0; c < VC; ++c) if (2 * t4 + (h & 1) + 8 * (h >> 1) >= there) vf[h][c] = make_uint4(0, 0, 0, 0);
    }
    // The block that is loaded.  next_k(): called as soon as K's registers are free.
    template <typename F> __device__ __forceinline__ void step(int there, float scale_log2, F&& next_k) {
        float s[NT][4];                                   // keys g and g + 8, rows 2 t4 and + 1
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
            #pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint32_t a0[4] = {kf[0][c].x, kf[1][c].x, kf[0][c].y, kf[1][c].y}, a1[4] = {kf[0][c].z, kf[1][c].z, kf[0][c].w, kf[1][c].w};
                mma_16816<T>(s[n], a0, qf[n][c].x, qf[n][c].y);
                mma_16816<T>(s[n], a1, qf[n][c].z, qf[n][c].w);
            }
        }
        next_k();
        uint32_t pt[NT][2];
        #pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (g >= there) s[n][0] = s[n][1] = -INFINITY;
            if (g + 8 >= there) s[n][2] = s[n][3] = -INFINITY;
            float alpha[2];
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = fmaxf(s[n][e], s[n][2 + e]);
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                const float most = fmaxf(m[n][e], x * scale_log2), ref = most == -INFINITY ? 0.f : most;      // nothing but -inf so far: weights of 0
                alpha[e] = fast_exp2(m[n][e] - ref);
                m[n][e] = most;
                s[n][e] = fast_exp2(fmaf(s[n][e], scale_log2, -ref));
                s[n][2 + e] = fast_exp2(fmaf(s[n][2 + e], scale_log2, -ref));
                l[n][e] = l[n][e] * alpha[e] + (s[n][e] + s[n][2 + e]);
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
                #pragma unroll
                for (int i = 0; i < D / 16; ++i) { o[n][i][0] *= alpha[0]; o[n][i][1] *= alpha[1]; o[n][i][2] *= alpha[0]; o[n][i][3] *= alpha[1]; }
            }
            // in 16 bits, as V is: half a step of each weight (prefill_tc.cuh); l has added them in fp32
            pt[n][0] = transposed_8x8(pack2<T>(s[n][0], s[n][1])); pt[n][1] = transposed_8x8(pack2<T>(s[n][2], s[n][3]));
        }
        #pragma unroll
        for (int c = 0; c < VC; ++c) {
            const uint32_t* v0 = reinterpret_cast<const uint32_t*>(&vf[0][c]); const uint32_t* v1 = reinterpret_cast<const uint32_t*>(&vf[1][c]);
            const uint32_t* v2 = reinterpret_cast<const uint32_t*>(&vf[2][c]); const uint32_t* v3 = reinterpret_cast<const uint32_t*>(&vf[3][c]);
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {__byte_perm(v0[i], v1[i], 0x5410), __byte_perm(v0[i], v1[i], 0x7632), __byte_perm(v2[i], v3[i], 0x5410), __byte_perm(v2[i], v3[i], 0x7632)};
                #pragma unroll
                for (int n = 0; n < NT; ++n) mma_16816<T>(o[n][c * 4 + i], a, pt[n][0], pt[n][1]);
            }
        }
    }
    // Row n * 8 + 2 t4 + e: put(row, maximum, sum over all lanes) by the lanes with g = 0, then every lane's columns, four at a time.
    template <typename ML, typename O4> __device__ __forceinline__ void result(ML&& put_ml, O4&& put_o) {
        #pragma unroll
        for (int n = 0; n < NT; ++n)
            #pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[n][e];
                #pragma unroll
                for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
                const int row = n * 8 + 2 * t4 + e;
                if (g == 0) put_ml(row, m[n][e], x);
                #pragma unroll
                for (int c = 0; c < VC; ++c)
                    #pragma unroll
                    for (int h = 0; h < 2; ++h)
                        put_o(row, 64 * c + 8 * g + 4 * h, make_float4(o[n][c * 4 + 2 * h][e], o[n][c * 4 + 2 * h][2 + e], o[n][c * 4 + 2 * h + 1][e], o[n][c * 4 + 2 * h + 1][2 + e]));
            }
    }
};

// The sequences' own keys, and the prefix's where it has no launch of its own.  `gridDim.x` CTAs per unit, which is (sequence, key head, 8 * NT
// query rows); a warp takes every (warps of the unit)-th block of 16 keys.  With the prefix apart the CTAs leave parts for
// merge_kernel; else they are a cluster and merge through distributed shared memory.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kOwnThreads, NT == 1 ? 4 : D == 64 ? 3 : 2)
own_kernel(const OwnParams p) {
    constexpr int R = 8 * NT;
    __shared__ __align__(16) float s_o[kOwnWarps][R][D + 4];
    __shared__ float s_ml[kOwnWarps][R][2];
    __shared__ float s_sum_ml[R][2];                      // the CTA's, for the cluster; its O takes the first warp's place
    __shared__ float s_w[R][kMostOwnCluster + kMostJoined];
    griddep_launch_dependents();                          // the merge may get ready
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int ctas = gridDim.x, rank = blockIdx.x, kvh = blockIdx.y / p.row_groups, r0 = (blockIdx.y % p.row_groups) * R, b = blockIdx.z;
    const int rows = min(R, p.group - r0), nQH = p.nKVH * p.group, head0 = kvh * p.group + r0;

    KeyWalk<T, D, NT> w;
    const int prefix_blocks = (p.prefix_here + kKeyBlock - 1) / kKeyBlock, stride = ctas * kOwnWarps;
    const T* const own_k = static_cast<const T*>(p.K) + b * p.own_batch + kvh * p.own_head; const T* const own_v = static_cast<const T*>(p.V) + b * p.own_batch + kvh * p.own_head;
    const T* const prefix_k = static_cast<const T*>(p.Kp) + kvh * p.prefix_head; const T* const prefix_v = static_cast<const T*>(p.Vp) + kvh * p.prefix_head;
    auto first_key = [&](int j) { return (j < prefix_blocks ? j : j - prefix_blocks) * kKeyBlock; };
    auto keys_of = [&](int j, int own) { return (j < prefix_blocks ? p.prefix_here : own) - first_key(j); };
    auto load_k = [&](int j, int own) { w.load_k((j < prefix_blocks ? prefix_k : own_k) + (long long)first_key(j) * D, keys_of(j, own)); };
    auto load_v = [&](int j, int own) { w.load_v((j < prefix_blocks ? prefix_v : own_v) + (long long)first_key(j) * D, keys_of(j, own)); };
    // the first block does not wait for the length: up to the cache's end the rows are there, whatever they hold
    int j = rank * kOwnWarps + warp;
    load_k(j, p.max_own);
    load_v(j, p.max_own);
    #pragma unroll
    for (int n = 0; n < NT; ++n)
        w.load_q(n, n * 8 + w.g < rows ? static_cast<const T*>(p.q) + b * p.q_batch + (long long)(head0 + n * 8 + w.g) * D : nullptr);
    const int own = p.max_own > 0 ? min(max(p.lengths[b], 0), p.max_own) : 0;
    const int blocks = prefix_blocks + (own + kKeyBlock - 1) / kKeyBlock;
    if (j < blocks) w.drop_v(keys_of(j, own));
    for (; j < blocks; j += stride) {
        w.step(keys_of(j, own), p.scale_log2, [&] { if (j + stride < blocks) load_k(j + stride, own); });
        if (j + stride < blocks) load_v(j + stride, own);
    }
    w.result([&](int row, float m, float l) { s_ml[warp][row][0] = m; s_ml[warp][row][1] = l; }, [&](int row, int d, float4 v) { *reinterpret_cast<float4*>(&s_o[warp][row][d]) = v; });
    __syncthreads();
    if (p.apart) {                                        // the CTA's result is a part
        const size_t row0 = (size_t(p.first_part + rank) * p.batch + b) * nQH + head0;
        for (int i = threadIdx.x; i < rows * (D / 4); i += kOwnThreads) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float most = -INFINITY, sum = 0.f;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            #pragma unroll
            for (int k = 0; k < kOwnWarps; ++k) most = fmaxf(most, s_ml[k][row][0]);
            #pragma unroll
            for (int k = 0; k < kOwnWarps; ++k) {
                const float f = weight_of(s_ml[k][row][0], most);
                const float4 v = *reinterpret_cast<const float4*>(&s_o[k][row][d]);
                sum += f * s_ml[k][row][1];
                x.x += f * v.x; x.y += f * v.y; x.z += f * v.z; x.w += f * v.w;
            }
            *reinterpret_cast<float4*>(&p.part_o[(row0 + row) * D + d]) = x;
            if (d == 0) *reinterpret_cast<float2*>(&p.part_ml[2 * (row0 + row)]) = make_float2(most, sum);
        }
        // One CTA's wait for the prefix's launch is this launch's: the merge waits for this one alone.  (All CTAs': those that are done
        // held the SMs that others could have begun on.)
        if (blockIdx.x + blockIdx.y + blockIdx.z == 0) griddep_wait();
        return;
    }
    // the CTA's, where a cluster follows
    if (ctas > 1) {
        for (int i = threadIdx.x; i < rows * D; i += kOwnThreads) {
            const int row = i / D, d = i % D;
            float most = -INFINITY, sum = 0.f, x = 0.f;
            for (int k = 0; k < kOwnWarps; ++k) most = fmaxf(most, s_ml[k][row][0]);
            for (int k = 0; k < kOwnWarps; ++k) { const float f = weight_of(s_ml[k][row][0], most); sum += f * s_ml[k][row][1]; x += f * s_o[k][row][d]; }
            s_o[0][row][d] = x;
            if (d == 0) { s_sum_ml[row][0] = most; s_sum_ml[row][1] = sum; }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (p.joined) griddep_wait();                         // the prefix's splits are there
    // every part's weight in the sum, 2^(m_i - m) / l, a warp per row: this unit's warps or CTAs, the prefix's splits
    const int parts = ctas > 1 ? ctas : kOwnWarps;
    const size_t part0 = size_t(b) * nQH + head0, next = size_t(p.batch) * nQH;
    for (int row = warp; row < rows; row += kOwnWarps) {
        float2 ml = make_float2(-INFINITY, 0.f), pml = make_float2(-INFINITY, kNoKey);
        if (lane < p.joined) pml = __ldcg(reinterpret_cast<const float2*>(&p.part_ml[2 * (part0 + row + lane * next)]));
        if (lane < parts)
            ml = ctas > 1 ? make_float2(load_cluster_f32(dme::smem_addr(&s_sum_ml[row][0]), lane), load_cluster_f32(dme::smem_addr(&s_sum_ml[row][1]), lane))
                          : make_float2(s_ml[lane][row][0], s_ml[lane][row][1]);
        float most = fmaxf(ml.x, pml.x);
        #pragma unroll
        for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        const float f = weight_of(ml.x, most), g = part_weight(pml, most);
        float sum = f * ml.y + (g == kNoKey ? 0.f : g * pml.y);
        #pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const float inv = p.joined + p.prefix_here + own > 0 ? 1.f / sum : 0.f;
        if (lane < parts) s_w[row][lane] = f * inv;
        if (lane < p.joined) s_w[row][kMostOwnCluster + lane] = g == kNoKey ? kNoKey : g * inv;
    }
    __syncthreads();
    // four columns per thread
    const int quads = rows * (D / 4), share = (quads + ctas - 1) / ctas, last = min(quads, (rank + 1) * share);
    for (int i = rank * share + threadIdx.x; i < last; i += kOwnThreads) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        const float* at = p.part_o + (part0 + row) * D + d;
        #pragma unroll 8
        for (int k = 0; k < p.joined; ++k) {
            const float f = s_w[row][kMostOwnCluster + k];
            float v[4];
            load_part<4>(at + k * next * D, v);
            #pragma unroll
            for (int e = 0; e < 4; ++e) if (f != kNoKey) x[e] += f * v[e];
        }
        for (int k = 0; k < parts; ++k) {
            const float4 v = ctas > 1 ? load_cluster_f32x4(dme::smem_addr(&s_o[0][row][d]), k) : *reinterpret_cast<const float4*>(&s_o[k][row][d]);
            const float f = s_w[row][k];
            x[0] += f * v.x; x[1] += f * v.y; x[2] += f * v.z; x[3] += f * v.w;
        }
        T* y = static_cast<T*>(p.o) + b * p.o_batch + (long long)(head0 + row) * D + d;
        *reinterpret_cast<uint2*>(y) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    }
    if (ctas > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");       // nobody leaves while a peer reads here
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// How a call is run.
struct SharedPlan {
    int splits, span;            // the prefix in a launch of its own: its splits, tiles of an item; 0: none, own_kernel reads the prefix
    bool joined;                 // own_kernel waits for the splits and merges them, no third launch
    int cluster, rows;           // CTAs and query rows (8 or 16) of a unit of own_kernel
    size_t off_ml, ws_bytes;
};

// Times in microseconds, from sizes alone, as they were measured over the range (sequences 2 to 256, prefixes of 100 to 32768 keys, 1 to 8
// key heads of 64 and 128, own caches up to 2000; of 460 drawn calls the mean is 1 % above the best form tried, one in ten is more than 5 % above it, the worst 1.34 times).  The sequences' own lengths are not known
// here: a little over half the caches' room.
//  * own_kernel alone: 4.5, and what it reads (the prefix for every sequence, from L2) at 7 TB/s or a warp's blocks of 16 keys at 0.8 each.
//    (32 / 8 heads of 128, 4 sequences, 512 keys in front: 6.5 against 9.0 with the prefix apart; 32 sequences, 2000 keys: 41 against 17.)
//  * the prefix apart: 5 for the launches and the merge; an item of the tcgen05 kernel takes 4.5 and 1.35 per key tile, 2.05 with two
//    query tiles; the own keys are read at 44 GB/s per SM, by the SMs that have no item and, once the items are done, by all; the parts are
//    written and read again.  (32 sequences, 2000 + up to 512 keys: 4 splits on 32 SMs 16.9, 8 on 64 18.9, 2 on 16 22.6.)
SharedPlan plan_shared(const b200p_shared_args& a) {
    SharedPlan pl{};
    const int sms = sm_count() > 0 ? sm_count() : 148, group = a.nQHeads / a.nKVHeads;
    pl.rows = group <= 8 ? 8 : 16;
    const long long units = (long long)a.batch * a.nKVHeads * ((group + pl.rows - 1) / pl.rows);
    auto cluster_for = [&](long long keys) {                    // CTAs of a unit: as many as find work and room
        int c = 1;
        while (c < kMostOwnCluster && units * c < 2 * sms && keys > 2 * kKeyBlock * kOwnWarps * c) c *= 2;
        return c;
    };
    pl.cluster = cluster_for((long long)a.max_own + a.prefix_len);
    if (a.prefix_len == 0) return pl;
    const double own_keys = 0.55 * a.max_own, key_bytes = 4.0 * a.D * a.nKVHeads;
    const double here_bytes = a.batch * (a.prefix_len + own_keys) * key_bytes;
    const double here_walk = 0.8 * ((a.prefix_len + own_keys) / (kKeyBlock * kOwnWarps * pl.cluster) + 1);
    const double here = 4.5 + (here_bytes / 7e6 > here_walk ? here_bytes / 7e6 : here_walk);
    const double own_work = a.batch * own_keys * key_bytes / 44e3;              // of one SM
    const int tokens = kBM / group, tiles = (a.batch + tokens - 1) / tokens, steps = (a.prefix_len + kBN - 1) / kBN, fixed = tuning(KNOB_SHARED_SPLITS, 0);
    double best = 0;
    int splits = 0, span = 0;
    const int first = fixed > 0 && fixed < kMostSplits ? fixed : kMostSplits;
    for (int per = (steps + first - 1) / first, next; per > 0; per = next) {    // key tiles of an item; the next is the smallest with fewer splits
        const int s = (steps + per - 1) / per;
        next = s > 1 && fixed == 0 ? (steps + s - 2) / (s - 1) : 0;
        for (int sp = 1; sp <= (tiles > 1 ? 2 : 1); ++sp) {
            const long long items = (long long)(tiles + sp - 1) / sp * a.nKVHeads * s;
            const double item = 4.5 + per * (sp == 1 ? 1.35 : 2.05), parts = double(s) * a.batch * a.nQHeads * a.D * 8 / 7.8e6;
            double t;
            if (items < sms) {
                const double alone = own_work / double(sms - items);            // the own keys on the SMs without an item
                t = alone + 2 <= item ? item : item + (alone + 2 - item) / alone * own_work / sms + 4;
            } else t = double((items + sms - 1) / sms) * item + own_work / sms + 5;
            if (best == 0 || t + parts < best) { best = t + parts; splits = s; span = sp; }
        }
    }
    const int forced = tuning(KNOB_SHARED_PREFIX, 0);
    if (splits > 0 && forced != 1 && (forced >= 2 || 5 + best < here)) {
        pl.splits = splits; pl.span = span;
        pl.cluster = cluster_for(a.max_own);
        // Where all of own_kernel's CTAs have room beside the items and there are few parts to add up for each, it may wait for them
        // and merge, which saves a launch (99 sequences, 2423 + up to 441 keys, 6 / 2 heads of 64, 14.9 -> 13.5 us; 145, 2984 + up to 306, 2 / 1,
        // 11.5 -> 9.9).  CTAs that wait where there is no room hold the SMs that others could begin on (48 of 32 / 4 heads of 64, 5000 + up to 1000,
        // 19.2 -> 26.4; 256, 32768 + up to 256, 32 / 8 of 128, 141 -> 157); short caches of heads of 64 are read soon enough all the same (103,
        // 4127 + up to 140, 16 / 4, 18.4 -> 16.1).  Many parts are quicker in merge_kernel's many warps. A unit's CTAs read group * splits * D
        // fp32 values of them, joined and apart: 5120 21.6 and 22.0 us (8 sequences, 12000 + up to 100 keys, 4 / 1 of 128), 12288 14.0 and 13.8 (4, 8000 + up to 100, 8 / 2),
        // 16384 22.8 and 18.9 (2, 15000 + up to 100, 8 / 1), 31744 18.2 and 14.0; below 6500 some lose too (16, 9000 + up to 100, 8 / 1, 6144: 29.0 and 25.9), above some gain 0.8.
        const long long items = (long long)((tiles + span - 1) / span) * a.nKVHeads * splits;
        const long long room = (a.D == 64 && a.max_own <= 160 ? sms : sms - items) * (pl.rows == 8 ? 4 : a.D == 64 ? 3 : 2);
        int c = pl.cluster;
        while (c > 1 && units * c > room && a.max_own <= 300 * c) c /= 2;
        pl.joined = splits <= kMostJoined && (forced == 3 || (forced != 2 && units * c <= room && group * splits * a.D <= 6500));
        if (pl.joined) pl.cluster = c;
        const size_t all = size_t(pl.splits + (pl.joined ? 0 : pl.cluster)) * a.batch * a.nQHeads;
        pl.off_ml = (all * a.D * 4 + 255) / 256 * 256;
        pl.ws_bytes = pl.off_ml + (all * 8 + 255) / 256 * 256;
    }
    return pl;
}

template <typename T, int D, int NT>
int launch_own(const OwnParams& p, int cluster, bool dependent, cudaStream_t st) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(cluster), unsigned(p.nKVH * p.row_groups), unsigned(p.batch)); cfg.blockDim = dim3(kOwnThreads); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1 && !p.apart) {
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
    const bool apart = pl.splits > 0;
    if (apart) {
        PackedParams p{};
        p.Q = q; p.K = Kp; p.V = Vp;
        p.seqQ = a.batch; p.seqK = a.prefix_len; p.batch = 1;
        p.nQH = a.nQHeads; p.nKVH = a.nKVHeads; p.group = group; p.splits = pl.splits; p.span = pl.span;
        p.scale_log2 = scale_log2;
        p.q_token = a.q_batch; p.q_head = D; p.k_token = p.v_token = D; p.k_head = p.v_head = a.prefix_head;
        p.part_o = part_o; p.part_ml = part_ml;
        if (int e = launch_packed<T, D, true, false>(p, a.dtype, st)) return e;
    }
    OwnParams w{};
    w.q = q; w.Kp = Kp; w.Vp = Vp; w.K = K; w.V = V; w.o = o; w.lengths = lengths;
    w.batch = a.batch; w.nKVH = a.nKVHeads; w.group = group; w.max_own = a.max_own; w.row_groups = (group + pl.rows - 1) / pl.rows;
    w.prefix_here = apart ? 0 : a.prefix_len;
    w.prefix_head = a.prefix_head; w.own_head = a.own_head; w.own_batch = a.own_batch; w.q_batch = a.q_batch; w.o_batch = a.o_batch;
    w.scale_log2 = scale_log2; w.apart = apart && !pl.joined; w.first_part = pl.splits; w.joined = pl.joined ? pl.splits : 0; w.part_o = part_o; w.part_ml = part_ml;
    if (int e = pl.rows == 8 ? launch_own<T, D, 1>(w, pl.cluster, apart, st) : launch_own<T, D, 2>(w, pl.cluster, apart, st)) return e;
    if (!apart || pl.joined) return B200P_OK;
    return launch_merge<T, D>(part_o, part_ml, pl.splits + pl.cluster, a.batch, a.nQHeads, o, a.o_batch, D, nullptr, nullptr, st);
}

int checked(const b200p_shared_args* args, b200p_shared_args* out) {
    if (!args) return B200P_E_NULL;
    b200p_shared_args a = *args;
    if (a.dtype != B200P_F16 && a.dtype != B200P_BF16) return B200P_E_DTYPE;
    if (a.D != 64 && a.D != 128) return B200P_E_DIM;
    if (a.nQHeads <= 0 || a.nKVHeads <= 0 || a.nQHeads % a.nKVHeads != 0) return B200P_E_DIM;
    if (a.batch < 0 || a.prefix_len < 0 || a.max_own < 0 || !(a.scale >= 0.f) || std::isinf(a.scale)) return B200P_E_LENGTH;
    if (a.prefix_len > kMostRows || a.max_own > kMostRows) return B200P_E_RANGE;
    if (a.nQHeads / a.nKVHeads > 128 || a.nQHeads > 65535 || a.batch > 65535 || (long long)a.batch * a.nQHeads > (1 << 28)) return B200P_E_RANGE;
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
