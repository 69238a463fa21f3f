// ---------------------------------------------------------------------------
// packed.cuh -- what the tcgen05 prefill kernel (prefill_tc.cuh, which includes this file) does differently for
// sequences of different lengths that lie one after the other:
//  * where its work items come from.  The lengths are known on the device only: a warp of every CTA walks over the offsets,
//    32 sequences at a time, and finds the CTA's items by number.  Items are numbered by falling number of key tiles; the grid has
//    a CTA for each of them, and a CTA that is done takes over the next one's number from the hardware (launch_control.cuh): the
//    heaviest items first, no SM idle while there are others, no counter in memory to clear ahead of a launch or to share.
//  * its rows.  A tile holds the heads of a group for 128 / group tokens, token by token: keys are read once for a group, a
//    prompt of 20 tokens fills 80 rows of a tile with 4 heads to a group, and the causal mask costs no more tiles than it would by head.
//  * what happens to rows that are no numbers.  A weight of zero times a value that is none (behind a causal row's position in
//    its key tile) gives none, and so does a tile of nothing but -inf scores ahead of finite ones.  Rows with such a result are done
//    again key by key (attn_rows.cuh), from those keys alone that the row sees, by the warp that has them: 32 rows 4 to 10 us a key.  A value that
//    is no number and seen costs every row that sees it as much (a tile of one head over 65536 keys, 282 ms for less than 1): it is right, not fast.
// ---------------------------------------------------------------------------
#pragma once
#include "attn_rows.cuh"
#include "launch_control.cuh"

namespace b200p {

// The next item is looked for when the K tile of this many steps before the item's end is asked for.  (1, 2, 3, 4: no difference.)
constexpr int kAskAhead = 2;

// What takes a time that grows with the sizes and holds up the CTA's other warps says every so often that it is at work (dme::say_alive), so
// that their bounded waits (2 s) go on: the walk over very many sequences, an item of very many key tiles, rows done again on long caches.
constexpr int kAliveChunks = 1024, kAliveTiles = 4096, kAliveKeys = 4096;

constexpr float kNoKey = -1.f;             // in place of a part's sum, whose O is not stored then

struct PackedParams : PrefillParams {      // seqQ, seqK: rows of Q and of K and V; batch: sequences; span, scale_log2, causal, nKVH, group
    const int *q_offsets, *k_offsets;      // without WALK none, one sequence of all rows
    const void *Q, *K, *V;
    void* O;
    long long q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    int tokens;                            // of a tile: 128 / group
    int o_wide;                            // rows of O start on 32 bytes
    int splits;                            // PARTIAL: items that share a block's keys
    float* part_o;                         // PARTIAL: [splits][seqQ][nQH][D]
    float* part_ml;                        // PARTIAL: [splits][seqQ][nQH][2]: maximum in log2 units, sum; kNoKey for the sum: the row sees no key
};

// One work item: up to two tiles of one sequence and key head, or a share of their keys.
struct PackedItem {
    int kvh, nmax;
    int first;                 // key tile of step 0
    int q0[2], n[2];           // per query tile: first token of the sequence, steps
    int q_row, k_row;          // the sequence's first rows
    int queries, keys, ahead;  // its lengths, and keys - queries
    int split;
};

// The tiles of a sequence's qb-th block: where they start, how many key tiles they have.
__device__ __forceinline__ void packed_tiles_of(const PackedParams& p, int qb, PackedItem& w) {
    w.ahead = w.keys - w.queries;
    #pragma unroll
    for (int t = 0; t < 2; ++t) {
        w.q0[t] = (qb * p.span + t) * p.tokens;
        w.n[t] = 0;
        if (t >= p.span || w.q0[t] >= w.queries) { w.q0[t] = w.queries; continue; }        // no such tile
        const int seen = p.causal ? min(w.keys, w.ahead + min(w.q0[t] + p.tokens, w.queries)) : w.keys;
        w.n[t] = seen > 0 ? (seen + kBN - 1) / kBN : 0;
    }
    w.nmax = max(w.n[0], w.n[1]);
}

// PARTIAL: the share of the block's keys that is split w.split.
__device__ __forceinline__ void packed_share(const PackedParams& p, PackedItem& w) {
    const int share = (w.nmax + p.splits - 1) / p.splits;
    w.first = w.split * share;
    #pragma unroll
    for (int t = 0; t < 2; ++t) w.n[t] = max(0, min(w.n[t] - w.first, share));
    w.nmax = max(w.n[0], w.n[1]);
}

// Without WALK: item `id` of the one sequence.
__device__ __forceinline__ PackedItem packed_split(const PackedParams& p, int id) {
    PackedItem w{};
    const int rest = id / p.splits, qb = rest / p.nKVH;
    w.split = id - rest * p.splits; w.kvh = rest - qb * p.nKVH;
    w.queries = p.seqQ; w.keys = p.seqK;
    packed_tiles_of(p, qb, w);
    packed_share(p, w);
    return w;
}

// Beyond 32 * 32 sequences the walk looks at all offsets once a level.  Measured, sequences of 0 to 8 tokens, 2 / 1 heads of 64, and the same with one
// of 3000 among them, which brings a dozen levels: 1024 sequences 52 and 97 us, 8192 0.29 and 1.3 ms, 65536 2.6 and 13.9 ms, 2^20 43 and 227 ms.
// Finds this CTA's items and calls publish(i, item) for them in order, the last time with kvh = -1, until it returns false.  One warp.
// answer, bar: shared memory for requests of further CTAs' items.
template <typename Publish>
__device__ __forceinline__ bool packed_walk(const PackedParams& p, void* answer, uint64_t* bar, uint64_t* alive, Publish&& publish) {
    constexpr unsigned kAll = 0xffffffffu;
    const int lane = threadIdx.x % 32;
    const int block = p.span * p.tokens, chunks = (p.batch + 31) / 32, per = p.nKVH * p.splits;
    int q = 0, k = 0, n = 0, m = 0;                             // this lane's sequence: first rows, lengths
    auto load = [&](int c) {
        const int b = c * 32 + lane;
        if (c % kAliveChunks == kAliveChunks - 1 && lane == 0) dme::say_alive(alive);
        q = k = n = m = 0;
        if (b >= p.batch) return;
        q = min(max(p.q_offsets[b], 0), p.seqQ); n = min(max(p.q_offsets[b + 1], q), p.seqQ) - q;
        k = min(max(p.k_offsets[b], 0), p.seqK); m = min(max(p.k_offsets[b + 1], k), p.seqK) - k;
    };
    int id = int(blockIdx.x), drawn = 0;
    // the next item's number, or -1; -2: the wait for it gave up.
    auto next_id = [&]() -> int {
        if (lane == 0) request_cta(answer, bar);
        const bool there = __all_sync(kAll, dme::wait(bar, uint32_t(drawn & 1), nullptr)) != 0;       // in any case: the answer arrives in this CTA's memory
        ++drawn;
        const int x = lane == 0 && there ? taken_cta(answer) : -1;
        __syncwarp();
        return there ? __shfl_sync(kAll, x, 0) : -2;
    };
    int most = 0, blocks = 0, chunk_most = 0;                   // key tiles of the longest sequence, blocks of all; lane c: of chunk c
    #pragma unroll 4
    for (int c = 0; c < chunks; ++c) {                          // (four loads under way)
        load(c);
        blocks += (n + block - 1) / block;
        const int tiles = __reduce_max_sync(kAll, n == 0 ? 0 : max(1, (m + kBN - 1) / kBN));
        if (lane == c) chunk_most = tiles;
        most = max(most, tiles);
    }
    blocks = __reduce_add_sync(kAll, blocks);
    // Blocks are numbered by levels of `unit` key tiles, the heaviest level first: a dozen levels balance as well as one for every
    // number of tiles, and are found faster (a visit of a level is some 300 cycles of divisions and shuffles).
    const int unit = max(1, (most + 11) / 12);
    // the sequence's first block (of `block` tokens) of this level or a heavier one; every block counts as having one tile at least
    auto first_of = [&](int level) {
        const int nb = (n + block - 1) / block, behind = (level - 1) * unit * kBN;
        if (level == 1) return 0;
        if (m <= behind) return nb;
        if (!p.causal) return 0;
        const int x = behind - (m - n);                         // a block whose last token is behind x sees more than `behind` keys
        return x < 0 ? 0 : min(nb, x / block);
    };
    int level = 0, c = 0, at = chunks == 1 ? 0 : -1;            // at: the chunk that is loaded
    int base = 0, first = 0, count = 0, upto = 0, total = -1;   // of the chunk at this level: blocks before it, lane's first, lane's, up to the lane's, all; -1: not counted
    auto restart = [&] { level = (most + unit - 1) / unit; c = 0; base = 0; total = -1; };
    restart();
    bool fine = true;
    for (int it = 0;;) {
        PackedItem w{};
        w.kvh = -1;
        const int entry = id >= 0 ? id / per : 0, rest = id - entry * per;
        if (id >= 0 && entry >= blocks) {                       // the grid has room for more items than there are
            id = next_id();
            if (id >= 0) continue;
        }
        fine = id != -2;
        if (id >= 0) {
            if (entry < base) restart();                        // numbers need not come in order
            for (;;) {
                if (total < 0) {
                    if (c < 32 && __shfl_sync(kAll, chunk_most, c & 31) <= (level - 1) * unit) total = 0;
                    else {
                        if (at != c) { load(c); at = c; }
                        first = first_of(level);
                        count = first_of(level + 1) - first;
                        upto = count;
                        #pragma unroll
                        for (int d = 1; d < 32; d <<= 1) { const int x = __shfl_up_sync(kAll, upto, d); if (lane >= d) upto += x; }
                        total = __shfl_sync(kAll, upto, 31);
                    }
                }
                if (entry - base < total || level == 0) break;
                base += total; total = -1;
                if (++c == chunks) { c = 0; --level; }
            }
            const int within = entry - base;
            const int src = __ffs(__ballot_sync(kAll, upto > within)) - 1;
            const int qb = __shfl_sync(kAll, first + upto - 1 - within, src);       // a sequence's last block of the level first
            w.kvh = rest / p.splits; w.split = rest - w.kvh * p.splits;
            w.q_row = __shfl_sync(kAll, q, src); w.k_row = __shfl_sync(kAll, k, src);
            w.queries = __shfl_sync(kAll, n, src); w.keys = __shfl_sync(kAll, m, src);
            packed_tiles_of(p, qb, w);
            if (p.splits > 1) packed_share(p, w);
        }
        const bool go_on = publish(it, w) && w.kvh >= 0;
        ++it;
        if (!go_on) break;
        id = next_id();
    }
    return fine;
}

// One query row once more, by the whole warp, from the n keys that it sees, and out: PARTIAL as fp32, not divided, with its
// maximum and sum, else as 16 bits.
template <typename T, int D, bool PARTIAL>
__device__ __forceinline__ void packed_row_again(const T* q, const T* K, const T* V, long long k_token, long long v_token, int n, float scale_log2, void* out, float* ml,
                                                 uint64_t* alive) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x % 32;
    float x[E];
    load_part<T, E>(q + lane * E, x);
    RowState<D> st;
    for (int j = 0; j < n; j += kAliveKeys) {
        attend_keys<T, D>(st, x, K + j * k_token, V + j * v_token, k_token, v_token, min(n - j, kAliveKeys), scale_log2);
        if (lane == 0) dme::say_alive(alive);
    }
    if constexpr (PARTIAL) {
        for (int i = 0; i < E; ++i) static_cast<float*>(out)[lane * E + i] = st.o[i];
        if (lane == 0) { ml[0] = st.m; ml[1] = st.l; }
    } else {
        for (int i = 0; i < E; ++i) static_cast<T*>(out)[lane * E + i] = from_float<T>(st.o[i] / st.l);       // every score -inf: 0 / 0
    }
}

// A row of a tile without keys (of this item's share): zeros, or a sum of nothing.
template <typename T, typename Sh>
__device__ __forceinline__ void packed_no_keys(const PackedParams& p, const PackedItem& w, int token, int g) {
    const int head = w.kvh * p.group + g;
    if constexpr (Sh::PARTIAL) {
        reinterpret_cast<float2*>(p.part_ml)[(size_t(w.split) * p.seqQ + w.q_row + token) * (p.nKVH * p.group) + head] = make_float2(-INFINITY, kNoKey);
    } else {
        uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.O) + (w.q_row + token) * p.o_token + head * p.o_head);
        for (int i = 0; i < Sh::DV / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
    }
}

// A tile's rows out, a row per thread: v is the thread's row of O, m and l its maximum and sum.
template <typename T, typename Sh>
__device__ __forceinline__ void packed_epilogue(const PackedParams& p, const PackedItem& w, uint32_t (&v)[Sh::DV], float m, float l, int nt, int q0, int row_token, bool live, int r,
                                                uint64_t* alive) {
    constexpr int D = Sh::DV;
    constexpr bool PARTIAL = Sh::PARTIAL;
    const int token = q0 + row_token, g = r - row_token * p.group;
    const int lo = w.first * kBN, hi = min(min(w.keys, p.causal ? w.ahead + token + 1 : w.keys), lo + nt * kBN);
    const bool sees = live && hi > lo;                          // some key of this item's share
    float z[8] = {l * 0.f};                                     // zeros, unless some element is no number or infinite
    #pragma unroll
    for (int i = 0; i < D; ++i) z[i % 8] = fmaf(__uint_as_float(v[i]), 0.f, z[i % 8]);
    const bool bad = sees && ((z[0] + z[1]) + (z[2] + z[3])) + ((z[4] + z[5]) + (z[6] + z[7])) != 0.f;
    // A row per thread, 32 bytes at a time (where rows start on 32): no barrier and no other lane's row in the way.  (Through a staging tile, as whole lines, by the
    // tile's threads and a tensor-map store or by each warp for itself: 16 prompts of 100 to 1500 tokens, heads of 128, 103 and 111 us
    // against 101.)
    unsigned char* mine = nullptr;
    if constexpr (PARTIAL) {
        const size_t row = (size_t(w.split) * p.seqQ + w.q_row + token) * (p.nKVH * p.group) + w.kvh * p.group + g;
        if (live) reinterpret_cast<float2*>(p.part_ml)[row] = sees ? make_float2(m, l) : make_float2(-INFINITY, kNoKey);
        if (sees) mine = reinterpret_cast<unsigned char*>(p.part_o + row * D);
    } else if (live) mine = reinterpret_cast<unsigned char*>(static_cast<T*>(p.O) + (w.q_row + token) * p.o_token + (w.kvh * p.group + g) * p.o_head);
    if (mine) {
        const float inv = 1.f / l;
        #pragma unroll
        for (int i = 0; i < D * (PARTIAL ? 4 : 2) / 32; ++i) {
            uint32_t x[8];
            #pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = i * 8 + e;                        // 32-bit word of the row
                if constexpr (PARTIAL) x[e] = v[k];
                else x[e] = sees ? pack2<T>(__uint_as_float(v[2 * k]) * inv, __uint_as_float(v[2 * k + 1]) * inv) : 0u;
            }
            if (PARTIAL || p.o_wide) VecIO<32>::store(mine + i * 32, x);
            else {
                reinterpret_cast<uint4*>(mine)[2 * i] = make_uint4(x[0], x[1], x[2], x[3]);
                reinterpret_cast<uint4*>(mine)[2 * i + 1] = make_uint4(x[4], x[5], x[6], x[7]);
            }
        }
    }
    unsigned again = __ballot_sync(0xffffffffu, bad);
    if (!again) return;
    __syncwarp();                                               // what is done again is written last
    for (; again; again &= again - 1) {
        const int src = __ffs(again) - 1;
        const int tok = __shfl_sync(0xffffffffu, token, src), head = w.kvh * p.group + __shfl_sync(0xffffffffu, g, src), n = __shfl_sync(0xffffffffu, hi, src) - lo;
        const long long key = (long long)w.k_row + lo;
        const size_t row = (size_t(w.split) * p.seqQ + w.q_row + tok) * (p.nKVH * p.group) + head;
        void* out = PARTIAL ? static_cast<void*>(p.part_o + row * D) : static_cast<void*>(static_cast<T*>(p.O) + (w.q_row + tok) * p.o_token + head * p.o_head);
        packed_row_again<T, D, PARTIAL>(static_cast<const T*>(p.Q) + (w.q_row + tok) * p.q_token + head * p.q_head, static_cast<const T*>(p.K) + key * p.k_token + w.kvh * p.k_head,
                                        static_cast<const T*>(p.V) + key * p.v_token + w.kvh * p.v_head, p.k_token, p.v_token, n, p.scale_log2, out, PARTIAL ? p.part_ml + 2 * row : nullptr, alive);
    }
}

} // namespace b200p
