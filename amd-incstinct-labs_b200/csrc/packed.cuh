// ---------------------------------------------------------------------------
// packed.cuh -- what the tcgen05 prefill kernel (prefill_tc.cuh, which includes this file) does differently for
// sequences of different lengths that lie one after the other:
//  * where its work items come from.  The lengths are known on the device only: a warp of every CTA walks over the offsets,
//    32 sequences at a time, and finds the CTA's items by number.  Items are numbered by falling number of key tiles, and CTA c
//    of g takes the numbers c, 2g-1-c, 2g+c, 4g-1-c, ...: the heaviest first, and a CTA that got a heavy one of a round gets a light
//    one of the next.  No counter to clear ahead of the launch, no state between launches, the same work for a CTA every time.
//  * its rows.  A tile holds the heads of a group for 128 / group tokens, token by token.
//  * how a tile is stored: tiles of whole tokens through the tensor map, a sequence's last one row by row, for the rows
//    behind it are the next sequence's.
//  * what happens to rows that are no numbers.  A weight of zero times a value that is none (behind a causal row's position in
//    its key tile) gives none, and so does a tile of nothing but -inf scores ahead of finite ones.  Rows with such a result are done
//    again key by key (attn_rows.cuh), from those keys alone that the row sees.
// ---------------------------------------------------------------------------
#pragma once
#include "attn_rows.cuh"

namespace b200p {

struct PackedParams : PrefillParams {      // seqQ, seqK: rows of Q and of K and V; batch: sequences; span, scale_log2, causal, nKVH, group
    const int *q_offsets, *k_offsets;      // null: one sequence of all rows
    const void *Q, *K, *V;
    void* O;
    long long q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    int tokens;                            // of a tile: 128 / group
    int splits;                            // PARTIAL: items that share a block's keys
    float* part_o;                         // PARTIAL: [splits][seqQ][nQH][D]
    float* part_ml;                        // PARTIAL: [splits][seqQ][nQH][2]: maximum in log2 units, sum; a sum of 0: no key
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

// Calls publish(i, item) for this CTA's items in order, the last one with kvh = -1, until it returns false.  One warp.
template <typename Publish>
__device__ __forceinline__ void packed_walk(const PackedParams& p, Publish&& publish) {
    constexpr unsigned kAll = 0xffffffffu;
    const int lane = threadIdx.x % 32;
    const int block = p.span * p.tokens, chunks = (p.batch + 31) / 32;
    int q = 0, k = 0, n = 0, m = 0;                             // this lane's sequence: first rows, lengths
    auto load = [&](int c) {
        const int b = c * 32 + lane;
        q = k = n = m = 0;
        if (b >= p.batch) return;
        int q1 = p.seqQ, k1 = p.seqK;
        if (p.q_offsets) {
            q = min(max(p.q_offsets[b], 0), p.seqQ); q1 = min(max(p.q_offsets[b + 1], q), p.seqQ);
            k = min(max(p.k_offsets[b], 0), p.seqK); k1 = min(max(p.k_offsets[b + 1], k), p.seqK);
        }
        n = q1 - q; m = k1 - k;
    };
    // the sequence's first block of `block` tokens that has `level` key tiles or more; every block counts as having one at least
    auto first_of = [&](int level) {
        const int nb = (n + block - 1) / block, behind = (level - 1) * kBN;
        if (level == 1) return 0;
        if (m <= behind) return nb;
        if (!p.causal) return 0;
        const int x = behind - (m - n);                         // a block whose last token is behind x sees more than `behind` keys
        return x < 0 ? 0 : min(nb, x / block);
    };
    int levels = 0, chunk_levels = 0, blocks = 0;               // lane c: of chunk c
    for (int c = 0; c < chunks; ++c) {
        load(c);
        blocks += (n + block - 1) / block;
        const int most = __reduce_max_sync(kAll, n == 0 ? 0 : max(1, (m + kBN - 1) / kBN));
        if (lane == c) chunk_levels = most;
        levels = max(levels, most);
    }
    blocks = __reduce_add_sync(kAll, blocks);
    const int per = p.nKVH * p.splits;
    int level = levels, c = 0, at = -1;                         // at: the chunk that is loaded
    if (chunks == 1) at = 0;
    int base = 0, first = 0, count = 0, upto = 0, total = -1;   // of the chunk at this level: blocks before it, lane's first, lane's, up to the lane's, all; -1: not counted
    for (int it = 0;; ++it) {
        const int g = int(gridDim.x), id = it * g + ((it & 1) ? g - 1 - int(blockIdx.x) : int(blockIdx.x));
        const int entry = id / per, rest = id - entry * per;
        PackedItem w{};
        w.kvh = -1;
        if (entry >= blocks) level = 0;                         // no more
        while (level > 0) {
            if (total < 0) {
                if (c < 32 && __shfl_sync(kAll, chunk_levels, c & 31) < level) total = 0;
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
            if (entry - base < total) break;
            base += total; total = -1;
            if (chunks == 1) {                                  // on to the next level that a block has: that of the last one before `first`
                const int before = min(m, p.causal ? m - n + first * block : m);
                level = __reduce_max_sync(kAll, first == 0 ? 0 : max(1, (before + kBN - 1) / kBN));
            } else if (++c == chunks) { c = 0; --level; }
        }
        if (level > 0) {
            const int within = entry - base;
            const int src = __ffs(__ballot_sync(kAll, upto > within)) - 1;
            const int qb = __shfl_sync(kAll, first + within - (upto - count), src);
            w.kvh = rest / p.splits; w.split = rest - w.kvh * p.splits;
            w.q_row = __shfl_sync(kAll, q, src); w.k_row = __shfl_sync(kAll, k, src);
            w.queries = __shfl_sync(kAll, n, src); w.keys = __shfl_sync(kAll, m, src);
            w.ahead = w.keys - w.queries;
            #pragma unroll
            for (int t = 0; t < 2; ++t) {
                w.q0[t] = qb * block + t * p.tokens;
                if (t >= p.span || w.q0[t] >= w.queries) { w.q0[t] = w.queries; continue; }        // no such tile
                const int seen = p.causal ? min(w.keys, w.ahead + min(w.q0[t] + p.tokens, w.queries)) : w.keys;
                w.n[t] = seen > 0 ? (seen + kBN - 1) / kBN : 0;
            }
            if (p.splits > 1) {
                const int share = (max(w.n[0], w.n[1]) + p.splits - 1) / p.splits;
                w.first = w.split * share;
                #pragma unroll
                for (int t = 0; t < 2; ++t) w.n[t] = max(0, min(w.n[t] - w.first, share));
            }
            w.nmax = max(w.n[0], w.n[1]);
        }
        if (!publish(it, w) || w.kvh < 0) return;
    }
}

// One query row once more, by the whole warp, from the n keys that it sees, and out: PARTIAL as fp32, not divided, with its
// maximum and sum, else as 16 bits.
template <typename T, int D, bool PARTIAL>
__device__ __forceinline__ void packed_row_again(const T* q, const T* K, const T* V, long long k_token, long long v_token, int n, float scale_log2, void* out, float* ml) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x % 32;
    float x[E];
    load_part<T, E>(q + lane * E, x);
    RowState<D> st;
    attend_keys<T, D>(st, x, K, V, k_token, v_token, n, scale_log2);
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
        reinterpret_cast<float2*>(p.part_ml)[(size_t(w.split) * p.seqQ + w.q_row + token) * (p.nKVH * p.group) + head] = make_float2(-INFINITY, 0.f);
    } else {
        uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(p.O) + (w.q_row + token) * p.o_token + head * p.o_head);
        for (int i = 0; i < Sh::DV / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
    }
}

// A tile's rows out: v is the thread's row of O, m and l its maximum and sum.
// any_of_tile: a barrier of the tile's threads that says whether any of them came with true.
template <typename T, typename Sh, typename Sync, typename Any>
__device__ __forceinline__ void packed_epilogue(const PackedParams& p, const PackedItem& w, uint32_t (&v)[Sh::DV], float m, float l, int nt, int q0, int row_token,
                                                bool live, int r, unsigned char* stage, bool issuer, Sync&& tile_sync, Any&& any_of_tile, const CUtensorMap* mapO) {
    constexpr int D = Sh::DV;
    constexpr bool PARTIAL = Sh::PARTIAL;
    const int token = q0 + row_token, g = r - row_token * p.group;
    const int lo = w.first * kBN, hi = min(min(w.keys, p.causal ? w.ahead + token + 1 : w.keys), lo + nt * kBN);
    const bool sees = live && hi > lo;                          // some key of this item's share
    float z = 0.f;
    if (sees) {
        #pragma unroll
        for (int i = 0; i < D; ++i) z = fmaf(__uint_as_float(v[i]), 0.f, z);
        z = fmaf(l, 0.f, z);
    }
    const bool bad = z != 0.f;                                  // some element is no number, or infinite
    const size_t part_row = (size_t(w.split) * p.seqQ + w.q_row + token) * (p.nKVH * p.group) + w.kvh * p.group + g;
    T* const o_row = static_cast<T*>(p.O) + (w.q_row + token) * p.o_token + (w.kvh * p.group + g) * p.o_head;
    bool some_bad = false;
    if constexpr (PARTIAL) {
        if (live) {
            reinterpret_cast<float2*>(p.part_ml)[part_row] = sees ? make_float2(m, l) : make_float2(-INFINITY, 0.f);
            if (sees) {
                float* o = p.part_o + part_row * D;
                #pragma unroll
                for (int i = 0; i < D; i += 8) VecIO<32>::store(o + i, *reinterpret_cast<uint32_t(*)[8]>(&v[i]));
            }
        }
        some_bad = __any_sync(0xffffffffu, bad);
    } else {
        const float inv = 1.f / l;
        #pragma unroll
        for (int hb = 0; hb < D / 64; ++hb) {
            if (issuer) dme::store_wait_read<0>();              // the previous store from this staging tile has read it out
            if (hb == 0) some_bad = any_of_tile(bad);
            else tile_sync();
            // the tensor map's box is all the tile's tokens: not past the sequence's end, and not where rows follow that must not be overtaken
            const bool whole = q0 + p.tokens <= w.queries && !some_bad;
            #pragma unroll
            for (int ch = 0; ch < 8; ++ch) {
                const int c0 = hb * 64 + ch * 8;
                uint32_t x[4];
                #pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[i] = sees ? pack2<T>(__uint_as_float(v[c0 + 2 * i]) * inv, __uint_as_float(v[c0 + 2 * i + 1]) * inv) : 0u;
                *reinterpret_cast<uint4*>(stage + swz128(r, ch)) = make_uint4(x[0], x[1], x[2], x[3]);
            }
            if (whole) {
                dme::fence_proxy_async_smem();
                tile_sync();
                if (issuer) {
                    dme::store_tile_4d(mapO, hb * 64, 0, w.q_row + q0, w.kvh, stage);
                    dme::store_commit();
                }
            } else {
                tile_sync();
                const int rows = min(w.queries - q0, p.tokens) * p.group;
                for (int i = r / 8; i < rows; i += 16) {        // eight lanes a row's 128 bytes
                    const int tok = i / p.group, head = w.kvh * p.group + i - tok * p.group;
                    T* o = static_cast<T*>(p.O) + (w.q_row + q0 + tok) * p.o_token + head * p.o_head + hb * 64 + (r % 8) * 8;
                    *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(stage + swz128(i, r % 8));
                }
            }
        }
    }
    if (!some_bad) return;
    if constexpr (PARTIAL) __syncwarp(); else tile_sync();      // what is done again is written last
    for (unsigned again = __ballot_sync(0xffffffffu, bad); again; again &= again - 1) {
        const int src = __ffs(again) - 1;
        const int tok = __shfl_sync(0xffffffffu, token, src), head = w.kvh * p.group + __shfl_sync(0xffffffffu, g, src), n = __shfl_sync(0xffffffffu, hi, src) - lo;
        const long long key = (long long)w.k_row + lo;
        void* out = PARTIAL ? static_cast<void*>(p.part_o + __shfl_sync(0xffffffffu, (unsigned long long)part_row, src) * D)
                            : reinterpret_cast<void*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(o_row), src));
        float* ml = PARTIAL ? p.part_ml + 2 * __shfl_sync(0xffffffffu, (unsigned long long)part_row, src) : nullptr;
        packed_row_again<T, D, PARTIAL>(static_cast<const T*>(p.Q) + (w.q_row + tok) * p.q_token + head * p.q_head, static_cast<const T*>(p.K) + key * p.k_token + w.kvh * p.k_head,
                                        static_cast<const T*>(p.V) + key * p.v_token + w.kvh * p.v_head, p.k_token, p.v_token, n, p.scale_log2, out, ml);
    }
}

} // namespace b200p
