// What the kernels of dense attention over the paged cache share: the tree of drafted tokens at the end of a sequence, and
// the cut of all (sequence, kv-head) units into one contiguous range of token tiles per CTA.
//
// A sequence of S cached tokens ends with the n tokens of a drafted tree, so that P = S - n tokens are its prefix. Node i of
// the tree sees every token of the prefix, and node j (token P + j) where bit j of its 128-bit mask word is set. The 4 n query
// rows of a kv-head are numbered 4 i + g (g = query head of the group).
#pragma once

#include "tcgen05.cuh"

namespace ha {

constexpr int kMaxNodes = 128;         // drafted tokens per sequence: the bits of a node's mask
constexpr int kMaskWords = kMaxNodes / 32;

// One call's sequences.
struct DenseSeqs {
    const int32_t* page_table;  // [B][max_pages]
    const int32_t* seq_lens;    // [B] cached tokens, drafts included
    const int32_t* tree_lens;   // [B] drafted tokens, or null: T of each
    const uint32_t* tree_mask;  // [B][T][4], or null: a chain (node i sees the nodes 0 .. i)
    int32_t* status;
    int B, Hkv, T, max_pages, num_pages;
};

// Length and drafted tokens of sequence b; both 0 where it has nothing to do (no drafts, or a length out of range).
__device__ __forceinline__ void dense_seq(const DenseSeqs& d, int b, bool reporter, int& S, int& n) {
    S = __ldg(d.seq_lens + b);
    n = d.tree_lens != nullptr ? __ldg(d.tree_lens + b) : d.T;
    if (n < 0 || n > d.T || (n > 0 && (S < n || S > d.max_pages * kPage))) {
        if (reporter) report(d.status, HA_ERR_BAD_SEQ_LEN);
        n = 0;
    }
    if (n == 0) S = 0;
}

__device__ __forceinline__ int dense_page(const DenseSeqs& d, int b, int page_index) {
    int page = __ldg(d.page_table + (size_t)b * d.max_pages + page_index);
    if (page < 0 || page >= d.num_pages) {  // reported, and read as page 0
        report(d.status, HA_ERR_BAD_PAGE);
        page = 0;
    }
    return page;
}

// Mask words of node i of sequence b.
__device__ __forceinline__ uint4 dense_mask(const DenseSeqs& d, int b, int i) {
    if (d.tree_mask != nullptr) return __ldg(reinterpret_cast<const uint4*>(d.tree_mask) + (size_t)b * d.T + i);
    uint4 m;
    auto upto = [&](int word) { return i >= 32 * word + 31 ? 0xffffffffu : (i < 32 * word ? 0u : (2u << (i & 31)) - 1u); };
    m.x = upto(0); m.y = upto(1); m.z = upto(2); m.w = upto(3);
    return m;
}
__device__ __forceinline__ bool dense_bit(const uint4& m, int j) {
    const uint32_t w = j < 64 ? (j < 32 ? m.x : m.y) : (j < 96 ? m.z : m.w);
    return (w >> (j & 31)) & 1u;
}

// The nodes below n as a set.
__device__ __forceinline__ uint4 first_nodes(int n) {
    auto word = [&](int k) { return n >= 32 * k + 32 ? 0xffffffffu : (n <= 32 * k ? 0u : (1u << (n - 32 * k)) - 1u); };
    return make_uint4(word(0), word(1), word(2), word(3));
}

// a / b for a >= 0, b > 0: in 32 bits where they fit
__device__ __forceinline__ long long dense_div(long long a, long long b) {
    return (a | b) >> 32 == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

// The cut. A unit is a (sequence, kv-head, group of kRows query rows); its tokens are tiles of kTile. The tiles of all units,
// in order, are cut into gridDim.x ranges of equal length: the CTAs finish together whatever the lengths of the sequences,
// and a unit lies in at most a few CTAs. A range covers whole units but for its first and its last one, so a CTA
// leaves at most two partial results: number 0 of its first unit, number 1 of its last.
template <int kTile, int kRows>
struct DenseCut {
    static __host__ __device__ __forceinline__ int groups(int n) { return (n * kGroup + kRows - 1) / kRows; }
    static __device__ __forceinline__ long long seq_tiles(const DenseSeqs& d, int b, bool reporter, int& S, int& n) {
        dense_seq(d, b, reporter, S, n);
        return (long long)((S + kTile - 1) / kTile) * groups(n) * d.Hkv;
    }
    // Tiles per CTA and the tiles in front of sequence b_stop, by a whole warp.
    static __device__ void count(const DenseSeqs& d, int ctas, int lane, int b_stop, long long& quota, long long& before) {
        long long total = 0, front = 0;
        for (int b = lane; b < d.B; b += 32) {
            int S, n;
            const long long t = seq_tiles(d, b, false, S, n);
            total += t;
            if (b < b_stop) front += t;
        }
        total = warp_sum(total);
        before = warp_sum(front);
        quota = quota_of(total, ctas);
    }
    static __device__ __forceinline__ long long quota_of(long long total, int ctas) { return max(1ll, dense_div(total + ctas - 1, ctas)); }
    static __device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) v += __shfl_xor_sync(0xffffffffu, v, i);
        return v;
    }
};

struct DenseSegment {
    int b, kvh, group, S, n;
    int tile0, tile1, tiles;  // [tile0, tile1) of the unit's tiles
    int slot;                 // of the CTA's two partial results, if the segment is not the whole unit
    __device__ bool whole() const { return tile0 == 0 && tile1 == tiles; }
};

// Walks over the segments of a CTA's range. Built and advanced by a whole warp, all lanes alike.
template <int kTile, int kRows>
struct DenseCursor {
    using Cut = DenseCut<kTile, kRows>;
    const DenseSeqs& d;
    int b, S, n, tiles, groups, unit, tile;
    bool first;
    long long left;
    __device__ DenseCursor(const DenseSeqs& d_, int lane, bool reporter) : d(d_), b(0), S(0), n(0), tiles(0), groups(0), unit(0), tile(0), first(true), left(0) {
        // lane = sequence; the last 32 sequences stay in registers (all of them, as a rule)
        int S_ = 0, n_ = 0;
        long long t = 0, total = 0;
        const int last = (d.B - 1) & ~31;
        for (int b0 = 0; b0 <= last; b0 += 32) {
            S_ = n_ = 0;
            t = b0 + lane < d.B ? Cut::seq_tiles(d, b0 + lane, reporter, S_, n_) : 0;
            total += t;
        }
        total = Cut::warp_sum(total);
        const long long quota = Cut::quota_of(total, gridDim.x), at = quota * blockIdx.x;
        if (at >= total) return;
        left = min(quota, total - at);
        long long before = 0;
        for (int b0 = 0; b0 <= last; b0 += 32) {
            if (last > 0) {
                S_ = n_ = 0;
                t = b0 + lane < d.B ? Cut::seq_tiles(d, b0 + lane, false, S_, n_) : 0;
            }
            long long incl = t;
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const long long u = __shfl_up_sync(0xffffffffu, incl, i);
                if (lane >= i) incl += u;
            }
            const uint32_t reached = __ballot_sync(0xffffffffu, before + incl > at);
            if (reached != 0) {
                const int l = __ffs(reached) - 1;
                const long long in = __shfl_sync(0xffffffffu, at - (before + incl - t), l);
                b = b0 + l;
                S = __shfl_sync(0xffffffffu, S_, l);
                n = __shfl_sync(0xffffffffu, n_, l);
                tiles = (S + kTile - 1) / kTile;
                groups = Cut::groups(n);
                unit = (int)dense_div(in, tiles);
                tile = (int)(in - (long long)unit * tiles);
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    __device__ bool next(DenseSegment& s) {
        if (left <= 0) return false;
        if (tile >= tiles) {  // on to the next unit
            tile = 0;
            if (++unit >= groups * d.Hkv) {
                unit = 0;
                do {
                    ++b;  // (left > 0: there is one)
                    dense_seq(d, b, false, S, n);
                } while (n == 0);
                tiles = (S + kTile - 1) / kTile;
                groups = Cut::groups(n);
            }
        }
        s.b = b; s.S = S; s.n = n; s.tiles = tiles;
        s.kvh = unit / groups;
        s.group = unit - s.kvh * groups;
        s.tile0 = tile;
        s.tile1 = (int)min((long long)tiles, tile + left);
        s.slot = first ? 0 : 1;
        left -= s.tile1 - s.tile0;
        tile = s.tile1;
        first = false;
        return true;
    }
};

// The matrix instructions (mma.sync and tcgen05 alike) cut their fp32 sums towards zero instead of rounding them. A score of 128
// products in 8 steps comes out smaller by 1.0 to 1.25e-7 of itself on average (measured against 64 bits, with and without
// channels of larger scale; what is left beside that is 4e-7 of rms at scores above 4, as with fp32 multiply-adds). In an exponent
// of 20 that is 2e-6 of a weight, always to the same side, so log-sum-exps and received weights are corrected by it.
constexpr double kScoreCut = 1.0 / (1 << 23);

// exp2 by the special-function unit: 2 ulp; 0 for -inf, NaN for NaN
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ha
