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

// a / b for a >= 0, b > 0 (unsigned: fewer instructions)
__device__ __forceinline__ int dense_div(int a, int b) { return (int)((uint32_t)a / (uint32_t)b); }
constexpr int kMaxTiles = 1 << 30;  // of all units of a call together, which the entry points check: counts of tiles are 32 bits

// The cut. A unit is a (sequence, kv-head, group of kRows query rows); its tokens are tiles of kTile. The tiles of all units,
// in order, are cut into gridDim.x ranges of equal length (the quota): the CTAs finish together whatever the lengths of the
// sequences, and a unit lies in at most a few CTAs. A range covers whole units but for its first and its last one, so a CTA
// leaves at most two partial results: number 0 of its first unit, number 1 of its last.
// A range that crosses from one unit into another pays for the end of a unit twice, which costs as much as kCross tiles (11 us in
// the tensor-core attention; 0: next to nothing). So where the next larger quotas up to kCross more let every unit begin a range of
// its own, the smallest of those is taken, and the units are seen as padded to whole ranges (their span): 20011 tokens x 8 kv-heads
// with 32 drafts 38.7 -> 31.0 us, 131072 x 8 with 8 drafts 110 -> 101, 40000 x 8 with 64 75 -> 68.
template <int kTile, int kRows, int kCross>
struct DenseCut {
    static __host__ __device__ __forceinline__ int groups(int n) { return (n * kGroup + kRows - 1) / kRows; }
    static __device__ __forceinline__ int tiles_of(int S) { return dense_div(S + kTile - 1, kTile); }
    static __device__ __forceinline__ int span_of(int tiles, int quota, bool whole) {
        return whole ? dense_div(tiles + quota - 1, quota) * quota : tiles;
    }
    // The quota for `total` tiles, by a whole warp; lane b has the units of sequence b and their tiles (if B <= 32).
    static __device__ __forceinline__ int quota_of(const DenseSeqs& d, int total, int ctas, int lane, int units, int tiles, bool& whole) {
        const int even = max(1, dense_div(total + ctas - 1, ctas));
        whole = false;
        if (kCross == 0 || d.B > 32 || d.B * d.Hkv > ctas) return even;
        const int mine = even + lane;  // lane i tries a quota larger by i
        int need = 0;
        for (int b = 0; b < d.B; ++b) need += __shfl_sync(0xffffffffu, units, b) * dense_div(__shfl_sync(0xffffffffu, tiles, b) + mine - 1, mine);
        const uint32_t fits = __ballot_sync(0xffffffffu, need <= ctas && lane <= kCross);
        whole = fits != 0;
        return whole ? even + __ffs(fits) - 1 : even;
    }
    // The quota, the (padded) tiles in front of sequence b_stop and the span of its units, by a whole warp.
    static __device__ void count(const DenseSeqs& d, int ctas, int lane, int b_stop, int& quota, int& before, int& span) {
        int S, n, units = 0, tiles = 0, total = 0;
        for (int b = lane; b < d.B; b += 32) {
            dense_seq(d, b, false, S, n);
            tiles = tiles_of(S);
            units = groups(n) * d.Hkv;
            total += tiles * units;
        }
        bool whole;
        quota = quota_of(d, warp_sum(total), ctas, lane, units, tiles, whole);
        before = 0;
        for (int b = lane; b < b_stop; b += 32) {
            dense_seq(d, b, false, S, n);
            before += span_of(tiles_of(S), quota, whole) * (groups(n) * d.Hkv);
        }
        before = warp_sum(before);
        dense_seq(d, b_stop, false, S, n);
        span = span_of(tiles_of(S), quota, whole);
    }
    static __device__ __forceinline__ int warp_sum(int v) {
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
template <int kTile, int kRows, int kCross>
struct DenseCursor {
    using Cut = DenseCut<kTile, kRows, kCross>;
    const DenseSeqs& d;
    int b, S, n, tiles, groups, unit, tile;
    bool first;
    int left;
    __device__ DenseCursor(const DenseSeqs& d_, int lane, bool reporter) : d(d_), b(0), S(0), n(0), tiles(0), groups(0), unit(0), tile(0), first(true), left(0) {
        // lane = sequence; the last 32 sequences stay in registers (all of them, as a rule)
        int S_ = 0, n_ = 0;
        int total = 0;
        const int last = (d.B - 1) & ~31;
        auto units_of = [&] { return Cut::groups(n_) * d.Hkv; };
        for (int b0 = 0; b0 <= last; b0 += 32) {
            S_ = n_ = 0;
            if (b0 + lane < d.B) dense_seq(d, b0 + lane, reporter, S_, n_);
            total += Cut::tiles_of(S_) * units_of();
        }
        total = Cut::warp_sum(total);
        bool whole;
        const int quota = Cut::quota_of(d, total, gridDim.x, lane, units_of(), Cut::tiles_of(S_), whole), at = quota * blockIdx.x;
        int before = 0;
        for (int b0 = 0; b0 <= last; b0 += 32) {
            if (last > 0) {
                S_ = n_ = 0;
                if (b0 + lane < d.B) dense_seq(d, b0 + lane, false, S_, n_);
            }
            const int t = Cut::span_of(Cut::tiles_of(S_), quota, whole) * units_of();
            int incl = t;
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, incl, i);
                if (lane >= i) incl += u;
            }
            const uint32_t reached = __ballot_sync(0xffffffffu, before + incl > at);
            if (reached != 0) {
                const int l = __ffs(reached) - 1;
                const int in = __shfl_sync(0xffffffffu, at - (before + incl - t), l);
                b = b0 + l;
                S = __shfl_sync(0xffffffffu, S_, l);
                n = __shfl_sync(0xffffffffu, n_, l);
                tiles = Cut::tiles_of(S);
                groups = Cut::groups(n);
                const int span = Cut::span_of(tiles, quota, whole);
                unit = dense_div(in, span);
                tile = in - unit * span;
                // (the last range may be shorter, and so may the last one of a unit that is padded)
                left = whole ? min(quota, (tiles - tile)) : min(quota, total - at);
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
                tiles = Cut::tiles_of(S);
                groups = Cut::groups(n);
            }
        }
        s.b = b; s.S = S; s.n = n; s.tiles = tiles;
        s.kvh = unit / groups;
        s.group = unit - s.kvh * groups;
        s.tile0 = tile;
        s.tile1 = min(tiles, tile + left);
        s.slot = first ? 0 : 1;
        left -= s.tile1 - s.tile0;
        tile = s.tile1;
        first = false;
        return true;
    }
};

// Where the call's small arrays are read by every CTA behind the programmatic wait: their lines are asked into L2 in front of it
// (a hint that reads nothing, so it does not matter whether the kernel in front still writes them). Whole CTA.
__device__ __forceinline__ void dense_prefetch(const DenseSeqs& d) {
    auto line = [](const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); };
    const int at = threadIdx.x * 32;  // 128 bytes
    if (at < d.B) {
        line(d.seq_lens + at);
        if (d.tree_lens != nullptr) line(d.tree_lens + at);
    }
    if (blockIdx.x == 0)
        for (size_t i = at; i < (size_t)d.B * d.max_pages && i < (1u << 16); i += blockDim.x * 32) line(d.page_table + i);
}

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
