// Dense attention of many query rows per kv-head over the paged cache, on the 5th-generation tensor cores (tcgen05): drafted
// trees of more than a few nodes.
//
// The mathematics of tree_attention.cuh with the rows of a kv-head (4 per node) on the 128 lanes of tensor memory. Per tile of
// 128 tokens S = Q K^T (128 x 128 sums), P = e^{S - m} by two threads per row, O += P V with P handed over in tensor memory as two bf16
// (hi + lo) in the columns S was read from. A CTA works on two such chains ("streams") at a time, so that one's softmax runs
// under the other's products:
//   * up to 128 rows (kWide == false): both streams have the same rows and take every second tile; their results are joined
//     at the end of the unit, each group of softmax warps reading a quarter of the columns of both.
//   * up to 256 rows (kWide): stream w has rows 128 w .. 128 w + 127, and a tile of K and V serves both.
//
// Roles of the warps: 0 issues the products, 1 loads K and V tiles by TMA (two boxes of 64 elements x 128 tokens, 128-byte
// swizzle) into a ring of 32 KB slots, K and V of a tile in turn, 2 - 17 are the softmax warps, eight per stream: a thread has 64 of
// a row's 128 columns, and the two halves of a row agree on its maximum through shared memory. Streams that take
// different tiles have a ring of three slots each, streams that share tiles a ring of five; a barrier is waited for in every
// phase by the one who uses it.
//
// One warp issues for both streams, P V of a tile and Q K^T of the stream's next one back to back: the streams then take turns at
// the tensor core (two issuers leave them in step: both wait for their softmax at the same time). S takes the place of P, so S
// complete means O complete too, and the softmax warps may rescale O (which they do only when a row's maximum has grown by more
// than 2^8) without another barrier. P is announced in two parts of 64 tokens (32 of each half): the first one's product runs under
// the exponentials of the second.
//
// What bounds it. A stream's turn is 24 products of 64 clocks (1536; the lo halves are 512 of them); the streams take turns every
// 2300 to 2450 clocks, the rest being the issuing warp's waits and the way from scores to weights (1400 clocks to the first half
// of P, 700 more to the second). Up to 128 rows: K and V of a tile take 2760 clocks at the copy rate, so a long cache is read at
// 4.8 to 5.7 TB/s (131072 tokens x 8 kv-heads with 8 drafts: 94 us in a burst, 111 after a second, floor 82). 256 rows: 4 x 131072
// x 8 with 64 drafts take 680 us in a burst (810 TFLOP/s, 1210 with the lo halves), where the power limit brings the clock to
// 1.36 GHz, and 775 to 830 in runs of a second. Short calls: 5 us until the first scores, 3 for the end of a unit, 4 for the second
// kernel (20011 x 8 with 32 drafts: 28 us with K and V in L2, 31 to 32 from memory).
// Loops are kept rolled where a CTA does only a few tiles: the instructions of its first tile come from memory, and took 9000 clocks
// where a tile takes 2500.
//
// The V rows behind a sequence's end, and V rows of drafts with an infinity or NaN in them, are zeroed in shared memory before
// the product sees them; the latter are added at the end to the rows that see them, by scalar arithmetic. What infinities of the
// prefix, which every row sees, make of a channel is looked up at the end (v_classes).
#pragma once

#include "tree_attention.cuh"

namespace ha {

constexpr int kTaTile = 128;                       // tokens per tile
constexpr uint32_t kTaSlot = 2 * 128 * 128;        // K or V of a tile: 32 KB
constexpr uint32_t kTaHalf = 128 * 128;            // 64 elements of 128 rows
constexpr int kTaLoadWarp = 1;
constexpr int kTaSoftWarp0 = 2;
constexpr int kTaSoftWarps = 16;
constexpr int kTaThreads = (kTaSoftWarp0 + kTaSoftWarps) * 32;

template <bool kWide>
struct TaLayout {
    static constexpr int kRows = kWide ? 256 : 128;
    static constexpr int kCross = kWide ? 4 : 8;           // what a second unit in a CTA's range costs, in tiles (DenseCut)
    static constexpr int kRings = kWide ? 1 : 2;
    static constexpr int kSlots = kWide ? 5 : 3;           // per ring
    static constexpr uint32_t kOffQ = 0;                   // 128 rows x 128 each, K-major, 128-byte swizzle
    static constexpr uint32_t kOffRing = (kWide ? 2 : 1) * kTaSlot;
    static constexpr uint32_t kOffMl = kOffQ;              // [2][2][128] float2, once the unit's products are complete
    static constexpr int kBarFull = 0;                     // [rings][slots] the loader's arrival and the bytes of two copies
    static constexpr int kBarEmpty = kBarFull + kRings * kSlots;  // [rings][slots] commit: the products have read the slot
    static constexpr int kBarS = kBarEmpty + kRings * kSlots;     // [2] commit: S complete (and every product in front)
    static constexpr int kBarP = kBarS + 2;                // [2][2 parts] 8 warps: P is written
    static constexpr int kBarO = kBarP + 4;                // [2] commit: the unit's last product is complete
    static constexpr int kBarQ = kBarO + 2;                // 16 warps: the unit's queries are in place, the last unit's results read
    static constexpr int kBarFinal = kBarQ + 1;            // commit: every product of the CTA is complete
    static constexpr int kBars = kBarFinal + 1;
    static constexpr uint32_t kOffMax = kOffRing + kRings * kSlots * kTaSlot;  // [2 streams][2 halves][128] floats: maxima of half rows
    static constexpr uint32_t kOffBar = kOffMax + 2 * 2 * 128 * 4;
    static constexpr uint32_t kOffTmem = kOffBar + kBars * 8;     // tmem base, abort flag
    static constexpr uint32_t kOffBad = (kOffTmem + 8 + 15) / 16 * 16;  // [4] nodes with an infinity or NaN in V
    static constexpr uint32_t kAlign = 256;                       // of the array as declared
    static constexpr uint32_t kSmemBytes = kOffBad + 16 + 1024 - kAlign;  // + slack to align the base to 1024 B
    static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
};

// V as the B operand of O (128 x 128) += P (128 x 16) V (16 x 128): the 128 output columns run along the 128-byte rows
// ("MN-major"), so blocks of 64 columns are kTaHalf apart and groups of 8 tokens 1024 bytes.
__device__ __forceinline__ uint32_t ta_v_desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | ((kTaHalf >> 4) << 16); }
// O += P V over half of a tile's tokens: k-steps 0, 1, 4, 5 from the given addresses on, the hi and the lo half of P of each (as
// tc_mma_ss_k128; `accumulate` is the first product's).
__device__ __forceinline__ void ta_mma_pv(uint32_t tmem_d, uint32_t tmem_p, uint64_t desc_v, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 r, %4, %4;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "add.u32 a, %1, 8;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], %2, %3, r;\n\t"
        "add.u32 a, %1, 16;\n\tadd.u64 b, %2, 128;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "add.u32 a, %1, 24;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "add.u32 a, %1, 64;\n\tadd.u64 b, %2, 512;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "add.u32 a, %1, 72;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "add.u32 a, %1, 80;\n\tadd.u64 b, %2, 640;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "add.u32 a, %1, 88;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, r;\n\t"
        "}\n" ::"r"(tmem_d), "r"(tmem_p), "l"(desc_v), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint32_t ta_pv_idesc() { return tc_idesc(128) | (1u << 16); }

// 32 tokens from token `base` on that a row with mask `m` (bits below n only) sees, one bit each.
__device__ __forceinline__ uint32_t visible32(const uint4& m, int base, int P, int S) {
    uint32_t vis;
    const int at = base - P;  // the first token's node, negative in the prefix
    if (at <= -32) vis = 0xffffffffu;
    else {
        auto word = [&](int w) { return w < 0 ? 0xffffffffu : (w == 0 ? m.x : (w == 1 ? m.y : (w == 2 ? m.z : (w == 3 ? m.w : 0u)))); };
        const int w = at >> 5;  // (rounds down)
        vis = __funnelshift_r(word(w), word(w + 1), at & 31);
    }
    const int left = S - base;
    return left >= 32 ? vis : (left <= 0 ? 0u : vis & ((1u << left) - 1u));
}

template <bool kWide>
__global__ void __launch_bounds__(kTaThreads, 1)
tree_attention_tc_kernel(const TreeAttentionParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using L = TaLayout<kWide>;
    using Cursor = DenseCursor<kTaTile, L::kRows, L::kCross>;
    extern __shared__ __align__(L::kAlign) unsigned char ta_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ta_smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = tc_smem_u32(smem), bars = sbase + L::kOffBar;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + L::kOffTmem);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::kOffTmem + 4);
    uint32_t* s_bad = reinterpret_cast<uint32_t*>(smem + L::kOffBad);
    float2* s_ml = reinterpret_cast<float2*>(smem + L::kOffMl);
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
    if (tid == 32 * kTaLoadWarp) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    if (tid == 0) {
        auto init = [&](int first, int n, uint32_t count) {
            for (int i = first; i < first + n; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar(i)), "r"(count));
        };
        init(L::kBarFull, L::kRings * L::kSlots, 1);
        init(L::kBarEmpty, L::kRings * L::kSlots, 1);
        init(L::kBarS, 2, 1);
        init(L::kBarP, 4, 8);
        init(L::kBarO, 2, 1);
        init(L::kBarQ, 1, kTaSoftWarps);
        init(L::kBarFinal, 1, 1);
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem_u32(s_tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *s_tmem;
    dense_prefetch(p.seqs);
    pdl_wait();
    pdl_launch_dependents();

    // every lane waits for itself; the warp then agrees, so that warp-wide instructions are never executed by a part of it
    auto wait = [&](int b, uint32_t parity) {
        const bool ok = tc_wait_soon(bar(b), parity, s_abort, p.seqs.status);
        return __all_sync(0xffffffffu, ok) != 0;
    };
    // tiles of the segment that stream w takes
    auto stream_tiles = [&](const DenseSegment& s, int w) { return kWide ? s.tile1 - s.tile0 : (s.tile1 - s.tile0 + 1 - w) / 2; };

    Cursor cur(p.seqs, lane, blockIdx.x == 0 && warp == kTaLoadWarp);  // (in front of the roles: the instructions come from memory once)
    DenseSegment seg;
    bool ok = true;

    if (warp == 0) {
        // ---- the issuer: P V of a stream's tile and Q K^T of its next one back to back, the streams in turn ----------------
        const uint32_t t_0 = __shfl_sync(0xffffffffu, tmem, 0);
        uint32_t use_0 = 0, use_1 = 0, tiles_0 = 0, tiles_1 = 0, segs = 0;  // ring slots and tiles so far
        auto wait_mma = [&](int b, uint32_t parity) {
            const bool done = wait(b, parity);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return done;
        };
        while (ok && cur.next(seg)) {
            if (!(ok = wait_mma(L::kBarQ, segs & 1))) break;
            ++segs;
            const int count0 = stream_tiles(seg, 0), count1 = stream_tiles(seg, 1);  // count1 = count0 or one less
            // Turn i of a stream: P V of its tile i - 1, then Q K^T of its tile i. A ring has K of a tile, V of it, K of the next ...; the
            // streams that share one go through it alike, and the second one releases the slots. (One copy of the code for all turns:
            // the first of them wait for instructions. Two waits a turn, two barriers each: a wait costs 300 clocks even
            // where the barriers are complete, the products of a turn 1536, and four waits made this warp the bound.)
#pragma unroll 1
            for (int turn = 0; turn < 2 * (count0 + 1) && ok; ++turn) {
                const int w = turn & 1, i = turn >> 1, count = w == 0 ? count0 : count1;
                if (i > count || count == 0) continue;
                uint32_t& use = w == 0 ? use_0 : use_1;
                const uint32_t ring = kWide || w == 0 ? 0u : (uint32_t)L::kSlots, t_s = t_0 + 128u * (uint32_t)w, t_o = t_s + 256u;
                const uint32_t v_use = use, k_use = i > 0 ? use + 1 : use;
                const uint32_t v_at = ring + v_use % L::kSlots, k_at = ring + k_use % L::kSlots;
                const int full_k = L::kBarFull + (int)k_at, full_v = L::kBarFull + (int)v_at;
                const uint32_t full_k_parity = (k_use / L::kSlots) & 1, full_v_parity = (v_use / L::kSlots) & 1;
                auto wait_both = [&](int b0, uint32_t parity0, int b1, uint32_t parity1) {
                    const bool done = tc_wait_both(bar(b0), parity0, bar(b1), parity1, s_abort, p.seqs.status);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    return done;
                };
                if (i > 0) {  // O += P V: the first 32 tokens of both halves of the tile, then the rest
                    const uint32_t parity = (w == 0 ? tiles_0 : tiles_1) & 1;
                    const uint64_t vd = tc_desc(ta_v_desc_lo(sbase + L::kOffRing + v_at * kTaSlot));
                    const int p0 = L::kBarP + 2 * w, p1 = p0 + 1;
                    if (!(ok = wait_both(full_v, full_v_parity, p0, parity))) break;
                    ta_mma_pv(t_o, t_s, vd, ta_pv_idesc(), i > 1 ? 1u : 0u);
                    if (!(ok = i < count ? wait_both(full_k, full_k_parity, p1, parity) : wait_both(p1, parity, p1, parity))) break;
                    ta_mma_pv(t_o, t_s + 32, vd + 256, ta_pv_idesc(), 1u);
                    if (!kWide || w == 1) tc_commit(bar(L::kBarEmpty + (int)v_at));
                    if (w == 0) ++tiles_0;
                    else ++tiles_1;
                    ++use;
                } else if (!(ok = wait_both(full_k, full_k_parity, full_k, full_k_parity))) break;
                if (i < count) {  // S = Q K^T
                    tc_mma_ss_k128<kTaHalf>(t_s, tc_desc(tc_desc_lo(sbase + L::kOffQ + (kWide ? (uint32_t)w * kTaSlot : 0u))),
                                            tc_desc(tc_desc_lo(sbase + L::kOffRing + k_at * kTaSlot)), tc_idesc(128));
                    tc_commit(bar(L::kBarS + w));
                    if (!kWide || w == 1) tc_commit(bar(L::kBarEmpty + (int)k_at));
                    ++use;
                }
            }
            // (for a unit without a tile for a stream too: its softmax warps then never run ahead of the issuer)
            if (ok) {
                tc_commit(bar(L::kBarO));
                tc_commit(bar(L::kBarO + 1));
            }
        }
        // the tensor core has finished everything issued above (after a time-out: one more bounded wait)
        tc_commit(bar(L::kBarFinal));
        for (int spin = 0; spin < (1 << 22) && __all_sync(0xffffffffu, tc_test(bar(L::kBarFinal), 0)) == 0; ++spin) {}
    } else if (warp >= kTaSoftWarp0) {
        // ---- softmax warps -----------------------------------------------------------------------------------------------
        // A warp that gives up goes on through the units without waiting, so that the barriers among these warps are
        // reached by all of them.
        const int group = (warp - kTaSoftWarp0) >> 2, w = group >> 1, half = group & 1;  // stream, half of the columns
        const int quarter = warp & 3, r = quarter * 32 + lane, ring = kWide ? 0 : w;      // quarter of the rows = tensor-memory lanes
        const int t_all = tid - kTaSoftWarp0 * 32, t_stream = t_all & 255;
        const uint32_t t_lane = tmem + ((uint32_t)quarter << 21), t_s = t_lane + 128u * (uint32_t)w + 64u * (uint32_t)half;
        const uint32_t t_o = t_lane + 256u + 128u * (uint32_t)w + 64u * (uint32_t)half;
        float* s_max = reinterpret_cast<float*>(smem + L::kOffMax) + w * 256;
        const unsigned char* ring_mem = smem + L::kOffRing + (size_t)(ring * L::kSlots) * kTaSlot;
        uint32_t use = 0, tiles = 0, seg_o = 0;
        const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2);
        while (cur.next(seg)) {
            const int P = seg.S - seg.n, row0 = seg.group * L::kRows + (kWide ? 128 * w : 0);
            const int rows_left = seg.n * kGroup - row0;  // may be <= 0 for the second half of a wide unit
            const bool idle = quarter * 32 >= rows_left;
            const int node = (row0 + r) >> 2;
            const bool mine = r < rows_left;
            // queries: row-major pieces of 16 bytes, rows behind the last one zero
            {
                constexpr int kThreads = kWide ? 256 : 512;
                const int t = kWide ? t_stream : t_all;
                unsigned char* dst = smem + L::kOffQ + (kWide ? (size_t)w * kTaSlot : 0);
                uint4 v[128 * 16 / kThreads];
#pragma unroll
                for (int k = 0; k < 128 * 16 / kThreads; ++k) {
                    const int i = t + k * kThreads, qr = i >> 4, c = i & 15;
                    v[k] = make_uint4(0, 0, 0, 0);
                    if (qr < rows_left)
                        v[k] = __ldg(reinterpret_cast<const uint4*>(p.q + seg.b * p.q_batch + (long long)((row0 + qr) >> 2) * p.q_node +
                                                                    (seg.kvh * kGroup + (qr & 3)) * p.q_head) + c);
                }
#pragma unroll
                for (int k = 0; k < 128 * 16 / kThreads; ++k) {
                    const int i = t + k * kThreads, qr = i >> 4, c = i & 15;
                    *reinterpret_cast<uint4*>(dst + (c >> 3) * kTaHalf + tc_swizzled(qr, c & 7)) = v[k];
                }
                if (warp == kTaSoftWarp0 && lane < kMaskWords) s_bad[lane] = 0;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) tc_arrive(bar(L::kBarQ));
            }
            uint4 mask = make_uint4(0, 0, 0, 0);
            if (mine && seg.tile1 * kTaTile > P) {
                mask = dense_mask(p.seqs, seg.b, node);
                const uint4 f = first_nodes(seg.n);
                mask.x &= f.x; mask.y &= f.y; mask.z &= f.z; mask.w &= f.w;
            }
            const int count = stream_tiles(seg, w);
            float m = -INFINITY, l = 0.0f;
            for (int i = 0; i < count; ++i, ++tiles, use += 2) {
                if (ok) ok = wait(L::kBarS + w, tiles & 1);
                const int tok0 = (seg.tile0 + (kWide ? i : 2 * i + w)) * kTaTile;
                const bool masked = tok0 + kTaTile > P;
                if (masked) {
                    // the tile has drafts or lies beyond the end: V rows are looked at by the threads that share the tile
                    const uint32_t v_use = use + 1, slot = v_use % L::kSlots;
                    if (ok) ok = wait(L::kBarFull + ring * L::kSlots + (int)slot, (v_use / L::kSlots) & 1);
                    const int t = kWide ? t_all : t_stream;  // the first 128 of them: a token each
                    unsigned char* row = const_cast<unsigned char*>(ring_mem) + slot * kTaSlot + (uint32_t)t * 128u;
                    const int j = tok0 + t;
                    if (ok && t < kTaTile && j >= P) {
                        bool drop = j >= seg.S;
                        if (!drop) {
#pragma unroll
                            for (int c = 0; c < 16; ++c)  // (in any order: the swizzle permutes pieces inside a row)
                                drop |= any_nonfinite(*reinterpret_cast<const uint4*>(row + (c >> 3) * kTaHalf + (c & 7) * 16));
                            if (drop) atomicOr(&s_bad[(j - P) >> 5], 1u << ((j - P) & 31));
                        }
                        if (drop)
                            for (int c = 0; c < 16; ++c) *reinterpret_cast<uint4*>(row + (c >> 3) * kTaHalf + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    if (kWide) asm volatile("bar.sync 1, 512;" ::: "memory");
                    else asm volatile("bar.sync %0, 256;" ::"r"(10 + w) : "memory");
                }
                if (idle) {
                    __syncwarp();
                    if (ok && lane < 2) tc_arrive(bar(L::kBarP + 2 * w + lane));
                    continue;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (masked) {  // tokens that the row does not see: taken out of S itself, so that the loops below are short
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        uint32_t v[16];
                        tc_ld16_issue(t_s + 16u * (uint32_t)q, v);
                        tc_ld16_wait(v);
                        const uint32_t vis = visible32(mask, tok0 + 64 * half + 16 * q, P, seg.S);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (((vis >> k) & 1u) == 0) v[k] = 0xff800000u;  // -inf
                        tc_st16(t_s + 16u * (uint32_t)q, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                // The scores are read twice, for the maximum and for the weights: held in between they would cost 64 registers.
                uint32_t sa[16], sb[16], sc[16], sd[16];
                float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
                auto largest = [&](uint32_t (&v)[16]) {
                    tc_ld16_wait(v);
#pragma unroll
                    for (int k = 0; k < 16; k += 4) {
                        x0 = fmaxf(x0, __uint_as_float(v[k]));
                        x1 = fmaxf(x1, __uint_as_float(v[k + 1]));
                        x2 = fmaxf(x2, __uint_as_float(v[k + 2]));
                        x3 = fmaxf(x3, __uint_as_float(v[k + 3]));
                    }
                };
                tc_ld16_issue(t_s, sa);
                tc_ld16_issue(t_s + 16u, sb);
                tc_ld16_issue(t_s + 32u, sc);
                tc_ld16_issue(t_s + 48u, sd);
                largest(sa);
                largest(sb);
                tc_ld16_issue(t_s, sa);  // (the second reading)
                largest(sc);
                largest(sd);
                tc_ld16_issue(t_s + 16u, sb);
                // The maximum of the row, from both halves: the reference of its exponents, to the last bit (2^-16 of it less, and the
                // weights of a score of 2^24 pass 2^128).
                const float mine_max = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * p.scale_log2;
                s_max[half * 128 + r] = mine_max;
                asm volatile("bar.sync %0, 64;" ::"r"(2 + 4 * w + quarter) : "memory");
                const float x = fmaxf(mine_max, s_max[(half ^ 1) * 128 + r]);
                if (!ok) continue;
                const bool grow = x > m + kRescaleAt;  // (from -inf: any score at all)
                if (__any_sync(0xffffffffu, grow)) {
                    const float alpha = grow ? exp2_approx(m - x) : 1.0f;
                    m = grow ? x : m;
                    l *= alpha;
                    if (i > 0) {
                    // O is complete: S of this tile was issued behind the product that wrote it
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        uint32_t o[16];
                        tc_ld16_issue(t_o + 16 * q, o);
                        tc_ld16_wait(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                        tc_st16(t_o + 16 * q, o);
                    }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                const f32x2 nref2 = pack2(-ref, -ref);
                f32x2 la = pack2(0.0f, 0.0f), lb = pack2(0.0f, 0.0f);
                auto weigh = [&](int q, uint32_t (&v)[16]) {
                    tc_ld16_wait(v);
                    uint32_t out[16];  // one k-step of the A operand: words 0 .. 7 the hi halves, 8 .. 15 the lo halves
#pragma unroll
                    for (int pr = 0; pr < 8; ++pr) {
                        float t0, t1;
                        unpack2(fma2(pack2(__uint_as_float(v[2 * pr]), __uint_as_float(v[2 * pr + 1])), scale2, nref2), t0, t1);
                        const float e0 = exp2_approx(t0), e1 = exp2_approx(t1);
                        if (pr & 1) lb = add2(lb, pack2(e0, e1));
                        else la = add2(la, pack2(e0, e1));
                        const uint32_t hi = tc_pack_bf16(e0, e1);
                        float l0, l1;  // e - hi, exact: the multiply-add takes the bf16 halves of hi as they are
                        asm("{\n\t.reg .b16 h0, h1;\n\tmov.b32 {h0, h1}, %2;\n\t"
                            "fma.rn.f32.bf16 %0, h0, %3, %4;\n\tfma.rn.f32.bf16 %1, h1, %3, %5;\n\t}"
                            : "=f"(l0), "=f"(l1) : "r"(hi), "h"((unsigned short)0xBF80), "f"(e0), "f"(e1));
                        out[pr] = hi;
                        out[pr + 8] = tc_pack_bf16(l0, l1);
                    }
                    if (q < 2) tc_ld16_issue(t_s + 16u * (uint32_t)(q + 2), v);
                    tc_st16(t_s + 16u * (uint32_t)q, out);
                };
#pragma unroll 1  // (a short loop: at the first tile the instructions come from memory)
                for (int part = 0; part < 2; ++part) {
                    weigh(2 * part, sa);
                    weigh(2 * part + 1, sb);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tc_arrive(bar(L::kBarP + 2 * w + part));
                }
                float a0, a1, b0, b1;
                unpack2(la, a0, a1);
                unpack2(lb, b0, b1);
                l += (a0 + a1) + (b0 + b1);
            }
            // ---- the unit's result -------------------------------------------------------------------------------------
            if (ok) ok = wait(L::kBarO + w, seg_o & 1);
            ++seg_o;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            // maxima and sums of the streams that share the rows
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            asm volatile("bar.sync 1, 512;" ::: "memory");  // (all products have read the queries, whose place this is)
            s_ml[(2 * w + half) * 128 + r] = make_float2(m, l);
            asm volatile("bar.sync 1, 512;" ::: "memory");
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float M = m, sum, f0 = 1.0f, f1 = 0.0f;
            if constexpr (kWide) {
                sum = l + s_ml[(2 * w + (half ^ 1)) * 128 + r].y;
            } else {
                const float2 a = s_ml[r], b = s_ml[256 + r];
                M = fmaxf(a.x, b.x);
                const float ref = M == -INFINITY ? 0.0f : M;
                f0 = exp2_approx(a.x - ref);
                f1 = exp2_approx(b.x - ref);
                sum = (a.y + s_ml[128 + r].y) * f0 + (b.y + s_ml[384 + r].y) * f1;
            }
            if (ok && !idle) {
                const bool second = !kWide && stream_tiles(seg, 1) > 0;  // (otherwise that stream's columns hold something else)
                const size_t out_row = ((size_t)seg.b * p.seqs.T + node) * ((size_t)p.seqs.Hkv * kGroup) + seg.kvh * kGroup + (r & 3);
                const int row_in = (kWide ? 128 * w : 0) + r;  // of the unit
                const float inv = 1.0f / sum;
                const uint32_t bad = s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
                const int q0 = kWide ? 4 * half : 2 * group, q1 = q0 + (kWide ? 4 : 2);
#pragma unroll 1
                for (int q = q0; q < q1; ++q) {
                    uint32_t o0[16], o1[16];
                    tc_ld16_issue(t_lane + 256u + (kWide ? 128u * (uint32_t)w : 0u) + 16 * q, o0);
                    if (second) tc_ld16_issue(t_lane + 384u + 16 * q, o1);
                    tc_ld16_wait(o0);
                    if (second) tc_ld16_wait(o1);
                    float acc[16];
                    bool nan = false;
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        acc[k] = __uint_as_float(o0[k]) * f0;
                        if (second) acc[k] = fmaf(__uint_as_float(o1[k]), f1, acc[k]);
                        nan |= acc[k] != acc[k];
                    }
                    nan = nan && mine && sum >= 0.0f;  // (with a sum of NaN the row is NaN)
                    if (__any_sync(0xffffffffu, nan)) {
                        const uint32_t classes = v_classes(p.k_pages, p.v_pages, p.seqs.page_table + (size_t)seg.b * p.seqs.max_pages, p.seqs.num_pages, p.seqs.Hkv,
                                                           seg.kvh, seg.tile0 * kTaTile, min(P, seg.tile1 * kTaTile), q);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (nan) acc[k] = class_value(class_of(classes, k), acc[k]);
                    }
                    if (mine) {
                        if (bad != 0) {
                            const __nv_bfloat16* qr = p.q + seg.b * p.q_batch + (long long)node * p.q_node + (seg.kvh * kGroup + (r & 3)) * p.q_head;
                            for (int t = 0; t < seg.n; ++t) {
                                if (((s_bad[t >> 5] >> (t & 31)) & 1u) == 0 || !dense_bit(mask, t)) continue;
                                const int j = P + t;
                                const size_t at = (((size_t)dense_page(p.seqs, seg.b, j / kPage) * p.seqs.Hkv + seg.kvh) * kPage + j % kPage) * kHeadDim;
                                float dot = 0.0f;
                                for (int d = 0; d < kHeadDim; ++d) dot = fmaf(__bfloat162float(qr[d]), __bfloat162float(p.k_pages[at + d]), dot);
                                const float e = exp2_approx(fmaf(dot, p.scale_log2, M == -INFINITY ? 0.0f : -M));
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    const float v = __bfloat162float(p.v_pages[at + 16 * q + k]);
                                    acc[k] = fmaf(value_class(v) == 0 || dot == -INFINITY ? e : 1.0f, v, acc[k]);  // (a weight that fp32 holds as 0 is not one)
                                }
                            }
                        }
                        if (seg.whole()) {
                            uint32_t words[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) words[k] = sum == 0.0f ? 0u : tc_pack_bf16(acc[2 * k] * inv, acc[2 * k + 1] * inv);
                            uint4* dst = reinterpret_cast<uint4*>(p.out + out_row * kHeadDim + 16 * q);
                            dst[0] = make_uint4(words[0], words[1], words[2], words[3]);
                            dst[1] = make_uint4(words[4], words[5], words[6], words[7]);
                        } else {
                            // [slot][dimensions / 4][row]: a warp's rows side by side
                            float4* dst = reinterpret_cast<float4*>(p.part_acc) + ((size_t)(2 * blockIdx.x + seg.slot) * (kHeadDim / 4) + 4 * q) * L::kRows + row_in;
#pragma unroll
                            for (int k = 0; k < 4; ++k) dst[(size_t)k * L::kRows] = make_float4(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3]);
                        }
                    }
                    __syncwarp();  // (the next piece is read by all lanes together)
                }
                if (mine && (kWide ? half : group) == 0) {
                    if (!seg.whole()) p.part_ml[(size_t)(2 * blockIdx.x + seg.slot) * L::kRows + row_in] = make_float2(M, sum);
                    else if (p.lse != nullptr) p.lse[out_row] = natural_lse(M, sum);
                }
            }
            // the queries and O make room for the next unit: every product of this one is complete, and what was read of the other
            // stream's is read before its next product (the queries' barrier)
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            asm volatile("bar.sync 1, 512;" ::: "memory");
        }
    } else if (warp == kTaLoadWarp) {
        // ---- the loading warp: lane l holds the l-th page of a window of 32; one lane copies -----------------------------
        uint32_t use[2] = {0, 0};
        auto copy = [&](int ring, const CUtensorMap* map, int y) {
            const uint32_t slot = use[ring] % L::kSlots, at = (uint32_t)(ring * L::kSlots) + slot, dst = sbase + L::kOffRing + at * kTaSlot;
            if (!tc_wait(bar(L::kBarEmpty + (int)at), ((use[ring] / L::kSlots) & 1) ^ 1, s_abort, p.seqs.status)) return false;
            const uint32_t full = bar(L::kBarFull + (int)at);
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"(kTaSlot) : "memory");
            tc_tma_load(dst, map, 0, y, full);
            tc_tma_load(dst + kTaHalf, map, 64, y, full);
            ++use[ring];
            return true;
        };
        while (ok && cur.next(seg)) {
            int base = -64, page_l = 0;
            for (int t = seg.tile0; t < seg.tile1 && ok; ++t) {
                const int pi = t / (kPage / kTaTile);
                if (pi - base >= 32) {
                    base = pi;
                    page_l = (base + lane) * kPage < seg.S ? dense_page(p.seqs, seg.b, base + lane) : 0;
                }
                const int page = __shfl_sync(0xffffffffu, page_l, pi - base);
                if (lane == 0) {
                    const int y = (int)(((size_t)page * p.seqs.Hkv + seg.kvh) * kPage) + (t % (kPage / kTaTile)) * kTaTile;
                    const int ring = kWide ? 0 : (t - seg.tile0) & 1;
                    ok = copy(ring, &k_map, y) && copy(ring, &v_map, y);
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
        }
        // no copy is left in flight when the CTA ends (they have all landed unless the CTA gave up early)
        if (lane == 0)
            for (int ring = 0; ring < L::kRings; ++ring)
                for (uint32_t j = use[ring] > (uint32_t)L::kSlots ? use[ring] - L::kSlots : 0; j < use[ring]; ++j)
                    for (int spin = 0; spin < (1 << 22) && !tc_test(bar(L::kBarFull + ring * L::kSlots + (int)(j % L::kSlots)), (j / L::kSlots) & 1); ++spin) {}
        __syncwarp();
    }

    // ---- release tensor memory -----------------------------------------------------------------------------------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The partial results of the units that several CTAs share: a thread has one row and four dimensions (of kSteps pieces of 16 in
// turn) of every second one of them, a warp 32 rows side by side (as they lie in the workspace), a CTA 32 rows x 16 kSteps dimensions;
// grid (Hkv * groups of T x 8 / kSteps, B, rows / 32). kBatch partial results are loaded together. Few units: each has many
// partial results, and the CTAs are made small (12 at once, one step). Many units: two or three each, and what counts is how many
// CTAs there are and how many fit an SM (2 at once, 4 steps; 16 sequences of 2000 tokens x 4 kv-heads with 48 drafts 70 -> 46 us a
// call, 64 of 600 x 8 with 20 148 -> 92).
constexpr int kTaMergeThreads = 256, kTaMergeParts = 8;
template <int kRows, int kBatch, int kSteps>
__global__ void __launch_bounds__(kTaMergeThreads) tree_merge_tc_kernel(const TreeAttentionParams p, int ctas) {
    using Cut = DenseCut<kTaTile, kRows, TaLayout<(kRows > 128)>::kCross>;
    constexpr int kGrid = kTaMergeParts / kSteps;
    __shared__ float4 s_acc[4][32];
    __shared__ float2 s_ml[4][32];
    __shared__ uint2 s_out[32][5];  // [row][4 x 4 dimensions] bf16 (a column of padding)
    // The lengths are read before the wait: the attention kernel in front does not write them, and what did has completed.
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3, half = threadIdx.x >> 7, b = blockIdx.y;
    const int max_groups = Cut::groups(p.seqs.T), x = blockIdx.x / kGrid, kvh = x / max_groups, group = x - kvh * max_groups;
    const int row0 = blockIdx.z * 32;
    int S, n;
    dense_seq(p.seqs, b, false, S, n);
    int quota, before, span;
    Cut::count(p.seqs, ctas, lane, b, quota, before, span);
    const int rows = min(kRows, n * kGroup - group * kRows);  // of the unit
    const int tiles = Cut::tiles_of(S), r = min(row0 + lane, rows - 1);
    const int start = before + (kvh * Cut::groups(n) + group) * span;
    const int c0 = dense_div(start, quota), c1 = dense_div(start + tiles - 1, quota), first_slot = 2 * c0 + (c0 * quota != start ? 1 : 0);
    pdl_wait();
    pdl_launch_dependents();
    if (row0 >= rows || c0 == c1) return;  // (c0 == c1: one CTA had the whole unit)
#pragma unroll 1
    for (int step = 0; step < kSteps; ++step) {
        const int d4 = ((int)(blockIdx.x % kGrid) * kSteps + step) * 4 + warp;
        const float4* part = reinterpret_cast<const float4*>(p.part_acc) + (size_t)d4 * kRows + r;
        float M = -INFINITY, sum = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto rescale = [&](float top) {  // -> the reference of what is added next
            const float ref = top == -INFINITY ? 0.0f : top, f = exp2_approx(M - ref);
            M = top;
            sum *= f;
            acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
            return ref;
        };
        auto add = [&](float2 ml, float4 a, float ref) {
            const float f = exp2_approx(ml.x - ref);
            sum = fmaf(ml.y, f, sum);
            acc.x = fmaf(a.x, f, acc.x); acc.y = fmaf(a.y, f, acc.y);
            acc.z = fmaf(a.z, f, acc.z); acc.w = fmaf(a.w, f, acc.w);
        };
        for (int cb = c0 + half; cb <= c1; cb += 2 * kBatch) {  // the loads of a batch in flight together
            float2 ml[kBatch];
            float4 a[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                const int c = cb + 2 * k;
                const size_t slot = (size_t)(c == c0 ? first_slot : 2 * c);
                ml[k] = make_float2(-INFINITY, 0.0f);
                a[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (c <= c1) {
                    ml[k] = __ldcg(&p.part_ml[slot * kRows + r]);
                    a[k] = __ldcg(part + slot * (kHeadDim / 4) * kRows);
                }
            }
            float top = M;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
            const float ref = rescale(top);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) add(ml[k], a[k], ref);
        }
        if (half == 1) {
            s_acc[warp][lane] = acc;
            s_ml[warp][lane] = make_float2(M, sum);
        }
        __syncthreads();
        auto out_row = [&](int row) {
            return ((size_t)b * p.seqs.T + (group * kRows + row) / kGroup) * ((size_t)p.seqs.Hkv * kGroup) + kvh * kGroup + (row & (kGroup - 1));
        };
        if (half == 0) {
            const float2 ml = s_ml[warp][lane];
            add(ml, s_acc[warp][lane], rescale(fmaxf(M, ml.x)));
            if (!(acc.x == acc.x && acc.y == acc.y && acc.z == acc.z && acc.w == acc.w) && sum > 0.0f) {
                // (infinite partial results whose factor fp32 holds as zero, or of both signs)
                uint32_t c[4] = {0, 0, 0, 0};
                for (int k = c0; k <= c1; ++k) {
                    const float4 a = __ldcg(part + (size_t)(k == c0 ? first_slot : 2 * k) * (kHeadDim / 4) * kRows);
                    c[0] |= value_class(a.x); c[1] |= value_class(a.y); c[2] |= value_class(a.z); c[3] |= value_class(a.w);
                }
                acc = make_float4(class_value(c[0], acc.x), class_value(c[1], acc.y), class_value(c[2], acc.z), class_value(c[3], acc.w));
            }
            const float inv = 1.0f / sum;
            s_out[lane][warp] = sum == 0.0f ? make_uint2(0, 0) : make_uint2(tc_pack_bf16(acc.x * inv, acc.y * inv), tc_pack_bf16(acc.z * inv, acc.w * inv));
            if (d4 == 0 && row0 + lane < rows && p.lse != nullptr) p.lse[out_row(row0 + lane)] = natural_lse(M, sum);
        }
        __syncthreads();  // (and the other half's results have been read)
        const int row = threadIdx.x >> 2, piece = threadIdx.x & 3;  // 32 bytes of a row: four threads
        if (half == 0 && row0 + row < rows) reinterpret_cast<uint2*>(p.out + out_row(row0 + row) * kHeadDim)[d4 - warp + piece] = s_out[row][piece];
        if (kSteps > 1) __syncthreads();
    }
}

}  // namespace ha
