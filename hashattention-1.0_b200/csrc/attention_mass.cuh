// The attention weight each cached token receives:
//
//   mass[j] += sum_{i in rows, g} e^{c q_ig.k_j - lse_ig}   over the rows that see token j
//
// per (sequence, kv-head), with the log-sum-exps the attention left: one more pass over K, no V. The transposed product
// S = K Q^T runs on the 5th-generation tensor cores (tcgen05): the 128 tokens of a tile are the lanes of tensor memory, the counted
// query rows its columns, so a thread adds up its token's weights without another one's help. The query rows (4 per counted node,
// up to 512) stay in shared memory as the B operand, N = 16 to 128 columns at a time, so few rows cost few products.
//
// Roles of the warps: 0 issues the products, 1 loads K tiles by TMA (two boxes of 64 elements x 128 tokens, 128-byte swizzle) into a
// ring of 32 KB slots, 4 - 19 turn scores into weights, in two groups of eight that take every second tile (two buffers of 128 columns
// of tensor memory each, so that the next products run under the exponentials; with one of 256 a group stood still for 1700 of 7500
// clocks): four quarters of the lanes times two halves of the columns. The halves of a token's sum meet
// in shared memory; a token's sum is formed in a fixed order and added by one thread in one piece (a reduction in L2: a load of the
// old value cost 1300 clocks a tile).
//
// With few rows the bytes of K bound it (one row per head, 4 x 32768 tokens x 8 kv-heads: 50.7 us, floor 42); with 256 and more
// the exponentials do: 16 a clock on an SM, 2048 clocks for the 128 x 256 scores whose K tile takes 1400 to arrive at the copy
// rate and whose products take 1024. A tile takes 3550 (64 nodes, 30011 + 50021 tokens x 8: 78.5 us): the units that take
// exponentials are busy 54 % of the time, the rest being a group's waits at each pass of 128 columns.
//
// Precision: c * s and lse are numbers of magnitude 10 to 50 whose difference is exponentiated. The multiply-add rounds only that
// difference. What the rounding of c to fp32 would add, and what the products leave of a score (kScoreCut), is taken out of lse in
// 64 bits (where weights matter, c s = lse); what is left is the rounding of lse * log2(e) to fp32, half an ulp of 16 to 64: up to
// 1.3e-6 of a row's weights, to either side. (A factor per row that takes that out as well was read from shared memory for every
// score: 4096 clocks for two tiles of 256 rows, as long as their exponentials take, on top of the same for lse.)
#pragma once

#include "tree_attention.cuh"

namespace ha {

struct AttentionMassParams {
    DenseSeqs seqs;
    const __nv_bfloat16* q;  // as in TreeAttentionParams
    long long q_batch, q_node, q_head;
    const float* lse;        // [B][T][Hq]
    const uint32_t* rows;    // [B][4] the nodes whose weights count, or null: all of the tree
    float* mass;             // [B][Hkv][max_pages * 256]
    float scale_log2;        // c * log2(e), rounded
    double lse_scale;        // log2(e) * scale_log2 / (c * log2(e)) * (1 - kScoreCut)
    int q_rows;              // rows of the query operand: 4 T, to a multiple of 16
    int slots;               // of the ring
};

constexpr int kMassTile = 128;
constexpr int kMassMaxRows = kMaxNodes * kGroup;
constexpr int kMassCols = 128;                  // columns of a buffer of tensor memory
constexpr uint32_t kMassSlot = 2 * 128 * 128;   // K of a tile: 32 KB
constexpr uint32_t kMassHalf = 128 * 128;
constexpr int kMassMaxSlots = 6;
constexpr int kMassWarp0 = 4;
constexpr int kMassWarps = 16;
constexpr int kMassThreads = (kMassWarp0 + kMassWarps) * 32;
// Shared memory: the fixed part, then the ring, then the queries (two halves of 64 elements, 128 bytes a row).
constexpr int kMassBarFull = 0;                               // [slots] the loader's arrival and the bytes of two copies
constexpr int kMassBarEmpty = kMassBarFull + kMassMaxSlots;   // [slots] commit: the products have read the tile
constexpr int kMassBarS = kMassBarEmpty + kMassMaxSlots;      // [2 groups][2 buffers] commit: scores complete
constexpr int kMassBarRead = kMassBarS + 4;                   // [2 groups][2 buffers] 8 warps: scores read
constexpr int kMassBarQ = kMassBarRead + 4;                   // 16 warps: the unit's queries are in place
constexpr int kMassBarFinal = kMassBarQ + 1;
constexpr int kMassBars = kMassBarFinal + 1;
constexpr uint32_t kMassOffLse = 0;                                    // [512] -lse in powers of two, rounded; -inf where there is no row or it is NaN
constexpr uint32_t kMassOffNode = kMassOffLse + kMassMaxRows * 4;      // [128] the counted nodes
constexpr uint32_t kMassOffVis = kMassOffNode + kMaxNodes * 4;         // [128 drafts] counted nodes that see the draft, one bit each
constexpr uint32_t kMassOffPart = kMassOffVis + kMaxNodes * 16;        // [2 groups][2 tiles][128] sums of the second half of the columns;
                                                                       // in front of a unit's tiles: [128] mask words of the counted nodes
constexpr uint32_t kMassOffBar = kMassOffPart + 2 * 2 * 128 * 4;
constexpr uint32_t kMassOffTmem = kMassOffBar + kMassBars * 8;
constexpr uint32_t kMassOffNan = (kMassOffTmem + 8 + 15) / 16 * 16;    // counted nodes with a row whose log-sum-exp is NaN, one bit each
constexpr uint32_t kMassOffRing = (kMassOffNan + 16 + 1023) / 1024 * 1024;
__host__ __device__ constexpr size_t mass_smem_bytes(int slots, int q_rows) { return kMassOffRing + (size_t)slots * kMassSlot + (size_t)q_rows * 256 + 1024; }
inline int mass_slots(int q_rows) {
    int slots = kMassMaxSlots;
    while (mass_smem_bytes(slots, q_rows) > 227 * 1024) --slots;
    return slots;
}

__device__ __forceinline__ uint4 counted_nodes(const uint32_t* rows, int b, int n) {
    uint4 set = first_nodes(n);
    if (rows != nullptr) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(rows) + b);
        set.x &= r.x; set.y &= r.y; set.z &= r.z; set.w &= r.w;
    }
    return set;
}

// A row whose log-sum-exp is NaN makes NaN of the tokens [j0, j1) that it sees. (In the exponent, where tokens that a row does not
// see are taken out by -inf, it would make NaN of those too.) By the threads that form weights; out of line, so that the kernel's end, whose
// instructions come from memory, stays short.
__device__ __noinline__ void mass_of_nan_rows(uint32_t* s_nan, const uint4* s_vis, bool nan_row, int t_all, float* mass, int j0, int j1, int P) {
    if (t_all < kMaskWords) s_nan[t_all] = 0;
    asm volatile("bar.sync 1, 512;" ::: "memory");
    if (nan_row) atomicOr(&s_nan[t_all >> 7], 1u << ((t_all >> 2) & 31));
    asm volatile("bar.sync 1, 512;" ::: "memory");
    const uint4 nan = *reinterpret_cast<const uint4*>(s_nan);
    for (int j = j0 + t_all; j < j1; j += kMassWarps * 32) {
        const uint4 v = j < P ? nan : s_vis[j - P];
        if (((v.x & nan.x) | (v.y & nan.y) | (v.z & nan.z) | (v.w & nan.w)) != 0) atomicAdd(mass + j, __uint_as_float(0x7fffffffu));
    }
    asm volatile("bar.sync 1, 512;" ::: "memory");
}

__global__ void __launch_bounds__(kMassThreads, 1) attention_mass_kernel(const AttentionMassParams p, const __grid_constant__ CUtensorMap k_map) {
    using Cursor = DenseCursor<kMassTile, kMassMaxRows, 0>;
    extern __shared__ unsigned char mass_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mass_smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = tc_smem_u32(smem), bars = sbase + kMassOffBar;
    const uint32_t off_q = kMassOffRing + (uint32_t)p.slots * kMassSlot, q_half = (uint32_t)p.q_rows * 128u;
    uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + kMassOffTmem);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + kMassOffTmem + 4);
    float* s_lse = reinterpret_cast<float*>(smem + kMassOffLse);
    int* s_node = reinterpret_cast<int*>(smem + kMassOffNode);
    uint4* s_mask = reinterpret_cast<uint4*>(smem + kMassOffPart);
    uint4* s_vis = reinterpret_cast<uint4*>(smem + kMassOffVis);
    float* s_part = reinterpret_cast<float*>(smem + kMassOffPart);
    uint32_t* s_nan = reinterpret_cast<uint32_t*>(smem + kMassOffNan);
    auto bar = [&](int i) { return bars + 8u * (uint32_t)i; };
    if (tid == 0) {
        auto init = [&](int first, int n, uint32_t count) {
            for (int i = first; i < first + n; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar(i)), "r"(count));
        };
        init(kMassBarFull, kMassMaxSlots, 1);
        init(kMassBarEmpty, kMassMaxSlots, 1);
        init(kMassBarS, 4, 1);
        init(kMassBarRead, 4, kMassWarps / 2);
        init(kMassBarQ, 1, kMassWarps);
        init(kMassBarFinal, 1, 1);
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
    if (tid == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    pdl_wait();
    pdl_launch_dependents();

    // every lane waits for itself; the warp then agrees, so that warp-wide instructions are never executed by a part of it
    auto wait = [&](int b, uint32_t parity) {
        const bool ok = tc_wait_soon(bar(b), parity, s_abort, p.seqs.status);
        return __all_sync(0xffffffffu, ok) != 0;
    };
    Cursor cur(p.seqs, lane, blockIdx.x == 0 && warp == 1);
    DenseSegment seg = {};
    bool ok = true;
    // Units of which no node counts are left out, by all roles alike. Otherwise: rows, and passes of up to 128 columns.
    auto rows_of_unit = [&](uint4& set) {
        set = counted_nodes(p.rows, seg.b, seg.n);
        return (__popc(set.x) + __popc(set.y) + __popc(set.z) + __popc(set.w)) * kGroup;
    };
    const uint32_t slots = (uint32_t)p.slots;

    if (warp == 0) {
        // ---- the issuer: pass by pass for two tiles, one of each group, in turn ----------------------------------------------
        uint32_t use = 0, items[2] = {0, 0}, segs = 0;  // tiles of the ring; passes of a group
        auto wait_mma = [&](int b, uint32_t parity) {
            const bool done = wait(b, parity);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return done;
        };
        while (ok && cur.next(seg)) {
            uint4 set;
            const int rows = rows_of_unit(set);
            if (rows == 0) continue;
            const int passes = (rows + kMassCols - 1) / kMassCols, count = seg.tile1 - seg.tile0;
            if (!(ok = wait_mma(kMassBarQ, segs & 1))) break;
            ++segs;
            for (int i = 0; i < count && ok; i += 2) {
                for (int pass = 0; pass < passes && ok; ++pass) {
                    const uint32_t cols = (uint32_t)min(kMassCols, (rows - pass * kMassCols + 15) & ~15);
                    for (int g = 0; g < 2 && i + g < count && ok; ++g) {
                        const uint32_t at = use + (uint32_t)g, slot = at % slots, item = items[g]++, buffer = 2u * (uint32_t)g + (item & 1);
                        // (the tile is there; the scores that the buffer held have been read)
                        const int full = kMassBarFull + (int)slot, read = kMassBarRead + (int)buffer;
                        ok = tc_wait_both(bar(full), (at / slots) & 1, bar(read), ((item >> 1) & 1) ^ 1, s_abort, p.seqs.status);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t k_lo = tc_desc_lo(sbase + kMassOffRing + slot * kMassSlot);
                        const uint32_t q_lo = tc_desc_lo(sbase + off_q + (uint32_t)(pass * kMassCols) * 128u);
#pragma unroll
                        for (uint32_t ks = 0; ks < 8; ++ks)
                            tc_mma_ss(tmem + buffer * kMassCols, tc_desc(k_lo + tc_koff(ks, kMassHalf)), tc_desc(q_lo + tc_koff(ks, q_half)), tc_idesc(cols),
                                      ks == 0 ? 0u : 1u);
                        tc_commit(bar(kMassBarS + (int)buffer));
                        if (pass == passes - 1) tc_commit(bar(kMassBarEmpty + (int)slot));
                    }
                }
                use += (uint32_t)min(2, count - i);
            }
        }
        tc_commit(bar(kMassBarFinal));
        for (int spin = 0; spin < (1 << 22) && __all_sync(0xffffffffu, tc_test(bar(kMassBarFinal), 0)) == 0; ++spin) {}
    } else if (warp == 1) {
        // ---- the loading warp: lane l holds the l-th page of a window of 32; one lane copies -----------------------------
        uint32_t use = 0;
        bool first = true;
        while (ok && cur.next(seg)) {
            uint4 set;
            const int rows = rows_of_unit(set);
            if (rows == 0) continue;
            int base = -64, page_l = 0;
            for (int t = seg.tile0; t < seg.tile1 && ok; ++t) {
                // Many query rows (32 KB and more) come in behind the first two tiles only, not behind a full ring's.
                if (first && rows >= 128 && t == seg.tile0 + 2 && !(ok = wait(kMassBarQ, 0))) break;
                const int pi = t / (kPage / kMassTile);
                if (pi - base >= 32) {
                    base = pi;
                    page_l = (base + lane) * kPage < seg.S ? dense_page(p.seqs, seg.b, base + lane) : 0;
                }
                const int page = __shfl_sync(0xffffffffu, page_l, pi - base);
                if (lane == 0) {
                    const uint32_t slot = use % slots, dst = sbase + kMassOffRing + slot * kMassSlot, full = bar(kMassBarFull + (int)slot);
                    const int y = (int)(((size_t)page * p.seqs.Hkv + seg.kvh) * kPage) + (t % (kPage / kMassTile)) * kMassTile;
                    ok = tc_wait(bar(kMassBarEmpty + (int)slot), ((use / slots) & 1) ^ 1, s_abort, p.seqs.status);
                    if (ok) {
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full), "r"(kMassSlot) : "memory");
                        tc_tma_load(dst, &k_map, 0, y, full);
                        tc_tma_load(dst + kMassHalf, &k_map, 64, y, full);
                        ++use;
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            first = false;
        }
        // no copy is left in flight when the CTA ends (they have all landed unless the CTA gave up early)
        if (lane == 0)
            for (uint32_t j = use > slots ? use - slots : 0; j < use; ++j)
                for (int spin = 0; spin < (1 << 22) && !tc_test(bar(kMassBarFull + (int)(j % slots)), (j / slots) & 1); ++spin) {}
        __syncwarp();
    } else if (warp >= kMassWarp0) {
        // ---- weights -----------------------------------------------------------------------------------------------------
        // A warp that gives up goes on through the units without waiting, so that the barriers among these warps are
        // reached by all of them.
        const int g = (warp - kMassWarp0) >> 3, part = ((warp - kMassWarp0) >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane;
        const int t_all = tid - kMassWarp0 * 32;
        const uint32_t t_g = tmem + ((uint32_t)quarter << 21) + (uint32_t)(2 * g * kMassCols);
        const f32x2 scale2 = pack2(p.scale_log2, p.scale_log2);
        uint32_t items = 0;
        while (cur.next(seg)) {
            uint4 set;
            const int rows = rows_of_unit(set);
            if (rows == 0) continue;
            const int passes = (rows + kMassCols - 1) / kMassCols, count = seg.tile1 - seg.tile0, padded = (rows + 15) & ~15, P = seg.S - seg.n;
            if (t_all < kMaxNodes && dense_bit(set, t_all)) {  // the counted nodes in order: a node's place is the number of those below it
                const uint4 below = first_nodes(t_all);
                s_node[__popc(set.x & below.x) + __popc(set.y & below.y) + __popc(set.z & below.z) + __popc(set.w & below.w)] = t_all;
            }
            asm volatile("bar.sync 1, 512;" ::: "memory");
            // The counted query rows. (Every product of the unit before has been read: the barrier at the end of the loop.) A row
            // that fills up the last 16 is a copy of the last one that counts for nothing.
#pragma unroll 4
            for (int i = t_all; i < padded * 16; i += kMassWarps * 32) {
                const int qr = i >> 4, c = i & 15, row = min(qr, rows - 1);
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.q + seg.b * p.q_batch + s_node[row >> 2] * p.q_node +
                                                                     (seg.kvh * kGroup + (row & 3)) * p.q_head) + c);
                *reinterpret_cast<uint4*>(smem + off_q + (c >> 3) * q_half + tc_swizzled(qr, c & 7)) = v;
            }
            bool nan_row = false;
            if (t_all < padded) {
                float l = -INFINITY;  // (so too for a row that sees nothing)
                if (t_all < rows) {
                    const float lse = __ldg(p.lse + ((size_t)seg.b * p.seqs.T + s_node[t_all >> 2]) * ((size_t)p.seqs.Hkv * kGroup) + seg.kvh * kGroup + (t_all & 3));
                    nan_row = lse != lse;
                    if (lse != -INFINITY && !nan_row) l = -(float)((double)lse * p.lse_scale);
                }
                s_lse[t_all] = l;
            }
            if (seg.tile1 * kMassTile > P) {  // which counted nodes see draft t_all
                const int nodes = rows / kGroup;
                if (t_all < nodes) s_mask[t_all] = dense_mask(p.seqs, seg.b, s_node[t_all]);
                asm volatile("bar.sync 1, 512;" ::: "memory");
                if (t_all < seg.n) {
                    const uint32_t* column = reinterpret_cast<const uint32_t*>(s_mask) + (t_all >> 5);
                    uint32_t words[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        words[w] = 0;
#pragma unroll 8
                        for (int k = 32 * w; k < min(nodes, 32 * w + 32); ++k) words[w] |= ((column[4 * k] >> (t_all & 31)) & 1u) << (k & 31);
                    }
                    s_vis[t_all] = make_uint4(words[0], words[1], words[2], words[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 1, 512;" ::: "memory");  // (what a thread reads below others have written)
            if (lane == 0) tc_arrive(bar(kMassBarQ));

            float* mass = p.mass + ((size_t)seg.b * p.seqs.Hkv + seg.kvh) * ((size_t)p.seqs.max_pages * kPage);
            for (int i = g; i < count; i += 2) {
                const int j = (seg.tile0 + i) * kMassTile + r;
                const bool masked = (seg.tile0 + i + 1) * kMassTile > P;
                uint4 vis = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
                if (masked && j >= P) vis = j < seg.S ? s_vis[j - P] : make_uint4(0, 0, 0, 0);
                f32x2 s0 = pack2(0.0f, 0.0f), s1 = s0;
                for (int pass = 0; pass < passes; ++pass, ++items) {
                    const int buffer = 2 * g + (int)(items & 1);
                    const uint32_t t_s = t_g + (items & 1) * kMassCols;
                    if (ok) ok = wait(kMassBarS + buffer, (items >> 1) & 1);
                    if (!ok) continue;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int cols = min(kMassCols, padded - pass * kMassCols), half = ((cols >> 4) + 1) >> 1;  // pieces of 16 columns of part 0
                    const int piece0 = part == 0 ? 0 : half, piece1 = part == 0 ? half : cols >> 4;
                    if (masked) {  // what does not count becomes -inf in tensor memory, so that the loop below has nothing to ask
#pragma unroll 1
                        for (int q = piece0; q < piece1; ++q) {
                            uint32_t v[16];
                            tc_ld16_issue(t_s + 16u * (uint32_t)q, v);
                            tc_ld16_wait(v);
                            const int node = (pass * kMassCols + 16 * q) >> 2;  // four nodes in 16 columns
                            const uint32_t word = node < 64 ? (node < 32 ? vis.x : vis.y) : (node < 96 ? vis.z : vis.w);
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                if (((word >> ((node + (k >> 2)) & 31)) & 1u) == 0) v[k] = 0xff800000u;
                            tc_st16(t_s + 16u * (uint32_t)q, v);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    uint32_t a[2][16];
                    if (piece0 < piece1) tc_ld16_issue(t_s + 16u * (uint32_t)piece0, a[0]);
                    auto piece = [&](int q, uint32_t (&v)[16], uint32_t (&ahead)[16]) {
                        tc_ld16_wait(v);
                        if (q + 1 < piece1) tc_ld16_issue(t_s + 16u * (uint32_t)(q + 1), ahead);
                        const int col = pass * kMassCols + 16 * q;
                        const float4* ls = reinterpret_cast<const float4*>(s_lse + col);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const float4 l4 = ls[n];
                            float x0, x1, x2, x3;
                            unpack2(fma2(pack2(__uint_as_float(v[4 * n]), __uint_as_float(v[4 * n + 1])), scale2, pack2(l4.x, l4.y)), x0, x1);
                            unpack2(fma2(pack2(__uint_as_float(v[4 * n + 2]), __uint_as_float(v[4 * n + 3])), scale2, pack2(l4.z, l4.w)), x2, x3);
                            s0 = add2(s0, pack2(exp2_approx(x0), exp2_approx(x1)));
                            s1 = add2(s1, pack2(exp2_approx(x2), exp2_approx(x3)));
                        }
                    };
                    for (int q = piece0; q < piece1; q += 2) {
                        piece(q, a[0], a[1]);
                        if (q + 1 < piece1) piece(q + 1, a[1], a[0]);
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tc_arrive(bar(kMassBarRead + buffer));
                }
                float a0, a1, b0, b1;
                unpack2(s0, a0, a1);
                unpack2(s1, b0, b1);
                const float sum = (a0 + a1) + (b0 + b1);
                float* others = s_part + (2 * g + ((i >> 1) & 1)) * 128;  // (written again two tiles on, behind a barrier of the one between)
                if (part == 1) others[r] = sum;
                asm volatile("bar.sync %0, 64;" ::"r"(2 + 4 * g + quarter) : "memory");
                if (part == 0 && ok && j < seg.S) atomicAdd(mass + j, sum + others[r]);  // (no other thread of the call adds a number to it)
            }
            // (the barrier at the end of a unit tells whether it has a row that is NaN)
            uint32_t any_nan;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 512, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                         : "=r"(any_nan) : "r"(nan_row ? 1u : 0u) : "memory");
            if (any_nan != 0) mass_of_nan_rows(s_nan, s_vis, nan_row, t_all, mass, seg.tile0 * kMassTile, min(seg.S, seg.tile1 * kMassTile), P);
        }
    }

    // ---- release tensor memory -----------------------------------------------------------------------------------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

}  // namespace ha
