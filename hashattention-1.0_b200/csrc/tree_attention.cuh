// Dense attention of a few query rows per kv-head over the paged cache (a decode step's token, or a small drafted tree), and
// the merge of partial results.
//
//   o_i = sum_j e^{c q_i.k_j - lse_i} v_j,   lse_i = log sum_j e^{c q_i.k_j},   j over the tokens that row i sees
//
// in one pass over K and V with a running maximum and sum per row. A CTA takes a range of token tiles (DenseCut) of 64 tokens:
// 32 KB of K and V, copied by TMA in the 128-byte swizzle into a ring of stages. Four warps take 16 tokens of a tile each and
// keep a maximum, a sum and 16 x 128 sums of their own; they meet at the end of a unit only.
//
// The products run on the warps' matrix instructions (m16n8k16, bf16 with fp32 sums): with 4 to 16 query rows, of which a tcgen05
// tile of 128 would be mostly padding, the bytes of K and V bound the kernel and not the products (from 5 nodes on the
// tensor-core kernel of tree_attention_tc.cuh is faster). 32 sequences of 16K to 64K tokens x 8 kv-heads take 775 to 840 us, 780 of
// which are the bytes at the copy rate; in a graph 16 x 16384 x 8 take 161 to 167 us (floor 164), 131072 x 8 87 (82), 8192 x 8
// 14 (15.5 with 4 nodes) and 701 x 8 6.4, of which the start and the second kernel are the most. The weights e^{s - m} are
// handed to the second product as two bf16 (hi + lo, 16 bits of mantissa), so that their rounding does not show beside
// the one of the bf16 output. The maximum a row's weights refer to moves only when a score passes it by more than 2^8: the
// sums are fp32 and do not mind, and rescaling 16 x 128 of them at every new maximum would.
//
// Tokens that a row does not see are taken out by selection, not by a weight of zero: an infinity or NaN in the K or V of a
// token that only other branches of the tree see stays with those. An infinity in a V row that a row does see is NaN in the products
// (the lo half of its weight is negative or zero as often as not), where the average, whose weights are above zero, is
// infinite. So a channel that came out NaN is looked up at the end, in the V rows themselves (v_classes): its average is
// NaN if one of them is, if both infinities are among them, or if one meets a weight that is zero by its score of -inf. That reads V
// again, but only then.
#pragma once

#include "dense_common.cuh"

namespace ha {

struct TreeAttentionParams {
    DenseSeqs seqs;
    const __nv_bfloat16* q;  // [B][T][Hq][128], strides in elements
    long long q_batch, q_node, q_head;
    __nv_bfloat16* out;      // [B][T][Hq][128]
    float* lse;              // [B][T][Hq] or null
    float2* part_ml;         // [2 * CTAs][rows] maximum (in powers of two) and sum of each partial result
    float* part_acc;         // [2 * CTAs][rows][128]
    const __nv_bfloat16* k_pages;  // [num_pages][Hkv][256][128]: single rows only, the tiles come by tensor map
    const __nv_bfloat16* v_pages;
    float scale_log2;        // c * log2(e)
};

constexpr int kRowsTile = 64;            // tokens per tile
constexpr int kRowsWarps = 4;            // consumer warps, 16 tokens each
constexpr int kRowsThreads = (kRowsWarps + 1) * 32;
constexpr uint32_t kRowsHalf = kRowsTile * 128;      // 64 rows x 64 elements
constexpr uint32_t kRowsStage = 4 * kRowsHalf;       // K and V of a tile: 32 KB
constexpr float kRescaleAt = 8.0f;       // a row's weights may grow to 2^8 before its sums are rescaled

struct RowsLayout {
    static constexpr int kRows = 16;  // 4 query heads x up to 4 nodes
    static constexpr int kStages = 5;
    static constexpr int kAccPitch = kHeadDim + 4;
    static constexpr uint32_t kOffAcc = kStages * kRowsStage;                               // [4 warps][kRows][kAccPitch] floats
    static constexpr uint32_t kOffMl = kOffAcc + kRowsWarps * kRows * kAccPitch * 4;        // [4 warps][kRows] float2
    static constexpr uint32_t kOffBar = kOffMl + kRowsWarps * kRows * 8;
    static constexpr uint32_t kOffAbort = kOffBar + 2 * kStages * 8;
    static constexpr uint32_t kSmemBytes = kOffAbort + 16 + 1024;  // + slack to align the base to 1024 B
    static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16-byte chunk `chunk` (0..15) of row `row` of a tile of kRowsTile rows: two halves of 64 elements, 128-byte swizzle
__device__ __forceinline__ uint32_t rows_at(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * kRowsHalf + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}
__device__ __forceinline__ bool any_nonfinite(uint4 w) {
    auto bad = [](uint32_t x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; };
    return bad(w.x) || bad(w.y) || bad(w.z) || bad(w.w);
}

// What a value makes of an average with weights above zero, as bits that add up by OR: 1 it is +inf or NaN, 2 it is -inf or NaN.
__device__ __forceinline__ uint32_t value_class(float v) { return v != v ? 3u : (v == INFINITY ? 1u : (v == -INFINITY ? 2u : 0u)); }
__device__ __forceinline__ float class_value(uint32_t c, float finite) {
    return c == 0 ? finite : (c == 1 ? INFINITY : (c == 2 ? -INFINITY : __uint_as_float(0x7fffffffu)));
}
// The classes of the channels 16 q .. 16 q + 15 of V over the tokens [t0, t1) of a sequence (table: its row of the page table), by a
// whole warp, a token per lane: bit k of the lower half and bit k of the upper half. For rows whose sum of weights is a number: where K is not
// finite, their score then is -inf, and zero times an infinity is NaN.
__device__ __noinline__ uint32_t v_classes(const __nv_bfloat16* k_pages, const __nv_bfloat16* v_pages, const int32_t* table, int num_pages, int Hkv, int kvh,
                                           int t0, int t1, int q) {
    uint32_t found = 0;
#pragma unroll 4
    for (int t = t0 + (int)(threadIdx.x & 31); t < t1; t += 32) {
        int page = __ldg(table + t / kPage);
        if (page < 0 || page >= num_pages) page = 0;  // (reported by the loading warp, which took the same)
        const size_t at = (((size_t)page * Hkv + kvh) * kPage + t % kPage) * kHeadDim;
        const uint4* row = reinterpret_cast<const uint4*>(v_pages + at) + 2 * q;
        const uint4 a = __ldg(row), b = __ldg(row + 1);
        if (any_nonfinite(a) || any_nonfinite(b)) {
            const uint32_t words[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            uint32_t of_token = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t lo = value_class(bf16_lo(words[k])), hi = value_class(bf16_hi(words[k]));
                of_token |= ((lo & 1u) | (hi & 1u) << 1) << (2 * k) | ((lo >> 1) | (hi >> 1) << 1) << (2 * k + 16);
            }
            bool weightless = false;
#pragma unroll 1
            for (int c = 0; c < 16; ++c) weightless |= any_nonfinite(__ldg(reinterpret_cast<const uint4*>(k_pages + at) + c));
            found |= weightless ? of_token | __funnelshift_l(of_token, of_token, 16) : of_token;
        }
    }
    return __reduce_or_sync(0xffffffffu, found);
}
__device__ __forceinline__ uint32_t class_of(uint32_t classes, int k) { return ((classes >> k) & 1u) | ((classes >> (16 + k)) & 1u) << 1; }

// Natural log-sum-exp of a row from its maximum (in powers of two, a score as the products gave it) and sum.
__device__ __forceinline__ float natural_lse(float M, float sum) {
    return sum == 0.0f ? -INFINITY : (fmaf(M, (float)kScoreCut, M) + log2f(sum)) * 0.6931471805599453f;
}

// The output row and log-sum-exp of (sequence, node, query head): 4 dimensions per lane.
__device__ __forceinline__ void store_row(const TreeAttentionParams& p, int b, int node, int qh, int lane, float4 acc, float M, float L) {
    const size_t row = ((size_t)b * p.seqs.T + node) * ((size_t)p.seqs.Hkv * kGroup) + qh;
    const float inv = 1.0f / L;
    uint2 w = make_uint2(0, 0);  // a row that sees nothing, or scores of -inf only: zeros
    if (L != 0.0f) {
        w.x = tc_pack_bf16(acc.x * inv, acc.y * inv);
        w.y = tc_pack_bf16(acc.z * inv, acc.w * inv);
    }
    reinterpret_cast<uint2*>(p.out + row * kHeadDim)[lane] = w;
    if (lane == 0 && p.lse != nullptr) p.lse[row] = natural_lse(M, L);
}

__global__ void __launch_bounds__(kRowsThreads, 1)
tree_attention_rows_kernel(const TreeAttentionParams p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using L = RowsLayout;
    using Cursor = DenseCursor<kRowsTile, L::kRows, 0>;
    extern __shared__ unsigned char rows_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(rows_smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = tc_smem_u32(smem), bars = sbase + L::kOffBar;
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::kOffAbort);
    auto full = [&](uint32_t s) { return bars + 8u * s; };
    auto empty = [&](uint32_t s) { return bars + 8u * (L::kStages + s); };
    if (tid == 0) {
        for (uint32_t s = 0; s < (uint32_t)L::kStages; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty(s)), "r"(kRowsWarps));
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
    }
    dense_prefetch(p.seqs);
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();

    Cursor cur(p.seqs, lane, blockIdx.x == 0 && warp == 0);
    DenseSegment seg;
    uint32_t it = 0;  // tiles so far: stage it % kStages, phase it / kStages
    if (warp == kRowsWarps) {
        // ---- the loading warp: lane l holds the l-th page of a window of 32; one lane copies -------------------------
        bool ok = true;
        while (ok && cur.next(seg)) {
            int base = -64, page_l = 0;
            for (int t = seg.tile0; t < seg.tile1 && ok; ++t, ++it) {
                const int pi = t / (kPage / kRowsTile);
                if (pi - base >= 32) {
                    base = pi;
                    page_l = (base + lane) * kPage < seg.S ? dense_page(p.seqs, seg.b, base + lane) : 0;
                }
                const int page = __shfl_sync(0xffffffffu, page_l, pi - base);
                if (lane == 0) {
                    const uint32_t s = it % L::kStages, dst = sbase + s * kRowsStage;
                    ok = tc_wait(empty(s), ((it / L::kStages) & 1) ^ 1, s_abort, p.seqs.status);
                    if (ok) {
                        const int y = (int)(((size_t)page * p.seqs.Hkv + seg.kvh) * kPage) + (t % (kPage / kRowsTile)) * kRowsTile;
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(s)), "r"(kRowsStage) : "memory");
                        tc_tma_load(dst, &k_map, 0, y, full(s));
                        tc_tma_load(dst + kRowsHalf, &k_map, 64, y, full(s));
                        tc_tma_load(dst + 2 * kRowsHalf, &v_map, 0, y, full(s));
                        tc_tma_load(dst + 3 * kRowsHalf, &v_map, 64, y, full(s));
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;  // (tile `it` was not issued)
            }
        }
        // no copy is left in flight when the CTA ends (they have all landed unless the CTA gave up early)
        if (lane == 0)
            for (uint32_t j = it > (uint32_t)L::kStages ? it - L::kStages : 0; j < it; ++j)
                for (int spin = 0; spin < (1 << 22) && !tc_test(full(j % L::kStages), (j / L::kStages) & 1); ++spin) {}
        return;
    }

    // ---- consumer warps ----------------------------------------------------------------------------------------------
    // A warp that gives up (another one's time-out included) goes on through the segments without waiting, so that
    // the barriers below are reached by all four.
    bool ok = true;
    float* s_acc = reinterpret_cast<float*>(smem + L::kOffAcc);
    float2* s_ml = reinterpret_cast<float2*>(smem + L::kOffMl);
    const uint32_t k_row = (uint32_t)(warp * 16 + ((lane >> 4) << 3) + (lane & 7)), k_chunk = (uint32_t)((lane >> 3) & 1);
    const uint32_t v_row = (uint32_t)(warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7)), v_chunk = (uint32_t)(lane >> 4);
    while (cur.next(seg)) {
        const int P = seg.S - seg.n;  // (a sequence's rows are one group)
        uint32_t qa[8][4];  // the query rows as the A operand: rows lane / 4 and + 8, elements 2 (lane % 4) and + 8
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 8 + (lane >> 2);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + seg.b * p.q_batch + (r >> 2) * p.q_node +
                                                                    (seg.kvh * kGroup + (r & 3)) * p.q_head) + (lane & 3);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                qa[ks][h] = r < seg.n * kGroup ? __ldg(src + ks * 8) : 0u;
                qa[ks][h + 2] = r < seg.n * kGroup ? __ldg(src + ks * 8 + 4) : 0u;
            }
        }
        float o[16][4] = {};
        float m[2], l[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) m[h] = -INFINITY, l[h] = 0.0f;

        for (int t = seg.tile0; t < seg.tile1; ++t, ++it) {
            const uint32_t s = it % L::kStages, kb = sbase + s * kRowsStage, vb = kb + 2 * kRowsHalf;
            if (ok) ok = __all_sync(0xffffffffu, tc_wait(full(s), (it / L::kStages) & 1, s_abort, p.seqs.status)) != 0;
            if (!ok) continue;
            const int tok0 = t * kRowsTile + warp * 16;
            float c[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                uint32_t kf[4];
                ldmatrix4(kb + rows_at(k_row, 2 * ks + k_chunk), kf);
                mma16816(c[0], qa[ks], kf[0], kf[1]);
                mma16816(c[1], qa[ks], kf[2], kf[3]);
            }
            uint32_t vkeep[2] = {0xffffffffu, 0xffffffffu}, bad = 0;  // V values to use; tokens of the tree with an infinity or NaN in V
            if (tok0 + 16 > P) {
                // tokens of the tree or behind the sequence's end
                bool nonfinite = false;
                const int vt = lane >> 1;
                if (tok0 + vt >= P && tok0 + vt < seg.S) {
#pragma unroll
                    for (int ch = 0; ch < 8; ++ch)
                        nonfinite |= any_nonfinite(*reinterpret_cast<const uint4*>(smem + (vb - sbase) + rows_at(warp * 16 + vt, (lane & 1) * 8 + ch)));
                }
                const uint32_t votes = __ballot_sync(0xffffffffu, nonfinite);
#pragma unroll
                for (int i = 0; i < 16; ++i) bad |= ((votes >> (2 * i)) & 3u) != 0 ? 1u << i : 0u;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tk = nt * 8 + (lane & 3) * 2 + e;
                        if (tok0 + tk >= seg.S || ((bad >> tk) & 1u)) vkeep[nt] &= e ? 0x0000ffffu : 0xffff0000u;
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int node = 2 * h + (lane >> 4);
                    const uint4 words = node < seg.n ? dense_mask(p.seqs, seg.b, node) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int j = tok0 + nt * 8 + (lane & 3) * 2 + e;
                            if (j >= seg.S || (j >= P && !dense_bit(words, j - P))) c[nt][2 * h + e] = -INFINITY;
                        }
                }
            }
            uint32_t ph[4], pl[4];
            bool grow = false;
            float alpha[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float x = fmaxf(fmaxf(c[0][2 * h], c[0][2 * h + 1]), fmaxf(c[1][2 * h], c[1][2 * h + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2)) * p.scale_log2;
                alpha[h] = 1.0f;
                if (x > m[h] + kRescaleAt) {  // (from -inf: any score at all)
                    alpha[h] = exp2_approx(m[h] - x);
                    m[h] = x;
                    grow = true;
                }
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int dt = 0; dt < 16; ++dt) {
                    o[dt][0] *= alpha[0]; o[dt][1] *= alpha[0];
                    o[dt][2] *= alpha[1]; o[dt][3] *= alpha[1];
                }
                l[0] *= alpha[0];
                l[1] *= alpha[1];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float ref = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float p0 = exp2_approx(fmaf(c[nt][2 * h], p.scale_log2, -ref));
                    const float p1 = exp2_approx(fmaf(c[nt][2 * h + 1], p.scale_log2, -ref));
                    l[h] += p0 + p1;
                    const uint32_t hi = tc_pack_bf16(p0, p1);
                    ph[2 * nt + h] = hi;
                    pl[2 * nt + h] = tc_pack_bf16(p0 - bf16_lo(hi), p1 - bf16_hi(hi));
                    c[nt][2 * h] = p0;
                    c[nt][2 * h + 1] = p1;
                }
            }
#pragma unroll
            for (int dt = 0; dt < 16; dt += 2) {
                uint32_t vf[4];
                ldmatrix4_trans(vb + rows_at(v_row, dt + v_chunk), vf);
                vf[0] &= vkeep[0]; vf[1] &= vkeep[1]; vf[2] &= vkeep[0]; vf[3] &= vkeep[1];
                mma16816(o[dt], ph, vf[0], vf[1]);
                mma16816(o[dt + 1], ph, vf[2], vf[3]);
                mma16816(o[dt], pl, vf[0], vf[1]);
                mma16816(o[dt + 1], pl, vf[2], vf[3]);
            }
            if (bad != 0) {
                // V rows with an infinity or NaN, one by one, for the rows that see them
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        for (int w = 0; w < 4; ++w) {
                            const int tk = nt * 8 + 2 * w + e;
                            if (((bad >> tk) & 1u) == 0) continue;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float pv = __shfl_sync(0xffffffffu, c[nt][2 * h + e], (lane & ~3) | w);
                                const int node = 2 * h + (lane >> 4);
                                if (node >= seg.n || !dense_bit(dense_mask(p.seqs, seg.b, node), tok0 + tk - P)) continue;
#pragma unroll
                                for (int dt = 0; dt < 16; ++dt) {
                                    const uint32_t w2 = *reinterpret_cast<const uint32_t*>(smem + (vb - sbase) + rows_at(warp * 16 + tk, dt) + (lane & 3) * 4);
                                    o[dt][2 * h] = fmaf(pv, bf16_lo(w2), o[dt][2 * h]);
                                    o[dt][2 * h + 1] = fmaf(pv, bf16_hi(w2), o[dt][2 * h + 1]);
                                }
                            }
                            __syncwarp();
                        }
            }
            __syncwarp();
            if (lane == 0) tc_arrive(empty(s));
        }

        // ---- the four warps' results: one row at a time per warp ------------------------------------------------------
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 8 + (lane >> 2);
            float sum = l[h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            if ((lane & 3) == 0) s_ml[warp * L::kRows + r] = make_float2(m[h], sum);
            float* dst = s_acc + (size_t)(warp * L::kRows + r) * L::kAccPitch + (lane & 3) * 2;
#pragma unroll
            for (int dt = 0; dt < 16; ++dt) *reinterpret_cast<float2*>(dst + dt * 8) = make_float2(o[dt][2 * h], o[dt][2 * h + 1]);
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kRowsWarps * 32) : "memory");
        const int rows = seg.n * kGroup;
        bool looked_up = false;  // what the prefix's V rows hold beside numbers, for a row that comes out NaN
        uint32_t prefix_classes = 0;
        for (int r = warp; r < rows; r += kRowsWarps) {
            float2 ml[kRowsWarps];
            float M = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                ml[w] = s_ml[w * L::kRows + r];
                M = fmaxf(M, ml[w].x);
            }
            const float ref = M == -INFINITY ? 0.0f : M;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float f = exp2_approx(ml[w].x - ref);
                const float4 a = *reinterpret_cast<const float4*>(s_acc + (size_t)(w * L::kRows + r) * L::kAccPitch + lane * 4);
                sum = fmaf(ml[w].y, f, sum);
                acc.x = fmaf(a.x, f, acc.x); acc.y = fmaf(a.y, f, acc.y);
                acc.z = fmaf(a.z, f, acc.z); acc.w = fmaf(a.w, f, acc.w);
            }
            if (__any_sync(0xffffffffu, !(acc.x == acc.x && acc.y == acc.y && acc.z == acc.z && acc.w == acc.w)) && sum >= 0.0f) {
                // (with a sum of NaN the row is NaN)
                auto classes = [&](int t0, int t1) {  // of the lane's four channels
                    uint32_t mine = 0;
                    for (int q = 0; q < 8; ++q) {
                        const uint32_t c = v_classes(p.k_pages, p.v_pages, p.seqs.page_table + (size_t)seg.b * p.seqs.max_pages, p.seqs.num_pages, p.seqs.Hkv, seg.kvh, t0, t1, q);
                        if (q == lane >> 2) mine = c >> (4 * (lane & 3));
                    }
                    return mine;
                };
                const int t0 = seg.tile0 * kRowsTile, t1 = min(seg.S, seg.tile1 * kRowsTile);
                if (!looked_up) prefix_classes = classes(t0, min(P, t1));
                looked_up = true;
                uint32_t c = prefix_classes;
                const uint4 words = dense_mask(p.seqs, seg.b, r >> 2);
                for (int t = max(P, t0); t < t1; ++t)
                    if (dense_bit(words, t - P)) c |= classes(t, t + 1);
                acc = make_float4(class_value(class_of(c, 0), acc.x), class_value(class_of(c, 1), acc.y),
                                  class_value(class_of(c, 2), acc.z), class_value(class_of(c, 3), acc.w));
            }
            if (seg.whole()) {
                if (ok) store_row(p, seg.b, r >> 2, seg.kvh * kGroup + (r & 3), lane, acc, M, sum);
            } else {
                const size_t at = (size_t)(2 * blockIdx.x + seg.slot) * L::kRows + r;
                if (lane == 0) p.part_ml[at] = make_float2(M, sum);
                reinterpret_cast<float4*>(p.part_acc + at * kHeadDim)[lane] = acc;
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kRowsWarps * 32) : "memory");
    }
}

// The partial results of the units that several CTAs share, a warp per query row; grid (Hkv, B, rows / 4).
constexpr int kTreeMergeWarps = 4;
__global__ void __launch_bounds__(kTreeMergeWarps * 32) tree_merge_rows_kernel(const TreeAttentionParams p, int ctas) {
    constexpr int kRows = RowsLayout::kRows;
    using Cut = DenseCut<kRowsTile, kRows, 0>;
    // The lengths are read before the wait: the attention kernel in front does not write them, and what did has completed.
    const int lane = threadIdx.x & 31, r = blockIdx.z * kTreeMergeWarps + (threadIdx.x >> 5), b = blockIdx.y, kvh = blockIdx.x;
    int S, n;
    dense_seq(p.seqs, b, false, S, n);
    int quota, before, span;
    Cut::count(p.seqs, ctas, lane, b, quota, before, span);
    const int tiles = Cut::tiles_of(S);
    const int start = before + kvh * span;
    const int c0 = dense_div(start, quota), c1 = dense_div(start + tiles - 1, quota);
    auto at = [&](int c) { return (size_t)(2 * c + (c == c0 && c0 * quota != start ? 1 : 0)) * kRows + r; };
    pdl_wait();
    pdl_launch_dependents();
    if (r >= n * kGroup || c0 == c1) return;  // (one CTA had the whole unit)

    // 16 partial results at a time, all of their loads in flight together, in an order that is always the same
    constexpr int kBatch = 16;
    float M = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int cb = c0; cb <= c1; cb += kBatch) {
        const bool mine = lane < kBatch && cb + lane <= c1;
        const float2 ml = mine ? __ldcg(&p.part_ml[at(cb + lane)]) : make_float2(-INFINITY, 0.0f);
        float4 a[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            a[i] = cb + i <= c1 ? __ldcg(reinterpret_cast<const float4*>(p.part_acc + at(cb + i) * kHeadDim) + lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float top = fmaxf(M, ml.x);
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
        const float ref = top == -INFINITY ? 0.0f : top, f0 = exp2_approx(M - ref);
        const float f = mine ? exp2_approx(ml.x - ref) : 0.0f;
        float part = ml.y * f;
#pragma unroll
        for (int i = 16; i > 0; i >>= 1) part += __shfl_xor_sync(0xffffffffu, part, i);
        M = top;
        sum = fmaf(sum, f0, part);
        acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const float w = __shfl_sync(0xffffffffu, f, i);
            acc.x = fmaf(a[i].x, w, acc.x); acc.y = fmaf(a[i].y, w, acc.y);
            acc.z = fmaf(a[i].z, w, acc.z); acc.w = fmaf(a[i].w, w, acc.w);
        }
    }
    if (__any_sync(0xffffffffu, !(acc.x == acc.x && acc.y == acc.y && acc.z == acc.z && acc.w == acc.w)) && sum > 0.0f) {
        // (infinite partial results whose factor fp32 holds as zero, or of both signs)
        uint32_t c[4] = {0, 0, 0, 0};
        for (int k = c0; k <= c1; ++k) {
            const float4 a = __ldcg(reinterpret_cast<const float4*>(p.part_acc + at(k) * kHeadDim) + lane);
            c[0] |= value_class(a.x); c[1] |= value_class(a.y); c[2] |= value_class(a.z); c[3] |= value_class(a.w);
        }
        acc = make_float4(class_value(c[0], acc.x), class_value(c[1], acc.y), class_value(c[2], acc.z), class_value(c[3], acc.w));
    }
    store_row(p, b, r >> 2, kvh * kGroup + (r & 3), lane, acc, M, sum);
}

}  // namespace ha
