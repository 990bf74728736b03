// The attention weight each cached token receives:
//
//   mass[j] += sum_{i in rows, g} e^{c q_ig.k_j - lse_ig}   over the rows that see token j
//
// per (sequence, kv-head), with the log-sum-exps the attention left: one more pass over K, no V. The transposed product
// K Q^T puts the tokens on the rows of the matrix instruction, so a token's sum stays inside a quad of lanes. No atomics: a
// token's sum is formed by one warp in a fixed order.
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
    float scale_log2;
};

constexpr int kMassTile = 64;
constexpr int kMassMaxRows = kMaxNodes * kGroup;
constexpr uint32_t kMassStage = 2 * kRowsHalf;  // K of a tile: 16 KB
constexpr int kMassStages = 4;
constexpr uint32_t kMassOffQ = kMassStages * kMassStage;               // [2 halves][512 rows][64] bf16, 128-byte swizzle
constexpr uint32_t kMassQHalf = kMassMaxRows * 128;
constexpr uint32_t kMassOffLse = kMassOffQ + 2 * kMassQHalf;           // [512] lse * log2(e), +inf where there is no row
constexpr uint32_t kMassOffMask = kMassOffLse + kMassMaxRows * 4;      // [128] mask words of the counted nodes
constexpr uint32_t kMassOffBar = kMassOffMask + kMaxNodes * 16;
constexpr uint32_t kMassOffAbort = kMassOffBar + 2 * kMassStages * 8;
constexpr uint32_t kMassSmemBytes = kMassOffAbort + 16 + 1024;
static_assert(kMassSmemBytes <= 227 * 1024, "shared memory of one CTA");

// The i-th set bit of a node set restricted to the nodes below n (-1: there are fewer).
__device__ __forceinline__ int nth_node(const uint4& set, int i) {
    const uint32_t w[4] = {set.x, set.y, set.z, set.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int c = __popc(w[k]);
        if (i < c) return 32 * k + (int)__fns(w[k], 0, i + 1);
        i -= c;
    }
    return -1;
}
__device__ __forceinline__ uint4 first_nodes(int n) {
    auto word = [&](int k) { return n >= 32 * k + 32 ? 0xffffffffu : (n <= 32 * k ? 0u : (1u << (n - 32 * k)) - 1u); };
    return make_uint4(word(0), word(1), word(2), word(3));
}
__device__ __forceinline__ uint4 counted_nodes(const uint32_t* rows, int b, int n) {
    uint4 set = first_nodes(n);
    if (rows != nullptr) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(rows) + b);
        set.x &= r.x; set.y &= r.y; set.z &= r.z; set.w &= r.w;
    }
    return set;
}

__global__ void __launch_bounds__(kRowsThreads, 1) attention_mass_rows_kernel(const AttentionMassParams p, const __grid_constant__ CUtensorMap k_map) {
    using Cursor = DenseCursor<kMassTile, kMassMaxRows>;
    extern __shared__ unsigned char mass_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(mass_smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t sbase = tc_smem_u32(smem), bars = sbase + kMassOffBar;
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + kMassOffAbort);
    float* s_lse = reinterpret_cast<float*>(smem + kMassOffLse);
    uint4* s_mask = reinterpret_cast<uint4*>(smem + kMassOffMask);
    auto full = [&](uint32_t s) { return bars + 8u * s; };
    auto empty = [&](uint32_t s) { return bars + 8u * (kMassStages + s); };
    if (tid == 0) {
        for (uint32_t s = 0; s < (uint32_t)kMassStages; ++s) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty(s)), "r"(kRowsWarps));
        }
        *s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();

    Cursor cur(p.seqs, lane, blockIdx.x == 0 && warp == 0);
    DenseSegment seg;
    uint32_t it = 0;
    if (warp == kRowsWarps) {
        bool ok = true;
        while (ok && cur.next(seg)) {
            int base = -64, page_l = 0;
            for (int t = seg.tile0; t < seg.tile1 && ok; ++t, ++it) {
                const int pi = t / (kPage / kMassTile);
                if (pi - base >= 32) {
                    base = pi;
                    page_l = (base + lane) * kPage < seg.S ? dense_page(p.seqs, seg.b, base + lane) : 0;
                }
                const int page = __shfl_sync(0xffffffffu, page_l, pi - base);
                if (lane == 0) {
                    const uint32_t s = it % kMassStages, dst = sbase + s * kMassStage;
                    ok = tc_wait(empty(s), ((it / kMassStages) & 1) ^ 1, s_abort, p.seqs.status);
                    if (ok) {
                        const int y = (int)(((size_t)page * p.seqs.Hkv + seg.kvh) * kPage) + (t % (kPage / kMassTile)) * kMassTile;
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(s)), "r"(kMassStage) : "memory");
                        tc_tma_load(dst, &k_map, 0, y, full(s));
                        tc_tma_load(dst + kRowsHalf, &k_map, 64, y, full(s));
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
                if (!ok) break;
            }
        }
        if (lane == 0)
            for (uint32_t j = it > (uint32_t)kMassStages ? it - kMassStages : 0; j < it; ++j)
                for (int spin = 0; spin < (1 << 22) && !tc_test(full(j % kMassStages), (j / kMassStages) & 1); ++spin) {}
        return;
    }

    bool ok = true;
    const uint32_t a_row = (uint32_t)(warp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7)), a_chunk = (uint32_t)(lane >> 4);
    const uint32_t q_row = (uint32_t)(lane & 7), q_chunk = (uint32_t)(lane >> 3);
    while (cur.next(seg)) {
        const int P = seg.S - seg.n;
        const uint4 set = counted_nodes(p.rows, seg.b, seg.n);
        const int nodes = __popc(set.x) + __popc(set.y) + __popc(set.z) + __popc(set.w), rows = nodes * kGroup, row_tiles = (rows + 7) / 8;
        // the counted query rows, 16 bytes per thread and step; a missing last row is a copy of the last one that counts for nothing
        for (int i = tid; i < row_tiles * 8 * 16; i += kRowsWarps * 32) {
            const int r = min(i >> 4, rows - 1), chunk = i & 15;
            const int node = nth_node(set, r >> 2);
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(p.q + seg.b * p.q_batch + node * p.q_node + (seg.kvh * kGroup + (r & 3)) * p.q_head) + chunk);
            *reinterpret_cast<uint4*>(smem + kMassOffQ + (chunk >> 3) * kMassQHalf + (uint32_t)(i >> 4) * 128u + (((uint32_t)(chunk & 7) ^ ((i >> 4) & 7u)) << 4)) = w;
        }
        for (int r = tid; r < row_tiles * 8; r += kRowsWarps * 32) {
            float x = INFINITY;
            if (r < rows) {
                const int node = nth_node(set, r >> 2);
                x = __ldg(p.lse + ((size_t)seg.b * p.seqs.T + node) * ((size_t)p.seqs.Hkv * kGroup) + seg.kvh * kGroup + (r & 3)) * 1.4426950408889634f;
                if ((r & 3) == 0) s_mask[r >> 2] = dense_mask(p.seqs, seg.b, node);
            }
            s_lse[r] = x;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kRowsWarps * 32) : "memory");
        float* mass = p.mass + ((size_t)seg.b * p.seqs.Hkv + seg.kvh) * ((size_t)p.seqs.max_pages * kPage);
        for (int t = seg.tile0; t < seg.tile1; ++t, ++it) {
            const uint32_t s = it % kMassStages, kb = sbase + s * kMassStage;
            if (ok) ok = __all_sync(0xffffffffu, tc_wait(full(s), (it / kMassStages) & 1, s_abort, p.seqs.status)) != 0;
            if (!ok) continue;
            const int tok0 = t * kMassTile + warp * 16;
            const int j0 = tok0 + (lane >> 2), j1 = j0 + 8;
            uint32_t ka[8][4];
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) ldmatrix4(kb + rows_at(a_row, 2 * ks + a_chunk), ka[ks]);
            __syncwarp();
            if (lane == 0) tc_arrive(empty(s));
            const bool masked = tok0 + 16 > P;
            float sum[2] = {0.0f, 0.0f};
            for (int rt = 0; rt < row_tiles; ++rt) {
                float c[4] = {};
#pragma unroll
                for (int k2 = 0; k2 < 4; ++k2) {
                    uint32_t qf[4];
                    const uint32_t chunk = 4 * k2 + q_chunk;
                    ldmatrix4(sbase + kMassOffQ + (chunk >> 3) * kMassQHalf + (rt * 8 + q_row) * 128u + (((chunk & 7u) ^ q_row) << 4), qf);
                    mma16816(c, ka[2 * k2], qf[0], qf[1]);
                    mma16816(c, ka[2 * k2 + 1], qf[2], qf[3]);
                }
                const int r = rt * 8 + (lane & 3) * 2;
                const float2 e = *reinterpret_cast<const float2*>(s_lse + r);
                float w0 = exp2_approx(fmaf(c[0], p.scale_log2, -e.x)), w1 = exp2_approx(fmaf(c[1], p.scale_log2, -e.y));
                float w2 = exp2_approx(fmaf(c[2], p.scale_log2, -e.x)), w3 = exp2_approx(fmaf(c[3], p.scale_log2, -e.y));
                if (masked) {  // (a quad's two rows belong to one node)
                    const uint4 words = s_mask[min(r >> 2, nodes - 1)];
                    if (j0 >= seg.S || (j0 >= P && !dense_bit(words, j0 - P))) w0 = w1 = 0.0f;
                    if (j1 >= seg.S || (j1 >= P && !dense_bit(words, j1 - P))) w2 = w3 = 0.0f;
                }
                sum[0] += w0 + w1;
                sum[1] += w2 + w3;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
                sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            }
            if ((lane & 3) == 0) {
                if (j0 < seg.S) mass[j0] += sum[0];
                if (j1 < seg.S) mass[j1] += sum[1];
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kRowsWarps * 32) : "memory");
    }
}

}  // namespace ha
