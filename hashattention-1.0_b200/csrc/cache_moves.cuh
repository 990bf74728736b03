// What a drafted tree and an eviction do to the paged cache besides attention: the tree's mask words, the accepted path,
// its rows moved to the front of the drafts, and the rows of a cache cut to a budget moved together. Rows move in place
// and only towards lower token numbers.
#pragma once

#include <cooperative_groups.h>

#include "attention_mass.cuh"

namespace ha {

// ---- mask words of a tree: bit j of node i <=> j is i or an ancestor of i ----------------------------------------------
// A thread per node; ancestors by pointer doubling: after round r a node knows its 2^r nearest ones. Latency bounds it: seven
// rounds of one shared-memory trip, where a walk up a chain of 128 nodes takes 128.
__global__ void __launch_bounds__(kMaxNodes) tree_mask_kernel(const int32_t* parents, const int32_t* tree_lens, int T, uint32_t* tree_mask, int32_t* status) {
    __shared__ uint4 s_set[2][kMaxNodes];
    __shared__ int s_up[2][kMaxNodes];
    pdl_wait();
    pdl_launch_dependents();
    const int i = threadIdx.x, b = blockIdx.x;
    int n = tree_lens != nullptr ? __ldg(tree_lens + b) : T;
    if (n < 0 || n > T) {
        if (i == 0) report(status, HA_ERR_BAD_SEQ_LEN);
        n = 0;
    }
    uint4 set = make_uint4(0, 0, 0, 0);
    int up = -1;
    if (i < n) {
        up = __ldg(parents + (size_t)b * T + i);
        if (up < -1 || up >= i) {  // a parent comes before its children
            report(status, HA_ERR_BAD_ARG);
            up = -1;
        }
        const uint32_t bit = 1u << (i & 31);
        if (i < 32) set.x = bit; else if (i < 64) set.y = bit; else if (i < 96) set.z = bit; else set.w = bit;
    }
    int buf = 0;
    for (int reach = 1; reach < n; reach *= 2) {
        s_set[buf][i] = set;
        s_up[buf][i] = up;
        __syncthreads();
        if (up >= 0) {
            const uint4 a = s_set[buf][up];
            set.x |= a.x; set.y |= a.y; set.z |= a.z; set.w |= a.w;
            up = s_up[buf][up];
        }
        buf ^= 1;
    }
    if (i < T) reinterpret_cast<uint4*>(tree_mask)[(size_t)b * T + i] = set;
}

// ---- the accepted path ---------------------------------------------------------------------------------------------------
// From node 0 on: the lowest child whose drafted token is the token the model puts behind its parent. A warp per sequence,
// four nodes per lane; a step of the path is four ballots, and nothing is stored until the path ends.
struct TreeAcceptParams {
    const long long* draft;
    const int32_t* parents;
    const long long* target;
    const int32_t* tree_lens;
    const int32_t* seq_lens;
    uint32_t* accepted;
    int32_t* count;
    long long* next_token;
    int32_t* new_lens;
    int32_t* status;
    int B, T;
};
constexpr int kAcceptWarps = 4;
__global__ void __launch_bounds__(kAcceptWarps * 32) tree_accept_kernel(const TreeAcceptParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, b = blockIdx.x * kAcceptWarps + (threadIdx.x >> 5);
    if (b >= p.B) return;
    const int S = __ldg(p.seq_lens + b);
    int n = p.tree_lens != nullptr ? __ldg(p.tree_lens + b) : p.T;
    if (n < 0 || n > p.T || S < n) {
        if (lane == 0) report(p.status, HA_ERR_BAD_SEQ_LEN);
        n = 0;
    }
    long long draft[kMaskWords], target[kMaskWords];
    int parent[kMaskWords];
#pragma unroll
    for (int k = 0; k < kMaskWords; ++k) {
        const int i = 32 * k + lane;
        const size_t at = (size_t)b * p.T + i;
        parent[k] = i < n ? __ldg(p.parents + at) : -1;
        draft[k] = i < n ? __ldg(p.draft + at) : 0;
        target[k] = i < n ? __ldg(p.target + at) : 0;
    }
    uint32_t words[kMaskWords] = {n > 0 ? 1u : 0u, 0, 0, 0};
    int at = 0, count = n > 0 ? 1 : 0;
    long long token = 0;
    for (int step = 0; step < n; ++step) {
        const long long t = at < 64 ? (at < 32 ? target[0] : target[1]) : (at < 96 ? target[2] : target[3]);
        token = __shfl_sync(0xffffffffu, t, at & 31);
        int next = -1;
#pragma unroll
        for (int k = kMaskWords - 1; k >= 0; --k) {
            // (a child comes after its parent: parents that say otherwise end the path)
            const uint32_t hit = __ballot_sync(0xffffffffu, parent[k] == at && 32 * k + lane > at && draft[k] == token);
            if (hit != 0) next = 32 * k + __ffs(hit) - 1;
        }
        if (next < 0) break;
        at = next;
#pragma unroll
        for (int k = 0; k < kMaskWords; ++k) words[k] |= (at >> 5) == k ? 1u << (at & 31) : 0u;
        ++count;
    }
    if (lane == 0) {
        reinterpret_cast<uint4*>(p.accepted)[b] = make_uint4(words[0], words[1], words[2], words[3]);
        p.count[b] = count;
        if (n > 0) p.next_token[b] = token;
        p.new_lens[b] = S - n + count;
    }
}

// ---- commit: the accepted nodes' rows P + a_k -> P + k ---------------------------------------------------------------------
// A CTA per (kv-head, sequence) holds every row that moves (up to 127 of 528 bytes) in registers before it writes the first
// one, so that nothing is overwritten unread.
struct TreeCommitParams {
    DenseSeqs seqs;
    const uint32_t* accepted;  // [B][4]
    uint4* k_pages;            // rows of 16 x 16 bytes
    uint4* v_pages;
    uint4* hash_pages;         // rows of 16 bytes, or null
    float* mass;               // [B][Hkv][max_pages * 256] or null
};
constexpr int kCommitThreads = 512;
constexpr int kCommitPieces = (kMaxNodes * 33 + kCommitThreads - 1) / kCommitThreads;  // 16-byte pieces per thread: 9
__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const TreeCommitParams p) {
    __shared__ int16_t s_src[kMaxNodes];   // node at place k of the accepted ones
    __shared__ int16_t s_move[kMaxNodes];  // the places whose rows move
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, kvh = blockIdx.x, b = blockIdx.y;
    const DenseSeqs& d = p.seqs;
    int S, n;
    dense_seq(d, b, tid == 0 && kvh == 0, S, n);
    if (n == 0) return;
    const uint4 set = [&] {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p.accepted) + b), f = first_nodes(n);
        return make_uint4(a.x & f.x, a.y & f.y, a.z & f.z, a.w & f.w);
    }();
    const uint32_t w[kMaskWords] = {set.x, set.y, set.z, set.w};
    const int count = __popc(w[0]) + __popc(w[1]) + __popc(w[2]) + __popc(w[3]);
    // Places 0 .. fixed - 1 hold the nodes of the same number: they stay.
    int fixed = 0;
#pragma unroll
    for (int k = 0; k < kMaskWords; ++k)
        if (fixed == 32 * k) fixed += w[k] == 0xffffffffu ? 32 : __ffs(~w[k]) - 1;
    const int moved = count - fixed;
    if (tid < kMaxNodes) {
        const int k = tid >> 5;
        int below = __popc(w[k] & ((1u << lane) - 1u));
#pragma unroll
        for (int q = 0; q < kMaskWords; ++q) below += q < k ? __popc(w[q]) : 0;
        if ((w[k] >> lane) & 1u) {
            s_src[below] = (int16_t)tid;
            if (below >= fixed) s_move[below - fixed] = (int16_t)below;
        }
    }
    __syncthreads();
    const int P = S - n;
    // the drafts lie on two pages at most
    const int page0 = P / kPage;
    const size_t base0 = ((size_t)dense_page(d, b, page0) * d.Hkv + kvh) * kPage;
    const size_t base1 = (S - 1) / kPage > page0 ? ((size_t)dense_page(d, b, page0 + 1) * d.Hkv + kvh) * kPage : base0;
    auto slot = [&](int token) { return (token / kPage == page0 ? base0 : base1) + token % kPage; };
    const int per_row = p.hash_pages != nullptr ? 33 : 32;
    uint4 v[kCommitPieces];
    auto piece = [&](int i, int node_or_place) {
        const size_t row = slot(P + node_or_place);
        const int c = i % per_row;
        return c < 16 ? p.k_pages + row * 16 + c : (c < 32 ? p.v_pages + row * 16 + (c - 16) : p.hash_pages + row);
    };
#pragma unroll
    for (int k = 0; k < kCommitPieces; ++k) {
        const int i = tid + k * kCommitThreads;
        if (i < moved * per_row) v[k] = __ldcg(piece(i, s_src[s_move[i / per_row]]));
    }
    float m = 0.0f;
    float* mass = p.mass != nullptr ? p.mass + ((size_t)b * d.Hkv + kvh) * ((size_t)d.max_pages * kPage) + P : nullptr;
    if (mass != nullptr && tid < count) m = __ldcg(mass + s_src[tid]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kCommitPieces; ++k) {
        const int i = tid + k * kCommitThreads;
        if (i < moved * per_row) *piece(i, s_move[i / per_row]) = v[k];
    }
    if (mass != nullptr && tid < n) mass[tid] = m;  // (n <= 128: places behind the accepted ones start from zero)
}

// ---- eviction: which tokens stay -------------------------------------------------------------------------------------------
// Per (sequence, kv-head): the sink, the recent tokens and the H candidates of the largest accumulated weight, ties by the
// lowest index, in their order. A cluster of 8 CTAs holds a row of weights in its shared memory (as unsigned keys that order
// as the weights do: weights that are not above zero, NaN included, are all 0), finds the H-th largest key by three
// histograms of 11, 10 and 10 bits that it adds up through distributed shared memory, and writes the list and the
// weights of the kept tokens. A warp owns a contiguous part, so that positions follow from counts of the parts in front.
struct EvictParams {
    const float* mass;       // [B][Hkv][pitch]
    float* mass_out;         // [B][Hkv][pitch] or null
    const int32_t* seq_lens;
    int32_t* lens_out;
    int32_t* kept;           // [B][Hkv][keep]
    const int32_t* page_table;
    uint4* k_pages;
    uint4* v_pages;
    uint4* hash_pages;       // or null
    int32_t* status;
    int B, Hkv, max_pages, num_pages;
    int keep, sink, recent;
    int share_max;           // keys of a CTA that its shared memory holds
};
constexpr int kEvictCtas = 8;
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;
constexpr int kEvictShareCap = 40960;  // 160 KB of keys; longer rows are read again by each step

struct EvictCounts {
    int above, level;  // kept whatever happens (sink, recent, above the threshold); at the threshold
};

__device__ __forceinline__ int evict_len(const int32_t* seq_lens, int b, int max_pages, bool reporter, int32_t* status) {
    const int S = __ldg(seq_lens + b);
    if (S < 0 || S > max_pages * kPage) {
        if (reporter) report(status, HA_ERR_BAD_SEQ_LEN);
        return -1;
    }
    return S;
}

__global__ void __cluster_dims__(kEvictCtas, 1, 1) __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ uint32_t s_keys[];
    __shared__ uint32_t s_hist[kEvictBins], s_total[kEvictBins];
    __shared__ uint32_t s_warp[kEvictWarps];
    __shared__ int s_bin;
    __shared__ uint32_t s_above;
    __shared__ EvictCounts s_cta, s_counts[kEvictWarps];
    cg::cluster_group cluster = cg::this_cluster();
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const size_t pitch = (size_t)p.max_pages * kPage, unit = (size_t)b * p.Hkv + kvh;
    const float* mass = p.mass + unit * pitch;
    float* mass_out = p.mass_out != nullptr ? p.mass_out + unit * pitch : nullptr;
    int32_t* kept = p.kept + unit * p.keep;
    const int S = evict_len(p.seq_lens, b, p.max_pages, rank == 0 && kvh == 0 && tid == 0, p.status);
    const int stay = S < 0 ? 0 : min(S, p.keep);
    if (rank == 0 && kvh == 0 && tid == 0) p.lens_out[b] = S < 0 ? __ldg(p.seq_lens + b) : stay;
    if (mass_out != nullptr)
        for (size_t i = stay + rank * kEvictThreads + tid; i < pitch; i += kEvictCtas * kEvictThreads) mass_out[i] = 0.0f;
    if (S <= p.keep) {  // (the same for the whole cluster)
        for (int i = rank * kEvictThreads + tid; i < stay; i += kEvictCtas * kEvictThreads) {
            kept[i] = i;
            if (mass_out != nullptr) mass_out[i] = __ldg(mass + i);
        }
        return;
    }
    const int lo = p.sink, hi = S - p.recent, H = p.keep - p.sink - p.recent;
    // this CTA's tokens, and this warp's part of them
    const int share = ((S + kEvictCtas - 1) / kEvictCtas + 127) & ~127;
    const int t0 = min(S, rank * share), t1 = min(S, t0 + share);
    const bool held = share <= p.share_max;
    auto key_of = [&](float v) { return v > 0.0f ? __float_as_uint(v) : 0u; };
    auto key_at = [&](int t) { return held ? s_keys[t - t0] : key_of(__ldg(mass + t)); };
    if (held)
        for (int t = t0 + tid; t < t1; t += kEvictThreads) s_keys[t - t0] = key_of(__ldg(mass + t));

    // the H-th largest candidate's key, from its upper bits down
    uint32_t prefix = 0, wanted = (uint32_t)H;  // keys that agree with `prefix` above the step's bits; still to be found among them
    uint32_t threshold = 0xffffffffu;
    if (H > 0) {
        const int shifts[3] = {20, 10, 0}, widths[3] = {11, 10, 10};
#pragma unroll
        for (int step = 0; step < 3; ++step) {
            const int shift = shifts[step], bins = 1 << widths[step];
            for (int i = tid; i < kEvictBins; i += kEvictThreads) s_hist[i] = 0;
            __syncthreads();
            for (int t = max(t0, lo) + tid; t < min(t1, hi); t += kEvictThreads) {
                const uint32_t k = key_at(t);
                if (step == 0 || (k >> (shift + widths[step])) == prefix) atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1u);
            }
            cluster.sync();
            // CTA r adds up the r-th eighth of the bins and hands the sums to all
            const int per = kEvictBins / kEvictCtas;
            if (tid < per) {
                uint32_t sum = 0;
#pragma unroll
                for (int r = 0; r < kEvictCtas; ++r) sum += *cluster.map_shared_rank(&s_hist[rank * per + tid], r);
#pragma unroll
                for (int r = 0; r < kEvictCtas; ++r) *cluster.map_shared_rank(&s_total[rank * per + tid], r) = sum;
            }
            cluster.sync();
            // the bin in which the wanted-th largest lies: thread i has 4 bins, from the top down
            uint32_t mine[4], sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                mine[q] = s_total[kEvictBins - 1 - (4 * tid + q)];
                sum += mine[q];
            }
            uint32_t incl = sum;
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, incl, i);
                if (lane >= i) incl += u;
            }
            if (lane == 31) s_warp[warp] = incl;
            __syncthreads();
            uint32_t front = incl - sum;
            for (int q = 0; q < warp; ++q) front += s_warp[q];
            if (front < wanted && wanted <= front + sum) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (front < wanted && wanted <= front + mine[q]) {
                        s_bin = kEvictBins - 1 - (4 * tid + q);
                        s_above = front;
                    }
                    front += mine[q];
                }
            }
            __syncthreads();
            prefix = (prefix << widths[step]) | (uint32_t)s_bin;
            wanted -= s_above;
        }
        threshold = prefix;
    }
    // wanted = tokens at the threshold that stay (the lowest ones)
    const int part = ((t1 - t0 + kEvictWarps - 1) / kEvictWarps + 31) & ~31;
    const int w0 = min(t1, t0 + warp * part), w1 = min(t1, w0 + part);
    auto classify = [&](int t, bool& above, bool& level) {
        above = level = false;
        if (t >= w1) return;
        if (t < lo || t >= hi) above = true;
        else if (H > 0) {
            const uint32_t k = key_at(t);
            above = k > threshold;
            level = k == threshold;
        }
    };
    EvictCounts mine = {0, 0};
    for (int t = w0 + lane; t - lane < w1; t += 32) {
        bool above, level;
        classify(t, above, level);
        mine.above += __popc(__ballot_sync(0xffffffffu, above));
        mine.level += __popc(__ballot_sync(0xffffffffu, level));
    }
    if (lane == 0) s_counts[warp] = mine;
    __syncthreads();
    EvictCounts front = {0, 0}, cta = {0, 0};
    for (int q = 0; q < kEvictWarps; ++q) {
        if (q < warp) front.above += s_counts[q].above, front.level += s_counts[q].level;
        cta.above += s_counts[q].above, cta.level += s_counts[q].level;
    }
    if (tid == 0) s_cta = cta;
    cluster.sync();
    for (int r = 0; r < rank; ++r) {
        const EvictCounts c = *cluster.map_shared_rank(&s_cta, r);
        front.above += c.above, front.level += c.level;
    }
    cluster.sync();  // no CTA leaves while another reads its shared memory
    const int quota = (int)wanted;
    const uint32_t below = (1u << lane) - 1u;
    for (int t = w0 + lane; t - lane < w1; t += 32) {
        bool above, level;
        classify(t, above, level);
        const uint32_t ma = __ballot_sync(0xffffffffu, above), ml = __ballot_sync(0xffffffffu, level);
        const int lrank = front.level + __popc(ml & below);
        if (above || (level && lrank < quota)) {
            const int at = front.above + __popc(ma & below) + min(lrank, quota);
            if (at < p.keep) {
                kept[at] = t;
                if (mass_out != nullptr) mass_out[at] = __ldg(mass + t);
            }
        }
        front.above += __popc(ma);
        front.level += __popc(ml);
    }
}

// ---- eviction: rows kept[i] -> i ------------------------------------------------------------------------------------------
// In place: kept is ascending, so a row never moves up and the row that place i receives lies at or behind every place written
// before. A CTA owns a 64-byte column of K or of V (or the code words) of one (sequence, kv-head) and takes its rows in order, a batch at
// a time: all loads of a batch are complete (a barrier) before its first store, and a later batch reads rows behind all
// places written so far, so its loads run ahead of those stores.
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 8;  // rows per thread and batch
template <int kPieces>        // 16-byte pieces of a row per CTA
__device__ __forceinline__ void evict_move(const EvictParams& p, uint4* pool, int row_pieces, int first_piece, int b, int kvh, int S) {
    constexpr int kRowsPer = kMoveThreads / kPieces, kBatch = kRowsPer * kMoveRows;
    const int32_t* kept = p.kept + ((size_t)b * p.Hkv + kvh) * p.keep;
    const int piece = first_piece + threadIdx.x % kPieces, r0 = threadIdx.x / kPieces;
    auto slot = [&](int token) {
        int page = __ldg(p.page_table + (size_t)b * p.max_pages + token / kPage);
        if (page < 0 || page >= p.num_pages) {
            report(p.status, HA_ERR_BAD_PAGE);
            return (size_t)-1;
        }
        return ((size_t)page * p.Hkv + kvh) * kPage + token % kPage;
    };
    uint4 v[2][kMoveRows];
    uint32_t have[2] = {0, 0};
    auto load = [&](int base, uint4 (&buf)[kMoveRows], uint32_t& mask) {
        int src[kMoveRows];
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
            const int i = base + k * kRowsPer + r0;
            src[k] = i < p.keep ? __ldcg(kept + i) : i;
        }
        mask = 0;
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
            const int i = base + k * kRowsPer + r0;
            if (src[k] > i && src[k] < S) {
                const size_t s = slot(src[k]);
                if (s != (size_t)-1) {
                    buf[k] = __ldcg(pool + s * row_pieces + piece);
                    mask |= 1u << k;
                }
            }
        }
    };
    auto store = [&](int base, const uint4 (&buf)[kMoveRows], uint32_t mask) {
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
            if ((mask >> k) & 1u) {
                const size_t s = slot(base + k * kRowsPer + r0);
                if (s != (size_t)-1) pool[s * row_pieces + piece] = buf[k];
            }
        }
    };
    load(0, v[0], have[0]);
    for (int base = 0; base < p.keep; base += 2 * kBatch) {
        load(base + kBatch, v[1], have[1]);
        __syncthreads();
        store(base, v[0], have[0]);
        load(base + 2 * kBatch, v[0], have[0]);
        __syncthreads();
        store(base + kBatch, v[1], have[1]);
    }
}
constexpr int kMoveColumns = 9;  // four of K, four of V, the code words
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int column = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int S = evict_len(p.seq_lens, b, p.max_pages, false, p.status);
    if (S <= p.keep) return;
    if (column < 8) evict_move<4>(p, column < 4 ? p.k_pages : p.v_pages, 16, (column & 3) * 4, b, kvh, S);
    else if (p.hash_pages != nullptr) evict_move<1>(p, p.hash_pages, 1, 0, b, kvh, S);
}

}  // namespace ha
