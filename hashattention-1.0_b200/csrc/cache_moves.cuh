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
    // The drafts lie on two pages at most. A page id out of range is no place to write to (page 0, which a reader may take instead, is
    // another sequence's): then nothing of the sequence's moves, on no kv-head, the weights included. The ids are the same for the whole CTA.
    const int page0 = P / kPage, page1 = (S - 1) / kPage;
    const int32_t* table = d.page_table + (size_t)b * d.max_pages;
    const int id0 = __ldg(table + page0), id1 = __ldg(table + page1);
    if (id0 < 0 || id0 >= d.num_pages || id1 < 0 || id1 >= d.num_pages) {
        if (tid == 0) report(d.status, HA_ERR_BAD_PAGE);
        return;
    }
    const size_t base0 = ((size_t)id0 * d.Hkv + kvh) * kPage, base1 = ((size_t)id1 * d.Hkv + kvh) * kPage;
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
    // (the barrier takes a predicate formed from what was loaded, so that no load is still on its way behind it)
    uint32_t arrived = __float_as_uint(m);
#pragma unroll
    for (int k = 0; k < kCommitPieces; ++k)
        if (tid + k * kCommitThreads < moved * per_row) arrived ^= v[k].x;
    __syncthreads_or(arrived == 0x5bd1e995u);
#pragma unroll
    for (int k = 0; k < kCommitPieces; ++k) {
        const int i = tid + k * kCommitThreads;
        if (i < moved * per_row) *piece(i, s_move[i / per_row]) = v[k];
    }
    if (mass != nullptr && tid < n) mass[tid] = m;  // (n <= 128: places behind the accepted ones start from zero)
}

// ---- eviction: which tokens stay -------------------------------------------------------------------------------------------
// Per (sequence, kv-head): the sink, the recent tokens and the H candidates of the largest accumulated weight, ties by the
// lowest index, in their order. The weights order as unsigned keys: their bits, or 0 where they are not above zero (NaN included).
// kCtas CTAs (a cluster, or one of them for short rows) hold a row of weights in shared memory, find the H-th largest key by
// three histograms of 11, 10 and 10 bits that they add up through distributed shared memory, and write the list and the weights
// of the kept tokens. A warp owns a contiguous part, so that positions follow from counts of the parts in front.
// What bounds it are the eight cluster barriers (about a microsecond each) and, for long rows, one trip of the weights.
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
    uint32_t* ticket;        // [1] next piece of the move (cleared by the selection)
    uint32_t* read;          // [B][Hkv][read_words] one bit per 64 kept rows: they have been read (cleared by the selection)
    int B, Hkv, max_pages, num_pages;
    int keep, sink, recent;
    int share_max;           // weights of a CTA that its shared memory holds
    int read_words;
};
constexpr int kEvictCtas = 8;
constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictBins = 2048;
constexpr int kEvictShareCap = 40960;  // 160 KB of weights; longer rows are read again by each step
// Capacities of up to this many tokens (the host does not know the lengths) take one CTA a row: no cluster barriers. Both kernels of a
// call, one CTA / a cluster, us, a quarter of the tokens kept, in a graph:
//   4096 tokens   8 rows 13.3 / 16.1, 64 rows 27.2 / 33.5, 256 rows 65 / 120
//   8192 tokens   8 rows 17.4 / 17.1, 64 rows 49.9 / 49.2, 256 rows 119 / 169
//   16384 tokens  8 rows 26.0 / 19.8, 64 rows 95.4 / 77.5
constexpr int kEvictOneCta = 8192;

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

template <int kCtas>
__global__ void __launch_bounds__(kEvictThreads) evict_select_kernel(const EvictParams p) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) float s_mass[];
    __shared__ uint32_t s_hist[kEvictBins], s_total[kEvictBins];
    __shared__ uint32_t s_warp[kEvictWarps];
    __shared__ int s_bin;
    __shared__ uint32_t s_above;
    __shared__ EvictCounts s_cta, s_counts[kEvictWarps];
    cg::cluster_group cluster = cg::this_cluster();
    auto sync_all = [&] {
        if constexpr (kCtas > 1) cluster.sync();
        else __syncthreads();
    };
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = kCtas > 1 ? blockIdx.x : 0, kvh = blockIdx.y, b = blockIdx.z, at_all = rank * kEvictThreads + tid;
    constexpr int kAll = kCtas * kEvictThreads;
    const size_t pitch = (size_t)p.max_pages * kPage, unit = (size_t)b * p.Hkv + kvh;
    const float* mass = p.mass + unit * pitch;
    float* mass_out = p.mass_out != nullptr ? p.mass_out + unit * pitch : nullptr;
    int32_t* kept = p.kept + unit * p.keep;
    for (int i = at_all; i < p.read_words; i += kAll) p.read[unit * p.read_words + i] = 0;
    if (unit == 0 && at_all == 0) *p.ticket = 0;
    const int S = evict_len(p.seq_lens, b, p.max_pages, at_all == 0 && kvh == 0, p.status);
    // (a refused length is reported and passed on, with the whole row of weights)
    const int stay = S < 0 ? (int)pitch : min(S, p.keep);
    if (at_all == 0 && kvh == 0) p.lens_out[b] = S < 0 ? __ldg(p.seq_lens + b) : stay;
    if (mass_out != nullptr) {
        const int first4 = (stay + 3) & ~3;
        if (at_all < first4 - stay) mass_out[stay + at_all] = 0.0f;
        for (size_t i = first4 / 4 + at_all; i < pitch / 4; i += kAll) reinterpret_cast<float4*>(mass_out)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (S <= p.keep) {  // (the same for the whole cluster)
        for (int i = at_all; i < stay; i += kAll) {
            if (S >= 0) kept[i] = i;
            if (mass_out != nullptr) mass_out[i] = __ldg(mass + i);
        }
        return;
    }
    const int lo = p.sink, hi = S - p.recent, H = p.keep - p.sink - p.recent;
    // this CTA's tokens
    const int share = ((S + kCtas - 1) / kCtas + 127) & ~127;
    const int t0 = min(S, rank * share), t1 = min(S, t0 + share);
    const bool held = share <= p.share_max;
    // four tokens from t on (t a multiple of 4; behind t1 there may be anything)
    auto mass4_at = [&](int t) {
        return held ? *reinterpret_cast<const float4*>(s_mass + (t - t0)) : __ldg(reinterpret_cast<const float4*>(mass + t));
    };
    auto key_of = [&](float v) { return v > 0.0f ? __float_as_uint(v) : 0u; };
    if (held) {
        // (rows are read to the next multiple of 4: the pitch is one of 256)
        const float4* src = reinterpret_cast<const float4*>(mass + t0);
        const int n4 = (t1 - t0 + 3) / 4;
#pragma unroll 4
        for (int i = tid; i < n4; i += kEvictThreads) reinterpret_cast<float4*>(s_mass)[i] = __ldg(src + i);
    }

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
            const int c0 = max(t0, lo), c1 = min(t1, hi);
#pragma unroll 2
            for (int t = t0 + 4 * tid; t < c1; t += 4 * kEvictThreads) {
                const float4 v = mass4_at(t);
                const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t k = key_of(e[q]);
                    if (t + q >= c0 && t + q < c1 && (step == 0 || (k >> (shift + widths[step])) == prefix))
                        atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1u);
                }
            }
            sync_all();
            const uint32_t* total = s_hist;
            if constexpr (kCtas > 1) {
                // CTA r adds up the r-th eighth of the bins and hands the sums to all
                constexpr int per = kEvictBins / kCtas;
                if (tid < per) {
                    uint32_t sum = 0;
#pragma unroll
                    for (int r = 0; r < kCtas; ++r) sum += *cluster.map_shared_rank(&s_hist[rank * per + tid], r);
#pragma unroll
                    for (int r = 0; r < kCtas; ++r) *cluster.map_shared_rank(&s_total[rank * per + tid], r) = sum;
                }
                cluster.sync();
                total = s_total;
            }
            // the bin in which the wanted-th largest lies: thread i has 4 bins, from the top down
            uint32_t mine[4], sum = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                mine[q] = total[kEvictBins - 1 - (4 * tid + q)];
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
    // wanted = tokens at the threshold that stay (the lowest ones); this warp's part of the CTA's tokens, four per lane and step
    const int part = ((t1 - t0 + kEvictWarps - 1) / kEvictWarps + 127) & ~127;
    const int w0 = min(t1, t0 + warp * part), w1 = min(t1, w0 + part);
    // of token t (weight v): 1 kept whatever happens, 1 << 16 at the threshold, 0 dropped
    auto classify = [&](int t, float v) -> uint32_t {
        if (t >= w1) return 0;
        if (t < lo || t >= hi) return 1;
        const uint32_t k = key_of(v);
        return H == 0 ? 0u : (k > threshold ? 1u : (k == threshold ? 1u << 16 : 0u));
    };
    EvictCounts mine = {0, 0};
#pragma unroll 2
    for (int t = w0 + 4 * lane; t < w1; t += 128) {
        const float4 v = mass4_at(t);
        const uint32_t c = classify(t, v.x) + classify(t + 1, v.y) + classify(t + 2, v.z) + classify(t + 3, v.w);
        mine.above += c & 0xffff;
        mine.level += c >> 16;
    }
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) {
        mine.above += __shfl_xor_sync(0xffffffffu, mine.above, i);
        mine.level += __shfl_xor_sync(0xffffffffu, mine.level, i);
    }
    if (lane == 0) s_counts[warp] = mine;
    __syncthreads();
    EvictCounts front = {0, 0}, cta = {0, 0};
    for (int q = 0; q < kEvictWarps; ++q) {
        if (q < warp) front.above += s_counts[q].above, front.level += s_counts[q].level;
        cta.above += s_counts[q].above, cta.level += s_counts[q].level;
    }
    if constexpr (kCtas > 1) {
        if (tid == 0) s_cta = cta;
        cluster.sync();
        for (int r = 0; r < rank; ++r) {
            const EvictCounts c = *cluster.map_shared_rank(&s_cta, r);
            front.above += c.above, front.level += c.level;
        }
        cluster.sync();  // no CTA leaves while another reads its shared memory
    }
    const int quota = (int)wanted;
    for (int t = w0 + 4 * lane; t - 4 * lane < w1; t += 128) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (t < w1) v = mass4_at(t);
        const float e[4] = {v.x, v.y, v.z, v.w};
        uint32_t c[4], sum = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            c[q] = classify(t + q, e[q]);
            sum += c[q];
        }
        uint32_t incl = sum;  // (128 tokens at most: no carry between the halves)
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) {
            const uint32_t u = __shfl_up_sync(0xffffffffu, incl, i);
            if (lane >= i) incl += u;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, incl, 31);
        int above = front.above + (int)((incl - sum) & 0xffff), level = front.level + (int)((incl - sum) >> 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (c[q] == 1u || (c[q] != 0u && level < quota)) {
                const int at = above + min(level, quota);
                if (at < p.keep) {
                    kept[at] = t + q;
                    if (mass_out != nullptr) mass_out[at] = e[q];
                }
            }
            above += c[q] & 0xffff;
            level += c[q] >> 16;
        }
        front.above += all & 0xffff;
        front.level += all >> 16;
    }
}

// ---- eviction: rows kept[i] -> i ------------------------------------------------------------------------------------------
// In place: kept is ascending, so a row never moves up, and place i may be written once the row that lies there, if it is a
// kept one, has been read; that row goes to a place up to i. The rows of a (sequence, kv-head) are moved in pieces of 64, handed
// out in order (a ticket); a CTA reads its piece into registers (a warp per row of K and V, 16 bytes per lane), says so, waits until
// the pieces in front of its own whose rows lie on its places have been read, and writes. The pieces it waits for have been handed
// out before, so they are on some running CTA and need nothing from this one; the wait is bounded all the same. Pieces of
// different units are handed out in turn and a list's rows lie far behind their places, so the wait is over before it begins.
// 4 x 131072 tokens x 8 kv-heads cut to 32768 move 1.1 GB in 212 us (5.2 TB/s, the rows 256 bytes at random places). With the
// next piece's rows in flight under this one's wait it took 270: the fence in front of the flag waits for them.
constexpr int kMoveThreads = 256;
constexpr int kMoveWarps = kMoveThreads / 32;
constexpr int kMovePiece = 64;                       // rows
constexpr int kMoveRows = kMovePiece / kMoveWarps;   // rows per warp
constexpr int kMoveCtasPerSm = 4;

struct MovePiece {
    uint32_t unit, piece;
    int src, dst;  // lanes 0 .. 7 of a warp: its rows, as row numbers of the pool (-1: nothing to do)
    bool moves;    // (the whole CTA) the sequence is cut
};
__device__ __forceinline__ MovePiece move_lookup(const EvictParams& p, uint32_t ticket, uint32_t units, uint32_t total, int warp, int lane) {
    MovePiece m;
    m.piece = ticket / units;
    m.unit = ticket - m.piece * units;
    m.src = m.dst = -1;
    m.moves = false;
    if (ticket >= total) return m;
    const int b = (int)(m.unit / (uint32_t)p.Hkv), kvh = (int)m.unit - b * p.Hkv;
    const int i = (int)m.piece * kMovePiece + warp * kMoveRows + lane;
    const bool looks = lane < kMoveRows && i < p.keep;
    const int S = evict_len(p.seq_lens, b, p.max_pages, false, p.status);
    const int token = looks ? __ldcg(p.kept + (size_t)m.unit * p.keep + i) : i;
    m.moves = S > p.keep;
    if (m.moves && looks && token > i && token < S) {
        const int32_t* table = p.page_table + (size_t)b * p.max_pages;
        const int from = __ldg(table + token / kPage), to = __ldg(table + i / kPage);
        if (from >= 0 && from < p.num_pages && to >= 0 && to < p.num_pages) {
            m.src = (from * p.Hkv + kvh) * kPage + token % kPage;
            m.dst = (to * p.Hkv + kvh) * kPage + i % kPage;
        } else report(p.status, HA_ERR_BAD_PAGE);
    }
    return m;
}

// The pieces [lo, hi) in front of `piece` that have rows on its places, by a whole warp: lo is the number of pieces whose last
// row lies in front of the places, hi that of those whose first row does not lie behind them.
__device__ __forceinline__ void move_conflicts(const int32_t* kept, int keep, int piece, int lane, int& lo, int& hi) {
    const int first = piece * kMovePiece, last = first + kMovePiece - 1;
    int base[2] = {0, 0}, left[2] = {piece, piece};  // the answers lie in [base, base + left]
    while (max(left[0], left[1]) > 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int step = (left[e] + 31) / 32;  // lane l looks at the last piece of the l-th part
            const int at = base[e] + min(left[e], (lane + 1) * step) - 1;
            bool in = false;
            if (left[e] > 0 && lane * step < left[e]) {
                const int row = e == 0 ? min(keep - 1, at * kMovePiece + kMovePiece - 1) : at * kMovePiece;
                const int token = __ldcg(kept + row);
                in = e == 0 ? token < first : token <= last;
            }
            const int parts = __popc(__ballot_sync(0xffffffffu, in));  // (ascending: the parts that lie in front as a whole)
            const int skip = min(left[e], parts * step);
            base[e] += skip;
            left[e] = max(0, min(left[e] - skip, step - 1));
        }
    }
    lo = base[0];
    hi = base[1];
}

__global__ void __launch_bounds__(kMoveThreads, kMoveCtasPerSm) evict_move_kernel(const EvictParams p) {
    __shared__ uint32_t s_ticket[2];
    __shared__ int s_ok;
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t units = (uint32_t)(p.B * p.Hkv), total = units * (uint32_t)((p.keep + kMovePiece - 1) / kMovePiece);
    if (tid == 0) s_ticket[0] = atomicAdd(p.ticket, 1u);
    __syncthreads();
    uint32_t ticket = s_ticket[0];
    MovePiece m = move_lookup(p, ticket, units, total, warp, lane);
    for (int round = 1; ticket < total; ++round) {
        if (tid == 0) s_ticket[round & 1] = atomicAdd(p.ticket, 1u);
        uint4 v[kMoveRows], code;
        const size_t column = lane & 15;
        const uint4* pool = (lane < 16 ? p.k_pages : p.v_pages) + column;
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k) {
            const int s = __shfl_sync(0xffffffffu, m.src, k);
            if (s >= 0) v[k] = __ldcg(pool + (size_t)s * 16);
        }
        if (m.src >= 0 && p.hash_pages != nullptr) code = __ldcg(p.hash_pages + m.src);
        int lo = 0, hi = 0;
        if (m.moves && warp == 0) move_conflicts(p.kept + (size_t)m.unit * p.keep, p.keep, (int)m.piece, lane, lo, hi);
        // Every thread's rows are read: the barrier takes a predicate formed from them, so that none is still on its way.
        uint32_t arrived = m.src >= 0 && p.hash_pages != nullptr ? code.x : 0u;
#pragma unroll
        for (int k = 0; k < kMoveRows; ++k)
            if (__shfl_sync(0xffffffffu, m.src, k) >= 0) arrived ^= v[k].x;
        __syncthreads_or(arrived == 0x5bd1e995u);
        if (m.moves && warp == 0) {
            uint32_t* read = p.read + (size_t)m.unit * p.read_words;
            if (lane == 0) {
                __threadfence();
                atomicOr(read + m.piece / 32, 1u << (m.piece & 31));
            }
            bool all = true;
            for (int w0 = lo / 32; w0 * 32 < hi && all; w0 += 32) {
                const int w = w0 + lane;
                uint32_t want = 0;  // bits lo .. hi - 1
                if (w * 32 < hi && w * 32 + 32 > lo) {
                    want = 0xffffffffu;
                    if (w * 32 < lo) want &= 0xffffffffu << (lo - w * 32);
                    if (w * 32 + 32 > hi) want &= 0xffffffffu >> (w * 32 + 32 - hi);
                }
                bool done = want == 0;
                for (int spin = 0; spin < (1 << 20); ++spin) {
                    if (!done) {
                        uint32_t have;
                        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(have) : "l"(read + w) : "memory");
                        done = (have & want) == want;
                    }
                    if (__all_sync(0xffffffffu, done) != 0) break;
                    __nanosleep(100);
                }
                all = __all_sync(0xffffffffu, done) != 0;
            }
            if (lane == 0) {
                __threadfence();
                if (!all) report(p.status, HA_ERR_TIMEOUT);
                s_ok = all ? 1 : 0;
            }
        }
        // the next piece's rows are looked up under this one's wait
        ticket = s_ticket[round & 1];
        const MovePiece next = move_lookup(p, ticket, units, total, warp, lane);
        __syncthreads();
        if (m.moves && s_ok != 0) {
            uint4* to_pool = (lane < 16 ? p.k_pages : p.v_pages) + column;
#pragma unroll
            for (int k = 0; k < kMoveRows; ++k) {
                const int s = __shfl_sync(0xffffffffu, m.src, k), t = __shfl_sync(0xffffffffu, m.dst, k);
                if (s >= 0) to_pool[(size_t)t * 16] = v[k];
            }
            if (m.src >= 0 && p.hash_pages != nullptr) p.hash_pages[m.dst] = code;
        }
        m = next;
        __syncthreads();  // (s_ok has been read)
    }
}

}  // namespace ha
