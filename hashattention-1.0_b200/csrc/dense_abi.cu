// extern "C" entry points of dense attention over the paged cache and of what goes with it (declared in include/hashattn.h):
// argument checks, workspace carving and kernel launches. As in hashattn_abi.cu nothing is allocated, nothing synchronises with
// the host and nothing throws.
#include <algorithm>
#include <cmath>

#include "cache_moves.cuh"
#include "host.cuh"
#include "tree_attention_tc.cuh"

namespace ha {
namespace {

constexpr int kDenseMaxCtas = 160;  // CTAs of the kernels that cut the cache into ranges; the workspace is sized for as many

int sm_count(int& sms) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1)
        return HA_ERR_LAUNCH;
    return HA_OK;
}

int check_tree(const ha_tree_t* t) {
    if (t == nullptr || t->max_nodes < 1) return HA_ERR_BAD_ARG;
    return t->max_nodes > kMaxNodes ? HA_ERR_UNSUPPORTED_DIM : HA_OK;
}

// Rows of a pool (page, kv-head, token of the page) are numbered in 32 bits.
bool too_many_rows(const ha_shape_t* s) { return (long long)s->num_pages * s->num_kv_heads * kPage > 0x7fffffffll; }

// The kernels count the tiles of 64 tokens of all sequences, heads and groups of 16 rows in 32 bits, and copy tiles by row number.
int check_tiles(const ha_shape_t* s, const ha_tree_t* t) {
    if (too_many_rows(s)) return HA_ERR_UNSUPPORTED_DIM;
    const double groups = (double)((t->max_nodes * kGroup + 15) / 16), tiles = (double)s->max_pages * (kPage / kRowsTile);
    return tiles > kMaxTiles / kRowsTile || tiles * groups * s->batch * s->num_kv_heads > kMaxTiles ? HA_ERR_UNSUPPORTED_DIM : HA_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

DenseSeqs seqs_of(const ha_shape_t* s, const ha_tree_t* t, const int32_t* page_table, const int32_t* seq_lens, int32_t* status) {
    DenseSeqs d;
    d.page_table = page_table;
    d.seq_lens = seq_lens;
    d.tree_lens = t->tree_lens;
    d.tree_mask = t->tree_mask;
    d.status = status;
    d.B = s->batch;
    d.Hkv = s->num_kv_heads;
    d.T = t->max_nodes;
    d.max_pages = s->max_pages;
    d.num_pages = s->num_pages;
    return d;
}

// Strides of q [B][T][Hq][128] in elements; rows of 16-byte pieces.
int q_strides_of(const ha_shape_t* s, const ha_tree_t* t, const int64_t* strides, long long& batch, long long& node, long long& head) {
    head = kHeadDim;
    node = head * s->num_kv_heads * kGroup;
    batch = node * t->max_nodes;
    if (strides != nullptr) {
        batch = strides[0];
        node = strides[1];
        head = strides[2];
    }
    return (batch | node | head) % 8 == 0 && batch >= 0 && node >= 0 && head >= 0 ? HA_OK : HA_ERR_BAD_ARG;
}

// Query rows per CTA of the attention of trees of up to max_nodes nodes: a kernel each. Measured on both sides of the borders, us:
//   4 nodes   16 rows on mma.sync / 128 on tcgen05   8192 tokens x 8 kv-heads 16.4 / 18.4, 8 x 33001 x 1 32.3 / 39.1, 16 x 16384 x 8 166 / 196
//   8 nodes   32 rows on mma.sync / 128 on tcgen05   21.8 / 18.8, 49.7 / 39.8, 292 / 197 (131072 x 8: 154 / 97)
//   40 nodes  groups of 128 rows / 256               20011 x 8 43.6 / 39.8; with 64 nodes 2 x 131072 x 8 444 / 361, 8192 x 8 29.5 / 30.6
int rows_of(int max_nodes) { return max_nodes * kGroup <= 16 ? 16 : (max_nodes * kGroup <= 128 ? 128 : 256); }

size_t tree_workspace(int max_nodes) {
    return (size_t)2 * kDenseMaxCtas * rows_of(max_nodes) * (sizeof(float2) + kHeadDim * sizeof(float));
}

// The attention kernel and the merge behind it.
template <int kTile, int kRows, int kCross>
int launch_tree(void (*kernel)(TreeAttentionParams, CUtensorMap, CUtensorMap), int threads, size_t smem_bytes, const ha_shape_t* shape,
                const TreeAttentionParams& p, cudaStream_t st) {
    int sms = 0;
    if (sm_count(sms) != HA_OK) return HA_ERR_LAUNCH;
    CUtensorMap k_map, v_map;
    const uint64_t rows = (uint64_t)shape->num_pages * shape->num_kv_heads * kPage;
    if (!encode_row_map(&k_map, p.k_pages, rows, kTile) || !encode_row_map(&v_map, p.v_pages, rows, kTile)) return HA_ERR_LAUNCH;
    // (a per-device function attribute: set at every call, so that a process driving several GPUs is served)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes) != cudaSuccess) return HA_ERR_LAUNCH;
    const int groups = DenseCut<kTile, kRows, kCross>::groups(p.seqs.T);
    const long long tiles = (long long)shape->batch * shape->num_kv_heads * groups * shape->max_pages * (kPage / kTile);
    const int ctas = (int)std::min<long long>(tiles, std::min(sms, kDenseMaxCtas));
    if (launch_smem(kernel, dim3(ctas), dim3(threads), smem_bytes, st, 1, p, k_map, v_map) != cudaSuccess) return HA_ERR_LAUNCH;
    const int rows_max = std::min(kRows, p.seqs.T * kGroup);
    cudaError_t e;
    if constexpr (kRows == RowsLayout::kRows) {
        const dim3 grid(shape->num_kv_heads, shape->batch, (rows_max + kTreeMergeWarps - 1) / kTreeMergeWarps);
        e = launch(tree_merge_rows_kernel, grid, dim3(kTreeMergeWarps * 32), st, 1, p, ctas);
    } else {
        const bool few = 4ll * shape->batch * shape->num_kv_heads * groups < ctas;  // units: many partial results of each
        const int parts = shape->num_kv_heads * groups * (few ? kTaMergeParts : kTaMergeParts / 4);
        e = launch(few ? tree_merge_tc_kernel<kRows, 12, 1> : tree_merge_tc_kernel<kRows, 2, 4>, dim3(parts, shape->batch, (rows_max + 31) / 32),
                   dim3(kTaMergeThreads), st, 1, p, ctas);
    }
    return e == cudaSuccess ? HA_OK : HA_ERR_LAUNCH;
}

// Words of one bit per 64 kept rows, for the largest budget a sequence can exceed.
int evict_read_words(const ha_shape_t* s) { return (s->max_pages * (kPage / kMovePiece) + 31) / 32; }
size_t evict_workspace(const ha_shape_t* s) { return 16 + (size_t)s->batch * s->num_kv_heads * evict_read_words(s) * sizeof(uint32_t); }

}  // namespace
}  // namespace ha

using namespace ha;

extern "C" {

size_t ha_tree_workspace_bytes(int32_t max_nodes) {
    return max_nodes < 1 || max_nodes > kMaxNodes ? 0 : tree_workspace(max_nodes);
}

int ha_tree_mask(const int32_t* parents, const int32_t* tree_lens, int32_t batch, int32_t max_nodes, uint32_t* tree_mask, int32_t* status, void* stream) {
    if (parents == nullptr || tree_mask == nullptr || batch < 1 || max_nodes < 1 || !aligned16(tree_mask)) return HA_ERR_BAD_ARG;
    if (max_nodes > kMaxNodes) return HA_ERR_UNSUPPORTED_DIM;
    return launch(tree_mask_kernel, dim3(batch), dim3(kMaxNodes), static_cast<cudaStream_t>(stream), 1, parents, tree_lens, (int)max_nodes, tree_mask,
                  status) == cudaSuccess ? HA_OK : HA_ERR_LAUNCH;
}

int ha_tree_accept(const int64_t* draft, const int32_t* parents, const int64_t* target, const int32_t* tree_lens, const int32_t* seq_lens,
                   int32_t batch, int32_t max_nodes, uint32_t* accepted, int32_t* count, int64_t* next_token, int32_t* new_lens,
                   int32_t* status, void* stream) {
    if (draft == nullptr || parents == nullptr || target == nullptr || seq_lens == nullptr || accepted == nullptr || count == nullptr ||
        next_token == nullptr || new_lens == nullptr || batch < 1 || max_nodes < 1 || !aligned16(accepted))
        return HA_ERR_BAD_ARG;
    if (max_nodes > kMaxNodes) return HA_ERR_UNSUPPORTED_DIM;
    if (new_lens == seq_lens) return HA_ERR_BAD_ARG;  // (the commits still need the lengths with all drafts)
    TreeAcceptParams p;
    p.draft = reinterpret_cast<const long long*>(draft);
    p.parents = parents;
    p.target = reinterpret_cast<const long long*>(target);
    p.tree_lens = tree_lens;
    p.seq_lens = seq_lens;
    p.accepted = accepted;
    p.count = count;
    p.next_token = reinterpret_cast<long long*>(next_token);
    p.new_lens = new_lens;
    p.status = status;
    p.B = batch;
    p.T = max_nodes;
    return launch(tree_accept_kernel, dim3((batch + kAcceptWarps - 1) / kAcceptWarps), dim3(kAcceptWarps * 32), static_cast<cudaStream_t>(stream), 1,
                  p) == cudaSuccess ? HA_OK : HA_ERR_LAUNCH;
}

int ha_tree_attention(const ha_shape_t* shape, const ha_tree_t* tree, const void* q, const int64_t* q_strides, const void* k_pages,
                      const void* v_pages, const int32_t* page_table, const int32_t* seq_lens, float sm_scale, void* out, float* lse,
                      void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
    int rc = check_shape(shape);
    if (rc == HA_OK) rc = check_tree(tree);
    if (rc == HA_OK) rc = check_tiles(shape, tree);
    if (rc != HA_OK) return rc;
    if (q == nullptr || k_pages == nullptr || v_pages == nullptr || page_table == nullptr || seq_lens == nullptr || out == nullptr || status == nullptr ||
        !(sm_scale > 0.0f) || !std::isfinite(sm_scale) || !aligned16(q) || !aligned16(out) || !aligned16(k_pages) || !aligned16(v_pages) ||
        !aligned16(tree->tree_mask) || !aligned16(workspace))
        return HA_ERR_BAD_ARG;
    if (workspace == nullptr || workspace_bytes < tree_workspace(tree->max_nodes)) return HA_ERR_WORKSPACE;
    TreeAttentionParams p;
    rc = q_strides_of(shape, tree, q_strides, p.q_batch, p.q_node, p.q_head);
    if (rc != HA_OK) return rc;
    p.seqs = seqs_of(shape, tree, page_table, seq_lens, status);
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.out = static_cast<__nv_bfloat16*>(out);
    p.lse = lse;
    const int rows = rows_of(tree->max_nodes);
    p.part_acc = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_acc + (size_t)2 * kDenseMaxCtas * rows * kHeadDim);
    p.scale_log2 = sm_scale * 1.4426950408889634f;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    p.k_pages = static_cast<const __nv_bfloat16*>(k_pages);
    p.v_pages = static_cast<const __nv_bfloat16*>(v_pages);
    if (rows == RowsLayout::kRows) return launch_tree<kRowsTile, RowsLayout::kRows, 0>(tree_attention_rows_kernel, kRowsThreads, RowsLayout::kSmemBytes, shape, p, st);
    if (rows == 128) return launch_tree<kTaTile, 128, TaLayout<false>::kCross>(tree_attention_tc_kernel<false>, kTaThreads, TaLayout<false>::kSmemBytes, shape, p, st);
    return launch_tree<kTaTile, 256, TaLayout<true>::kCross>(tree_attention_tc_kernel<true>, kTaThreads, TaLayout<true>::kSmemBytes, shape, p, st);
}

int ha_attention_mass(const ha_shape_t* shape, const ha_tree_t* tree, const void* q, const int64_t* q_strides, const float* lse, const uint32_t* rows,
                      const void* k_pages, const int32_t* page_table, const int32_t* seq_lens, float sm_scale, float* mass, int32_t* status,
                      void* stream) {
    int rc = check_shape(shape);
    if (rc == HA_OK) rc = check_tree(tree);
    if (rc == HA_OK) rc = check_tiles(shape, tree);
    if (rc != HA_OK) return rc;
    if (q == nullptr || lse == nullptr || k_pages == nullptr || page_table == nullptr || seq_lens == nullptr || mass == nullptr || status == nullptr ||
        !(sm_scale > 0.0f) || !std::isfinite(sm_scale) || !aligned16(q) || !aligned16(k_pages) || !aligned16(tree->tree_mask) || !aligned16(rows) ||
        !aligned16(mass))
        return HA_ERR_BAD_ARG;
    AttentionMassParams p;
    rc = q_strides_of(shape, tree, q_strides, p.q_batch, p.q_node, p.q_head);
    if (rc != HA_OK) return rc;
    p.seqs = seqs_of(shape, tree, page_table, seq_lens, status);
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.lse = lse;
    p.rows = rows;
    p.mass = mass;
    const double exact = (double)sm_scale * 1.4426950408889634074;
    p.scale_log2 = (float)exact;
    p.lse_scale = 1.4426950408889634074 * ((double)p.scale_log2 / exact) * (1.0 - kScoreCut);
    p.q_rows = (tree->max_nodes * kGroup + 15) & ~15;
    p.slots = mass_slots(p.q_rows);
    const size_t smem = mass_smem_bytes(p.slots, p.q_rows);
    int sms = 0;
    CUtensorMap k_map;
    if (sm_count(sms) != HA_OK || !encode_row_map(&k_map, k_pages, (uint64_t)shape->num_pages * shape->num_kv_heads * kPage, kMassTile) ||
        cudaFuncSetAttribute(attention_mass_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return HA_ERR_LAUNCH;
    const long long tiles = (long long)shape->batch * shape->num_kv_heads * shape->max_pages * (kPage / kMassTile);
    const int ctas = (int)std::min<long long>(tiles, sms);
    return launch_smem(attention_mass_kernel, dim3(ctas), dim3(kMassThreads), smem, static_cast<cudaStream_t>(stream), 1, p, k_map) == cudaSuccess
               ? HA_OK : HA_ERR_LAUNCH;
}

int ha_tree_commit(const ha_shape_t* shape, const ha_tree_t* tree, const uint32_t* accepted, void* k_pages, void* v_pages, uint32_t* hash_pages,
                   const int32_t* page_table, const int32_t* seq_lens, float* mass, int32_t* status, void* stream) {
    int rc = check_shape(shape);
    if (rc == HA_OK) rc = check_tree(tree);
    if (rc != HA_OK) return rc;
    if (accepted == nullptr || k_pages == nullptr || v_pages == nullptr || page_table == nullptr || seq_lens == nullptr || status == nullptr ||
        !aligned16(accepted) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(hash_pages))
        return HA_ERR_BAD_ARG;
    TreeCommitParams p;
    p.seqs = seqs_of(shape, tree, page_table, seq_lens, status);
    p.accepted = accepted;
    p.k_pages = static_cast<uint4*>(k_pages);
    p.v_pages = static_cast<uint4*>(v_pages);
    p.hash_pages = reinterpret_cast<uint4*>(hash_pages);
    p.mass = mass;
    return launch(tree_commit_kernel, dim3(shape->num_kv_heads, shape->batch), dim3(kCommitThreads), static_cast<cudaStream_t>(stream), 1, p) ==
                   cudaSuccess ? HA_OK : HA_ERR_LAUNCH;
}

size_t ha_evict_workspace_bytes(const ha_shape_t* shape) { return check_shape(shape) == HA_OK ? evict_workspace(shape) : 0; }

int ha_cache_evict(const ha_shape_t* shape, int32_t keep_tokens, int32_t init_budget, int32_t recent_budget, const float* mass, void* k_pages,
                   void* v_pages, uint32_t* hash_pages, const int32_t* page_table, const int32_t* seq_lens, int32_t* kept, float* mass_out,
                   int32_t* lens_out, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
    const int rc = check_shape(shape);
    if (rc != HA_OK) return rc;
    if (mass == nullptr || k_pages == nullptr || v_pages == nullptr || page_table == nullptr || seq_lens == nullptr || kept == nullptr ||
        lens_out == nullptr || status == nullptr || mass == mass_out || seq_lens == lens_out || !aligned16(k_pages) || !aligned16(v_pages) ||
        !aligned16(hash_pages) || !aligned16(mass) || !aligned16(mass_out) || !aligned16(workspace) || keep_tokens < 1 || init_budget < 0 ||
        recent_budget < 0 || (long long)init_budget + recent_budget > keep_tokens)
        return HA_ERR_BAD_ARG;
    if (workspace == nullptr || workspace_bytes < evict_workspace(shape)) return HA_ERR_WORKSPACE;
    if (too_many_rows(shape)) return HA_ERR_UNSUPPORTED_DIM;
    const long long capacity = (long long)shape->max_pages * kPage;
    EvictParams p;
    p.mass = mass;
    p.mass_out = mass_out;
    p.seq_lens = seq_lens;
    p.lens_out = lens_out;
    p.kept = kept;
    p.page_table = page_table;
    p.k_pages = static_cast<uint4*>(k_pages);
    p.v_pages = static_cast<uint4*>(v_pages);
    p.hash_pages = reinterpret_cast<uint4*>(hash_pages);
    p.status = status;
    p.ticket = static_cast<uint32_t*>(workspace);
    p.read = p.ticket + 4;
    p.read_words = evict_read_words(shape);
    p.B = shape->batch;
    p.Hkv = shape->num_kv_heads;
    p.max_pages = shape->max_pages;
    p.num_pages = shape->num_pages;
    p.keep = keep_tokens;
    p.sink = init_budget;
    p.recent = recent_budget;
    int sms = 0;
    if (sm_count(sms) != HA_OK) return HA_ERR_LAUNCH;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool one = capacity <= kEvictOneCta;
    const int ctas = one ? 1 : kEvictCtas;
    p.share_max = (int)std::min<long long>(((capacity + ctas - 1) / ctas + 127) & ~127ll, kEvictShareCap);
    const size_t smem = (size_t)p.share_max * sizeof(float);
    auto select = one ? evict_select_kernel<1> : evict_select_kernel<kEvictCtas>;
    if (cudaFuncSetAttribute(select, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        launch_smem(select, dim3(ctas, shape->num_kv_heads, shape->batch), dim3(kEvictThreads), smem, st, one ? 1 : kEvictCtas, p) != cudaSuccess)
        return HA_ERR_LAUNCH;
    // (sequences are no longer than the capacity, so larger budgets move nothing)
    if (keep_tokens >= capacity) return HA_OK;
    const long long pieces = (long long)shape->batch * shape->num_kv_heads * ((keep_tokens + kMovePiece - 1) / kMovePiece);
    return launch(evict_move_kernel, dim3((unsigned)std::min<long long>(pieces, (long long)sms * kMoveCtasPerSm)), dim3(kMoveThreads), st, 1, p) ==
                   cudaSuccess ? HA_OK : HA_ERR_LAUNCH;
}

}  // extern "C"
