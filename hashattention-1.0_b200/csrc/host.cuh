// Host-side helpers shared by the files that hold the C entry points: shape checks, kernel launches, tensor maps.
#pragma once

#include <atomic>
#include <utility>

#include <cuda.h>

#include "common.cuh"

namespace ha {

inline int check_shape(const ha_shape_t* s) {
    if (s == nullptr) return HA_ERR_BAD_ARG;
    if (s->gqa_group != kGroup || s->head_dim != kHeadDim || s->page_size != kPage)
        return HA_ERR_UNSUPPORTED_DIM;
    if (s->batch < 1 || s->num_kv_heads < 1 || s->max_pages < 1 || s->num_pages < 1 ||
        s->sel_stride < 1)
        return HA_ERR_BAD_ARG;
    if (s->batch > 65535 || s->num_kv_heads * kGroup > 65535 || s->max_pages > 65535)
        return HA_ERR_UNSUPPORTED_DIM;
    return HA_OK;
}

// Every kernel is launched with programmatic stream serialization (it may start while its
// predecessor drains and synchronises itself with griddepcontrol.wait); cluster_x > 1 adds a
// thread-block cluster along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_smem(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem_bytes, cudaStream_t stream, int cluster_x,
                        Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster_x > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster_x;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    cfg.attrs = attr;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t stream, int cluster_x, Args&&... args) {
    return launch_smem(kernel, grid, block, 0, stream, cluster_x, std::forward<Args>(args)...);
}

// cuTensorMapEncodeTiled, looked up once through the runtime (the library does not link against libcuda).
// The K or V pool as a 2-d tensor [rows = pages x kv heads x page size][128]: boxes of 64 elements x box_rows rows, written
// to shared memory in the 128-byte swizzle.
inline bool encode_row_map(CUtensorMap* map, const void* pages, uint64_t rows, int box_rows) {
    typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static std::atomic<encode_fn> cached{nullptr};
    encode_fn fn = cached.load();
    if (fn == nullptr) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || sym == nullptr)
            return false;
        fn = reinterpret_cast<encode_fn>(sym);
        cached.store(fn);
    }
    const cuuint64_t dims[2] = {(cuuint64_t)kHeadDim, rows};
    const cuuint64_t strides[1] = {(cuuint64_t)kHeadDim * sizeof(__nv_bfloat16)};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    auto encode = [&] {
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pages), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a thread's first call: it has no context until the runtime gives it its device's
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
        r = encode();
    }
    return r == CUDA_SUCCESS;
}

}  // namespace ha
