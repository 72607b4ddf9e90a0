// Host side of the ragged attention kernels: tensor maps, launches, and what a kernel plans before it runs.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "attention_args.cuh"

namespace eptq {

struct AttentionPlan {
    int shares;         // blocks of the launch
    int tile_rows;      // rows of a piece
    bool may_cut;       // whether a tile may be cut, by what the host knows
};

AttentionPlan attention_rows_plan(const EptqAttention& a);
AttentionPlan attention_tcgen05_plan(const EptqAttention& a);
int launch_attention_rows(const EptqAttention& a, AttentionArgs& p, int dev, cudaStream_t stream);
int launch_attention_tcgen05(const EptqAttention& a, AttentionArgs& p, int dev, cudaStream_t stream);

PFN_cuTensorMapEncodeTiled_v12000 attention_map_encoder();

// Heads of one key/value head that share a row tile: all of them, or the most that divide them and fit its rows.
inline int heads_in(int kv_group, int rows) {
    int n = kv_group < rows ? kv_group : rows;
    while (kv_group % n != 0) --n;
    return n;
}

// Boxes in 128-byte swizzle, 64 columns wide; what lies outside the tensor reads as zeros.  strides[i], in elements, is that
// of dims[i + 1].
inline bool encode_map(CUtensorMap* map, int dtype, const void* base, int rank, const cuuint64_t* dims, const int64_t* strides, const cuuint32_t* box) {
    cuuint64_t bytes[4];
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<cuuint64_t>(strides[i]) * 2;
    return attention_map_encoder()(map, dtype == EPTQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                                   const_cast<void*>(base), dims, bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// (n_pages, n_kv_heads, page_size, head_dim) caches as boxes of `rows` keys of one head on one page.  A cache without pages
// is never read (its requests have no keys): any address stands for it.
inline bool encode_page_maps(CUtensorMap* k, CUtensorMap* v, const EptqAttention& a, int rows) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.page_size), static_cast<cuuint64_t>(a.n_kv_heads),
                                static_cast<cuuint64_t>(a.n_pages > 0 ? a.n_pages : 1)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1};
    const int64_t ks[3] = {a.head_dim, static_cast<int64_t>(a.page_size) * a.head_dim, a.k_stride};
    const int64_t vs[3] = {a.head_dim, static_cast<int64_t>(a.page_size) * a.head_dim, a.v_stride};
    return encode_map(k, a.dtype, a.n_pages > 0 ? a.k : a.q, 4, dims, ks, box) && encode_map(v, a.dtype, a.n_pages > 0 ? a.v : a.q, 4, dims, vs, box);
}

// Launch that may start its set-up before the previous kernel of the stream has ended (the kernels wait on their own).
template <typename... KArgs, typename... Args>
int launch_dependent(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return EPTQ_ERR_LAUNCH;
    }
    count_launch(EPTQ_KERNEL_OTHER);
    return EPTQ_OK;
}

}  // namespace eptq
