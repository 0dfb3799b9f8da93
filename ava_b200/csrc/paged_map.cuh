// A store's pools as tensors for TMA: boxes of some keys of one page and key head, up to 128 bytes of channels wide.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "serving.cuh"
#include "tc_common.cuh"

namespace ava {

// A pool as a tensor of [pages][...][...][channels] with the smaller of the head and place strides inside, as long as the
// strides nest (each a multiple of the one inside it and at least its extent): what a tensor map describes.
struct PoolShape {
    bool heads_inside;
    uint64_t dims[4], strides[3];
};
inline bool pool_shape(const ava_paged_store& s, PoolShape* p) {
    const int64_t el = s.dtype == AVA_BF16 ? 2 : 4;
    p->heads_inside = s.head_stride <= s.place_stride;
    const int64_t n1 = p->heads_inside ? s.kv_heads : s.page_size, n2 = p->heads_inside ? s.page_size : s.kv_heads;
    int64_t s1 = p->heads_inside ? s.head_stride : s.place_stride, s2 = p->heads_inside ? s.place_stride : s.head_stride, s3 = s.page_stride;
    if (n1 == 1) s1 = s.head_size;     // the stride of a single head or place says nothing
    if (n2 == 1) s2 = n1 * s1;
    if (s.n_pages == 1) s3 = n2 * s2;
    if (s1 < s.head_size || s1 * el % 16 || s2 < n1 * s1 || s2 % s1 || s3 < n2 * s2 || s3 % s2 || s3 * el >= (1ll << 40)) return false;
    const uint64_t d[4] = {(uint64_t)s.head_size, (uint64_t)n1, (uint64_t)n2, (uint64_t)s.n_pages};
    for (int i = 0; i < 4; ++i) p->dims[i] = d[i];
    p->strides[0] = (uint64_t)(s1 * el);
    p->strides[1] = (uint64_t)(s2 * el);
    p->strides[2] = (uint64_t)(s3 * el);
    return true;
}
// boxes of `keys` keys, their channels' columns of up to 128 bytes swizzled by that width
inline bool pool_map(CUtensorMap* map, const void* base, int dtype, const PoolShape& p, int keys) {
    tcc::EncodeFn fn = tcc::encode_fn();
    if (!fn) return false;
    const cuuint32_t el = dtype == AVA_BF16 ? 2 : 4, wide = p.dims[0] * el < 128 ? (cuuint32_t)p.dims[0] : 128 / el;
    const cuuint64_t dims[4] = {p.dims[0], p.dims[1], p.dims[2], p.dims[3]}, strides[3] = {p.strides[0], p.strides[1], p.strides[2]};
    const cuuint32_t box[4] = {wide, p.heads_inside ? 1u : (cuuint32_t)keys, p.heads_inside ? (cuuint32_t)keys : 1u, 1}, es[4] = {1, 1, 1, 1};
    return fn(map, dtype == AVA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, const_cast<void*>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, wide * el == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

#ifdef __CUDACC__
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int page, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(page), "r"(tcc::s32(bar))
                 : "memory");
}
#endif

}  // namespace ava
