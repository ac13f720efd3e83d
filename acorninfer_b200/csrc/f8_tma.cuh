// The 8-bit cache's pages on their way into shared memory: what the two kernels that read them by TMA share.
#pragma once

#include "f8_cache.cuh"
#include "tcgen05_helpers.cuh"

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// Four or eight bytes global -> shared, and this thread's arrival at `bar` once its copies so far are there (the barrier's
// count has room for it).
template <int BYTES> __device__ __forceinline__ void cp_async_bytes(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(bar) : "memory");
}

// The row of key `key` of a stage whose boxes are 2^log_box keys and then as many values (a key's value: 2^log_box further).
__device__ __forceinline__ int f8_stage_row(int key, int log_box) {
    return ((key >> log_box) << (log_box + 1)) + (key & ((1 << log_box) - 1));
}

// A map over codes [planes, rows, D bytes], boxes of box_rows rows of every plane.
static int make_code_map(CUtensorMap* map, const void* base, int64_t rows, int planes, int64_t plane_bytes, int d, int box_rows,
                         CUtensorMapSwizzle swizzle) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr || rows > 0x7fffffff) return ACORN_ERR_UNSUPPORTED;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)d, (cuuint64_t)plane_bytes};
    const cuuint32_t box[3] = {(cuuint32_t)d, (cuuint32_t)box_rows, (cuuint32_t)planes};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 20000 + (int)r;
}

// Keys and values through one map whose planes are the two tensors (the one at the lower address first), where their distance
// fits a map's stride; a map each otherwise (mk: the keys', mv: the values').
static int make_code_maps(CUtensorMap* mk, CUtensorMap* mv, const F8AttnParams& p, int64_t num_pages, int d, int box_rows,
                          CUtensorMapSwizzle swizzle, int* joint, int* v_first) {
    const int64_t rows = (num_pages * p.nkv) << p.logP, apart = p.v_pages - p.k_pages, distance = apart < 0 ? -apart : apart;
    *joint = distance > 0 && distance < (int64_t)1 << 40 && distance % 16 == 0;
    *v_first = *joint && apart < 0;
    const int rc = make_code_map(mk, *v_first ? p.v_pages : p.k_pages, rows, *joint ? 2 : 1, *joint ? distance : rows * d, d, box_rows, swizzle);
    return rc ? rc : make_code_map(mv, p.v_pages, rows, 1, rows * d, d, box_rows, swizzle);
}
