// tmap.h -- host-side tensor maps (cuTensorMapEncodeTiled) of the GEMM kernels.
#pragma once

#include <cuda.h>

#include <atomic>
#include <mutex>
#include <string>

#include "nq_internal.h"

namespace nq {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Binds the current device's context to a host thread that has none yet.  The runtime does so by itself,
// the driver's cuTensorMapEncodeTiled does not (CUDA_ERROR_INVALID_CONTEXT): a product may be the
// first thing that a thread does.
inline nq_status_t bind_context() {
    typedef CUresult (*CtxGetCurrentFn)(CUcontext*);
    static std::atomic<CtxGetCurrentFn> cached{nullptr};
    CtxGetCurrentFn f = cached.load(std::memory_order_acquire);
    if (!f) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t e = cudaGetDriverEntryPoint("cuCtxGetCurrent", &p, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) return fail(NQ_ERROR_CUDA, "cuCtxGetCurrent entry point not found");
        f = reinterpret_cast<CtxGetCurrentFn>(p);
        cached.store(f, std::memory_order_release);
    }
    CUcontext ctx = nullptr;
    if (f(&ctx) == CUDA_SUCCESS && ctx) return NQ_SUCCESS;
    int dev = -1;
    NQ_CHECK_CUDA(cudaGetDevice(&dev), "cudaGetDevice");
    NQ_CHECK_CUDA(cudaSetDevice(dev), "cudaSetDevice");
    return NQ_SUCCESS;
}

inline nq_status_t get_encode_fn(EncodeTiledFn* fn) {
    static std::atomic<EncodeTiledFn> cached{nullptr};
    static std::mutex mu;
    EncodeTiledFn f = cached.load(std::memory_order_acquire);
    if (!f) {
        std::lock_guard<std::mutex> lk(mu);
        f = cached.load(std::memory_order_relaxed);
        if (!f) {
            void* p = nullptr;
            cudaDriverEntryPointQueryResult q;
            cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
            if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p)
                return fail(NQ_ERROR_CUDA, "cuTensorMapEncodeTiled entry point not found");
            f = reinterpret_cast<EncodeTiledFn>(p);
            cached.store(f, std::memory_order_release);
        }
    }
    *fn = f;
    return bind_context();
}

// 2-D uint8 tensor map: inner extent `inner`, `outer` rows of `ld` bytes,
// box {box_inner, box_outer}, 128-byte swizzle, zero fill out of bounds.
inline nq_status_t make_map(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer, uint64_t ld,
                     uint32_t box_inner, uint32_t box_outer,
                     CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    EncodeTiledFn fn;
    nq_status_t st = get_encode_fn(&fn);
    if (st != NQ_SUCCESS) return st;
    cuuint64_t dims[2] = {inner, outer};
    cuuint64_t strides[1] = {ld};
    cuuint32_t box[2] = {box_inner, box_outer};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NQ_ERROR_CUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
    return NQ_SUCCESS;
}

}  // namespace nq
