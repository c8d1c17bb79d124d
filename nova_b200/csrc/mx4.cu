// mx4.cu -- microscaled 4-bit formats: quantize and dequantize.
#include <algorithm>
#include <string>

#include "mx4.cuh"
#include "nq_internal.h"
#include "ptx.cuh"

namespace nq {
namespace {

using namespace dev;

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t block_umax(uint32_t m, int parity) {
    __shared__ uint32_t s_max[2][32];
    m = __reduce_max_sync(0xffffffffu, m);
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) s_max[parity][w] = m;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, l < (blockDim.x >> 5) ? s_max[parity][l] : 0u);
}

// One block per row; NVFP4 reads the row twice (its maximum first).
template <class In, int F, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx4_quant(const In* __restrict__ src, size_t ld, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ bscales, float* __restrict__ rscales, int rows,
                                                        int cols) {
    pdl_launch_dependents();
    pdl_wait();
    const int nvec = (cols + 7) / 8;
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int pitch_words = static_cast<int>(mx4_pitch(cols) / 4);
    const int nstep = words * Mx4Traits<F>::word_lanes;
    int parity = 0;
    for (long long rl = blockIdx.x; rl < rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = src + row * ld;
        float level = 0.0f;
        bool ok = true;
        if (F == kNVFP4) {
            uint32_t m = 0;
            for (int v = threadIdx.x; v < nvec; v += kThreads) {
                float f[8];
                unpack8<In>(load_raw8<In, VEC>(x, v, cols), f);
                m = max(m, amax_bits8(f));
            }
            m = block_umax(m, parity);
            ok = m < kInfBits;
            level = nv_row_level(m);
            if (threadIdx.x == 0) rscales[row] = nv_row_scale(m, level);
        }
        for (int v = threadIdx.x; v - static_cast<int>(threadIdx.x & 31) < nstep; v += kThreads) {
            float f[8];
            unpack8<In>(load_raw8<In, VEC>(x, v, cols), f);
            uint32_t byte;
            const uint32_t c = mx4_encode<F>(f, level, ok, &byte);
            mx4_store<F>(codes + row * mx4_pitch(cols), bscales, row, v, pitch_words, words, c, byte);
        }
    }
}

template <class T, int F, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx4_dequant(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ bscales,
                                                          const float* __restrict__ rscales, T* __restrict__ dst, int rows,
                                                          int cols) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int L = Mx4Traits<F>::block_lanes;
    const int nvec = (cols + 7) / 8;
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    for (long long rl = blockIdx.x; rl < rows; rl += gridDim.x) {
        const int row = static_cast<int>(rl);
        const float g = rscales ? __ldg(rscales + row) : 1.0f;
        const uint32_t* code = reinterpret_cast<const uint32_t*>(codes + row * mx4_pitch(cols));
        for (int v = threadIdx.x; v < nvec; v += kThreads) {
            const int b = v / L;
            const float s = mx4_scale_value(F, __ldg(bscales + mx4_scale_offset(row, b / 4, words) + b % 4));
            float f[8];
            e2m1_decode8(__ldg(code + v), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(__fmul_rn(f[e], s), g);
            store_raw8<T, VEC>(dst + static_cast<size_t>(row) * cols, v, cols, pack8<T>(f));
        }
    }
}

// ---- host side -------------------------------------------------------------------
nq_status_t bad(const char* who, const char* what) {
    return fail(NQ_ERROR_INVALID_VALUE, std::string(who) + ": " + what);
}

nq_status_t check_matrix(const char* who, int rows, int cols, nq_mx4_format_t fmt, nq_dtype_t dt) {
    if (rows < 0 || cols < 0) return bad(who, "negative size");
    if (cols > (1 << 30)) return fail(NQ_ERROR_UNSUPPORTED, std::string(who) + ": more than 2^30 columns");
    if (fmt != NQ_MXFP4 && fmt != NQ_NVFP4) return bad(who, "format");
    if (dt != NQ_F32 && dt != NQ_BF16) return bad(who, "dtype must be NQ_F32 or NQ_BF16");
    return NQ_SUCCESS;
}

}  // namespace
}  // namespace nq

extern "C" {

size_t nq_mx4_row_bytes(int cols) { return cols < 0 ? 0 : nq::dev::mx4_pitch(cols); }

size_t nq_mx4_scale_bytes(int rows, int cols, nq_mx4_format_t fmt) {
    if (rows < 0 || cols < 0 || (fmt != NQ_MXFP4 && fmt != NQ_NVFP4)) return 0;
    return (static_cast<size_t>(rows) + 127) / 128 * nq::dev::mx4_words(cols, fmt == NQ_MXFP4 ? 32 : 16) * 512;
}

nq_status_t nq_quantize_rows_mx4(const void* src, nq_dtype_t src_dtype, int src_stride, uint8_t* codes,
                                 uint8_t* block_scales, float* row_scales, int rows, int cols, nq_mx4_format_t fmt,
                                 nq_stream_t s) {
    const char* who = "nq_quantize_rows_mx4";
    nq_status_t st = nq::check_matrix(who, rows, cols, fmt, src_dtype);
    if (st != NQ_SUCCESS) return st;
    if (src_stride && src_stride < cols) return nq::bad(who, "the row stride is smaller than cols");
    if (rows == 0 || cols == 0) return NQ_SUCCESS;
    if (!src || !codes || !block_scales) return nq::bad(who, "null pointer");
    if (fmt == NQ_NVFP4 && !row_scales) return nq::bad(who, "NQ_NVFP4 needs row scales");
    if (fmt == NQ_MXFP4 && row_scales) return nq::bad(who, "NQ_MXFP4 has no row scales");
    if (!nq::aligned16(codes) || !nq::aligned16(block_scales)) return nq::bad(who, "codes and block scales must be 16-byte aligned");
    if (!nq::aligned_to(src, src_dtype) || !nq::aligned_to(row_scales, NQ_F32)) return nq::bad(who, "a pointer is not aligned to its type");
    nq::DeviceInfo di;
    st = nq::current_device(&di);
    if (st != NQ_SUCCESS) return st;
    const size_t ld = src_stride ? src_stride : cols;
    const bool vec = cols % 8 == 0 && ld * (src_dtype == NQ_BF16 ? 2 : 4) % 16 == 0 && nq::aligned16(src);
    const int grid = static_cast<int>(std::min<long long>(rows, static_cast<long long>(di.sm_count) * 8));
    auto go = [&](auto kern, const auto* typed) {
        return nq::cuda_status(nq::launch_pdl(kern, dim3(grid), dim3(nq::kThreads), 0, s, typed, ld, codes, block_scales,
                                              row_scales, rows, cols),
                               who);
    };
    using namespace nq;
    const float* f = static_cast<const float*>(src);
    const uint16_t* h = static_cast<const uint16_t*>(src);
    if (fmt == NQ_MXFP4) {
        if (src_dtype == NQ_F32) return vec ? go(k_mx4_quant<float, kMXFP4, true>, f) : go(k_mx4_quant<float, kMXFP4, false>, f);
        return vec ? go(k_mx4_quant<uint16_t, kMXFP4, true>, h) : go(k_mx4_quant<uint16_t, kMXFP4, false>, h);
    }
    if (src_dtype == NQ_F32) return vec ? go(k_mx4_quant<float, kNVFP4, true>, f) : go(k_mx4_quant<float, kNVFP4, false>, f);
    return vec ? go(k_mx4_quant<uint16_t, kNVFP4, true>, h) : go(k_mx4_quant<uint16_t, kNVFP4, false>, h);
}

nq_status_t nq_dequantize_rows_mx4(const uint8_t* codes, const uint8_t* block_scales, const float* row_scales, void* dst,
                                   nq_dtype_t dst_dtype, int rows, int cols, nq_mx4_format_t fmt, nq_stream_t s) {
    const char* who = "nq_dequantize_rows_mx4";
    nq_status_t st = nq::check_matrix(who, rows, cols, fmt, dst_dtype);
    if (st != NQ_SUCCESS) return st;
    if (rows == 0 || cols == 0) return NQ_SUCCESS;
    if (!codes || !block_scales || !dst) return nq::bad(who, "null pointer");
    if (!nq::aligned16(codes) || !nq::aligned16(block_scales)) return nq::bad(who, "codes and block scales must be 16-byte aligned");
    if (!nq::aligned_to(dst, dst_dtype) || !nq::aligned_to(row_scales, NQ_F32)) return nq::bad(who, "a pointer is not aligned to its type");
    nq::DeviceInfo di;
    st = nq::current_device(&di);
    if (st != NQ_SUCCESS) return st;
    const bool vec = cols % 8 == 0 && nq::aligned16(dst);
    const int grid = static_cast<int>(std::min<long long>(rows, static_cast<long long>(di.sm_count) * 8));
    auto go = [&](auto kern, auto* typed) {
        return nq::cuda_status(nq::launch_pdl(kern, dim3(grid), dim3(nq::kThreads), 0, s, codes, block_scales, row_scales,
                                              typed, rows, cols),
                               who);
    };
    using namespace nq;
    float* f = static_cast<float*>(dst);
    uint16_t* h = static_cast<uint16_t*>(dst);
    if (fmt == NQ_MXFP4) {
        if (dst_dtype == NQ_F32) return vec ? go(k_mx4_dequant<float, kMXFP4, true>, f) : go(k_mx4_dequant<float, kMXFP4, false>, f);
        return vec ? go(k_mx4_dequant<uint16_t, kMXFP4, true>, h) : go(k_mx4_dequant<uint16_t, kMXFP4, false>, h);
    }
    if (dst_dtype == NQ_F32) return vec ? go(k_mx4_dequant<float, kNVFP4, true>, f) : go(k_mx4_dequant<float, kNVFP4, false>, f);
    return vec ? go(k_mx4_dequant<uint16_t, kNVFP4, true>, h) : go(k_mx4_dequant<uint16_t, kNVFP4, false>, h);
}

}  // extern "C"
