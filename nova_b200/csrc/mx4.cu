// mx4.cu -- microscaled 4-bit formats: quantize and dequantize (HBM-bound).
//
// Aligned rows with 16 columns a lane: 28672 x 8192 bf16 to MXFP4 96 us, to NVFP4
// 91 us (6.2 and 6.6 TB/s), back to bf16 100 and 104 us (5.9 TB/s); 8192 x 4096
// 15.0 and 15.5 us.  With 8 columns a lane NVFP4 took 113 us and the way back 116.
// Unaligned rows move one column a lane (16384 x 4111 bf16 to NVFP4 55 us).
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

template <bool VEC>
__device__ __forceinline__ uint8_t* warp_buf() {
    if constexpr (VEC) {
        return nullptr;
    } else {
        __shared__ uint4 s_buf[32 * kWarpBuf / 16];
        return reinterpret_cast<uint8_t*>(s_buf) + (threadIdx.x >> 5) * kWarpBuf;
    }
}

// One block per row; NVFP4 reads the row twice (its maximum first).  For rows too wide for k_mx4_quant.
template <class In, int F, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx4_quant_wide(const In* __restrict__ src, size_t ld, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ bscales, float* __restrict__ rscales,
                                                             int rows, int cols) {
    pdl_launch_dependents();
    pdl_wait();
    uint8_t* buf = warp_buf<VEC>();
    const int nvec = (cols + 7) / 8;
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int nstep = words * Mx4Traits<F>::word_lanes;
    const int lane = lane_of();
    int parity = 0;
    for (long long rl = blockIdx.x; rl < rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = src + row * ld;
        const Mx4Row to = mx4_row(codes, bscales, row, cols, words);
        NvRow nr{};
        if (F == kNVFP4) {
            uint32_t m = 0;
            for (int v = threadIdx.x; v - lane < nvec; v += kThreads)
                m = max(m, amax_bits_raw<In>(load_vec<In, VEC>(x, v, cols, buf)));
            m = block_umax(m, parity);
            nr = nv_row(m);
            if (threadIdx.x == 0) rscales[row] = nv_row_scale(m, nr.level);
        }
        for (int v = threadIdx.x; v - lane < nstep; v += kThreads) {
            const Raw8<In> r = load_vec<In, VEC>(x, v, cols, buf);
            uint32_t byte;
            const uint32_t c = mx4_encode<F, sizeof(In) == 4>(unpack8<In>(r), amax_bits_raw<In>(r), nr, &byte);
            mx4_store<F>(to, v, c, byte);
        }
    }
}

// Rows held in registers, NV vectors of 8 columns a thread, by one warp (WARP) or
// one block; each row is read once.
template <class In, int F, bool VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_mx4_quant(const In* __restrict__ src, size_t ld,
                                                                 uint8_t* __restrict__ codes, uint8_t* __restrict__ bscales,
                                                                 float* __restrict__ rscales, int rows, int cols) {
    pdl_launch_dependents();
    uint8_t* buf = warp_buf<VEC>();
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int width = WARP ? 32 : blockDim.x;
    const int t0 = WARP ? lane_of() : threadIdx.x;
    const int per = WARP ? blockDim.x >> 5 : 1;
    pdl_wait();
    int parity = 0;
    for (long long rl = static_cast<long long>(blockIdx.x) * per + (WARP ? threadIdx.x >> 5 : 0); rl < rows;
         rl += static_cast<long long>(gridDim.x) * per, parity ^= 1) {
        const int row = static_cast<int>(rl);
        Raw8<In> x[NV];
        load_vecs<In, VEC, NV>(x, src + row * ld, t0, width, cols, buf);
        const Mx4Row to = mx4_row(codes, bscales, row, cols, words);
        uint32_t am[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) am[i] = amax_bits_raw<In>(x[i]);
        NvRow nr{};
        if (F == kNVFP4) {
            uint32_t m = am[0];
#pragma unroll
            for (int i = 1; i < NV; ++i) m = max(m, am[i]);
            m = WARP ? __reduce_max_sync(0xffffffffu, m) : block_umax(m, parity);
            nr = nv_row(m);
            if (t0 == 0) rscales[row] = nv_row_scale(m, nr.level);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            uint32_t byte;
            const uint32_t c = mx4_encode<F, sizeof(In) == 4>(unpack8<In>(x[i]), am[i], nr, &byte);
            mx4_store<F>(to, t0 + i * width, c, byte);
        }
    }
}

// The same with 16 columns a lane: NV of them, by one warp or one block.
template <class In, int F, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_mx4_quant16(const In* __restrict__ src, size_t ld,
                                                                   uint8_t* __restrict__ codes, uint8_t* __restrict__ bscales,
                                                                   float* __restrict__ rscales, int rows, int cols) {
    pdl_launch_dependents();
    constexpr int WL = F == kNVFP4 ? 4 : 8;  // lanes in a word of 4 scales
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int nvec = cols / 16;
    const int width = WARP ? 32 : blockDim.x;
    const int t0 = WARP ? lane_of() : threadIdx.x;
    const int per = WARP ? blockDim.x >> 5 : 1;
    // few rows: their first bytes to L2 (which is coherent) while the kernel before ends (with a 1 x 8192 x
    // 8192 product behind it 14.3 -> 13.4 us)
    if (NV == 1 && !WARP && blockIdx.x < rows && t0 < nvec) prefetch_l2(src + blockIdx.x * ld + 16 * t0);
    pdl_wait();
    int parity = 0;
    for (long long rl = static_cast<long long>(blockIdx.x) * per + (WARP ? threadIdx.x >> 5 : 0); rl < rows;
         rl += static_cast<long long>(gridDim.x) * per, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* p = src + row * ld;
        Raw16<In> x[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = t0 + i * width;
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j)
                x[i].q[j] = v < nvec ? ld_global_32(p + 16 * static_cast<size_t>(v) + 8 * j) : Word32{};
        }
        const Mx4Row to = mx4_row(codes, bscales, row, cols, words);
        uint32_t am[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) am[i] = max(amax_bits_raw<In>(half_of<In>(x[i], 0)), amax_bits_raw<In>(half_of<In>(x[i], 1)));
        NvRow nr{};
        if (F == kNVFP4) {
            uint32_t m = am[0];
#pragma unroll
            for (int i = 1; i < NV; ++i) m = max(m, am[i]);
            m = WARP ? __reduce_max_sync(0xffffffffu, m) : block_umax(m, parity);
            nr = nv_row(m);
            if (t0 == 0) rscales[row] = nv_row_scale(m, nr.level);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = t0 + i * width;
            if (F == kMXFP4) am[i] = max(am[i], __shfl_xor_sync(0xffffffffu, am[i], 1));
            const Mx4Block k = mx4_block<F, sizeof(In) == 4>(am[i], nr);
            if (v < nvec)
                reinterpret_cast<uint2*>(to.codes)[v] = make_uint2(mx4_codes8<F, sizeof(In) == 4>(unpack8<In>(half_of<In>(x[i], 0)), k),
                                                                   mx4_codes8<F, sizeof(In) == 4>(unpack8<In>(half_of<In>(x[i], 1)), k));
            // columns up to a whole 32 are zero; MXFP4's last half block pairs with nothing
            else if (2 * v < to.pitch_words) reinterpret_cast<uint2*>(to.codes)[v] = make_uint2(0u, 0u);
            uint32_t w = k.byte | (__shfl_down_sync(0xffffffffu, k.byte, WL / 4) << 8);
            w |= __shfl_down_sync(0xffffffffu, w, WL / 2) << 16;
            if (v % WL == 0 && v / WL < words) *reinterpret_cast<uint32_t*>(to.scales + static_cast<size_t>(v / WL) * 512) = w;
        }
    }
}

template <class T, int F>
__global__ void __launch_bounds__(kThreads) k_mx4_dequant16(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ bscales,
                                                            const float* __restrict__ rscales, T* __restrict__ dst, int rows,
                                                            int cols, int width) {
    pdl_launch_dependents();
    constexpr int L = F == kNVFP4 ? 1 : 2;  // lanes in a block
    const int nvec = cols / 16;
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int t0 = threadIdx.x % width;
    const int per = blockDim.x / width;
    pdl_wait();
    for (long long rl = static_cast<long long>(blockIdx.x) * per + threadIdx.x / width; rl < rows;
         rl += static_cast<long long>(gridDim.x) * per) {
        const int row = static_cast<int>(rl);
        const float g = rscales ? __ldg(rscales + row) : 1.0f;
        const uint2* code = reinterpret_cast<const uint2*>(codes + row * mx4_pitch(cols));
        const uint8_t* scale = bscales + mx4_scale_offset(row, 0, words);
        T* out = dst + static_cast<size_t>(row) * cols;
        for (int v0 = t0; v0 < nvec; v0 += 4 * width) {
            uint2 c[4];
            uint32_t s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = v0 + i * width, b = v / L;
                c[i] = v < nvec ? __ldg(code + v) : make_uint2(0u, 0u);
                s[i] = v < nvec ? __ldg(scale + static_cast<size_t>(b / 4) * 512 + b % 4) : 0u;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = v0 + i * width;
                if (v >= nvec) break;
                const float sv = mx4_scale_value(F, s[i]);
                F8 f[2];
                e2m1_decode8(c[i].x, f[0]);
                e2m1_decode8(c[i].y, f[1]);
                Word32 o[sizeof(T) / 2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[h].p[j] = mul2(f[h].p[j], both(sv));
                        if (rscales) f[h].p[j] = mul2(f[h].p[j], both(g));
                        if constexpr (sizeof(T) == 2) {
                            o[0].w[4 * h + j] = f32x2_to_bf16x2(f[h].p[j].x, f[h].p[j].y);
                        } else {
                            o[h].w[2 * j] = __float_as_uint(f[h].p[j].x);
                            o[h].w[2 * j + 1] = __float_as_uint(f[h].p[j].y);
                        }
                    }
                }
#pragma unroll
                for (int h = 0; h < static_cast<int>(sizeof(T) / 2); ++h) st_global_32(out + 16 * static_cast<size_t>(v) + 8 * h, o[h]);
            }
        }
    }
}

// `width` threads a row, four vectors a thread in flight.
template <class T, int F, bool VEC>
__global__ void __launch_bounds__(kThreads) k_mx4_dequant(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ bscales,
                                                          const float* __restrict__ rscales, T* __restrict__ dst, int rows,
                                                          int cols, int width) {
    pdl_launch_dependents();
    uint8_t* buf = warp_buf<VEC>();
    constexpr int L = Mx4Traits<F>::block_lanes;
    const int nvec = (cols + 7) / 8;
    const int words = mx4_words(cols, Mx4Traits<F>::block);
    const int t0 = threadIdx.x % width;
    const int per = blockDim.x / width;
    pdl_wait();
    for (long long rl = static_cast<long long>(blockIdx.x) * per + threadIdx.x / width; rl < rows;
         rl += static_cast<long long>(gridDim.x) * per) {
        const int row = static_cast<int>(rl);
        const float g = rscales ? __ldg(rscales + row) : 1.0f;
        const uint32_t* code = reinterpret_cast<const uint32_t*>(codes + row * mx4_pitch(cols));
        const uint8_t* scale = bscales + mx4_scale_offset(row, 0, words);
        T* out = dst + static_cast<size_t>(row) * cols;
        for (int v0 = t0; v0 - lane_of() < nvec; v0 += 4 * width) {
            uint32_t c[4], s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = v0 + i * width, b = v / L;
                c[i] = v < nvec ? __ldg(code + v) : 0u;
                s[i] = v < nvec ? __ldg(scale + static_cast<size_t>(b / 4) * 512 + b % 4) : 0u;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                F8 f;
                e2m1_decode8(c[i], f);
                const float sv = mx4_scale_value(F, s[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f.p[j] = mul2(f.p[j], both(sv));
                    if (rscales) f.p[j] = mul2(f.p[j], both(g));
                }
                store_vec<T, VEC>(out, v0 + i * width, cols, pack8<T>(f), buf);
            }
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

struct QuantArgs {
    size_t ld;
    uint8_t* codes;
    uint8_t* bscales;
    float* rscales;
    int rows, cols;
};

template <class In, int F, bool VEC, int NV, bool WARP>
nq_status_t launch_quant(const In* src, const QuantArgs& a, int threads, const DeviceInfo& di, cudaStream_t s) {
    auto kern = k_mx4_quant<In, F, VEC, NV, WARP>;
    const long long blocks = WARP ? (static_cast<long long>(a.rows) + threads / 32 - 1) / (threads / 32) : a.rows;
    const int grid = persistent_grid(kern, threads, 0, blocks, di);
    return cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), 0, s, src, a.ld, a.codes, a.bscales, a.rscales, a.rows, a.cols),
                       "nq_quantize_rows_mx4");
}

template <class In, int F, int NV, bool WARP>
nq_status_t launch_quant16(const In* src, const QuantArgs& a, int threads, const DeviceInfo& di, cudaStream_t s) {
    auto kern = k_mx4_quant16<In, F, NV, WARP>;
    const long long blocks = WARP ? (static_cast<long long>(a.rows) + threads / 32 - 1) / (threads / 32) : a.rows;
    const int grid = persistent_grid(kern, threads, 0, blocks, di);
    return cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), 0, s, src, a.ld, a.codes, a.bscales, a.rscales, a.rows, a.cols),
                       "nq_quantize_rows_mx4");
}

template <class In, int F, bool VEC>
nq_status_t quant_impl(const void* p, const QuantArgs& a, const DeviceInfo& di, cudaStream_t s) {
    constexpr int NVMAX = sizeof(In) == 2 ? 4 : 2;  // 64 bytes a thread
    const In* src = static_cast<const In*>(p);
    const int nvec = mx4_words(a.cols, Mx4Traits<F>::block) * Mx4Traits<F>::word_lanes;  // whole scale words
    if (VEC && a.cols % 16 == 0 && a.ld * sizeof(In) % 32 == 0 && reinterpret_cast<uintptr_t>(p) % 32 == 0) {
        constexpr int NV16 = sizeof(In) == 2 ? 2 : 1;  // 64 bytes a thread
        const int n16 = nvec / 2;
        // (below 32 of them lanes would idle: 65536 x 256 bf16 18.2 us against 10.1 with 8 columns a lane)
        if (n16 < 32 && nvec <= 32) return launch_quant<In, F, VEC, 1, true>(src, a, 256, di, s);
        if (n16 <= 32 * NV16) return launch_quant16<In, F, NV16, true>(src, a, 256, di, s);
        if (a.rows < 2 * di.sm_count && n16 <= 1024) return launch_quant16<In, F, 1, false>(src, a, (n16 + 31) / 32 * 32, di, s);
        const int threads16 = ((n16 + NV16 - 1) / NV16 + 31) / 32 * 32;
        if (threads16 <= 1024) return launch_quant16<In, F, NV16, false>(src, a, threads16, di, s);
    }
    if (nvec <= 32) return launch_quant<In, F, VEC, 1, true>(src, a, 256, di, s);
    if (nvec <= 32 * NVMAX) return launch_quant<In, F, VEC, NVMAX, true>(src, a, 256, di, s);
    if (a.rows < 2 * di.sm_count && nvec <= 1024) return launch_quant<In, F, VEC, 1, false>(src, a, (nvec + 31) / 32 * 32, di, s);
    // the most vectors a thread, or half of them where that leaves fewer lanes idle
    auto lanes = [&](int nv) { return ((nvec + nv - 1) / nv + 31) / 32 * 32; };
    const int threads = lanes(NVMAX), half = lanes(NVMAX / 2);
    if (half <= 512 && half * (NVMAX / 2) < threads * NVMAX) return launch_quant<In, F, VEC, NVMAX / 2, false>(src, a, half, di, s);
    if (threads <= 1024) return launch_quant<In, F, VEC, NVMAX, false>(src, a, threads, di, s);
    const int grid = static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(di.sm_count) * 8));
    return cuda_status(launch_pdl(k_mx4_quant_wide<In, F, VEC>, dim3(grid), dim3(kThreads), 0, s, src, a.ld, a.codes, a.bscales,
                                  a.rscales, a.rows, a.cols),
                       "nq_quantize_rows_mx4 (wide)");
}

template <class T, int F>
nq_status_t dequant_impl(const uint8_t* codes, const uint8_t* bscales, const float* rscales, void* dst, int rows, int cols,
                         bool vec, const DeviceInfo& di, cudaStream_t s) {
    // `width` lanes a row with four vectors each (few rows: one each), as many rows as make a block of
    // up to 256 threads
    auto go = [&](auto kern, int nvec) {
        const int width = std::min(kThreads, rows < 2 * di.sm_count ? (nvec + 31) / 32 * 32 : (nvec + 127) / 128 * 32);
        const int per = kThreads / width;
        const long long blocks = (static_cast<long long>(rows) + per - 1) / per;
        const int grid = static_cast<int>(std::min<long long>(blocks, static_cast<long long>(di.sm_count) * 8));
        return cuda_status(launch_pdl(kern, dim3(grid), dim3(width * per), 0, s, codes, bscales, rscales, static_cast<T*>(dst), rows,
                                      cols, width),
                           "nq_dequantize_rows_mx4");
    };
    if (cols % 16 == 0 && reinterpret_cast<uintptr_t>(dst) % 32 == 0) return go(k_mx4_dequant16<T, F>, cols / 16);
    return go(vec ? k_mx4_dequant<T, F, true> : k_mx4_dequant<T, F, false>, (cols + 7) / 8);
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
    const nq::QuantArgs a{ld, codes, block_scales, row_scales, rows, cols};
    using namespace nq;
    if (fmt == NQ_MXFP4) {
        if (src_dtype == NQ_F32) return vec ? quant_impl<float, kMXFP4, true>(src, a, di, s) : quant_impl<float, kMXFP4, false>(src, a, di, s);
        return vec ? quant_impl<uint16_t, kMXFP4, true>(src, a, di, s) : quant_impl<uint16_t, kMXFP4, false>(src, a, di, s);
    }
    if (src_dtype == NQ_F32) return vec ? quant_impl<float, kNVFP4, true>(src, a, di, s) : quant_impl<float, kNVFP4, false>(src, a, di, s);
    return vec ? quant_impl<uint16_t, kNVFP4, true>(src, a, di, s) : quant_impl<uint16_t, kNVFP4, false>(src, a, di, s);
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
    using namespace nq;
    if (fmt == NQ_MXFP4)
        return dst_dtype == NQ_F32 ? dequant_impl<float, kMXFP4>(codes, block_scales, row_scales, dst, rows, cols, vec, di, s)
                                   : dequant_impl<uint16_t, kMXFP4>(codes, block_scales, row_scales, dst, rows, cols, vec, di, s);
    return dst_dtype == NQ_F32 ? dequant_impl<float, kNVFP4>(codes, block_scales, row_scales, dst, rows, cols, vec, di, s)
                               : dequant_impl<uint16_t, kNVFP4>(codes, block_scales, row_scales, dst, rows, cols, vec, di, s);
}

}  // extern "C"
