// norm.cu -- RMS norm with the residual's addition and an 8- or 4-bit quantized
// output, and its gradient (all HBM-bound).
//
//   h = x + residual, t = h w, r = 1 / sqrt(mean(h^2) + eps), y = t r
// The row's factor r is positive and common to a row, so it cancels in the
// 8-bit and NVFP4 codes (ratios of t to its row or block maximum) and only
// enters their row scale: one reduction per row yields both sum(h^2) and
// max |t|, and nothing waits for r but the scale.  MXFP4 scales are powers of two of y
// itself, so its codes are those of t r.
#include <algorithm>
#include <cfloat>
#include <mutex>
#include <string>

#include "mx4.cuh"
#include "nq_internal.h"
#include "ptx.cuh"

namespace nq {
namespace {

using namespace dev;

// Quantized output of the forward kernels: the 8-bit formats, the 4-bit ones, none.
enum Out : int { kOutE4M3 = 0, kOutE5M2 = 1, kOutINT8 = 2, kOutMX = 3, kOutNV = 4, kOutNone = 5 };

struct NormArgs {
    const void* x;
    const void* res;     // or NULL
    const void* w;
    void* sum;           // or NULL
    void* y;             // or NULL
    uint8_t* codes;      // or NULL (kOutNone)
    uint8_t* bscales;    // 4-bit block scales
    float* scales;       // per row (8-bit, NVFP4)
    int rows, cols;
    size_t x_stride, res_stride;
    float eps;
    int w_bf16;
};

template <bool VEC>
__device__ __forceinline__ void load_weight8(const void* w, int w_bf16, int v, int cols, float (&f)[8]) {
    if (w_bf16) unpack8<uint16_t>(load_raw8<uint16_t, VEC>(static_cast<const uint16_t*>(w), v, cols), f);
    else unpack8<float>(load_raw8<float, VEC>(static_cast<const float*>(w), v, cols), f);
}

// h = x + residual rounded to the type: the stored value is the one normalized.
template <class In>
__device__ __forceinline__ Raw8<In> add8(const Raw8<In>& x, const Raw8<In>& res) {
    float a[8], b[8];
    unpack8<In>(x, a);
    unpack8<In>(res, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = __fadd_rn(a[e], b[e]);
    return pack8<In>(a);
}

// Sum of `s` and maximum of `m` over the block (every thread gets both).  Two
// buffers used in turn make one barrier per call enough.
__device__ __forceinline__ void block_sum_max(float& s, uint32_t& m, int parity) {
    __shared__ float s_sum[2][32];
    __shared__ uint32_t s_max[2][32];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) {
        s_sum[parity][w] = s;
        s_max[parity][w] = m;
    }
    __syncthreads();
    const int nw = blockDim.x >> 5;
    s = l < nw ? s_sum[parity][l] : 0.0f;
    m = l < nw ? s_max[parity][l] : 0u;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
}

// What a row's reduction gives the encoder.
struct RowNorm {
    float r;      // 1 / rms
    float level;  // 8 bits: qmax / T; NVFP4: A
    bool ok;      // every t of the row is finite
};
template <int OUT>
__device__ __forceinline__ RowNorm row_norm(float sumsq, uint32_t tmax, int cols, float eps, float* scale) {
    RowNorm n;
    n.r = __frsqrt_rn(__fadd_rn(__fdiv_rn(sumsq, static_cast<float>(cols)), eps));
    n.ok = tmax < kInfBits;
    n.level = 0.0f;
    if (OUT <= kOutINT8) {
        constexpr float qmax = FmtTraits<OUT <= kOutINT8 ? OUT : 0>::qmax;
        const float T = fmaxf(__uint_as_float(tmax), 0x1p-110f);
        n.level = __fdiv_rn(qmax, T);
        *scale = !n.ok ? __uint_as_float(0x7FC00000u) : (tmax == 0u ? 1.0f : __fdiv_rn(__fmul_rn(n.r, T), qmax));
    } else if (OUT == kOutNV) {
        n.level = nv_row_level(tmax);
        const float g = nv_row_scale(tmax, n.level);
        *scale = tmax == 0u ? 1.0f : __fmul_rn(n.r, g);
    }
    return n;
}

// Encodes and stores this thread's 8 columns of a row (every lane takes part).
template <class In, int OUT, bool VEC>
__device__ __forceinline__ void emit8(const NormArgs& a, int row, int v, int pitch_words, int words, const float (&t)[8],
                                      const RowNorm& n) {
    if (a.y || OUT == kOutMX) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __fmul_rn(t[e], n.r);
        if (a.y) store_raw8<In, VEC>(static_cast<In*>(a.y) + static_cast<size_t>(row) * a.cols, v, a.cols, pack8<In>(y));
        if (OUT == kOutMX) {
            uint32_t byte;
            const uint32_t c = mx4_encode<kMXFP4>(y, 0.0f, true, &byte);
            mx4_store<kMXFP4>(a.codes + row * mx4_pitch(a.cols), a.bscales, row, v, pitch_words, words, c, byte);
        }
    }
    if (OUT == kOutNV) {
        uint32_t byte;
        const uint32_t c = mx4_encode<kNVFP4>(t, n.level, n.ok, &byte);
        mx4_store<kNVFP4>(a.codes + row * mx4_pitch(a.cols), a.bscales, row, v, pitch_words, words, c, byte);
    }
    if (OUT <= kOutINT8) {
        constexpr int F = OUT <= kOutINT8 ? OUT : 0;
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = ocp_encode2<F>(__fmul_rn(t[2 * i], n.level), __fmul_rn(t[2 * i + 1], n.level));
        uint8_t* o = a.codes + static_cast<size_t>(row) * a.cols + 8 * static_cast<size_t>(v);
        if (VEC) {
            if (8 * v < a.cols) *reinterpret_cast<uint2*>(o) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * v + e < a.cols) o[e] = static_cast<uint8_t>(c[e / 2] >> (8 * (e & 1)));
        }
    }
}

// One block per row in two passes: the reduction, then the encoding of the row
// read again (from sum where it is stored).  Any width and alignment.
template <class In, int OUT, bool VEC>
__global__ void __launch_bounds__(256) k_norm_two_pass(const NormArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int F = OUT == kOutNV ? kNVFP4 : kMXFP4;
    const int nvec = (a.cols + 7) / 8;
    const bool four = OUT == kOutMX || OUT == kOutNV;
    const int words = four ? mx4_words(a.cols, Mx4Traits<F>::block) : 0;
    const int pitch_words = static_cast<int>(mx4_pitch(a.cols) / 4);
    const int nstep = four ? words * Mx4Traits<F>::word_lanes : nvec;
    int parity = 0;
    for (long long rl = blockIdx.x; rl < a.rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = static_cast<const In*>(a.x) + row * a.x_stride;
        const In* res = a.res ? static_cast<const In*>(a.res) + row * a.res_stride : nullptr;
        In* sum = a.sum ? static_cast<In*>(a.sum) + static_cast<size_t>(row) * a.cols : nullptr;
        auto load_h = [&](int v) {
            const Raw8<In> h = load_raw8<In, VEC>(x, v, a.cols);
            return res ? add8<In>(h, load_raw8<In, VEC>(res, v, a.cols)) : h;
        };
        float ss = 0.0f;
        uint32_t tm = 0;
        for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
            const Raw8<In> hr = load_h(v);
            if (sum) store_raw8<In, VEC>(sum, v, a.cols, hr);
            float h[8], w[8];
            unpack8<In>(hr, h);
            load_weight8<VEC>(a.w, a.w_bf16, v, a.cols, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = __fmaf_rn(h[e], h[e], ss);
                w[e] = __fmul_rn(h[e], w[e]);
            }
            tm = max(tm, amax_bits8(w));
        }
        block_sum_max(ss, tm, parity);
        float scale = 0.0f;
        const RowNorm n = row_norm<OUT>(ss, tm, a.cols, a.eps, &scale);
        if (threadIdx.x == 0 && (OUT <= kOutINT8 || OUT == kOutNV)) a.scales[row] = scale;
        for (int v = threadIdx.x; v - static_cast<int>(threadIdx.x & 31) < nstep; v += blockDim.x) {
            float t[8], w[8];
            unpack8<In>(sum ? load_raw8<In, VEC>(sum, v, a.cols) : load_h(v), t);
            load_weight8<VEC>(a.w, a.w_bf16, v, a.cols, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = __fmul_rn(t[e], w[e]);
            emit8<In, OUT, VEC>(a, row, v, pitch_words, words, t, n);
        }
    }
}

// ---- gradient ---------------------------------------------------------------------
struct GradArgs {
    const void* h;
    const void* w;
    const void* dy;
    const void* dsum;  // or NULL
    void* dx;          // or NULL
    int rows, cols;
    size_t h_stride;
    float eps;
    int w_bf16;
};

// Sum of two values over the block.
__device__ __forceinline__ void block_sum2(float& s, float& g, int parity) {
    __shared__ float s_a[2][32], s_b[2][32];
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        g += __shfl_xor_sync(0xffffffffu, g, o);
    }
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) {
        s_a[parity][w] = s;
        s_b[parity][w] = g;
    }
    __syncthreads();
    const int nw = blockDim.x >> 5;
    s = l < nw ? s_a[parity][l] : 0.0f;
    g = l < nw ? s_b[parity][l] : 0.0f;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        g += __shfl_xor_sync(0xffffffffu, g, o);
    }
}

// dx = dsum + r g - h (r^3 mean(g h)), g = dy w, one block per row in two
// passes; r of every row also goes to `rs` for the weight's gradient.
template <class In, bool VEC>
__global__ void __launch_bounds__(256) k_norm_grad_rows(const GradArgs a, float* __restrict__ rs) {
    pdl_launch_dependents();
    pdl_wait();
    const int nvec = (a.cols + 7) / 8;
    int parity = 0;
    for (long long rl = blockIdx.x; rl < a.rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* hp = static_cast<const In*>(a.h) + row * a.h_stride;
        const size_t at = static_cast<size_t>(row) * a.cols;
        const In* dyp = static_cast<const In*>(a.dy) + at;
        float ss = 0.0f, sg = 0.0f;
        for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
            float h[8], g[8], w[8];
            unpack8<In>(load_raw8<In, VEC>(hp, v, a.cols), h);
            unpack8<In>(load_raw8<In, VEC>(dyp, v, a.cols), g);
            load_weight8<VEC>(a.w, a.w_bf16, v, a.cols, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ss = __fmaf_rn(h[e], h[e], ss);
                sg = __fmaf_rn(__fmul_rn(g[e], w[e]), h[e], sg);
            }
        }
        block_sum2(ss, sg, parity);
        const float n = static_cast<float>(a.cols);
        const float r = __frsqrt_rn(__fadd_rn(__fdiv_rn(ss, n), a.eps));
        if (threadIdx.x == 0) rs[row] = r;
        if (!a.dx) continue;
        // c h = r (mean(g n) n) with n = h r, the bounded form: |mean(g n)| <= max |g| sqrt(cols)
        const float c = __fmul_rn(__fdiv_rn(__fmul_rn(sg, r), n), r);
        for (int v = threadIdx.x; v < nvec; v += blockDim.x) {
            float h[8], g[8], w[8];
            unpack8<In>(load_raw8<In, VEC>(hp, v, a.cols), h);
            unpack8<In>(load_raw8<In, VEC>(dyp, v, a.cols), g);
            load_weight8<VEC>(a.w, a.w_bf16, v, a.cols, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = __fmul_rn(r, __fmaf_rn(-h[e], c, __fmul_rn(g[e], w[e])));
            if (a.dsum) {
                float d[8];
                unpack8<In>(load_raw8<In, VEC>(static_cast<const In*>(a.dsum) + at, v, a.cols), d);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[e] = __fadd_rn(g[e], d[e]);
            }
            store_raw8<In, VEC>(static_cast<In*>(a.dx) + at, v, a.cols, pack8<In>(g));
        }
    }
}

// Partial weight gradients: block (x, y) sums dy h r of 256 columns over row
// chunk y, in row order; k_sum_chunks adds the chunks in order.
template <class In>
__global__ void __launch_bounds__(256) k_norm_grad_weight(const GradArgs a, const float* __restrict__ rs, int rows_per_chunk,
                                                          float* __restrict__ part) {
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    const int r0 = blockIdx.y * rows_per_chunk, r1 = min(a.rows, r0 + rows_per_chunk);
    float s = 0.0f;
    for (int row = r0; row < r1; ++row) {
        float h, d;
        if (sizeof(In) == 4) {
            h = static_cast<const float*>(a.h)[row * a.h_stride + c];
            d = static_cast<const float*>(a.dy)[static_cast<size_t>(row) * a.cols + c];
        } else {
            h = bf16_bits_to_f32(static_cast<const uint16_t*>(a.h)[row * a.h_stride + c]);
            d = bf16_bits_to_f32(static_cast<const uint16_t*>(a.dy)[static_cast<size_t>(row) * a.cols + c]);
        }
        s = __fmaf_rn(__fmul_rn(h, rs[row]), d, s);
    }
    part[static_cast<size_t>(blockIdx.y) * a.cols + c] = s;
}
__global__ void __launch_bounds__(256) k_sum_chunks(const float* __restrict__ part, int chunks, int cols, float* __restrict__ dw) {
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int k = 0; k < chunks; ++k) s = __fadd_rn(s, part[static_cast<size_t>(k) * cols + c]);
    dw[c] = s;
}

// ---- host side -------------------------------------------------------------------
nq_status_t bad(const char* who, const char* what) {
    return fail(NQ_ERROR_INVALID_VALUE, std::string(who) + ": " + what);
}

bool strided_ok(size_t stride, size_t esize) { return stride * esize % 16 == 0; }

// Checks a descriptor; x_stride / residual_stride come back with 0 replaced.
nq_status_t check_desc(const char* who, const nq_rmsnorm_desc_t* d, size_t* xs, size_t* rs) {
    if (!d) return bad(who, "null descriptor");
    if (d->rows < 0 || d->cols < 0) return bad(who, "negative size");
    if (d->cols > (1 << 30)) return fail(NQ_ERROR_UNSUPPORTED, std::string(who) + ": more than 2^30 columns");
    if (d->dtype != NQ_F32 && d->dtype != NQ_BF16) return bad(who, "dtype must be NQ_F32 or NQ_BF16");
    if (d->weight_dtype != NQ_F32 && d->weight_dtype != NQ_BF16) return bad(who, "weight_dtype must be NQ_F32 or NQ_BF16");
    if (!(d->eps > 0.0f) || !(d->eps <= FLT_MAX)) return bad(who, "eps must be positive and finite");
    if ((d->x_stride && d->x_stride < d->cols) || (d->residual_stride && d->residual_stride < d->cols))
        return bad(who, "a row stride is smaller than cols");
    *xs = d->x_stride ? d->x_stride : d->cols;
    *rs = d->residual_stride ? d->residual_stride : d->cols;
    return NQ_SUCCESS;
}

template <class In, int OUT, bool VEC>
nq_status_t launch_norm(const NormArgs& a, const DeviceInfo& di, cudaStream_t s, const char* who) {
    const int grid = static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(di.sm_count) * 8));
    return cuda_status(launch_pdl(k_norm_two_pass<In, OUT, VEC>, dim3(grid), dim3(256), 0, s, a), who);
}

template <int OUT>
nq_status_t norm_out(const NormArgs& a, bool bf16, bool vec, const DeviceInfo& di, cudaStream_t s, const char* who) {
    if (bf16) return vec ? launch_norm<uint16_t, OUT, true>(a, di, s, who) : launch_norm<uint16_t, OUT, false>(a, di, s, who);
    return vec ? launch_norm<float, OUT, true>(a, di, s, who) : launch_norm<float, OUT, false>(a, di, s, who);
}

nq_status_t norm_impl(const char* who, const nq_rmsnorm_desc_t* d, const void* x, const void* residual, const void* weight,
                      void* sum, void* y, uint8_t* codes, uint8_t* bscales, float* scales, int out, cudaStream_t s) {
    size_t xs, rs;
    nq_status_t st = check_desc(who, d, &xs, &rs);
    if (st != NQ_SUCCESS) return st;
    if (d->rows == 0 || d->cols == 0) return NQ_SUCCESS;
    if (!x || !weight) return bad(who, "null pointer");
    if (!codes && !y) return bad(who, "neither y nor codes asked for");
    const bool four = out == kOutMX || out == kOutNV;
    if (codes) {
        if (four && !bscales) return bad(who, "codes without block scales");
        if (out != kOutMX && !scales) return bad(who, "codes without row scales");
        if (out == kOutMX && scales) return bad(who, "NQ_MXFP4 has no row scales");
        if (four && (!aligned16(codes) || !aligned16(bscales))) return bad(who, "4-bit codes and scales must be 16-byte aligned");
    } else {
        if (scales || bscales) return bad(who, "scales without codes");
        out = kOutNone;
    }
    if (sum && !residual) return bad(who, "sum without a residual");
    if ((sum && sum == x && xs != static_cast<size_t>(d->cols)) ||
        (sum && sum == residual && rs != static_cast<size_t>(d->cols)))
        return bad(who, "sum in place of a strided tensor");
    if (!aligned_to(x, d->dtype) || !aligned_to(residual, d->dtype) || !aligned_to(sum, d->dtype) || !aligned_to(y, d->dtype) ||
        !aligned_to(weight, d->weight_dtype) || !aligned_to(scales, NQ_F32))
        return bad(who, "a pointer is not aligned to its type");
    if (y && (y == x || y == residual || y == sum)) return bad(who, "y must not be x, residual or sum");
    DeviceInfo di;
    st = current_device(&di);
    if (st != NQ_SUCCESS) return st;
    const size_t es = d->dtype == NQ_BF16 ? 2 : 4;
    const bool vec = d->cols % 8 == 0 && strided_ok(xs, es) && (!residual || strided_ok(rs, es)) && aligned16(x) &&
                     aligned16(residual) && aligned16(weight) && aligned16(sum) && aligned16(y) && aligned16(codes);
    const NormArgs a{x, residual, weight, sum, y, codes, bscales, scales, d->rows, d->cols, xs, rs, d->eps,
                     d->weight_dtype == NQ_BF16};
    const bool bf = d->dtype == NQ_BF16;
    switch (out) {
        case kOutE4M3: return norm_out<kOutE4M3>(a, bf, vec, di, s, who);
        case kOutE5M2: return norm_out<kOutE5M2>(a, bf, vec, di, s, who);
        case kOutINT8: return norm_out<kOutINT8>(a, bf, vec, di, s, who);
        case kOutMX: return norm_out<kOutMX>(a, bf, vec, di, s, who);
        case kOutNV: return norm_out<kOutNV>(a, bf, vec, di, s, who);
        default: return norm_out<kOutNone>(a, bf, vec, di, s, who);
    }
}

template <class In>
nq_status_t grad_impl(const GradArgs& a, float* dw, bool vec, const DeviceInfo& di, cudaStream_t s) {
    const char* who = "nq_rmsnorm_backward";
    const int chunks = static_cast<int>(std::min<long long>(64, a.rows));
    const int per = (a.rows + chunks - 1) / chunks;
    void* scratch = nullptr;
    const size_t rs_bytes = (static_cast<size_t>(a.rows) * 4 + 255) / 256 * 256;
    nq_status_t st = scratch_alloc(&scratch, rs_bytes + static_cast<size_t>(chunks) * a.cols * 4, s);
    if (st != NQ_SUCCESS) return st;
    float* rs = static_cast<float*>(scratch);
    float* part = reinterpret_cast<float*>(static_cast<char*>(scratch) + rs_bytes);
    const int grid = static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(di.sm_count) * 8));
    cudaError_t e = vec ? launch_pdl(k_norm_grad_rows<In, true>, dim3(grid), dim3(256), 0, s, a, rs)
                        : launch_pdl(k_norm_grad_rows<In, false>, dim3(grid), dim3(256), 0, s, a, rs);
    if (e == cudaSuccess && dw) {
        const int cb = (a.cols + 255) / 256;
        e = launch_pdl(k_norm_grad_weight<In>, dim3(cb, chunks), dim3(256), 0, s, a, static_cast<const float*>(rs), per, part);
        if (e == cudaSuccess)
            e = launch_pdl(k_sum_chunks, dim3(cb), dim3(256), 0, s, static_cast<const float*>(part), chunks, a.cols, dw);
    }
    scratch_free(scratch, s);
    return cuda_status(e, who);
}

}  // namespace
}  // namespace nq

extern "C" {

nq_status_t nq_rmsnorm_quantize(const nq_rmsnorm_desc_t* desc, const void* x, const void* residual, const void* weight,
                                void* sum, void* y, uint8_t* codes, float* scales, nq_format_t fmt, nq_stream_t s) {
    if (fmt != NQ_E4M3 && fmt != NQ_E5M2 && fmt != NQ_INT8)
        return nq::fail(NQ_ERROR_INVALID_VALUE, "nq_rmsnorm_quantize: format");
    return nq::norm_impl("nq_rmsnorm_quantize", desc, x, residual, weight, sum, y, codes, nullptr, scales,
                         static_cast<int>(fmt), s);
}

nq_status_t nq_rmsnorm_quantize_mx4(const nq_rmsnorm_desc_t* desc, const void* x, const void* residual, const void* weight,
                                    void* sum, void* y, uint8_t* codes, uint8_t* block_scales, float* row_scales,
                                    nq_mx4_format_t fmt, nq_stream_t s) {
    if (fmt != NQ_MXFP4 && fmt != NQ_NVFP4) return nq::fail(NQ_ERROR_INVALID_VALUE, "nq_rmsnorm_quantize_mx4: format");
    return nq::norm_impl("nq_rmsnorm_quantize_mx4", desc, x, residual, weight, sum, y, codes, block_scales, row_scales,
                         fmt == NQ_MXFP4 ? nq::kOutMX : nq::kOutNV, s);
}

nq_status_t nq_rmsnorm_backward(const nq_rmsnorm_desc_t* desc, const void* h, const void* weight, const void* grad_y,
                                const void* grad_sum, void* grad_x, float* grad_weight, nq_stream_t s) {
    const char* who = "nq_rmsnorm_backward";
    size_t xs, rs;
    nq_status_t st = nq::check_desc(who, desc, &xs, &rs);
    if (st != NQ_SUCCESS) return st;
    if (!grad_x && !grad_weight) return nq::bad(who, "neither grad_x nor grad_weight asked for");
    if (desc->cols == 0) return NQ_SUCCESS;
    if (desc->rows == 0) {
        if (!grad_weight) return NQ_SUCCESS;
        return nq::cuda_status(cudaMemsetAsync(grad_weight, 0, static_cast<size_t>(desc->cols) * 4, s), who);
    }
    if (!h || !weight || !grad_y) return nq::bad(who, "null pointer");
    if (grad_x && (grad_x == h || grad_x == grad_y)) return nq::bad(who, "grad_x must not be h or grad_y");
    if (grad_weight && (grad_weight == weight || grad_weight == grad_x)) return nq::bad(who, "grad_weight must be its own tensor");
    if (!nq::aligned_to(h, desc->dtype) || !nq::aligned_to(grad_y, desc->dtype) || !nq::aligned_to(grad_sum, desc->dtype) ||
        !nq::aligned_to(grad_x, desc->dtype) || !nq::aligned_to(weight, desc->weight_dtype) || !nq::aligned_to(grad_weight, NQ_F32))
        return nq::bad(who, "a pointer is not aligned to its type");
    nq::DeviceInfo di;
    st = nq::current_device(&di);
    if (st != NQ_SUCCESS) return st;
    const bool bf = desc->dtype == NQ_BF16;
    const bool vec = desc->cols % 8 == 0 && nq::strided_ok(xs, bf ? 2 : 4) && nq::aligned16(h) && nq::aligned16(weight) &&
                     nq::aligned16(grad_y) && nq::aligned16(grad_sum) && nq::aligned16(grad_x);
    const nq::GradArgs a{h, weight, grad_y, grad_sum, grad_x, desc->rows, desc->cols, xs, desc->eps,
                         desc->weight_dtype == NQ_BF16};
    return bf ? nq::grad_impl<uint16_t>(a, grad_weight, vec, di, s) : nq::grad_impl<float>(a, grad_weight, vec, di, s);
}

}  // extern "C"
