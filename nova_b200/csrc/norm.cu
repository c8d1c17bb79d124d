// norm.cu -- RMS norm with the residual's addition and an 8- or 4-bit quantized
// output, and its gradient (all HBM-bound).
//
//   h = x + residual, t = h w, r = 1 / sqrt(mean(h^2) + eps), y = t r
// The row's factor r is positive and common to a row, so it cancels in the
// 8-bit and NVFP4 codes (ratios of t to its row or block maximum) and only
// enters their row scale: one reduction per row yields both sum(h^2) and
// max |t|, and nothing waits for r but the scale.  MXFP4 scales are powers of two of y
// itself, so its codes are those of t r.
//
// Which kernel: rows in registers (k_norm_rows: a warp or a block a row); many
// aligned rows through a bulk-copy ring (k_norm_ring: 16384 x 8192 bf16 with
// residual, E4M3: 153 us, 6.1 TB/s, against 165 from registers, in a graph of passes; to NVFP4 237, bound
// by the encode's arithmetic; 16384 columns lose by it, 298 against 285); dense rows of odd widths cut where
// memory is (k_norm_cut: 16384 x 5003 bf16 120 us against 187); rows too wide for
// registers in two passes.  One row: 2.7 us a launch in a graph.  The gradient: 8192 x 4096
// bf16 51 us (5.2 TB/s), of which the partial rows' sum takes 4.5; 4096 x 16384 bf16 160, fp32 326.
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
    float eps, inv_cols;
    int w_kind;  // bit 0: bf16, bit 1: 16-byte aligned
    int shift0;  // columns from a boundary of 8 to row 0 where all tensors agree on it, else -1 (k_norm_cut)
};

// The warp's buffer for rows that are not aligned (one kWarpBuf per warp).
template <bool VEC>
__device__ __forceinline__ uint8_t* warp_buf() {
    if constexpr (VEC) {
        return nullptr;
    } else {
        __shared__ uint4 s_buf[32 * kWarpBuf / 16];
        return reinterpret_cast<uint8_t*>(s_buf) + (threadIdx.x >> 5) * kWarpBuf;
    }
}

// Columns [8v, 8v + 8) of the weight; a vector starts on a 16-byte boundary
// wherever the weight itself does, whatever the rows do (w_vec).
template <class W>
__device__ __forceinline__ F8 load_weight8_of(const W* w, bool w_vec, int v, int cols) {
    if (w_vec && 8 * v + 8 <= cols) {
        Raw8<W> r;
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(W) / 2); ++j)
            r.q[j] = __ldg(reinterpret_cast<const uint4*>(w + 8 * static_cast<size_t>(v)) + j);
        return unpack8<W>(r);
    }
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = 8 * v + e;
        f[e] = c >= cols ? 0.0f : (sizeof(W) == 4 ? __ldg(reinterpret_cast<const float*>(w) + c)
                                                  : bf16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t*>(w) + c)));
    }
    return F8{{{f[0], f[1]}, {f[2], f[3]}, {f[4], f[5]}, {f[6], f[7]}}};
}
__device__ __forceinline__ F8 load_weight8(const void* w, int w_kind, int v, int cols) {
    return (w_kind & 1) ? load_weight8_of(static_cast<const uint16_t*>(w), w_kind & 2, v, cols)
                        : load_weight8_of(static_cast<const float*>(w), w_kind & 2, v, cols);
}

// h = x + residual rounded to the type: the stored value is the one normalized.
template <class In>
__device__ __forceinline__ Raw8<In> add8(const Raw8<In>& x, const Raw8<In>& res) {
    F8 a = unpack8<In>(x);
    const F8 b = unpack8<In>(res);
#pragma unroll
    for (int i = 0; i < 4; ++i) a.p[i] = add2(a.p[i], b.p[i]);
    return pack8<In>(a);
}
// t = h w; ss += h^2, tm = max(tm, |t|).
__device__ __forceinline__ F8 row_terms(const F8& h, const F8& w, float2& ss, uint32_t& tm) {
    F8 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ss = fma2(h.p[i], h.p[i], ss);
        t.p[i] = mul2(h.p[i], w.p[i]);
    }
    tm = max(tm, amax_bits8(t));
    return t;
}

// Sum of `s` and maximum of `m` over the block (every thread gets both).  Two
// buffers used in turn make one barrier per call enough.
__device__ __forceinline__ void block_sum_max(float& s, uint32_t& m, int parity) {
    __shared__ float s_sum[2][32];
    __shared__ uint32_t s_max[2][32];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = __reduce_max_sync(0xffffffffu, m);
    const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
    if (l == 0) {
        s_sum[parity][w] = s;
        s_max[parity][w] = m;
    }
    __syncthreads();
    const int nw = blockDim.x >> 5;
    s = l < nw ? s_sum[parity][l] : 0.0f;
    m = __reduce_max_sync(0xffffffffu, l < nw ? s_max[parity][l] : 0u);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
}

// What a row's reduction gives the encoder.
struct RowNorm {
    float r;             // 1 / rms (where it is needed: y, MXFP4)
    float mul, tn, inv;  // 8 bits: qmax p and T p for a power of two p, and the reciprocal of T p
    NvRow nv;            // NVFP4
};
__device__ __forceinline__ float row_r(float sumsq, float inv_cols, float eps) {
    return rsqrtf(__fmaf_rn(sumsq, inv_cols, eps));
}
// The quotient t qmax / T of an 8-bit code: numerator rounded (exact for bf16 tensors), then a
// product with the reciprocal, its remainder, one correction: the quotient correctly
// rounded.  (Quotients of bf16 products are ratios of small integers and fall on
// rounding borders; the product alone puts them to either side.)
// Numerator and denominator carry a power of two by the row's T: 2^-16 from 1 on, so that
// |t| qmax 2^-16 <= 0.875 T whatever the format, and 2^32 below, so that neither the numerator of a code
// that is not zero nor a remainder is subnormal (T >= 2^-110).
__device__ __forceinline__ float2 code_quotient(float2 t, const RowNorm& n) {
    const float2 num = mul2(t, both(n.mul));
    const float2 q = mul2(num, both(n.inv));
    return fma2(fma2(q, both(-n.tn), num), both(n.inv), q);
}
// Row scales of the 8-bit formats and of NVFP4 (tmax: magnitude bits of the largest t).
template <int F>
__device__ __forceinline__ float row_scale8(float r, uint32_t tmax) {
    if (tmax >= kInfBits) return __uint_as_float(0x7FC00000u);
    return tmax == 0u ? 1.0f : __fdiv_rn(__fmul_rn(r, fmaxf(__uint_as_float(tmax), 0x1p-110f)), FmtTraits<F>::qmax);
}
__device__ __forceinline__ float row_scale_nv(float r, uint32_t tmax, float level) {
    return tmax == 0u ? 1.0f : __fmul_rn(r, nv_row_scale(tmax, level));
}
// `first`: this thread stores the row's scale (the only place, besides y and
// MXFP4, where r and its divisions are needed).
template <int OUT>
__device__ __forceinline__ RowNorm row_norm(const NormArgs& a, int row, float sumsq, uint32_t tmax, bool first) {
    RowNorm n{};
    if (a.y || OUT == kOutMX) n.r = row_r(sumsq, a.inv_cols, a.eps);
    if (OUT <= kOutINT8) {
        constexpr float qmax = FmtTraits<OUT <= kOutINT8 ? OUT : 0>::qmax;
        const float T = fmaxf(__uint_as_float(tmax), 0x1p-110f);
        const float p = T < 1.0f ? 0x1p32f : 0x1p-16f;
        n.mul = qmax * p;
        n.tn = T * p;
        n.inv = __frcp_rn(n.tn);
        if (first) a.scales[row] = row_scale8<OUT <= kOutINT8 ? OUT : 0>(row_r(sumsq, a.inv_cols, a.eps), tmax);
    } else if (OUT == kOutNV) {
        n.nv = nv_row(tmax);
        if (first) a.scales[row] = row_scale_nv(row_r(sumsq, a.inv_cols, a.eps), tmax, n.nv.level);
    }
    return n;
}

constexpr float kFar = 0x1p-80f;
// Rows whose sum(h^2) is out of fp32's range (a finite |h| from 1.8e19 on may do that): what
// depends on r -- the row scale, y, MXFP4 codes -- once more, with the sum of (h 2^-80)^2, which
// 2^30 finite columns keep in range.  The other codes are right as they are.  A block or warp
// that met such a row does this for all its rows when it is through with them: inside the loop over
// rows it cost the kernels up to 17%.  (A sum within a factor of two of the border is taken here
// too: the same r but for rounding.)  One such row among 16384 x 8192 bf16: 438 us for 153; a NaN,
// whose r is a NaN already, costs nothing.  h comes from sum where that is stored, which may have
// taken the place of an input.
template <class In, int OUT, bool WARP>
__device__ __forceinline__ void redo_far_rows_of(const NormArgs& a, long long first, long long step, int t0, int width) {
    auto value = [](const In* p, int c) {
        if constexpr (sizeof(In) == 4) return p[c];
        else return bf16_bits_to_f32(p[c]);
    };
    auto weight = [&](int c) {
        return (a.w_kind & 1) ? bf16_bits_to_f32(static_cast<const uint16_t*>(a.w)[c]) : static_cast<const float*>(a.w)[c];
    };
    if (WARP) __syncwarp();
    else __syncthreads();
    int parity = 0;
    for (long long rl = first; rl < a.rows; rl += step, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = a.sum ? static_cast<const In*>(a.sum) + static_cast<size_t>(row) * a.cols
                            : static_cast<const In*>(a.x) + row * a.x_stride;
        const In* res = a.res && !a.sum ? static_cast<const In*>(a.res) + row * a.res_stride : nullptr;
        auto load_h = [&](int c) {
            float h = value(x, c);
            if (res) h = __fadd_rn(h, value(res, c));
            if (res && sizeof(In) == 2) h = bf16_bits_to_f32(f32x2_to_bf16x2(h, 0.0f) & 0xFFFFu);
            return h;
        };
        float s = 0.0f;
        uint32_t tm = 0;
#pragma unroll 4
        for (int c = t0; c < a.cols; c += width) {
            const float h = load_h(c), hs = __fmul_rn(h, kFar);
            s = __fmaf_rn(hs, hs, s);
            tm = max(tm, __float_as_uint(__fmul_rn(h, weight(c))) & 0x7FFFFFFFu);
        }
        if (WARP) {
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            tm = __reduce_max_sync(0xffffffffu, tm);
        } else {
            block_sum_max(s, tm, parity);
        }
        if (s < 0.5f * FLT_MAX * kFar * kFar) continue;
        const float r = kFar * row_r(s, a.inv_cols, a.eps * kFar * kFar);
        if (t0 == 0) {
            if (OUT <= kOutINT8) a.scales[row] = row_scale8<OUT <= kOutINT8 ? OUT : 0>(r, tm);
            if (OUT == kOutNV) a.scales[row] = row_scale_nv(r, tm, nv_row(tm).level);
        }
        if (a.y) {
            In* y = static_cast<In*>(a.y) + static_cast<size_t>(row) * a.cols;
#pragma unroll 1
            for (int c = t0; c < a.cols; c += width) {
                const float v = __fmul_rn(__fmul_rn(load_h(c), weight(c)), r);
                if constexpr (sizeof(In) == 4) y[c] = v;
                else y[c] = static_cast<uint16_t>(f32x2_to_bf16x2(v, 0.0f));
            }
        }
        if (OUT == kOutMX) {
            const Mx4Row to = mx4_row(a.codes, a.bscales, row, a.cols, mx4_words(a.cols, 32));
#pragma unroll 1
            for (int b = t0; 32 * b < a.cols; b += width) {
                auto y8 = [&](int q) {  // columns [32 b + 8 q, + 8)
                    float e[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int c = 32 * b + 8 * q + k;
                        e[k] = c < a.cols ? __fmul_rn(__fmul_rn(load_h(c), weight(c)), r) : 0.0f;
                    }
                    return F8{{{e[0], e[1]}, {e[2], e[3]}, {e[4], e[5]}, {e[6], e[7]}}};
                };
                uint32_t m = 0;
#pragma unroll 1
                for (int q = 0; q < 4; ++q) m = max(m, amax_bits8(y8(q)));
                const Mx4Block k = mx4_block<kMXFP4, false>(m, NvRow{});
#pragma unroll 1
                for (int q = 0; q < 4; ++q) to.codes[4 * b + q] = mx4_codes8<kMXFP4, false>(y8(q), k);
                to.scales[static_cast<size_t>(b / 4) * 512 + b % 4] = static_cast<uint8_t>(k.byte);
            }
        }
    }
}

// Called or inline, as the loop before it compiles better: 65536 x 203 bf16 to E4M3 50 us called, 57
// inline; 65536 x 1024 bf16 to MXFP4 84 called, 73 inline.
template <class In, int OUT, bool WARP>
__device__ __noinline__ void redo_far_call(const NormArgs& a, long long first, long long step, int t0, int width) {
    redo_far_rows_of<In, OUT, WARP>(a, first, step, t0, width);
}
template <class In, int OUT, bool WARP>
__device__ __forceinline__ void redo_far_rows(const NormArgs& a, long long first, long long step, int t0, int width) {
    if (OUT == kOutMX) redo_far_rows_of<In, OUT, WARP>(a, first, step, t0, width);
    else redo_far_call<In, OUT, WARP>(a, first, step, t0, width);
}

// Encodes and stores this thread's 8 columns of a row (every lane takes part).
template <class In, int OUT, bool VEC>
__device__ __forceinline__ void emit8(const NormArgs& a, int row, int v, const Mx4Row& to, const F8& t, const RowNorm& n, uint8_t* buf) {
    if (a.y || OUT == kOutMX) {
        F8 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.p[i] = mul2(t.p[i], both(n.r));
        if (a.y) store_vec<In, VEC>(static_cast<In*>(a.y) + static_cast<size_t>(row) * a.cols, v, a.cols, pack8<In>(y), buf);
        if (OUT == kOutMX) {
            uint32_t byte;
            const uint32_t c = mx4_encode<kMXFP4, false>(y, amax_bits8(y), n.nv, &byte);
            mx4_store<kMXFP4>(to, v, c, byte);
        }
    }
    if (OUT == kOutNV) {
        uint32_t byte;
        const uint32_t c = mx4_encode<kNVFP4, true>(t, amax_bits8(t), n.nv, &byte);
        mx4_store<kNVFP4>(to, v, c, byte);
    }
    if (OUT <= kOutINT8) {
        constexpr int F = OUT <= kOutINT8 ? OUT : 0;
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 q = code_quotient(t.p[i], n);
            c[i] = ocp_encode2<F>(q.x, q.y);
        }
        store_codes8<VEC>(a.codes + static_cast<size_t>(row) * a.cols, v, a.cols, make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16)), buf);
    }
}

// One block per row in two passes: the reduction, then the encoding of the row
// read again (from sum where it is stored).  For rows too wide for k_norm_rows.
template <class In, int OUT, bool VEC>
__global__ void __launch_bounds__(256) k_norm_two_pass(const __grid_constant__ NormArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    uint8_t* buf = warp_buf<VEC>();
    constexpr int F = OUT == kOutNV ? kNVFP4 : kMXFP4;
    const int nvec = (a.cols + 7) / 8;
    const bool four = OUT == kOutMX || OUT == kOutNV;
    const int words = four ? mx4_words(a.cols, Mx4Traits<F>::block) : 0;
    const int nstep = four ? words * Mx4Traits<F>::word_lanes : nvec;
    const int lane = lane_of();
    int parity = 0;
    bool far = false;  // some row's sum(h^2) left fp32's range
    for (long long rl = blockIdx.x; rl < a.rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = static_cast<const In*>(a.x) + row * a.x_stride;
        const In* res = a.res ? static_cast<const In*>(a.res) + row * a.res_stride : nullptr;
        In* sum = a.sum ? static_cast<In*>(a.sum) + static_cast<size_t>(row) * a.cols : nullptr;
        auto load_h = [&](int v) {
            const Raw8<In> h = load_vec<In, VEC>(x, v, a.cols, buf);
            return res ? add8<In>(h, load_vec<In, VEC>(res, v, a.cols, buf)) : h;
        };
        float2 s2 = both(0.0f);
        uint32_t tm = 0;
        for (int v = threadIdx.x; v - lane < nvec; v += blockDim.x) {
            const Raw8<In> hr = load_h(v);
            if (sum) store_vec<In, VEC>(sum, v, a.cols, hr, buf);
            (void)row_terms(unpack8<In>(hr), load_weight8(a.w, a.w_kind, v, a.cols), s2, tm);
        }
        float ss = s2.x + s2.y;
        block_sum_max(ss, tm, parity);  // (its barrier also orders the unaligned rows' stores before the loads below)
        const Mx4Row to = four ? mx4_row(a.codes, a.bscales, row, a.cols, words) : Mx4Row{};
        far |= ss > FLT_MAX;
        const RowNorm n = row_norm<OUT>(a, row, ss, tm, threadIdx.x == 0);
        for (int v = threadIdx.x; v - lane < nstep; v += blockDim.x) {
            F8 t = unpack8<In>(sum ? load_vec<In, VEC>(sum, v, a.cols, buf) : load_h(v));
            const F8 w = load_weight8(a.w, a.w_kind, v, a.cols);
#pragma unroll
            for (int i = 0; i < 4; ++i) t.p[i] = mul2(t.p[i], w.p[i]);
            emit8<In, OUT, VEC>(a, row, v, to, t, n, buf);
        }
    }
    if (far) redo_far_rows<In, OUT, false>(a, blockIdx.x, gridDim.x, threadIdx.x, blockDim.x);
}

// Rows held in registers: a row is read once, 8 columns a vector and NV vectors
// a thread, by one warp (WARP, 8 rows a block) or one block; the block's
// threads are as many as the row needs.
template <class In, int OUT, bool VEC, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) k_norm_rows(const __grid_constant__ NormArgs a) {
    pdl_launch_dependents();
    uint8_t* buf = warp_buf<VEC>();
    constexpr int F = OUT == kOutNV ? kNVFP4 : kMXFP4;
    const bool four = OUT == kOutMX || OUT == kOutNV;
    const int words = four ? mx4_words(a.cols, Mx4Traits<F>::block) : 0;
    const int width = WARP ? 32 : blockDim.x;
    const int t0 = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int per = WARP ? blockDim.x >> 5 : 1;  // rows a block takes at once
    if (VEC && NV == 1 && !WARP && blockIdx.x < a.rows && 8 * t0 < a.cols) {
        // few rows: their first bytes to L2 (which is coherent) while the kernel before ends
        prefetch_l2(static_cast<const In*>(a.x) + blockIdx.x * a.x_stride + 8 * t0);
        if (a.res) prefetch_l2(static_cast<const In*>(a.res) + blockIdx.x * a.res_stride + 8 * t0);
        prefetch_l2(static_cast<const uint8_t*>(a.w) + ((a.w_kind & 1) ? 16 : 32) * static_cast<size_t>(t0));
    }
    pdl_wait();
    int parity = 0;
    bool far = false;  // some row's sum(h^2) left fp32's range
    for (long long rl = static_cast<long long>(blockIdx.x) * per + (WARP ? threadIdx.x >> 5 : 0); rl < a.rows;
         rl += static_cast<long long>(gridDim.x) * per, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* x = static_cast<const In*>(a.x) + row * a.x_stride;
        Raw8<In> h[NV];
        load_vecs<In, VEC, NV>(h, x, t0, width, a.cols, buf);
        if (a.res) {
            const In* res = static_cast<const In*>(a.res) + row * a.res_stride;
            Raw8<In> q[NV];
            load_vecs<In, VEC, NV>(q, res, t0, width, a.cols, buf);
#pragma unroll
            for (int i = 0; i < NV; ++i) h[i] = add8<In>(h[i], q[i]);
            if (a.sum) {
                In* sum = static_cast<In*>(a.sum) + static_cast<size_t>(row) * a.cols;
#pragma unroll
                for (int i = 0; i < NV; ++i) store_vec<In, VEC>(sum, t0 + i * width, a.cols, h[i], buf);
            }
        }
        float2 s2 = both(0.0f);
        uint32_t tm = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            (void)row_terms(unpack8<In>(h[i]), load_weight8(a.w, a.w_kind, t0 + i * width, a.cols), s2, tm);
        float ss = s2.x + s2.y;
        if (WARP) {
#pragma unroll
            for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            tm = __reduce_max_sync(0xffffffffu, tm);
        } else {
            block_sum_max(ss, tm, parity);
        }
        const Mx4Row to = four ? mx4_row(a.codes, a.bscales, row, a.cols, words) : Mx4Row{};
        far |= ss > FLT_MAX;
        const RowNorm n = row_norm<OUT>(a, row, ss, tm, t0 == 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = t0 + i * width;
            F8 t = unpack8<In>(h[i]);
            const F8 w = load_weight8(a.w, a.w_kind, v, a.cols);
#pragma unroll
            for (int j = 0; j < 4; ++j) t.p[j] = mul2(t.p[j], w.p[j]);
            emit8<In, OUT, VEC>(a, row, v, to, t, n, buf);
        }
    }
    if (far)
        redo_far_rows<In, OUT, WARP>(a, static_cast<long long>(blockIdx.x) * per + (WARP ? threadIdx.x >> 5 : 0),
                                     static_cast<long long>(gridDim.x) * per, t0, width);
}

// Dense rows of a width that is not a multiple of 8, 8-bit output: all tensors are
// equally far off a 16-byte boundary (a.shift0 columns, more with every row), so
// the columns are cut into vectors where memory is: vector v of a row that lies
// s columns behind a boundary holds columns [8v - s, 8v - s + 8), whole words of every
// tensor, codes included, but for the row's ends.  Only the weight is read through
// a window.  (1021 x 5003 fp32: 12.3 us one column a lane.)
template <class In>
__device__ __forceinline__ Raw8<In> load_cut(const In* row, int c0, int cols) {
    Raw8<In> r;
    if (c0 >= 0 && c0 + 8 <= cols) {
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j) r.q[j] = reinterpret_cast<const uint4*>(row + c0)[j];
        return r;
    }
    F8 f{};
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int c = c0 + k;
        e[k] = c < 0 || c >= cols ? 0.0f : (sizeof(In) == 4 ? reinterpret_cast<const float*>(row)[c]
                                                            : bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[c]));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) f.p[k] = make_float2(e[2 * k], e[2 * k + 1]);
    return pack8<In>(f);
}
template <class In>
__device__ __forceinline__ void store_cut(In* row, int c0, int cols, const Raw8<In>& r) {
    if (c0 >= 0 && c0 + 8 <= cols) {
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j) reinterpret_cast<uint4*>(row + c0)[j] = r.q[j];
        return;
    }
    const uint32_t w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[sizeof(In) / 2 - 1].x, r.q[sizeof(In) / 2 - 1].y,
                           r.q[sizeof(In) / 2 - 1].z, r.q[sizeof(In) / 2 - 1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int c = c0 + k;
        if (c < 0 || c >= cols) continue;
        if (sizeof(In) == 4) reinterpret_cast<uint32_t*>(row)[c] = w[k];
        else reinterpret_cast<uint16_t*>(row)[c] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
    }
}
// Eight columns of the weight from any column on.
__device__ __forceinline__ F8 load_weight_cut(const void* w, int w_kind, int c0, int cols) {
    if (w_kind & 1) return unpack8<uint16_t>([&] {
        Raw8<uint16_t> r;
        const uint16_t* p = static_cast<const uint16_t*>(w);
        uint32_t e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = c0 + k < 0 || c0 + k >= cols ? 0u : __ldg(p + c0 + k);
        r.q[0] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        return r;
    }());
    const float* p = static_cast<const float*>(w);
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = c0 + k < 0 || c0 + k >= cols ? 0.0f : __ldg(p + c0 + k);
    return F8{{{e[0], e[1]}, {e[2], e[3]}, {e[4], e[5]}, {e[6], e[7]}}};
}

template <class In, int OUT, int NV, bool SMALL>
__global__ void __launch_bounds__(SMALL ? 320 : 1024, SMALL ? 4 : 1) k_norm_cut(const __grid_constant__ NormArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int width = blockDim.x, t0 = threadIdx.x;
    int parity = 0;
    bool far = false;  // some row's sum(h^2) left fp32's range
    for (long long rl = blockIdx.x; rl < a.rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const int s = static_cast<int>((a.shift0 + rl * a.cols) & 7);
        const size_t at = static_cast<size_t>(row) * a.cols;
        const In* x = static_cast<const In*>(a.x) + row * a.x_stride;
        Raw8<In> h[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k) h[k] = load_cut<In>(x, 8 * (t0 + k * width) - s, a.cols);
        if (a.res) {
            const In* res = static_cast<const In*>(a.res) + row * a.res_stride;
            Raw8<In> q[NV];
#pragma unroll
            for (int k = 0; k < NV; ++k) q[k] = load_cut<In>(res, 8 * (t0 + k * width) - s, a.cols);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                h[k] = add8<In>(h[k], q[k]);
                if (a.sum) store_cut<In>(static_cast<In*>(a.sum) + at, 8 * (t0 + k * width) - s, a.cols, h[k]);
            }
        }
        float2 s2 = both(0.0f);
        uint32_t tm = 0;
        F8 t[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            t[k] = row_terms(unpack8<In>(h[k]), load_weight_cut(a.w, a.w_kind, 8 * (t0 + k * width) - s, a.cols), s2, tm);
        float ss = s2.x + s2.y;
        block_sum_max(ss, tm, parity);
        far |= ss > FLT_MAX;
        const RowNorm n = row_norm<OUT>(a, row, ss, tm, t0 == 0);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int c0 = 8 * (t0 + k * width) - s;
            if (a.y) {
                F8 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y.p[i] = mul2(t[k].p[i], both(n.r));
                store_cut<In>(static_cast<In*>(a.y) + at, c0, a.cols, pack8<In>(y));
            }
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 q = code_quotient(t[k].p[i], n);
                c[i] = ocp_encode2<OUT>(q.x, q.y);
            }
            uint8_t* o = a.codes + at;
            if (c0 >= 0 && c0 + 8 <= a.cols) {
                *reinterpret_cast<uint2*>(o + c0) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (c0 + e >= 0 && c0 + e < a.cols) o[c0 + e] = static_cast<uint8_t>(c[e / 2] >> (8 * (e & 1)));
            }
        }
    }
    if (far) redo_far_rows<In, OUT, false>(a, blockIdx.x, gridDim.x, t0, width);
}

// Many aligned rows: they come through a ring in shared memory by 1-D bulk
// copies, so that the next rows stream in while one is reduced and encoded.
// (Registers for as many blocks as the ring leaves room for: without the bound 16384 x 4096 bf16
// to NVFP4 takes 133 us for 116.)
template <class In, int OUT, int NV>
__global__ void __launch_bounds__(sizeof(In) == 2 ? 256 : 512, sizeof(In) == 2 ? (NV == 2 ? 3 : 2) : 0) k_norm_ring(const __grid_constant__ NormArgs a, int stages, uint32_t* err) {
    extern __shared__ __align__(128) uint8_t n_smem[];
    pdl_launch_dependents();
    constexpr int F = OUT == kOutNV ? kNVFP4 : kMXFP4;
    const bool four = OUT == kOutMX || OUT == kOutNV;
    const int words = four ? mx4_words(a.cols, Mx4Traits<F>::block) : 0;
    const int width = blockDim.x, t0 = threadIdx.x;
    const uint32_t rb = static_cast<uint32_t>(a.cols) * sizeof(In);
    const uint32_t stage_bytes = (a.res ? 2u : 1u) * rb;
    uint64_t* full = reinterpret_cast<uint64_t*>(n_smem + static_cast<size_t>(stages) * stage_bytes);
    if (t0 == 0) {
        for (int k = 0; k < stages; ++k) mbar_init(&full[k], 1);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    long long last = -1;  // the last row issued
    auto issue = [&](long long i) {
        const long long row = blockIdx.x + i * gridDim.x;
        if (row >= a.rows) return;
        const int st = static_cast<int>(i % stages);
        uint8_t* s = n_smem + static_cast<size_t>(st) * stage_bytes;
        last = i;
        mbar_arrive_expect_tx(&full[st], stage_bytes);
        bulk_load_1d(s, static_cast<const In*>(a.x) + static_cast<size_t>(row) * a.x_stride, rb, &full[st]);
        if (a.res) bulk_load_1d(s + rb, static_cast<const In*>(a.res) + static_cast<size_t>(row) * a.res_stride, rb, &full[st]);
    };
    if (t0 == 0)
        for (int i = 0; i < stages; ++i) issue(i);
    int st = 0, parity = 0;
    bool far = false;
    uint32_t phase = 0;
    bool ok = true;  // after a wait that ran out (error bit set) a thread waits and issues no more
    for (long long i = 0; blockIdx.x + i * gridDim.x < a.rows; ++i, parity ^= 1) {
        const int row = static_cast<int>(blockIdx.x + i * gridDim.x);
        ok = ok && mbar_wait(&full[st], phase, err);
        const In* s = reinterpret_cast<const In*>(n_smem + static_cast<size_t>(st) * stage_bytes);
        Raw8<In> h[NV];
        load_vecs<In, true, NV>(h, s, t0, width, a.cols, nullptr);
        if (a.res) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int v = t0 + k * width;
                h[k] = add8<In>(h[k], load_vec<In, true>(s + a.cols, v, a.cols, nullptr));
                if (a.sum) store_vec<In, true>(static_cast<In*>(a.sum) + static_cast<size_t>(row) * a.cols, v, a.cols, h[k], nullptr);
            }
        }
        float2 s2 = both(0.0f);
        uint32_t tm = 0;
        F8 t[NV];
#pragma unroll
        for (int k = 0; k < NV; ++k)
            t[k] = row_terms(unpack8<In>(h[k]), load_weight8(a.w, a.w_kind, t0 + k * width, a.cols), s2, tm);
        float ss = s2.x + s2.y;
        block_sum_max(ss, tm, parity);
        if (t0 == 0 && ok) issue(i + stages);  // every thread has read the stage
        const Mx4Row to = four ? mx4_row(a.codes, a.bscales, row, a.cols, words) : Mx4Row{};
        far |= ss > FLT_MAX;
        const RowNorm n = row_norm<OUT>(a, row, ss, tm, t0 == 0);
#pragma unroll
        for (int k = 0; k < NV; ++k) emit8<In, OUT, true>(a, row, t0 + k * width, to, t[k], n, nullptr);
        if (++st == stages) { st = 0; phase ^= 1u; }
    }
    if (!ok && t0 == 0)  // copies still in flight land before the block ends
        for (long long k = max(0ll, last - stages + 1); k <= last; ++k)
            mbar_wait(&full[k % stages], static_cast<uint32_t>(k / stages) & 1u, nullptr);
    if (far) redo_far_rows<In, OUT, false>(a, blockIdx.x, gridDim.x, t0, width);
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
    float eps, inv_cols;
    int w_kind;  // bit 0: bf16, bit 1: 16-byte aligned
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

// Row terms of the gradient: dx = dsum + r (g - m n), n = h r, m = mean(g n).  |m| <= max |g|: in
// range whatever r is (r^2, in the form r g - r^2 m h, leaves fp32 for rows of 1e18 or of 1e-19).
struct RowGrad {
    float r, m;
};
__device__ __forceinline__ RowGrad row_grad(const GradArgs& a, float sumsq, float sgh) {
    RowGrad q;
    q.r = row_r(sumsq, a.inv_cols, a.eps);
    q.m = __fmul_rn(__fmul_rn(sgh, q.r), a.inv_cols);
    return q;
}
__device__ __forceinline__ bool row_grad_ok(float sumsq, float sgh) { return sumsq <= FLT_MAX && fabsf(sgh) <= FLT_MAX; }
// The same where a sum is out of range, from those with h 2^-80 in the place of h (sumsq: sum(h^2) itself).
__device__ __forceinline__ RowGrad row_grad_far(const GradArgs& a, float sumsq, float far_sumsq, float far_sgh) {
    const float r = sumsq <= FLT_MAX ? row_r(sumsq, a.inv_cols, a.eps) / kFar : row_r(far_sumsq, a.inv_cols, a.eps * kFar * kFar);
    RowGrad q;
    q.r = r * kFar;
    q.m = __fmul_rn(__fmul_rn(far_sgh, r), a.inv_cols);
    return q;
}
// (sums of a vector for it)
__device__ __forceinline__ void grad_far_terms(const F8& h, const F8& gw, float2& ss, float2& sg) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = mul2(h.p[i], both(kFar));
        ss = fma2(f, f, ss);
        sg = fma2(gw.p[i], f, sg);
    }
}
// gw = g w; ss += h^2, sg += gw h.
__device__ __forceinline__ F8 grad_terms(const F8& h, const F8& g, const F8& w, float2& ss, float2& sg) {
    F8 gw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        ss = fma2(h.p[i], h.p[i], ss);
        gw.p[i] = mul2(g.p[i], w.p[i]);
        sg = fma2(gw.p[i], h.p[i], sg);
    }
    return gw;
}
// r (gw - m n) [+ d]
__device__ __forceinline__ F8 grad_dx(const F8& n, const F8& gw, const RowGrad& q, bool has_d, const F8& d) {
    F8 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o.p[i] = fma2(both(-q.m), n.p[i], gw.p[i]);
        o.p[i] = has_d ? fma2(both(q.r), o.p[i], d.p[i]) : mul2(both(q.r), o.p[i]);
    }
    return o;
}

// One block per row in two passes, for rows too wide for k_norm_grad; r of every
// row also goes to `rs` for the weight's gradient.
template <class In, bool VEC>
__global__ void __launch_bounds__(256) k_norm_grad_rows(const GradArgs a, float* __restrict__ rs) {
    pdl_launch_dependents();
    pdl_wait();
    uint8_t* buf = warp_buf<VEC>();
    const int nvec = (a.cols + 7) / 8;
    const int lane = lane_of();
    int parity = 0;
    for (long long rl = blockIdx.x; rl < a.rows; rl += gridDim.x, parity ^= 1) {
        const int row = static_cast<int>(rl);
        const In* hp = static_cast<const In*>(a.h) + row * a.h_stride;
        const size_t at = static_cast<size_t>(row) * a.cols;
        const In* dyp = static_cast<const In*>(a.dy) + at;
        float2 s2 = both(0.0f), g2 = both(0.0f);
        for (int v = threadIdx.x; v - lane < nvec; v += blockDim.x)
            (void)grad_terms(unpack8<In>(load_vec<In, VEC>(hp, v, a.cols, buf)), unpack8<In>(load_vec<In, VEC>(dyp, v, a.cols, buf)),
                             load_weight8(a.w, a.w_kind, v, a.cols), s2, g2);
        float ss = s2.x + s2.y, sg = g2.x + g2.y;
        block_sum2(ss, sg, parity);
        RowGrad q = row_grad(a, ss, sg);
        if (!row_grad_ok(ss, sg)) {
            s2 = g2 = both(0.0f);
            for (int v = threadIdx.x; v - lane < nvec; v += blockDim.x) {
                F8 g = unpack8<In>(load_vec<In, VEC>(dyp, v, a.cols, buf));
                const F8 w = load_weight8(a.w, a.w_kind, v, a.cols);
#pragma unroll
                for (int i = 0; i < 4; ++i) g.p[i] = mul2(g.p[i], w.p[i]);
                grad_far_terms(unpack8<In>(load_vec<In, VEC>(hp, v, a.cols, buf)), g, s2, g2);
            }
            float fs = s2.x + s2.y, fg = g2.x + g2.y;
            __syncthreads();  // the buffers of block_sum2 are free again
            block_sum2(fs, fg, parity);
            q = row_grad_far(a, ss, fs, fg);
        }
        if (threadIdx.x == 0) rs[row] = q.r;
        if (!a.dx) continue;
        for (int v = threadIdx.x; v - lane < nvec; v += blockDim.x) {
            F8 n = unpack8<In>(load_vec<In, VEC>(hp, v, a.cols, buf));
            const F8 w = load_weight8(a.w, a.w_kind, v, a.cols);
            F8 g = unpack8<In>(load_vec<In, VEC>(dyp, v, a.cols, buf)), d{};
            if (a.dsum) d = unpack8<In>(load_vec<In, VEC>(static_cast<const In*>(a.dsum) + at, v, a.cols, buf));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                n.p[i] = mul2(n.p[i], both(q.r));
                g.p[i] = mul2(g.p[i], w.p[i]);
            }
            store_vec<In, VEC>(static_cast<In*>(a.dx) + at, v, a.cols, pack8<In>(grad_dx(n, g, q, a.dsum, d)), buf);
        }
    }
}

// A row in registers: its vectors as loaded.
template <class In, int NV>
struct GradRow {
    Raw8<In> h[NV], g[NV], d[NV];
};
// The row's sums over the block, its dx, and its share of the weight's gradient.
// next() runs once every thread of the block has read the row.
template <class In, bool VEC, int NV, class Next>
__device__ __forceinline__ void grad_row(const GradArgs& a, const GradRow<In, NV>& r, size_t at, int t0, int width, int parity,
                                         F8 (&acc)[NV], uint8_t* buf, Next next) {
    // Of four vectors the products are formed again where they are needed: kept beside the branch
    // below, they spill (4096 x 16384 bf16: 167 us for 160).
    constexpr bool KEEP = NV < 4;
    float2 s2 = both(0.0f), g2 = both(0.0f);
    F8 gw[KEEP ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const F8 p = grad_terms(unpack8<In>(r.h[i]), unpack8<In>(r.g[i]), load_weight8(a.w, a.w_kind, t0 + i * width, a.cols), s2, g2);
        if constexpr (KEEP) gw[i] = p;
    }
    auto product = [&](int i) {
        if constexpr (KEEP) return gw[i];
        int v = t0 + i * width;
        asm volatile("" : "+r"(v));  // (a load of its own)
        F8 p = unpack8<In>(r.g[i]);
        const F8 w = load_weight8(a.w, a.w_kind, v, a.cols);
#pragma unroll
        for (int j = 0; j < 4; ++j) p.p[j] = mul2(p.p[j], w.p[j]);
        return p;
    };
    float ss = s2.x + s2.y, sg = g2.x + g2.y;
    block_sum2(ss, sg, parity);
    next();
    RowGrad q = row_grad(a, ss, sg);
    if (!row_grad_ok(ss, sg)) {
        s2 = g2 = both(0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) grad_far_terms(unpack8<In>(r.h[i]), product(i), s2, g2);
        float fs = s2.x + s2.y, fg = g2.x + g2.y;
        __syncthreads();  // the buffers of block_sum2 are free again
        block_sum2(fs, fg, parity);
        q = row_grad_far(a, ss, fs, fg);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        F8 n = unpack8<In>(r.h[i]);
        const F8 g = unpack8<In>(r.g[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            n.p[j] = mul2(n.p[j], both(q.r));
            acc[i].p[j] = fma2(n.p[j], g.p[j], acc[i].p[j]);
        }
        if (a.dx) {
            F8 d{};
            if (a.dsum) d = unpack8<In>(r.d[i]);
            store_vec<In, VEC>(static_cast<In*>(a.dx) + at, t0 + i * width, a.cols,
                               pack8<In>(grad_dx(n, product(i), q, a.dsum, d)), buf);
        }
    }
}

// Rows read once: dx, and the weight's gradient summed over the block's rows
// (blockIdx.x, + gridDim.x, ...) in registers, one partial row a block.
// Aligned rows (VEC) come through a ring in shared memory by 1-D bulk copies:
// the next rows stream in while one is reduced, without registers for
// them (8192 x 4096 bf16: 79 us with loads straight to registers).
template <class In, bool VEC, int NV>
__global__ void __launch_bounds__(512) k_norm_grad(const GradArgs a, int stages, float* __restrict__ part, uint32_t* err) {
    extern __shared__ __align__(128) uint8_t g_smem[];
    pdl_launch_dependents();
    uint8_t* buf = warp_buf<VEC>();
    const int t0 = threadIdx.x, width = blockDim.x;
    const bool has_d = a.dsum && a.dx;
    F8 acc[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[i] = F8{};
    int parity = 0;
    if constexpr (VEC) {
        const uint32_t rb = static_cast<uint32_t>(a.cols) * sizeof(In);
        const uint32_t stage_bytes = (has_d ? 3u : 2u) * rb;
        uint64_t* full = reinterpret_cast<uint64_t*>(g_smem + static_cast<size_t>(stages) * stage_bytes);
        if (t0 == 0) {
            for (int k = 0; k < stages; ++k) mbar_init(&full[k], 1);
            fence_mbar_init();
        }
        __syncthreads();
        pdl_wait();
        auto issue = [&](long long i) {
            const long long row = blockIdx.x + i * gridDim.x;
            if (row >= a.rows) return;
            const int st = static_cast<int>(i % stages);
            uint8_t* s = g_smem + static_cast<size_t>(st) * stage_bytes;
            mbar_arrive_expect_tx(&full[st], stage_bytes);
            bulk_load_1d(s, static_cast<const In*>(a.h) + static_cast<size_t>(row) * a.h_stride, rb, &full[st]);
            bulk_load_1d(s + rb, static_cast<const In*>(a.dy) + static_cast<size_t>(row) * a.cols, rb, &full[st]);
            if (has_d) bulk_load_1d(s + 2 * rb, static_cast<const In*>(a.dsum) + static_cast<size_t>(row) * a.cols, rb, &full[st]);
        };
        if (t0 == 0)
            for (int i = 0; i < stages; ++i) issue(i);
        int st = 0;
        uint32_t phase = 0;
        long long i = 0;
        bool ok = true;
        for (; blockIdx.x + i * gridDim.x < a.rows; ++i, parity ^= 1) {
            const size_t row = static_cast<size_t>(blockIdx.x + i * gridDim.x);
            ok = mbar_wait(&full[st], phase, err);
            if (!__syncthreads_and(ok)) {
                ok = false;
                break;
            }
            const uint8_t* s = g_smem + static_cast<size_t>(st) * stage_bytes;
            GradRow<In, NV> r;
            load_vecs<In, true, NV>(r.h, reinterpret_cast<const In*>(s), t0, width, a.cols, nullptr);
            load_vecs<In, true, NV>(r.g, reinterpret_cast<const In*>(s + rb), t0, width, a.cols, nullptr);
            if (has_d) load_vecs<In, true, NV>(r.d, reinterpret_cast<const In*>(s + 2 * rb), t0, width, a.cols, nullptr);
            grad_row<In, true, NV>(a, r, row * a.cols, t0, width, parity, acc, nullptr, [&]() {
                if (t0 == 0) issue(i + stages);
            });
            if (++st == stages) { st = 0; phase ^= 1u; }
        }
        if (!ok && t0 == 0)  // the copies in flight land before the block ends
            for (int k = 0; k < stages && blockIdx.x + (i + k) * gridDim.x < a.rows; ++k) {
                mbar_wait(&full[st], phase, nullptr);
                if (++st == stages) { st = 0; phase ^= 1u; }
            }
    } else {
        pdl_wait();
        for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
            const size_t at = static_cast<size_t>(row) * a.cols;
            GradRow<In, NV> r;
            load_vecs<In, VEC, NV>(r.h, static_cast<const In*>(a.h) + static_cast<size_t>(row) * a.h_stride, t0, width, a.cols, buf);
            load_vecs<In, VEC, NV>(r.g, static_cast<const In*>(a.dy) + at, t0, width, a.cols, buf);
            if (has_d) load_vecs<In, VEC, NV>(r.d, static_cast<const In*>(a.dsum) + at, t0, width, a.cols, buf);
            grad_row<In, VEC, NV>(a, r, at, t0, width, parity, acc, buf, []() {});
        }
    }
    if (!part) return;
    float* mine = part + static_cast<size_t>(blockIdx.x) * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) store_vec<float, VEC>(mine, t0 + i * width, a.cols, pack8<float>(acc[i]), buf);
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
// dw[c] = sum of the partial rows: 32 columns a block, warp k adds rows k, k + 32,
// ... and the warps are added in order.
__global__ void __launch_bounds__(1024) k_sum_chunks(const float* __restrict__ part, int chunks, int cols, float* __restrict__ dw) {
    __shared__ float s_part[32][33];
    pdl_launch_dependents();
    pdl_wait();
    const int c = blockIdx.x * 32 + lane_of(), k0 = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (int k = k0; k < chunks; k += 32) s = __fadd_rn(s, part[static_cast<size_t>(k) * cols + c]);
    }
    s_part[k0][lane_of()] = s;
    __syncthreads();
    if (k0 == 0 && c < cols) {
        s = s_part[0][lane_of()];
#pragma unroll
        for (int k = 1; k < 32; ++k) s = __fadd_rn(s, s_part[k][lane_of()]);
        dw[c] = s;
    }
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
    if (!(d->eps >= FLT_MIN) || !(d->eps <= FLT_MAX)) return bad(who, "eps must be at least FLT_MIN (1.18e-38) and finite");
    if ((d->x_stride && d->x_stride < d->cols) || (d->residual_stride && d->residual_stride < d->cols))
        return bad(who, "a row stride is smaller than cols");
    *xs = d->x_stride ? d->x_stride : d->cols;
    *rs = d->residual_stride ? d->residual_stride : d->cols;
    return NQ_SUCCESS;
}

template <class In, int OUT, bool VEC, int NV, bool WARP>
nq_status_t launch_norm_rows(const NormArgs& a, int threads, const DeviceInfo& di, cudaStream_t s, const char* who) {
    auto kern = k_norm_rows<In, OUT, VEC, NV, WARP>;
    const long long blocks = WARP ? (static_cast<long long>(a.rows) + threads / 32 - 1) / (threads / 32) : a.rows;
    const int grid = persistent_grid(kern, threads, 0, blocks, di);
    return cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), 0, s, a), who);
}

constexpr size_t kRingSmem = 200 * 1024;

template <class In, int OUT, int NV>
nq_status_t launch_norm_ring(const NormArgs& a, int nvec, const DeviceInfo& di, cudaStream_t s, const char* who) {
    auto kern = k_norm_ring<In, OUT, NV>;
    const int threads = ((nvec + NV - 1) / NV + 31) / 32 * 32;
    const size_t row = static_cast<size_t>(a.cols) * sizeof(In) * (a.res ? 2 : 1);
    const int stages = static_cast<int>(std::max<size_t>(2, std::min<size_t>(4, 96 * 1024 / row)));
    const size_t smem = stages * (row + 8);
    static std::mutex mu;
    static std::atomic<uint64_t> attr_set{0};
    nq_status_t st = once_per_device(attr_set, mu, di.device, [&]() -> nq_status_t {
        NQ_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRingSmem)),
                      "cudaFuncSetAttribute(nq_rmsnorm)");
        return NQ_SUCCESS;
    });
    if (st != NQ_SUCCESS) return st;
    const int grid = persistent_grid(kern, threads, smem, a.rows, di);
    return cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), smem, s, a, stages, device_error_word()), who);
}

template <class In, int OUT, int NV, bool SMALL>
nq_status_t launch_norm_cut(const NormArgs& a, int threads, const DeviceInfo& di, cudaStream_t s, const char* who) {
    auto kern = k_norm_cut<In, OUT, NV, SMALL>;
    const int grid = persistent_grid(kern, threads, 0, a.rows, di);
    return cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), 0, s, a), who);
}

template <class In, int OUT, bool VEC>
nq_status_t launch_norm(const NormArgs& a, const DeviceInfo& di, cudaStream_t s, const char* who) {
    constexpr int NVMAX = sizeof(In) == 2 ? 4 : 2;  // 64 bytes a thread of each tensor
    int nvec = (a.cols + 7) / 8;
    if (OUT == kOutMX) nvec = mx4_words(a.cols, 32) * 16;  // whole scale words
    if (OUT == kOutNV) nvec = mx4_words(a.cols, 16) * 8;
    if constexpr (OUT <= kOutINT8 && !VEC) {
        if (a.shift0 >= 0 && nvec + 1 <= 1024 * NVMAX) {
            const int cut = nvec + 1;  // a row may begin inside its first vector
            if (cut <= 256) return launch_norm_cut<In, OUT, 1, true>(a, (cut + 31) / 32 * 32, di, s, who);
            const int threads = ((cut + NVMAX - 1) / NVMAX + 31) / 32 * 32;
            if constexpr (sizeof(In) == 4)
                if (threads <= 320) return launch_norm_cut<In, OUT, NVMAX, true>(a, threads, di, s, who);
            return launch_norm_cut<In, OUT, NVMAX, false>(a, threads, di, s, who);
        }
    }
    if (nvec <= 32 * NVMAX) {
        if (nvec <= 32) return launch_norm_rows<In, OUT, VEC, 1, true>(a, 256, di, s, who);
        return launch_norm_rows<In, OUT, VEC, NVMAX, true>(a, 256, di, s, who);
    }
    if (a.rows < 2 * di.sm_count && nvec <= 1024)
        return launch_norm_rows<In, OUT, VEC, 1, false>(a, (nvec + 31) / 32 * 32, di, s, who);
    const int threads = ((nvec + NVMAX - 1) / NVMAX + 31) / 32 * 32;
    if (VEC && a.rows >= 4 * di.sm_count && nvec <= 1024) {
        if (nvec <= 512) return launch_norm_ring<In, OUT, NVMAX / 2>(a, nvec, di, s, who);
        return launch_norm_ring<In, OUT, NVMAX>(a, nvec, di, s, who);
    }
    if (threads <= 1024) return launch_norm_rows<In, OUT, VEC, NVMAX, false>(a, threads, di, s, who);
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
                     aligned16(residual) && aligned16(sum) && aligned16(y) && aligned16(codes);
    // the tensors' common distance from a boundary of 8 columns, row for row
    auto off = [&](const void* p, size_t e) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) / e % 8); };
    const bool agree = xs % 8 == static_cast<size_t>(d->cols) % 8 && (!residual || rs % 8 == static_cast<size_t>(d->cols) % 8) &&
                       (!residual || off(residual, es) == off(x, es)) && (!sum || off(sum, es) == off(x, es)) &&
                       (!y || off(y, es) == off(x, es)) && codes && off(codes, 1) == off(x, es);
    const NormArgs a{x, residual, weight, sum, y, codes, bscales, scales, d->rows, d->cols, xs, rs, d->eps, 1.0f / d->cols,
                     (d->weight_dtype == NQ_BF16 ? 1 : 0) | (aligned16(weight) ? 2 : 0), agree ? off(x, es) : -1};
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

nq_status_t sum_chunks(const float* part, int chunks, int cols, float* dw, cudaStream_t s) {
    return cuda_status(launch_pdl(k_sum_chunks, dim3((cols + 31) / 32), dim3(1024), 0, s, part, chunks, cols, dw),
                       "nq_rmsnorm_backward (weight)");
}

constexpr size_t kGradSmem = 200 * 1024;

template <class In, bool VEC, int NV>
nq_status_t launch_grad(const GradArgs& a, float* dw, const DeviceInfo& di, cudaStream_t s) {
    auto kern = k_norm_grad<In, VEC, NV>;
    const int threads = ((a.cols + 8 * NV - 1) / (8 * NV) + 31) / 32 * 32;
    int stages = 0;
    size_t smem = 0;
    if (VEC) {
        // two to four rows ahead, up to 60 KB of them a block, or two rows where those are more
        // (room for dsum even where dx is not asked for: the grid, and with it the order of
        // the weight gradient's sum, does not depend on dx)
        const size_t row = static_cast<size_t>(a.cols) * sizeof(In) * (a.dsum ? 3 : 2);
        stages = static_cast<int>(std::max<size_t>(2, std::min<size_t>(4, 60 * 1024 / row)));
        smem = stages * (row + 8);
        static std::mutex mu;
        static std::atomic<uint64_t> attr_set{0};
        nq_status_t st = once_per_device(attr_set, mu, di.device, [&]() -> nq_status_t {
            NQ_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kGradSmem + 64)),
                          "cudaFuncSetAttribute(nq_rmsnorm_backward)");
            return NQ_SUCCESS;
        });
        if (st != NQ_SUCCESS) return st;
    }
    const int grid = persistent_grid(kern, threads, smem, a.rows, di);
    void* part = nullptr;
    nq_status_t st = NQ_SUCCESS;
    if (dw) st = scratch_alloc(&part, static_cast<size_t>(grid) * a.cols * 4, s);
    if (st != NQ_SUCCESS) return st;
    st = cuda_status(launch_pdl(kern, dim3(grid), dim3(threads), smem, s, a, stages, static_cast<float*>(part), device_error_word()),
                     "nq_rmsnorm_backward");
    if (st == NQ_SUCCESS && dw) st = sum_chunks(static_cast<const float*>(part), grid, a.cols, dw, s);
    scratch_free(part, s);
    return st;
}

template <class In, bool VEC>
nq_status_t grad_impl(const GradArgs& a, float* dw, const DeviceInfo& di, cudaStream_t s) {
    // vectors a thread: one up to 64 threads' worth, then two, then (bf16) four
    const int nvec = (a.cols + 7) / 8;
    if (nvec <= 64) return launch_grad<In, VEC, 1>(a, dw, di, s);
    if (nvec <= 1024) return launch_grad<In, VEC, 2>(a, dw, di, s);
    if (sizeof(In) == 2 && nvec <= 2048) return launch_grad<In, VEC, sizeof(In) == 2 ? 4 : 2>(a, dw, di, s);
    const int chunks = static_cast<int>(std::min<long long>(64, a.rows));
    const int per = (a.rows + chunks - 1) / chunks;
    void* scratch = nullptr;
    const size_t rs_bytes = (static_cast<size_t>(a.rows) * 4 + 255) / 256 * 256;
    nq_status_t st = scratch_alloc(&scratch, rs_bytes + static_cast<size_t>(chunks) * a.cols * 4, s);
    if (st != NQ_SUCCESS) return st;
    float* rs = static_cast<float*>(scratch);
    float* part = reinterpret_cast<float*>(static_cast<char*>(scratch) + rs_bytes);
    const int grid = static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(di.sm_count) * 8));
    cudaError_t e = launch_pdl(k_norm_grad_rows<In, VEC>, dim3(grid), dim3(256), 0, s, a, rs);
    if (e == cudaSuccess && dw)
        e = launch_pdl(k_norm_grad_weight<In>, dim3((a.cols + 255) / 256, chunks), dim3(256), 0, s, a,
                       static_cast<const float*>(rs), per, part);
    st = cuda_status(e, "nq_rmsnorm_backward");
    if (st == NQ_SUCCESS && dw) st = sum_chunks(part, chunks, a.cols, dw, s);
    scratch_free(scratch, s);
    return st;
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
    const bool vec = desc->cols % 8 == 0 && nq::strided_ok(xs, bf ? 2 : 4) && nq::aligned16(h) &&
                     nq::aligned16(grad_y) && nq::aligned16(grad_sum) && nq::aligned16(grad_x);
    const nq::GradArgs a{h, weight, grad_y, grad_sum, grad_x, desc->rows, desc->cols, xs, desc->eps, 1.0f / desc->cols,
                         (desc->weight_dtype == NQ_BF16 ? 1 : 0) | (nq::aligned16(weight) ? 2 : 0)};
    if (bf) return vec ? nq::grad_impl<uint16_t, true>(a, grad_weight, di, s) : nq::grad_impl<uint16_t, false>(a, grad_weight, di, s);
    return vec ? nq::grad_impl<float, true>(a, grad_weight, di, s) : nq::grad_impl<float, false>(a, grad_weight, di, s);
}

}  // extern "C"
