// mx4.cuh -- the microscaled 4-bit formats on the device.
//
// Elements are E2M1 (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a
// byte with the even column in the low nibble.
//   MXFP4: blocks of 32 columns, scale 2^(floor(log2 amax) - 2), one E8M0 byte
//     (the biased exponent).  The division by it is exact, so a code is the
//     correctly rounded E2M1 value.
//   NVFP4: blocks of 16 columns, scale s = E4M3(448 amax_block / A) with
//     A = max(amax_row, 2688 * 2^-110), element code E2M1(x * 2688 / (s A)) and
//     one fp32 scale A / 2688 for the row (6 * 448 = 2688: the row's largest
//     value is 6 * 448 * scale).  An all-zero row has scale 1.
//
// A thread holds 8 consecutive columns of a row: 2 lanes make an NVFP4 block,
// 4 an MXFP4 block; 8 (16) lanes make one 4-byte word of four scales.
#pragma once

#include "codec.cuh"

namespace nq {
namespace dev {

enum Mx4 : int { kMXFP4 = 0, kNVFP4 = 1 };

template <int F>
struct Mx4Traits {
    static constexpr int block = F == kMXFP4 ? 32 : 16;
    static constexpr int block_lanes = block / 8;      // lanes of 8 columns in a block
    static constexpr int word_lanes = 4 * block_lanes;  // lanes in a word of 4 scales
};

// Bytes of a row of codes: whole 32-column groups, so rows are 16-byte aligned.
__host__ __device__ __forceinline__ size_t mx4_pitch(int cols) {
    return (static_cast<size_t>(cols) + 31) / 32 * 16;
}
// 4-byte words of scales in a row.
__host__ __device__ __forceinline__ int mx4_words(int cols, int block) {
    return static_cast<int>((static_cast<long long>(cols) + 4 * block - 1) / (4 * block));
}
// Byte offset of a row's scale word in the tiled layout: 512-byte tiles of 128
// rows x 4 blocks, rows r and r + 32 four bytes apart -- what one
// tcgen05.cp.32x128b moves into the tensor memory columns of a 128-row operand.
__host__ __device__ __forceinline__ size_t mx4_scale_offset(int row, int word, int words) {
    return (static_cast<size_t>(row >> 7) * words + word) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// 8 floats -> 8 E2M1 codes (round to nearest even, saturating), v[0] lowest.
__device__ __forceinline__ uint32_t e2m1_encode8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// 8 codes -> 8 floats (exact).
__device__ __forceinline__ void e2m1_decode8(uint32_t c, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float mx4_scale_value(int fmt, uint32_t byte) {
    if (fmt == kNVFP4) return ocp_decode2<kE4M3>(byte).x;
    if (byte == 0xFFu) return __uint_as_float(0x7FC00000u);
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);  // 2^(byte - 127)
}

// Magnitude bits of the largest of 8 values: infinities and NaN order above
// every finite value, so a block or row that holds one is seen from its maximum.
__device__ __forceinline__ uint32_t amax_bits8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    return m;
}
constexpr uint32_t kInfBits = 0x7F800000u;

// The row's level A of NVFP4 and its stored scale.  Rows below 2688 * 2^-110
// keep A there, so no reciprocal below overflows; a row with an infinity or
// NaN has scale NaN (its codes and block scales are zero).
__device__ __forceinline__ float nv_row_level(uint32_t row_amax_bits) {
    return fmaxf(__uint_as_float(row_amax_bits), 2688.0f * 0x1p-110f);
}
__device__ __forceinline__ float nv_row_scale(uint32_t row_amax_bits, float level) {
    if (row_amax_bits == 0u) return 1.0f;
    if (row_amax_bits >= kInfBits) return __uint_as_float(0x7FC00000u);
    return __fdiv_rn(level, 2688.0f);
}

// Codes of this thread's 8 columns and the scale byte of its block.  Every lane
// of the warp takes part.  level: nv_row_level (NVFP4); ok: the row is finite
// (NVFP4 only; MXFP4 decides by block).
template <int F>
__device__ __forceinline__ uint32_t mx4_encode(const float (&v)[8], float level, bool ok, uint32_t* byte) {
    uint32_t a = amax_bits8(v);
    a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
    float q[8];
    if (F == kMXFP4) {
        a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
        const int e = max(static_cast<int>(a >> 23) - 2, 0);
        ok = a < kInfBits;
        *byte = ok ? static_cast<uint32_t>(e) : 0xFFu;
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e), exact
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __fmul_rn(v[i], inv);
    } else {
        // Both quotients of bf16 values often fall right on a rounding border
        // (they are ratios of small integers).  The first is a correctly rounded
        // division of exact operands, so a border stays a border and goes to
        // even; the second is a product with a rounded reciprocal, brought back
        // onto the grid of 2^-17 by adding and subtracting 96 (|q| < 9): its
        // error is below 2^-20 and a bf16 quotient that is no border is at
        // least 2^-15 away from one.
        const float lv = level * 0x1p-10f;
        const float s = __fdiv_rn(__uint_as_float(a) * 0.4375f, lv);
        *byte = ok ? ocp_encode2<kE4M3>(s, 0.0f) & 0xFFu : 0u;
        const float sv = ocp_decode2<kE4M3>(*byte).x;
        const float inv = sv > 0.0f ? __fdiv_rn(2.625f, __fmul_rn(sv, lv)) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __fsub_rn(__fmaf_rn(v[i], inv, 96.0f), 96.0f);
    }
    return ok ? e2m1_encode8(q) : 0u;
}

// The word of four scale bytes of this lane's group of word_lanes lanes (every
// lane of the warp takes part; the group's first lane stores it).
template <int F>
__device__ __forceinline__ uint32_t mx4_scale_word(uint32_t byte) {
    constexpr int L = Mx4Traits<F>::block_lanes;
    uint32_t w = byte | (__shfl_down_sync(0xffffffffu, byte, L) << 8);
    w |= __shfl_down_sync(0xffffffffu, w, 2 * L) << 16;
    return w;
}

// Stores one warp step of a quantised row: 8 columns a lane from column 8 * v.
template <int F>
__device__ __forceinline__ void mx4_store(uint8_t* codes_row, uint8_t* scales, int row, int v, int pitch_words, int words,
                                          uint32_t code, uint32_t byte) {
    const uint32_t w = mx4_scale_word<F>(byte);
    constexpr int WL = Mx4Traits<F>::word_lanes;
    if (v < pitch_words) reinterpret_cast<uint32_t*>(codes_row)[v] = code;
    if (v % WL == 0 && v / WL < words)
        *reinterpret_cast<uint32_t*>(scales + mx4_scale_offset(row, v / WL, words)) = w;
}

// ---- rows of fp32 / bf16 in vectors of 8 columns -----------------------------------
// A vector v holds columns [8v, 8v + 8) of a row, zero behind the last column.
// The lanes of a warp hold consecutive vectors and load and store together.
//   VEC: rows start on 16-byte boundaries and cols is a multiple of 8; a lane
//     moves its vector as 16-byte words.
//   else: the warp's 256 columns move one column a lane (whole sectors for any
//     alignment) and change hands through kWarpBuf bytes of the warp's shared
//     memory.  Eight scalar accesses 8 columns apart per lane instead made
//     every access of the warp touch 32 sectors (1021 x 5003 fp32 norm: 27 us).
constexpr int kWarpBuf = 1024;
__device__ __forceinline__ int lane_of() { return threadIdx.x & 31; }

template <class In>
struct Raw8 {
    uint4 q[sizeof(In) / 2];
};
template <class In>
__device__ __forceinline__ void unpack8(const Raw8<In>& r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = vec_elem<In>(r.q[sizeof(In) == 4 ? e / 4 : 0], sizeof(In) == 4 ? e % 4 : e);
}
// Rounds 8 values to the type (nearest even).
template <class In>
__device__ __forceinline__ Raw8<In> pack8(const float (&v)[8]) {
    Raw8<In> r;
    if constexpr (sizeof(In) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r.q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                                __float_as_uint(v[4 * i + 3]));
    } else {
        r.q[0] = make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]), f32x2_to_bf16x2(v[4], v[5]),
                            f32x2_to_bf16x2(v[6], v[7]));
    }
    return r;
}

// Vectors v0 + i * width, i < NV, of a row; all loads are issued before any use.
template <class In, bool VEC, int NV>
__device__ __forceinline__ void load_vecs(Raw8<In> (&r)[NV], const In* row, int v0, int width, int cols, uint8_t* buf) {
    if (VEC) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int v = v0 + i * width;
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j)
                r[i].q[j] = 8 * v < cols ? reinterpret_cast<const uint4*>(row + 8 * static_cast<size_t>(v))[j] : make_uint4(0, 0, 0, 0);
        }
    } else {
        In* b = reinterpret_cast<In*>(buf);
        In s[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c0 = 8 * (v0 + i * width - lane_of()) + lane_of();
#pragma unroll
            for (int e = 0; e < 8; ++e) s[i][e] = c0 + 32 * e < cols ? row[c0 + 32 * e] : In(0);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) b[32 * e + lane_of()] = s[i][e];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j)
                r[i].q[j] = reinterpret_cast<const uint4*>(b + 8 * lane_of())[j];
        }
    }
}
template <class In, bool VEC>
__device__ __forceinline__ Raw8<In> load_vec(const In* row, int v, int cols, uint8_t* buf) {
    Raw8<In> r[1];
    load_vecs<In, VEC, 1>(r, row, v, 0, cols, buf);
    return r[0];
}
template <class In, bool VEC>
__device__ __forceinline__ void store_vec(In* row, int v, int cols, const Raw8<In>& r, uint8_t* buf) {
    if (VEC) {
        if (8 * v >= cols) return;
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(In) / 2); ++i)
            reinterpret_cast<uint4*>(row + 8 * static_cast<size_t>(v))[i] = r.q[i];
    } else {
        In* b = reinterpret_cast<In*>(buf);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(In) / 2); ++j) reinterpret_cast<uint4*>(b + 8 * lane_of())[j] = r.q[j];
        __syncwarp();
        const int c0 = 8 * (v - lane_of()) + lane_of();
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + 32 * e < cols) row[c0 + 32 * e] = b[32 * e + lane_of()];
    }
}
// 8 one-byte codes a lane.
template <bool VEC>
__device__ __forceinline__ void store_codes8(uint8_t* row, int v, int cols, const uint2& c, uint8_t* buf) {
    if (VEC) {
        if (8 * v < cols) *reinterpret_cast<uint2*>(row + 8 * static_cast<size_t>(v)) = c;
    } else {
        __syncwarp();
        reinterpret_cast<uint2*>(buf)[lane_of()] = c;
        __syncwarp();
        const int c0 = 8 * (v - lane_of()) + lane_of();
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c0 + 32 * e < cols) row[c0 + 32 * e] = buf[32 * e + lane_of()];
    }
}

}  // namespace dev
}  // namespace nq
