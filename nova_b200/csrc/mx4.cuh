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

// Two fp32 operations an instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r, x = *reinterpret_cast<uint64_t*>(&a), y = *reinterpret_cast<uint64_t*>(&b);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r, x = *reinterpret_cast<uint64_t*>(&a), y = *reinterpret_cast<uint64_t*>(&b);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r, x = *reinterpret_cast<uint64_t*>(&a), y = *reinterpret_cast<uint64_t*>(&b), z = *reinterpret_cast<uint64_t*>(&c);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// Eight columns as four pairs.
struct F8 {
    float2 p[4];
    __device__ __forceinline__ float operator[](int e) const { return (e & 1) ? p[e >> 1].y : p[e >> 1].x; }
};

// 8 floats -> 8 E2M1 codes (round to nearest even, saturating), v[0] lowest.
__device__ __forceinline__ uint32_t e2m1_encode8(const F8& v) {
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
__device__ __forceinline__ void e2m1_decode8(uint32_t c, F8& v) {
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
        v.p[i] = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    }
}
__device__ __forceinline__ float mx4_scale_value(int fmt, uint32_t byte) {
    if (fmt == kNVFP4) return ocp_decode2<kE4M3>(byte).x;
    if (byte == 0xFFu) return __uint_as_float(0x7FC00000u);
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);  // 2^(byte - 127)
}

// Magnitude bits of the largest of 8 values: infinities and NaN order above
// every finite value, so a block or row that holds one is seen from its maximum.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t amax_bits8(const F8& v) {
    const float a = max3_nan(fabsf(v[0]), fabsf(v[1]), fabsf(v[2]));
    const float b = max3_nan(fabsf(v[3]), fabsf(v[4]), fabsf(v[5]));
    return __float_as_uint(max3_nan(max3_nan(fabsf(v[6]), fabsf(v[7]), a), b, b)) & 0x7FFFFFFFu;
}
constexpr uint32_t kInfBits = 0x7F800000u;

// Row terms of NVFP4 from the row's largest magnitude.
struct NvRow {
    float level;    // A
    float to_s;     // 448 / A
    float to_code;  // 2688 / A
    bool ok;        // the row is finite
};
// Rows below 2688 * 2^-110 keep A there, so nothing below overflows; a row with
// an infinity or NaN has scale NaN (its codes and block scales are zero).
__device__ __forceinline__ NvRow nv_row(uint32_t row_amax_bits) {
    NvRow r;
    r.level = fmaxf(__uint_as_float(row_amax_bits), 2688.0f * 0x1p-110f);
    r.to_s = __fdiv_rn(448.0f, r.level);
    r.to_code = __fmul_rn(6.0f, r.to_s);
    r.ok = row_amax_bits < kInfBits;
    return r;
}
__device__ __forceinline__ float nv_row_scale(uint32_t row_amax_bits, float level) {
    if (row_amax_bits == 0u) return 1.0f;
    if (row_amax_bits >= kInfBits) return __uint_as_float(0x7FC00000u);
    return __fdiv_rn(level, 2688.0f);
}
__device__ __forceinline__ float rcp_approx(float x) {  // relative error below 2^-22
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Scale byte of a block from the magnitude bits of its largest value, and the
// factor that takes its values to E2M1's range.
struct Mx4Block {
    uint32_t byte;
    float inv;
    double unit;  // NVFP4, FIX: s A
    bool ok;      // codes are not forced to zero
};
// A rounded quotient on a grid (below) stands on a rounding border: `exact` is the sign of the
// true quotient's distance from it, and a step that no rounding to a few bits sees.
__device__ __forceinline__ float nudge(float q, double exact) {
    return exact > 0.0 ? q * (1.0f + 0x1p-20f) : (exact < 0.0 ? q * (1.0f - 0x1p-20f) : q);
}
// NVFP4's quotients.  Those of bf16 values often fall right on a rounding border
// (they are ratios of small integers), and have to stay there to go to even.
// Products with rounded reciprocals move them by less than 2^-22 of themselves (codes:
// 2^-21.4, of at most 5), so they are brought onto a grid first: the scale's quotient
// to 20 mantissa bits, the code's to multiples of 2^-17 (96 added and
// subtracted; |q| < 9).  Quotients of bf16 values that are no border are at least 2^-13
// (relative) and 2^-15 away from one, so they round as the true quotient does.
// FIX, for values of more bits: a quotient that the grid puts on a border (about
// one in 10^5) is compared with it exactly, in products of double.  With two correctly
// rounded divisions a lane instead the quantize was bound by its arithmetic (8192 x
// 4096 bf16: 25.1 us).
template <int F, bool FIX>
__device__ __forceinline__ Mx4Block mx4_block(uint32_t a, const NvRow& row) {
    Mx4Block k;
    k.unit = 0.0;
    if (F == kMXFP4) {
        const int e = max(static_cast<int>(a >> 23) - 2, 0);
        k.ok = a < kInfBits;
        k.byte = k.ok ? static_cast<uint32_t>(e) : 0xFFu;
        k.inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);  // 2^(127 - e), exact
    } else {
        k.ok = row.ok;
        const uint32_t g = (__float_as_uint(__fmul_rn(__uint_as_float(a), row.to_s)) + 4u) & ~7u;
        float s = __uint_as_float(g);
        if (FIX && (g & 0x7FFFFu) == 0u && g != 0u)  // borders of E4M3 have four mantissa bits
            s = nudge(s, 448.0 * __uint_as_float(a) - static_cast<double>(s) * row.level);
        k.byte = k.ok ? ocp_encode2<kE4M3>(s, 0.0f) & 0xFFu : 0u;
        const float sv = ocp_decode2<kE4M3>(k.byte).x;
        k.inv = sv > 0.0f ? __fmul_rn(rcp_approx(sv), row.to_code) : 0.0f;
        if (FIX) k.unit = static_cast<double>(sv) * row.level;
    }
    return k;
}
template <int F, bool FIX>
__device__ __forceinline__ uint32_t mx4_codes8(const F8& v, const Mx4Block& k) {
    F8 q;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        q.p[i] = F == kMXFP4 ? mul2(v.p[i], both(k.inv)) : add2(fma2(v.p[i], both(k.inv), both(96.0f)), both(-96.0f));
    if (F == kNVFP4 && FIX) {
        // borders of E2M1 are multiples of 1/4 (adding 1.5 * 2^21 rounds to them)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 r = add2(add2(q.p[i], both(3145728.0f)), both(-3145728.0f));
            if (r.x == q.p[i].x && r.x != 0.0f)
                q.p[i].x = nudge(r.x, 2688.0 * fabsf(v.p[i].x) - static_cast<double>(fabsf(r.x)) * k.unit);
            if (r.y == q.p[i].y && r.y != 0.0f)
                q.p[i].y = nudge(r.y, 2688.0 * fabsf(v.p[i].y) - static_cast<double>(fabsf(r.y)) * k.unit);
        }
    }
    return k.ok ? e2m1_encode8(q) : 0u;
}
// Codes of this thread's 8 columns and the scale byte of its block.  Every lane
// of the warp takes part.  a: magnitude bits of the largest of the 8 (amax_bits8).
template <int F, bool FIX>
__device__ __forceinline__ uint32_t mx4_encode(const F8& v, uint32_t a, const NvRow& row, uint32_t* byte) {
    a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
    if (F == kMXFP4) a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
    const Mx4Block k = mx4_block<F, FIX>(a, row);
    *byte = k.byte;
    return mx4_codes8<F, FIX>(v, k);
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

// Where a quantised row goes.
struct Mx4Row {
    uint32_t* codes;
    uint8_t* scales;  // its word 0; word w is 512 w bytes on
    int pitch_words, words;
};
__device__ __forceinline__ Mx4Row mx4_row(uint8_t* codes, uint8_t* scales, int row, int cols, int words) {
    const size_t pitch = mx4_pitch(cols);
    return Mx4Row{reinterpret_cast<uint32_t*>(codes + row * pitch), scales + mx4_scale_offset(row, 0, words),
                  static_cast<int>(pitch / 4), words};
}
// Stores one warp step of it: 8 columns a lane from column 8 * v.
template <int F>
__device__ __forceinline__ void mx4_store(const Mx4Row& r, int v, uint32_t code, uint32_t byte) {
    const uint32_t w = mx4_scale_word<F>(byte);
    constexpr int WL = Mx4Traits<F>::word_lanes;
    if (v < r.pitch_words) r.codes[v] = code;
    if (v % WL == 0 && v / WL < r.words) *reinterpret_cast<uint32_t*>(r.scales + static_cast<size_t>(v / WL) * 512) = w;
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
__device__ __forceinline__ F8 unpack8(const Raw8<In>& r) {
    F8 f;
    if constexpr (sizeof(In) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f.p[2 * i] = make_float2(__uint_as_float(r.q[i].x), __uint_as_float(r.q[i].y));
            f.p[2 * i + 1] = make_float2(__uint_as_float(r.q[i].z), __uint_as_float(r.q[i].w));
        }
    } else {
        const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) f.p[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
    return f;
}
// amax_bits8 of a vector as loaded; bf16 two values an instruction.
template <class In>
__device__ __forceinline__ uint32_t amax_bits_raw(const Raw8<In>& r) {
    if constexpr (sizeof(In) == 2) {
        const uint4& q = r.q[0];
        const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu), __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
        return max(m & 0xFFFF0000u, m << 16);
    } else {
        return amax_bits8(unpack8<In>(r));
    }
}
// Rounds 8 values to the type (nearest even).
template <class In>
__device__ __forceinline__ Raw8<In> pack8(const F8& v) {
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

// ---- 16 columns a lane (rows on 32-byte boundaries, cols a multiple of 16) ---------------
// A lane holds an NVFP4 block or half an MXFP4 block: half the exchanges between
// lanes and half the work per scale of the 8-column form, and 32-byte accesses.
struct Word32 {
    uint32_t w[8];
};
__device__ __forceinline__ Word32 ld_global_32(const void* p) {
    Word32 r;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
                 : "l"(p));
    return r;
}
__device__ __forceinline__ void st_global_32(void* p, const Word32& r) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                 "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                 : "memory");
}
template <class In>
struct Raw16 {
    Word32 q[sizeof(In) / 2];
};
// Half `i` (0, 1) as a vector of 8 columns.
template <class In>
__device__ __forceinline__ Raw8<In> half_of(const Raw16<In>& r, int i) {
    Raw8<In> h;
    if constexpr (sizeof(In) == 2) {
        h.q[0] = make_uint4(r.q[0].w[4 * i], r.q[0].w[4 * i + 1], r.q[0].w[4 * i + 2], r.q[0].w[4 * i + 3]);
    } else {
        h.q[0] = make_uint4(r.q[i].w[0], r.q[i].w[1], r.q[i].w[2], r.q[i].w[3]);
        h.q[1] = make_uint4(r.q[i].w[4], r.q[i].w[5], r.q[i].w[6], r.q[i].w[7]);
    }
    return h;
}

}  // namespace dev
}  // namespace nq
