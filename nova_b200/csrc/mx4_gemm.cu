// mx4_gemm.cu -- product of two microscaled 4-bit operands on the sm_100a
// tensor cores (tcgen05 kind::mxf4 / kind::mxf4nvf4 with block scaling).
//
// Codes come in by TMA as bytes (two codes each, 128-byte swizzle: 256 columns
// of K a stage); block scales by TMA too, as the 512-byte tiles their layout
// consists of, then by tcgen05.cp into tensor memory, where the MMAs read them.
//
// k_mx4_pair (more than 64 rows): a cluster of two CTAs computes 256 x 256
//   tiles with cta_group::2, persistent, banded tile order.
// k_mx4_decode (up to 64 rows): operands swapped -- 128 rows of B are the MMA's
//   M side, the rows of A its N side; units of 128 rows whole, or their k-blocks
//   shared out so that every SM streams the same number of bytes.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>
#include <string>

#include "mx4.cuh"
#include "nq_internal.h"
#include "ptx.cuh"
#include "tmap.h"

namespace nq {
namespace {

using namespace dev;

constexpr int BKB = 128;  // bytes of codes of a row in a stage
constexpr int BK = 256;   // columns of K in a stage

struct MxEpi {
    void* out;
    int out_bf16;
    int tma_out;  // rows of the output are whole 16-byte units: stores by TMA
    float alpha;
    const float* row_scale;
    const float* col_scale;
    const float* bias;
};

// (acc * (alpha * row)) * col + bias, one rounding per step (absent vectors are 1 and -0).
__device__ __forceinline__ float mx_epi(float acc, float row, float cs, float b) {
    return __fadd_rn(__fmul_rn(__fmul_rn(acc, row), cs), b);
}
// Keeps the compiler from using registers that tcgen05.ld fills before the wait
// that precedes this call.
template <int NR>
__device__ __forceinline__ void after_tmem_ld(uint32_t (&r)[NR]) {
#pragma unroll
    for (int j = 0; j < NR; ++j) asm volatile("" : "+r"(r[j]));
}

// out = epi(0): products over no columns.
__global__ void __launch_bounds__(256) k_mx4_empty(int M, int N, MxEpi ep) {
    const size_t total = static_cast<size_t>(M) * N;
    for (size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x; i < total; i += static_cast<size_t>(gridDim.x) * 256) {
        const int n = static_cast<int>(i % N);
        const float v = ep.bias ? ep.bias[n] : 0.0f;
        if (ep.out_bf16) static_cast<uint16_t*>(ep.out)[i] = static_cast<uint16_t>(f32x2_to_bf16x2(v, 0.0f));
        else static_cast<float*>(ep.out)[i] = v;
    }
}

// ---------------- CTA pair, 256 x 256 tiles ----------------
// Bound by the tensor pipe and, run back to back, by the board's power: 4096^3
// MXFP4 27.4 us (5.0 PFLOP/s) on operands that stay in L2, 30.2 on changing ones, 34.8 for seconds on
// end at 1.61 GHz; 8192^3 NVFP4 194 us (5.7 PFLOP/s, tensor pipe 74%
// active, DRAM traffic 211 MB of 210), 8192 x 14336 x 4096 NVFP4 218 us (4.4
// PFLOP/s) for seconds on end, with SM clocks at 1.46 GHz under the cap.  Of those
// 218 us the operands' way into shared memory and the epilogue take about 30 each
// (the MMAs alone, on data already there: 161); the accumulators' handover between
// tiles takes about 1600 cycles of a tile's 10800.  Tiles of 256 x 192 with two whole
// accumulators hide that, but load 19% more and end at the same time (211 against
// 210 us, MXFP4) at a lower clock; stores from registers instead of
// staged TMA stores measured the same.
template <bool MX, bool BF16>
struct PairCfg {
    static constexpr int WORDS = MX ? 2 : 4;          // scale words (tiles) a stage
    static constexpr int A_BYTES = 128 * BKB;         // this CTA's 128 rows of A
    static constexpr int B_BYTES = 128 * BKB;         // its half of B's 256 rows
    static constexpr int SFA_BYTES = WORDS * 512;     // its rows' scales
    static constexpr int SFB_BYTES = 2 * WORDS * 512;  // all 256 rows' scales: both CTAs need them
    static constexpr int STAGE = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int STAGES = BF16 ? 5 : 4;
    static constexpr int SLOT = 32 * 32 * (BF16 ? 2 : 4);  // a 32 x 32 chunk of outputs
    static constexpr int EPI_WARPS = 8;
    static constexpr int COLS = EPI_WARPS * 256;      // per warp: a chunk's column scales and biases
    static constexpr int SMEM = 1024 + STAGES * STAGE + EPI_WARPS * 2 * SLOT + COLS + 256;
    static constexpr int THREADS = 32 * (2 + EPI_WARPS);
    // Tensor memory: the accumulators of consecutive tiles share half of their
    // columns, [0, 256) and [128, 384); behind them a ring of 10 scale words (4
    // columns for A, 8 for B): two and a half stages of NVFP4, all five of MXFP4.
    static constexpr int ACC1 = 128;
    static constexpr int SF = 384;
    static constexpr int RING = 10;
    static constexpr bool SF_WAIT = WORDS * STAGES > RING;
};

constexpr int M_BAND = 32;
// Bands of 32 row tiles; inside a band the row tiles run fastest, so that the
// clusters in flight share few panels of A and B.
__device__ __forceinline__ void pair_tile(int tile, int m_tiles, int n_tiles, int& mb, int& nb) {
    const int band = tile / (M_BAND * n_tiles);
    const int rows = min(M_BAND, m_tiles - band * M_BAND);
    const int local = tile - band * M_BAND * n_tiles;
    mb = band * M_BAND + local % rows;
    nb = local / rows;
}

// The i-th 32-column chunk of a tile that an epilogue warp of column group g
// drains: the half that the next tile's accumulator overlays comes first.
__device__ __forceinline__ int chunk_of(int acc, int g, int i) {
    return (((i < 2) == (acc == 0)) ? 4 : 0) + 2 * g + (i & 1);
}

// Tiles [0, whole) are dealt round-robin; where the rest fill at most half the
// clusters, each of them is done as two 256 x 128 halves by two clusters.
struct PairUnit {
    int tile;
    int half;  // 0: the whole tile, 1 / 2: its columns [0, 128) / [128, 256)
};
__device__ __forceinline__ int pair_units(int tiles, int whole, int cluster, int nclusters) {
    const int n = whole > cluster ? (whole - cluster + nclusters - 1) / nclusters : 0;
    return n + (cluster < 2 * (tiles - whole) ? 1 : 0);
}
__device__ __forceinline__ PairUnit pair_unit(int whole, int cluster, int nclusters, int j) {
    const int tile = cluster + j * nclusters;
    return tile < whole ? PairUnit{tile, 0} : PairUnit{whole + cluster / 2, 1 + (cluster & 1)};
}

template <bool MX, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg<MX, BF16>::THREADS, 1)
    k_mx4_pair(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
               const __grid_constant__ CUtensorMap tmBh, const __grid_constant__ CUtensorMap tmSA,
               const __grid_constant__ CUtensorMap tmSB, const __grid_constant__ CUtensorMap tmC, int M, int N, int K,
               int whole, MxEpi ep, uint32_t* err) {
    using C = PairCfg<MX, BF16>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sA = smem;
    uint8_t* sB = sA + C::STAGES * C::A_BYTES;
    uint8_t* sSA = sB + C::STAGES * C::B_BYTES;
    uint8_t* sSB = sSA + C::STAGES * C::SFA_BYTES;
    uint8_t* sEpi = sSB + C::STAGES * C::SFB_BYTES;
    uint8_t* sCols = sEpi + C::EPI_WARPS * 2 * C::SLOT;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sCols + C::COLS);
    uint64_t* full = bars;                  // [STAGES] leader: both CTAs' TMA -> MMA
    uint64_t* empty = full + C::STAGES;     // [STAGES] MMA -> each CTA's producer
    uint64_t* tfull = empty + C::STAGES;    // [2] MMA -> each CTA's epilogue
    uint64_t* tempty = tfull + 2;           // leader: 16 epilogue warps -> MMA, once a tile
    uint64_t* done = tempty + 1;            // leader: MMA drain
    uint64_t* mid = done + 1;               // [STAGES] leader: a stage's first two MMAs are complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mid + C::STAGES);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int cluster = blockIdx.x >> 1;
    const int nclusters = gridDim.x >> 1;
    const int m_tiles = (M + 255) / 256;
    const int n_tiles = (N + 255) / 256;
    const int kblocks = (K + BK - 1) / BK;
    const int units = pair_units(m_tiles * n_tiles, whole, cluster, nclusters);

    // Up to pdl_wait() nothing touches memory that an earlier kernel may write.
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&mid[s], 1);
        }
        mbar_init(&tfull[0], 1);
        mbar_init(&tfull[1], 1);
        mbar_init(tempty, 2 * C::EPI_WARPS);
        mbar_init(done, 1);
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        tma_prefetch_desc(&tmBh);
        tma_prefetch_desc(&tmSA);
        tma_prefetch_desc(&tmSB);
        if (ep.tma_out) tma_prefetch_desc(&tmC);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    pdl_wait();

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs) ----------------
        if (elect_one()) {
            const uint32_t full_leader = mapa_shared(smem_u32(full), 0);
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int j = 0; j < units && ok; ++j) {
                const PairUnit un = pair_unit(whole, cluster, nclusters, j);
                int mb, nb;
                pair_tile(un.tile, m_tiles, n_tiles, mb, nb);
                const int hi = un.half == 2 ? 1 : 0;
                const int brow = nb * 256 + (un.half ? 128 * hi + static_cast<int>(rank) * 64 : static_cast<int>(rank) * 128);
                for (int kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, err)) { ok = false; break; }
                    if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * (un.half ? C::STAGE - C::B_BYTES / 2 : C::STAGE));
                    const uint32_t fb = full_leader + 8u * stage;
                    tma_load_2d_pair(sA + stage * C::A_BYTES, &tmA, fb, kb * BKB, mb * 256 + rank * 128);
                    tma_load_2d_pair(sB + stage * C::B_BYTES, un.half ? &tmBh : &tmB, fb, kb * BKB, brow);
                    // 8-byte elements: 64 to a 512-byte scale tile; row blocks of 128
                    tma_load_2d_pair(sSA + stage * C::SFA_BYTES, &tmSA, fb, kb * C::WORDS * 64, mb * 2 + rank);
                    tma_load_2d_pair(sSB + stage * C::SFB_BYTES, &tmSB, fb, kb * C::WORDS * 64, nb * 2 + hi);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok) {
                for (int s = 0; s < C::STAGES; ++s) mbar_wait(&empty[s], phase ^ 1u, nullptr);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (leader CTA only) ----------------
        if (rank == 0 && elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            int it = 0;
            int word = 0;       // of the scale ring
            long long seq = 0;  // k-blocks issued
            for (; it < units && ok; ++it) {
                const uint32_t idesc = make_idesc_mx4(MX, 256u, pair_unit(whole, cluster, nclusters, it).half ? 128u : 256u);
                const uint32_t d_tmem = tmem_base + ((it & 1) ? C::ACC1 : 0);
                for (int kb = 0; kb < kblocks; ++kb, ++seq) {
                    if (!mbar_wait(&full[stage], phase, err)) { ok = false; break; }
                    if (C::SF_WAIT && seq >= 2) {
                        // The MMAs that read these scale words before are complete: the last of
                        // them are the first two of two k-blocks ago.  (The order of one thread's
                        // tcgen05 operations covers copy -> MMA, not MMA -> copy.)  Where the ring
                        // holds every stage's words, the stage itself says so.
                        int st = stage - 2;
                        uint32_t ph = phase;
                        if (st < 0) { st += C::STAGES; ph ^= 1u; }
                        if (!mbar_wait(&mid[st], ph, err)) { ok = false; break; }
                    }
                    tc_fence_after();
                    // Descriptors once a stage, then their address fields (16-byte units) by
                    // addition: built one by one they held the single issuing thread
                    // behind the tensor pipe (250 -> 230 us at 8192 x 14336 x 4096).
                    const uint64_t ga = smem_desc_rows16(smem_u32(sSA + stage * C::SFA_BYTES));
                    const uint64_t gb = smem_desc_rows16(smem_u32(sSB + stage * C::SFB_BYTES));
                    const uint64_t ad = smem_desc_sw128(smem_u32(sA + stage * C::A_BYTES), 16u, 1024u);
                    const uint64_t bd = smem_desc_sw128(smem_u32(sB + stage * C::B_BYTES), 16u, 1024u);
                    uint32_t sf[C::WORDS];
#pragma unroll
                    for (int w = 0; w < C::WORDS; ++w) {
                        sf[w] = tmem_base + C::SF + 12u * static_cast<uint32_t>(word);
                        if (++word == C::RING) word = 0;
                        tmem_cp_scales_pair(sf[w], ga + 32 * w);
                        tmem_cp_scales_pair(sf[w] + 4, gb + 32 * w);
                        tmem_cp_scales_pair(sf[w] + 8, gb + 32 * (C::WORDS + w));
                    }
                    if (kb == 0 && it > 0) {
                        // the previous tile's shared columns (and all of the tile before it) are drained
                        if (!mbar_wait(tempty, static_cast<uint32_t>(it - 1) & 1u, err)) { ok = false; break; }
                        tc_fence_after();
                    }
                    const int mmas = min(4, (K - kb * BK + 63) / 64);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (kk < mmas) {
                            const int w = MX ? kk / 2 : kk;
                            const uint32_t id = idesc | (MX ? idesc_scale_ids(2u * (kk & 1)) : 0u);
                            mma_mx4_pair<MX>(d_tmem, ad + 2 * kk, bd + 2 * kk, id, sf[w], sf[w] + 4, (kb > 0 || kk > 0) ? 1u : 0u);
                        }
                        if (C::SF_WAIT && kk == 1) tc_commit_pair_mc(&mid[stage], 0x1);
                    }
                    tc_commit_pair_mc(&empty[stage], 0x3);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
                if (ok) tc_commit_pair_mc(&tfull[it & 1], 0x3);
            }
            tc_commit_pair_mc(done, 0x1);
            mbar_wait(done, 0, err);
        }
    } else {
        // ---------------- epilogue (warps 2..9 of both CTAs) ----------------
        const int quarter = warp & 3;      // tensor memory lanes [32 * quarter, +32)
        const int g = (warp - 2) >> 2;     // column group: which four of the eight chunks
        const uint32_t tempty_leader = mapa_shared(smem_u32(tempty), 0);
        uint8_t* slots = sEpi + (warp - 2) * 2 * C::SLOT;
        float* cols = reinterpret_cast<float*>(sCols + (warp - 2) * 256);  // 32 column scales, 32 biases
        const bool has_cols = ep.col_scale, has_bias = ep.bias;
        int it = 0;
        int chunk_seq = 0;
        for (; it < units; ++it) {
            const int acc = it & 1;
            const PairUnit un = pair_unit(whole, cluster, nclusters, it);
            int mb, nb;
            pair_tile(un.tile, m_tiles, n_tiles, mb, nb);
            // the four chunks of a whole tile, or the two of a half in accumulator columns [0, 128)
            const int nchunks = un.half ? 2 : 4;
            const int half0 = un.half == 2 ? 128 : 0;
            auto chunk = [&](int i) { return un.half ? 2 * g + i : chunk_of(acc, g, i); };
            const int row0 = mb * 256 + static_cast<int>(rank) * 128 + quarter * 32;
            const int row = row0 + lane;
            const float f1 = (ep.row_scale && row < M) ? __fmul_rn(ep.alpha, __ldg(ep.row_scale + row)) : ep.alpha;
            const float2 f = make_float2(f1, f1);
            float cs[4], bs[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = min(nb * 256 + half0 + 32 * chunk(i) + lane, N - 1);
                cs[i] = ep.col_scale ? __ldg(ep.col_scale + c) : 1.0f;
                bs[i] = ep.bias ? __ldg(ep.bias + c) : -0.0f;
            }
            const bool ok = mbar_wait(&tfull[acc], static_cast<uint32_t>(it >> 1) & 1u, err);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (acc ? C::ACC1 : 0);
            uint32_t r[2][32];
            tmem_ld_32x32b_x32(taddr + 32 * chunk(0), r[0]);
            tmem_ld_32x32b_x32(taddr + 32 * chunk(1), r[1]);
            tmem_ld_wait();
            after_tmem_ld(r[0]);
            after_tmem_ld(r[1]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(tempty);
                else mbar_arrive_remote(tempty_leader);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= nchunks) break;
                const int col0 = nb * 256 + half0 + 32 * chunk(i);
                uint32_t (&cur)[32] = r[i & 1];
                if (i >= 2) {
                    tmem_ld_wait();
                    after_tmem_ld(cur);
                }
                if (col0 < N && row0 < M) {
                    uint8_t* slot = slots + (chunk_seq & 1) * C::SLOT;
                    if (ep.tma_out && lane == 0) bulk_wait_group_read<1>();  // the store two chunks ago has read this slot
                    if (has_cols) cols[lane] = cs[i];
                    if (has_bias) cols[32 + lane] = bs[i];
                    __syncwarp();
                    constexpr int PER = BF16 ? 8 : 4;  // outputs in 16 bytes
#pragma unroll
                    for (int j = 0; j < 32 / PER; ++j) {
                        float v[PER];
#pragma unroll
                        for (int t = 0; t < PER; t += 4) {
                            float2 lo = mul2(make_float2(__uint_as_float(cur[PER * j + t]), __uint_as_float(cur[PER * j + t + 1])), f);
                            float2 hi = mul2(make_float2(__uint_as_float(cur[PER * j + t + 2]), __uint_as_float(cur[PER * j + t + 3])), f);
                            if (has_cols) {
                                const float4 c4 = *reinterpret_cast<const float4*>(cols + PER * j + t);
                                lo = mul2(lo, make_float2(c4.x, c4.y));
                                hi = mul2(hi, make_float2(c4.z, c4.w));
                            }
                            if (has_bias) {
                                const float4 b4 = *reinterpret_cast<const float4*>(cols + 32 + PER * j + t);
                                lo = add2(lo, make_float2(b4.x, b4.y));
                                hi = add2(hi, make_float2(b4.z, b4.w));
                            }
                            v[t] = lo.x;
                            v[t + 1] = lo.y;
                            v[t + 2] = hi.x;
                            v[t + 3] = hi.y;
                        }
                        if (BF16) {
                            // 64-byte rows, 16-byte unit j at j ^ ((row >> 1) & 3)
                            *reinterpret_cast<uint4*>(slot + lane * 64 + 16 * (j ^ ((lane >> 1) & 3))) =
                                make_uint4(f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3]),
                                           f32x2_to_bf16x2(v[4 % PER], v[5 % PER]), f32x2_to_bf16x2(v[6 % PER], v[7 % PER]));
                        } else {
                            // 128-byte rows, 16-byte unit j at j ^ (row & 7)
                            *reinterpret_cast<uint4*>(slot + lane * 128 + 16 * (j ^ (lane & 7))) =
                                make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                        }
                    }
                    if (ep.tma_out) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&tmC, slot, col0, row0);
                            bulk_commit_group();
                        }
                    } else {
                        __syncwarp();
                        // a row of 32 outputs per step, one lane each
                        for (int q = 0; q < 32 && row0 + q < M; ++q) {
                            if (col0 + lane >= N) break;
                            const size_t at = static_cast<size_t>(row0 + q) * N + col0 + lane;
                            if (BF16)
                                static_cast<uint16_t*>(ep.out)[at] = *reinterpret_cast<const uint16_t*>(
                                    slot + q * 64 + 16 * ((lane >> 3) ^ ((q >> 1) & 3)) + 2 * (lane & 7));
                            else
                                static_cast<float*>(ep.out)[at] = *reinterpret_cast<const float*>(
                                    slot + q * 128 + 16 * ((lane >> 2) ^ (q & 7)) + 4 * (lane & 3));
                        }
                        __syncwarp();
                    }
                    ++chunk_seq;
                }
                if (i + 2 < nchunks) tmem_ld_32x32b_x32(taddr + 32 * chunk(i + 2), cur);
            }
        }
        if (lane == 0) bulk_wait_group_all();
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ---------------- up to 64 rows: swapped operands ----------------
// Units of 128 rows of B (the MMA's M side), dealt whole to the CTAs, or with
// `split` their k-blocks shared out: the k-blocks of all units in order are cut into one contiguous range a
// CTA.  The CTA that holds a unit's first k-block finishes it; a CTA that starts
// inside a unit parks its accumulators in its workspace row and raises its
// flag, and the owner adds the parts in range order: no atomics, the same sums
// every time.  Ranges go to the CTAs in reverse, so an owner waits for CTAs of
// lower index only: those are placed before it, and a grid that shares the GPU
// with another one still finishes.
// Bound by HBM where B is large: 16 x 28672 x 8192 NVFP4 23.8 us, 5.6 TB/s of B's
// codes and scales (85% of the measured copy rate; 64 rows 26.8 us).  What is missing: the first
// loads' latency, SMs that finish up to 3 us apart, the last epilogue.
template <bool MX, int BT>
struct DecodeCfg {
    static constexpr int WORDS = MX ? 2 : 4;
    static constexpr int W_BYTES = 128 * BKB;
    static constexpr int X_BYTES = BT * BKB;
    static constexpr int SF_BYTES = WORDS * 512;
    static constexpr int STAGE = W_BYTES + X_BYTES + 2 * SF_BYTES;
    static constexpr int OUT_BYTES = BT * 128 * 4;  // a slice of outputs or of raw accumulators
    static constexpr int BUDGET = 216 * 1024 - 2 * OUT_BYTES;
    static constexpr int STAGES = BUDGET / STAGE < 8 ? BUDGET / STAGE : 8;
    static constexpr int SMEM = 1024 + STAGES * STAGE + 2 * OUT_BYTES + BT * 4 + 256;
    static constexpr int SF = 128;           // tensor memory columns of the scales (accumulators below)
    static constexpr int SF_SLOT = 8 * WORDS;  // a slot for every stage's scales
    static_assert(SF + STAGES * SF_SLOT <= 512, "tensor memory");
    static constexpr int THREADS = 192;
};

__device__ __forceinline__ long long range_begin(long long total, int c, int G) { return total * c / G; }

// The later ranges [first, last] that hold the rest of a slice ending at k-block
// slice_end, when range `cta`'s part of it ends at s1 (first > last: none).
__device__ __forceinline__ void later_ranges(long long total, int cta, int G, long long s1, long long slice_end, int* first,
                                             int* last) {
    *first = cta + 1;
    *last = cta;
    if (s1 < slice_end) {
        int c = cta + 1;
        while (c + 1 < G && range_begin(total, c + 1, G) < slice_end) ++c;
        *last = c;
    }
}

template <bool MX, int BT>
__global__ void __launch_bounds__(192, 1)
    k_mx4_decode(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                 const __grid_constant__ CUtensorMap tmSW, const __grid_constant__ CUtensorMap tmSX,
                 const __grid_constant__ CUtensorMap tmO, int M, int N, int K, int split, MxEpi ep, uint32_t* ws, uint32_t* flags,
                 uint32_t* err) {
    using C = DecodeCfg<MX, BT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sX = sW + C::STAGES * C::W_BYTES;
    uint8_t* sSW = sX + C::STAGES * C::X_BYTES;
    uint8_t* sSX = sSW + C::STAGES * C::SF_BYTES;
    uint8_t* sOut = sSX + C::STAGES * C::SF_BYTES;                          // outputs or a part to park
    uint32_t* sPart = reinterpret_cast<uint32_t*>(sOut + C::OUT_BYTES);     // a later CTA's parked part
    float* sRs = reinterpret_cast<float*>(sOut + 2 * C::OUT_BYTES);
    uint64_t* full = reinterpret_cast<uint64_t*>(sRs + BT);
    uint64_t* empty = full + C::STAGES;
    uint64_t* tfull = empty + C::STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* done = tempty + 2;
    uint64_t* pfull = done + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pfull + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int G = gridDim.x;
    const int kblocks = (K + BK - 1) / BK;
    const int unit_n = (N + 127) / 128;
    const long long total = static_cast<long long>(unit_n) * kblocks;
    const int cta = G - 1 - static_cast<int>(blockIdx.x);  // this CTA's range (split)
    // work positions: k-blocks [b0, b1) of all units in order, or units b0, b0 + G, ... below b1
    const long long b0 = split ? range_begin(total, cta, G) : blockIdx.x;
    const long long b1 = split ? range_begin(total, cta + 1, G) : unit_n;
    struct Seg {
        int unit, kb0, kb1;
        long long next;
    };
    auto segment = [&](long long pos) {
        if (!split) return Seg{static_cast<int>(pos), 0, kblocks, pos + G};
        const int unit = static_cast<int>(pos / kblocks);
        const long long u0 = static_cast<long long>(unit) * kblocks;
        const long long next = min(b1, u0 + kblocks);
        return Seg{unit, static_cast<int>(pos - u0), static_cast<int>(next - u0), next};
    };
    // split: does this CTA's last segment own a unit whose rest is one later range's?
    int lc_first = 1, lc_last = 0;
    bool last_fetch = false;
    if (split) {
        const int last = static_cast<int>((b1 - 1) / kblocks);
        later_ranges(total, cta, G, b1, static_cast<long long>(last + 1) * kblocks, &lc_first, &lc_last);
        last_fetch = b0 <= static_cast<long long>(last) * kblocks && lc_last == lc_first;
    }

    // Up to pdl_wait() nothing touches memory that an earlier kernel may write
    // (the prefetch only fills L2, which is coherent).
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 128);
        }
        mbar_init(done, 1);
        mbar_init(pfull, 1);
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmSW);
        tma_prefetch_desc(&tmSX);
        if (ep.tma_out) tma_prefetch_desc(&tmO);
        const Seg g = segment(b0);
        for (int kb = g.kb0; kb < g.kb1 && kb < g.kb0 + 2 * C::STAGES; ++kb) {  // (a quantize before it takes about 3 us)
            tma_prefetch_l2_2d(&tmW, kb * BKB, g.unit * 128);
            tma_prefetch_l2_2d(&tmSW, kb * C::WORDS * 64, g.unit);
        }
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (long long pos = b0; pos < b1 && ok;) {
                const Seg g = segment(pos);
                pos = g.next;
                for (int kb = g.kb0; kb < g.kb1; ++kb) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, err)) { ok = false; break; }
                    mbar_arrive_expect_tx(&full[stage], C::STAGE);
                    tma_load_2d(sW + stage * C::W_BYTES, &tmW, &full[stage], kb * BKB, g.unit * 128);
                    tma_load_2d(sSW + stage * C::SF_BYTES, &tmSW, &full[stage], kb * C::WORDS * 64, g.unit);
                    tma_load_2d(sX + stage * C::X_BYTES, &tmX, &full[stage], kb * BKB, 0);
                    tma_load_2d(sSX + stage * C::SF_BYTES, &tmSX, &full[stage], kb * C::WORDS * 64, 0);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
            if (!ok) {
                // the copies in flight land before the CTA ends: the stages are freed by the MMAs that read them
                for (int s = 0; s < C::STAGES; ++s) mbar_wait(&empty[s], phase ^ 1u, nullptr);
            }
            if (last_fetch) {
                // the later CTA parked its part long ago (it was the start of its range)
                if (wait_flag_geq(flags + lc_first * 4, 1u, err)) {
                    fence_proxy_async_global();
                    mbar_arrive_expect_tx(pfull, C::OUT_BYTES);
                    bulk_load_1d(sPart, ws + static_cast<size_t>(lc_first) * BT * 128, C::OUT_BYTES, pfull);
                } else {
                    mbar_arrive(pfull);
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = make_idesc_mx4(MX, 128u, BT);
            int stage = 0;
            uint32_t phase = 0;
            int seg = 0;
            bool ok = true;
            for (long long pos = b0; pos < b1 && ok; ++seg) {
                const Seg g = segment(pos);
                pos = g.next;
                const int acc = seg & 1;
                if (!mbar_wait(&tempty[acc], ((static_cast<uint32_t>(seg) >> 1) & 1u) ^ 1u, err)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BT);
                for (int kb = g.kb0; kb < g.kb1; ++kb) {
                    if (!mbar_wait(&full[stage], phase, err)) { ok = false; break; }
                    tc_fence_after();
                    // (the MMAs that read this slot before have freed the stage)
                    const uint32_t sfw = tmem_base + C::SF + static_cast<uint32_t>(stage) * C::SF_SLOT;
                    const uint32_t sfx = sfw + 4 * C::WORDS;
                    const uint64_t gw = smem_desc_rows16(smem_u32(sSW + stage * C::SF_BYTES));
                    const uint64_t gx = smem_desc_rows16(smem_u32(sSX + stage * C::SF_BYTES));
                    const uint64_t ad = smem_desc_sw128(smem_u32(sW + stage * C::W_BYTES), 16u, 1024u);
                    const uint64_t bd = smem_desc_sw128(smem_u32(sX + stage * C::X_BYTES), 16u, 1024u);
#pragma unroll
                    for (int w = 0; w < C::WORDS; ++w) {
                        tmem_cp_scales(sfw + 4 * w, gw + 32 * w);
                        tmem_cp_scales(sfx + 4 * w, gx + 32 * w);
                    }
                    const int mmas = min(4, (K - kb * BK + 63) / 64);
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (kk >= mmas) break;
                        const int w = MX ? kk / 2 : kk;
                        const uint32_t id = idesc | (MX ? idesc_scale_ids(2u * (kk & 1)) : 0u);
                        mma_mx4<MX>(d_tmem, ad + 2 * kk, bd + 2 * kk, id, sfw + 4 * w, sfx + 4 * w, (kb > g.kb0 || kk > 0) ? 1u : 0u);
                    }
                    tc_commit(&empty[stage]);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
                if (ok) tc_commit(&tfull[acc]);
            }
            tc_commit(done);
            mbar_wait(done, 0, err);
        }
    } else {
        const int quarter = warp & 3;
        const int nl = quarter * 32 + lane;  // row of B within the slice
        const bool issuer = threadIdx.x == 64;
        // After a wait that ran out (error bit set) the warps still pass every
        // named barrier in the same order, with garbage data: none may leave
        // the protocol early while the others wait at a barrier.
        bool failed = false;
        int seg = 0;
        if (threadIdx.x < 64 + BT) {  // (read behind the barriers below)
            const int t = threadIdx.x - 64;
            sRs[t] = (ep.row_scale && t < M) ? __fmul_rn(ep.alpha, __ldg(ep.row_scale + t)) : ep.alpha;
        }
        uint32_t* sOut32 = reinterpret_cast<uint32_t*>(sOut);
        for (long long pos = b0; pos < b1; ++seg) {
            const Seg g = segment(pos);
            pos = g.next;
            const bool head = g.kb0 == 0;  // this CTA holds the unit's first k-block
            const int acc = seg & 1;
            const uint32_t tpar = (static_cast<uint32_t>(seg) >> 1) & 1u;
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BT);
            int c_first = 1, c_last = 0;
            if (split && head)
                later_ranges(total, cta, G, g.next, static_cast<long long>(g.unit + 1) * kblocks, &c_first, &c_last);
            const bool parts = c_last >= c_first;
            const bool fetched = parts && g.next == b1 && last_fetch;  // the producer bulk-loads the part
            const int n = g.unit * 128 + nl;
            const bool mine = n < N;
            const float cs = head && ep.col_scale && mine ? __ldg(ep.col_scale + n) : 1.0f;
            const float bs = head && ep.bias && mine ? __ldg(ep.bias + n) : -0.0f;
            if (parts && !fetched) {
                if (lane == 0)
                    for (int c = c_first; c <= c_last; ++c) wait_flag_geq(flags + c * 4, 1u, err);
                __syncwarp();
            }
            if (fetched && !failed && !__all_sync(0xffffffffu, mbar_wait(pfull, 0, err))) failed = true;
            if (!failed && !__all_sync(0xffffffffu, mbar_wait(&tfull[acc], tpar, err))) failed = true;
            tc_fence_after();
            // the previous bulk store has read sOut, and every warp has passed its
            // flag wait (so the flags can be cleared below)
            named_bar_sync(1, 128);
            uint32_t r[BT];  // this thread's row of B against every row of A
#pragma unroll
            for (int c = 0; c < BT; c += 16) tmem_ld_32x32b_x16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(r + c));
            tmem_ld_wait();
            after_tmem_ld(r);
            if (!head) {
#pragma unroll
                for (int j = 0; j < BT; ++j) sOut32[j * 128 + nl] = r[j];
            } else {
                if (fetched) {
#pragma unroll
                    for (int j = 0; j < BT; ++j)
                        r[j] = __float_as_uint(__fadd_rn(__uint_as_float(r[j]), __uint_as_float(sPart[j * 128 + nl])));
                } else if (parts) {
                    // a whole part's loads in flight at once
                    for (int cc = c_first; cc <= c_last; ++cc) {
                        const uint32_t* part = ws + static_cast<size_t>(cc) * BT * 128 + nl;
                        uint32_t q[BT];
#pragma unroll
                        for (int j = 0; j < BT; ++j) q[j] = __ldcg(part + j * 128);
#pragma unroll
                        for (int j = 0; j < BT; ++j) r[j] = __float_as_uint(__fadd_rn(__uint_as_float(r[j]), __uint_as_float(q[j])));
                    }
                }
                // [row of A][row of B] in the output type
#pragma unroll
                for (int j = 0; j < BT; j += 2) {
                    const float v0 = mx_epi(__uint_as_float(r[j]), sRs[j], cs, bs);
                    const float v1 = mx_epi(__uint_as_float(r[j + 1]), sRs[j + 1], cs, bs);
                    if (ep.out_bf16) {
                        const uint32_t p2 = f32x2_to_bf16x2(v0, v1);
                        reinterpret_cast<uint16_t*>(sOut)[j * 128 + nl] = static_cast<uint16_t>(p2);
                        reinterpret_cast<uint16_t*>(sOut)[(j + 1) * 128 + nl] = static_cast<uint16_t>(p2 >> 16);
                    } else {
                        sOut32[j * 128 + nl] = __float_as_uint(v0);
                        sOut32[(j + 1) * 128 + nl] = __float_as_uint(v1);
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(&tempty[acc]);
            fence_proxy_async_smem();
            named_bar_sync(1, 128);
            if (!head) {
                // park with one bulk store, then raise the flag
                if (issuer) {
                    bulk_store_1d(ws + static_cast<size_t>(cta) * BT * 128, sOut, C::OUT_BYTES);
                    bulk_commit_group();
                    bulk_wait_group<0>();  // the part is in global memory
                    fence_proxy_async_global();
                    __threadfence();
                    atomicAdd(flags + cta * 4, 1u);
                }
            } else {
                if (ep.tma_out) {
                    if (issuer) {
                        tma_store_2d(&tmO, sOut, g.unit * 128, 0);  // clips rows >= M and columns >= N
                        bulk_commit_group();
                        bulk_wait_group_read<0>();
                    }
                } else if (mine) {
                    for (int t = 0; t < M; ++t) {
                        const size_t at = static_cast<size_t>(t) * N + n;
                        if (ep.out_bf16) static_cast<uint16_t*>(ep.out)[at] = reinterpret_cast<uint16_t*>(sOut)[t * 128 + nl];
                        else static_cast<uint32_t*>(ep.out)[at] = sOut32[t * 128 + nl];
                    }
                }
                // each parked part has exactly one reader (a CTA parks at most the
                // first segment of its range): clear its flag for the next launch
                if (issuer)
                    for (int cc = c_first; cc <= c_last; ++cc) flags[cc * 4] = 0u;
            }
        }
        if (issuer) bulk_wait_group<0>();
    }
    __syncwarp();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ---------------- host side ----------------
// 2-D map of block scales: rows of `words` 512-byte tiles (8-byte elements, 64
// to a tile), one row per 128 rows of the operand.
nq_status_t make_scale_map(CUtensorMap* map, const void* base, int rows, int words, uint32_t box_words, uint32_t box_rows) {
    EncodeTiledFn fn;
    nq_status_t st = get_encode_fn(&fn);
    if (st != NQ_SUCCESS) return st;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(words) * 64, (static_cast<cuuint64_t>(rows) + 127) / 128};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(words) * 512};
    cuuint32_t box[2] = {box_words * 64, box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NQ_ERROR_CUDA, "cuTensorMapEncodeTiled (scales) failed (" + std::to_string(int(r)) + ")");
    return NQ_SUCCESS;
}

nq_status_t make_out_map(CUtensorMap* map, const MxEpi& ep, int m, int n, uint32_t box_cols, uint32_t box_rows, bool swizzle) {
    EncodeTiledFn fn;
    nq_status_t st = get_encode_fn(&fn);
    if (st != NQ_SUCCESS) return st;
    const int es = ep.out_bf16 ? 2 : 4;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(n), static_cast<cuuint64_t>(m)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(n) * es};
    cuuint32_t box[2] = {box_cols, box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapSwizzle sw = !swizzle ? CU_TENSOR_MAP_SWIZZLE_NONE
                                           : (ep.out_bf16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    CUresult r = fn(map, ep.out_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, ep.out, dims,
                    strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NQ_ERROR_CUDA, "cuTensorMapEncodeTiled (output) failed (" + std::to_string(int(r)) + ")");
    return NQ_SUCCESS;
}

struct Operands {
    const uint8_t *a, *sa, *b, *sb;
    int m, n, k;
};

template <class F>
nq_status_t smem_attr(F kern, int bytes, int device, std::atomic<uint64_t>* flags) {
    static std::mutex mu;
    return once_per_device(*flags, mu, device, [&]() -> nq_status_t {
        NQ_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                      "cudaFuncSetAttribute(nq_gemm_mx4)");
        return NQ_SUCCESS;
    });
}

template <bool MX, bool BF16>
nq_status_t launch_pair(const Operands& o, const MxEpi& ep, const DeviceInfo& di, cudaStream_t s) {
    using C = PairCfg<MX, BF16>;
    const uint64_t pitch = mx4_pitch(o.k);
    const int words = mx4_words(o.k, MX ? 32 : 16);
    CUtensorMap ma, mb, mbh, msa, msb, mc;
    std::memset(&mc, 0, sizeof(mc));
    nq_status_t st = make_map(&ma, o.a, pitch, o.m, pitch, BKB, 128);
    if (st == NQ_SUCCESS) st = make_map(&mb, o.b, pitch, o.n, pitch, BKB, 128);
    if (st == NQ_SUCCESS) st = make_map(&mbh, o.b, pitch, o.n, pitch, BKB, 64);
    if (st == NQ_SUCCESS) st = make_scale_map(&msa, o.sa, o.m, words, C::WORDS, 1);
    if (st == NQ_SUCCESS) st = make_scale_map(&msb, o.sb, o.n, words, C::WORDS, 2);
    if (st == NQ_SUCCESS && ep.tma_out) st = make_out_map(&mc, ep, o.m, o.n, 32, 32, true);
    if (st != NQ_SUCCESS) return st;
    auto kern = k_mx4_pair<MX, BF16>;
    static std::atomic<uint64_t> attr_set{0};
    st = smem_attr(kern, C::SMEM, di.device, &attr_set);
    if (st != NQ_SUCCESS) return st;
    static std::atomic<int> max_clusters[64];
    int resident = max_clusters[di.device & 63].load(std::memory_order_relaxed);
    if (!resident) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (di.sm_count / 2));
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        if (cudaOccupancyMaxActiveClusters(&resident, kern, &cfg) != cudaSuccess || resident <= 0) {
            cudaGetLastError();
            resident = di.sm_count / 2;
        }
        max_clusters[di.device & 63].store(resident, std::memory_order_relaxed);
    }
    const long long tiles = static_cast<long long>((o.m + 255) / 256) * ((o.n + 255) / 256);
    if (tiles > (1 << 30)) return fail(NQ_ERROR_UNSUPPORTED, "nq_gemm_mx4: more than 2^30 output tiles");
    // A last wave that fills at most half the clusters runs as half tiles: the
    // tail takes half a tile's time (4096^3, 3.46 waves: 28.9 -> 27.4 us).
    const int rest = static_cast<int>(tiles % resident);
    const int whole = static_cast<int>(2 * rest <= resident ? tiles - rest : tiles);
    const long long units = whole < tiles ? std::max<long long>(std::min<long long>(whole, resident), 2 * rest) : tiles;
    const int clusters = static_cast<int>(std::max<long long>(1, std::min<long long>(units, resident)));
    return cuda_status(launch_pdl(kern, dim3(2 * clusters), dim3(C::THREADS), C::SMEM, s, ma, mb, mbh, msa, msb, mc, o.m, o.n, o.k,
                                  whole, ep, device_error_word()),
                       "nq_gemm_mx4 (CTA pair)");
}

template <bool MX, int BT>
nq_status_t launch_decode(const Operands& o, const MxEpi& ep, int split, int grid, const DeviceInfo& di, cudaStream_t s) {
    using C = DecodeCfg<MX, BT>;
    const uint64_t pitch = mx4_pitch(o.k);
    const int words = mx4_words(o.k, MX ? 32 : 16);
    CUtensorMap mw, mx, msw, msx, mo;
    std::memset(&mo, 0, sizeof(mo));
    nq_status_t st = make_map(&mw, o.b, pitch, o.n, pitch, BKB, 128);
    if (st == NQ_SUCCESS) st = make_map(&mx, o.a, pitch, o.m, pitch, BKB, BT);
    if (st == NQ_SUCCESS) st = make_scale_map(&msw, o.sb, o.n, words, C::WORDS, 1);
    if (st == NQ_SUCCESS) st = make_scale_map(&msx, o.sa, o.m, words, C::WORDS, 1);
    if (st == NQ_SUCCESS && ep.tma_out) st = make_out_map(&mo, ep, o.m, o.n, 128, BT, false);
    if (st != NQ_SUCCESS) return st;
    auto kern = k_mx4_decode<MX, BT>;
    static std::atomic<uint64_t> attr_set{0};
    st = smem_attr(kern, C::SMEM, di.device, &attr_set);
    if (st != NQ_SUCCESS) return st;
    uint32_t* flags = nullptr;
    void* ws = nullptr;
    cudaError_t e = cudaSuccess;
    if (split) {
        // per CTA one parked part and one flag (stride 4) of the stream's flag words,
        // which every launch leaves cleared
        const size_t ws_bytes = static_cast<size_t>(grid) * C::OUT_BYTES;
        const size_t fl_bytes = static_cast<size_t>(grid) * 4 * 4;
        st = stream_flags(&flags, grid * 4, s);
        if (st != NQ_SUCCESS) return st;
        st = scratch_alloc(&ws, ws_bytes + (flags ? 0 : fl_bytes), s);
        if (st != NQ_SUCCESS) return st;
        if (!flags) {
            // inside a graph capture: flags of this launch, cleared by a memset node
            flags = reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + ws_bytes);
            e = cudaMemsetAsync(flags, 0, fl_bytes, s);
        }
    }
    if (e == cudaSuccess)
        e = launch_pdl(kern, dim3(grid), dim3(C::THREADS), C::SMEM, s, mw, mx, msw, msx, mo, o.m, o.n, o.k, split, ep,
                       static_cast<uint32_t*>(ws), flags, device_error_word());
    scratch_free(ws, s);
    return cuda_status(e, "nq_gemm_mx4 (few rows)");
}

template <bool MX>
nq_status_t decode(const Operands& o, const MxEpi& ep, int split, int grid, const DeviceInfo& di, cudaStream_t s) {
    if (o.m <= 16) return launch_decode<MX, 16>(o, ep, split, grid, di, s);
    if (o.m <= 32) return launch_decode<MX, 32>(o, ep, split, grid, di, s);
    return launch_decode<MX, 64>(o, ep, split, grid, di, s);
}

// Whole units or shared-out k-blocks, and on how many CTAs: the smallest of a few
// estimates (us).  A k-block takes a CTA 0.27 us (its MMAs and copies) or its
// share of HBM, whichever is longer (fewer CTAs reach two thirds of it); whole units cost 2.9 us besides, shared-out
// ones 4.2 us and a part's way through memory for each CTA of a unit (0.45 us at 16
// rows, 1 us at 64).  Measured, NVFP4, whole / shared out: 16 x 28672 x 8192 26.7 /
// 24.7, 1 x 4096 x 4096 7.4 / 7.6, 4 x 4096 x 28672 32.9 / 17.0, 16 x 5000 x 3000
// 6.4 / 7.5.
struct DecodePlan {
    int split, grid;
};
DecodePlan plan_decode(const Operands& o, bool mx, int sms) {
    const long long units = (static_cast<long long>(o.n) + 127) / 128;
    const long long kblocks = (o.k + BK - 1) / BK;
    const double share = (mx ? 17.4e3 : 18.4e3) * sms / 6.5e6;  // us a k-block with every SM streaming
    auto t_kb = [&](double active) { return std::max(0.27, std::min(share, 1.5 * share * active / sms)); };
    DecodePlan best{0, static_cast<int>(std::min<long long>(units, sms))};
    const long long rest = units % sms;
    double best_us = 2.9 + static_cast<double>(kblocks) *
                               (static_cast<double>(units / sms) * t_kb(sms) + (rest ? t_kb(static_cast<double>(rest)) : 0.0));
    const double part_us = o.m <= 16 ? 0.45 : (o.m <= 32 ? 0.6 : 1.0);
    auto offer = [&](long long grid, double parts) {
        if (grid < 1 || grid > units * kblocks) return;
        const double us = 4.2 + parts * part_us + static_cast<double>(units * kblocks) / grid * t_kb(static_cast<double>(grid));
        if (us < best_us) {
            best_us = us;
            best = DecodePlan{1, static_cast<int>(grid)};
        }
    };
    offer(sms, static_cast<double>(sms) / units + 1.0);
    for (long long p = 2; p <= kblocks && units * p <= sms; ++p) offer(units * p, static_cast<double>(p));
    return best;
}

template <bool MX>
nq_status_t launch_gemm(const Operands& o, const MxEpi& ep, const DeviceInfo& di, cudaStream_t s) {
    if (o.m <= 64) {
        const DecodePlan p = plan_decode(o, MX, di.sm_count);
        return decode<MX>(o, ep, p.split, p.grid, di, s);
    }
    return ep.out_bf16 ? launch_pair<MX, true>(o, ep, di, s) : launch_pair<MX, false>(o, ep, di, s);
}

nq_status_t bad(const char* what) { return fail(NQ_ERROR_INVALID_VALUE, std::string("nq_gemm_mx4: ") + what); }

}  // namespace
}  // namespace nq

extern "C" nq_status_t nq_gemm_mx4(const nq_gemm_mx4_desc_t* d, const uint8_t* a_codes, const uint8_t* a_scales,
                                   const uint8_t* b_codes, const uint8_t* b_scales, void* out, nq_stream_t s) {
    using namespace nq;
    if (!d) return bad("null descriptor");
    if (d->m < 0 || d->n < 0 || d->k < 0) return bad("negative size");
    if (d->k > (1 << 30)) return fail(NQ_ERROR_UNSUPPORTED, "nq_gemm_mx4: more than 2^30 columns");
    if (d->m > (1 << 30) || d->n > (1 << 30)) return fail(NQ_ERROR_UNSUPPORTED, "nq_gemm_mx4: more than 2^30 rows");
    if (d->format != NQ_MXFP4 && d->format != NQ_NVFP4) return bad("format");
    if (d->out_dtype != NQ_F32 && d->out_dtype != NQ_BF16) return bad("out_dtype must be NQ_F32 or NQ_BF16");
    if (d->m == 0 || d->n == 0) return NQ_SUCCESS;
    if (!out || (d->k > 0 && (!a_codes || !a_scales || !b_codes || !b_scales))) return bad("null pointer");
    if (!aligned16(a_codes) || !aligned16(a_scales) || !aligned16(b_codes) || !aligned16(b_scales))
        return bad("codes and block scales must be 16-byte aligned");
    if (!aligned_to(out, d->out_dtype) || !aligned_to(d->row_scale, NQ_F32) || !aligned_to(d->col_scale, NQ_F32) ||
        !aligned_to(d->bias, NQ_F32))
        return bad("a pointer is not aligned to its type");
    DeviceInfo di;
    nq_status_t st = current_device(&di);
    if (st != NQ_SUCCESS) return st;
    const bool bf = d->out_dtype == NQ_BF16;
    const MxEpi ep{out, bf, aligned16(out) && static_cast<size_t>(d->n) * (bf ? 2 : 4) % 16 == 0, d->alpha,
                   d->row_scale, d->col_scale, d->bias};
    if (d->k == 0) {
        k_mx4_empty<<<di.sm_count, 256, 0, s>>>(d->m, d->n, ep);
        NQ_LAUNCH_CHECK("nq_gemm_mx4 (no columns)");
        return NQ_SUCCESS;
    }
    const Operands o{a_codes, a_scales, b_codes, b_scales, d->m, d->n, d->k};
    return d->format == NQ_MXFP4 ? launch_gemm<true>(o, ep, di, s) : launch_gemm<false>(o, ep, di, s);
}
