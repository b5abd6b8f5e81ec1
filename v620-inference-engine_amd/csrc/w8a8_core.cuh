// Shared main loop of the int8 x int8 products (W8A8): one block computes a
// BM x BN tile of Q (int8 rows, K long) times W^T (int8 weight rows, as the
// checkpoint holds them: row-major), summed exactly in int32 on
// v_mfma_i32_32x32x32_i8.
//
// The sums are whole numbers, so neither the tile, nor how K is split over
// stages and waves, nor the batch changes a result: every shape of this loop
// gives the same bits, and a variant is chosen by speed alone.
//
// Schedule. K runs in stages of 128 bytes through NS buffers of LDS, filled by
// direct global -> LDS loads (a wave instruction moves 8 rows of 128 bytes,
// whole cache lines, from any row addresses: gathered rows cost the same as
// neighbours) NS - 1 stages ahead. One barrier per stage: a wave waits for its
// own loads of the stage, and the barrier then makes everyone's visible and
// tells that the buffer of the stage before is free for the next loads.
// The waves are WM x WN over the tile and KW over the 32-wide slabs of a
// stage; the KW partial sums meet in LDS at the end.
#pragma once

#include <type_traits>

#include "q4_common.cuh"

namespace qwq4 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int W8_KB = 128;  // K bytes per stage

// What a lane loads for K columns past the row's end (K need not be a
// multiple of 128): zeros, from memory that is always there.
static __device__ const uint4 w8_zeros = {0u, 0u, 0u, 0u};

// Byte offset of 16-byte chunk c (0..7) of row r in a [rows][128] stage. A
// fragment read takes 32 consecutive rows at chunk c (lanes 0-31) and c + 1
// (lanes 32-63); under this XOR its 16-lane parts fall on distinct banks.
__device__ __forceinline__ int w8_swz_x(int r) { return (r & 7) ^ ((r >> 3) & 1); }
__device__ __forceinline__ int w8_swz(int r, int c) { return r * W8_KB + ((c ^ w8_swz_x(r)) << 4); }

__device__ __forceinline__ i32x16 w8_mfma(const uint4 &a, const uint4 &b, const i32x16 &c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0,
                                                 0);
}

template <int BM_, int BN_, int WM_, int WN_, int KW_, int NS_>
struct W8Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KW = KW_, NS = NS_;
    static constexpr int NW = WM * WN * KW, THREADS = NW * WAVE;
    static constexpr int MT = BM / 32 / WM, NT = BN / 32 / WN;  // 32 x 32 tiles per wave
    static constexpr int AJ = BM / 8 / NW, BJ = BN / 8 / NW;    // load instructions per wave and stage
    static constexpr int STAGE = (BM + BN) * W8_KB;             // bytes of one buffer
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "tile");
    static_assert(KW == 1 || KW == 2 || KW == 4, "a stage has 4 slabs");
    static_assert(NS >= 2 && NS <= 4 && (KW == 1 || KW <= NS + 1), "one buffer per partial sum");
    static_assert(KW == 1 || WM * WN == 1, "partial sums are exchanged per wave tile");
    static_assert(KW == 1 || BM * BN * 4 <= STAGE, "a partial sum fits a buffer");

    // The tile row that part j of this lane's loads belongs to: A rows for
    // j < AJ, weight rows likewise for j < BJ.
    __device__ static __forceinline__ int load_row(int j) {
        return (j * NW + int(threadIdx.x) / WAVE) * 8 + int(threadIdx.x) % WAVE / 8;
    }
    // The chunk of that row it loads (the LDS slot is lane % 8).
    __device__ static __forceinline__ int load_chunk(int j) {
        return (int(threadIdx.x) % 8) ^ w8_swz_x(load_row(j));
    }
    // Wave coordinates, and the tile row / column of a lane's accumulator
    // element: row 32 i + ..(r), column 32 j + lane % 32 of the wave's part.
    __device__ static __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE); }
    __device__ static __forceinline__ int m_of(int i, int r) {
        return (wave() / KW / WN * MT + i) * 32 + 8 * (r / 4) + 4 * (int(threadIdx.x) % WAVE / 32) + r % 4;
    }
    __device__ static __forceinline__ int n_of(int j) {
        return (wave() / KW % WN * NT + j) * 32 + int(threadIdx.x) % 32;
    }
};

// Waits until at most N vector-memory operations of this wave are in flight
// and its LDS reads are done, then the block's barrier. Nothing that touches
// memory moves across.
template <int N>
__device__ __forceinline__ void w8_stage_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (0 << 8));  // vmcnt N, lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// acc += the tile's sums over K (a multiple of 16, >= 16). ap[j] / bp[j]: the
// start of the int8 row load_row(j) of Q / W (any valid row where the tile
// passes the matrix). With KW > 1 the sums end in the waves with wave % KW
// == 0 (acc of the others is void); returns whether this wave holds sums.
// The LDS is not free for reuse until the block's next barrier. (USE tags the
// caller: each call site instantiates its own specialization; the host
// compilation pass rejects a second call site of a shared one.)
template <class S, int USE>
__device__ __forceinline__ bool w8_tile(const int8_t *(&ap)[S::AJ], const int8_t *(&bp)[S::BJ], int K,
                                        i32x16 (&acc)[S::MT][S::NT]) {
    constexpr int NS = S::NS, LPW = S::AJ + S::BJ;
    __shared__ __align__(16) unsigned char s0[S::STAGE], s1[S::STAGE];
    __shared__ __align__(16) unsigned char s2[NS > 2 ? S::STAGE : 16], s3[NS > 3 ? S::STAGE : 16];
    const int wave = S::wave(), lane = int(threadIdx.x) % WAVE, l32 = lane % 32, lh = lane / 32;
    const int nk = (K + W8_KB - 1) / W8_KB;
    // (distinct arrays picked at compile time: the compiler then sees that the
    // loads in flight into one do not touch the buffer being read)
    auto buf = [&](auto i) -> unsigned char * {
        if constexpr (decltype(i)::value == 0) return s0;
        else if constexpr (decltype(i)::value == 1) return s1;
        else if constexpr (decltype(i)::value == 2) return s2;
        else return s3;
    };
    auto issue = [&](int ks, unsigned char *dst) {
        const int k0 = ks * W8_KB;
        if (k0 + W8_KB <= K) {
#pragma unroll
            for (int j = 0; j < S::AJ; ++j)
                __builtin_amdgcn_global_load_lds(ap[j] + k0 + S::load_chunk(j) * 16, dst + (j * S::NW + wave) * 1024, 16,
                                                 0, 0);
#pragma unroll
            for (int j = 0; j < S::BJ; ++j)
                __builtin_amdgcn_global_load_lds(bp[j] + k0 + S::load_chunk(j) * 16,
                                                 dst + S::BM * W8_KB + (j * S::NW + wave) * 1024, 16, 0, 0);
        } else {
            const int8_t *z = reinterpret_cast<const int8_t *>(&w8_zeros);
#pragma unroll
            for (int j = 0; j < S::AJ; ++j) {
                const int k = k0 + S::load_chunk(j) * 16;
                __builtin_amdgcn_global_load_lds(k < K ? ap[j] + k : z, dst + (j * S::NW + wave) * 1024, 16, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < S::BJ; ++j) {
                const int k = k0 + S::load_chunk(j) * 16;
                __builtin_amdgcn_global_load_lds(k < K ? bp[j] + k : z, dst + S::BM * W8_KB + (j * S::NW + wave) * 1024,
                                                 16, 0, 0);
            }
        }
    };
    const int wm = wave / S::KW / S::WN, wn = wave / S::KW % S::WN, kw = wave % S::KW;
    auto compute = [&](const unsigned char *a) {
        const unsigned char *b = a + S::BM * W8_KB;
#pragma unroll
        for (int q0 = 0; q0 < 4; q0 += S::KW) {
            const int q = q0 + kw;
            uint4 af[S::MT], bf[S::NT];
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
                af[i] = *reinterpret_cast<const uint4 *>(a + w8_swz((wm * S::MT + i) * 32 + l32, 2 * q + lh));
#pragma unroll
            for (int j = 0; j < S::NT; ++j)
                bf[j] = *reinterpret_cast<const uint4 *>(b + w8_swz((wn * S::NT + j) * 32 + l32, 2 * q + lh));
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j) acc[i][j] = w8_mfma(af[i], bf[j], acc[i][j]);
        }
    };
    auto step = [&](auto i, int ks) {
        constexpr int I = decltype(i)::value;
        if (ks + NS - 2 < nk) w8_stage_barrier<(NS - 2) * LPW>();
        else w8_stage_barrier<0>();
        if (ks + NS - 1 < nk) issue(ks + NS - 1, buf(std::integral_constant<int, (I + NS - 1) % NS>{}));
        compute(buf(i));
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    issue(0, s0);
    if constexpr (NS > 2) {
        if (nk > 1) issue(1, s1);
    }
    if constexpr (NS > 3) {
        if (nk > 2) issue(2, s2);
    }
    for (int ks = 0; ks < nk; ks += NS) {
        step(I0{}, ks);
        if (ks + 1 < nk) step(I1{}, ks + 1);
        if constexpr (NS > 2) {
            if (ks + 2 < nk) step(I2{}, ks + 2);
        }
        if constexpr (NS > 3) {
            if (ks + 3 < nk) step(I3{}, ks + 3);
        }
    }
    if constexpr (S::KW > 1) {
        __syncthreads();  // the last stage is read
        auto part = [&](int w) -> int * {
            return reinterpret_cast<int *>(w == 1 ? s0 : w == 2 ? s1 : s2);
        };
        if (kw > 0) {
            int *p = part(kw);
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) p[((i * S::NT + j) * 16 + r) * WAVE + lane] = acc[i][j][r];
        }
        __syncthreads();
        if (kw > 0) return false;
#pragma unroll
        for (int w = 1; w < S::KW; ++w) {
            const int *p = part(w);
#pragma unroll
            for (int i = 0; i < S::MT; ++i)
#pragma unroll
                for (int j = 0; j < S::NT; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] += p[((i * S::NT + j) * 16 + r) * WAVE + lane];
        }
    }
    return true;
}

template <class S>
__device__ __forceinline__ void w8_clear(i32x16 (&acc)[S::MT][S::NT]) {
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int j = 0; j < S::NT; ++j) acc[i][j] = i32x16{};
}

// The sum's value: the whole number rounded once to fp32 (it can pass 2^24),
// times the weight row's scale, times the token's.
__device__ __forceinline__ float w8_value(int sum, float sw, float sx) { return float(sum) * sw * sx; }

// One element of an output of type QW_T_F32 (0), QW_T_BF16 (1) or QW_T_F16
// (2; finite values beyond +-65504 saturate).
__device__ __forceinline__ void w8_store(void *y, int type, int64_t at, float v) {
    if (type == 0) static_cast<float *>(y)[at] = v;
    else if (type == 1) static_cast<uint16_t *>(y)[at] = f32_to_bf16_rne(v);
    else static_cast<_Float16 *>(y)[at] = f32_to_f16_satfinite(v);
}

}  // namespace qwq4
