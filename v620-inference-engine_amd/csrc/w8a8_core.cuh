// Shared main loop of the int8 x int8 products (W8A8): one block computes a
// BM x BN tile of Q (int8 rows, K long) times W^T (int8 weight rows, as the
// checkpoint holds them: row-major), summed exactly in int32 on
// v_mfma_i32_32x32x32_i8.
//
// The sums are whole numbers, so neither the tile, nor the order of K, nor the
// batch changes a result: every shape of this loop gives the same bits, and a variant is chosen by speed alone.
//
// Schedule. K runs in stages of 128 bytes through NS buffers of LDS, filled by
// direct global -> LDS loads (a wave instruction moves 8 rows of 128 bytes,
// whole cache lines, from any row addresses: gathered rows cost the same as
// neighbours) NS - 1 stages ahead. One barrier per stage: a wave waits for its
// own loads of the stage, and the barrier then makes everyone's visible and
// tells that the buffer of the stage before is free for the next loads.
// The waves are WM x WN over the tile.
#pragma once

#include <type_traits>

#include "q4_common.cuh"

namespace qwq4 {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// What a lane loads for K columns past the row's end (K need not be a
// multiple of 128): zeros, from memory that is always there.
static __device__ const uint4 w8_zeros = {0u, 0u, 0u, 0u};

__device__ __forceinline__ i32x16 w8_mfma(const uint4 &a, const uint4 &b, const i32x16 &c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0,
                                                 0);
}

template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct W8A8Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KB = 128, NS = NS_;
    static constexpr int NW = WM * WN, THREADS = NW * WAVE;
    static constexpr int MT = BM / 32 / WM, NT = BN / 32 / WN;  // 32 x 32 tiles per wave
    static constexpr int CH = KB / 16, RPL = 1024 / KB;         // chunks per row, rows per load instruction
    static constexpr int AJ = BM / RPL / NW, BJ = BN / RPL / NW;  // load instructions per wave and stage
    static constexpr int NQ = KB / 32;                          // slabs per stage
    static_assert(BM % (RPL * NW) == 0 && BN % (RPL * NW) == 0 && BM % (32 * WM) == 0 && BN % (32 * WN) == 0, "tile");
    static_assert(NS >= 2 && NS <= 4 && NQ % 2 == 0, "the fragments alternate between two sets of registers");

    // Byte offset of 16-byte chunk c of row r in a [rows][KB] buffer. A
    // fragment read takes 32 consecutive rows at chunk c (lanes 0-31) and
    // c + 1 (lanes 32-63); under this XOR each 16 lanes of it fall on the 64
    // banks once.
    __device__ static __forceinline__ int swz_x(int r) { return (r & 7) ^ ((r >> 3) & 1); }
    __device__ static __forceinline__ int swz(int r, int c) { return r * KB + ((c ^ swz_x(r)) << 4); }
    // The tile row that part j of this lane's loads belongs to: A rows for
    // j < AJ, weight rows likewise for j < BJ.
    __device__ static __forceinline__ int load_row(int j) {
        return (j * NW + int(threadIdx.x) / WAVE) * RPL + int(threadIdx.x) % WAVE / CH;
    }
    // The chunk of that row it loads (its place in the row is lane % CH).
    __device__ static __forceinline__ int load_chunk(int j) { return (int(threadIdx.x) % CH) ^ swz_x(load_row(j)); }
    // The wave's place over the tile: its first row of Q and of W. Element r
    // of accumulator (i, j) is row m_base() + 32 i + lane % 32 of Q and row
    // n_base() + 32 j + n_of(r) of W.
    __device__ static __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE); }
    __device__ static __forceinline__ int m_base() { return wave() / WN * MT * 32; }
    __device__ static __forceinline__ int n_base() { return wave() % WN * NT * 32; }
    __device__ static __forceinline__ int n_of(int r) { return 8 * (r / 4) + 4 * (int(threadIdx.x) % WAVE / 32) + r % 4; }
    // LDS that a wave has to itself after the sums, of the weights' buffers
    // (whole banks' turns: several waves share a buffer, three of 10922 bytes in
    // the tall expert tiles, and each of them starts aligned)
    static constexpr int SPARE = BN * KB / ((NW + NS - 1) / NS) / 128 * 128;
    static_assert(SPARE % 16 == 0, "16-byte pieces go through it");
};

// The stage buffers of shape S; a kernel that runs several shapes takes those
// of its largest for all of them. STREAM: the weights are read by no other
// block, and go past the caches' replacement (non-temporal loads).
template <class S, int USE, bool STREAM = false>
struct W8Lds {
    static constexpr int W_AUX = STREAM ? 2 : 0;
    template <int I>
    __device__ static __forceinline__ unsigned char *a() {
        __shared__ __align__(16) unsigned char s[I < S::NS ? S::BM * S::KB : 16];
        return s;
    }
    template <int I>
    __device__ static __forceinline__ unsigned char *b() {
        __shared__ __align__(16) unsigned char s[I < S::NS ? S::BN * S::KB : 16];
        return s;
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
// passes the matrix).
// spare: S::SPARE bytes of LDS for this wave until the block's next barrier,
// which has to come before another tile. (USE tags the caller: each call site
// instantiates its own specialization; the host compilation pass rejects a
// second call site of a shared one.)
template <class S, int USE, class L = W8Lds<S, USE>>
__device__ __forceinline__ void w8_tile(const int8_t *(&ap)[S::AJ], const int8_t *(&bp)[S::BJ], int K,
                                        i32x16 (&acc)[S::MT][S::NT], unsigned char *&spare) {
    constexpr int NS = S::NS, LPW = S::AJ + S::BJ;
    // (distinct arrays picked at compile time: the compiler then sees that the
    // loads in flight into one do not touch the buffer being read)
    unsigned char *const sa0 = L::template a<0>(), *const sa1 = L::template a<1>(), *const sa2 = L::template a<2>(),
                  *const sa3 = L::template a<3>();
    unsigned char *const sb0 = L::template b<0>(), *const sb1 = L::template b<1>(), *const sb2 = L::template b<2>(),
                  *const sb3 = L::template b<3>();
    const int wave = S::wave(), lane = int(threadIdx.x) % WAVE, l32 = lane % 32, lh = lane / 32;
    const int nk = (K + S::KB - 1) / S::KB;
    auto buf_a = [&](auto i) -> unsigned char * {
        if constexpr (decltype(i)::value == 0) return sa0;
        else if constexpr (decltype(i)::value == 1) return sa1;
        else if constexpr (decltype(i)::value == 2) return sa2;
        else return sa3;
    };
    auto buf_b = [&](auto i) -> unsigned char * {
        if constexpr (decltype(i)::value == 0) return sb0;
        else if constexpr (decltype(i)::value == 1) return sb1;
        else if constexpr (decltype(i)::value == 2) return sb2;
        else return sb3;
    };
    // Load n of a stage's LPW. Past the end of the rows (the last stage of a K
    // that is no multiple of KB) Q's chunks are zeros and W's any of the row's:
    // a select rather than a branch, whose two sides would share their last
    // load, whose buffer the compiler then no longer knows. All of a lane's
    // loads are of one chunk.
    static_assert(S::NW % 2 == 0, "load_chunk(j) is load_chunk(0)");
    const int8_t *zeros = reinterpret_cast<const int8_t *>(&w8_zeros);
    auto issue_one = [&](int ks, int n, unsigned char *da, unsigned char *db) {
        const int k = ks * S::KB + S::load_chunk(0) * 16;
        if (n < S::AJ)
            __builtin_amdgcn_global_load_lds(k < K ? ap[n] + k : zeros, da + (n * S::NW + wave) * 1024, 16, 0, 0);
        else
            __builtin_amdgcn_global_load_lds(bp[n - S::AJ] + min(k, K - 16),
                                             db + ((n - S::AJ) * S::NW + wave) * 1024, 16, 0, L::W_AUX);
    };
    auto issue = [&](int ks, unsigned char *da, unsigned char *db) {
#pragma unroll
        for (int n = 0; n < LPW; ++n) issue_one(ks, n, da, db);
    };
    const int wm = wave / S::WN, wn = wave % S::WN;
    // Fragments of slab n of a stage, read while the slab
    // before is multiplied. (The scheduling barrier keeps the reads in front:
    // left to itself the compiler moves them behind the products, and every
    // slab then waits for its own.)
    constexpr int NQ = S::NQ;
    uint4 af[2][S::MT], bf[2][S::NT];
    auto read = [&](int p, const unsigned char *a, const unsigned char *b, int n) {
        const int c = 2 * n + lh;
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
            af[p][i] = *reinterpret_cast<const uint4 *>(a + S::swz((wm * S::MT + i) * 32 + l32, c));
#pragma unroll
        for (int j = 0; j < S::NT; ++j)
            bf[p][j] = *reinterpret_cast<const uint4 *>(b + S::swz((wn * S::NT + j) * 32 + l32, c));
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int p) {
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
            for (int j = 0; j < S::NT; ++j) acc[i][j] = w8_mfma(bf[p][j], af[p][i], acc[i][j]);
    };
    // The same with the loads of stage ks between the products: in front of
    // them they would hold up all waves at once, behind the barrier.
    auto multiply_and_issue = [&](int p, int ks, unsigned char *da, unsigned char *db) {
        constexpr int TILES = S::MT * S::NT, PER = (LPW + TILES - 1) / TILES;
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int i = t / S::NT, j = t % S::NT;
            acc[i][j] = w8_mfma(bf[p][j], af[p][i], acc[i][j]);
#pragma unroll
            for (int n = t * PER; n < (t + 1) * PER && n < LPW; ++n) issue_one(ks, n, da, db);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // A stage up to its last slab, whose fragments are then held in set 1; the
    // first slab's are in set 0.
    auto inner = [&](const unsigned char *a, const unsigned char *b) {
#pragma unroll
        for (int n = 0; n + 1 < NQ; ++n) {
            read((n + 1) % 2, a, b, n + 1);
            multiply(n % 2);
        }
    };
    // From stage ks in buffer I to the next. Before the last slab of ks is
    // multiplied, the block meets: the next stage has landed and this one's
    // buffer is read, so the next stage's first fragments and the loads of
    // stage ks + NS go out, and the products behind them cover the wait. (There
    // is a stage ks + NS: these steps have no branch. Around one the compiler
    // moves the sums, or waits for all loads.)
    auto step = [&](auto i, int ks) {
        constexpr int I = decltype(i)::value;
        constexpr std::integral_constant<int, (I + 1) % NS> next{};
        w8_stage_barrier<(NS - 2) * LPW>();
        read(0, buf_a(next), buf_b(next), 0);
        multiply_and_issue(1, ks + NS, buf_a(i), buf_b(i));
        inner(buf_a(next), buf_b(next));
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    // (a K of fewer stages loads its last one again, where nobody reads it)
    issue(0, sa0, sb0);
    issue(min(1, nk - 1), sa1, sb1);
    if constexpr (NS > 2) issue(min(2, nk - 1), sa2, sb2);
    if constexpr (NS > 3) issue(min(3, nk - 1), sa3, sb3);
    w8_stage_barrier<(NS - 1) * LPW>();
    read(0, sa0, sb0, 0);
    inner(sa0, sb0);
    int ks = 0;
    for (; ks + 2 * NS - 1 < nk; ks += NS) {
        step(I0{}, ks);
        step(I1{}, ks + 1);
        if constexpr (NS > 2) step(I2{}, ks + 2);
        if constexpr (NS > 3) step(I3{}, ks + 3);
    }
    // The last stages (up to 2 NS - 1; ks is at buffer 0 again), in one piece
    // of code for every buffer.
    auto pick_a = [&](int i) { return i == 0 ? sa0 : i == 1 ? sa1 : i == 2 ? sa2 : sa3; };
    auto pick_b = [&](int i) { return i == 0 ? sb0 : i == 1 ? sb1 : i == 2 ? sb2 : sb3; };
    auto last = [&](int s) {
        const int cur = s % NS, next = (s + 1) % NS;
        if (s + NS <= nk) w8_stage_barrier<(NS - 2) * LPW>();
        else w8_stage_barrier<0>();
        read(0, pick_a(next), pick_b(next), 0);
        if (s + NS < nk) issue(s + NS, pick_a(cur), pick_b(cur));
        multiply(1);
        inner(pick_a(next), pick_b(next));
    };
    for (; ks < nk - 1; ++ks) last(ks);
    multiply(1);
    // The last stage is read, and no load is in flight any more (a K of one
    // stage has not waited for those that nobody reads): the buffers are free.
    w8_stage_barrier<0>();
    const int w = wave % NS;
    spare = (w == 0 ? sb0 : w == 1 ? sb1 : w == 2 ? sb2 : sb3) + wave / NS * S::SPARE;
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
__device__ __forceinline__ uint16_t w8_bits16(int type, float v) {
    return type == 1 ? __builtin_bit_cast(uint16_t, __bf16(v)) : __builtin_bit_cast(uint16_t, f32_to_f16_satfinite(v));
}
__device__ __forceinline__ void w8_store(void *y, int type, int64_t at, float v) {
    if (type == 0) static_cast<float *>(y)[at] = v;
    else static_cast<uint16_t *>(y)[at] = w8_bits16(type, v);
}

// The wave's values to rows of Y: value(i, c, r) is that of row 32 i +
// lane % 32 of the wave's, column 32 c + S::n_of(r) of its NC * 32; row(m)
// gives where row m of them starts in Y (in elements; negative: no such row)
// and columns from `cols` on are left out. Through the wave's spare LDS, 32
// rows at a time, so that a row goes out in 16-byte pieces next to each other
// (stored as the accumulators hold them, 32 rows of 8 bytes an instruction,
// a 4096 x 12288 product took 20 us longer).
template <class S, int NC, int BYTES, class ValueF, class RowF>
__device__ __forceinline__ void w8_store_rows(unsigned char *spare, void *Y, int type, int cols, ValueF value, RowF row) {
    constexpr int FIT = (S::SPARE / 32 - 16) / (32 * BYTES);
    constexpr int CG = FIT >= NC ? NC : FIT >= 2 && NC % 2 == 0 ? 2 : 1;  // 32-column groups at a time
    static_assert(FIT >= 1, "32 columns fit");
    constexpr int LD = CG * 32 * BYTES + 16, PIECES = CG * 32 * BYTES / 16, PER = 16 / BYTES;
    const int lane = int(threadIdx.x) % WAVE, l32 = lane % 32, lh = lane / 32;
    unsigned char *y8 = static_cast<unsigned char *>(Y);
#pragma unroll
    for (int i = 0; i < S::MT; ++i)
#pragma unroll
        for (int c0 = 0; c0 < NC; c0 += CG) {
#pragma unroll
            for (int c = 0; c < CG; ++c)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = value(i, c0 + c, 4 * u + e);
                    unsigned char *at = spare + l32 * LD + (c * 32 + 8 * u + 4 * lh) * BYTES;
                    if constexpr (BYTES == 4) {
                        *reinterpret_cast<float4 *>(at) = make_float4(v[0], v[1], v[2], v[3]);
                    } else {
                        *reinterpret_cast<uint2 *>(at) =
                            make_uint2(w8_bits16(type, v[0]) | uint32_t(w8_bits16(type, v[1])) << 16,
                                       w8_bits16(type, v[2]) | uint32_t(w8_bits16(type, v[3])) << 16);
                    }
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int p = 0; p < PIECES / 2; ++p) {
                const int m = (p * WAVE + lane) / PIECES, piece = (p * WAVE + lane) % PIECES;
                const uint4 w = *reinterpret_cast<const uint4 *>(spare + m * LD + piece * 16);
                const int n = c0 * 32 + piece * PER;
                const int64_t at = row(32 * i + m);
                if (at < 0 || n >= cols) continue;
                unsigned char *dst = y8 + (at + n) * BYTES;
                if (n + PER <= cols && reinterpret_cast<uintptr_t>(dst) % 16 == 0) {
                    *reinterpret_cast<uint4 *>(dst) = w;
                } else {
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        if (n + e >= cols) break;
                        if constexpr (BYTES == 4) reinterpret_cast<uint32_t *>(dst)[e] = words[e];
                        else reinterpret_cast<uint16_t *>(dst)[e] = uint16_t(words[e / 2] >> (16 * (e % 2)));
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
}

// w8_store_rows for either width of the output's type.
template <class S, int NC, class ValueF, class RowF>
__device__ __forceinline__ void w8_output(unsigned char *spare, void *Y, int type, int cols, ValueF value, RowF row) {
    if (type == 0) {
        w8_store_rows<S, NC, 4>(spare, Y, type, cols, value, row);
    } else {
        w8_store_rows<S, NC, 2>(spare, Y, type, cols, value, row);
    }
}

}  // namespace qwq4
