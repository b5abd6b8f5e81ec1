// Dense W8A8: int8 rows with a scale per token times int8 weights with a scale
// per output row, and the rows' quantiser.
//
//   s_t = max_k |x_tk| / 127 (1 for a row of zeros, at least 2^-126)
//   q_tk = rint(x_tk * (1 / s_t))
//   y_tn = float(sum_k q_tk w_nk) * sw_n * s_t
//
// The engine's int8 copy of its dense weights (src/engine/weight_convert.cpp:92-108)
// keeps 16-bit rows and a scale per 16 or 32 columns, so its products
// (src/kernels/gemv.hip:75-136) cannot be summed in whole numbers; with one
// scale per row and token they are, over all of K, on the int8 MFMA.
#include <type_traits>

#include "q4_kernels.hpp"
#include "w8a8_core.cuh"
#include "w8a8_gemv.cuh"

namespace qwq4 {

// ------------------------------------------------------------ quantiser
// A row by G threads (64: a wave, four rows a block; 256: the block), 16
// elements per thread and turn. C > 0: the row is held in C turns' registers
// and read once; C = 0: any length, read twice (the second time from the
// caches).
template <int XT, bool VEC, int G, int C>
__global__ __launch_bounds__(256) void quant_tokens_kernel(const void *__restrict__ x, int64_t ldx, int T, int K,
                                                           int8_t *__restrict__ q, int64_t ldq,
                                                           float *__restrict__ scale) {
    const int li = int(threadIdx.x) % G;
    const int t = min(int(blockIdx.x) * (256 / G) + int(threadIdx.x) / G, T - 1);  // (spare waves repeat the last row)
    const int64_t at = int64_t(t) * ldx;
    uint4 *out = reinterpret_cast<uint4 *>(q + int64_t(t) * ldq);
    const int n = K / 16;
    uint32_t top = 0u;
    W8Raw<XT, VEC> raw[C > 0 ? C : 1];
    if constexpr (C > 0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (li + c * G < n) raw[c].load(x, at + (li + c * G) * 16);
            else raw[c].clear();
        }
#pragma unroll
        for (int c = 0; c < C; ++c) top = raw[c].top(top);
    } else {
        for (int i = li; i < n; i += G) {
            raw[0].load(x, at + i * 16);
            top = raw[0].top(top);
        }
    }
    top = wave_top(top);
    if constexpr (G == 256) {
        __shared__ uint32_t s_top[4];
        if (li % WAVE == 0) s_top[li / WAVE] = top;
        __syncthreads();
        top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    }
    bool finite;
    const float sc = w8_scale(top, finite), inv = 1.f / sc;
    if constexpr (C > 0) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (li + c * G < n) out[li + c * G] = raw[c].quantised(inv, finite);
    } else {
        for (int i = li; i < n; i += G) {
            raw[0].load(x, at + i * 16);
            out[i] = raw[0].quantised(inv, finite);
        }
    }
    if (li == 0) scale[t] = sc;
}

// Rows up to 2048 by a wave each, longer ones by a block, from registers up to
// 16384.
template <int XT, bool VEC>
static void launch_quant_x(const void *x, int64_t ldx, int T, int K, int8_t *q, int64_t ldq, float *scale,
                           hipStream_t s) {
    const unsigned quads = unsigned((T + 3) / 4);
    if (K <= 1024) quant_tokens_kernel<XT, VEC, 64, 1><<<quads, 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else if (K <= 2048) quant_tokens_kernel<XT, VEC, 64, 2><<<quads, 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else if (K <= 4096) quant_tokens_kernel<XT, VEC, 256, 1><<<unsigned(T), 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else if (K <= 8192) quant_tokens_kernel<XT, VEC, 256, 2><<<unsigned(T), 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else if (K <= 16384) quant_tokens_kernel<XT, VEC, 256, 4><<<unsigned(T), 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else quant_tokens_kernel<XT, VEC, 256, 0><<<unsigned(T), 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
}

void launch_quant_tokens(const void *x, int x_type, int64_t ldx, int T, int K, int8_t *q, int64_t ldq, float *scale,
                         hipStream_t s) {
    w8_by_rows(x, x_type, ldx, T, [&](auto xt, auto vec) {
        launch_quant_x<decltype(xt)::value, decltype(vec)::value>(x, ldx, T, K, q, ldq, scale, s);
    });
}

// ------------------------------------------------------------ product
// Tile of block b among mt x nt. Blocks go to the 8 XCDs in turn; each XCD gets
// a run of tiles in an order that walks the columns of bands GM tiles tall, so
// that the tiles it works on together form a patch whose rows and weights its
// L2 holds once
// (4096 x 12288 x 4096: 225 us against 261 with the tiles row by row, bands of
// 2 to 8 alike).
template <int GM>
__device__ __forceinline__ void w8_place(int b, int mt, int nt, int &m, int &n) {
    const int per = mt * nt / 8, rest = mt * nt % 8, xcd = b % 8;
    const int t = xcd * per + min(xcd, rest) + b / 8;
    const int band = t / (GM * nt), at = t % (GM * nt), tall = min(GM, mt - band * GM);
    m = band * GM + at % tall;
    n = at / tall;
}

template <class S>
__global__ __launch_bounds__(S::THREADS) void w8a8_gemm_kernel(W8GemmArgs a) {
    int mi, ni;
    w8_place<S::BM >= 256 ? 4 : 8>(int(blockIdx.x), (a.T + S::BM - 1) / S::BM, (a.N + S::BN - 1) / S::BN, mi,
                                     ni);
    const int m0 = mi * S::BM, n0 = ni * S::BN;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::AJ; ++j) ap[j] = a.q + int64_t(min(m0 + S::load_row(j), a.T - 1)) * a.ldq;
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) bp[j] = a.W + int64_t(min(n0 + S::load_row(j), a.N - 1)) * a.ldw;
    i32x16 acc[S::MT][S::NT];
    w8_clear<S>(acc);
    unsigned char *spare;
    w8_tile<S, 0>(ap, bp, a.K, acc, spare);
    const int m_first = m0 + S::m_base(), n_first = n0 + S::n_base(), l32 = int(threadIdx.x) % 32;
    float sx[S::MT], sw[S::NT][16];
#pragma unroll
    for (int i = 0; i < S::MT; ++i) sx[i] = a.sx[min(m_first + 32 * i + l32, a.T - 1)];
#pragma unroll
    for (int j = 0; j < S::NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) sw[j][r] = a.sw[min(n_first + 32 * j + S::n_of(r), a.N - 1)];
    auto value = [&](int i, int j, int r) { return w8_value(acc[i][j][r], sw[j][r], sx[i]); };
    w8_output<S, S::NT>(spare, a.Y, a.y_type, a.N - n_first, value, [&](int m) -> int64_t {
        return m_first + m < a.T ? int64_t(m_first + m) * a.ldy + n_first : -1;
    });
}

template <class S>
static void launch_shape(const W8GemmArgs &a, hipStream_t s) {
    const unsigned tiles = unsigned((a.T + S::BM - 1) / S::BM) * unsigned((a.N + S::BN - 1) / S::BN);
    w8a8_gemm_kernel<S><<<tiles, S::THREADS, 0, s>>>(a);
}

// ------------------------------------------------------------ tens of tokens
// Tiles of 32 tokens by 32 NT weight rows whose four waves split K. Such a tile
// has little to multiply and is bound by the latency of its loads, so each wave
// runs alone: it loads every fourth 128-byte stage of K into two buffers of its
// own, waits for its own loads only, and no barrier joins the waves before
// their sums meet. (With a barrier per stage and four buffers shared by the
// waves: 37 x 4096 x 6144 15.2 us, here 8.3; 20 x 4096 x 4096 12.0 and 7.0, weights
// in the last-level cache; from memory 10.2 and 8.1 here. Three or four buffers
// or eight waves a block: no better, and fewer blocks on a CU.)
template <int NT_>
struct W8Split {
    static constexpr int NT = NT_, NS = 2, KW = 4, THREADS = KW * WAVE, BN = 32 * NT, LPW = 4 + 4 * NT;
    // Stage buffer I: [waves][rows][128 bytes].
    template <int I>
    __device__ static __forceinline__ unsigned char *a() {
        __shared__ __align__(16) unsigned char s[KW * 4096];
        return s;
    }
    template <int I>
    __device__ static __forceinline__ unsigned char *b() {
        __shared__ __align__(16) unsigned char s[KW * NT * 4096];
        return s;
    }
};

// Until at most N of this wave's loads are in flight, and its LDS reads done.
template <int N>
__device__ __forceinline__ void w8_wave_wait() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (0 << 8));
    asm volatile("" ::: "memory");
}

template <class S>
__device__ __forceinline__ void w8_split_tile(const W8GemmArgs &a) {
    constexpr int NT = S::NT, NS = S::NS, KW = S::KW, LPW = S::LPW;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE), lane = int(threadIdx.x) % WAVE;
    const int l32 = lane % 32, lh = lane / 32;
    int mi, ni;
    w8_place<8>(int(blockIdx.x), (a.T + 31) / 32, (a.N + S::BN - 1) / S::BN, mi, ni);
    const int m0 = mi * 32, n0 = ni * S::BN;
    // (this thread's part of the output: row l32, columns 32 j + col .. + 3)
    const int col = 8 * wave + 4 * lh;
    float sw[NT][4];
    const float sx = a.sx[min(m0 + l32, a.T - 1)];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[j][e] = a.sw[min(n0 + 32 * j + col + e, a.N - 1)];
    const int8_t *ap[4], *bp[4 * NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) ap[j] = a.q + int64_t(min(m0 + 8 * j + lane / 8, a.T - 1)) * a.ldq;
#pragma unroll
    for (int j = 0; j < 4 * NT; ++j) bp[j] = a.W + int64_t(min(n0 + 8 * j + lane / 8, a.N - 1)) * a.ldw;
    // (16-byte chunk c of row r lies at place c ^ (r & 7) ^ (r >> 3 & 1) of its 128 bytes: without bank conflicts)
    const int c0 = (lane % 8) ^ (lane / 8), place = (l32 & 7) ^ ((l32 >> 3) & 1);
    const int nk = (a.K + 127) / 128, n = (nk - wave + KW - 1) / KW;  // stages wave, wave + KW, .. of K
    const int8_t *zeros = reinterpret_cast<const int8_t *>(&w8_zeros);
    unsigned char *const sa0 = S::template a<0>() + wave * 4096, *const sa1 = S::template a<1>() + wave * 4096;
    unsigned char *const sb0 = S::template b<0>() + wave * NT * 4096, *const sb1 = S::template b<1>() + wave * NT * 4096;
    auto issue = [&](int i, unsigned char *da, unsigned char *db) {
        const int k0 = min(wave + KW * i, nk - 1) * 128;  // (past the last: again, where nobody reads it)
#pragma unroll
        for (int j = 0; j < 4 + 4 * NT; ++j) {
            const int k = k0 + (c0 ^ (j & 1)) * 16;
            if (j < 4) __builtin_amdgcn_global_load_lds(k < a.K ? ap[j] + k : zeros, da + j * 1024, 16, 0, 0);
            else __builtin_amdgcn_global_load_lds(bp[j - 4] + min(k, a.K - 16), db + (j - 4) * 1024, 16, 0, 0);
        }
    };
    i32x16 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = i32x16{};
    // One stage, landed: its fragments are read, and with MORE the loads of
    // stage `next` go into its buffers, in front of the products.
    auto stage = [&](unsigned char *sa, unsigned char *sb, auto more, int next) {
        uint4 af[4], bf[4][NT];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int at = ((2 * s + lh) ^ place) << 4;
            af[s] = *reinterpret_cast<const uint4 *>(sa + l32 * 128 + at);
#pragma unroll
            for (int j = 0; j < NT; ++j) bf[s][j] = *reinterpret_cast<const uint4 *>(sb + (32 * j + l32) * 128 + at);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (decltype(more)::value) {
            w8_wave_wait<63>();
            issue(next, sa, sb);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j] = w8_mfma(bf[s][j], af[s], acc[j]);
    };
    issue(0, sa0, sb0);
    issue(1, sa1, sb1);
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
    int i = 0;
    auto turn = [&](unsigned char *sa, unsigned char *sb, int at) {
        w8_wave_wait<(NS - 1) * LPW>();
        stage(sa, sb, yes, at + NS);
    };
    for (; i + NS < n; i += NS) {
        turn(sa0, sb0, i);
        turn(sa1, sb1, i + 1);
    }
    // the last one or two (of a K of few stages: none), both on their way
    auto last = [&](unsigned char *sa, unsigned char *sb) { stage(sa, sb, no, 0); };
    if (i < n) {
        w8_wave_wait<(NS - 1) * LPW>();
        last(sa0, sb0);
    }
    if (i + 1 < n) {
        w8_wave_wait<0>();
        last(sa1, sb1);
    }
    // the waves' sums through their buffers; each wave then has a quarter of the columns
    w8_wave_wait<0>();
    int *part = reinterpret_cast<int *>(sb0);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) part[(j * 16 + r) * WAVE + lane] = acc[j][r];
    __syncthreads();
    const int *parts = reinterpret_cast<const int *>(S::template b<0>());
    const int m = m0 + l32;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < KW; ++w) sum += parts[(w * NT * 16 + j * 16 + 4 * wave + e) * WAVE + lane];
            v[e] = w8_value(sum, sw[j][e], sx);
        }
        const int at = n0 + 32 * j + col;
        if (m >= a.T) continue;
        const int64_t y = int64_t(m) * a.ldy + at;
        if (a.y_type == 0) {
            float *p = static_cast<float *>(a.Y) + y;
            if (at + 4 <= a.N && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
                *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
                continue;
            }
        } else {
            uint16_t *p = static_cast<uint16_t *>(a.Y) + y;
            if (at + 4 <= a.N && reinterpret_cast<uintptr_t>(p) % 8 == 0) {
                *reinterpret_cast<uint2 *>(p) =
                    make_uint2(w8_bits16(a.y_type, v[0]) | uint32_t(w8_bits16(a.y_type, v[1])) << 16,
                               w8_bits16(a.y_type, v[2]) | uint32_t(w8_bits16(a.y_type, v[3])) << 16);
                continue;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (at + e < a.N) w8_store(a.Y, a.y_type, y + e, v[e]);
    }
}

template <class S>
__global__ __launch_bounds__(S::THREADS) void w8a8_split_kernel(W8GemmArgs a) {
    w8_split_tile<S>(a);
}

template <int NT>
static void launch_split(const W8GemmArgs &a, hipStream_t s) {
    using S = W8Split<NT>;
    const unsigned tiles = unsigned((a.T + 31) / 32) * unsigned((a.N + S::BN - 1) / S::BN);
    w8a8_split_kernel<S><<<tiles, S::THREADS, 0, s>>>(a);
}

// ------------------------------------------------------------ few tokens
// Up to 2 tokens the product is a stream of the weights (w8a8_gemv.cuh), 8 G
// rows of them per block, bound by memory and by the launch's ramp (one token,
// 4096 -> 12288, rows quantised on the way: 12.1 us, 4.2 TB/s; a large copy
// reaches 5.2). Times here and at launch_w8a8_gemm: calls in a graph over 0.8 GB
// of weights in turn, which no cache holds. Streamed and in tiles of 32, K 4096:
// 1 row to 4096 5.2 and 6.6 us, to 12288 11.7 and 13.5; 2 rows 5.9 and 6.6, 12.5
// and 13.6. (4 rows, weights in the last-level cache: 6.9 and 6.4, 14.5 and 12.3.)
// From 16- or 32-bit rows the block quantises them itself, which saves the
// quantiser's launch (one token: 6.0 against 7.3 us and 12.1 against 13.7; two:
// 7.4 against 7.9 and 14.2 against 14.6).
template <int XT, bool VEC, int TM, int G>
__global__ __launch_bounds__(256) void w8a8_gemv_kernel(W8GemmArgs a, const void *x, int64_t ldx) {
    extern __shared__ __align__(16) unsigned char s_q[];
    const int n0 = int(blockIdx.x) * 8 * G;
    const int8_t *w[G];
#pragma unroll
    for (int g = 0; g < G; ++g) w[g] = a.W + int64_t(min(n0 + 8 * g + gemv_row(), a.N - 1)) * a.ldw;
    W8Stream<G> v;
    v.load(w, a.K, gemv_wave());
    auto token = [&](int t) { return int64_t(min(t, a.T - 1)); };
    float sx[TM];
    if constexpr (XT == 3) gemv_stage_i8<TM>(a.q, a.ldq, a.sx, a.K, s_q, sx, token);
    else gemv_stage<XT, VEC, TM>(x, ldx, a.K, s_q, sx, token);
    gemv_sums<TM, G>(v, w, a.K, s_q, [&](auto sum) {
        for (int i = int(threadIdx.x); i < TM * 8 * G; i += 256) {
            const int t = i / (8 * G), r = i % (8 * G), n = n0 + r;
            if (t < a.T && n < a.N)
                w8_store(a.Y, a.y_type, int64_t(t) * a.ldy + n, w8_value(sum(t, r), a.sw[n], gemv_pick(sx, t)));
        }
    });
}

static bool gemv_takes(int T, int K) { return T <= 2 && gemv_lds(T, K) <= W8_GEMV_LDS; }

template <int XT, bool VEC>
static void launch_gemv(const W8GemmArgs &a, const void *x, int64_t ldx, hipStream_t s) {
    // (16 rows a block where that leaves blocks enough: 2 tokens and 12288 rows
    // take 14.2 us against 15.3 with 8, 8192 rows 11.1 and 11.0, 4096 rows 8.0
    // and 7.7. One token has less to gain from it: 12288 rows 12.4 and 11.5.)
    auto run = [&](auto tm) {
        constexpr int TM = decltype(tm)::value;
        const size_t lds = gemv_lds(TM, a.K);
        if (a.N >= 8192)
            w8a8_gemv_kernel<XT, VEC, TM, 2><<<unsigned((a.N + 15) / 16), 256, lds, s>>>(a, x, ldx);
        else w8a8_gemv_kernel<XT, VEC, TM, 1><<<unsigned((a.N + 7) / 8), 256, lds, s>>>(a, x, ldx);
    };
    if (a.T <= 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
}

// One or two tokens stream the weights. Else the largest tile that makes about
// a block for every CU (us, weights from memory; rows x weight rows x K, tiles of
// 256 and 128: 4096 x 12288 x 4096: 190, 235; 1024 x 12288 x 4096: 60, 78; 1024 x
// 4096 x 4096: 54, 34; of 256, 128, 64: 256 x 12288 x 4096: 58, 35, 34; 256 x 4096 x
// 4096: 56, 32, 13.9). Where those of 32 are no more than two rounds of the CUs,
// or there are no more than 32 rows, those, two side by side between one round
// and two (tiles of 64, of 32, of 32 x 64: 64 x 4096 x 4096, 256 of 32: 13.4, 8.3,
// 10.3; 32 x 9216 x 4096, 288: 15.6, 14.4, 13.3; 128 x 4096 x 4096, 512: 13.3, 11.3,
// 10.5; 96 x 6144 x 4096, 576: 13.3, 15.6, 18.2; 150 x 4096 x 4096, 640: 12.4, 14.0,
// 16.9; 16 x 20480 x 4096, 640: 25.2, 20.4, 25.0; 8 x 100000 x 4096: 87, 75, 92).
void launch_w8a8_gemm(const W8GemmArgs &a, hipStream_t s) {
    auto tiles = [&](int b) { return int64_t((a.T + b - 1) / b) * ((a.N + b - 1) / b); };
    if (gemv_takes(a.T, a.K)) launch_gemv<3, true>(a, nullptr, 0, s);
    else if (a.T > 128 && tiles(256) >= 192) launch_shape<W8A8Shape<256, 256, 2, 4, 2>>(a, s);
    else if (a.T > 64 && tiles(128) >= 128) launch_shape<W8A8Shape<128, 128, 2, 2, 2>>(a, s);
    else if (a.T > 32 && tiles(32) > 512) launch_shape<W8A8Shape<64, 64, 2, 2, 4>>(a, s);
    else if (tiles(32) > 256 && tiles(32) <= 512) launch_split<2>(a, s);
    else launch_split<1>(a, s);
}

static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

// (none where the product's blocks quantise the rows)
size_t w8a8_workspace_bytes(int T, int K) {
    return gemv_takes(T, K) ? 0 : up256(size_t(T) * size_t(K)) + up256(size_t(T) * 4);
}

void launch_w8a8_linear(W8GemmArgs a, const void *x, int x_type, int64_t ldx, void *ws, hipStream_t s) {
    if (gemv_takes(a.T, a.K)) {
        w8_by_rows(x, x_type, ldx, a.T, [&](auto xt, auto vec) {
            launch_gemv<decltype(xt)::value, decltype(vec)::value>(a, x, ldx, s);
        });
        return;
    }
    int8_t *q = static_cast<int8_t *>(ws);
    float *sx = reinterpret_cast<float *>(q + up256(size_t(a.T) * size_t(a.K)));
    launch_quant_tokens(x, x_type, ldx, a.T, a.K, q, a.K, sx, s);
    a.q = q;
    a.ldq = a.K;
    a.sx = sx;
    launch_w8a8_gemm(a, s);
}

}  // namespace qwq4
