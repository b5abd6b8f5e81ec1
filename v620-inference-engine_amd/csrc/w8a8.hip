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
    if (!w8_tile<S, 0>(ap, bp, a.K, acc, spare)) return;
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

// ------------------------------------------------------------ few tokens
// Up to 4 tokens the product is a stream of the weights (w8a8_gemv.cuh), 8 G
// rows of them per block, bound by memory (one token, 4096 -> 12288: 9.9 us,
// 5.1 TB/s; a large copy reaches 5.2). Device times from bf16 rows of 4096:
//                          1 token   2      4      8
//   4096 rows, streamed    4.7 us    6.1    8.1    11.1
//              tiles       10.7      10.6   11.1   11.1
//   12288 rows, streamed   9.9       11.5   14.5   18.8
//               tiles      14.3      14.5   14.3   14.8
// For one or two tokens the block quantises their rows itself, which saves the
// quantiser's launch (one token: 4.7 against 5.8 us and 9.9 against 11.5; two:
// 6.1 against 6.6 and 11.5 against 12.2).
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

static bool gemv_takes(int T, int K) { return T <= 4 && gemv_lds(T, K) <= W8_GEMV_LDS; }

template <int XT, bool VEC>
static void launch_gemv(const W8GemmArgs &a, const void *x, int64_t ldx, hipStream_t s) {
    // (16 rows a block where that leaves blocks enough: 2 tokens and 12288 rows
    // take 11.5 us against 13.8 with 8, 4096 rows 6.3 against 6.1)
    auto run = [&](auto tm) {
        constexpr int TM = decltype(tm)::value;
        const size_t lds = gemv_lds(TM, a.K);
        if (a.N >= 8192)
            w8a8_gemv_kernel<XT, VEC, TM, 2><<<unsigned((a.N + 15) / 16), 256, lds, s>>>(a, x, ldx);
        else w8a8_gemv_kernel<XT, VEC, TM, 1><<<unsigned((a.N + 7) / 8), 256, lds, s>>>(a, x, ldx);
    };
    if (a.T <= 1) run(std::integral_constant<int, 1>{});
    else if (a.T <= 2) run(std::integral_constant<int, 2>{});
    else if constexpr (XT == 3) run(std::integral_constant<int, 4>{});
}

// Few tokens stream the weights; else the largest tile that still makes about
// a block for every CU. Measured (us; rows x weight rows x K, tiles of 256, 128,
// 64, 32): 4096 x 12288 x 4096: 237, 270, 406, 685; 1024 x 4096 x 4096: 55, 34, 36,
// 71; 600 x 4096 x 6144: 75, 46, 38, 61; 256 x 4096 x 4096: 55, 31, 12.9, 21.7;
// 37 x 12288 x 4096: 52, 33, 14.5, 17.5; 37 x 4096 x 6144: 74, 45, 16.6, 15.2.
void launch_w8a8_gemm(const W8GemmArgs &a, hipStream_t s) {
    auto tiles = [&](int b) { return int64_t((a.T + b - 1) / b) * ((a.N + b - 1) / b); };
    if (gemv_takes(a.T, a.K)) launch_gemv<3, true>(a, nullptr, 0, s);
    else if (a.T > 128 && tiles(256) >= 192) launch_shape<W8A8Shape<256, 256, 2, 4, 1, 2>>(a, s);
    else if (a.T > 64 && tiles(128) >= 128) launch_shape<W8A8Shape<128, 128, 2, 2, 1, 2>>(a, s);
    else if (a.T > 32 && tiles(64) >= 128) launch_shape<W8A8Shape<64, 64, 2, 2, 1, 4>>(a, s);
    else launch_shape<W8A8Shape<32, 32, 1, 1, 4, 4>>(a, s);
}

static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

size_t w8a8_workspace_bytes(int T, int K) { return up256(size_t(T) * size_t(K)) + up256(size_t(T) * 4); }

void launch_w8a8_linear(W8GemmArgs a, const void *x, int x_type, int64_t ldx, void *ws, hipStream_t s) {
    if (a.T <= 2 && gemv_takes(a.T, a.K)) {
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
