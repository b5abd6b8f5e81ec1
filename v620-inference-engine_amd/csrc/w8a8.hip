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

namespace qwq4 {

// ------------------------------------------------------------ quantiser
// The row scale of a maximum, and whether a row's values are all finite: a
// row that is not gets scale NaN and zeros. (The maximum is taken over the
// magnitudes' bit patterns: an infinity or NaN then has the largest.)
__device__ __forceinline__ float w8_scale(uint32_t top, bool &finite) {
    finite = top < 0x7f800000u;
    const float mx = __builtin_bit_cast(float, top);
    return !finite ? __builtin_nanf("") : top ? fmaxf(mx / 127.f, 1.17549435e-38f) : 1.f;
}

// 16 consecutive elements of a row of type XT as loaded, and their values.
// VEC: the row is 16-byte aligned.
template <int XT, bool VEC>
struct W8Raw {
    static constexpr int W = XT == 0 ? 16 : 8;
    uint32_t w[W];
    __device__ __forceinline__ void load(const void *x, int64_t at) {
        if constexpr (VEC) {
            const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint32_t *>(x) + (XT == 0 ? at : at / 2));
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const uint4 v = p[i];
                w[4 * i] = v.x;
                w[4 * i + 1] = v.y;
                w[4 * i + 2] = v.z;
                w[4 * i + 3] = v.w;
            }
        } else if constexpr (XT == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = static_cast<const uint32_t *>(x)[at + i];
        } else {
            const uint16_t *p = static_cast<const uint16_t *>(x) + at;
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = uint32_t(p[2 * i]) | uint32_t(p[2 * i + 1]) << 16;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (XT == 0) return __builtin_bit_cast(float, w[i]);
        const uint16_t b = uint16_t(w[i / 2] >> (16 * (i % 2)));
        return XT == 1 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
    }
    // (the words are taken anew afterwards: the values would otherwise stay
    // in registers, two to a word)
    __device__ __forceinline__ uint32_t top(uint32_t t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) t = max(t, __builtin_bit_cast(uint32_t, value(i)) & 0x7fffffffu);
#pragma unroll
        for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
        return t;
    }
    __device__ __forceinline__ uint4 quantised(float inv, bool finite) const {
        uint32_t q[4] = {0u, 0u, 0u, 0u};
        if (finite) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                q[i / 4] |= uint32_t(int(__builtin_rintf(value(i) * inv)) & 0xff) << (8 * (i % 4));
        }
        return make_uint4(q[0], q[1], q[2], q[3]);
    }
};

__device__ __forceinline__ uint32_t wave_top(uint32_t t) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) t = max(t, uint32_t(__shfl_xor(int(t), o)));
    return t;
}

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

// f with the rows' type and whether each is 16-byte aligned, as constants
template <class F>
static void by_rows(const void *x, int x_type, int64_t ldx, int T, F f) {
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx * (x_type == 0 ? 4 : 2) % 16 == 0);
    auto run = [&](auto xt) {
        if (vec) f(xt, std::true_type{});
        else f(xt, std::false_type{});
    };
    if (x_type == 0) run(std::integral_constant<int, 0>{});
    else if (x_type == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
}

void launch_quant_tokens(const void *x, int x_type, int64_t ldx, int T, int K, int8_t *q, int64_t ldq, float *scale,
                         hipStream_t s) {
    by_rows(x, x_type, ldx, T, [&](auto xt, auto vec) {
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
// Up to 8 tokens the product is a stream of the weights. A block takes 8 G
// weight rows, its 4 waves the 128-byte steps of K in turn: a wave instruction
// reads 128 bytes of each of 8 rows (whole cache lines of the row-major
// matrix), lane (row, chunk) multiplies its 16 bytes by the tokens' in LDS
// with v_dot4, and the 8 chunks and 4 waves are added at the end. For one or
// two tokens the block quantises their rows itself (XT 0 to 2; 3: int8 rows
// with their scales): that hides behind the first weights, which are requested
// before, and saves the quantiser's launch (one token, 4096 -> 12288 from bf16:
// 12.6 us against 15.2 in two launches).
template <int XT, bool VEC, int TM, int G>
__global__ __launch_bounds__(256) void w8a8_gemv_kernel(W8GemmArgs a, const void *x, int64_t ldx) {
    extern __shared__ __align__(16) unsigned char s_q[];  // [TM][kp]: the rows' 8 bits, zeros from K on
    __shared__ uint32_t s_top[TM][4];
    __shared__ int s_sum[4][TM][8 * G];
    const int tid = int(threadIdx.x), wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int K = a.K, n16 = K / 16, steps = (K + 127) / 128, kp = steps * 128;
    const int n0 = int(blockIdx.x) * 8 * G;
    constexpr int U = 8;  // steps a wave has on their way per row
    const int8_t *w[G];
#pragma unroll
    for (int g = 0; g < G; ++g) w[g] = a.W + int64_t(min(n0 + 8 * g + lane / 8, a.N - 1)) * a.ldw;
    i32x4 v[U][G];
    // steps s0 + 4 u of the wave; past the row's end any of its bytes (the
    // tokens' are zeros there)
    auto load = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int g = 0; g < G; ++g)
                v[u][g] = __builtin_nontemporal_load(reinterpret_cast<const i32x4 *>(
                    w[g] + 16 * int64_t(min((s0 + 4 * u) * 8 + lane % 8, n16 - 1))));
    };
    load(wave);
    float sx[TM];
    if constexpr (XT == 3) {
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const uint4 *q = reinterpret_cast<const uint4 *>(a.q + int64_t(min(t, a.T - 1)) * a.ldq);
            for (int i = tid; i < kp / 16; i += 256)
                *reinterpret_cast<uint4 *>(s_q + t * kp + 16 * i) = i < n16 ? q[i] : make_uint4(0u, 0u, 0u, 0u);
            sx[t] = a.sx[min(t, a.T - 1)];
        }
    } else {
        constexpr int C = 2;  // the first C turns' elements are kept (rows up to 8192), the rest read again
        W8Raw<XT, VEC> raw[TM][C];
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const int64_t at = min(t, a.T - 1) * ldx;
            uint32_t top = 0u;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (tid + 256 * c < n16) raw[t][c].load(x, at + (tid + 256 * c) * 16);
                else raw[t][c].clear();
            }
#pragma unroll
            for (int c = 0; c < C; ++c) top = raw[t][c].top(top);
            for (int i = tid + 256 * C; i < n16; i += 256) {
                W8Raw<XT, VEC> r;
                r.load(x, at + i * 16);
                top = r.top(top);
            }
            top = wave_top(top);
            if (lane == 0) s_top[t][wave] = top;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            bool finite;
            sx[t] = w8_scale(max(max(s_top[t][0], s_top[t][1]), max(s_top[t][2], s_top[t][3])), finite);
            const float inv = 1.f / sx[t];
            auto put = [&](int i, const W8Raw<XT, VEC> &r) {
                *reinterpret_cast<uint4 *>(s_q + t * kp + 16 * i) = r.quantised(inv, finite);
            };
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (tid + 256 * c < kp / 16) put(tid + 256 * c, raw[t][c]);  // (zeros from K on)
            for (int i = tid + 256 * C; i < kp / 16; i += 256) {
                W8Raw<XT, VEC> r;
                if (i < n16) r.load(x, min(t, a.T - 1) * ldx + i * 16);
                else r.clear();
                put(i, r);
            }
        }
    }
    __syncthreads();
    int acc[TM][G];
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) acc[t][g] = 0;
    for (int s0 = wave; s0 < steps; s0 += 4 * U) {
        if (s0 != wave) load(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + 4 * u >= steps) break;
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const i32x4 q = *reinterpret_cast<const i32x4 *>(s_q + t * kp + (s0 + 4 * u) * 128 + lane % 8 * 16);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][g] = __builtin_amdgcn_sdot4(v[u][g][e], q[e], acc[t][g], false);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) acc[t][g] += __shfl_xor(acc[t][g], o);
            if (lane % 8 == 0) s_sum[wave][t][8 * g + lane / 8] = acc[t][g];
        }
    __syncthreads();
    for (int i = tid; i < TM * 8 * G; i += 256) {
        const int t = i / (8 * G), r = i % (8 * G), n = n0 + r;
        if (t >= a.T || n >= a.N) continue;
        float s = sx[0];
#pragma unroll
        for (int u = 1; u < TM; ++u) s = t == u ? sx[u] : s;
        w8_store(a.Y, a.y_type, int64_t(t) * a.ldy + n,
                 w8_value(s_sum[0][t][r] + s_sum[1][t][r] + s_sum[2][t][r] + s_sum[3][t][r], a.sw[n], s));
    }
}

constexpr int W8_GEMV_LDS = 64 << 10;  // what a block stages of the tokens' rows at most

static bool gemv_takes(int T, int K) {
    const int tm = T <= 1 ? 1 : T <= 2 ? 2 : T <= 4 ? 4 : 8;
    return T <= 8 && int64_t(tm) * ((K + 127) / 128 * 128) <= W8_GEMV_LDS;
}

template <int XT, bool VEC>
static void launch_gemv(const W8GemmArgs &a, const void *x, int64_t ldx, hipStream_t s) {
    auto run = [&](auto tm) {
        constexpr int TM = decltype(tm)::value;
        const size_t lds = size_t(TM) * size_t((a.K + 127) / 128 * 128);
        if (a.N >= 8192)
            w8a8_gemv_kernel<XT, VEC, TM, 2><<<unsigned((a.N + 15) / 16), 256, lds, s>>>(a, x, ldx);
        else w8a8_gemv_kernel<XT, VEC, TM, 1><<<unsigned((a.N + 7) / 8), 256, lds, s>>>(a, x, ldx);
    };
    if (a.T <= 1) run(std::integral_constant<int, 1>{});
    else if (a.T <= 2) run(std::integral_constant<int, 2>{});
    else if constexpr (XT == 3) {
        if (a.T <= 4) run(std::integral_constant<int, 4>{});
        else run(std::integral_constant<int, 8>{});
    }
}

// Few tokens stream the weights; else the largest tile that still makes about
// a block for every CU.
void launch_w8a8_gemm(const W8GemmArgs &a, hipStream_t s) {
    auto tiles = [&](int b) { return int64_t((a.T + b - 1) / b) * ((a.N + b - 1) / b); };
    if (gemv_takes(a.T, a.K)) launch_gemv<3, true>(a, nullptr, 0, s);
    else if (a.T > 128 && tiles(256) >= 192) launch_shape<W8Shape<256, 256, 2, 4, 1, 128, 2>>(a, s);
    else if (a.T > 64 && tiles(128) >= 128) launch_shape<W8Shape<128, 128, 2, 2, 1, 128, 2>>(a, s);
    else if (a.T > 32 && tiles(64) >= 128) launch_shape<W8Shape<64, 64, 2, 2, 1, 128, 4>>(a, s);
    else launch_shape<W8Shape<32, 32, 1, 1, 4, 128, 4>>(a, s);
}

static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

size_t w8a8_workspace_bytes(int T, int K) { return up256(size_t(T) * size_t(K)) + up256(size_t(T) * 4); }

void launch_w8a8_linear(W8GemmArgs a, const void *x, int x_type, int64_t ldx, void *ws, hipStream_t s) {
    if (a.T <= 2 && gemv_takes(a.T, a.K)) {
        by_rows(x, x_type, ldx, a.T, [&](auto xt, auto vec) {
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
