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
    __device__ __forceinline__ uint32_t top(uint32_t t) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) t = max(t, __builtin_bit_cast(uint32_t, value(i)) & 0x7fffffffu);
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

void launch_quant_tokens(const void *x, int x_type, int64_t ldx, int T, int K, int8_t *q, int64_t ldq, float *scale,
                         hipStream_t s) {
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx * (x_type == 0 ? 4 : 2) % 16 == 0);
    auto run = [&](auto xt) {
        if (vec) launch_quant_x<decltype(xt)::value, true>(x, ldx, T, K, q, ldq, scale, s);
        else launch_quant_x<decltype(xt)::value, false>(x, ldx, T, K, q, ldq, scale, s);
    };
    if (x_type == 0) run(std::integral_constant<int, 0>{});
    else if (x_type == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
}

// ------------------------------------------------------------ product
template <class S>
__global__ __launch_bounds__(S::THREADS) void w8a8_gemm_kernel(W8GemmArgs a) {
    const int nt = (a.N + S::BN - 1) / S::BN;
    const int m0 = int(blockIdx.x) / nt * S::BM, n0 = int(blockIdx.x) % nt * S::BN;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::AJ; ++j) ap[j] = a.q + int64_t(min(m0 + S::load_row(j), a.T - 1)) * a.ldq;
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) bp[j] = a.W + int64_t(min(n0 + S::load_row(j), a.N - 1)) * a.ldw;
    i32x16 acc[S::MT][S::NT];
    w8_clear<S>(acc);
    if (!w8_tile<S, 0>(ap, bp, a.K, acc)) return;
#pragma unroll
    for (int j = 0; j < S::NT; ++j) {
        const int n = n0 + S::n_of(j);
        if (n >= a.N) continue;
        const float sw = a.sw[n];
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + S::m_of(i, r);
                if (m < a.T) w8_store(a.Y, a.y_type, int64_t(m) * a.ldy + n, w8_value(acc[i][j][r], sw, a.sx[m]));
            }
    }
}

template <class S>
static void launch_shape(const W8GemmArgs &a, hipStream_t s) {
    const unsigned tiles = unsigned((a.T + S::BM - 1) / S::BM) * unsigned((a.N + S::BN - 1) / S::BN);
    w8a8_gemm_kernel<S><<<tiles, S::THREADS, 0, s>>>(a);
}

void launch_w8a8_gemm(const W8GemmArgs &a, hipStream_t s) {
    if (a.T <= 64) launch_shape<W8Shape<32, 32, 1, 1, 4, 4>>(a, s);
    else if (a.T <= 1024) launch_shape<W8Shape<128, 128, 2, 2, 1, 2>>(a, s);
    else launch_shape<W8Shape<256, 256, 2, 4, 1, 2>>(a, s);
}

static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

size_t w8a8_workspace_bytes(int T, int K) { return up256(size_t(T) * size_t(K)) + up256(size_t(T) * 4); }

void launch_w8a8_linear(W8GemmArgs a, const void *x, int x_type, int64_t ldx, void *ws, hipStream_t s) {
    int8_t *q = static_cast<int8_t *>(ws);
    float *sx = reinterpret_cast<float *>(q + up256(size_t(a.T) * size_t(a.K)));
    launch_quant_tokens(x, x_type, ldx, a.T, a.K, q, a.K, sx, s);
    a.q = q;
    a.ldq = a.K;
    a.sx = sx;
    launch_w8a8_gemm(a, s);
}

}  // namespace qwq4
