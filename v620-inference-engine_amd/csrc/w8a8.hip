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
template <int XT>
__device__ __forceinline__ float w8_load(const void *x, int64_t i) {
    if constexpr (XT == 0) return static_cast<const float *>(x)[i];
    else if constexpr (XT == 1) return bf16_bits_to_f32(static_cast<const uint16_t *>(x)[i]);
    else return f16_bits_to_f32(static_cast<const uint16_t *>(x)[i]);
}

// One row by one wave: two passes over it, 16 elements per lane and turn.
template <int XT>
__global__ __launch_bounds__(256) void quant_tokens_kernel(const void *__restrict__ x, int64_t ldx, int T, int K,
                                                           int8_t *__restrict__ q, int64_t ldq,
                                                           float *__restrict__ scale) {
    const int t = int(blockIdx.x) * 4 + int(threadIdx.x) / WAVE, lane = int(threadIdx.x) % WAVE;
    if (t >= T) return;
    const int64_t at = int64_t(t) * ldx;
    float mx = 0.f;
    bool bad = false;
    for (int k = lane; k < K; k += WAVE) {
        const float v = fabsf(w8_load<XT>(x, at + k));
        bad |= !(v <= 3.402823466e38f);
        mx = fmaxf(mx, v);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    bad = __any(bad);
    const float sc = bad ? __builtin_nanf("") : mx > 0.f ? fmaxf(mx / 127.f, 1.17549435e-38f) : 1.f, inv = 1.f / sc;
    for (int k0 = lane * 16; k0 < K; k0 += WAVE * 16) {
        uint32_t pk[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float v = bad ? 0.f : __builtin_rintf(w8_load<XT>(x, at + k0 + j) * inv);
            pk[j / 4] |= uint32_t(int(v) & 0xff) << (8 * (j % 4));
        }
        *reinterpret_cast<uint4 *>(q + int64_t(t) * ldq + k0) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    }
    if (lane == 0) scale[t] = sc;
}

void launch_quant_tokens(const void *x, int x_type, int64_t ldx, int T, int K, int8_t *q, int64_t ldq, float *scale,
                         hipStream_t s) {
    const unsigned blocks = unsigned((T + 3) / 4);
    if (x_type == 0) quant_tokens_kernel<0><<<blocks, 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else if (x_type == 1) quant_tokens_kernel<1><<<blocks, 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
    else quant_tokens_kernel<2><<<blocks, 256, 0, s>>>(x, ldx, T, K, q, ldq, scale);
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
