// The W8A8 products of few tokens: a stream of the weights. Shared by the dense
// product (w8a8.hip) and the routed experts (moe_w8a8.hip).
//
// A block of 4 waves takes 8 G weight rows. The waves take the 128-byte steps
// of K in turn; a wave instruction reads 128 bytes of each of 8 rows (whole
// cache lines of the row-major matrix), lane (row, chunk) multiplies its 16
// bytes by the tokens' in LDS with v_dot4, and the 8 chunks and 4 waves are
// added at the end, in whole numbers. The first weights are requested before
// the tokens' rows are staged (and, where they come as 16- or 32-bit rows,
// quantised), which hides behind them.
#pragma once

#include <type_traits>

#include "w8a8_core.cuh"

namespace qwq4 {

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


// f with the rows' type and whether each is 16-byte aligned, as constants
template <class F>
inline void w8_by_rows(const void *x, int x_type, int64_t ldx, int T, F f) {
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (T == 1 || ldx * (x_type == 0 ? 4 : 2) % 16 == 0);
    auto run = [&](auto xt) {
        if (vec) f(xt, std::true_type{});
        else f(xt, std::false_type{});
    };
    if (x_type == 0) run(std::integral_constant<int, 0>{});
    else if (x_type == 1) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 2>{});
}

// ------------------------------------------------------------ the stream
constexpr int GEMV_U = 8;                // steps a wave has on their way per row
constexpr size_t W8_GEMV_LDS = 64 << 10;  // bytes a block stages of the tokens' rows at most

// LDS of T tokens' rows (staged for 1, 2, 4 or 8)
__host__ __device__ inline size_t gemv_lds(int T, int K) {
    return size_t(T <= 1 ? 1 : T <= 2 ? 2 : T <= 4 ? 4 : 8) * size_t((K + 127) / 128 * 128);
}

__device__ __forceinline__ int gemv_wave() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE); }
__device__ __forceinline__ int gemv_row() { return int(threadIdx.x) % WAVE / 8; }  // the lane's row of 8

template <int G>
struct W8Stream {
    i32x4 v[GEMV_U][G];
    // steps s0, s0 + 4, .. of the rows (those there are); past a row's end any
    // of its bytes (the tokens' are zeros there)
    __device__ __forceinline__ void load(const int8_t *const (&w)[G], int K, int s0) {
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u) {
            if ((s0 + 4 * u) * 128 >= K) break;
#pragma unroll
            for (int g = 0; g < G; ++g)
                v[u][g] = __builtin_nontemporal_load(reinterpret_cast<const i32x4 *>(
                    w[g] + 16 * int64_t(min((s0 + 4 * u) * 8 + int(threadIdx.x) % 8, K / 16 - 1))));
        }
    }
};

// TM tokens' int8 rows into LDS, zeros from K on; token(t): row of q and sx.
template <int TM, class TokenF>
__device__ __forceinline__ void gemv_stage_i8(const int8_t *q, int64_t ldq, const float *scales, int K,
                                              unsigned char *s_q, float (&sx)[TM], TokenF token) {
    const int n16 = K / 16, kp = (K + 127) / 128 * 128;
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const uint4 *p = reinterpret_cast<const uint4 *>(q + token(t) * ldq);
        for (int i = int(threadIdx.x); i < kp / 16; i += 256)
            *reinterpret_cast<uint4 *>(s_q + t * kp + 16 * i) = i < n16 ? p[i] : make_uint4(0u, 0u, 0u, 0u);
        sx[t] = scales[token(t)];
    }
    __syncthreads();
}

// The same from rows of type XT, quantised on the way.
template <int XT, bool VEC, int TM, class TokenF>
__device__ __forceinline__ void gemv_stage(const void *x, int64_t ldx, int K, unsigned char *s_q, float (&sx)[TM],
                                           TokenF token) {
    __shared__ uint32_t s_top[TM][4];
    const int tid = int(threadIdx.x), n16 = K / 16, kp = (K + 127) / 128 * 128;
    constexpr int C = 2;  // the first C turns' elements are kept (rows up to 8192), the rest read again
    W8Raw<XT, VEC> raw[TM][C];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int64_t at = token(t) * ldx;
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
        if (tid % WAVE == 0) s_top[t][tid / WAVE] = top;
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
            if (i < n16) r.load(x, token(t) * ldx + i * 16);
            else r.clear();
            put(i, r);
        }
    }
    __syncthreads();
}

// The sums of TM staged tokens with the 8 G rows w (v: their first steps,
// loaded): out(sum) is run by every thread, sum(t, r) being that of token t
// with row r. A barrier has to come before the next staging.
template <int TM, int G, class OutF>
__device__ __forceinline__ void gemv_sums(W8Stream<G> &v, const int8_t *const (&w)[G], int K,
                                          const unsigned char *s_q, OutF out) {
    __shared__ int s_sum[4][TM][8 * G];
    const int tid = int(threadIdx.x), lane = tid % WAVE, steps = (K + 127) / 128, kp = steps * 128;
    int acc[TM][G];
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) acc[t][g] = 0;
    const int first = gemv_wave();
    for (int s0 = first; s0 < steps; s0 += 4 * GEMV_U) {
        if (s0 != first) v.load(w, K, s0);
#pragma unroll
        for (int u = 0; u < GEMV_U; ++u) {
            if (s0 + 4 * u >= steps) break;
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const i32x4 q = *reinterpret_cast<const i32x4 *>(s_q + t * kp + (s0 + 4 * u) * 128 + lane % 8 * 16);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[t][g] = __builtin_amdgcn_sdot4(v.v[u][g][e], q[e], acc[t][g], false);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TM; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) acc[t][g] += __shfl_xor(acc[t][g], o);
            if (lane % 8 == 0) s_sum[first][t][8 * g + lane / 8] = acc[t][g];
        }
    __syncthreads();
    auto sum = [&](int t, int r) { return s_sum[0][t][r] + s_sum[1][t][r] + s_sum[2][t][r] + s_sum[3][t][r]; };
    out(sum);
}

// sx[t] for a t that is not a constant
template <int TM>
__device__ __forceinline__ float gemv_pick(const float (&sx)[TM], int t) {
    float s = sx[0];
#pragma unroll
    for (int u = 1; u < TM; ++u) s = t == u ? sx[u] : s;
    return s;
}

}  // namespace qwq4
