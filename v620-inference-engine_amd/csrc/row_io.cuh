// Rows of fp32, bf16 or fp16 elements: vector loads and stores through fp32
// values, and the dispatch over element types.
#pragma once

#include <type_traits>

#include "q4_common.cuh"

namespace qwq4 {

// (16-bit elements and the words that move them change places as values: an
// array of the one read through a pointer to the other is undefined, and has
// lost a store)
template <int V>
struct Halves {
    uint16_t h[V];
};

// V consecutive elements of type TY (QW_T_*), V a vector load's worth (16
// bytes: 4 or 8) or 1.
template <int TY, int V>
__device__ __forceinline__ void row_load(const void *x, int64_t i, float (&v)[V]) {
    if constexpr (TY == 0 && V == 1) {
        v[0] = static_cast<const float *>(x)[i];
    } else if constexpr (TY == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i + j);
            v[j] = f.x;
            v[j + 1] = f.y;
            v[j + 2] = f.z;
            v[j + 3] = f.w;
        }
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(x) + i;
        Halves<V> b;
        if constexpr (V == 8) b = __builtin_bit_cast(Halves<V>, *reinterpret_cast<const uint4 *>(p));
        else if constexpr (V == 4) b = __builtin_bit_cast(Halves<V>, *reinterpret_cast<const uint2 *>(p));
        else b.h[0] = p[0];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = TY == 1 ? bf16_bits_to_f32(b.h[j]) : f16_bits_to_f32(b.h[j]);
    }
}
// fp32 -> the nearest fp16, infinite beyond its range. (The value is taken as it
// is: the compiler would otherwise join the conversion with the multiplication
// before it, which then rounds once, and differently in 16-byte pieces and single
// elements.)
__device__ __forceinline__ _Float16 f32_to_f16_rne(float v) {
    asm volatile("" : "+v"(v));
    return _Float16(v);
}

// Finite values beyond fp16's +-65504 become those (activations), or, as type
// GRAD_F16, infinities (gradients: a loss scaler has to see them). A flag at run
// time would cost the forward 3% (4096 tokens of 8 choices, 4096 wide: 59.3 us
// against 57.7).
constexpr int GRAD_F16 = 3;
template <int TY, int V>
__device__ __forceinline__ void row_store(void *y, int64_t i, const float (&v)[V]) {
    if constexpr (TY == 0 && V == 1) {
        static_cast<float *>(y)[i] = v[0];
    } else if constexpr (TY == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4)
            *reinterpret_cast<float4 *>(static_cast<float *>(y) + i + j) =
                make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
        uint16_t *p = static_cast<uint16_t *>(y) + i;
        Halves<V> b;
#pragma unroll
        for (int j = 0; j < V; ++j)
            b.h[j] = TY == 1   ? f32_to_bf16_rne(v[j])
                   : TY == 2 ? __builtin_bit_cast(uint16_t, f32_to_f16_satfinite(v[j]))
                             : __builtin_bit_cast(uint16_t, f32_to_f16_rne(v[j]));
        if constexpr (V == 8) *reinterpret_cast<uint4 *>(p) = __builtin_bit_cast(uint4, b);
        else if constexpr (V == 4) *reinterpret_cast<uint2 *>(p) = __builtin_bit_cast(uint2, b);
        else p[0] = b.h[0];
    }
}

// Elements per thread: 8 of 16-bit rows or 4 of fp32 rows (16-byte loads of
// the rows that are read k times), where every row starts on what the widest
// of them needs, else 1.
inline bool rows_aligned(const void *p, int type, int64_t ld, int V) {
    const int64_t z = type == 0 ? 4 : 2, a = V * z < 16 ? V * z : 16;
    return !p || (reinterpret_cast<uintptr_t>(p) % size_t(a) == 0 && ld * z % a == 0);
}

// fp32 pairs -> 16-bit pairs (nearest even) and back
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 f = {a, b};
    if constexpr (__is_same(T, BF16)) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
}
template <class T>
__device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b) {
    if constexpr (__is_same(T, BF16)) {
        a = __builtin_bit_cast(float, w << 16);
        b = __builtin_bit_cast(float, w & 0xffff0000u);
    } else {
        a = f16_bits_to_f32(uint16_t(w));
        b = f16_bits_to_f32(uint16_t(w >> 16));
    }
}

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// 8 elements of a row as they lie (16-byte aligned), and their values.
template <int YT>
struct RowPiece {
    uint4 w[YT == 0 ? 2 : 1];
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        const char *at = static_cast<const char *>(p) + i * (YT == 0 ? 4 : 2);
        w[0] = reinterpret_cast<const uint4 *>(at)[0];
        if constexpr (YT == 0) w[1] = reinterpret_cast<const uint4 *>(at)[1];
    }
    // the same past the caches, for rows that nobody reads or writes again soon
    __device__ __forceinline__ void load_stream(const void *p, int64_t i) {
        const u32x4 *at = reinterpret_cast<const u32x4 *>(static_cast<const char *>(p) + i * (YT == 0 ? 4 : 2));
#pragma unroll
        for (int n = 0; n < (YT == 0 ? 2 : 1); ++n) w[n] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(at + n));
    }
    __device__ __forceinline__ void store_stream(void *p, int64_t i) const {
        u32x4 *at = reinterpret_cast<u32x4 *>(static_cast<char *>(p) + i * (YT == 0 ? 4 : 2));
#pragma unroll
        for (int n = 0; n < (YT == 0 ? 2 : 1); ++n) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, w[n]), at + n);
    }
    // (fp16: finite values beyond its range saturate, or, as a gradient, become infinite)
    template <bool GRAD>
    __device__ __forceinline__ void set(float (&v)[8]) {
        if constexpr (YT == 0) {
            w[0] = __builtin_bit_cast(uint4, f32x4{v[0], v[1], v[2], v[3]});
            w[1] = __builtin_bit_cast(uint4, f32x4{v[4], v[5], v[6], v[7]});
        } else {
            using T = std::conditional_t<YT == 1, BF16, F16>;
            if constexpr (YT != 1 && !GRAD) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __builtin_isfinite(v[j]) ? fminf(fmaxf(v[j], -65504.f), 65504.f) : v[j];
            }
            w[0] = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        if constexpr (YT == 0) {
            const f32x4 a = __builtin_bit_cast(f32x4, w[0]), b = __builtin_bit_cast(f32x4, w[1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j], v[j + 4] = b[j];
        } else {
            using T = std::conditional_t<YT == 1, BF16, F16>;
            unpack2<T>(w[0].x, v[0], v[1]);
            unpack2<T>(w[0].y, v[2], v[3]);
            unpack2<T>(w[0].z, v[4], v[5]);
            unpack2<T>(w[0].w, v[6], v[7]);
        }
    }
};

template <int N>
using Int = std::integral_constant<int, N>;

// f with a type code as a constant
template <class F>
inline void by_type(int type, F f) {
    if (type == 0) f(Int<0>{});
    else if (type == 1) f(Int<1>{});
    else f(Int<2>{});
}

}  // namespace qwq4
