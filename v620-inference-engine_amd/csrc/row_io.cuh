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
