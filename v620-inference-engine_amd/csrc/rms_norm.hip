// Root-mean-square norm of rows, with the residual's addition in front and an
// output in 16 bits, fp32 or int8 with a scale per row, and its gradients.
//
//   h = x + residual,  r = 1 / sqrt(mean(h^2) + eps),  y = h r w
//   int8: u = h w,  c = max |u| / 127,  q = rint(u (1 / c)),  scale = r c
//   g = dy w,  dh = r (g - h r^2 mean(g h)) + dres,  dw = sum_t dy h r
//
// The 8-bit values do not depend on r (it cancels in u / max |u|), so the
// row's sum of squares and its largest |u| come out of the same pass, and q
// does not change with the order of the sum. Sums are in fp32; h is
// normalised as added, the residual is rounded to its own type beside it.
#include <algorithm>

#include "q4_kernels.hpp"
#include "row_io.cuh"

namespace qwq4 {

// 8 elements from index j on of a row of n (VEC: n is a multiple of 8 and the
// row starts on 16 bytes), those behind the row's end as zeros. A piece that
// starts anywhere is moved in one access too, which memory takes off its alignment
// (single elements throughout: 1024 rows of 16380 98 us for 34, of 4100 72 for 34), and
// only the last one of a row, if it is not whole, element by element. The same
// threads have the same elements either way: a row's bits do not depend on how it lies.
template <int TY, bool VEC>
__device__ __forceinline__ void part_load(const void *x, int64_t row, int j, int n, float (&v)[8]) {
    if constexpr (VEC) {
        row_load<TY, 8>(x, row + j, v);
    } else if (j + 8 <= n) {
        RowPiece<TY> w;
        __builtin_memcpy(&w, static_cast<const char *>(x) + (row + j) * (TY == 0 ? 4 : 2), sizeof(w));
        w.values(v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float one[1];
            row_load<TY, 1>(x, row + min(j + e, n - 1), one);
            v[e] = j + e < n ? one[0] : 0.f;
        }
    }
}
template <int TY, bool VEC>
__device__ __forceinline__ void part_store(void *y, int64_t row, int j, int n, const float (&v)[8]) {
    if constexpr (VEC) {
        row_store<TY, 8>(y, row + j, v);
    } else if (j + 8 <= n) {
        constexpr int Z = TY == 0 ? 4 : 2;
        __align__(16) char w[8 * Z];
        row_store<TY, 8>(w, 0, v);
        __builtin_memcpy(static_cast<char *>(y) + (row + j) * Z, w, sizeof(w));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float one[1] = {v[e]};
            if (j + e < n) row_store<TY, 1>(y, row + j + e, one);
        }
    }
}

// The same with a type known at run time (one for the whole launch). Stores
// only: with three loads to choose from at run time the compiler has left
// values undefined that the third passes by.
template <bool VEC>
__device__ __forceinline__ void any_store(void *y, int type, int64_t row, int j, int n, const float (&v)[8]) {
    if (type == 0) part_store<0, VEC>(y, row, j, n, v);
    else if (type == 1) part_store<1, VEC>(y, row, j, n, v);
    else part_store<2, VEC>(y, row, j, n, v);
}

// the sum over groups of G lanes
template <int G>
__device__ __forceinline__ float group_add(float v) {
#pragma unroll
    for (int o = G / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// 8 elements of h = x + residual (RT < 0: no residual).
template <int XT, int RT, bool VEC>
__device__ __forceinline__ void load_h(const NormArgs &a, int64_t x0, int64_t r0, int j, float (&h)[8]) {
    part_load<XT, VEC>(a.x, x0, j, a.H, h);
    if constexpr (RT >= 0) {
        float r[8];
        part_load<RT, VEC>(a.res, r0, j, a.H, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[e] += r[e];
    }
}

// A row by G threads (16: a wave takes four; 64: a wave; 256: the block), 8
// elements per thread and turn. C > 0: the row is held in C turns' registers
// and read once; C = 0: any length, read twice (the second time from the
// caches; the residual is written then, since it may lie on its input).
// Bound by memory.
template <int XT, int RT, int WT, bool I8, bool VEC, int G, int C>
__global__ __launch_bounds__(256) void rms_norm_kernel(NormArgs a) {
    const int li = int(threadIdx.x) % G, H = a.H;
    const int64_t t = int64_t(blockIdx.x) * (256 / G) + int(threadIdx.x) / G;
    if (t >= a.T) return;  // (whole groups, where G < 256: they meet no barrier)
    const int64_t x0 = t * a.ldx, r0 = t * a.ldr, o0 = t * a.ldro, y0 = t * a.ldy;
    float h[C > 0 ? C : 1][8], w[C > 0 ? C : 1][8];
    float sum = 0.f;
    uint32_t top = 0u;
    auto count = [&](const float (&v)[8], const float (&wv)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum = __builtin_fmaf(v[e], v[e], sum);
            if constexpr (I8) top = max(top, __builtin_bit_cast(uint32_t, v[e] * wv[e]) & 0x7fffffffu);
        }
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if (j < H) {
                load_h<XT, RT, VEC>(a, x0, r0, j, h[c]);
                part_load<WT, VEC>(a.w, 0, j, H, w[c]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[c][e] = w[c][e] = 0.f;
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if constexpr (RT >= 0) {
                if (j < H) part_store<RT, VEC>(a.res_out, o0, j, H, h[c]);
            }
            count(h[c], w[c]);
        }
    } else {
        for (int j = li * 8; j < H; j += G * 8) {
            load_h<XT, RT, VEC>(a, x0, r0, j, h[0]);
            if constexpr (I8) part_load<WT, VEC>(a.w, 0, j, H, w[0]);
            count(h[0], w[0]);
        }
    }
    sum = group_add<G < WAVE ? G : WAVE>(sum);
    if constexpr (I8) {
#pragma unroll
        for (int o = (G < WAVE ? G : WAVE) / 2; o >= 1; o >>= 1) top = max(top, uint32_t(__shfl_xor(int(top), o)));
    }
    if constexpr (G == 256) {
        __shared__ float s_sum[4];
        __shared__ uint32_t s_top[4];
        if (li % WAVE == 0) {
            s_sum[li / WAVE] = sum;
            if constexpr (I8) s_top[li / WAVE] = top;
        }
        __syncthreads();
        sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        if constexpr (I8) top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    }
    const float r = 1.f / sqrtf(sum / float(H) + a.eps);
    // (as the quantiser of rows: a row of zeros has step 1, an infinity or a NaN gives a NaN scale)
    const bool finite = top < 0x7f800000u;
    float step = 1.f, inv = 1.f;
    if constexpr (I8) {
        step = !finite ? __builtin_nanf("") : top ? fmaxf(__builtin_bit_cast(float, top) / 127.f, 1.17549435e-38f) : 1.f;
        inv = 1.f / step;
    }
    auto put = [&](int j, const float (&v)[8], const float (&wv)[8]) {
        if constexpr (I8) {
            uint32_t q[2] = {0u, 0u};
            if (finite) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    q[e / 4] |= uint32_t(int(__builtin_rintf(v[e] * wv[e] * inv)) & 0xff) << (8 * (e % 4));
            }
            int8_t *p = static_cast<int8_t *>(a.y) + y0 + j;
            if constexpr (VEC) {
                *reinterpret_cast<uint2 *>(p) = make_uint2(q[0], q[1]);
            } else if (j + 8 <= H) {
                __builtin_memcpy(p, q, sizeof(q));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j + e < H) p[e] = int8_t(q[e / 4] >> (8 * (e % 4)));
            }
        } else {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = v[e] * r * wv[e];
            any_store<VEC>(a.y, a.y_type, y0, j, H, o);
        }
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if (j < H) put(j, h[c], w[c]);
        }
    } else {
        for (int j = li * 8; j < H; j += G * 8) {
            load_h<XT, RT, VEC>(a, x0, r0, j, h[0]);
            part_load<WT, VEC>(a.w, 0, j, H, w[0]);
            if constexpr (RT >= 0) part_store<RT, VEC>(a.res_out, o0, j, H, h[0]);
            put(j, h[0], w[0]);
        }
    }
    if constexpr (I8) {
        if (li == 0) a.scale[t] = step * r;
    }
}

template <int XT, int RT, int WT, bool I8>
static void launch_norm(const NormArgs &a, hipStream_t s) {
    auto run = [&](auto vec, auto g, auto c) {
        constexpr int G = decltype(g)::value, ROWS = 256 / G;
        rms_norm_kernel<XT, RT, WT, I8, decltype(vec)::value, G, decltype(c)::value>
            <<<unsigned((a.T + ROWS - 1) / ROWS), 256, 0, s>>>(a);
    };
    // (16.8 million elements in bf16 with a residual: rows of 64 by waves 100 us, by 16 lanes 29; of 520 by blocks 37, by
    // waves 28)
    auto by_length = [&](auto vec) {
        if (a.H <= 128) run(vec, Int<16>{}, Int<1>{});
        else if (a.H <= 256) run(vec, Int<16>{}, Int<2>{});
        else if (a.H <= 512) run(vec, Int<64>{}, Int<1>{});
        else if (a.H <= 1024) run(vec, Int<64>{}, Int<2>{});
        else if (a.H <= 2048) run(vec, Int<256>{}, Int<1>{});
        else if (a.H <= 4096) run(vec, Int<256>{}, Int<2>{});
        else if (a.H <= 8192) run(vec, Int<256>{}, Int<4>{});
        else run(vec, Int<256>{}, Int<0>{});
    };
    const int64_t one = a.T == 1 ? 0 : 1;  // (a single row's stride does not matter)
    const bool out = I8 ? reinterpret_cast<uintptr_t>(a.y) % 8 == 0 && one * a.ldy % 8 == 0
                        : rows_aligned(a.y, a.y_type, one * a.ldy, 8);
    if (a.H % 8 == 0 && out && rows_aligned(a.x, XT, one * a.ldx, 8) && rows_aligned(a.w, WT, 0, 8) &&
        (RT < 0 || (rows_aligned(a.res, RT, one * a.ldr, 8) && rows_aligned(a.res_out, RT, one * a.ldro, 8))))
        by_length(std::true_type{});
    else
        by_length(std::false_type{});
}

void launch_rms_norm(const NormArgs &a, hipStream_t s) {
    by_type(a.x_type, [&](auto xt) {
        constexpr int XT = decltype(xt)::value;
        auto run = [&](auto rt, auto wt) {
            constexpr int RT = decltype(rt)::value, WT = decltype(wt)::value;
            if (a.scale) launch_norm<XT, RT, WT, true>(a, s);
            else launch_norm<XT, RT, WT, false>(a, s);
        };
        auto by_residual = [&](auto wt) {
            if (!a.res) run(Int<-1>{}, wt);
            else if (a.res_type == 0) run(Int<0>{}, wt);
            else run(xt, wt);
        };
        if (a.w_type == 0) by_residual(Int<0>{});
        else by_residual(xt);
    });
}

// ------------------------------------------------------------ gradients
// 8 elements of a row on their way, as they lie (unpacked, those of rows that start
// anywhere would take twice the registers: 1024 bf16 rows of 16380 120 us for 38). The
// last piece of such a row is its last 8 elements in one access, moved to their places,
// with zeros behind them, when the values are asked for. SHORT: a row may have fewer than 8.
template <int TY, bool VEC, bool SHORT>
struct Part {
    RowPiece<TY> w;
    using E = std::conditional_t<TY == 0, uint32_t, uint16_t>;
    struct Eight {
        E e[8];
    };
    __device__ __forceinline__ void load(const void *x, int64_t row, int j, int n) {
        if constexpr (VEC) {
            w.load(x, row + j);
            return;
        }
        const E *p = static_cast<const E *>(x) + row;
        if (SHORT && n < 8) {
            Eight one;
#pragma unroll
            for (int e = 0; e < 8; ++e) one.e[e] = p[min(e, n - 1)];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= n) one.e[e] = 0;
            w = __builtin_bit_cast(RowPiece<TY>, one);
        } else {
            __builtin_memcpy(&w, p + min(j, n - 8), sizeof(w));
        }
    }
    template <class T>
    __device__ __forceinline__ static void to_places(T (&v)[8], int j, int n) {
        if (VEC || j + 8 <= n || (SHORT && n < 8)) return;
        const int by = j + 8 - n;
#pragma unroll
        for (int s = 4; s >= 1; s >>= 1) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = !(by & s) ? v[e] : e + s < 8 ? v[(e + s) % 8] : T(0);
        }
    }
    __device__ __forceinline__ void values(float (&v)[8], int j, int n) const {
        w.values(v);
        to_places(v, j, n);
    }
    // the elements at their places for good: w.values has them (for what is read once and used for every row)
    __device__ __forceinline__ void settle(int j, int n) {
        if constexpr (VEC) return;
        Eight v = __builtin_bit_cast(Eight, w);
        to_places(v.e, j, n);
        w = __builtin_bit_cast(RowPiece<TY>, v);
    }
};

// A row by G of the block's TH threads (16, 64: groups of a wave, which meet no
// barrier but the last; more: of waves), 8 elements per thread and C turns each. A
// group takes every (groups of the grid)-th row, with the next one on its way
// while the current one's sums are made (but in blocks of 1024), and keeps its
// columns' part of dw in registers; the block adds its groups' parts and a second
// launch the blocks', in order. Bound by memory.
template <int DT, int HT, int WT, bool VEC, int G, int TH, int C>
__global__ __launch_bounds__(TH) void rms_norm_backward_kernel(NormGradArgs a) {
    constexpr int NW = TH / WAVE, GROUPS = TH / G;
    constexpr bool BLOCK = G > WAVE;  // (groups of waves: all of a block's take their rows together)
    __shared__ float s_sum[2][2][NW];
    const int tid = int(threadIdx.x), H = a.H;
    const int group = GROUPS == 1 ? 0 : BLOCK ? __builtin_amdgcn_readfirstlane(tid / G) : tid / G, li = tid - group * G;
    // (with the next row on its way a block of 1024 spills 57 to 113 registers: 512 fp32 rows of 16384 70 us for 45)
    constexpr bool SHORT = G == 16, AHEAD = G < 1024;
    struct Row {
        Part<HT, VEC, SHORT> h[C], res[C];
        Part<DT, VEC, SHORT> d[C];
    } next;
    Part<WT, VEC, SHORT> wp[C];
    float dw[C][8];
    auto load = [&](int64_t t) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if (j >= H) continue;
            next.h[c].load(a.h, t * a.ldh, j, H);
            next.d[c].load(a.dy, t * a.lddy, j, H);
            if (a.dres) next.res[c].load(a.dres, t * a.lddr, j, H);
        }
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int j = (li + c * G) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[c][e] = 0.f;
        if (j < H) {
            wp[c].load(a.w, 0, j, H);
            wp[c].settle(j, H);
        }
    }
    const int64_t t0 = int64_t(blockIdx.x) * GROUPS + group, step = int64_t(gridDim.x) * GROUPS;
    if (AHEAD && t0 < a.T) load(t0);
    int p = 0;
    for (int64_t t = t0; t - (BLOCK ? group : 0) < a.T; t += step, p ^= 1) {
        const bool live = !BLOCK || GROUPS == 1 || t < a.T;
        if (!AHEAD && t < a.T) load(t);
        const Row row = next;
        if (AHEAD && t + step < a.T) load(t + step);
        float h[C][8], g[C][8], sum = 0.f, dot = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if (j >= H) continue;
            float w[8];
            row.h[c].values(h[c], j, H);
            row.d[c].values(g[c], j, H);
            wp[c].w.values(w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum = __builtin_fmaf(h[c][e], h[c][e], sum);
                dot = __builtin_fmaf(g[c][e] * w[e], h[c][e], dot);
            }
        }
#pragma unroll
        for (int o = (BLOCK ? WAVE : G) / 2; o >= 1; o >>= 1) {
            sum += __shfl_xor(sum, o);
            dot += __shfl_xor(dot, o);
        }
        if constexpr (BLOCK) {
            if (tid % WAVE == 0) {
                s_sum[p][0][tid / WAVE] = sum;
                s_sum[p][1][tid / WAVE] = dot;
            }
            __syncthreads();  // (one per row: the next row's sums go to the other pair of lists)
            sum = dot = 0.f;
#pragma unroll
            for (int i = 0; i < G / WAVE; ++i) {
                sum += s_sum[p][0][group * (G / WAVE) + i];
                dot += s_sum[p][1][group * (G / WAVE) + i];
            }
        }
        const float r = 1.f / sqrtf(sum / float(H) + a.eps), k = r * r * (dot / float(H));
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
            if (j >= H || !live) continue;
            float o[8], w[8];
            wp[c].w.values(w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                o[e] = r * (g[c][e] * w[e] - h[c][e] * k);
                dw[c][e] = __builtin_fmaf(g[c][e], h[c][e] * r, dw[c][e]);
            }
            if (a.dres) {
                float res[8];
                row.res[c].values(res, j, H);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += res[e];
            }
            part_store<HT == 2 ? GRAD_F16 : HT, VEC>(a.dx, t * a.lddx, j, H, o);
        }
    }
    if (!a.dw) return;
    float *part = a.part + int64_t(blockIdx.x) * H;
    if constexpr (G == TH) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int j = (li + c * G) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (j + e < H) part[j + e] = dw[c][e];
        }
    } else {
        constexpr int SETS = BLOCK ? GROUPS : NW;  // (a wave's groups first)
        __shared__ float s_dw[SETS][C * G * 8];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int o = G; o < WAVE; o <<= 1) dw[c][e] += __shfl_xor(dw[c][e], o);
                if (BLOCK || tid % WAVE < G) s_dw[tid / (BLOCK ? G : WAVE)][(li + c * G) * 8 + e] = dw[c][e];
            }
        __syncthreads();
        for (int j = tid; j < H; j += TH) {
            float sum = s_dw[0][j];
#pragma unroll
            for (int i = 1; i < SETS; ++i) sum += s_dw[i][j];
            part[j] = sum;
        }
    }
}

// dw[j] = the blocks' parts in order: 64 columns a block, each of 16 waves
// adding a run of the parts.
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float *__restrict__ part, int parts, int H,
                                                           float *__restrict__ dw) {
    __shared__ float s[16][WAVE];
    const int lane = int(threadIdx.x) % WAVE, wave = int(threadIdx.x) / WAVE;
    const int64_t j = int64_t(blockIdx.x) * WAVE + lane;
    const int per = (parts + 15) / 16, b0 = wave * per, b1 = min(parts, b0 + per);
    float sum = 0.f;
    if (j < H) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) sum += part[int64_t(b) * H + j];
    }
    s[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && j < H) {
#pragma unroll
        for (int i = 1; i < 16; ++i) sum += s[i][lane];
        dw[j] = sum;
    }
}

// Blocks of the gradients' launch, of T groups: as many parts of dw are written
// and read (4096 rows of 4096 in 512 parts 32.5 us for 29.6, 1024 of 16384 52 for
// 37). Two blocks a CU only where waves take rows of up to 2048, 32 KB of LDS a block.
static int norm_grad_blocks(int T, int H) { return std::min(T, H <= 1024 || H > 2048 ? 256 : 512); }

size_t rms_norm_backward_workspace_bytes(int T, int H) { return size_t(norm_grad_blocks(T, H)) * size_t(H) * 4; }

template <int DT, int HT, int WT>
static void launch_norm_grad(const NormGradArgs &a, hipStream_t s) {
    int blocks = 0;
    auto run = [&](auto vec, auto g, auto th, auto c) {
        constexpr int G = decltype(g)::value, TH = decltype(th)::value;
        blocks = norm_grad_blocks((a.T + TH / G - 1) / (TH / G), a.H);
        rms_norm_backward_kernel<DT, HT, WT, decltype(vec)::value, G, TH, decltype(c)::value>
            <<<unsigned(blocks), TH, 0, s>>>(a);
    };
    // Short rows by parts of a wave: no barrier, and every thread has work (16.8 million elements in bf16, a block or a
    // wave a row, and as here: rows of 64 545 us and 42, of 256 140 and 22, of 1024 49 and 22). Rows of 16 bits by as few
    // waves as registers allow: of 2048 29 us in blocks, 24 in waves; of 2560 32 and 26; of 16384 37 and 34. fp32 would
    // spill so, and does (13 to 51 registers) above 8192. How the rows lie is not asked: their bits would depend on it.
    auto by_length = [&](auto vec) {
        constexpr bool HALF = HT != 0;
        if (a.H <= 128) return run(vec, Int<16>{}, Int<512>{}, Int<1>{});
        if (a.H <= 256) return run(vec, Int<16>{}, Int<512>{}, Int<2>{});
        if (a.H <= 512) return run(vec, Int<64>{}, Int<512>{}, Int<1>{});
        if (a.H <= 1024) return run(vec, Int<64>{}, Int<512>{}, Int<2>{});
        if constexpr (HALF) {
            if (a.H <= 2048) return run(vec, Int<64>{}, Int<256>{}, Int<4>{});
            if (a.H <= 128 * 24) return run(vec, Int<128>{}, Int<512>{}, Int<3>{});
        }
        if (a.H <= 2048) return run(vec, Int<128>{}, Int<512>{}, Int<2>{});
        if (a.H <= 4096) return run(vec, Int<256>{}, Int<512>{}, Int<2>{});
        if (a.H <= 8192) return run(vec, Int<512>{}, Int<512>{}, Int<2>{});
        if constexpr (HALF) return run(vec, Int<512>{}, Int<512>{}, Int<4>{});
        else return run(vec, Int<1024>{}, Int<1024>{}, Int<2>{});
    };
    const int64_t one = a.T == 1 ? 0 : 1;  // (a single row's stride does not matter)
    if (a.H % 8 == 0 && rows_aligned(a.dy, DT, one * a.lddy, 8) && rows_aligned(a.h, HT, one * a.ldh, 8) &&
        rows_aligned(a.w, WT, 0, 8) && rows_aligned(a.dres, HT, one * a.lddr, 8) &&
        rows_aligned(a.dx, HT, one * a.lddx, 8))
        by_length(std::true_type{});
    else
        by_length(std::false_type{});
    if (a.dw) rms_norm_dw_kernel<<<unsigned((a.H + WAVE - 1) / WAVE), 1024, 0, s>>>(a.part, blocks, a.H, a.dw);
}

void launch_rms_norm_backward(const NormGradArgs &a, hipStream_t s) {
    by_type(a.dy_type, [&](auto dt) {
        auto run = [&](auto ht, auto wt) {
            launch_norm_grad<decltype(dt)::value, decltype(ht)::value, decltype(wt)::value>(a, s);
        };
        auto by_row = [&](auto wt) {
            if (a.h_type == 0) run(Int<0>{}, wt);
            else run(dt, wt);
        };
        if (a.w_type == 0) by_row(Int<0>{});
        else by_row(dt);
    });
}

}  // namespace qwq4
