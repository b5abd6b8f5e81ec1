// Tokens sorted by expert and back: the slots of given expert choices, the
// rows in slot order, and the weighted rows back at their tokens, with the
// gradients.
//
//   slot(t, i) = place of the choice e[t][i] among all, by (expert, t, i)
//   xs[slot(t, i)] = x[t]                                    permute
//   out[t] = sum_i w[t][i] yp[slot(t, i)]                    unpermute
//   dyp[slot(t, i)] = w[t][i] dout[t]                        its gradients
//   dw[t][i] = <yp[slot(t, i)], dout[t]>
// The gradient of permute is unpermute with all weights 1. Choices outside
// 0 .. E - 1 (an expert that another rank holds, in the engine's
// expert-parallel layout, src/core/shard.hpp:34) have no slot (-1) and add
// nothing. No atomics on values: every sum has a fixed order.
#include <algorithm>
#include <type_traits>

#include "q4_common.cuh"
#include "q4_kernels.hpp"

namespace qwq4 {

// ------------------------------------------------------------ sort
// Exclusive scan over the values of the first E threads (1024-thread block);
// the total is returned in every thread.
__device__ __forceinline__ int rows_scan_excl(int v, int *s_w, int &total) {
    const int lane = int(threadIdx.x) % WAVE, wave = int(threadIdx.x) / WAVE;
    int inc = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int u = __shfl_up(inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == WAVE - 1) s_w[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < int(blockDim.x) / WAVE; ++w) {
        before += w < wave ? s_w[w] : 0;
        all += s_w[w];
    }
    __syncthreads();
    total = all;
    return before + inc - v;
}

// Every block counts the choices of all pairs and of the pairs before its own
// (LDS atomics on counters: their order does not matter), scans the totals
// over the experts, and gives its pairs their slots, 64 pairs a turn: a
// pair's rank among the turn's pairs of the same expert is a popcount below
// its bit in the lanes that hold that expert. No block reads what another
// writes, so one launch needs no hand-off.
__global__ __launch_bounds__(1024) void sort_kernel(SortArgs a, int per) {
    __shared__ int s_all[1024], s_at[1024], s_w[16];
    const int tid = int(threadIdx.x), E = a.E, P = a.T * a.topk;
    const int p0 = int(blockIdx.x) * per, p1 = min(p0 + per, P);
    s_all[tid] = 0;
    s_at[tid] = 0;
    __syncthreads();
    for (int i = tid; i < P; i += 1024) {
        const int e = a.top_e[i];
        if (e >= 0 && e < E) {
            atomicAdd(&s_all[e], 1);
            if (i < p0) atomicAdd(&s_at[e], 1);
        }
    }
    __syncthreads();
    const int c = s_all[tid];
    int total;
    const int off = rows_scan_excl(c, s_w, total);
    s_at[tid] += off;
    if (blockIdx.x == 0) {
        int n_act, n_tiles = 0;
        const int act = rows_scan_excl(c > 0, s_w, n_act);
        const int ntl = a.tile_m != 0 ? tile_count(c, a.tile_m) : 0;
        const int tile0 = a.tile_m != 0 ? rows_scan_excl(ntl, s_w, n_tiles) : 0;
        if (tid < E) {
            a.offsets[tid] = off;
            a.counts[tid] = c;
            if (c > 0) a.active[act] = tid;
            for (int j = 0, m0 = 0; j < ntl; ++j, m0 += tile_rows(c - m0, a.tile_m)) {
                a.tile_e[tile0 + j] = tid;
                a.tile_m0[tile0 + j] = m0;
            }
        }
        if (tid == 0) {
            a.offsets[E] = total;
            *a.n_active = n_act;
            if (a.tile_m != 0) *a.n_tiles = n_tiles;
        }
        for (int i = total + tid; i < P; i += 1024) a.pair_tok[i] = -1;
    }
    __syncthreads();
    if (tid >= WAVE) return;
    for (int i0 = p0; i0 < p1; i0 += WAVE) {
        const int i = i0 + tid;
        const int e = i < p1 ? a.top_e[i] : -1;
        const bool kept = e >= 0 && e < E;
        unsigned long long same = __ballot(kept);
        for (int b = 0; b < 10; ++b) {
            const unsigned long long m = __ballot((e >> b) & 1);
            same &= (e >> b) & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << tid) - 1ull));
        const int slot = kept ? s_at[e] + rank : -1;
        if (i < p1) a.tok_slot[i] = slot;
        if (kept) a.pair_tok[slot] = i / a.topk;
        __builtin_amdgcn_wave_barrier();
        if (kept && rank == 0) s_at[e] += __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

void launch_sort(const SortArgs &a, hipStream_t s) {
    const int P = a.T * a.topk;
    const int blocks = std::min(256, (P + WAVE - 1) / WAVE);
    const int per = ((P + blocks - 1) / blocks + WAVE - 1) / WAVE * WAVE;
    sort_kernel<<<unsigned((P + per - 1) / per), 1024, 0, s>>>(a, per);
}

// ------------------------------------------------------------ rows
// U: what a thread moves at once (the row length and strides are in units of U).
template <class U>
__global__ __launch_bounds__(256) void permute_kernel(const U *__restrict__ x, int64_t ldx, int T, int topk, int n,
                                                      const int32_t *__restrict__ tok_slot, U *__restrict__ xs,
                                                      int64_t ldxs) {
    const int t = int(blockIdx.x), P = T * topk;
    for (int j = int(threadIdx.x); j < n; j += 256) {
        const U v = x[t * ldx + j];
        for (int i = 0; i < topk; ++i) {
            const int slot = tok_slot[int64_t(t) * topk + i];
            if (slot >= 0 && slot < P) xs[slot * ldxs + j] = v;
        }
    }
}

void launch_permute(const void *x, int64_t ldx, int elem_bytes, int T, int topk, int H, const int32_t *tok_slot,
                    void *xs, int64_t ldxs, hipStream_t s) {
    const int64_t b = int64_t(H) * elem_bytes, sx = ldx * elem_bytes, ss = ldxs * elem_bytes;
    auto run = [&](auto u) {
        using U = decltype(u);
        constexpr int64_t z = sizeof(U);
        permute_kernel<U><<<unsigned(T), 256, 0, s>>>(static_cast<const U *>(x), sx / z, T, topk, int(b / z), tok_slot,
                                                      static_cast<U *>(xs), ss / z);
    };
    const uint64_t all = uint64_t(b) | uint64_t(sx) | uint64_t(ss) | reinterpret_cast<uintptr_t>(x) |
                         reinterpret_cast<uintptr_t>(xs);
    if (all % 16 == 0) run(uint4{});
    else if (all % 4 == 0) run(uint32_t{});
    else if (all % 2 == 0) run(uint16_t{});
    else run(uint8_t{});
}

template <int TY>
__device__ __forceinline__ float row_load(const void *x, int64_t i) {
    if constexpr (TY == 0) return static_cast<const float *>(x)[i];
    else if constexpr (TY == 1) return bf16_bits_to_f32(static_cast<const uint16_t *>(x)[i]);
    else return f16_bits_to_f32(static_cast<const uint16_t *>(x)[i]);
}
template <int TY>
__device__ __forceinline__ void row_store(void *y, int64_t i, float v) {
    if constexpr (TY == 0) static_cast<float *>(y)[i] = v;
    else if constexpr (TY == 1) static_cast<uint16_t *>(y)[i] = f32_to_bf16_rne(v);
    else static_cast<_Float16 *>(y)[i] = f32_to_f16_satfinite(v);
}

template <int YT, int OT>
__global__ __launch_bounds__(256) void unpermute_kernel(const void *__restrict__ yp, int64_t ldy,
                                                        const int32_t *__restrict__ tok_slot,
                                                        const float *__restrict__ tok_w, int T, int topk, int H,
                                                        void *__restrict__ out, int64_t ldo) {
    const int t = int(blockIdx.x), P = T * topk;
    for (int j = int(threadIdx.x); j < H; j += 256) {
        float sum = 0.f;
        for (int i = 0; i < topk; ++i) {
            const int64_t at = int64_t(t) * topk + i;
            const int slot = tok_slot[at];
            if (slot >= 0 && slot < P) sum = __builtin_fmaf(tok_w ? tok_w[at] : 1.f, row_load<YT>(yp, slot * ldy + j), sum);
        }
        row_store<OT>(out, t * ldo + j, sum);
    }
}

void launch_unpermute(const void *yp, int yp_type, int64_t ldy, const int32_t *tok_slot, const float *tok_w, int T,
                      int topk, int H, void *out, int out_type, int64_t ldo, hipStream_t s) {
    auto run = [&](auto yt, auto ot) {
        unpermute_kernel<decltype(yt)::value, decltype(ot)::value><<<unsigned(T), 256, 0, s>>>(
            yp, ldy, tok_slot, tok_w, T, topk, H, out, ldo);
    };
    auto by_out = [&](auto yt) {
        if (out_type == 0) run(yt, std::integral_constant<int, 0>{});
        else if (out_type == 1) run(yt, std::integral_constant<int, 1>{});
        else run(yt, std::integral_constant<int, 2>{});
    };
    if (yp_type == 0) by_out(std::integral_constant<int, 0>{});
    else if (yp_type == 1) by_out(std::integral_constant<int, 1>{});
    else by_out(std::integral_constant<int, 2>{});
}

// One wave per choice (t, i).
template <int DT, int YT>
__global__ __launch_bounds__(256) void unpermute_backward_kernel(UnpermuteGradArgs a) {
    const int P = a.T * a.topk, p = int(blockIdx.x) * 4 + int(threadIdx.x) / WAVE, lane = int(threadIdx.x) % WAVE;
    if (p >= P) return;
    const int t = p / a.topk, slot = a.tok_slot[p];
    const bool kept = slot >= 0 && slot < P;
    const float w = a.tok_w ? a.tok_w[p] : 1.f;
    float sum = 0.f;
    for (int j = lane; kept && j < a.H; j += WAVE) {
        const float d = row_load<DT>(a.dout, t * a.ldd + j);
        if (a.dw) sum = __builtin_fmaf(row_load<YT>(a.yp, slot * a.ldy + j), d, sum);
        if (a.dyp) row_store<YT>(a.dyp, slot * a.lddy + j, w * d);
    }
    if (!a.dw) return;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) a.dw[p] = sum;
}

void launch_unpermute_backward(const UnpermuteGradArgs &a, hipStream_t s) {
    const unsigned blocks = unsigned((int64_t(a.T) * a.topk + 3) / 4);
    auto run = [&](auto dt, auto yt) {
        unpermute_backward_kernel<decltype(dt)::value, decltype(yt)::value><<<blocks, 256, 0, s>>>(a);
    };
    auto by_y = [&](auto dt) {
        if (a.yp_type == 0) run(dt, std::integral_constant<int, 0>{});
        else if (a.yp_type == 1) run(dt, std::integral_constant<int, 1>{});
        else run(dt, std::integral_constant<int, 2>{});
    };
    if (a.dout_type == 0) by_y(std::integral_constant<int, 0>{});
    else if (a.dout_type == 1) by_y(std::integral_constant<int, 1>{});
    else by_y(std::integral_constant<int, 2>{});
}

}  // namespace qwq4
