// Tokens sorted by expert and back: the slots of given expert choices, the
// rows in slot order, and the weighted rows back at their tokens, with the
// gradients.
//
//   slot(t, i) = place of the choice e[t][i] among all, by (expert, t, i)
//   xs[slot(t, i)] = x[t]                                    permute
//   out[t] = sum_i w[t][i] yp[slot(t, i)]                    unpermute
//   dyp[slot(t, i)] = w[t][i] dout[t]                        its gradients
//   dw[t][i] = <yp[slot(t, i)], dout[t]>
// The gradient of permute is unpermute with all weights 1 (and fp16 that
// overflows instead of saturating). Choices outside
// 0 .. E - 1 (an expert that another rank holds, in the engine's
// expert-parallel layout, src/core/shard.hpp:34) have no slot (-1) and add
// nothing. No atomics on values: every sum has a fixed order.
#include <algorithm>
#include <type_traits>

#include "q4_kernels.hpp"
#include "row_io.cuh"

namespace qwq4 {

// ------------------------------------------------------------ sort
// Exclusive scans of three values per thread over the 1024-thread block: v
// becomes the sums before the thread's, total the sums of all.
__device__ __forceinline__ void rows_scan_excl(int (&v)[3], int (*s_w)[16], int (&total)[3]) {
    const int lane = int(threadIdx.x) % WAVE, wave = int(threadIdx.x) / WAVE;
    int inc[3];
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        inc[c] = v[c];
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) {
            const int u = __shfl_up(inc[c], o);
            if (lane >= o) inc[c] += u;
        }
        if (lane == WAVE - 1) s_w[c][wave] = inc[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 3; ++c) {
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? s_w[c][w] : 0;
            all += s_w[c][w];
        }
        total[c] = all;
        v[c] = before + inc[c] - v[c];
    }
}

// Every block counts the choices of all pairs and of the pairs before its own
// (LDS atomics on counters: their order does not matter), scans the totals
// over the experts, and gives its pairs their slots, 64 pairs a turn: a
// pair's rank among the turn's pairs of the same expert is a popcount below
// its bit in the lanes that hold that expert. No block reads what another
// writes, so one launch needs no hand-off.
__global__ __launch_bounds__(1024) void sort_kernel(SortArgs a, int per) {
    __shared__ int s_rest[1024], s_at[1024], s_w[3][16];
    const int tid = int(threadIdx.x), E = a.E, P = a.T * a.topk;
    const int p0 = int(blockIdx.x) * per, p1 = min(p0 + per, P);
    s_rest[tid] = 0;
    s_at[tid] = 0;
    __syncthreads();
    // the pairs before the block's own (s_at) and the others (s_rest), eight
    // choices requested per thread before their counts
    for (int i0 = tid; i0 < P; i0 += 8 * 1024) {
        int e[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) e[u] = a.top_e[min(i0 + u * 1024, P - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * 1024;
            if (i < P && e[u] >= 0 && e[u] < E) atomicAdd(i < p0 ? &s_at[e[u]] : &s_rest[e[u]], 1);
        }
    }
    __syncthreads();
    const int c = s_at[tid] + s_rest[tid];
    const int ntl = a.tile_m != 0 ? tile_count(c, a.tile_m) : 0;
    int at[3] = {c, c > 0, ntl}, all[3];  // slots, experts with any, list entries
    rows_scan_excl(at, s_w, all);
    const int off = at[0], total = all[0];
    s_at[tid] += off;
    if (blockIdx.x == 0) {
        if (tid < E) {
            a.offsets[tid] = off;
            a.counts[tid] = c;
            if (c > 0) a.active[at[1]] = tid;
            for (int j = 0, m0 = 0; j < ntl; ++j, m0 += tile_rows(c - m0, a.tile_m)) {
                a.tile_e[at[2] + j] = tid;
                a.tile_m0[at[2] + j] = m0;
            }
        }
        if (tid == 0) {
            a.offsets[E] = total;
            *a.n_active = all[1];
            if (a.tile_m != 0) *a.n_tiles = all[2];
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

// A thread's V columns of one token: up to 8 selections' rows requested
// together, then added in selection order. Bound by memory: 4096 tokens of 8
// choices, 4096 bf16 wide, take 63 us (4.8 TB/s; a large copy reaches 5.2).
template <int YT, int OT, int V>
__global__ __launch_bounds__(256) void unpermute_kernel(const void *__restrict__ yp, int64_t ldy,
                                                        const int32_t *__restrict__ tok_slot,
                                                        const float *__restrict__ tok_w, int T, int topk, int H,
                                                        void *__restrict__ out, int64_t ldo, int cols) {
    const int t = int(blockIdx.x) / cols, P = T * topk;
    const int32_t *slots = tok_slot + int64_t(t) * topk;
    const float *weights = tok_w ? tok_w + int64_t(t) * topk : nullptr;
    for (int j = (int(blockIdx.x) % cols * int(blockDim.x) + int(threadIdx.x)) * V; j < H;
         j += cols * int(blockDim.x) * V) {
        float sum[V];
#pragma unroll
        for (int c = 0; c < V; ++c) sum[c] = 0.f;
        for (int i0 = 0; i0 < topk; i0 += 8) {
            float v[8][V], w[8];
            bool kept[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int i = min(i0 + u, topk - 1), slot = slots[i];
                kept[u] = i0 + u < topk && slot >= 0 && slot < P;
                w[u] = weights ? weights[i] : 1.f;
                if (kept[u]) row_load<YT, V>(yp, slot * ldy + j, v[u]);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (kept[u]) {
#pragma unroll
                    for (int c = 0; c < V; ++c) sum[c] = __builtin_fmaf(w[u], v[u][c], sum[c]);
                }
            }
        }
        row_store<OT, V>(out, t * ldo + j, sum);
    }
}

void launch_unpermute(const void *yp, int yp_type, int64_t ldy, const int32_t *tok_slot, const float *tok_w, int T,
                      int topk, int H, void *out, int out_type, int64_t ldo, bool saturate, hipStream_t s) {
    auto run = [&](auto yt, auto ot, auto v) {
        constexpr int V = decltype(v)::value;
        const int items = (H + V - 1) / V, threads = items > 128 ? 256 : items > 64 ? 128 : 64;
        // (a grid holds less than 2^32 threads: with very many tokens a block takes more of a row)
        const int cols = std::max(1, std::min((items + threads - 1) / threads, (1 << 23) / T));
        unpermute_kernel<decltype(yt)::value, decltype(ot)::value, V><<<unsigned(T) * unsigned(cols), threads, 0, s>>>(
            yp, ldy, tok_slot, tok_w, T, topk, H, out, ldo, cols);
    };
    by_type(yp_type, [&](auto yt) {
        auto store_as = [&](auto ot) {
            constexpr int V = decltype(yt)::value == 0 ? 4 : 8;
            if (H % V == 0 && rows_aligned(yp, yp_type, ldy, V) && rows_aligned(out, out_type, ldo, V))
                run(yt, ot, Int<V>{});
            else run(yt, ot, Int<1>{});
        };
        if (out_type == 2 && !saturate) store_as(Int<GRAD_F16>{});
        else by_type(out_type, store_as);
    });
}

// One choice by one wave; each lane has 4 vectors' worth of both rows on
// their way.
template <int DT, int YT, int V>
__device__ __forceinline__ void choice_backward(const UnpermuteGradArgs &a, int t, int i) {
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t at = int64_t(t) * a.topk + i, d0 = t * a.ldd;
    const int slot = a.tok_slot[at];
    const float w = a.tok_w ? a.tok_w[at] : 1.f;
    float sum = 0.f;
    if (slot >= 0 && slot < a.T * a.topk) {
        const int64_t y0 = slot * a.ldy, g0 = slot * a.lddy;
        for (int j0 = lane * V; j0 < a.H; j0 += 4 * WAVE * V) {
            float d[4][V], y[4][V];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * WAVE * V;
                if (j < a.H) {
                    row_load<DT, V>(a.dout, d0 + j, d[u]);
                    if (a.dw) row_load<YT, V>(a.yp, y0 + j, y[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * WAVE * V;
                if (j >= a.H) continue;
                if (a.dw) {
#pragma unroll
                    for (int c = 0; c < V; ++c) sum = __builtin_fmaf(y[u][c], d[u][c], sum);
                }
                if (a.dyp) {
                    float g[V];
#pragma unroll
                    for (int c = 0; c < V; ++c) g[c] = w * d[u][c];
                    row_store<YT == 2 ? GRAD_F16 : YT, V>(a.dyp, g0 + j, g);
                }
            }
        }
    }
    if (!a.dw) return;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) a.dw[at] = sum;
}

// A wave per choice, a block per token (up to 16 choices at once): the
// token's dout row is read by all of them from the nearest cache. Bound by
// memory: 4096 tokens of 8 choices, 4096 bf16 wide, take 122 us (4.7 TB/s of
// what they read and write; a large copy reaches 5.2).
template <int DT, int YT, int V>
__global__ __launch_bounds__(1024) void unpermute_backward_kernel(UnpermuteGradArgs a) {
    for (int t = int(blockIdx.x); t < a.T; t += int(gridDim.x))
        for (int i = int(threadIdx.x) / WAVE; i < a.topk; i += int(blockDim.x) / WAVE)
            choice_backward<DT, YT, V>(a, t, i);
}

void launch_unpermute_backward(const UnpermuteGradArgs &a, hipStream_t s) {
    const unsigned threads = unsigned(WAVE) * unsigned(a.topk < 16 ? a.topk : 16);
    const unsigned blocks = unsigned(std::min(a.T, 1 << 21));  // (a grid holds less than 2^32 threads)
    by_type(a.dout_type, [&](auto dt) {
        by_type(a.yp_type, [&](auto yt) {
            constexpr int DT = decltype(dt)::value, YT = decltype(yt)::value, V = YT == 0 ? 4 : 8;
            if (a.H % V == 0 && rows_aligned(a.dout, DT, a.ldd, V) && (!a.dw || rows_aligned(a.yp, YT, a.ldy, V)) &&
                rows_aligned(a.dyp, YT, a.lddy, V))
                unpermute_backward_kernel<DT, YT, V><<<blocks, threads, 0, s>>>(a);
            else unpermute_backward_kernel<DT, YT, 1><<<blocks, threads, 0, s>>>(a);
        });
    });
}

}  // namespace qwq4
