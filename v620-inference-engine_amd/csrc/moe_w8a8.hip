// Routed experts in W8A8: int8 weights with a scale per output row, rows
// quantised with a scale per token (w8a8.hip), for any batch. The role of
// qw_moe_experts_w4a8 (the engine's int8-activation experts,
// src/kernels/moe_w4a8.hip:13-215) for checkpoints quantised to 8 bits, where
// the sums run over all of K in whole numbers and are scaled once.
//
//   h[p]  = fp16(silu(g) * u),  g, u = W8A8 products of x[pair_tok[p]]
//   yp[p] = W8A8 product of h[p], quantised per slot
#include <type_traits>

#include "q4_kernels.hpp"
#include "w8a8_core.cuh"

namespace qwq4 {

constexpr int MW8_TILE_M = -32;  // the routing's mixed tiles of 32 to 160 slots

int moe_w8a8_tile_m() { return MW8_TILE_M; }

// A list entry: expert e, its slots base .. base + M - 1.
struct MW8Entry {
    int e, base, M;
};
__device__ __forceinline__ bool mw8_entry(const MoeW8A8Args &a, int tile, MW8Entry &t) {
    if (tile >= *a.n_tiles) return false;
    t.e = a.tile_e[tile];
    const int m0 = a.tile_m0[tile], rem = a.offsets[t.e + 1] - a.offsets[t.e] - m0;
    t.base = a.offsets[t.e] + m0;
    t.M = min(tile_rows(rem, MW8_TILE_M), rem);
    return true;
}

// gate/up: of every 64 weight rows of the tile the first 32 are gate rows, the
// others the up rows of the same 32 columns of h: a wave holds both.
template <class S>
__global__ __launch_bounds__(S::THREADS) void moe_gate_up_w8a8_kernel(MoeW8A8Args a) {
    static_assert(S::NT % 2 == 0, "a wave holds gate and up of a column");
    const int nt = (a.F + S::BN / 2 - 1) / (S::BN / 2);
    MW8Entry t;
    if (!mw8_entry(a, int(blockIdx.x) / nt, t)) return;
    const int j0 = int(blockIdx.x) % nt * (S::BN / 2);
    const int64_t eF = int64_t(t.e) * a.F;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) {
        const int r = S::load_row(j);
        bp[j] = ((r / 32) % 2 ? a.uw : a.gw) + (eF + min(j0 + r / 64 * 32 + r % 32, a.F - 1)) * a.H;
    }
    const int32_t *pt = a.pair_tok + t.base;
    for (int m0 = 0; m0 < t.M; m0 += S::BM) {
        if (m0 > 0) __syncthreads();  // the tile before is read
#pragma unroll
        for (int j = 0; j < S::AJ; ++j) ap[j] = a.qx + int64_t(pt[min(m0 + S::load_row(j), t.M - 1)]) * a.H;
        i32x16 acc[S::MT][S::NT];
        w8_clear<S>(acc);
        unsigned char *spare;
        if (!w8_tile<S, 1>(ap, bp, a.H, acc, spare)) continue;
        const int m_first = m0 + S::m_base(), col = j0 + S::n_base() / 2, l32 = int(threadIdx.x) % 32;
        float sx[S::MT], sg[S::NT / 2][16], su[S::NT / 2][16];
#pragma unroll
        for (int i = 0; i < S::MT; ++i) sx[i] = a.sx[pt[min(m_first + 32 * i + l32, t.M - 1)]];
#pragma unroll
        for (int c = 0; c < S::NT / 2; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t n = eF + min(col + 32 * c + S::n_of(r), a.F - 1);
                sg[c][r] = a.gs[n];
                su[c][r] = a.us[n];
            }
        auto value = [&](int i, int c, int r) {
            const float g = w8_value(acc[i][2 * c][r], sg[c][r], sx[i]);
            return silu_ref(g) * w8_value(acc[i][2 * c + 1][r], su[c][r], sx[i]);
        };
        w8_output<S, S::NT / 2>(spare, a.h, 2, a.F - col, value, [&](int m) -> int64_t {
            return m_first + m < t.M ? int64_t(t.base + m_first + m) * a.F + col : -1;
        });
    }
}

template <class S>
__global__ __launch_bounds__(S::THREADS) void moe_down_w8a8_kernel(MoeW8A8Args a) {
    const int nt = (a.H + S::BN - 1) / S::BN;
    MW8Entry t;
    if (!mw8_entry(a, int(blockIdx.x) / nt, t)) return;
    const int n0 = int(blockIdx.x) % nt * S::BN;
    const int64_t eH = int64_t(t.e) * a.H;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) bp[j] = a.dw + (eH + min(n0 + S::load_row(j), a.H - 1)) * a.F;
    for (int m0 = 0; m0 < t.M; m0 += S::BM) {
        if (m0 > 0) __syncthreads();  // the tile before is read
#pragma unroll
        for (int j = 0; j < S::AJ; ++j) ap[j] = a.qh + int64_t(t.base + min(m0 + S::load_row(j), t.M - 1)) * a.F;
        i32x16 acc[S::MT][S::NT];
        w8_clear<S>(acc);
        unsigned char *spare;
        if (!w8_tile<S, 2>(ap, bp, a.F, acc, spare)) continue;
        const int m_first = m0 + S::m_base(), n_first = n0 + S::n_base(), l32 = int(threadIdx.x) % 32;
        float sx[S::MT], sw[S::NT][16];
#pragma unroll
        for (int i = 0; i < S::MT; ++i) sx[i] = a.sh[t.base + min(m_first + 32 * i + l32, t.M - 1)];
#pragma unroll
        for (int j = 0; j < S::NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) sw[j][r] = a.ds[eH + min(n_first + 32 * j + S::n_of(r), a.H - 1)];
        auto value = [&](int i, int j, int r) { return w8_value(acc[i][j][r], sw[j][r], sx[i]); };
        w8_output<S, S::NT>(spare, a.yp, a.yp_type, a.H - n_first, value, [&](int m) -> int64_t {
            return m_first + m < t.M ? int64_t(t.base + m_first + m) * a.H + n_first : -1;
        });
    }
}

static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

size_t moe_w8a8_workspace_bytes(int T, int topk, int H, int F) {
    const size_t P = size_t(T) * size_t(topk);
    return up256(size_t(T) * size_t(H)) + up256(size_t(T) * 4) + up256(P * size_t(F)) + up256(P * 4);
}

// x quantised, gate/up, h quantised, down: four launches on one stream.
void launch_moe_w8a8(MoeW8A8Args a, const void *x, int x_type, int T, int topk, void *ws, hipStream_t s) {
    const size_t P = size_t(T) * size_t(topk);
    int8_t *w = static_cast<int8_t *>(ws);
    int8_t *qx = w;
    w += up256(size_t(T) * size_t(a.H));
    float *sx = reinterpret_cast<float *>(w);
    w += up256(size_t(T) * 4);
    int8_t *qh = w;
    w += up256(P * size_t(a.F));
    float *sh = reinterpret_cast<float *>(w);
    a.qx = qx;
    a.sx = sx;
    a.qh = qh;
    a.sh = sh;
    const unsigned tiles = unsigned(P / size_t(-MW8_TILE_M)) + unsigned(a.E);
    launch_quant_tokens(x, x_type, a.H, T, a.H, qx, a.H, sx, s);
    using S = W8Shape<64, 128, 2, 2, 1, 128, 2>;
    moe_gate_up_w8a8_kernel<S><<<tiles * unsigned((a.F + S::BN / 2 - 1) / (S::BN / 2)), S::THREADS, 0, s>>>(a);
    launch_quant_tokens(a.h, 2, a.F, int(P), a.F, qh, a.F, sh, s);
    moe_down_w8a8_kernel<S><<<tiles * unsigned((a.H + S::BN - 1) / S::BN), S::THREADS, 0, s>>>(a);
}

}  // namespace qwq4
