// Routed experts in W8A8: int8 weights with a scale per output row, rows
// quantised with a scale per token (w8a8.hip), for any batch. The role of
// qw_moe_experts_w4a8 (the engine's int8-activation experts,
// src/kernels/moe_w4a8.hip:13-215) for checkpoints quantised to 8 bits, where
// the sums run over all of K in whole numbers and are scaled once.
//
//   h[p]  = fp16(silu(g) * u),  g, u = W8A8 products of x[pair_tok[p]]
//   yp[p] = W8A8 product of h[p], quantised per slot
//
// Work is the routing's tile list (an entry: an expert and 32 to 160 of its
// slots) times blocks of weight rows. A block runs its entry in tiles of 128 or
// 64 slots on the int8 MFMA (w8a8_core.cuh); for few tokens (up to 16, or 4 with
// small experts) it streams the weights past the slots' rows in LDS
// (w8a8_gemv.cuh). The sums being whole numbers, both give a slot the same bits.
#include <algorithm>
#include <type_traits>

#include "q4_kernels.hpp"
#include "w8a8_core.cuh"
#include "w8a8_gemv.cuh"

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

// ------------------------------------------------------------ tiles
// Entry and block of weight rows of block b, nt of them per entry: an entry's
// blocks go to one XCD (blocks go to the 8 in turn), whose L2 then holds the
// entry's rows once.
__device__ __forceinline__ int mw8_place(int b, int nt, int &col) {
    col = b / 8 % nt;
    return b / 8 / nt * 8 + b % 8;
}

// The tile heights of a launch; the first is what its buffers are made for. An
// entry of up to 160 slots takes its weights once or twice; heights of 192,
// 128 and 64 (once, two buffers) took 1521 us where these take 1437 (4096
// tokens, 256 experts of 1536), tiles of 128 x 128 in two buffers 1477.
template <bool LARGE>
struct MW8Tiles {
    using H1 = W8A8Shape<128, 256, 2, 4, 3>;
    using H0 = W8A8Shape<64, 256, 2, 4, 3>;
};
template <>
struct MW8Tiles<false> {
    using H1 = W8A8Shape<64, 128, 2, 2, 2>;
    using H0 = H1;
};

// gate/up of slots m0 .. of the entry: of every 64 weight rows of the tile the
// first 32 are gate rows, the others the up rows of the same 32 columns of h: a
// wave holds both.
template <class S, class L>
__device__ __forceinline__ void gate_up_tile(const MoeW8A8Args &a, const MW8Entry &t, int m0, int j0) {
    static_assert(S::NT % 2 == 0, "a wave holds gate and up of a column");
    const int64_t eF = int64_t(t.e) * a.F;
    const int32_t *pt = a.pair_tok + t.base;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) {
        const int r = S::load_row(j);
        bp[j] = ((r / 32) % 2 ? a.uw : a.gw) + (eF + min(j0 + r / 64 * 32 + r % 32, a.F - 1)) * a.H;
    }
#pragma unroll
    for (int j = 0; j < S::AJ; ++j) ap[j] = a.qx + int64_t(pt[min(m0 + S::load_row(j), t.M - 1)]) * a.H;
    i32x16 acc[S::MT][S::NT];
    w8_clear<S>(acc);
    unsigned char *spare;
    w8_tile<S, 1, L>(ap, bp, a.H, acc, spare);
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

template <class S, class L>
__device__ __forceinline__ void down_tile(const MoeW8A8Args &a, const MW8Entry &t, int m0, int n0) {
    const int64_t eH = int64_t(t.e) * a.H;
    const int8_t *ap[S::AJ], *bp[S::BJ];
#pragma unroll
    for (int j = 0; j < S::BJ; ++j) bp[j] = a.dw + (eH + min(n0 + S::load_row(j), a.H - 1)) * a.F;
#pragma unroll
    for (int j = 0; j < S::AJ; ++j) ap[j] = a.qh + int64_t(t.base + min(m0 + S::load_row(j), t.M - 1)) * a.F;
    i32x16 acc[S::MT][S::NT];
    w8_clear<S>(acc);
    unsigned char *spare;
    w8_tile<S, 2, L>(ap, bp, a.F, acc, spare);
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

// DOWN: the down projection, else gate/up. Where experts have few slots their
// weights are read once and streamed past the caches (250 tokens, 256 experts:
// 755 -> 697 us, 7.0 TB/s); with several entries an expert the second finds them
// there (4096 tokens: streamed 1729 us, else 1435).
template <bool DOWN, bool LARGE>
__global__ __launch_bounds__(MW8Tiles<LARGE>::H1::THREADS, 2) void moe_w8a8_kernel(MoeW8A8Args a) {
    using T = MW8Tiles<LARGE>;
    using L = W8Lds<typename T::H1, DOWN ? 2 : 1, !LARGE>;
    constexpr int COLS = DOWN ? T::H1::BN : T::H1::BN / 2;
    int col;
    MW8Entry t;
    if (!mw8_entry(a, mw8_place(int(blockIdx.x), ((DOWN ? a.H : a.F) + COLS - 1) / COLS, col), t)) return;
    auto tile = [&](auto shape, int m0) {
        using S = decltype(shape);
        if constexpr (DOWN) down_tile<S, L>(a, t, m0, col * COLS);
        else gate_up_tile<S, L>(a, t, m0, col * COLS);
        return S::BM;
    };
    for (int m0 = 0; m0 < t.M;) {
        if (m0 > 0) __syncthreads();  // the tile before is read
        if constexpr (!LARGE) m0 += tile(typename T::H0{}, m0);
        else if (t.M - m0 > T::H0::BM) m0 += tile(typename T::H1{}, m0);
        else m0 += tile(typename T::H0{}, m0);
    }
}

template <bool LARGE>
static void launch_moe_tiles(MoeW8A8Args a, unsigned tiles, size_t P, int8_t *qh, float *sh, hipStream_t s) {
    constexpr int BN = MW8Tiles<LARGE>::H1::BN, THREADS = MW8Tiles<LARGE>::H1::THREADS;
    const unsigned rows = (tiles + 7) / 8 * 8;  // (whole turns of the 8 XCDs)
    moe_w8a8_kernel<false, LARGE><<<rows * unsigned((a.F + BN / 2 - 1) / (BN / 2)), THREADS, 0, s>>>(a);
    launch_quant_tokens(a.h, 2, a.F, int(P), a.F, qh, a.F, sh, s);
    moe_w8a8_kernel<true, LARGE><<<rows * unsigned((a.H + BN - 1) / BN), THREADS, 0, s>>>(a);
}

// ------------------------------------------------------------ few tokens
// f with the number of slots to stage together as a constant: 1, 2 or (rows
// that come quantised) 4 or 8.
template <int XT, class F>
__device__ __forceinline__ void mw8_by_slots(int M, F f) {
    if (M <= 1) f(std::integral_constant<int, 1>{});
    else if (XT != 3 || M <= 2) f(std::integral_constant<int, 2>{});
    else if (M <= 4) f(std::integral_constant<int, 4>{});
    else f(std::integral_constant<int, 8>{});
}

// gate/up of an entry: 8 columns of h per block, from rows x of type XT (3:
// a.qx, a.sx).
template <int XT, bool VEC>
__global__ __launch_bounds__(256) void moe_gate_up_gemv_kernel(MoeW8A8Args a, const void *x) {
    extern __shared__ __align__(16) unsigned char s_q[];
    const int nt = (a.F + 7) / 8, j0 = int(blockIdx.x) % nt * 8;
    MW8Entry t;
    if (!mw8_entry(a, int(blockIdx.x) / nt, t)) return;
    const int64_t eF = int64_t(t.e) * a.F, row = eF + min(j0 + gemv_row(), a.F - 1);
    const int8_t *w[2] = {a.gw + row * a.H, a.uw + row * a.H};
    const int32_t *pt = a.pair_tok + t.base;
    mw8_by_slots<XT>(t.M, [&](auto tm) {
        constexpr int TM = decltype(tm)::value;
        for (int m0 = 0; m0 < t.M; m0 += TM) {
            W8Stream<2> v;
            v.load(w, a.H, gemv_wave());
            auto token = [&](int m) { return int64_t(pt[min(m0 + m, t.M - 1)]); };
            float sx[TM];
            if (m0 > 0) __syncthreads();
            if constexpr (XT == 3) gemv_stage_i8<TM>(a.qx, a.H, a.sx, a.H, s_q, sx, token);
            else gemv_stage<XT, VEC, TM>(x, a.H, a.H, s_q, sx, token);
            gemv_sums<TM, 2>(v, w, a.H, s_q, [&](auto sum) {
                const int m = int(threadIdx.x) / 8, j = j0 + int(threadIdx.x) % 8;
                if (m >= TM || m0 + m >= t.M || j >= a.F) return;
                const float s = gemv_pick(sx, m);
                const float g = w8_value(sum(m, int(threadIdx.x) % 8), a.gs[eF + j], s);
                const float u = w8_value(sum(m, 8 + int(threadIdx.x) % 8), a.us[eF + j], s);
                w8_store(a.h, 2, int64_t(t.base + m0 + m) * a.F + j, silu_ref(g) * u);
            });
        }
    });
}

// down of an entry: 16 rows per block, from h (XT 2) or a.qh, a.sh (3).
template <int XT, bool VEC>
__global__ __launch_bounds__(256) void moe_down_gemv_kernel(MoeW8A8Args a) {
    extern __shared__ __align__(16) unsigned char s_q[];
    const int nt = (a.H + 15) / 16, n0 = int(blockIdx.x) % nt * 16;
    MW8Entry t;
    if (!mw8_entry(a, int(blockIdx.x) / nt, t)) return;
    const int64_t eH = int64_t(t.e) * a.H;
    const int8_t *w[2] = {a.dw + (eH + min(n0 + gemv_row(), a.H - 1)) * a.F,
                          a.dw + (eH + min(n0 + 8 + gemv_row(), a.H - 1)) * a.F};
    mw8_by_slots<XT>(t.M, [&](auto tm) {
        constexpr int TM = decltype(tm)::value;
        for (int m0 = 0; m0 < t.M; m0 += TM) {
            W8Stream<2> v;
            v.load(w, a.F, gemv_wave());
            auto slot = [&](int m) { return int64_t(t.base + min(m0 + m, t.M - 1)); };
            float sx[TM];
            if (m0 > 0) __syncthreads();
            if constexpr (XT == 3) gemv_stage_i8<TM>(a.qh, a.F, a.sh, a.F, s_q, sx, slot);
            else gemv_stage<XT, VEC, TM>(a.h, a.F, a.F, s_q, sx, slot);
            gemv_sums<TM, 2>(v, w, a.F, s_q, [&](auto sum) {
                const int m = int(threadIdx.x) / 16, n = n0 + int(threadIdx.x) % 16;
                if (m < TM && m0 + m < t.M && n < a.H)
                    w8_store(a.yp, a.yp_type, int64_t(t.base + m0 + m) * a.H + n,
                             w8_value(sum(m, int(threadIdx.x) % 16), a.ds[eH + n], gemv_pick(sx, m)));
            });
        }
    });
}

// ------------------------------------------------------------ launches
static size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

size_t moe_w8a8_workspace_bytes(int T, int topk, int H, int F) {
    const size_t P = size_t(T) * size_t(topk);
    return up256(size_t(T) * size_t(H)) + up256(size_t(T) * 4) + up256(P * size_t(F)) + up256(P * 4);
}

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
    // entries of the list at most (each has a slot)
    const unsigned tiles = unsigned(std::min(P, P / size_t(-MW8_TILE_M) + size_t(a.E)));
    auto blocks = [](int rows, int per) { return unsigned((rows + per - 1) / per); };
    // Streamed or in tiles (device us, 8 of 256 experts of 4096 x 1536): 1 token
    // 35.7 and 46.0, 8 tokens 166 and 179, 16 tokens 276 and 277; 8 of 64: 6
    // tokens 115 and 128, 8 tokens 140 and 150. Small experts leave a block of the
    // streaming kernels little to read per row staged, and turn sooner: 6 of 64
    // of 2048 x 1024, 4 tokens 37.6 and 41.5, 6 tokens 45.9 and 43.1, 16 tokens
    // 80 and 59; 8 of 128 of 2048 x 768, 4 tokens 39.8 and 40.3, 8 tokens 57 and
    // 50.
    const bool stream = T <= (size_t(a.H) * size_t(a.F) >= (4u << 20) ? 16 : 4) &&
                        gemv_lds(8, std::max(a.H, a.F)) <= W8_GEMV_LDS;
    if (stream && T <= 2) {
        // one or two tokens: the blocks quantise the rows they stage (two
        // launches less: 35.7 us against 39.4 and 59.4 against 63.4)
        const unsigned gu = tiles * blocks(a.F, 8), dn = tiles * blocks(a.H, 16);
        w8_by_rows(x, x_type, a.H, T, [&](auto xt, auto vec) {
            moe_gate_up_gemv_kernel<decltype(xt)::value, decltype(vec)::value>
                <<<gu, 256, gemv_lds(2, a.H), s>>>(a, x);
        });
        w8_by_rows(a.h, 2, a.F, int(P), [&](auto, auto vec) {
            moe_down_gemv_kernel<2, decltype(vec)::value><<<dn, 256, gemv_lds(2, a.F), s>>>(a);
        });
    } else if (stream) {
        launch_quant_tokens(x, x_type, a.H, T, a.H, qx, a.H, sx, s);
        moe_gate_up_gemv_kernel<3, true><<<tiles * blocks(a.F, 8), 256, gemv_lds(8, a.H), s>>>(a, nullptr);
        launch_quant_tokens(a.h, 2, a.F, int(P), a.F, qh, a.F, sh, s);
        moe_down_gemv_kernel<3, true><<<tiles * blocks(a.H, 16), 256, gemv_lds(8, a.F), s>>>(a);
    } else {
        launch_quant_tokens(x, x_type, a.H, T, a.H, qx, a.H, sx, s);
        // tall tiles from 24 slots per expert (8 of 256 experts: 512 tokens, 16
        // each, 912 us tall and 855 low; 768: 1019 and 1014; 896: 945 and 1002;
        // 1024: 972 and 1059; 1536: 1053 and 1256)
        if (P > size_t(24) * size_t(a.E)) launch_moe_tiles<true>(a, tiles, P, qh, sh, s);
        else launch_moe_tiles<false>(a, tiles, P, qh, sh, s);
    }
}

}  // namespace qwq4
