// Low-rank adapters of many requests beside a projection that all share, and
// their gradients.
//
//   v_t = A[id_t] x_t                              shrink: [R][K] x [K]
//   y_t += scaling[id_t] B[id_t] v_t               expand: [N][R] x [R]
//   dv_t = B[id_t]^T dy_t                          shrink, with B transposed
//   dx_t += scaling[id_t] A[id_t]^T dv_t           expand, with A transposed
//   dA[l] = scaling[l] sum_t dv_t x_t^T,  dB[l] = scaling[l] sum_t dy_t v_t^T     over the tokens of adapter l
//
// A token with an id outside 0 .. L - 1 has no adapter. Tokens need no order:
// a tile of tokens is taken once for each adapter in it, with the others'
// results dropped, so a batch of long requests pays one product per tile and
// a batch of single tokens reads each adapter's weights where it has to
// anyway. All products run on the 16-bit MFMA with sums in fp32. v is kept in
// fp32; where it meets 16-bit weights again it goes in as two (16-bit outputs)
// or three (fp32 outputs) 16-bit parts: with ranks of tens the added products cost
// less than the rows' traffic. In bf16 their sum is v to 2^-17 or exactly. In fp16,
// scaled by the token's largest, it is to 2^-22 or exactly down to 2^-15 of that, and
// below to 2^-39 of it. The fewer bits of 16-bit outputs are a choice: 2^-17 stands
// beside the output's own 2^-8, and a third part would not fit the one step of the
// MFMA that covers two of rank 16.
#include <algorithm>
#include <type_traits>

#include "q4_kernels.hpp"
#include "row_io.cuh"

namespace qwq4 {

// 8 fp32 values as PARTS operands of 8 16-bit values that add up to them.
template <class T, int PARTS>
__device__ __forceinline__ void split8(const float (&f)[8], uint4 (&part)[PARTS]) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = f[j];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = pack2<T>(r[2 * j], r[2 * j + 1]);
            if (p + 1 < PARTS) {
                float a, b;
                unpack2<T>(w[j], a, b);
                r[2 * j] -= a;
                r[2 * j + 1] -= b;
            }
        }
        part[p] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

__device__ __forceinline__ void load8(const float *p, float (&f)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// 8 columns of 8 rows of 16-bit elements, a row in each register group, as a column in each.
__device__ __forceinline__ void turn8(const uint4 (&row)[8], uint4 (&column)[8]) {
    uint32_t d[8][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e][0] = row[e].x, d[e][1] = row[e].y, d[e][2] = row[e].z, d[e][3] = row[e].w;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = __builtin_amdgcn_perm(d[2 * e + 1][j / 2], d[2 * e][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
        column[j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The adapters among a wave's tokens (lane i: token i's, or -1), every `of`-th
// from `from` on: f(adapter, mask of its tokens). The same in every wave that
// asks for the same tokens.
template <class F>
__device__ __forceinline__ void each_adapter(int id, int from, int of, F f) {
    unsigned long long left = __ballot(id >= 0);
    for (int j = 0; left; ++j) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const unsigned long long mine = __ballot(id == a);
        left &= ~mine;
        if (j % of == from) f(a, mine);
    }
}

__device__ __forceinline__ int adapter_of(const int32_t *ids, int t, int T, int L) {
    if (t >= T) return -1;
    const int id = ids[t];
    return id >= 0 && id < L ? id : -1;
}

// ------------------------------------------------------------ shrink
// A wave's 16 rows of 64 16-bit elements on their way from memory to MFMA
// operands: read with eight lanes to a row (a 128-byte line each, where the
// operand's lane order would touch 16 lines with every 16 lanes and move 7
// bytes a cycle), turned in LDS. The 16-byte piece p of row r lies at place p ^ (r &
// 7) of its row: without bank conflicts both ways.
struct Turned {
    uint4 w[2];
    // the lane's places, in bytes behind the first element of `rows` (or the last one again) from `row0` on
    __device__ static __forceinline__ void places(uint32_t (&at)[2], int row0, int rows, uint32_t stride) {
        const int lane = int(threadIdx.x) % WAVE;
#pragma unroll
        for (int i = 0; i < 2; ++i) at[i] = (uint32_t(min(row0 + 8 * i + lane / 8, rows - 1)) * stride + lane % 8 * 8) * 2;
    }
    // from: the same in every lane (places of 32 bits beside it: half the registers of pointers); the first n of the 64
    // elements exist, and of the rows those in `rows` are asked for
    __device__ __forceinline__ void load(const uint16_t *from, const uint32_t (&at)[2], int n, uint32_t rows = ~0u) {
        const int lane = int(threadIdx.x) % WAVE;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = lane % 8 * 8 < n && ((rows >> (8 * i + lane / 8)) & 1) ? *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(from) + at[i])
                      : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void put(uint4 *lds) const {
        const int lane = int(threadIdx.x) % WAVE, r = lane / 8;
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < 2; ++i) lds[(8 * i + r) * 8 + (lane % 8 ^ r)] = w[i];
        wave_lds_order();
    }
    // the operand of the first or second 32 elements
    __device__ static __forceinline__ uint4 operand(const uint4 *lds, int h) {
        const int lane = int(threadIdx.x) % WAVE, c = lane % 16, g = lane / 16;
        return lds[c * 8 + ((4 * h + g) ^ (c & 7))];
    }
    // (a wave's LDS accesses complete in order; the compiler must keep them so)
    __device__ static __forceinline__ void wave_lds_order() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
    }
};

// The same for 16 columns of 64 rows of weights that lie with the ranks inside
// ([K][R]): read as they lie, and turned by LDS's transposing reads (four rows of 16
// elements to 16 lanes, each of which gets a column). Against a transposed copy in
// the workspace: gradients of 601 tokens of rank 64 30 us for 36, of 4096 of rank 32 58 for
// 65; of rank 128, whose rows' pieces of 32 bytes cost the loads more, 179 for 172.
struct TurnedColumns {
    uint4 w[2];
    // the lane's places in bytes, the ranks from r0 on (behind the last one the last ones again, whose sums nothing takes)
    __device__ static __forceinline__ void places(uint32_t (&at)[2], int r0, int R) {
        const int lane = int(threadIdx.x) % WAVE;
#pragma unroll
        for (int i = 0; i < 2; ++i) at[i] = uint32_t((32 * i + lane / 2) * R + min(r0 + lane % 2 * 8, R - 8)) * 2;
    }
    // the first n of the 64 rows exist
    __device__ __forceinline__ void load(const uint16_t *from, const uint32_t (&at)[2], int n) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = 32 * i + int(threadIdx.x) % WAVE / 2 < n
                       ? *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(from) + at[i])
                       : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void put(uint4 *lds) const {
        const int lane = int(threadIdx.x) % WAVE;
        Turned::wave_lds_order();
#pragma unroll
        for (int i = 0; i < 2; ++i) lds[WAVE * i + lane] = w[i];
        Turned::wave_lds_order();
    }
    __device__ static __forceinline__ uint4 operand(uint4 *lds, int h) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const int lane = int(threadIdx.x) % WAVE, c = lane % 16, g = lane / 16;
        short *row = reinterpret_cast<short *>(lds) + (32 * h + 8 * g + c / 4) * 16 + c % 4 * 4;
        auto four = [&](int k) {
            return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                 (__attribute__((address_space(3))) s16x4 *)(row + k * 16)));
        };
        const uint2 a = four(0), b = four(4);
        return make_uint4(a.x, a.y, b.x, b.y);
    }
};

// v[t][r] = sum_k A[id_t][r][k] x[t][k] for 16 tokens and 16 RF ranks by a block
// whose 16 waves take a run of 64-wide steps of K each and join their sums in
// LDS, in order: a row's bits depend on neither the batch nor its place in it.
// Every wave has U steps of rows and weights on their way: a step's registers are
// loaded again as soon as it lies in LDS (three steps of 16 ranks or two of 64: no
// faster, or spilled: 110 us for 102 with 4096 x 12288 of rank 64). Rows of other
// adapters are not read. A CU takes in rows and weights at 30 to 40 bytes a cycle,
// which bounds it: 4096 rows of 4096 in 11 us (3.1 TB/s of rows, as much again of
// weights out of L2), of 12288 in 29 (3.5). INSIDE: the ranks lie inside, A is [K][R].
template <class T16, int RF, bool INSIDE>
__global__ __launch_bounds__(1024) void lora_shrink_kernel(LoraShrinkArgs a) {
    constexpr int NW = 16, U = RF <= 2 ? 2 : 1;
    __shared__ uint4 s_turn[NW][2][128];  // (4 KB a wave, and then the waves' sums)
    f32x4(*s_part)[RF][WAVE] = reinterpret_cast<f32x4(*)[RF][WAVE]>(s_turn);
    static_assert(sizeof(f32x4) * NW * RF * WAVE <= sizeof(s_turn), "the sums fit");
    const int lane = int(threadIdx.x) % WAVE, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    const int c = lane % 16, g = lane / 16, t0 = int(blockIdx.x) * 16, t = t0 + c;
    const int r0 = int(blockIdx.z) * (16 * RF);
    const int id = lane < 16 ? adapter_of(a.ids, t0 + lane, a.T, a.L) : -1;
    const int steps = (a.K + 63) / 64, per = (steps + NW - 1) / NW, end = min(steps, (wave + 1) * per);
    const uint16_t *x = a.x + t0 * a.ldx;
    uint32_t xat[2], wat[RF][2];  // (16 strides are below 2^31 bytes, as R K is)
    Turned::places(xat, 0, a.T - t0, uint32_t(a.ldx));
#pragma unroll
    for (int f = 0; f < RF; ++f) {
        if constexpr (INSIDE) TurnedColumns::places(wat[f], r0 + 16 * f, a.R);
        else Turned::places(wat[f], r0 + 16 * f, a.R, uint32_t(a.K));
    }
    each_adapter(id, int(blockIdx.y), int(gridDim.y), [&](int l, unsigned long long mine) {
        const uint16_t *A = a.A + int64_t(l) * a.R * a.K;
        f32x4 acc[RF];
#pragma unroll
        for (int f = 0; f < RF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
        Turned nx[U];
        std::conditional_t<INSIDE, TurnedColumns, Turned> nw[U][RF];
        auto load = [&](int u, int step) {
            if (step >= end) return;
            const int k = step * 64, n = a.K - k;
            nx[u].load(x + k, xat, n, uint32_t(mine));
#pragma unroll
            for (int f = 0; f < RF; ++f) nw[u][f].load(A + (INSIDE ? int64_t(k) * a.R : k), wat[f], n);
        };
        const int first = wave * per;
#pragma unroll
        for (int u = 0; u < U; ++u) load(u, first + u);
        for (int s0 = first; s0 < end; s0 += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s0 + u >= end) continue;
                nx[u].put(s_turn[wave][0]);
                uint4 xf[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) xf[h] = Turned::operand(s_turn[wave][0], h);
#pragma unroll
                for (int f = 0; f < RF; ++f) {
                    nw[u][f].put(s_turn[wave][1]);
                    if (f + 1 == RF) load(u, s0 + u + U);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        acc[f] = mfma16<T16>(nw[u][f].operand(s_turn[wave][1], h), xf[h], acc[f]);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int f = 0; f < RF; ++f) s_part[wave][f][lane] = acc[f];
        __syncthreads();
        const int f = wave, r = r0 + 16 * f + 4 * g;  // (a wave adds a piece: RF <= 16)
        if (f < RF && r < a.R && ((mine >> c) & 1)) {
            f32x4 sum = s_part[0][f][lane];
#pragma unroll
            for (int i = 1; i < NW; ++i) sum += s_part[i][f][lane];
            *reinterpret_cast<f32x4 *>(a.v + int64_t(t) * a.R + r) = sum;
        }
        __syncthreads();
    });
}

void launch_lora_shrink(const LoraShrinkArgs &a, hipStream_t s) {
    const int tiles = (a.T + 15) / 16;
    // Adapters of a tile in parallel while there are few tiles (37 requests with an adapter each: every block takes
    // one), all of a tile's by one block where the tiles fill the chip; ranks likewise, 16 or up to 64 a block.
    const int side = std::max(1, std::min({256 / tiles, 16, a.L, a.T}));
    auto run = [&](auto t16, auto rf) {
        constexpr int RF = decltype(rf)::value;
        const dim3 grid{unsigned(tiles), unsigned(side), unsigned((a.R + 16 * RF - 1) / (16 * RF))};
        if (a.inside) lora_shrink_kernel<decltype(t16), RF, true><<<grid, 1024, 0, s>>>(a);
        else lora_shrink_kernel<decltype(t16), RF, false><<<grid, 1024, 0, s>>>(a);
    };
    auto by_rank = [&](auto t16) {
        if (a.R <= 16 || tiles * side < 128) run(t16, Int<1>{});
        else if (a.R <= 32) run(t16, Int<2>{});
        else run(t16, Int<4>{});
    };
    if (a.f16) by_rank(F16{});
    else by_rank(BF16{});
}

// out[l] = the parts of adapter l that have tokens, in order (none: zeros).
__device__ __forceinline__ void join_parts(const LoraJoinArgs &a, int block) {
    const int blocks = a.blocks(), l = block / blocks;
    if (l >= a.L) return;
    const int64_t i = (int64_t(block % blocks) * 256 + int(threadIdx.x)) * 4;
    const bool second = i >= a.n[0];
    float *out = a.out[second];
    const int64_t at = second ? i - a.n[0] : i, each = a.n[second];
    // (which parts have any, before the rows of those are asked for)
    const int lane = int(threadIdx.x) % WAVE;
    unsigned long long which = __ballot(lane < a.parts && a.count[min(lane, a.parts - 1) * a.L + l] > 0);
    if (at >= each) return;
    const float *p = a.part[second] + l * each + at;
    const int64_t step = a.L * each;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    while (which) {
        f32x4 v[4];
        int n = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (!which) continue;
            v[u] = *reinterpret_cast<const f32x4 *>(p + step * __builtin_ctzll(which));
            which &= which - 1;
            ++n;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (u < n) sum += v[u];
    }
    *reinterpret_cast<f32x4 *>(out + l * each + at) = sum;
}

// ------------------------------------------------------------ expand
// out[t][n] = y[t][n] + scaling[id_t] sum_r B[id_t][n][r] v[t][r]: 16 tokens by 128
// columns a wave at a time. The columns are dealt to 8 MFMAs so that a lane holds 8
// neighbouring ones of four tokens and 16 lanes a row's 128: rows are read and
// written in 256-byte runs (four lanes to a token's 64 columns: 47 us where this
// takes 43, 4096 x 12288 in bf16), past the caches (kept in them: 5 us more). K of the
// MFMA runs over the R values of each of v's parts in turn. fp16 parts are of v
// times a power of two per token, so that none of them overflows or loses bits to the
// range. Bound by memory.
// ONE: one step of the MFMA covers all parts; its weights stay in registers, and a
// wave takes NT = a.tiles (at most 4) tiles of 16 tokens one after the other.
// Else the rows of B lie in LDS, 16-byte piece p of a row at place p ^ (row / 8 & 7):
// without bank conflicts. The block's four waves take a tile each of the same 128
// columns (NT = 4), or 128 columns each of one tile (NT = 1).
// COLUMNS: the columns lie inside, B is [R][N]: a lane reads its 8 columns of 8 ranks
// and turns them in registers; and the blocks behind the expanding ones join the
// parts of the weights' gradients (as much work as in a launch of its own, but
// without that launch's 3 us or so).
template <class T16, int YT, bool ONE, bool COLUMNS>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraExpandArgs a, LoraJoinArgs join) {
    constexpr bool HALF = __is_same(T16, F16);
    constexpr int PARTS = YT == 0 ? 3 : 2;
    if constexpr (COLUMNS) {
        if (int(blockIdx.z) >= a.side) {
            join_parts(join, ((int(blockIdx.z) - a.side) * int(gridDim.y) + int(blockIdx.y)) * int(gridDim.x) + int(blockIdx.x));
            return;
        }
    }
    extern __shared__ uint4 s_weights[];  // ONE: none; [columns R / 8]
    const int lane = int(threadIdx.x) % WAVE, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    const int c = lane % 16, g = lane / 16;
    const int NT = a.tiles, t0 = int(blockIdx.y) * (16 * NT);
    const bool share = !ONE && NT == 4;
    const int n0 = (share ? int(blockIdx.x) : int(blockIdx.x) * 4 + wave) * 128;
    if (ONE && n0 >= a.N) return;  // (no barrier below)
    const int at = n0 + 8 * c;    // the lane's columns
    const bool in = at < a.N;     // (N is a multiple of 8)
    const int id = lane < 16 * NT ? adapter_of(a.ids, t0 + lane, a.T, a.L) : -1;
    const int octets = a.R / 8, steps = ONE ? 1 : (PARTS * octets + 3) / 4;
    if (a.out != a.y && blockIdx.z == 0) {  // (rows without an adapter)
        const unsigned long long none = ~__ballot(id >= 0);
        for (int i = share ? 4 * wave : 0; i < 16 * NT; i += share ? 16 : 4) {
            const int t = t0 + i + g;
            if (t < a.T && in && ((none >> (i + g)) & 1)) {
                RowPiece<YT> y;
                y.load_stream(a.y, t * a.ldy + at);
                y.store_stream(a.out, t * a.ldo + at);
            }
        }
    }
    uint4 *lds = s_weights + (share ? 0 : wave * 128 * octets);
    each_adapter(id, int(blockIdx.z), a.side, [&](int l, unsigned long long mine) {
        const float scale = a.scaling ? a.scaling[l] : 1.f;
        // the wave's rows, min(128, N - n0) of them, or its columns
        const uint16_t *B = a.B + int64_t(l) * a.N * a.R + (COLUMNS ? min(at, a.N - 8) : n0 * a.R);
        // COLUMNS: octet o of the lane's columns' ranks
        auto octet = [&](int o, uint4 (&w)[8]) {
            uint4 rank[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) rank[j] = *reinterpret_cast<const uint4 *>(B + uint32_t(8 * o + j) * uint32_t(a.N));
            turn8(rank, w);
        };
        // the tokens of tile i that are this adapter's, and their rows
        auto tokens = [&](int i) { return i < NT ? uint32_t(mine >> (16 * i)) & 0xffffu : 0u; };
        auto rows = [&](int i, RowPiece<YT> (&y)[4]) {
            const uint32_t here = tokens(i) >> (4 * g);
            const int64_t row = int64_t(t0 + 16 * i + 4 * g) * a.ldy + at;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (in && ((here >> e) & 1)) y[e].load_stream(a.y, row + e * a.ldy);
        };
        RowPiece<YT> next[4];
        rows(share ? wave : 0, next);
        // place o of v's parts and what it is: octet ro of part p (none from PARTS on)
        auto place = [&](int q, int &p) {
            const int o = 4 * q + g;
            p = ONE ? (o >= octets) + (o >= 2 * octets) + (PARTS == 3 && o >= 3 * octets) : o / octets;
            return p < PARTS ? o - p * octets : 0;
        };
        uint4 wf[8];
        if constexpr (ONE) {
            int p;
            const int ro = place(0, p);
            if constexpr (COLUMNS) octet(ro, wf);
            else {
                const uint16_t *w = B + min(8 * c, a.N - 8 - n0) * a.R + 8 * ro;
#pragma unroll
                for (int j = 0; j < 8; ++j) wf[j] = *reinterpret_cast<const uint4 *>(w + j * a.R);
            }
        } else if constexpr (COLUMNS) {
            for (int o = (share ? 4 * wave : 0) + g; o < octets; o += share ? 16 : 4) {
                octet(o, wf);
#pragma unroll
                for (int j = 0; j < 8; ++j) lds[((8 * c + j) * octets + o) ^ (c & 7)] = wf[j];
            }
            __syncthreads();
        } else {
            const int n = min(128, a.N - n0) * octets;
            const uint32_t inverse = (65536u + uint32_t(octets) - 1) / uint32_t(octets);  // (exact below 4096)
#pragma unroll 4
            for (int i = share ? int(threadIdx.x) : lane; i < n; i += share ? 4 * WAVE : WAVE)
                lds[i ^ int(((uint32_t(i) * inverse >> 16) >> 3) & 7)] = reinterpret_cast<const uint4 *>(B)[i];
            __syncthreads();
        }
        auto tile = [&](int i, const RowPiece<YT> (&y)[4]) {
            const uint32_t here = tokens(i);
            if (!here) return;
            const bool own = (here >> c) & 1;  // (token c's values of v are this lane's operand)
            const float *v = a.v + int64_t(t0 + 16 * i + c) * a.R;
            int shift = 0;
            if constexpr (HALF) {
                float top = 0.f;
                for (int o = g; own && o < octets; o += 4) {
                    float f[8];
                    load8(v + 8 * o, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(f[j] * scale));
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                // (2^shift top below 2^15)
                shift = 141 - int((__builtin_bit_cast(uint32_t, top) >> 23) & 255u);
            }
            f32x4 acc[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int q = 0; q < steps; ++q) {
                int p;
                const int ro = place(q, p);
                if constexpr (!ONE) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) wf[j] = lds[((8 * c + j) * octets + ro) ^ (c & 7)];
                }
                float f[8] = {};
                if (own && p < PARTS) {
                    load8(v + 8 * ro, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        f[j] *= scale;
                        if constexpr (HALF) f[j] = __builtin_ldexpf(f[j], shift);
                    }
                }
                uint4 part[PARTS];
                split8<T16, PARTS>(f, part);
                uint4 vf = part[0];
                if (p == 1) vf = part[1];
                if constexpr (PARTS == 3) {
                    if (p == 2) vf = part[2];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] = mfma16<T16>(vf, wf[j], acc[j]);
            }
            const int64_t row = int64_t(t0 + 16 * i + 4 * g) * a.ldo + at;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                int back = 0;
                if constexpr (HALF) back = -__shfl(shift, 4 * g + e);  // (token 4 g + e's, from the lane that scaled it)
                if (!in || !((here >> (4 * g + e)) & 1)) continue;
                float f[8];
                y[e].values(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float d = acc[j][e];
                    if constexpr (HALF) d = __builtin_ldexpf(d, back);
                    f[j] += d;
                }
                RowPiece<YT> o;
                o.template set<YT == GRAD_F16>(f);
                o.store_stream(a.out, row + e * a.ldo);
            }
        };
        if constexpr (ONE) {
#pragma unroll 1
            for (int i = 0; i < NT; ++i) {
                RowPiece<YT> y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = next[e];
                rows(i + 1, next);
                tile(i, y);
            }
        } else {
            tile(share ? wave : 0, next);
            __syncthreads();  // (the weights are read)
        }
    });
}

void launch_lora_expand(LoraExpandArgs a, const LoraJoinArgs &join, hipStream_t s) {
    auto run = [&](auto t16, auto yt, auto columns) {
        constexpr bool COLUMNS = decltype(columns)::value;
        constexpr int YT = decltype(yt)::value;
        const bool one = (YT == 0 ? 3 : 2) * a.R <= 32;
        // ONE: the weights are read once for all tiles of a block, but first of all the chip is to be filled (one tile
        // for two: 2048 x 4096 of rank 16 19.5 us for 16.8); two serve up to the largest calls (four: 4096 x 12288 of
        // rank 16 55.4 us for 54.0, 16384 x 12288 187 for 191). Then the adapters of a block's tokens side by side.
        // Else the waves share the columns' weights (with columns of their own a CU holds a third as many waves: 4096 x
        // 4096 of rank 128 85 us for 53, 4096 x 12288 of rank 64 90 for 77), but where 64 tokens may be of many adapters
        // (shared: 64 tokens of 64, 4096 columns of rank 64 22.5 us for 19.8; 1024 mixed ones of 64, rank 32 81 for 56).
        const bool share = !one && (a.T >= 64 * a.L || a.R > 64);  // (at most 64 KB of weights a block)
        const int wide = share ? 128 : 512, tiles = (a.T + 15) / 16, cols = (a.N + wide - 1) / wide;
        a.tiles = share || (one && tiles * cols >= 16384) ? 4 : one && tiles * cols >= 1024 ? 2 : 1;
        const int groups = (tiles + a.tiles - 1) / a.tiles;
        a.side = std::max(1, std::min({1024 / (groups * cols), 16 * a.tiles, a.L, a.T}));
        const int joining = join.L ? (join.L * join.blocks() + groups * cols - 1) / (groups * cols) : 0;
        const dim3 grid{unsigned(cols), unsigned(groups), unsigned(a.side + joining)};
        const size_t lds = one ? 0 : size_t(share ? 256 : 1024) * size_t(a.R);
        if (one) lora_expand_kernel<decltype(t16), YT, true, COLUMNS><<<grid, 256, lds, s>>>(a, join);
        else lora_expand_kernel<decltype(t16), YT, false, COLUMNS><<<grid, 256, lds, s>>>(a, join);
    };
    auto by_16 = [&](auto yt) {
        if (a.f16) run(F16{}, yt, Int<0>{});
        else run(BF16{}, yt, Int<0>{});
    };
    if (!a.columns) by_type(a.y_type, by_16);
    else if (a.f16) run(F16{}, Int<GRAD_F16>{}, Int<1>{});
    else run(BF16{}, Int<1>{}, Int<1>{});
}

// ------------------------------------------------------------ gradients
constexpr int OUTER_COLS = 512;     // columns of a block
constexpr int OUTER_TOKENS = 1024;  // tokens whose ids it looks at at once

// 8 fp16 values as two bf16 operands: their first 8 bits, and the last 3, which are left behind them exactly.
__device__ __forceinline__ void halves_of_f16(const uint4 &w, uint4 &high, uint4 &low) {
    const uint32_t in[4] = {w.x, w.y, w.z, w.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t top[2], rest[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float f = f16_bits_to_f32(uint16_t(in[i] >> (16 * e)));
            top[e] = __builtin_bit_cast(uint32_t, f) & 0xffff0000u;
            rest[e] = __builtin_bit_cast(uint32_t, f - __builtin_bit_cast(float, top[e]));
        }
        h[i] = __builtin_amdgcn_perm(top[1], top[0], 0x07060302u);
        l[i] = __builtin_amdgcn_perm(rest[1], rest[0], 0x07060302u);
    }
    high = make_uint4(h[0], h[1], h[2], h[3]);
    low = make_uint4(l[0], l[1], l[2], l[3]);
}

// G[r][c] = scaling sum_t u[t][r] m[t][c] over the tokens of one adapter in one
// part of the batch: 128 columns a wave, 16 RF ranks. The tokens are listed in
// LDS in order. The sum runs over tokens, whose values lie a row apart: a lane
// loads 8 columns of 8 tokens and turns them in registers (v_perm) into 8
// operands of one column each, so the wide rows come in 16-byte loads and
// never pass through LDS. u goes in as three bf16 parts whose sum it is. fp16 rows go
// in as two bf16 parts, also exactly, so that small factors keep their bits beside
// large ones, which fp16 has no range for: as two fp16 parts of u times a power of two
// per rank, a factor of 2e-8 of the largest was off by 1%. (u's third part times the
// rows' second one is left out: below 2^-25 of the product. A whole call with 4096 fp16
// tokens of rank 16, 4096 and 12288 columns: 81 us for 76 with two fp16 parts.) 4096
// tokens of 4096 and 12288 columns, 16 ranks: 31 us, 4.3 TB/s; alike with two steps on
// their way, with u turned once for the four waves, or a block for all adapters of a part.
template <bool HALF, int RF>
__global__ __launch_bounds__(256) void lora_outer_kernel(LoraOuterArgs a) {
    __shared__ uint32_t s_tok[OUTER_TOKENS];
    __shared__ int s_count[4];
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int c = lane % 16, g = lane / 16;
    const int part = int(blockIdx.z), l = int(blockIdx.y) % a.L, r0 = int(blockIdx.y) / a.L * (16 * RF);
    const bool second = int(blockIdx.x) >= a.m[0].blocks();
    const LoraOuterSide &m = a.m[second];
    const int c0 = (int(blockIdx.x) - (second ? a.m[0].blocks() : 0)) * OUTER_COLS + wave * 128;
    const int from = part * a.per, end = min(a.T, from + a.per);
    const uint16_t *col = m.m + min(c0 + 8 * c, m.C - 8);
    const uint32_t ldm = uint32_t(m.ldm), R = uint32_t(a.R);

    f32x4 acc[RF][8];
#pragma unroll
    for (int f = 0; f < RF; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    int total = 0;
    for (int b0 = from; b0 < end; b0 += OUTER_TOKENS) {
        int n = 0;
        const int b1 = min(end, b0 + OUTER_TOKENS);
        for (int b = b0; b < b1; b += 256) {
            const int t = b + tid;
            const bool mine = t < b1 && a.ids[t] == l;
            const unsigned long long which = __ballot(mine);
            if (lane == 0) s_count[wave] = __popcll(which);
            __syncthreads();
            int before = n;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                before += w < wave ? s_count[w] : 0;
                n += s_count[w];
            }
            if (mine) s_tok[before + __popcll(which & ((1ull << lane) - 1ull))] = uint32_t(t);
            __syncthreads();
        }
        total += n;
        const int steps = c0 < m.C ? (n + 31) / 32 : 0;
        uint4 next[8];
        float nu[RF][8];
        auto load = [&](int s) {
            uint32_t t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = s_tok[min(32 * s + 8 * g + e, n - 1)];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                next[e] = *reinterpret_cast<const uint4 *>(col + uint64_t(t[e]) * ldm);
#pragma unroll
                for (int f = 0; f < RF; ++f) nu[f][e] = m.u[t[e] * R + uint32_t(min(r0 + 16 * f + c, a.R - 1))];
            }
            // (behind the list: nothing, whatever the repeated row holds)
            if (32 * s + 32 > n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (32 * s + 8 * g + e < n) continue;
                    next[e] = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int f = 0; f < RF; ++f) nu[f][e] = 0.f;
                }
            }
        };
        if (steps > 0) load(0);
        for (int s = 0; s < steps; ++s) {
            uint4 column[8], q[RF][3];
            turn8(next, column);
#pragma unroll
            for (int f = 0; f < RF; ++f) split8<BF16, 3>(nu[f], q[f]);
            if (s + 1 < steps) load(s + 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint4 high = column[j], low;
                if constexpr (HALF) halves_of_f16(column[j], high, low);
#pragma unroll
                for (int f = 0; f < RF; ++f) {
#pragma unroll
                    for (int p = 0; p < 3; ++p) acc[f][j] = mfma16<BF16>(q[f][p], high, acc[f][j]);
                    if constexpr (HALF) {
#pragma unroll
                        for (int p = 0; p < 2; ++p) acc[f][j] = mfma16<BF16>(q[f][p], low, acc[f][j]);
                    }
                }
            }
        }
        __syncthreads();  // (the list is read)
    }
    if (a.parts > 1 && blockIdx.x == 0 && r0 == 0 && tid == 0) a.count[part * a.L + l] = total;
    if (total == 0 && a.parts > 1) return;  // (the joining launch goes by the count)

    if (c0 + 8 * c >= m.C) return;
    const float scale = a.scaling && total ? a.scaling[l] : 1.f;  // (without tokens: zeros, whatever a free slot's is)
    float *out = m.out + (int64_t(part) * a.L + l) * a.R * m.C;
#pragma unroll
    for (int f = 0; f < RF; ++f) {
        const int r = r0 + 16 * f + 4 * g;
        if (r >= a.R) continue;
        if (m.by_column) {  // [C][R]
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<f32x4 *>(out + int64_t(c0 + 8 * c + j) * a.R + r) = acc[f][j] * scale;
        } else {  // [R][C]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float *p = out + int64_t(r + i) * m.C + c0 + 8 * c;
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<f32x4 *>(p + j) =
                        f32x4{acc[f][j][i], acc[f][j + 1][i], acc[f][j + 2][i], acc[f][j + 3][i]} * scale;
            }
        }
    }
}

__global__ __launch_bounds__(256) void lora_outer_join_kernel(LoraJoinArgs a) { join_parts(a, int(blockIdx.x)); }

// Parts of the batch whose sums over tokens run side by side, at most
// MAX_PARTS: until about 2048 blocks are there (one whose adapter has no token in
// its part ends at once), of 128 tokens or more. Every part has room for every
// adapter's sums, 64 KB a block at most: with fewer than 4096 blocks in several parts,
// below 256 MB.
constexpr int MAX_PARTS = 64;
static int outer_ranks(int R) { return R <= 16 ? 16 : 32; }
static int outer_parts(int T, int K, int N, int R, int L) {
    const int ranks = outer_ranks(R);
    const int64_t blocks = int64_t((K + OUTER_COLS - 1) / OUTER_COLS + (N + OUTER_COLS - 1) / OUTER_COLS) *
                           ((R + ranks - 1) / ranks) * L;
    return int(std::max<int64_t>(1, std::min<int64_t>({(2048 + blocks - 1) / blocks, (T + 127) / 128, MAX_PARTS})));
}

// Workspace of the gradients: dv, and the parts of dA and dB with their counts,
// each at a multiple of 256 bytes.
struct LoraSpace {
    size_t dv, pa, pb, count, bytes;
    LoraSpace(int T, int K, int N, int R, int L, int parts) {
        size_t end = 0;
        auto take = [&](size_t n) {
            const size_t at0 = end;
            end = (end + n + 255) / 256 * 256;
            return at0;
        };
        const size_t rk = size_t(L) * R * K, rn = size_t(L) * R * N;
        dv = take(size_t(T) * R * 4);
        pa = take(parts > 1 ? rk * 4 * parts : 0);
        pb = take(parts > 1 ? rn * 4 * parts : 0);
        count = take(parts > 1 ? size_t(L) * parts * 4 : 0);
        bytes = end;
    }
};

size_t lora_backward_workspace_bytes(int T, int K, int N, int R, int L) {
    return LoraSpace(T, K, N, R, L, outer_parts(T, K, N, R, L)).bytes;
}

// What is left to join: nothing (L = 0) where the batch is one part.
static LoraJoinArgs launch_lora_outer(const LoraGradArgs &a, char *base, const LoraSpace &at, int parts,
                                      const float *dv, hipStream_t s) {
    float *pa = parts > 1 ? reinterpret_cast<float *>(base + at.pa) : a.dA;
    float *pb = parts > 1 ? reinterpret_cast<float *>(base + at.pb) : a.dB;
    LoraOuterArgs o{};
    // (a side that is not wanted has no columns)
    o.m[0] = LoraOuterSide{a.x, a.ldx, dv, a.dA ? a.K : 0, pa, false};
    o.m[1] = LoraOuterSide{a.dy, a.lddy, a.v, a.dB ? a.N : 0, pb, true};
    o.ids = a.ids;
    o.scaling = a.scaling;
    o.T = a.T;
    o.R = a.R;
    o.L = a.L;
    o.parts = parts;
    o.per = (a.T + parts - 1) / parts;
    o.count = reinterpret_cast<int *>(base + at.count);
    const int ranks = outer_ranks(a.R);
    const dim3 grid(unsigned(o.m[0].blocks() + o.m[1].blocks()), unsigned((a.R + ranks - 1) / ranks * a.L),
                    unsigned(parts));
    auto run = [&](auto half) {
        if (ranks == 16) lora_outer_kernel<decltype(half)::value, 1><<<grid, 256, 0, s>>>(o);
        else lora_outer_kernel<decltype(half)::value, 2><<<grid, 256, 0, s>>>(o);
    };
    if (a.f16) run(std::true_type{});
    else run(std::false_type{});
    if (parts == 1) return LoraJoinArgs{};
    return LoraJoinArgs{{pa, pb}, {a.dA, a.dB}, {a.dA ? int64_t(a.R) * a.K : 0, a.dB ? int64_t(a.R) * a.N : 0}, o.count,
                        a.L, parts};
}

void launch_lora_backward(const LoraGradArgs &a, void *ws, hipStream_t s) {
    const int parts = outer_parts(a.T, a.K, a.N, a.R, a.L);
    const LoraSpace at(a.T, a.K, a.N, a.R, a.L, parts);
    char *base = static_cast<char *>(ws);
    float *dv = reinterpret_cast<float *>(base + at.dv);
    if (a.dx || a.dA)
        launch_lora_shrink(LoraShrinkArgs{a.dy, a.lddy, a.B, a.ids, a.T, a.N, a.R, a.L, dv, a.f16, true}, s);
    LoraJoinArgs join{};
    if (a.dA || a.dB) join = launch_lora_outer(a, base, at, parts, dv, s);
    if (a.dx)
        launch_lora_expand(LoraExpandArgs{dv, a.A, a.ids, a.scaling, a.T, a.K, a.R, a.L, a.f16, a.dx, a.lddx, a.dx_out,
                                          a.lddxo, a.f16 ? 2 : 1, true},
                           join, s);
    else if (join.L) lora_outer_join_kernel<<<unsigned(join.L * join.blocks()), 256, 0, s>>>(join);
}

}  // namespace qwq4
