// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits, and the gradient of the first two.
//
//   lse = log sum_j exp(l_j),  logp = l_tok - lse,  H = lse - sum_j p_j l_j
//   dl_j = dlogp ([j = tok] - p_j) - dH p_j (log p_j + H),   p_j = exp(l_j - lse)
//
// One pass over the row: each lane keeps the largest value m so far,
// S = sum exp(l - m) and U = sum exp(l - m) (l - m), rescaled when m grows;
// then lse = m + log S and H = log S - U / S. A masked logit (-infinity) adds
// nothing to either sum. A row that masks everything has lse and logp of
// -infinity and entropy 0; one with a NaN or +infinity gives NaN.
#include <algorithm>
#include <climits>

#include "q4_kernels.hpp"
#include "row_io.cuh"

namespace qwq4 {

constexpr float LOG2E = 1.44269504088896341f;
// exp(x - y) of sums: below this nothing is left in fp32
constexpr float NEARLY_NONE = -200.f;

__device__ __forceinline__ float exp_fast(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
__device__ __forceinline__ float neg_inf() { return -__builtin_huge_valf(); }

struct SoftStats {
    float m, s, u;
    __device__ __forceinline__ void clear() {
        m = neg_inf();
        s = u = 0.f;
    }
    // The sums moved to a maximum of at least top (which they then have);
    // returns what values are to be taken relative to.
    __device__ __forceinline__ float raise(float top) {
        const float to = fmaxf(m, top), ref = to == neg_inf() ? 0.f : to;
        const float d = m - ref, f = exp_fast(d);  // (0 while nothing but masked values came)
        u = f * __builtin_fmaf(fmaxf(d, NEARLY_NONE), s, u);
        s *= f;
        m = to;
        return ref;
    }
    // (the difference is bounded where it is a factor: 0 times a masked value's would be a NaN)
    __device__ __forceinline__ void add(float v, float ref) {
        const float d = v - ref, e = exp_fast(d);
        s += e;
        u = __builtin_fmaf(e, fmaxf(d, NEARLY_NONE), u);
    }
    __device__ __forceinline__ void join(SoftStats o) {
        const float top = fmaxf(m, o.m);
        raise(top);
        o.raise(top);
        s += o.s;
        u += o.u;
    }
};

__device__ __forceinline__ SoftStats wave_join(SoftStats a) {
    float top = a.m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    a.raise(top);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        a.s += __shfl_xor(a.s, o);
        a.u += __shfl_xor(a.u, o);
    }
    return a;
}

// Order of alternatives: by value, ties by the lowest index (unused places of
// a list hold -infinity and INT_MAX: last).
__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// whole numbers in the order of the values
__device__ __forceinline__ int ordered(float v) {
    const int b = __builtin_bit_cast(int, v);
    return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int b) { return __builtin_bit_cast(float, b >= 0 ? b : b ^ 0x7fffffff); }

__device__ __forceinline__ float lane_value(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// v of the lane before (lane 0: its own)
__device__ __forceinline__ int lane_before(int v) { return __builtin_amdgcn_update_dpp(v, v, 0x138, 0xf, 0xf, false); }

// A wave's most likely values so far, in order, the i-th in lane i (exact for
// the first k; what lies behind them is whatever was pushed out).
struct TopList {
    float v, last_v;  // the lane's, the k-th
    int i, last_i, k;
    __device__ __forceinline__ void clear(int n) {
        v = last_v = neg_inf();
        i = last_i = INT_MAX;
        k = n;
    }
    __device__ __forceinline__ void set_last() {
        last_v = lane_value(v, k - 1);
        last_i = __builtin_amdgcn_readlane(i, k - 1);
    }
    __device__ __forceinline__ bool wants(float w, int j) const { return ahead(w, j, last_v, last_i); }
    // (w, j: the same in every lane)
    __device__ __forceinline__ void insert(float w, int j) {
        const int lane = int(threadIdx.x) % WAVE;
        const int at = __popcll(__ballot(ahead(v, i, w, j)));
        const int pv = lane_before(__builtin_bit_cast(int, v)), pi = lane_before(i);
        v = lane == at ? w : lane > at ? __builtin_bit_cast(float, pv) : v;
        i = lane == at ? j : lane > at ? pi : i;
        set_last();
    }
    // The list of the 64 lanes' own (w, j), sorted (a bitonic network).
    __device__ __forceinline__ void seed(float w, int j) {
        const int lane = int(threadIdx.x) % WAVE;
        v = w;
        i = j;
#pragma unroll
        for (int n = 2; n <= WAVE; n *= 2)
#pragma unroll
            for (int o = n / 2; o >= 1; o /= 2) {
                const float ov = __shfl_xor(v, o);
                const int oi = __shfl_xor(i, o);
                const bool down = (lane & n) == 0, low = (lane & o) == 0;
                if (ahead(ov, oi, v, i) == (down == low)) {  // (equal pairs are both unused: swapped or not is alike)
                    v = ov;
                    i = oi;
                }
            }
        set_last();
    }
};

// 8 logits as loaded, and their values.
template <int TY>
struct Raw8 {
    uint32_t b[TY == 0 ? 8 : 4];
    __device__ __forceinline__ void load(const void *p) {
#pragma unroll
        for (int i = 0; i < (TY == 0 ? 2 : 1); ++i) {
            const uint4 w = static_cast<const uint4 *>(p)[i];
            b[4 * i] = w.x, b[4 * i + 1] = w.y, b[4 * i + 2] = w.z, b[4 * i + 3] = w.w;
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (TY == 0) v[j] = __builtin_bit_cast(float, b[j]);
            else if constexpr (TY == 1) v[j] = __builtin_bit_cast(float, j % 2 ? b[j / 2] & 0xffff0000u : b[j / 2] << 16);
            else v[j] = f16_bits_to_f32(uint16_t(b[j / 2] >> (16 * (j % 2))));
        }
    }
};

// A row as single elements up to the first 16-byte boundary, pieces of 8, and
// single elements behind the last piece.
struct RowCut {
    int head, pieces, tail;
    __device__ __forceinline__ RowCut(const void *row, int bytes, int n) {
        const int per = 16 / bytes, off = int(reinterpret_cast<uintptr_t>(row) / unsigned(bytes) % unsigned(per));
        head = min((per - off) % per, n);
        pieces = (n - head) / 8;
        tail = n - head - 8 * pieces;
    }
};

template <int TY>
__device__ __forceinline__ float logit_at(const void *row, int64_t j) {
    float v[1];
    row_load<TY, 1>(row, j, v);
    return v[0];
}

// What a row's sums say, by one thread.
template <int TY>
__device__ __forceinline__ float finish_row(const LogprobArgs &a, int64_t t, const void *row, SoftStats st) {
    const bool none = st.m == neg_inf() && st.s == 0.f;  // (nothing but masked values)
    const float log_s = logf(st.s), lse = none ? neg_inf() : st.m + log_s;
    const int tok = a.tokens[t];
    float lp = 0.f;
    if (tok >= 0 && tok < a.V) lp = none ? neg_inf() : logit_at<TY>(row, tok) - lse;
    a.logp[t] = lp;
    a.entropy[t] = none ? 0.f : log_s - st.u / st.s;
    a.lse[t] = lse;
    return lse;
}

__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t t, int rank, float v, int i, float lse) {
    const bool bad = lse != lse;
    a.top_i[t * a.top + rank] = bad ? -1 : i;
    a.top_v[t * a.top + rank] = bad ? lse : lse == neg_inf() ? lse : v - lse;
}

// Places of n lists (sorted, k entries each, in LDS) in the order of all:
// put(rank, v, i) for the first k. An entry's rank is its own place and, for
// every other list, how many of that are ahead of it.
template <class Put>
__device__ __forceinline__ void merge_lists(const float *lv, const int *li, int n, int k, Put put) {
    for (int e = int(threadIdx.x); e < n * k; e += int(blockDim.x)) {
        const int own = e / k;
        const float v = lv[e];
        const int i = li[e];
        int rank = e % k;
        for (int q = 0; q < n && rank < k; ++q) {
            if (q == own) continue;
            int lo = 0, hi = k;  // (how many of list q are ahead; unused places go by their list's number)
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const float w = lv[q * k + mid];
                const int j = li[q * k + mid];
                if (ahead(w, j, v, i) || (w == v && j == i && q < own)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < k) put(rank, v, i);
    }
}

// Part `split` of row t by a block of four waves, each taking every fourth
// step of 64 U pieces. TOP: a wave keeps a list of the most likely values; a
// piece is looked at value by value only where its largest would come into the
// list and is not below the last of another wave's.
template <int TY, bool TOP, int U>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
    constexpr int Z = TY == 0 ? 4 : 2;
    __shared__ int s_last;
    __shared__ float s_st[4][3];
    __shared__ float s_lv[TOP ? 4 * WAVE : 1];
    __shared__ int s_li[TOP ? 4 * WAVE : 1];
    const int lane = int(threadIdx.x) % WAVE, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    const int64_t t = int64_t(blockIdx.x) / a.splits;
    const int split = int(blockIdx.x) % a.splits;
    const char *row = static_cast<const char *>(a.logits) + t * a.ld * Z;
    const RowCut cut(row, Z, a.V);
    const char *body = row + int64_t(cut.head) * Z;
    const int steps = (cut.pieces + WAVE * U - 1) / (WAVE * U);
    const int per = (steps + a.splits - 1) / a.splits, first = split * per, end = min(steps, first + per);
    if constexpr (TOP) {
        if (threadIdx.x == 0) s_last = INT_MIN;
        __syncthreads();
    }
    SoftStats st;
    st.clear();
    TopList list;
    list.clear(a.top);
    bool empty = true;

    // the values of one step, `mine` of them in order from index at: into the sums and the list
    auto take = [&](const float (&v)[8], float largest, int at, bool have, int seeded) {
        if constexpr (TOP) {
            const float other = unordered(__hip_atomic_load(&s_last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            auto wanted = [&] { return __ballot(have && list.wants(largest, at) && !(largest < other)); };
            unsigned long long lanes = wanted();
            if (!lanes) return;
            while (lanes) {
                const int l = __builtin_ctzll(lanes);
                float w = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) w = lane == j ? lane_value(v[j], l) : w;
                const int i0 = __builtin_amdgcn_readlane(at, l), skip = __builtin_amdgcn_readlane(seeded, l);
                const int i = i0 + lane;
                unsigned long long which = __ballot(lane < 8 && i != skip && list.wants(w, i));
                while (which) {
                    const int j = __builtin_ctzll(which);
                    which &= which - 1;
                    const float x = lane_value(w, j);
                    if (list.wants(x, i0 + j)) list.insert(x, i0 + j);
                }
                lanes = l == WAVE - 1 ? 0 : wanted() & (~0ull << (l + 1));
            }
            if (lane == 0 && list.last_i != INT_MAX)
                __hip_atomic_fetch_max(&s_last, ordered(list.last_v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
    };

    // (single elements before and behind the pieces: by the first wave)
    if (split == 0 && wave == 0 && cut.head + cut.tail > 0) {
        const int at = lane < cut.head ? lane : cut.head + 8 * cut.pieces + lane - cut.head;
        const bool have = lane < cut.head + cut.tail;
        const float v = have ? logit_at<TY>(row, at) : neg_inf();
        st.add(v, st.raise(v));
        if constexpr (TOP) {
            unsigned long long lanes = __ballot(have);
            while (lanes) {
                const int l = __builtin_ctzll(lanes);
                lanes &= lanes - 1;
                const float x = lane_value(v, l);
                const int i = __builtin_amdgcn_readlane(at, l);
                if (list.wants(x, i)) list.insert(x, i);
            }
        }
    }

    Raw8<TY> raw[U], next[U];
    auto load = [&](int step, Raw8<TY> (&r)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = min((step * U + u) * WAVE + lane, cut.pieces - 1);
            r[u].load(body + int64_t(p) * (8 * Z));
        }
    };
    int step = first + wave;
    if (step < end) load(step, next);
    for (; step < end; step += 4) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = next[u];
        if (step + 4 < end) load(step + 4, next);
        float v[U][8], largest[U], all = neg_inf();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            raw[u].values(v[u]);
            if ((step * U + u) * WAVE + lane >= cut.pieces) {  // (only in a row's last step)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = neg_inf();
            }
            largest[u] = v[u][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) largest[u] = fmaxf(largest[u], v[u][j]);
            all = fmaxf(all, largest[u]);
        }
        const float ref = st.raise(all);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) st.add(v[u][j], ref);
        if constexpr (TOP) {
            int seeded = -1;
            if (empty && list.last_i == INT_MAX && a.top > 1) {
                // the lanes' largest are the list to begin with: few other values of the step come before its k-th
                float w = neg_inf();
                int i = INT_MAX;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int p = (step * U + u) * WAVE + lane, at = cut.head + 8 * p;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (p < cut.pieces && ahead(v[u][j], at + j, w, i)) {
                            w = v[u][j];
                            i = at + j;
                        }
                }
                // (what the row's head and tail put into the list goes in again behind)
                TopList before = list;
                list.seed(w, i);
                seeded = i;
                unsigned long long lanes = __ballot(before.i != INT_MAX);
                while (lanes) {
                    const int l = __builtin_ctzll(lanes);
                    lanes &= lanes - 1;
                    const float x = lane_value(before.v, l);
                    const int j = __builtin_amdgcn_readlane(before.i, l);
                    if (list.wants(x, j)) list.insert(x, j);
                }
            }
            empty = false;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = (step * U + u) * WAVE + lane;
                take(v[u], largest[u], cut.head + 8 * p, p < cut.pieces, seeded);
            }
        }
    }

    st = wave_join(st);
    if (lane == 0) {
        s_st[wave][0] = st.m;
        s_st[wave][1] = st.s;
        s_st[wave][2] = st.u;
    }
    if constexpr (TOP) {
        if (lane < a.top) {
            s_lv[wave * a.top + lane] = list.v;
            s_li[wave * a.top + lane] = list.i;
        }
    }
    __syncthreads();
    st = SoftStats{s_st[0][0], s_st[0][1], s_st[0][2]};
#pragma unroll
    for (int w = 1; w < 4; ++w) st.join(SoftStats{s_st[w][0], s_st[w][1], s_st[w][2]});
    if (a.splits == 1) {
        __shared__ float s_lse;
        if (threadIdx.x == 0) s_lse = finish_row<TY>(a, t, row, st);
        if constexpr (TOP) {
            __syncthreads();
            const float lse = s_lse;
            merge_lists(s_lv, s_li, 4, a.top, [&](int rank, float v, int i) { put_top(a, t, rank, v, i, lse); });
        }
        return;
    }
    const int64_t part = t * a.splits + split;
    if (threadIdx.x == 0) {
        a.part_st[3 * part] = st.m;
        a.part_st[3 * part + 1] = st.s;
        a.part_st[3 * part + 2] = st.u;
    }
    if constexpr (TOP) {
        merge_lists(s_lv, s_li, 4, a.top, [&](int rank, float v, int i) {
            a.part_v[part * a.top + rank] = v;
            a.part_i[part * a.top + rank] = i;
        });
    }
}

constexpr int MAX_SPLITS = 64;

// The parts of a row joined, in order, by a block.
template <int TY>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    extern __shared__ float s_lists[];
    __shared__ float s_lse;
    const int64_t t = blockIdx.x;
    const int n = a.splits * a.top;
    float *lv = s_lists;
    int *li = reinterpret_cast<int *>(s_lists + n);
    for (int e = int(threadIdx.x); e < n; e += 256) {
        lv[e] = a.part_v[t * n + e];
        li[e] = a.part_i[t * n + e];
    }
    if (threadIdx.x < WAVE) {
        SoftStats st;
        st.clear();
        if (int(threadIdx.x) < a.splits) {
            const float *p = a.part_st + 3 * (t * a.splits + int(threadIdx.x));
            st = SoftStats{p[0], p[1], p[2]};
        }
        st = wave_join(st);
        constexpr int Z = TY == 0 ? 4 : 2;
        if (threadIdx.x == 0)
            s_lse = finish_row<TY>(a, t, static_cast<const char *>(a.logits) + t * a.ld * Z, st);
    }
    __syncthreads();
    const float lse = s_lse;
    merge_lists(lv, li, a.splits, a.top, [&](int rank, float v, int i) { put_top(a, t, rank, v, i, lse); });
}

// Pieces of a step by the row count, and parts of a row: enough blocks for the
// chip, at least one step for each wave.
static int logprob_unroll(int T) { return T >= 64 ? 4 : 2; }
int logprob_splits(int T, int V) {
    const int wave = 8 * WAVE * logprob_unroll(T), steps = std::max(1, V / wave);
    return std::max(1, std::min({(2048 + T - 1) / T, (steps + 3) / 4, MAX_SPLITS}));
}

size_t logprobs_workspace_bytes(int T, int V, int top) {
    const int n = logprob_splits(T, V);
    return n == 1 ? 0 : size_t(T) * size_t(n) * (12 + 8 * size_t(top));
}

void launch_logprobs(LogprobArgs a, void *ws, hipStream_t s) {
    a.splits = logprob_splits(a.T, a.V);
    const size_t parts = size_t(a.T) * size_t(a.splits);
    a.part_st = static_cast<float *>(ws);
    a.part_v = a.part_st + 3 * parts;
    a.part_i = reinterpret_cast<int *>(a.part_v + parts * size_t(a.top));
    by_type(a.type, [&](auto ty) {
        constexpr int TY = decltype(ty)::value;
        auto run = [&](auto u) {
            constexpr int U = decltype(u)::value;
            if (a.top) logprobs_kernel<TY, true, U><<<unsigned(parts), 256, 0, s>>>(a);
            else logprobs_kernel<TY, false, U><<<unsigned(parts), 256, 0, s>>>(a);
        };
        if (logprob_unroll(a.T) == 4) run(Int<4>{});
        else run(Int<2>{});
        if (a.splits > 1)
            logprobs_join_kernel<TY><<<unsigned(a.T), 256, size_t(a.splits) * size_t(a.top) * 8, s>>>(a);
    });
}

// ------------------------------------------------------------ gradient
// d of value v, at index i of a row.
struct LogprobRow {
    float lse, g, gh, h;
    int tok;
    bool none;
    __device__ __forceinline__ LogprobRow(const LogprobGradArgs &a, int64_t t) {
        lse = a.lse[t];
        tok = a.tokens[t];
        g = a.dlogp && tok >= 0 && tok < a.V ? a.dlogp[t] : 0.f;
        gh = a.dentropy ? a.dentropy[t] : 0.f;
        h = a.dentropy ? a.entropy[t] : 0.f;
        none = lse == neg_inf();  // (a row of masked values: no gradient)
    }
    __device__ __forceinline__ float value(float v, int i) const {
        const float lp = v - lse, p = exp_fast(lp);
        // p (g + gh (lp + H)), the log bounded where p is 0 (not a NaN)
        const float d = -p * __builtin_fmaf(gh, (lp < NEARLY_NONE ? NEARLY_NONE : lp) + h, g) + (i == tok ? g : 0.f);
        return none ? 0.f : d;
    }
};

// A row in parts of 256 threads with pieces of 8 (V8) or single elements; U
// pieces per thread requested together. Bound by memory: the logits read, the
// gradient written (in the same place, if the caller likes).
template <int TY, bool V8>
__global__ __launch_bounds__(256) void logprobs_backward_kernel(LogprobGradArgs a, int parts) {
    constexpr int Z = TY == 0 ? 4 : 2, U = 4, OT = TY == 2 ? GRAD_F16 : TY;
    const int64_t t = int64_t(blockIdx.x) / parts;
    const int part = int(blockIdx.x) % parts, tid = int(threadIdx.x);
    const LogprobRow r(a, t);
    const char *in = static_cast<const char *>(a.logits) + t * a.ld * Z;
    char *out = static_cast<char *>(a.dlogits) + t * a.ldd * Z;
    auto single = [&](int i) {
        float v[1] = {r.value(logit_at<TY>(in, i), i)};
        row_store<OT, 1>(out, i, v);
    };
    if constexpr (V8) {
        const RowCut cut(in, Z, a.V);
        const char *bi = in + int64_t(cut.head) * Z;
        for (int64_t p0 = int64_t(part) * (256 * U) + tid; p0 < cut.pieces; p0 += int64_t(parts) * (256 * U)) {
            Raw8<TY> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p0 + 256 * u < cut.pieces) raw[u].load(bi + (p0 + 256 * u) * (8 * Z));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t p = p0 + 256 * u;
                if (p >= cut.pieces) continue;
                const int i = cut.head + 8 * int(p);
                float v[8];
                raw[u].values(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = r.value(v[j], i + j);
                row_store<OT, 8>(out, i, v);
            }
        }
        if (part == 0 && tid < cut.head + cut.tail) single(tid < cut.head ? tid : 8 * cut.pieces + tid);
    } else {
        for (int64_t i = int64_t(part) * 256 + tid; i < a.V; i += int64_t(parts) * 256) single(int(i));
    }
}

void launch_logprobs_backward(const LogprobGradArgs &a, hipStream_t s) {
    by_type(a.type, [&](auto ty) {
        constexpr int TY = decltype(ty)::value, Z = TY == 0 ? 4 : 2;
        // (pieces of 8 start on 16 bytes in both rows, or in neither)
        const bool same = (reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.dlogits)) % 16 == 0 &&
                          (a.T == 1 || (a.ld - a.ldd) * Z % 16 == 0);
        const int per = same ? 8 * 4 * 256 : 8 * 256;
        // (a grid holds less than 2^32 threads)
        const int parts = std::max(1, std::min((a.V + per - 1) / per, (1 << 23) / a.T));
        const unsigned blocks = unsigned(a.T) * unsigned(parts);
        if (same) logprobs_backward_kernel<TY, true><<<blocks, 256, 0, s>>>(a, parts);
        else logprobs_backward_kernel<TY, false><<<blocks, 256, 0, s>>>(a, parts);
    });
}

}  // namespace qwq4
