// Log probabilities of given tokens, the entropy and the most likely tokens of
// rows of logits, and the gradient of the first two.
//
//   lse = log sum_j exp(l_j),  logp = l_tok - lse,  H = lse - sum_j p_j l_j
//   dl_j = dlogp ([j = tok] - p_j) - dH p_j (log p_j + H),   p_j = exp(l_j - lse)
//
// One pass over the row: each lane keeps the largest value m so far,
// S = sum exp(l - m) and U = sum exp(l - m) (l - m), rescaled when m grows;
// then lse = m + log S, logp = (l_tok - m) - log S and H = log S - U / S. A masked logit
// (-infinity) adds nothing to either sum. A row that masks everything has lse and logp of
// -infinity and entropy 0; one with a NaN or +infinity gives NaN.
#include <algorithm>
#include <climits>

#include "q4_kernels.hpp"
#include "row_io.cuh"

namespace qwq4 {

constexpr float LOG2E = 1.44269504088896341f;
// exp(x - y) of sums: below this nothing is left in fp32
constexpr float NEARLY_NONE = -200.f;

// (the product with log2 e is rounded: 2^-24 |d| of the result beside the exponential's own)
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
    // The values of one step, summed among themselves first: next to a likely
    // token each of the others alone is too small to change the sum so far, all
    // of them are not. (The difference is bounded where it is a factor: 0 times
    // a masked value's would be a NaN.)
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N][8], float ref) {
        float ps[4] = {}, pu[4] = {};
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = v[n][j] - ref, e = exp_fast(d);
                ps[j % 4] += e;
                pu[j % 4] = __builtin_fmaf(e, fmaxf(d, NEARLY_NONE), pu[j % 4]);
            }
        s += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        u += (pu[0] + pu[1]) + (pu[2] + pu[3]);
    }
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
// (Without branches: they would make every comparison wait for the one before.)
__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return (v > w) | ((v == w) & (i < j)); }

// whole numbers in the order of the values
__device__ __forceinline__ int ordered(float v) {
    const int b = __builtin_bit_cast(int, v);
    return b >= 0 ? b : b ^ 0x7fffffff;
}
__device__ __forceinline__ float unordered(int b) { return __builtin_bit_cast(float, b >= 0 ? b : b ^ 0x7fffffff); }

// The same order in one number (both zeros are one value): 0 is an unused
// place, behind every value; a NaN has none.
typedef unsigned long long TopKey;
__device__ __forceinline__ TopKey top_key(float v, int i) {
    const TopKey high = uint32_t(ordered(v + 0.f)) ^ 0x80000000u;
    return i == INT_MAX || v != v ? 0 : high << 32 | uint32_t(~i);
}
__device__ __forceinline__ float key_value(TopKey k) { return unordered(int(uint32_t(k >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int key_index(TopKey k) { return int(~uint32_t(k)); }

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

// The log probability of value v is (v - m) - log S: both differences are small and
// exact to their own last bit, where lse = m + log S is rounded to a step of m (a row
// whose values are all -1e9 would have lost log S).
struct RowLog {
    float m, log_s;  // -infinity both: nothing but masked values; log_s NaN: a NaN or +infinity among the values
    __device__ __forceinline__ float of(float v) const { return log_s == neg_inf() ? log_s : (v - m) - log_s; }
};

// What a row's sums say, by one thread.
template <int TY>
__device__ __forceinline__ RowLog finish_row(const LogprobArgs &a, int64_t t, const void *row, SoftStats st) {
    const bool none = st.m == neg_inf() && st.s == 0.f;  // (nothing but masked values)
    const RowLog r{st.m, logf(st.s)};
    const int tok = a.tokens[t];
    a.logp[t] = tok >= 0 && tok < a.V ? r.of(logit_at<TY>(row, tok)) : 0.f;
    a.entropy[t] = none ? 0.f : r.log_s - st.u / st.s;
    a.lse[t] = none ? neg_inf() : r.m + r.log_s;
    return r;
}

__device__ __forceinline__ void put_top(const LogprobArgs &a, int64_t t, int rank, TopKey key, RowLog r) {
    const bool bad = r.log_s != r.log_s;
    a.top_i[t * a.top + rank] = bad ? -1 : key_index(key);
    a.top_v[t * a.top + rank] = bad ? r.log_s : r.of(key_value(key));
}

// put(rank, key) for the first k of n keys in LDS, none alike (0 for the places
// behind the n-th): a key's rank is how many are ahead of it. Every comparison
// is independent of the others, where a search or a sorted list would wait.
template <class Put>
__device__ __forceinline__ void rank_keys(const TopKey *keys, int n, int k, Put put) {
    for (int e = int(threadIdx.x); e < n; e += int(blockDim.x)) {
        const TopKey own = keys[e];
        int rank = 0;
#pragma unroll 16
        for (int c = 0; c < n; ++c) rank += int(keys[c] > own);
        if (rank < k) put(rank, own);
    }
    for (int e = n + int(threadIdx.x); e < k; e += int(blockDim.x)) put(e, TopKey(0));
}

// Part `split` of row t by a block of four waves, each taking every fourth
// step of 64 U pieces. TOP: the largest value of each lane's step is left in LDS
// on the way. The lanes make 64 groups (a lane of each wave; 256, the lanes alone, for
// k > 32: of 64 groups as many as k are hardly a bound, 4096 rows of 151936 and k = 64
// 387 us for 248); the k-th of the groups' largest has k values at or above it, and
// only steps whose largest is not below it are read a second time: of such a row and
// k = 5, some 6 of 4736, from which some 5 values go to the list that is ranked. (A
// sorted list per wave kept up to date on the way: 5 alternatives 45 us more in 4096
// rows, 20 alternatives 130. Each lane reading its own steps again, one after the
// other: 13 and 38 more, and 200 rows 41 us for 25.) Where more than the list takes
// are left (rows with thousands of equal values, fewer than k unmasked ones), the
// part is read again into sorted lists. Bound by memory: 4096 rows 224 us, 5.6 TB/s.
constexpr int MAX_SPLITS = 64;  // parts of a row at most
constexpr int TOP_SLOTS = 32, TOP_LIST = 512;
template <int TY, bool TOP, int U>
__global__ __launch_bounds__(256) void logprobs_kernel(LogprobArgs a) {
    constexpr int Z = TY == 0 ? 4 : 2;
    extern __shared__ float s_max[];  // TOP: [slots][256]
    __shared__ int s_n, s_again;
    __shared__ uint16_t s_slots[TOP ? TOP_LIST : 1];
    __shared__ float s_st[4][3], s_bound;
    __shared__ RowLog s_log;
    __shared__ __align__(16) float s_lane[TOP ? 256 : 1];
    __shared__ TopKey s_keys[TOP ? TOP_LIST : 1];
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int64_t t = int64_t(blockIdx.x) / a.splits;
    const int split = int(blockIdx.x) % a.splits;
    const char *row = static_cast<const char *>(a.logits) + t * a.ld * Z;
    const RowCut cut(row, Z, a.V);
    const char *body = row + int64_t(cut.head) * Z;
    const int steps = (cut.pieces + WAVE * U - 1) / (WAVE * U);
    const int per = (steps + a.splits - 1) / a.splits, first = split * per, end = min(steps, first + per);
    if (TOP && tid == 0) s_n = s_again = 0;
    // (single elements before and behind the pieces: one each by the first lanes)
    const int alone = tid < cut.head ? tid : 8 * cut.pieces + tid;
    const bool has_alone = split == 0 && tid < cut.head + cut.tail;
    const float extra = has_alone ? logit_at<TY>(row, alone) : neg_inf();
    SoftStats st;
    st.clear();
    st.add(extra, st.raise(extra));

    auto load = [&](int step, Raw8<TY> (&r)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = min((step * U + u) * WAVE + lane, cut.pieces - 1);
            r[u].load(body + int64_t(p) * (8 * Z));
        }
    };
    // a step's values, -infinity behind the last piece (only in a row's last step)
    auto values = [&](int step, const Raw8<TY> (&r)[U], float (&v)[U][8]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            r[u].values(v[u]);
            if ((step * U + u) * WAVE + lane >= cut.pieces) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = neg_inf();
            }
        }
    };
    Raw8<TY> raw[U], next[U];
    float slot_max = neg_inf();
    int slot = 0, in_slot = 0;
    int step = first + wave;
    if (step < end) load(step, next);
    for (; step < end; step += 4) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = next[u];
        if (step + 4 < end) load(step + 4, next);
        float v[U][8], largest = neg_inf();
        values(step, raw, v);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) largest = fmaxf(largest, v[u][j]);
        const float ref = st.raise(largest);
        st.add(v, ref);
        if constexpr (TOP) {
            slot_max = fmaxf(slot_max, largest);
            if (++in_slot == a.slot_steps) {
                s_max[slot * 256 + tid] = slot_max;
                ++slot;
                in_slot = 0;
                slot_max = neg_inf();
            }
        }
    }
    if constexpr (TOP) {
        if (in_slot) s_max[slot++ * 256 + tid] = slot_max;
        s_lane[tid] = st.m;
    }
    st = wave_join(st);
    if (lane == 0) {
        s_st[wave][0] = st.m;
        s_st[wave][1] = st.s;
        s_st[wave][2] = st.u;
    }
    __syncthreads();
    if (!TOP || wave == 3) {
        st = SoftStats{s_st[0][0], s_st[0][1], s_st[0][2]};
#pragma unroll
        for (int w = 1; w < 4; ++w) st.join(SoftStats{s_st[w][0], s_st[w][1], s_st[w][2]});
        if (tid == (TOP ? 3 * WAVE : 0)) {
            if (a.splits == 1) {
                s_log = finish_row<TY>(a, t, row, st);
            } else {
                float *p = a.part_st + 3 * (t * a.splits + split);
                p[0] = st.m;
                p[1] = st.s;
                p[2] = st.u;
            }
        }
    }
    if constexpr (!TOP) return;

    if (a.top > WAVE / 2) {
        const float own = s_lane[tid];
        int rank = 0;
#pragma unroll 4
        for (int l = 0; l < 256; l += 4) {
            const float4 other = *reinterpret_cast<const float4 *>(&s_lane[l]);
            rank += int((other.x > own) | ((other.x == own) & (l < tid)));
            rank += int((other.y > own) | ((other.y == own) & (l + 1 < tid)));
            rank += int((other.z > own) | ((other.z == own) & (l + 2 < tid)));
            rank += int((other.w > own) | ((other.w == own) & (l + 3 < tid)));
        }
        if (rank == a.top - 1) s_bound = own;
    } else if (wave == 0) {
        const float own = fmaxf(fmaxf(s_lane[lane], s_lane[lane + 64]), fmaxf(s_lane[lane + 128], s_lane[lane + 192]));
        int rank = 0;
#pragma unroll 16
        for (int l = 0; l < WAVE; ++l) {
            const float other = lane_value(own, l);
            rank += int((other > own) | ((other == own) & (l < lane)));
        }
        if (rank == a.top - 1) s_bound = own;
    }
    __syncthreads();
    const float bound = s_bound;
    auto keep = [&](float x, int at) {
        if (!(x >= bound)) return;
        const int n = atomicAdd(&s_n, 1);
        if (n < TOP_LIST) s_keys[n] = top_key(x, at);
    };
    if (has_alone) keep(extra, alone);
    // (listed before they are read again, a piece a thread: all of them are asked for at once)
#pragma unroll 4
    for (int k = 0; k < slot; ++k) {
        if (!(s_max[k * 256 + tid] >= bound)) continue;
        const int i = atomicAdd(&s_again, 1);
        if (i < TOP_LIST) s_slots[i] = uint16_t(k * 256 + tid);
    }
    __syncthreads();
    const int each = a.slot_steps * U;  // pieces of a slot
    for (int i = tid; i < min(s_again, TOP_LIST) * each; i += 256) {
        const int at = s_slots[i / each], c = i % each / U, u = i % U;
        const int again = first + at % 256 / WAVE + 4 * (at / 256 * a.slot_steps + c);
        const int p = (again * U + u) * WAVE + at % WAVE;
        if (again >= end || p >= cut.pieces) continue;
        Raw8<TY> piece;
        piece.load(body + int64_t(p) * (8 * Z));
        float v[8];
        piece.values(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) keep(v[j], cut.head + 8 * p + j);
    }
    __syncthreads();
    int n = s_n;
    if (max(n, s_again) > TOP_LIST) {
        TopList list;
        list.clear(a.top);
        auto take = [&](float w, int i, bool have) {
            unsigned long long which = __ballot(have && list.wants(w, i));
            while (which) {
                const int l = __builtin_ctzll(which);
                which &= which - 1;
                const float x = lane_value(w, l);
                const int j = __builtin_amdgcn_readlane(i, l);
                if (list.wants(x, j)) list.insert(x, j);
            }
        };
        take(extra, alone, has_alone);
        for (int again = first + wave; again < end; again += 4) {
            load(again, raw);
            float v[U][8];
            values(again, raw, v);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = (again * U + u) * WAVE + lane;
#pragma unroll
                for (int j = 0; j < 8; ++j) take(v[u][j], cut.head + 8 * p + j, p < cut.pieces);
            }
        }
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
        const bool used = lane < a.top && list.i != INT_MAX;  // (the first so many places)
        const int places = __popcll(__ballot(used));
        int base = 0;
        if (lane == 0) base = atomicAdd(&s_n, places);
        base = __builtin_amdgcn_readlane(base, 0);
        if (used) s_keys[base + lane] = top_key(list.v, list.i);
        __syncthreads();
        n = s_n;
    }
    const RowLog log = a.splits == 1 ? s_log : RowLog{0.f, 0.f};
    const int64_t part = t * a.splits + split;
    rank_keys(s_keys, n, a.top, [&](int rank, TopKey key) {
        if (a.splits == 1) put_top(a, t, rank, key, log);
        else a.part_key[part * a.top + rank] = key;
    });
}

// The parts of a row joined, in order, by a block. With j the least such that
// the parts' first j keys are k or more, the ceil(k / j)-th of the parts' j-th
// keys has k keys at or ahead of it: what is behind it is left out, and the rest
// ranked. (Of 19 parts of 20 keys each some 30 are left, and most if only the
// parts' last keys are gone by.)
template <int TY>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogprobArgs a) {
    __shared__ TopKey s_last, s_keys[MAX_SPLITS * WAVE];
    __shared__ int s_n;
    __shared__ RowLog s_log;
    const int tid = int(threadIdx.x), n = a.splits * a.top;
    const int64_t t = blockIdx.x;
    const TopKey *parts = a.part_key + t * n;
    const int j = (a.top + a.splits - 1) / a.splits, m = j ? (a.top + j - 1) / j : 0;
    if (tid == 0) {
        s_last = 1;
        s_n = 0;
    }
    if (a.top && tid < WAVE) s_keys[tid] = tid < a.splits ? parts[tid * a.top + j - 1] : 0;
    __syncthreads();
    if (a.top && tid < WAVE) {
        const TopKey own = s_keys[tid];
        int rank = 0;
#pragma unroll 16
        for (int l = 0; l < WAVE; ++l) rank += int(s_keys[l] > own);
        if (rank == m - 1 && own) s_last = own;  // (keys differ: one lane)
    }
    if (tid >= 192) {
        const int lane = tid - 192;
        SoftStats st;
        st.clear();
        if (lane < a.splits) {
            const float *p = a.part_st + 3 * (t * a.splits + lane);
            st = SoftStats{p[0], p[1], p[2]};
        }
        st = wave_join(st);
        constexpr int Z = TY == 0 ? 4 : 2;
        if (lane == 0) s_log = finish_row<TY>(a, t, static_cast<const char *>(a.logits) + t * a.ld * Z, st);
    }
    if (!a.top) return;
    __syncthreads();
    const TopKey last = s_last;
    for (int e = tid; e < n; e += 256) {
        const TopKey key = parts[e];
        if (key >= last) s_keys[atomicAdd(&s_n, 1)] = key;
    }
    __syncthreads();
    const RowLog log = s_log;
    rank_keys(s_keys, s_n, a.top, [&](int rank, TopKey key) { put_top(a, t, rank, key, log); });
}

// A block takes a row, or a part of it while there are too few blocks for the
// chip, with at least a step for each wave: two blocks a CU (eight: every block
// has a tail in which it looks for its alternatives, and there are rows to join:
// 1000 rows of 50257 and 5 alternatives 34 us for 25, of 151936 68 for 63).
constexpr int LOGPROB_U = 4;
static int logprob_splits(int T, int V) {
    const int steps = std::max(1, V / (8 * WAVE * LOGPROB_U));
    return std::max(1, std::min({(512 + T - 1) / T, (steps + 3) / 4, MAX_SPLITS}));
}

size_t logprobs_workspace_bytes(int T, int V, int top) {
    const int n = logprob_splits(T, V);
    return n == 1 ? 0 : size_t(T) * size_t(n) * (12 + 8 * size_t(top));
}

void launch_logprobs(LogprobArgs a, void *ws, hipStream_t s) {
    a.splits = logprob_splits(a.T, a.V);
    const size_t parts = size_t(a.T) * size_t(a.splits);
    a.part_key = static_cast<unsigned long long *>(ws);
    a.part_st = reinterpret_cast<float *>(a.part_key + parts * size_t(a.top));
    by_type(a.type, [&](auto ty) {
        constexpr int TY = decltype(ty)::value;
        // (a wave's steps at most; a row's cut can only make them fewer)
        const int steps = (a.V / 8 + WAVE * LOGPROB_U - 1) / (WAVE * LOGPROB_U);
        const int wave = ((steps + a.splits - 1) / a.splits + 3) / 4;
        a.slot_steps = std::max(1, (wave + TOP_SLOTS - 1) / TOP_SLOTS);
        const size_t lds = size_t((wave + a.slot_steps - 1) / a.slot_steps) * 1024;
        if (a.top) logprobs_kernel<TY, true, LOGPROB_U><<<unsigned(parts), 256, lds, s>>>(a);
        else logprobs_kernel<TY, false, LOGPROB_U><<<unsigned(parts), 256, 0, s>>>(a);
        if (a.splits > 1) logprobs_join_kernel<TY><<<unsigned(a.T), 256, 0, s>>>(a);
    });
}

// ------------------------------------------------------------ gradient
// lse is given rounded, and p = exp(l - lse) is off by as much: by half a step of it,
// 2^-24 |lse|. Rows whose |lse| is above this (half a step of 2^-19 in fp32 rows, 2^-15
// in 16-bit ones, next to half a step of 2^-24 and 2^-11 of what is written) have their
// sum of p made first, and its log taken off too.
template <int TY>
constexpr float FAR_ROW = TY == 0 ? 64.f : 1024.f;

// d of value v, at index i of a row.
struct LogprobRow {
    float lse, g, gh, h;
    float power;  // of two that p is off by
    int tok;
    bool none;
    __device__ __forceinline__ LogprobRow(const LogprobGradArgs &a, int64_t t) {
        lse = a.lse[t];
        power = 0.f;
        tok = a.tokens[t];
        g = a.dlogp && tok >= 0 && tok < a.V ? a.dlogp[t] : 0.f;
        gh = a.dentropy ? a.dentropy[t] : 0.f;
        h = a.dentropy ? a.entropy[t] : 0.f;
        none = lse == neg_inf();  // (a row of masked values: no gradient)
    }
    // What rounding took from lse, from the row's sum of exp(l - lse): a step of it at most,
    // or the sum is not one that lse is of (a part of a longer row's values).
    __device__ __forceinline__ void put_right(float sum) {
        const float rest = logf(sum);
        if (!(fabsf(rest) <= 0x1p-23f * fabsf(lse))) return;
        power = -rest * LOG2E;
        h -= rest;
    }
    __device__ __forceinline__ float value(float v, int i) const {
        const float lp = v - lse, p = __builtin_amdgcn_exp2f(__builtin_fmaf(lp, LOG2E, power));
        // p (g + gh (lp + H)), the log bounded where p is 0 (not a NaN)
        const float d = -p * __builtin_fmaf(gh, (lp < NEARLY_NONE ? NEARLY_NONE : lp) + h, g) + (i == tok ? g : 0.f);
        return none ? 0.f : d;
    }
};

// A row in parts of 256 threads with pieces of 8 (V8) or single elements; U
// pieces per thread requested together. Bound by memory: the logits read, the
// gradient written (in the same place, if the caller likes): 601 bf16 rows of 151936 65
// us. A row far from zero is read twice, by one block alone, since the gradient may lie on
// it (601 such rows 173 us, one 52 us for 4.5; 2100 fp32 rows of 32000 167 us for 101, and
// 376 where that block was each row's first and came to two of the XCDs).
template <int TY, bool V8>
__global__ __launch_bounds__(256) void logprobs_backward_kernel(LogprobGradArgs a, int parts) {
    constexpr int Z = TY == 0 ? 4 : 2, U = 4, OT = TY == 2 ? GRAD_F16 : TY;
    const int64_t t = int64_t(blockIdx.x) / parts;
    int part = int(blockIdx.x) % parts;
    const int tid = int(threadIdx.x);
    LogprobRow r(a, t);
    const char *in = static_cast<const char *>(a.logits) + t * a.ld * Z;
    char *out = static_cast<char *>(a.dlogits) + t * a.ldd * Z;
    const RowCut cut(in, Z, a.V);
    const char *body = in + int64_t(cut.head) * Z;
    Raw8<TY> raw[U];
    auto load = [&](int64_t p0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p0 + 256 * u < cut.pieces) raw[u].load(body + (p0 + 256 * u) * (8 * Z));
    };
    int64_t p0 = int64_t(part) * (256 * U) + tid;
    if constexpr (V8) load(p0);  // (asked for beside lse: behind it, 601 rows of 151936 80 us for 66)
    const bool far = fabsf(r.lse) > FAR_ROW<TY> && fabsf(r.lse) < __builtin_huge_valf();
    const bool alone = tid < cut.head + cut.tail;
    const int at = tid < cut.head ? tid : 8 * cut.pieces + tid;  // the thread's single element
    if (far) {
        if (part != (t + t / 8) % parts) return;  // (another part from row to row: all XCDs have a share)
        part = 0;
        parts = 1;
        __shared__ float s_sum[4];
        float sum = alone ? exp_fast(logit_at<TY>(in, at) - r.lse) : 0.f;
        for (int64_t p = tid; p < cut.pieces; p += 256 * U) {
            load(p);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p + 256 * u >= cut.pieces) continue;
                float v[8];
                raw[u].values(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = exp_fast(v[j] - r.lse);
                sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
            }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
        if (tid % WAVE == 0) s_sum[tid / WAVE] = sum;
        __syncthreads();  // (and nothing of the row is overwritten before all of it is read)
        r.put_right((s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
        p0 = tid;
        if constexpr (V8) load(p0);
    }
    auto single = [&](int i) {
        float v[1] = {r.value(logit_at<TY>(in, i), i)};
        row_store<OT, 1>(out, i, v);
    };
    if constexpr (V8) {
        while (p0 < cut.pieces) {
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
            p0 += int64_t(parts) * (256 * U);
            load(p0);
        }
        if (alone && part == 0) single(at);
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
