// Log probabilities of given tokens under rows of logits, the rows' entropies and their k likeliest tokens, one pass over
// the logits.  For a row z with reference m (its maximum when the pass ends):
//   S = sum exp(z - m),  T = sum exp(z - m) (m - z):   log p(t) = (z_t - m) - log S,   entropy = log S + T / S
// (every term of T is >= 0, so the entropy loses nothing by cancellation; natural units).  S, T and m are float32; over long rows
// S and T are summed with compensation.
// Partial results over different references join by f = exp(m' - m): S = S + f S', T = T + f (T' + (m - m') S').
//
// What is masked: -inf has probability 0 and is never among the likeliest (id -1, log p -inf where fewer than k tokens
// remain); a row that allows nothing gives log p = -inf, entropy 0; the lowest finite value is a value like any other.
// A NaN or +inf anywhere makes S NaN, and the row's results NaN with ids -1.
// Ties go to the lower index: candidates are ranked by (value, index), never by the order in which they were found.
//
// Bandwidth-bound for rows that number in the hundreds (2 or 4 bytes per logit against about ten issue slots), bound by
// latency below.  Rows up to 1024 tokens stay in the registers of a group of lanes; longer ones are streamed by a
// work-group each, or by several where rows are few, whose results a second launch joins.
#include "oasr_common.h"

namespace oasr {
namespace scores {

constexpr float kLowest = -3.402823466e38f;       // the lowest finite float32
constexpr float kLargest = 3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 64;
constexpr int kShort = 1024;                      // tokens that a wave holds in registers
constexpr int kCandidates = 512;                  // kept in LDS per row before ranking

struct Args {
    const void* logits;
    int64_t ld, rows;           // rows of results
    int vocab, given, top;
    const int32_t* tokens;      // [rows][given]
    const int32_t* frames;      // null: result row r reads logits row r; else row (r / width) * frames_per + frames[r]
    int64_t width, frames_per;
    float* logprobs;            // [rows][given]
    float* entropy;             // [rows]
    int32_t* ids;               // [rows][top]
    float* best;                // [rows][top]
    int splits;                 // work-groups per row
    float* part;                // [rows][splits][4]: m, S, T
    uint2* cand;                // [rows][splits][top]: (ordered value, index), best first
};

// The order of float values as the order of unsigned integers; -0 equals 0.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t b = __float_as_uint(f + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t kOrderedLowest = 0x00800000u;  // ordered(kLowest): -inf lies below

__device__ __forceinline__ bool before(uint32_t va, uint32_t ia, uint32_t vb, uint32_t ib) { return va > vb || (va == vb && ia < ib); }

// Reductions over aligned groups of lanes without LDS: neighbours by data-parallel moves inside a row of 16 lanes (the mirrored
// partner serves as well as the exclusive-or one, since its four or eight lanes agree by then), rows by lane swaps.  `op` takes
// two values of any struct of 32-bit words and must be symmetric.  Every lane ends with the group's result.
template <int CTRL, typename T>
__device__ __forceinline__ T lane_move(const T& v) {
    constexpr int N = sizeof(T) / 4;
    int w[N];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], CTRL, 0xf, 0xf, true);
    T r;
    __builtin_memcpy(&r, w, sizeof(T));
    return r;
}
template <bool HALVES, typename T>
__device__ __forceinline__ void lane_swap(const T& v, T& a, T& b) {     // rows 0 1 2 3 -> a: 0 0 2 2, b: 1 1 3 3 (halves alike)
    constexpr int N = sizeof(T) / 4;
    unsigned w[N], wa[N], wb[N];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const auto p = HALVES ? __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false)
                              : __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);
        wa[i] = p[0];
        wb[i] = p[1];
    }
    __builtin_memcpy(&a, wa, sizeof(T));
    __builtin_memcpy(&b, wb, sizeof(T));
}
template <typename T, typename Op>
__device__ __forceinline__ T group_reduce(T v, int lanes, Op op) {      // lanes: 1, 2, 4 .. 64, uniform
    if (lanes > 1) v = op(v, lane_move<0xB1>(v));       // quad_perm [1 0 3 2]
    if (lanes > 2) v = op(v, lane_move<0x4E>(v));       // quad_perm [2 3 0 1]
    if (lanes > 4) v = op(v, lane_move<0x141>(v));      // row_half_mirror
    if (lanes > 8) v = op(v, lane_move<0x140>(v));      // row_mirror
    T a, b;
    if (lanes > 16) {
        lane_swap<false>(v, a, b);
        v = op(a, b);
    }
    if (lanes > 32) {
        lane_swap<true>(v, a, b);
        v = op(a, b);
    }
    return v;
}
struct Pick {
    uint32_t value, index;      // ordered value; the lower index wins a tie
};
__device__ __forceinline__ Pick better(const Pick& a, const Pick& b) { return before(b.value, b.index, a.value, a.index) ? b : a; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }
__device__ __forceinline__ uint32_t larger_word(uint32_t a, uint32_t b) { return a > b ? a : b; }

// 16 bytes of logits from any element's address.
template <typename E>
struct Chunk;
template <>
struct Chunk<float> {
    static constexpr int N = 4;
    struct __attribute__((packed, aligned(4))) Raw {
        float v[4];
    };
    static __device__ __forceinline__ void load(const float* p, float (&z)[4]) {
        const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = r.v[e];
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct Chunk<uint16_t> {
    static constexpr int N = 8;
    struct __attribute__((packed, aligned(2))) Raw {
        uint32_t v[4];
    };
    static __device__ __forceinline__ void load(const uint16_t* p, float (&z)[8]) {
        const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            z[2 * e] = __uint_as_float(r.v[e] << 16);
            z[2 * e + 1] = __uint_as_float(r.v[e] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ float one(const uint16_t* p) { return bf2f(*p); }
};

// Where result row r reads its logits: >= 0 the logits row, -1 absent (no token here), -2 a frame that does not exist.
__device__ __forceinline__ int64_t source_row(const Args& p, int64_t r) {
    if (!p.frames) return r;
    const int32_t f = p.frames[r];
    if (p.tokens[r] < 0 || f < 0) return -1;
    return f < p.frames_per ? r / p.width * p.frames_per + f : -2;
}

__device__ __forceinline__ float nan32() { return __uint_as_float(0x7fc00000u); }

// One given token's log probability.
template <typename E>
__device__ __forceinline__ float token_logprob(const E* row, int vocab, int32_t token, float m, float s, float log_s) {
    if (token < 0) return 0.f;                        // no token given here
    if (token >= vocab || s != s) return nan32();
    if (s == 0.f) return -INFINITY;
    return (Chunk<E>::one(row + token) - m) - log_s;
}

__device__ __forceinline__ float row_entropy(float s, float t, float log_s) { return s == 0.f ? 0.f : log_s + t / s; }

// One of the likeliest: rank `at` of row r.
__device__ __forceinline__ void write_best(const Args& p, int64_t r, int at, uint32_t value, uint32_t index, float m, float log_s) {
    p.ids[r * p.top + at] = (int32_t)index;
    p.best[r * p.top + at] = (unordered(value) - m) - log_s;
}
__device__ __forceinline__ void write_none(const Args& p, int64_t r, int at, float value) {
    p.ids[r * p.top + at] = -1;
    p.best[r * p.top + at] = value;
}

// A value that at least `count` lanes of the wave reach, and as few more as the ties of the count-th largest make.
__device__ __forceinline__ uint32_t wave_nth_largest(uint32_t v, int count) {
    uint32_t at = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = at | 1u << bit;
        const int reach = __popcll(__ballot(v >= trial));
        if (reach >= count) at = trial;
        if (reach == count) break;
    }
    return at;
}

// Orders a wave's own LDS writes before its reads of them.
#define OASR_SCORES_WAVE_LDS()                                          \
    do {                                                                \
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local"); \
        __builtin_amdgcn_wave_barrier();                                \
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local"); \
    } while (0)

// ---- short rows: a group of 2^g lanes holds a row in registers, C chunks of four per lane -----------------------------
// Four consecutive values, of which the first `left` exist (the rest -inf).
template <typename E>
__device__ __forceinline__ void load_four(const E* p, int left, float (&z)[4]);
template <>
__device__ __forceinline__ void load_four<float>(const float* p, int left, float (&z)[4]) {
    if (left >= 4) {
        Chunk<float>::load(p, z);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = e < left ? p[e] : -INFINITY;
    }
}
template <>
__device__ __forceinline__ void load_four<uint16_t>(const uint16_t* p, int left, float (&z)[4]) {
    struct __attribute__((packed, aligned(2))) Raw {
        uint32_t v[2];
    };
    if (left >= 4) {
        const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            z[2 * e] = __uint_as_float(r.v[e] << 16);
            z[2 * e + 1] = __uint_as_float(r.v[e] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = e < left ? bf2f(p[e]) : -INFINITY;
    }
}

template <typename E, int C>
__global__ __launch_bounds__(256) void token_scores_short_kernel(const Args p, int lanes_log2) {
    constexpr int kList = C > 1 ? 64 : 1;             // candidates of a wave's row, where a row takes the whole wave
    __shared__ Pick lists[4][kList];
    const int lane = threadIdx.x & 63, group = C > 1 ? 64 : 1 << lanes_log2, sub = lane & (group - 1);
    const int wave_in = threadIdx.x >> 6;
    const int64_t wave = (int64_t)blockIdx.x * 4 + wave_in;
    const int64_t r = C > 1 ? wave : (wave << (6 - lanes_log2)) + (lane >> lanes_log2);
    const bool live = r < p.rows;
    const int64_t src = live ? source_row(p, r) : -1;
    const E* row = reinterpret_cast<const E*>(p.logits) + (src < 0 ? 0 : src) * p.ld;
    float z[4 * C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = 4 * (sub + c * group);
        float four[4];
        load_four<E>(row + at, src >= 0 ? p.vocab - at : 0, four);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[4 * c + e] = four[e];
    }
    float own = z[0];
#pragma unroll
    for (int j = 1; j < 4 * C; ++j) own = fmaxf(own, z[j]);
    const float m = group_reduce(fmaxf(own, kLowest), group, larger);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < 4 * C; ++j) {
        const float x = m - z[j], e = __builtin_amdgcn_exp2f(x * -kLog2e);      // NaN for NaN, and for +inf against itself
        s += e;
        t = fmaf(e, fminf(x, kLargest), t);
    }
    s = group_reduce(s, group, sum_of);
    t = group_reduce(t, group, sum_of);
    const float log_s = logf(s);
    if (live && p.given > 0)
        for (int i = sub; i < p.given; i += group) {
            float v = 0.f;
            if (src >= 0) v = token_logprob(row, p.vocab, p.tokens[r * p.given + i], m, s, log_s);
            if (src == -2) v = nan32();
            p.logprobs[r * p.given + i] = v;
        }
    if (live && p.entropy && sub == 0) p.entropy[r] = src >= 0 ? row_entropy(s, t, log_s) : (src == -2 ? nan32() : 0.f);
    if (p.top == 0) return;
    const bool usable = src >= 0 && s == s;
    const float absent = src == -1 || usable ? -INFINITY : nan32();
    if (C == 1) {
        // several rows per wave: one round per alternative.  The group's largest value is a reduction of one word, the first lane
        // that holds it wins - a lane's four tokens are neighbours, so that is the lowest index - writes it and drops it.  (Values
        // reduced together with their indices: 100000 x 100 with 5 alternatives 43 us, this way 31.)
        const uint64_t mates = (group == 64 ? ~0ull : (1ull << group) - 1) << (lane - sub);
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = usable && ordered(z[j]) >= kOrderedLowest ? ordered(z[j]) : 0;
        for (int k = 0; k < p.top; ++k) {
            const uint32_t mine = max(max(u[0], u[1]), max(u[2], u[3]));
            const uint32_t best = group_reduce(mine, group, larger_word);
            if (lane == __builtin_ctzll(__ballot(mine == best) & mates)) {
                const int at = u[0] == best ? 0 : u[1] == best ? 1 : u[2] == best ? 2 : 3;
                if (live) {
                    if (best) write_best(p, r, k, best, (uint32_t)(4 * sub + at), m, log_s);
                    else write_none(p, r, k, absent);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (at == j) u[j] = 0;
            }
        }
        return;
    }
    // a whole wave per row: the values that reach the top-th largest of the lanes' own largest go to a list, and are
    // ranked there; a list that overflows (ties) is left, and the rounds below take its place
    const uint32_t bound = max(wave_nth_largest(ordered(own), p.top), kOrderedLowest);
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4 * C; ++j) {
        const uint32_t u = ordered(z[j]);
        const uint64_t hits = __ballot(usable && u >= bound);
        const int at = n + __popcll(hits & ((1ull << lane) - 1));
        if ((hits >> lane & 1) && at < kList) lists[wave_in][at] = {u, (uint32_t)(4 * (sub + (j >> 2) * group) + (j & 3))};
        n += __popcll(hits);
    }
    if (n <= kList) {
        OASR_SCORES_WAVE_LDS();
        if (!live) return;
        if (lane < n) {
            const Pick me = lists[wave_in][lane];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += before(lists[wave_in][o].value, lists[wave_in][o].index, me.value, me.index);
            if (rank < p.top) write_best(p, r, rank, me.value, me.index, m, log_s);
        }
        if (lane >= n && lane < p.top) write_none(p, r, lane, absent);
        return;
    }
    uint32_t taken = 0;                               // this lane's values that are out already
    for (int k = 0; k < p.top; ++k) {
        Pick best = {0, 0xffffffffu};
#pragma unroll
        for (int j = 0; j < 4 * C; ++j) {
            const uint32_t u = ordered(z[j]), at = 4 * (sub + (j >> 2) * group) + (j & 3);
            if (!(taken >> j & 1) && u >= bound) best = better(best, {u, at});
        }
        best = group_reduce(best, group, better);
#pragma unroll
        for (int j = 0; j < 4 * C; ++j)
            if (best.index == 4 * (sub + (j >> 2) * group) + (j & 3)) taken |= 1u << j;
        if (live && sub == 0) {
            if (usable && best.value) write_best(p, r, k, best.value, best.index, m, log_s);
            else write_none(p, r, k, absent);
        }
    }
}

// ---- long rows --------------------------------------------------------------------------------------------------------
// A wave's running sums: the reference m is shared by the wave, so that it rises rarely and rescaling costs little.
struct Sums {
    float m, s, t;
};

// A lane's running sums with what their additions rounded away (cs, ct: what the sums hold too much), so that the error of
// a sum does not grow with the row: one of 2^26 tokens gives a lane 4096 terms, and with terms that all round the same way the plain
// sum of 4096 is off by 2^-14.6 of itself, of 65536 by 2^-10.6.
struct LaneSums {
    float m, s, t, cs, ct;
};
__device__ __forceinline__ void add_compensated(float& sum, float& excess, float v) {
    const float y = v - excess, next = sum + y;
    excess = (next - sum) - y;
    sum = next;
}

// A lane's largest value, the chunk at which the step that held it began, and the largest of its other steps.
struct Tops {
    float first, second;
    int where;
};

template <int N>
__device__ __forceinline__ void add_values(LaneSums& a, Tops& top, int at, const float (&z)[N]) {
    float b = z[0];
#pragma unroll
    for (int j = 1; j < N; ++j) b = fmaxf(b, z[j]);
    top.second = fmaxf(top.second, fminf(top.first, b));
    top.where = b > top.first ? at : top.where;
    top.first = fmaxf(top.first, b);
    if (__any(b > a.m)) {
        const float m = fmaxf(a.m, group_reduce(b, 64, larger));
        const float d = fminf(m - a.m, kLargest), f = __builtin_amdgcn_exp2f(d * -kLog2e);
        a.t = f > 0.f ? f * fmaf(d, a.s, a.t) : 0.f * a.s;     // NaN stays NaN
        a.ct = f > 0.f ? f * fmaf(d, a.cs, a.ct) : 0.f;
        a.s *= f;
        a.cs *= f;
        a.m = m;
    }
    // the step's own sums first: sixteen terms are too few to matter, and one compensated addition per step costs little
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float x = a.m - z[j], e = __builtin_amdgcn_exp2f(x * -kLog2e);
        s = j ? s + e : e;
        t = j ? fmaf(e, fminf(x, kLargest), t) : e * fminf(x, kLargest);
    }
    add_compensated(a.s, a.cs, s);
    add_compensated(a.t, a.ct, t);
}

// Joins sums over another reference.
__device__ __forceinline__ void join(Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m);
    auto onto = [&](const Sums& x, float& s, float& t) {
        const float d = fminf(m - x.m, kLargest), f = __builtin_amdgcn_exp2f(d * -kLog2e);
        s = f * x.s;
        t = f > 0.f ? f * fmaf(d, x.s, x.t) : 0.f * x.s;
    };
    float s0, t0, s1, t1;
    onto(a, s0, t0);
    onto(b, s1, t1);
    a = {m, s0 + s1, t0 + t1};
}

template <typename E, int T, bool SPLIT>
__global__ __launch_bounds__(T) void token_scores_long_kernel(const Args p) {
    constexpr int N = Chunk<E>::N, W = T / 64, U = 16 / N;      // U chunks = 16 values per lane and step
    __shared__ Sums wave_sums[W];
    __shared__ uint32_t wave_bound[W], found, holding, single;
    __shared__ uint16_t holders[T];
    __shared__ int steps[T];
    __shared__ uint2 cand[kCandidates];
    __shared__ uint2 wave_pick[W];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r = SPLIT ? blockIdx.x / p.splits : blockIdx.x;
    const int split = SPLIT ? blockIdx.x % p.splits : 0;
    const int64_t src = source_row(p, r);
    if (src < 0) {                                              // uniform: nothing to read
        if (split == 0) {
            const float nothing = src == -2 ? nan32() : 0.f;
            for (int i = tid; i < p.given; i += T) p.logprobs[r * p.given + i] = nothing;
            if (tid == 0 && p.entropy) p.entropy[r] = nothing;
            if (tid < p.top) write_none(p, r, tid, src == -2 ? nan32() : -INFINITY);
        }
        return;
    }
    const E* row = reinterpret_cast<const E*>(p.logits) + src * p.ld;
    // this work-group's chunks, and for the last split the values behind the last whole chunk
    const int chunks = p.vocab / N;
    const int lo = SPLIT ? (int)((int64_t)chunks * split / p.splits) : 0;
    const int hi = SPLIT ? (int)((int64_t)chunks * (split + 1) / p.splits) : chunks;
    const int tail = !SPLIT || split == p.splits - 1 ? p.vocab - chunks * N : 0;

    LaneSums own = {kLowest, 0.f, 0.f, 0.f, 0.f};
    Tops top = {-INFINITY, -INFINITY, hi};
    int base = lo;
    for (; base + U * T <= hi; base += U * T) {
        float z[16];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float some[N];
            Chunk<E>::load(row + (int64_t)(base + u * T + tid) * N, some);
#pragma unroll
            for (int e = 0; e < N; ++e) z[u * N + e] = some[e];
        }
        add_values(own, top, base, z);
    }
    for (; base < hi; base += T) {
        float some[N];
        if (base + tid < hi) {
            Chunk<E>::load(row + (int64_t)(base + tid) * N, some);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) some[e] = -INFINITY;
        }
        add_values(own, top, base, some);
    }
    if (tail) {                                                 // uniform
        const float last[1] = {tid < tail ? Chunk<E>::one(row + (int64_t)chunks * N + tid) : -INFINITY};
        add_values(own, top, hi, last);                       // no chunk: offered below by itself
    }
    Sums a = {own.m, group_reduce(own.s - own.cs, 64, sum_of), group_reduce(own.t - own.ct, 64, sum_of)};
    // A bound that at least `top` values reach: the least over the waves of each wave's ceil(top / W)-th largest lane.
    const uint32_t mine = ordered(top.first);
    const uint32_t reach = p.top > 0 ? wave_nth_largest(mine, (p.top + W - 1) / W) : 0;
    if (lane == 0) {
        wave_sums[wave] = a;
        wave_bound[wave] = reach;
    }
    if (tid == 0) found = holding = single = 0;
    __syncthreads();
    a = wave_sums[0];
    uint32_t bound = wave_bound[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
        join(a, wave_sums[w]);
        bound = bound < wave_bound[w] ? bound : wave_bound[w];
    }
    bound = bound > kOrderedLowest ? bound : kOrderedLowest;
    const float log_s = logf(a.s);
    if (SPLIT) {
        if (tid == 0) {
            float* o = p.part + (r * p.splits + split) * 4;
            o[0] = a.m;
            o[1] = a.s;
            o[2] = a.t;
        }
    } else {
        for (int i = tid; i < p.given; i += T)
            p.logprobs[r * p.given + i] = token_logprob(row, p.vocab, p.tokens[r * p.given + i], a.m, a.s, log_s);
        if (tid == 0 && p.entropy) p.entropy[r] = row_entropy(a.s, a.t, log_s);
    }
    if (p.top == 0) return;
    uint2* const list = SPLIT ? p.cand + (r * p.splits + split) * p.top : nullptr;
    auto emit = [&](int at, uint32_t v, uint32_t i) {
        if (SPLIT) list[at] = make_uint2(v, i);
        else write_best(p, r, at, v, i, a.m, log_s);
    };
    auto emit_none = [&](int at) {
        if (SPLIT) list[at] = make_uint2(0, 0xffffffffu);
        else write_none(p, r, at, a.s != a.s ? nan32() : -INFINITY);
    };
    if (a.s != a.s) {                                           // uniform
        if (tid < p.top) emit_none(tid);
        return;
    }
    // Every value at or above the bound becomes a candidate.  Only lanes whose own largest reaches it hold any, and as a rule in
    // one step only: that step's U chunks are read again; where a second step reaches the bound too, all of the lane's (`each`
    // chunks, T apart).  The whole work-group reads, a chunk per thread, so that it costs one latency.  (Reading all chunks of every
    // such lane touches nearly every line of a row a second time: 8192 x 32000 with 20 alternatives 131 us, this way 112.)
    auto offer = [&](float z, uint32_t index) {
        const uint32_t u = ordered(z);
        if (u >= bound) {
            const uint32_t at = atomicAdd(&found, 1u);
            if (at < kCandidates) cand[at] = make_uint2(u, index);
        }
    };
    if (mine >= bound) {
        if (ordered(top.second) >= bound) holders[atomicAdd(&holding, 1u)] = (uint16_t)tid;
        else steps[atomicAdd(&single, 1u)] = top.where + tid;
    }
    __syncthreads();
    const uint32_t ones = single * U, each = (uint32_t)(hi - lo + T - 1) / T, reads = ones + holding * each;
    for (uint32_t i = tid; i < reads; i += T) {
        int c;
        if (i < ones) {
            c = steps[i / U] + (int)(i % U) * T;                // past a last, single chunk: another of the lane's, below the bound
        } else {
            const uint32_t q = (i - ones) / each;
            c = lo + holders[q] + (int)(i - ones - q * each) * T;
        }
        if (c < hi) {
            float some[N];
            Chunk<E>::load(row + (int64_t)c * N, some);
#pragma unroll
            for (int e = 0; e < N; ++e) offer(some[e], (uint32_t)c * N + e);
        }
    }
    if (mine >= bound && tid < tail) offer(Chunk<E>::one(row + (int64_t)chunks * N + tid), (uint32_t)chunks * N + tid);
    __syncthreads();
    const int n = (int)found;
    if (n <= kCandidates) {
        for (int c = tid; c < n; c += T) {
            const uint2 me = cand[c];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += before(cand[o].x, cand[o].y, me.x, me.y);
            if (rank < p.top) emit(rank, me.x, me.y);
        }
        for (int k = n + tid; k < p.top; k += T) emit_none(k);
        return;
    }
    // Too many values reach the bound (long runs of equal ones): the next in order, one after the other.
    uint2 last = make_uint2(0xffffffffu, 0u);
    for (int k = 0; k < p.top; ++k) {
        uint32_t v = 0, idx = 0xffffffffu;
        auto look = [&](float z, uint32_t index) {
            const uint32_t u = ordered(z);
            if (u >= kOrderedLowest && before(last.x, last.y, u, index) && before(u, index, v, idx)) {
                v = u;
                idx = index;
            }
        };
        for (int c = lo + tid; c < hi; c += T) {
            float z[N];
            Chunk<E>::load(row + (int64_t)c * N, z);
#pragma unroll
            for (int e = 0; e < N; ++e) look(z[e], (uint32_t)c * N + e);
        }
        if (tid < tail) look(Chunk<E>::one(row + (int64_t)chunks * N + tid), (uint32_t)chunks * N + tid);
        const Pick best = group_reduce(Pick{v, idx}, 64, better);
        if (lane == 0) wave_pick[wave] = make_uint2(best.value, best.index);
        __syncthreads();
        last = wave_pick[0];
        for (int w = 1; w < W; ++w)
            if (before(wave_pick[w].x, wave_pick[w].y, last.x, last.y)) last = wave_pick[w];
        __syncthreads();                                        // picked before the next round writes
        if (tid == 0) {
            if (last.x) emit(k, last.x, last.y);
            else emit_none(k);
        }
        if (!last.x) last = make_uint2(0, 0xffffffffu);
    }
}

// Joins the splits of a row: one wave per row, lane s holds split s and, in LDS, its list.
template <typename E>
__global__ __launch_bounds__(64) void token_scores_join_kernel(const Args p) {
    constexpr int kJoined = 128;
    __shared__ uint2 lists[kMaxSplits * kMaxTop];
    __shared__ Pick joined[kJoined];
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x, src = source_row(p, r);
    if (src < 0) return;                                        // written by the first split
    const E* row = reinterpret_cast<const E*>(p.logits) + src * p.ld;
    for (int i = lane; i < p.splits * p.top; i += 64) lists[i] = p.cand[r * p.splits * p.top + i];
    Sums a = {kLowest, 0.f, 0.f};
    if (lane < p.splits) {
        const float* o = p.part + (r * p.splits + lane) * 4;
        a = {o[0], o[1], o[2]};
    }
    a = group_reduce(a, 64, [](Sums x, const Sums& y) {
        join(x, y);
        return x;
    });
    const float log_s = logf(a.s);
    for (int i = lane; i < p.given; i += 64)
        p.logprobs[r * p.given + i] = token_logprob(row, p.vocab, p.tokens[r * p.given + i], a.m, a.s, log_s);
    if (lane == 0 && p.entropy) p.entropy[r] = row_entropy(a.s, a.t, log_s);
    if (p.top == 0) return;
    if (a.s != a.s) {
        if (lane < p.top) write_none(p, r, lane, nan32());
        return;
    }
    __syncthreads();
    // A value that at least `top` entries reach: of each list the first `depth`, of enough lists.  What reaches it - few entries
    // more than `top`, as a rule - is collected and ranked; ties may make it too many, and then the heads are picked in turn.
    const int depth = (p.top + p.splits - 1) / p.splits, first = lane * p.top;
    const uint32_t mark = lane < p.splits ? lists[first + depth - 1].x : 0;
    const uint32_t bound = max(wave_nth_largest(mark, (p.top + depth - 1) / depth), 1u);       // 0: no entry
    int n = 0;
    for (int e = 0; e < p.top; ++e) {
        const uint2 entry = lane < p.splits ? lists[first + e] : make_uint2(0, 0);
        const uint64_t hits = __ballot(entry.x >= bound);
        if (!hits) break;
        const int at = n + __popcll(hits & ((1ull << lane) - 1));
        if (entry.x >= bound && at < kJoined) joined[at] = {entry.x, entry.y};
        n += __popcll(hits);
    }
    __syncthreads();
    if (n <= kJoined) {
        for (int c = lane; c < n; c += 64) {
            const Pick me = joined[c];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += before(joined[o].value, joined[o].index, me.value, me.index);
            if (rank < p.top) write_best(p, r, rank, me.value, me.index, a.m, log_s);
        }
        for (int k = n + lane; k < p.top; k += 64) write_none(p, r, k, -INFINITY);
        return;
    }
    const uint2 none = make_uint2(0, 0xffffffffu);
    int at = first;
    const int end = lane < p.splits ? at + p.top : at;
    uint2 head = at < end ? lists[at] : none;
    for (int k = 0; k < p.top; ++k) {
        const Pick best = group_reduce(Pick{head.x, head.y}, 64, better);
        if (lane == 0) {
            if (best.value) write_best(p, r, k, best.value, best.index, a.m, log_s);
            else write_none(p, r, k, -INFINITY);
        }
        if (best.value && head.x == best.value && head.y == best.index) head = ++at < end ? lists[at] : none;   // the winner's next
    }
}

// Work-groups per row.  Cutting a row costs a second launch (some 4 us), which pays for few and very long rows only: parts of
// 8192 tokens (one row of 131072: 9.7 against 14.7 us, 64 rows 14.3 against 18.0; one row of 32000: 9.1 against 7.6, 200 rows of
// 131072 bf16 21.9 against 20.9).
static int splits_for(int64_t rows, int64_t vocab) {
    if (vocab <= 65536 || rows > 128) return 1;
    int64_t s = (vocab + 8191) / 8192;
    if (s > 1024 / rows) s = 1024 / rows;
    return (int)(s > kMaxSplits ? kMaxSplits : s);
}

static int64_t workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
    if (rows <= 0 || vocab <= 0 || top < 0) return 0;
    const int64_t s = splits_for(rows, vocab);
    return s == 1 ? 0 : round_up(rows * s * 16, 256) + rows * s * top * 8;
}

template <typename E>
static void launch(const Args& p, hipStream_t st) {
    if (p.vocab <= kShort) {
        int g = 0;
        while (g < 6 && (4 << g) < p.vocab) ++g;
        const int64_t per_wg = (int64_t)4 << (6 - g);
        const dim3 grid((unsigned)((p.rows + per_wg - 1) / per_wg)), blk(256);
        if (p.vocab <= 256) hipLaunchKernelGGL((token_scores_short_kernel<E, 1>), grid, blk, 0, st, p, g);
        else if (p.vocab <= 512) hipLaunchKernelGGL((token_scores_short_kernel<E, 2>), grid, blk, 0, st, p, g);
        else hipLaunchKernelGGL((token_scores_short_kernel<E, 4>), grid, blk, 0, st, p, g);     // (eight: 20000 x 2000 bf16 41 us, streamed 25)
    } else if (p.splits > 1) {
        hipLaunchKernelGGL((token_scores_long_kernel<E, 256, true>), dim3((unsigned)(p.rows * p.splits)), dim3(256), 0, st, p);
        hipLaunchKernelGGL((token_scores_join_kernel<E>), dim3((unsigned)p.rows), dim3(64), 0, st, p);
    } else {
        // Few long rows: wider work-groups keep the chip busier (256 x 65536 bf16: 512 threads 14.7 us, 256 threads 18.9; 400 x 50257
        // float32: 20.8 and 24.5; but 513 x 50257 bf16: 21.4 and 20.6).  Many or shorter ones: narrower work-groups interleave better
        // and have fewer lanes to rank (8192 x 32000 bf16: 512 threads 131 us, 256 threads 103; 16000 x 5000: 256 threads 61,
        // 128 threads 45, one wave 41; 2048 x 5000: 13.7, 10.6 and 11.1; 1024 x 32000: 19.6, 22.7 and 33.3).  Rows from memory, not
        // from a cache that an earlier call filled.
        const dim3 grid((unsigned)p.rows);
        const int64_t bytes = (int64_t)p.vocab * (int64_t)sizeof(E);
        const bool brief = p.vocab <= 10240;
        const bool wide = (p.rows <= 400 && bytes >= 61440) || (p.rows <= 640 && bytes >= 131072);
        if (wide) hipLaunchKernelGGL((token_scores_long_kernel<E, 512, false>), grid, dim3(512), 0, st, p);
        else if (brief && p.rows >= 4096) hipLaunchKernelGGL((token_scores_long_kernel<E, 64, false>), grid, dim3(64), 0, st, p);
        else if (p.vocab <= 5120 || (brief && p.rows >= 1024)) hipLaunchKernelGGL((token_scores_long_kernel<E, 128, false>), grid, dim3(128), 0, st, p);
        else hipLaunchKernelGGL((token_scores_long_kernel<E, 256, false>), grid, dim3(256), 0, st, p);
    }
}

static int run(const char* what, Args& p, int32_t dtype, void* workspace, int64_t bytes, hipStream_t st) {
    OASR_REQUIRE(dtype == OASR_F32 || dtype == OASR_BF16, "%s: dtype must be OASR_F32 or OASR_BF16", what);
    OASR_REQUIRE(p.rows >= 0 && p.rows < ((int64_t)1 << 24), "%s: rows must lie in [0, 2^24)", what);      // 256 threads each at most
    OASR_REQUIRE(p.vocab > 0 && p.vocab < (1 << 30), "%s: vocab must lie in [1, 2^30)", what);
    OASR_REQUIRE(p.ld >= p.vocab, "%s: ld=%lld does not cover the vocabulary", what, (long long)p.ld);
    OASR_REQUIRE(p.given >= 0, "%s: the count of given tokens is negative", what);
    OASR_REQUIRE(p.top >= 0 && p.top <= kMaxTop, "%s: top must lie in [0, %d]", what, kMaxTop);
    if (p.rows == 0) return OASR_OK;
    OASR_REQUIRE(p.logits && (p.given == 0 || (p.tokens && p.logprobs)) && (p.top == 0 || (p.ids && p.best)), "%s: null pointer", what);
    const uintptr_t words = (uintptr_t)p.tokens | (uintptr_t)p.frames | (uintptr_t)p.logprobs | (uintptr_t)p.entropy | (uintptr_t)p.ids |
                            (uintptr_t)p.best;
    OASR_REQUIRE(((uintptr_t)p.logits & (dtype == OASR_F32 ? 3 : 1)) == 0 && (words & 3) == 0, "%s: misaligned pointer", what);
    p.splits = splits_for(p.rows, p.vocab);
    const int64_t need = workspace_bytes(p.rows, p.vocab, p.top);
    if (need > 0) {
        if (bytes < need) {
            set_error("%s: workspace needs %lld bytes, got %lld", what, (long long)need, (long long)bytes);
            return OASR_ECAPACITY;
        }
        OASR_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "%s: workspace missing or not 256-byte aligned", what);
        p.part = static_cast<float*>(workspace);
        p.cand = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + round_up(p.rows * p.splits * 16, 256));
    }
    if (dtype == OASR_F32) launch<float>(p, st);
    else launch<uint16_t>(p, st);
    OASR_CHECK_LAUNCH(what);
    return OASR_OK;
}

}  // namespace scores
}  // namespace oasr

using namespace oasr;

extern "C" {

int64_t oasr_token_scores_workspace_bytes(int64_t rows, int64_t vocab, int32_t top) { return scores::workspace_bytes(rows, vocab, top); }

int oasr_token_scores(const void* logits, int32_t dtype, int64_t ld, int64_t rows, int32_t vocab, const int32_t* tokens,
                      int32_t given, float* logprobs, float* entropy, int32_t top, int32_t* ids, float* best, void* workspace,
                      int64_t workspace_bytes, void* stream) {
    scores::Args p = {};
    p.logits = logits;
    p.ld = ld;
    p.rows = rows;
    p.vocab = vocab;
    p.given = given;
    p.top = top;
    p.tokens = tokens;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.ids = ids;
    p.best = best;
    return scores::run("token_scores", p, dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

int oasr_ctc_token_scores(const void* logits, int32_t dtype, int64_t ld, int32_t vocab, int32_t batch, int64_t t_pad,
                          const int32_t* tokens, const int32_t* frames, int64_t width, float* logprobs, float* entropy,
                          int32_t top, int32_t* ids, float* best, void* workspace, int64_t workspace_bytes, void* stream) {
    OASR_REQUIRE(batch >= 0 && t_pad > 0 && width >= 0 && width < ((int64_t)1 << 31), "ctc_token_scores: bad batch, t_pad or width");
    if (batch == 0 || width == 0) return OASR_OK;
    OASR_REQUIRE(frames && tokens && logprobs, "ctc_token_scores: null pointer");
    scores::Args p = {};
    p.logits = logits;
    p.ld = ld;
    p.rows = batch * width;
    p.vocab = vocab;
    p.given = 1;
    p.top = top;
    p.tokens = tokens;
    p.frames = frames;
    p.width = width;
    p.frames_per = t_pad;
    p.logprobs = logprobs;
    p.entropy = entropy;
    p.ids = ids;
    p.best = best;
    return scores::run("ctc_token_scores", p, dtype, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"
