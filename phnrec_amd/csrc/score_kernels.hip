// score_kernels.hip -- lcrc_score (include/lcrc_pipeline.h): ln p of given classes, entropy and the k best classes of every
// row of logits or posteriors.
//     l(c) = x(c) or ln x(c);  m = max x (logits), 0 (posteriors);  e(c) = exp(x(c) - m) or x(c)
//     S = sum e, T = sum e * (l - m);  ln p(c) = (l(c) - m) - ln S;  entropy = ln S - T / S
// Every row is read once.  All accesses are 16 bytes wide: a row is cut into chunks of 16 bytes from its start, the last one
// moved back so that it ends with the row (what it holds twice is masked), so any alignment of an element is served and
// nothing outside the row is touched.
//
// NaN, +inf (and posteriors below 0) need no test for each value: they leave S at NaN or inf (a maximum skips NaN, but exp
// carries it; inf - inf is NaN), a negative posterior shows in the rows' minimum.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_dev.h"

namespace phnrec {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = kScoreThreads;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kLowest = -3.40282346638528859812e38f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

// W consecutive elements, 16 bytes where W is 16 / sizeof(X)
template <typename X, int W>
struct Chunk {
    X v[W];
    __device__ __forceinline__ float operator[](int i) const { return to_f32(v[i]); }
};
template <typename X, int W>
__device__ __forceinline__ Chunk<X, W> load_chunk(const X *p)
{
    Chunk<X, W> c;
    __builtin_memcpy(&c, p, sizeof(c));             // element-aligned: one unaligned 16-byte load
    return c;
}

// ---- reductions ----
// over the 16 lanes of a row of lanes; every lane gets the same bits (each step adds the same two numbers in both places)
template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)); }
template <int CTRL>
__device__ __forceinline__ double dpp(double v)
{
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xf, 0xf, false);
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xf, 0xf, false), lo);
}
template <typename V, typename Op>
__device__ __forceinline__ V reduce16(V v, Op op)
{
    v = op(v, dpp<0x128>(v));                       // row_ror:8, 4, 2, 1
    v = op(v, dpp<0x124>(v));
    v = op(v, dpp<0x122>(v));
    return op(v, dpp<0x121>(v));
}
// over 8 lanes: their pairs, their pairs of pairs, the two halves mirrored
template <typename V, typename Op>
__device__ __forceinline__ V reduce8(V v, Op op)
{
    v = op(v, dpp<0xb1>(v));                        // quad_perm 1 0 3 2, quad_perm 2 3 0 1, row_half_mirror
    v = op(v, dpp<0x4e>(v));
    return op(v, dpp<0x141>(v));
}
template <typename Op>
__device__ __forceinline__ float reduce64(float v, Op op)
{
    v = reduce16(v, op);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
struct Max { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return __builtin_elementwise_max(a, b); } };
struct Min { __device__ __forceinline__ float operator()(float a, float b) const { return fminf(a, b); } };
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };

// ---- a row's statistics ----
struct Stats {
    float m, S, T;      // S is NaN or inf in a row that is no distribution; m: logits: the maximum, posteriors: T of small values
};

// the sums over one value (logits: m is the row's or the running maximum)
template <bool PROBS>
__device__ __forceinline__ void add_value(float v, Stats &s)
{
    if constexpr (PROBS) {
        // Both ends of f32's range: T is kept in units of 256 ln 2, so that it leaves the range no sooner than S does, and apart
        // for values below 2^-64, times 2^64: their products would be subnormal, rounded to a multiple of 2^-149 (a row of 100
        // values of 1e-45 had an entropy of 79 instead of 4.6).  The scaling also keeps v_log_f32 off what it flushes.
        const bool small = v < 0x1p-64f;
        const float w = small ? v * 0x1p64f : v;
        const float l = fmaf(__builtin_amdgcn_logf(w), 0x1p-8f, small ? -64 * 0x1p-8f : 0.0f);
        const float t = v > 0.0f ? w * l : 0.0f;
        s.S += v;
        s.T += small ? 0.0f : t;
        s.m += small ? t : 0.0f;
    } else {
        const float d = v - s.m;
        const float e = __builtin_amdgcn_exp2f(d * kLog2e);
        s.S += e;
        s.T = fmaf(e, fmaxf(d, -1e30f), s.T);       // (0 * -inf)
    }
}
template <bool PROBS>
struct Row {
    float m, S, T, ln_s;
    bool bad, none;
    __device__ __forceinline__ Row(const Stats &s, bool negative)
        : m(s.m), S(s.S), T(s.T), ln_s(PROBS ? logf(s.S) : __builtin_amdgcn_logf(s.S) * kLn2), bad(negative || !(s.S < INFINITY)), none(!(s.S > 0.0f)) {}
    __device__ __forceinline__ float ln_p(float v) const
    {
        if (bad) return NAN;
        if (none) return -INFINITY;
        return (PROBS ? logf(v) : v - m) - ln_s;
    }
    __device__ __forceinline__ float entropy() const { return bad ? NAN : none ? 0.0f : ln_s - (PROBS ? (T / S + m / (S * 0x1p64f)) * (256.0f * kLn2) : T * __builtin_amdgcn_rcpf(S)); }
};

// A label of a row and its class's value, asked for before the row is worked on: two loads that wait for one another.
struct Label {
    int c;
    float v;
    bool wanted;
    template <typename X>
    __device__ __forceinline__ Label(const lcrc_score_args &a, const X *x, size_t r, int j) : wanted(a.logp && j < a.n_labels)
    {
        c = wanted ? a.labels[r * a.n_labels + j] : -1;
        v = to_f32(x[c < 0 || c >= a.cols ? 0 : c]);
    }
    template <bool PROBS>
    __device__ __forceinline__ void put(const lcrc_score_args &a, const Row<PROBS> &row, size_t r, int j) const
    {
        if (wanted) a.logp[r * a.n_labels + j] = c < 0 ? 0.0f : c >= a.cols ? NAN : row.ln_p(v);
    }
};
__device__ __forceinline__ bool wants_top(const lcrc_score_args &a) { return a.k > 0 && (a.top_index || a.top_logp); }

// ---- short rows: 8 lanes to a row ----
// A value and its column as ONE double: the f32 value (its conversion leaves 29 bits free) and the column in the free bits,
// complemented where that makes the lower column the larger number.  So one v_max_f64, a full-rate instruction, orders values
// and columns together, and a lane keeps its K best by K maxima and K - 1 minima for each value.  -inf sits at -2^200, below
// every f32; what is no class at all at -inf.
__device__ __forceinline__ double pair_of(float v, int c)
{
    const double d = fmax((double)(v + 0.0f), -0x1p200);
    const int hi = __double2hiint(d);
    return __hiloint2double(hi, __double2loint(d) | ((c ^ ~(hi >> 31)) & 0x1fffffff));
}
__device__ __forceinline__ int column_of(double d)
{
    return (__double2loint(d) ^ ~(__double2hiint(d) >> 31)) & 0x1fffffff;
}
__device__ __forceinline__ float value_of(double d)
{
    return (float)__hiloint2double(__double2hiint(d), __double2loint(d) & ~0x1fffffff);
}

// Maximum and minimum of such numbers.  Written out: the compiler puts a quieting maximum in front of every operand that it does
// not know to be no NaN, 40 of the kernel's 560 instructions.  (settled: for a result that is read across lanes at once)
__device__ __forceinline__ double larger(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double smaller(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
struct Larger {
    __device__ __forceinline__ double operator()(double a, double b) const
    {
        double r;
        asm("v_max_f64 %0, %1, %2\n\ts_nop 1" : "=v"(r) : "v"(a), "v"(b));        // two states before a DPP read
        return r;
    }
};
__device__ __forceinline__ double settled(double a)
{
    asm("s_nop 1" : "+v"(a));
    return a;
}

// J chunks of W values to a lane: up to 8 J W columns; K: the longest list of best classes.
// Bound by instructions: 524288 x 186 f32 with 3 best 94 us = 4.3 TB/s, a third of its instructions f64 maxima and what builds their
// operands (16 lanes to a row: 102 us; rows prefetched by fewer, longer-lived workgroups: slower by 10).  8192 x 138 with 5
// best: 5.7 us.
template <typename X, bool PROBS, int W, int J, int K>
__global__ __launch_bounds__(kThreads) void score_short_kernel(const lcrc_score_args a)
{
    const int lane = threadIdx.x & 7, cols = a.cols;
    const size_t stride = (size_t)gridDim.x * (kThreads / 8);
    for (size_t r = (size_t)blockIdx.x * (kThreads / 8) + threadIdx.x / 8; r < (size_t)a.rows; r += stride) {
        const X *x = static_cast<const X *>(a.x) + r * (size_t)a.ld;
        Chunk<X, W> raw[J];
#pragma unroll
        for (int j = 0; j < J; j++) raw[j] = load_chunk<X, W>(x + min((8 * j + lane) * W, cols - W));
        const Label label(a, x, r, lane);
        // (launch(): so many chunks of every lane are whole, the others may be cut off by the row's end or lie behind it)
        constexpr int kWhole = J <= 4 ? J - 1 : J - 2;
        const auto at = [&](int j) { return (8 * j + lane) * W; };
        const auto live = [&](int j, int i) { return j < kWhole || min(at(j), cols - W) + i >= at(j); };
        const auto column = [&](int j, int i) { return (j < kWhole ? at(j) : min(at(j), cols - W)) + i; };
        float m = kLowest, least = 0.0f;
        Stats s = {0.0f, 0.0f, 0.0f};
        if constexpr (!PROBS) {
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < W; i++) m = fmaxf(m, raw[j][i]);       // (what is there twice does no harm)
            s.m = m = reduce8(m, Max());
        }
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int i = 0; i < W; i++) {
                const float v = live(j, i) ? raw[j][i] : PROBS ? 0.0f : -INFINITY;
                if constexpr (PROBS) least = fminf(least, v);
                add_value<PROBS>(v, s);
            }
        s.S = reduce8(s.S, Add());
        s.T = reduce8(s.T, Add());
        if constexpr (PROBS) s.m = reduce8(s.m, Add()), least = reduce8(least, Min());
        const Row<PROBS> row(s, least < 0.0f);
        if (a.entropy && lane == 0) a.entropy[r] = row.entropy();
        label.put(a, row, r, lane);
        if (a.logp && a.n_labels > 8)
            for (int j = lane + 8; j < a.n_labels; j += 8) Label(a, x, r, j).put(a, row, r, j);
        if constexpr (K > 0) {
            double best[K];
#pragma unroll
            for (int q = 0; q < K; q++) best[q] = -INFINITY;
#pragma unroll
            for (int j = 0; j < J; j++)
#pragma unroll
                for (int i = 0; i < W; i++) {
                    double d = pair_of(raw[j][i], column(j, i));
                    if (!live(j, i)) d = -INFINITY;
#pragma unroll
                    for (int q = 0; q < K; q++) {
                        const double upper = larger(best[q], d);
                        if (q + 1 < K) d = smaller(best[q], d);
                        best[q] = upper;
                    }
                }
            double mine = 0.0;
            for (int n = 0; n < a.k; n++) {                  // the best head of the 8 lists, taken off its list
                const double top = reduce8(settled(best[0]), Larger());
                const bool won = best[0] == top;
#pragma unroll
                for (int q = 0; q < K; q++) best[q] = won ? (q + 1 < K ? best[q + 1] : -INFINITY) : best[q];
                if (lane == n) mine = top;
            }
            if (lane < a.k) {
                if (a.top_index) a.top_index[r * a.k + lane] = row.bad ? -1 : column_of(mine);
                if (a.top_logp) a.top_logp[r * a.k + lane] = row.ln_p(value_of(mine));
            }
        }
    }
}

// ---- longer rows, longer lists: the best classes by a threshold ----
// A key orders values, then columns (or chunks, or positions): 32 bits that rise with the value, -0 and +0 alike, and the
// complement of the column below them; 0 is below every key of a value.
__device__ __forceinline__ unsigned ordered(float x)
{
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ u64 make_key(float x, int c) { return ((u64)ordered(x) << 32) | (0xffffffffu - (unsigned)c); }
__device__ __forceinline__ int key_column(u64 k) { return (int)(0xffffffffu - (unsigned)k); }
__device__ __forceinline__ float key_value(u64 k)
{
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float(o ^ (~(unsigned)((int)o >> 31) | 0x80000000u));
}

// A bar that at least k (1 <= k <= 64) of the wave's 64 G keys reach, and no more than k where their upper halves differ:
// bit by bit from the top, a candidate stands if k keys reach it, and the search ends when exactly k do.  One compare a bit and
// key on the vector side, the count on the scalar side.  Equal upper halves (equal values) are told apart by the lower ones.
template <int G>
__device__ __forceinline__ int count_from(const unsigned (&v)[G], unsigned t)
{
    int n = 0;
#pragma unroll
    for (int q = 0; q < G; q++) n += __popcll(__ballot(v[q] >= t));
    return n;
}
template <int G>
__device__ __forceinline__ unsigned bar_of(const unsigned (&v)[G], int k, int *reached)
{
    unsigned res = 0;
    int n = 64 * G;
    if constexpr (G == 1) {
        for (int bit = 31; bit >= 0 && n != k; bit--) {
            const unsigned t = res | (1u << bit);
            const int c = count_from(v, t);
            if (c >= k) res = t, n = c;
        }
    } else {                                    // a workgroup waits for it: two bits at a time, three counts side by side
        for (int bit = 30; bit >= 0 && n != k; bit -= 2) {
            const unsigned t1 = res | (1u << bit), t2 = res | (2u << bit), t3 = res | (3u << bit);
            const int c1 = count_from(v, t1), c2 = count_from(v, t2), c3 = count_from(v, t3);
            if (c3 >= k) res = t3, n = c3;
            else if (c2 >= k) res = t2, n = c2;
            else if (c1 >= k) res = t1, n = c1;
        }
    }
    *reached = n;
    return res;
}
template <int G>
__device__ __forceinline__ u64 bar_of(const u64 (&key)[G], int k)
{
    unsigned hi[G], lo[G];
#pragma unroll
    for (int q = 0; q < G; q++) hi[q] = (unsigned)(key[q] >> 32);
    int n;
    const unsigned h = bar_of(hi, k, &n);
    if (n == k || h == 0) return (u64)h << 32;
    // more than k: they stand at exactly h or above (all bits are decided); the lower half decides among those at h
    const int more = h == 0xffffffffu ? 0 : count_from(hi, h + 1);
#pragma unroll
    for (int q = 0; q < G; q++) lo[q] = hi[q] == h ? (unsigned)key[q] : 0;
    return ((u64)h << 32) | bar_of(lo, k - more, &n);
}

constexpr int kCandidates = 512;       // candidates a team holds (more: the slow way)

// A team of threads that works on one row: T threads, one wave or a whole workgroup.
// TOGETHER: a wave that looks through its values in step, and needs no counter in memory.
template <int T, bool TOGETHER = false>
struct Team {
    static constexpr int kWaves = T / 64;
    struct Shared {
        u64 cand[kCandidates];
        u64 best[T > 64 ? T : 1];
        float slot[4 * kWaves];
        u64 kslot[kWaves];
        int count;
    };
    Shared &sh;
    const int t;
    __device__ __forceinline__ Team(Shared &s) : sh(s), t(threadIdx.x % T) {}
    __device__ __forceinline__ void sync() const
    {
        if constexpr (T > 64) __syncthreads();
        else {                                                  // one wave: its LDS accesses are in order
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
    // the team's statistics from its threads': S and T move to the team's maximum
    template <bool PROBS>
    __device__ __forceinline__ Stats join(Stats s, float &least)
    {
        Stats all;
        const auto moved = [](Stats &v, float m) {
            if constexpr (!PROBS) {
                const float d = fmaxf(v.m - m, -1e30f), f = __builtin_amdgcn_exp2f(d * kLog2e);
                v.T = f * fmaf(v.S, d, v.T);
                v.S *= f;
            }
        };
        if constexpr (PROBS) all.m = reduce64(s.m, Add());
        else all.m = reduce64(s.m, Max());
        moved(s, all.m);
        all.S = reduce64(s.S, Add());
        all.T = reduce64(s.T, Add());
        least = PROBS ? reduce64(least, Min()) : 0.0f;
        if constexpr (T > 64) {
            sync();
            if ((t & 63) == 0) {
                float *p = sh.slot + 4 * (t >> 6);
                p[0] = all.m, p[1] = all.S, p[2] = all.T, p[3] = least;
            }
            sync();
            float m = sh.slot[0];
            for (int w = 1; w < kWaves; w++) m = PROBS ? m + sh.slot[4 * w] : fmaxf(m, sh.slot[4 * w]);
            s = {m, 0.0f, 0.0f};
            for (int w = 0; w < kWaves; w++) {
                Stats v = {sh.slot[4 * w], sh.slot[4 * w + 1], sh.slot[4 * w + 2]};
                moved(v, m);
                s.S += v.S, s.T += v.T;
                least = fminf(least, sh.slot[4 * w + 3]);
            }
            all = s;
        }
        return all;
    }
    __device__ __forceinline__ u64 max_key(u64 v)
    {
        for (int d = 32; d >= 1; d >>= 1) {
            const u64 o = __shfl_xor(v, d);
            v = o > v ? o : v;
        }
        if constexpr (T > 64) {
            sync();
            if ((t & 63) == 0) sh.kslot[t >> 6] = v;
            sync();
            for (int w = 0; w < kWaves; w++) v = sh.kslot[w] > v ? sh.kslot[w] : v;
        }
        return v;
    }
    // The k best of the team's values, best first: out(rank, key), by the thread that finds it.
    //   first          the best (value, chunk) of this thread's share, as a key, 0 where it has none
    //   scan(bar, f)   f(live, value, chunk, column) for what this thread holds, at least for the values whose keys reach the
    //                  bar; by a whole wave together where the team is one
    //   again(f)       the same for all that it holds, any number of times
    // The threads are put into 64 G groups.  The k-th best of the groups' bests is reached by at least k values, so
    // the k best are among the values that reach it, and only threads with such a group look at their values again.  With
    // 256 groups some 74 of random values remain for k = 64, 17 for k = 16 (from 64 groups 300 and 18).  They are ranked by
    // counting.  Rows made so that more remain than fit are done one rank after another.
    template <typename Scan, typename Again, typename Out>
    __device__ __forceinline__ void top(int k, u64 first, const Scan &scan, const Again &again, const Out &out)
    {
        constexpr int G = T > 64 ? 4 : 1;
        u64 group[G];
        if (!TOGETHER && t == 0) sh.count = 0;
        if constexpr (T > 64) {
            sh.best[t] = first;
            sync();
#pragma unroll
            for (int q = 0; q < G; q++) {
                group[q] = 0;
                for (int w = q; w < kWaves; w += G) group[q] = max(group[q], sh.best[64 * w + (t & 63)]);
            }
        } else {
            group[0] = first;
            sync();
        }
        const u64 bar = bar_of(group, k);
        const float least = key_value(bar);
        const auto reaches = [&](float v, int chunk) {          // (a bar between two values can lie at a NaN: no help then)
            return !(v < least) && make_key(v, chunk) >= bar;
        };
        int n = 0;
        if constexpr (!TOGETHER) {
            if (first >= bar && first != 0)
                scan(bar, [&](bool live, float v, int chunk, int c) {
                    if (live && reaches(v, chunk)) {
                        const int at = atomicAdd(&sh.count, 1);      // (any order: they are ranked by their keys)
                        if (at < kCandidates) sh.cand[at] = make_key(v, c);
                    }
                });
            sync();
            n = sh.count;
        } else {
            scan(bar, [&](bool live, float v, int chunk, int c) {
                const bool hit = live && reaches(v, chunk);
                const u64 all = __ballot(hit);
                const int at = n + __builtin_amdgcn_mbcnt_hi((unsigned)(all >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)all, 0));
                if (hit && at < kCandidates) sh.cand[at] = make_key(v, c);
                n += __popcll(all);
            });
            sync();
        }
        if (n <= kCandidates) {
            for (int i = t; i < n; i += T) {
                const u64 key = sh.cand[i];
                int rank = 0;
#pragma unroll 8
                for (int q = 0; q < n; q++) rank += sh.cand[q] > key ? 1 : 0;
                if (rank < k) out(rank, key);
            }
        } else {
            u64 last = ~0ull;
            for (int q = 0; q < k; q++) {
                u64 best = 0;
                again([&](bool live, float v, int, int c) {
                    const u64 key = make_key(v, c);
                    if (live && key < last && key > best) best = key;
                });
                last = max_key(best);
                if (t == 0) out(q, last);
            }
        }
        sync();                                                 // (the lists are free for the next row)
    }
};

__device__ __forceinline__ void put_bad(const lcrc_score_args &a, size_t r, int rank)
{
    if (a.top_index) a.top_index[r * a.k + rank] = -1;
    if (a.top_logp) a.top_logp[r * a.k + rank] = NAN;
}
template <bool PROBS>
__device__ __forceinline__ void put_top(const lcrc_score_args &a, size_t r, const Row<PROBS> &row, int rank, u64 key)
{
    if (a.top_index) a.top_index[r * a.k + rank] = key_column(key);
    if (a.top_logp) a.top_logp[r * a.k + rank] = row.ln_p(key_value(key));
}

// ---- a wave to a row, the row in its registers: a chunk of 16 bytes to a lane (rows of up to 64 chunks, k beyond the lists') ----
// Bound by the fixed part of the search (bar, ballots, ranks): 524288 x 186 f32 with 20 best 297 us.
template <typename X, bool PROBS>
__global__ __launch_bounds__(kThreads) void score_wave_kernel(const lcrc_score_args a)
{
    constexpr int W = 16 / sizeof(X);
    __shared__ typename Team<64, true>::Shared shared[kThreads / 64];
    Team<64, true> team(shared[threadIdx.x >> 6]);
    const int lane = team.t, cols = a.cols, start = min(lane * W, cols - W), from = lane * W - start;
    const size_t stride = (size_t)gridDim.x * (kThreads / 64);
    for (size_t r = (size_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); r < (size_t)a.rows; r += stride) {
        const X *x = static_cast<const X *>(a.x) + r * (size_t)a.ld;
        const Chunk<X, W> raw = load_chunk<X, W>(x + start);
        const Label label(a, x, r, lane);
        float least = 0.0f;
        Stats s = {0.0f, 0.0f, 0.0f};
        float most = raw[W - 1];                    // of the chunk, without what it shares with the one before
#pragma unroll
        for (int i = 0; i < W - 1; i++) most = i >= from ? fmaxf(most, raw[i]) : most;
        if constexpr (!PROBS) s.m = reduce64(fmaxf(most, kLowest), Max());         // (lanes behind the end: the last chunk's)
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float v = i >= from ? raw[i] : PROBS ? 0.0f : -INFINITY;
            if constexpr (PROBS) least = fminf(least, v);
            add_value<PROBS>(v, s);
        }
        s.S = reduce64(s.S, Add());
        s.T = reduce64(s.T, Add());
        if constexpr (PROBS) s.m = reduce64(s.m, Add()), least = reduce64(least, Min());
        const Row<PROBS> row(s, least < 0.0f);
        if (a.entropy && lane == 0) a.entropy[r] = row.entropy();
        label.put(a, row, r, lane);
        if (!wants_top(a)) continue;
        if (row.bad) {
            if (lane < a.k) put_bad(a, r, lane);
            continue;
        }
        const u64 first = from < W ? make_key(most, lane) : 0;
        const auto scan = [&](const auto &f) {
#pragma unroll
            for (int i = 0; i < W; i++) f(i >= from, raw[i], lane, start + i);
        };
        team.top(a.k, first, [&](u64, const auto &f) { scan(f); }, scan, [&](int rank, u64 key) { put_top<PROBS>(a, r, row, rank, key); });
    }
}

// ---- long rows: a workgroup to a row, or to a part of one ----
struct Part {
    int parts;                  // of a row
    int chunks;                 // in a part
    float4 *stats;              // [rows][parts]: m, S, T, the least value  (parts > 1)
    u64 *keys;                  // [rows][parts][k], best first, 0 where a part has fewer
};

// (T = 64: a wave to a row, four of them in a workgroup)
// U chunks on their way to a thread; about 12 instruction slots a value, four of them the exponential's.  12000 x 8192 f32 with
// 5 best 80 us = 4.9 TB/s, a copy's rate; 2051 x 50001 bf16 with 16 best 65 us = 3.2 TB/s (256 threads; 512: 68, 1024: 146 --
// fewer workgroups are left to load while others search); the first version, k passes over the row, 1706.
template <typename X, bool PROBS, int T>
__global__ __launch_bounds__(kThreads) void score_long_kernel(const lcrc_score_args a, const Part p)
{
    constexpr int W = 16 / sizeof(X), U = 4;
    constexpr int kTeams = kThreads / T;
    __shared__ typename Team<T>::Shared shared[kTeams];
    Team<T> team(shared[threadIdx.x / T]);
    const int t = team.t, cols = a.cols, n_chunks = (cols + W - 1) / W;
    const bool want_top = wants_top(a);
    const size_t jobs = (size_t)a.rows * p.parts;
    for (size_t job = (size_t)blockIdx.x * kTeams + threadIdx.x / T; job < jobs; job += (size_t)gridDim.x * kTeams) {
        const size_t r = job / p.parts;
        const int from = (int)(job - r * p.parts) * p.chunks, to = min(from + p.chunks, n_chunks);
        const X *x = static_cast<const X *>(a.x) + r * (size_t)a.ld;
        const Label label(a, x, r, p.parts == 1 ? t : kScoreMaxLabels);
        Stats s = {PROBS ? 0.0f : kLowest, 0.0f, 0.0f};
        float least = 0.0f, most = -INFINITY, second = -INFINITY;       // the best chunk, and the best value of the others
        int most_at = -1;
        // U chunks, T apart; CHECKED: some of them may lie behind the part's end or be the row's last one
        const auto take = [&](int c0, auto checked) {
            constexpr bool CHECKED = decltype(checked)::value;
            Chunk<X, W> raw[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long at = (c0 + u * T) * (long long)W;
                raw[u] = load_chunk<X, W>(x + (CHECKED ? min(at, (long long)cols - W) : at));
            }
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + u * T;
                if (CHECKED && c >= to) break;
                // (values that the row's last chunk shares with the one before it are that one's)
                const int twice = CHECKED ? (int)max(0ll, (c + 1) * (long long)W - cols) : 0;
                float v = raw[u][W - 1];
#pragma unroll
                for (int i = 0; i < W - 1; i++)
                    if (i >= twice) v = fmaxf(v, raw[u][i]);
                const bool better = v > most || most_at < 0;
                second = fmaxf(second, better ? most : v);
                most = better ? v : most;
                most_at = better ? c : most_at;
                top = fmaxf(top, v);
            }
            if constexpr (!PROBS)
                if (top > s.m + 8.0f || (s.m == kLowest && top > s.m)) {     // the reference moves in steps: seldom
                    const float d = fmaxf(s.m - top, -1e30f), f = __builtin_amdgcn_exp2f(d * kLog2e);
                    s.T = f * fmaf(s.S, d, s.T);
                    s.S *= f;
                    s.m = top;
                }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int c = c0 + u * T;
                if (CHECKED && c >= to) break;
                const int twice = CHECKED ? (int)max(0ll, (c + 1) * (long long)W - cols) : 0;
#pragma unroll
                for (int i = 0; i < W; i++) {
                    const float v = i >= twice ? raw[u][i] : PROBS ? 0.0f : -INFINITY;
                    if constexpr (PROBS) least = fminf(least, v);
                    add_value<PROBS>(v, s);
                }
            }
        };
        const int whole = min(to, cols / W);        // chunks before it need no checks
        int c0 = from + t;
        for (; c0 - t + U * T <= whole; c0 += U * T) take(c0, std::false_type());
        for (; c0 < to; c0 += U * T) take(c0, std::true_type());
        s = team.template join<PROBS>(s, least);
        const Row<PROBS> row(s, least < 0.0f);
        if (p.parts == 1) {
            if (a.entropy && t == 0) a.entropy[r] = row.entropy();
            label.put(a, row, r, t);
        } else if (t == 0) p.stats[job] = float4{s.m, s.S, s.T, least};
        if (!want_top) continue;
        if (row.bad) {
            if (p.parts == 1 && t < a.k) put_bad(a, r, t);
            continue;                               // (a bad part makes its row bad: its list is not read)
        }
        u64 *list = p.keys + job * a.k;
        if (p.parts > 1) {
            // a part with fewer values than k leaves zeros at its list's end
            const long long here = min((long long)to * W, (long long)cols) - (long long)from * W;
            if (t < a.k && t >= here) list[t] = 0;
        }
        const auto look_at = [&](const Chunk<X, W> &raw, int c, const auto &f) {
            const long long at = c * (long long)W, start = min(at, (long long)cols - W);
#pragma unroll
            for (int i = 0; i < W; i++) f(start + i >= at, raw[i], c, (int)start + i);
        };
        const auto chunk = [&](int c) { return load_chunk<X, W>(x + min(c * (long long)W, (long long)cols - W)); };
        // bar: what f is looking for; mostly a thread has it in its best chunk alone
        const auto scan = [&](u64 bar, const auto &f) {
            if (ordered(second) < (unsigned)(bar >> 32)) {
                if (most_at >= 0) look_at(chunk(most_at), most_at, f);
                return;
            }
            for (int c = from + t; c < to; c += U * T) {
                Chunk<X, W> raw[U];
#pragma unroll
                for (int u = 0; u < U; u++) raw[u] = chunk(min(c + u * T, to - 1));
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (c + u * T < to) look_at(raw[u], c + u * T, f);
            }
        };
        const u64 first = most_at < 0 ? 0 : make_key(most, most_at);
        team.top(a.k, first, scan, [&](const auto &f) { scan(0, f); }, [&](int rank, u64 key) {
            if (p.parts == 1) put_top<PROBS>(a, r, row, rank, key);
            else list[rank] = key;
        });
    }
}

// joins the parts of each row.  All latency: 49 parts of 64 best 11 us, as much as the parts take (3 x 200003 f16).
template <typename X, bool PROBS>
__global__ __launch_bounds__(kThreads) void score_join_kernel(const lcrc_score_args a, const Part p)
{
    __shared__ Team<kThreads>::Shared shared;
    Team<kThreads> team(shared);
    const int t = team.t;
    for (size_t r = blockIdx.x; r < (size_t)a.rows; r += gridDim.x) {
        const X *x = static_cast<const X *>(a.x) + r * (size_t)a.ld;
        const Label label(a, x, r, t);
        Stats s = {PROBS ? 0.0f : kLowest, 0.0f, 0.0f};
        float least = 0.0f;
        if (t < p.parts) {                          // (parts <= kThreads)
            const float4 v = p.stats[r * p.parts + t];
            s = {v.x, v.y, v.z};
            least = v.w;
        }
        s = team.template join<PROBS>(s, least);
        const Row<PROBS> row(s, least < 0.0f);
        if (a.entropy && t == 0) a.entropy[r] = row.entropy();
        label.put(a, row, r, t);
        if (!wants_top(a)) continue;
        if (row.bad) {
            if (t < a.k) put_bad(a, r, t);
            continue;
        }
        // the parts' lists, rank by rank: the best ones lie with different threads; a key is a chunk of its own (its column)
        const u64 *keys = p.keys + r * p.parts * a.k;
        const int n = p.parts * a.k;
        // (kThreads keys further: so many ranks and lists further, without a division)
        const int by_rank = kThreads / p.parts, by_list = kThreads % p.parts, rank0 = t / p.parts, list0 = t % p.parts;
        const auto each = [&](const auto &f) {
            int rank = rank0, list = list0;
#pragma unroll 8
            for (int i = t; i < n; i += kThreads) {
                f(keys[list * a.k + rank]);
                rank += by_rank, list += by_list;
                if (list >= p.parts) list -= p.parts, rank++;
            }
        };
        u64 first = 0;
        each([&](u64 key) { first = max(first, key); });
        const auto scan = [&](u64, const auto &f) {
            each([&](u64 key) { f(key != 0, key_value(key), key_column(key), key_column(key)); });
        };
        team.top(a.k, first, scan, [&](const auto &f) { scan(0, f); }, [&](int rank, u64 key) { put_top<PROBS>(a, r, row, rank, key); });
    }
}

// ---- which kernel, on what grid ----
int most_blocks = 1 << 22;               // beyond it the workgroups take several rows each (lcrc_debug_score_blocks)

// Lists of 1, 3, 5 and 8 best and seven lengths of rows, since what a row does not need is not free (524288 rows f32, us; in the
// next longer list or length): 138 columns, 1 best 67 (76), 3 best 81 (97), 5 best 105 (162); lengths of 24 and 48 chunks: 80
// columns with 5 best 69 (77), 138 columns 105 (126), 300 columns bf16 162 (245).
template <typename X, bool PROBS, int W, int J>
void launch_short(const lcrc_score_args &a, int k, hipStream_t stream)
{
    const int blocks = (int)std::min<long long>(((long long)a.rows + kThreads / 8 - 1) / (kThreads / 8), most_blocks);
    if (k == 0) score_short_kernel<X, PROBS, W, J, 0><<<blocks, kThreads, 0, stream>>>(a);
    else if (k == 1) score_short_kernel<X, PROBS, W, J, 1><<<blocks, kThreads, 0, stream>>>(a);
    else if (k <= 3) score_short_kernel<X, PROBS, W, J, 3><<<blocks, kThreads, 0, stream>>>(a);
    else if (k <= 5) score_short_kernel<X, PROBS, W, J, 5><<<blocks, kThreads, 0, stream>>>(a);
    else score_short_kernel<X, PROBS, W, J, 8><<<blocks, kThreads, 0, stream>>>(a);
}

template <typename X, bool PROBS>
hipError_t launch(const lcrc_score_args &a, hipStream_t stream)
{
    constexpr int W = 16 / sizeof(X);
    const int k = a.top_index || a.top_logp ? a.k : 0, chunks = (a.cols - 1) / W + 1;
    if (a.cols < W) launch_short<X, PROBS, 1, 1>(a, k, stream);          // (k <= cols < 8)
    else if (k <= 8 && chunks <= 8) launch_short<X, PROBS, W, 1>(a, k, stream);
    else if (k <= 8 && chunks <= 16) launch_short<X, PROBS, W, 2>(a, k, stream);
    else if (k <= 8 && chunks <= 24) launch_short<X, PROBS, W, 3>(a, k, stream);
    else if (k <= 8 && chunks <= 32) launch_short<X, PROBS, W, 4>(a, k, stream);
    else if (k <= 8 && chunks <= 48) launch_short<X, PROBS, W, 6>(a, k, stream);
    else if (k <= 8 && chunks <= 64) launch_short<X, PROBS, W, 8>(a, k, stream);
    else if (chunks <= kScoreWaveChunks) {
        const int blocks = (int)std::min<long long>(((long long)a.rows + 3) / 4, most_blocks);
        const Part p = {1, chunks, nullptr, nullptr};
        if (chunks <= kScoreHeldChunks) score_wave_kernel<X, PROBS><<<blocks, kThreads, 0, stream>>>(a);
        else score_long_kernel<X, PROBS, 64><<<blocks, kThreads, 0, stream>>>(a, p);
    } else {
        const ScoreParts cut = score_parts(a.rows, a.cols, a.type);
        const size_t jobs = (size_t)a.rows * cut.parts;
        float4 *const stats = static_cast<float4 *>(a.workspace);
        const Part p = {cut.parts, cut.chunks, stats, reinterpret_cast<u64 *>(stats + (cut.parts > 1 ? jobs : 0))};
        score_long_kernel<X, PROBS, kThreads><<<(int)std::min<size_t>(jobs, (size_t)most_blocks), kThreads, 0, stream>>>(a, p);
        if (p.parts > 1) {
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            score_join_kernel<X, PROBS><<<std::min(a.rows, most_blocks), kThreads, 0, stream>>>(a, p);
        }
    }
    return hipGetLastError();
}

}  // namespace

int score_most_blocks(int most)
{
    const int before = most_blocks;
    most_blocks = most;
    return before;
}

hipError_t score_launch(const lcrc_score_args &a, hipStream_t stream)
{
    const auto go = [&](auto x) {
        typedef decltype(x) X;
        return a.form == LCRC_SCORE_PROBS ? launch<X, true>(a, stream) : launch<X, false>(a, stream);
    };
    if (a.type == LCRC_T_F32) return go(float());
    if (a.type == LCRC_T_F16) return go(_Float16());
    return go(__bf16());
}

}  // namespace phnrec
