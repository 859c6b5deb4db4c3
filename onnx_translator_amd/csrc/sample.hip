// sample.hip — sample_forward for gfx950: a token per row of logits by temperature, top-k,
// top-p and min-p from a given random number.
//
// Row x, temperature t, w_i = exp((x_i - max) / t).  Kept are: of the k largest x (equal ones
// by index) those whose larger ones weigh less than p of the k's weight, and of these the ones
// with w_i >= m.  So the kept set is all values above some value, and of those equal to it the
// first few by index: no sort, the border value is found digit by digit in histograms (counts
// for k, weights for p).  The token is the first kept index at which the kept weights, added up
// in index order, pass u times their sum.
//
// Weights are computed in double and summed as 64-bit fixed-point numbers: whole numbers, so
// every order of adding gives the same sum, histograms may be filled by atomics and the borders
// p and u fall where the sums in index order have them, whoever adds.  (In float32 sums a token
// beside a border would depend on the order: of 131072 tokens one row in some thousands.)  Rows that
// are spread over blocks are summed span by span against the span's largest weight and rounded once
// more when those sums are taken against the row's, by half of 2^-shift for each span or bin of a span: less
// than the weights' own roundings add up to, but a border as near as that may fall on the other
// side of a token than in a row that one block does, or with the spans that begin at another column.
#include "attention.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace tohip {
namespace {

struct SampleArgs {
    const void *x, *u;
    const float *temperature, *top_p, *min_p;          // null: not given
    IndexVec top_k;
    void* token;
    float* logprob;                                    // may be null
    int64_t ld;                                        // columns
    int rows, V, token64, u64;
    int shift;                                         // weights are whole numbers of 2^-shift
};

typedef unsigned long long u64;

// ---- one weight ------------------------------------------------------------------------
// Order-preserving key of a logit that is no NaN: -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = f2u(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return u2f(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }
// Value and index as one number: larger for larger values, and of equal ones for lower indices.
__device__ __forceinline__ u64 rank_of(float x, int i) { return ((u64)key_of(x) << 32) | (uint32_t)~i; }
__device__ __forceinline__ int index_of(u64 rank) { return (int)~(uint32_t)rank; }
__device__ __forceinline__ float value_of(u64 rank) { return of_key((uint32_t)(rank >> 32)); }

// A logit as a number whose differences are numbers too: +inf as one beyond all others.
__device__ __forceinline__ double finite(float x) { return __builtin_fmin((double)x, 1e300); }

// Against the largest of some logits: weights 2^((x - top) per).
struct Weights {
    double top, per;
    int shift;                         // in whole numbers of 2^-shift, at most 51

    // log2 of the weight, -100 for what weighs nothing in 64 bits (-inf among it)
    __device__ __forceinline__ double log2_of(float x) const { return __builtin_fmax((finite(x) - top) * per, -100.0); }
    // 2^y for -100 <= y <= 0, as the bits of 2^52 + the weight rounded to the nearest whole number:
    // the polynomial through 2^f at the eleven Chebyshev points of |f| <= 1/2 (off by 2^-51.5 of
    // itself), with whole part and shift put into its exponent.  Without a branch, and the factors
    // as scalars: else each costs two moves, more than the product.
    __device__ __forceinline__ u64 bits(double y) const {
        constexpr double kC[11] = {1.0, 0.69314718055995, 0.24022650695910097, 0.05550410866444772, 0.009618129107606888,
                                   0.0013333558230164974, 0.0001540353044173605, 1.5252657260200837e-05,
                                   1.321544258792169e-06, 1.0208690299958306e-07, 7.072585949269223e-09};
        const double n = y + 0x1.8p52, f = y - (n - 0x1.8p52);      // (n's low bits: the whole part)
        double v = kC[10];
#pragma unroll
        for (int i = 9; i >= 0; i--) {
            double c = kC[i];
            asm("" : "+s"(c));
            v = __builtin_fma(v, f, c);
        }
        const u64 b = __builtin_bit_cast(u64, v);
        const uint32_t hi = (uint32_t)(b >> 32) + (((uint32_t)__builtin_bit_cast(u64, n) + (uint32_t)shift) << 20);
        return __builtin_bit_cast(u64, __builtin_bit_cast(double, ((u64)hi << 32) | (uint32_t)b) + 0x1p52);
    }
    static constexpr u64 kBias = 0x4330000000000000ull;              // 2^52's bits
    __device__ __forceinline__ u64 of_log2(double y) const { return bits(y) - kBias; }
    __device__ __forceinline__ u64 of(float x) const { return of_log2(log2_of(x)); }
    template <int N> __device__ __forceinline__ u64 sum(const float (&x)[N]) const {
        u64 s = 0;
#pragma unroll
        for (int e = 0; e < N; e++) s += bits(log2_of(x[e]));
        return s - (u64)N * kBias;
    }
};

// ---- sums ---------------------------------------------------------------------------------
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned lanes_before(unsigned v) {      // (0 where there is none)
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS> __device__ __forceinline__ u64 lanes_before(u64 v) {
    return ((u64)lanes_before<CTRL, ROWS>((unsigned)(v >> 32)) << 32) | lanes_before<CTRL, ROWS>((unsigned)v);
}
// Sums of the wave's lanes up to and with each.
template <class T> __device__ __forceinline__ T wave_scan(T v) {
    v += lanes_before<0x111, 0xF>(v);                  // row_shr 1, 2, 4, 8: in rows of 16 lanes
    v += lanes_before<0x112, 0xF>(v);
    v += lanes_before<0x114, 0xF>(v);
    v += lanes_before<0x118, 0xF>(v);
    v += lanes_before<0x142, 0xA>(v);                  // lane 15 of the row before to rows 1 and 3
    v += lanes_before<0x143, 0xC>(v);                  // lane 31 to rows 2 and 3
    return v;
}
struct Add {
    template <class T> __device__ __forceinline__ T operator()(T x, T y) const { return x + y; }
};
struct Max {
    __device__ __forceinline__ float operator()(float x, float y) const { return fmaxf(x, y); }
};
struct Min {
    __device__ __forceinline__ int operator()(int x, int y) const { return x < y ? x : y; }
    __device__ __forceinline__ float operator()(float x, float y) const { return fminf(x, y); }
};

// Sums over a block of NT threads.  to: LDS of a number per wave.
template <int NT> struct Block {
    static constexpr int kWaves = NT / 64;
    // Of all threads before this one, and of all.
    static __device__ __forceinline__ u64 before(u64 v, u64* to, u64& total) {
        const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
        const u64 s = wave_scan(v);
        __syncthreads();                               // (the last call's are read)
        if (lane == 63) to[w] = s;
        __syncthreads();
        u64 b = 0;
        total = 0;
#pragma unroll
        for (int i = 0; i < kWaves; i++) {
            const u64 x = to[i];
            b += i < w ? x : 0;
            total += x;
        }
        return b + s - v;
    }
    template <class T, class OP> static __device__ __forceinline__ T reduce(T v, u64* waves, OP op) {
        T* to = reinterpret_cast<T*>(waves);
        v = wave_allreduce(v, op);
        __syncthreads();
        if (((int)threadIdx.x & 63) == 0) to[threadIdx.x >> 6] = v;
        __syncthreads();
        v = to[0];
#pragma unroll
        for (int i = 1; i < kWaves; i++) v = op(v, to[i]);
        return v;
    }
};

// ---- a row's settings ------------------------------------------------------------------------
struct Settings {
    double per, t, p, m;               // log2 e / t; m in [0, 1]
    int64_t k;
    bool greedy, by_k, by_p;

    __device__ __forceinline__ Settings(const SampleArgs& a, int64_t row) {
        t = a.temperature ? (double)a.temperature[row] : 1.0;
        p = a.top_p ? (double)a.top_p[row] : 1.0;
        const double low = a.min_p ? (double)a.min_p[row] : 0.0;
        m = low >= 1.0 ? 1.0 : low > 0.0 ? low : 0.0;  // (NaN: 0)
        k = a.top_k.p ? a.top_k[row] : 0;
        greedy = !(t > 0.0);
        by_k = k > 0 && k < a.V;
        by_p = p < 1.0;
        per = __builtin_fmax(1.4426950408889634 / t, 1e-60);      // (not 0: an infinite logit is beyond all others)
    }
    __device__ __forceinline__ bool filters() const { return by_k || by_p || m > 0.0; }
    // The whole number that the weights before a kept value stay below, of `total`.
    __device__ __forceinline__ u64 want(u64 total) const {
        const double w = __builtin_ceil(p * (double)total);
        return !(w >= 1.0) ? 1 : w >= (double)total ? total : (u64)w;
    }
    // 2^y (of a weight) against min-p, in double.
    __device__ __forceinline__ bool passes(double y) const { return !(m > 0.0) || exp2(y) >= m; }
    // A value that no logit passing min-p is below.
    __device__ __forceinline__ float least(float top) const {
        if (top == INFINITY) return top;
        const double x = (double)top + t * log(m);
        const float f = (float)(x - 1e-6 * __builtin_fabs(x) - 1e-30);
        return f == f ? f : -INFINITY;
    }
};
// The number below which the first of the kept weights, added up, are drawn.
__device__ __forceinline__ u64 draw_target(const SampleArgs& a, int64_t row, u64 all) {
    const double u = a.u64 ? ((const double*)a.u)[row] : (double)((const float*)a.u)[row];
    const double at = u * (double)all;
    const u64 target = !(at > 0.0) ? 0 : at >= (double)all ? all - 1 : (u64)at;
    return target < all ? target : all - 1;
}
__device__ __forceinline__ void put_token(const SampleArgs& a, int64_t row, int64_t token, float logprob) {
    if (a.token64) ((int64_t*)a.token)[row] = token;
    else ((int32_t*)a.token)[row] = (int32_t)token;
    if (a.logprob) a.logprob[row] = logprob;
}
__device__ __forceinline__ void put_drawn(const SampleArgs& a, int64_t row, int token, double y, u64 all) {
    put_token(a, row, token, (float)((y + (double)a.shift) * 0.6931471805599453 - log((double)all)));
}

// ---- logits ----------------------------------------------------------------------------------
// The logits of a row by 16-byte chunks from the one that holds its first on; -inf outside the row
// and for NaN.
template <int DT> struct RowChunks {
    static constexpr int ES = DT == kF32 ? 4 : 2, VEC = 16 / ES;
    const char* base;
    int first, V;                                      // index 0 is place `first` of the chunk at base

    __device__ __forceinline__ RowChunks(const SampleArgs& a, int64_t row) {
        const char* p = (const char*)a.x + row * a.ld * ES;
        first = (int)((uintptr_t)p & 15) / ES;
        base = p - first * ES;
        V = a.V;
    }
    __device__ __forceinline__ uint4 whole(int i) const { return *reinterpret_cast<const uint4*>(base + (int64_t)(i + first) * ES); }
    __device__ __forceinline__ uint4 part(int i) const {
        const char* p = base + (int64_t)(i + first) * ES;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (DT == kF32) {
                w[e] = i + e >= 0 && i + e < V ? ((const uint32_t*)p)[e] : 0xFF800000u;
            } else {
                constexpr uint32_t none = DT == kBF16 ? 0xFF80u : 0xFC00u;
                const uint32_t lo = i + 2 * e >= 0 && i + 2 * e < V ? ((const uint16_t*)p)[2 * e] : none;
                const uint32_t hi = i + 2 * e + 1 >= 0 && i + 2 * e + 1 < V ? ((const uint16_t*)p)[2 * e + 1] : none;
                w[e] = lo | (hi << 16);
            }
        }
        return uint4{w[0], w[1], w[2], w[3]};
    }
    // N chunks at at(0), at(1), ..., all of them between the indices lo and hi of a wave's (so that
    // inside a row the loads go out together).
    template <int N, class AT> __device__ __forceinline__ void chunks(int lo, int hi, AT at, uint4 (&q)[N]) const {
        if (lo >= 0 && hi <= V) {
#pragma unroll
            for (int c = 0; c < N; c++) q[c] = whole(at(c));
        } else {
#pragma unroll
            for (int c = 0; c < N; c++) q[c] = part(at(c));
        }
    }
    static __device__ __forceinline__ void open(uint4 q, float* x) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (DT == kF32) {
                x[e] = u2f(w[e]);
            } else if constexpr (DT == kBF16) {
                x[2 * e] = u2f(w[e] << 16);
                x[2 * e + 1] = u2f(w[e] & 0xFFFF0000u);
            } else {
                x[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
                x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) x[e] = x[e] != x[e] ? -INFINITY : x[e];
    }
};

constexpr int kBins = 2048;

// The first of n sums (thread t has those from n / NT t on, by at(i)) up to and with which they reach
// `want` (from 1 on): its number and the sum before it; -1: they do not.  found: LDS of two.
template <int NT, int N, class AT> __device__ __forceinline__ int reach(AT at, u64 want, u64* waves, u64* found, u64& before, u64& total) {
    u64 v[N], sum = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        v[e] = at(N * (int)threadIdx.x + e);
        sum += v[e];
    }
    if (threadIdx.x == 0) found[0] = ~0ull;
    u64 b = Block<NT>::before(sum, waves, total);
    if (b < want && want <= b + sum) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            if (b < want && want <= b + v[e]) {
                found[0] = (u64)(N * (int)threadIdx.x + e);
                found[1] = b;
            }
            b += v[e];
        }
    }
    __syncthreads();
    before = found[1];
    return (int)found[0];
}

// ---- few candidates --------------------------------------------------------------------------
// Where the kept tokens are known to be among at most kMost candidates these go on without the row.
// Up to kFew are ranked by counting the larger ones, which takes no barrier between its reads (100
// candidates: 5 us; with one read after the other 14); of more the border is found in bins of the
// value, and only its bin's are ranked (500 candidates: 6 us; two sorts took 25).
constexpr int kMost = 2048, kFew = 128;

template <int NT> struct Candidates {
    u64 waves[Block<NT>::kWaves], found[2];
    u64 rank[kMost], bins[kBins];
    u64 few[kMost];                    // ranks; up to kFew: with their amounts behind them
    unsigned count, few_count;
};

// Adds the logits of a wave's lanes that the bits of `in` name to a list of at most `most` (every lane
// calls: their places are found all at once); count goes on past it.
template <int N, class I> __device__ __forceinline__ void add_candidates(u64* list, unsigned* count, unsigned most, unsigned in, const float (&x)[N], I index) {
    const unsigned n = (unsigned)__builtin_popcount(in), upto = wave_scan(n), sum = (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
    if (!sum) return;
    unsigned at = ((int)threadIdx.x & 63) == 0 ? atomicAdd(count, sum) : 0;
    at = (unsigned)__builtin_amdgcn_readfirstlane((int)at) + upto - n;
#pragma unroll
    for (int e = 0; e < N; e++) {
        if (in >> e & 1) {
            if (at < most) list[at] = rank_of(x[e], index(e));
            at++;
        }
    }
}

// f(rank, amount) for n ranks and amounts in LDS (which have room for a multiple of eight), eight reads
// of each at a time: one after the other they wait for LDS 128 cycles each.
template <class F> __device__ __forceinline__ void each_few(const u64* rank, const u64* amount, int n, F f) {
    for (int j = 0; j < n; j += 8) {
        u64 r[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) r[e] = rank[j + e];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = amount[j + e];
#pragma unroll
        for (int e = 0; e < 8; e++) f(r[e], j + e < n ? v[e] : 0);
    }
}

// n numbers in LDS, n a power of two, in falling order.  (Pairs at most 64 apart lie in one wave's part.)
template <int NT> __device__ __forceinline__ void sort_falling(u64* v, int n) {
    __syncthreads();
    for (int size = 2; size <= n; size *= 2) {
        for (int step = size / 2; step > 0; step /= 2) {
            if (step >= 64) __syncthreads();
            else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            for (int t = (int)threadIdx.x; t < n / 2; t += NT) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const u64 x = v[i], y = v[j];
                if ((x < y) == ((i & size) == 0)) {
                    v[i] = y;
                    v[j] = x;
                }
            }
            if (step == 64) __syncthreads();
        }
    }
    __syncthreads();
}

// Of the ranks in a list, from the largest down, the last one before which amounts of less than `want`
// lie, `base` among them (0: all are such).  amount(rank): 0 for one that does not count.  lo, hi: bounds
// of their values.  bins: LDS of kBins, few of kMost.
template <int NT, class A> __device__ __forceinline__ u64 border_of(u64* list, int count, float lo, float hi, u64 base, u64 want, A amount, u64* bins, u64* few,
                                                    unsigned* few_count, u64* waves, u64* found) {
    const int tid = (int)threadIdx.x;
    u64 above = base, total;
    int n = count;
    u64* from = list;
    if (count > kFew) {
        const float scale = (float)(kBins - 1) / (hi - lo);
        auto bin_of = [&](u64 rank) {                  // (NaN of equal or infinite ones: bin 0)
            const float f = (hi - value_of(rank)) * scale;
            return f > 0.0f ? (int)fminf(f, kBins - 1) : 0;
        };
        __syncthreads();
        for (int i = tid; i < kBins; i += NT) bins[i] = 0;
        if (tid == 0) *few_count = 0;
        __syncthreads();
        for (int i = tid; i < count; i += NT) {
            const u64 v = amount(list[i]);
            if (v) atomicAdd(&bins[bin_of(list[i])], v);
        }
        __syncthreads();
        const int bin = reach<NT, kBins / NT>([&](int i) { return bins[i]; }, want - base, waves, found, above, total);
        above += base;
        if (bin < 0) return 0;
        for (int i = tid; i < count; i += NT)
            if (bin_of(list[i]) == bin && amount(list[i])) few[atomicAdd(few_count, 1u)] = list[i];
        __syncthreads();
        n = (int)*few_count;
        from = few;
    }
    if (tid == 0) found[0] = ~0ull;
    if (n <= kFew) {
        const u64 mine = tid < n ? from[tid] : 0, own = mine ? amount(mine) : 0;
        u64* amounts = few + kFew;
        if (tid < n) amounts[tid] = own;
        __syncthreads();
        u64 before = above, all = above;
        if (tid < (n + 63) / 64 * 64) {
            each_few(from, amounts, n, [&](u64 rank, u64 v) {
                before += rank > mine ? v : 0;
                all += v;
            });
        }
        if (tid == 0) found[1] = all;
        if (own && before < want) atomicMin(&found[0], mine);
        __syncthreads();
        const u64 border = found[1] < want ? 0 : found[0];
        __syncthreads();
        return border;
    }
    int m = 2 * kFew;
    while (m < n) m *= 2;
    for (int i = n + tid; i < m; i += NT) few[i] = 0;
    sort_falling<NT>(few, m);
    constexpr int E = kMost / NT;
    u64 v[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        v[e] = E * tid + e < n ? amount(few[E * tid + e]) : 0;
        sum += v[e];
    }
    u64 before = above + Block<NT>::before(sum, waves, total);
#pragma unroll
    for (int e = 0; e < E; e++) {
        if (v[e] && before < want) atomicMin(&found[0], few[E * tid + e]);
        before += v[e];
    }
    __syncthreads();
    const u64 border = found[0];
    __syncthreads();
    return border;
}

// Draws from the c.count <= kMost candidates of top-k or of min-p alone (they hold all that those keep;
// none is below `least`).
template <int NT> __device__ __forceinline__ void draw_candidates(const SampleArgs& a, int64_t row, const Settings& g, const Weights& w, float least, float top,
                                                                  Candidates<NT>& c) {
    const int tid = (int)threadIdx.x;
    __syncthreads();
    const int count = (int)c.count, most = g.by_k && g.k < count ? (int)g.k : count;
    if (count <= kFew) {
        // a candidate per thread; the larger ones and their weights, then the kept ones before it
        u64 *mass = c.few, *kept = c.few + kFew;
        const u64 mine = tid < count ? c.rank[tid] : 0;
        const double y = mine ? w.log2_of(value_of(mine)) : -100.0;
        const u64 own = mine ? w.of_log2(y) : 0;
        if (tid < (count + 7) / 8 * 8) {
            c.rank[tid] = mine;                        // (0 behind the last)
            mass[tid] = own;
        }
        __syncthreads();
        int larger = 0;
        u64 above = 0;
        if (tid < (count + 63) / 64 * 64) {
            each_few(c.rank, mass, count, [&](u64 rank, u64 v) {
                larger += rank > mine;
                above += rank > mine ? v : 0;
            });
        }
        const bool ranked = mine && larger < most;
        u64 total = 0;
        if (g.by_p) total = Block<NT>::reduce(ranked ? own : 0, c.waves, Add());
        const bool keep = ranked && (!g.by_p || above < g.want(total)) && g.passes(y);
        if (tid < count) kept[tid] = keep ? own : 0;
        const u64 all = Block<NT>::reduce(keep ? own : 0, c.waves, Add());
        const u64 target = draw_target(a, row, all);
        u64 before = 0;
        if (keep) {
            each_few(c.rank, kept, count, [&](u64 rank, u64 v) { before += (uint32_t)rank > (uint32_t)mine ? v : 0; });      // (~index)
            if (before <= target && target < before + own) put_drawn(a, row, index_of(mine), y, all);
        }
        return;
    }
    if (!(least > -INFINITY)) {                        // (few logits in all)
        least = top;
        for (int i = tid; i < count; i += NT) least = fminf(least, value_of(c.rank[i]));
        least = Block<NT>::reduce(least, c.waves, Min());
    }
    u64 border = 0, total;
    if (most < count)
        border = border_of<NT>(c.rank, count, least, top, 0, (u64)most, [](u64) { return (u64)1; }, c.bins, c.few, &c.few_count, c.waves, c.found);
    if (g.by_p) {
        auto weight = [&](u64 rank) { return rank >= border ? w.of(value_of(rank)) : 0; };
        u64 sum = 0;
        for (int i = tid; i < count; i += NT) sum += weight(c.rank[i]);
        sum = Block<NT>::reduce(sum, c.waves, Add());
        const u64 by_p = border_of<NT>(c.rank, count, least, top, 0, g.want(sum), weight, c.bins, c.few, &c.few_count, c.waves, c.found);
        border = by_p > border ? by_p : border;
    }
    // the kept weights by index, then those of the bin that the target falls into
    const int per = (a.V + kBins - 1) / kBins;
    auto kept = [&](u64 rank) {
        const double y = w.log2_of(value_of(rank));
        return rank >= border && g.passes(y) ? w.of_log2(y) : 0;
    };
    __syncthreads();
    for (int i = tid; i < kBins; i += NT) c.bins[i] = 0;
    if (tid == 0) c.few_count = 0;
    __syncthreads();
    u64 sum = 0;
    for (int i = tid; i < count; i += NT) {
        const u64 v = kept(c.rank[i]);
        if (v) atomicAdd(&c.bins[index_of(c.rank[i]) / per], v);
        sum += v;
    }
    const u64 all = Block<NT>::reduce(sum, c.waves, Add()), target = draw_target(a, row, all);
    u64 before;
    const int bin = reach<NT, kBins / NT>([&](int i) { return c.bins[i]; }, target + 1, c.waves, c.found, before, total);
    for (int i = tid; i < count; i += NT)
        if (index_of(c.rank[i]) / per == bin && kept(c.rank[i])) c.few[atomicAdd(&c.few_count, 1u)] = c.rank[i];
    __syncthreads();
    const int n = (int)c.few_count;
    for (int i = tid; i < n; i += NT) {
        const u64 mine = c.few[i], own = kept(mine);
        u64 at = before;
        for (int j = 0; j < n; j++) at += (uint32_t)c.few[j] > (uint32_t)mine ? kept(c.few[j]) : 0;
        if (at <= target && target < at + own) put_drawn(a, row, index_of(mine), w.log2_of(value_of(mine)), all);
    }
}

// ---- any number of candidates, in one block ---------------------------------------------------
constexpr int kEach = 8;                               // logits of a thread in a tile, in index order
constexpr int kHeld = 4;                               // tiles that a block holds in registers
constexpr int kMaxTiles = 2048, kRowThreads = 1024, kShortThreads = 256;      // (16 M columns)

template <int NT> struct Histograms {
    u64 waves[Block<NT>::kWaves];
    u64 bins[kBins];
    u64 tile_mass[kMaxTiles];
    uint32_t tile_ties[kMaxTiles];
    u64 found[2];
};
template <int NT> union SampleShared {
    Histograms<NT> h;
    Candidates<NT> c;
};

// A row in tiles, from its first chunk on; HELD: all of them (at most kHeld) stay in registers.
template <int DT, int NT, bool HELD> struct SampleRow : RowChunks<DT> {
    typedef RowChunks<DT> Chunks;
    static constexpr int PER = kEach / Chunks::VEC;    // chunks of a thread in a tile
    static constexpr int kTile = NT * kEach;
    int tiles;
    uint4 held[HELD ? kHeld : 1][PER];

    __device__ __forceinline__ SampleRow(const SampleArgs& a, int64_t row) : Chunks(a, row) {
        tiles = (this->first + this->V + kTile - 1) / kTile;
        if constexpr (HELD) {
#pragma unroll
            for (int i = 0; i < kHeld; i++) raw(i, held[i]);
        }
    }
    __device__ __forceinline__ int index(int tile) const { return tile * kTile + (int)threadIdx.x * kEach - this->first; }
    __device__ __forceinline__ void raw(int tile, uint4 (&q)[PER]) const {
        const int lo = tile * kTile + __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63) * kEach - this->first;
        this->chunks(lo, lo + 64 * kEach, [&](int c) { return index(tile) + c * Chunks::VEC; }, q);
    }
    __device__ __forceinline__ void load(int tile, float (&x)[kEach]) const {
        uint4 q[PER];
        raw(tile, q);
#pragma unroll
        for (int c = 0; c < PER; c++) Chunks::open(q[c], x + c * Chunks::VEC);
    }
    // f(tile, logits) for every tile in index order
    template <class F> __device__ __forceinline__ void each(F f) const { each(f, 0, tiles); }
    // ... from tile `from` on (0 where they are held) and before `to`.
    template <class F> __device__ __forceinline__ void each(F f, int from, int to) const {
        if constexpr (HELD) {
#pragma unroll
            for (int tile = 0; tile < kHeld; tile++) {
                if (tile >= to) break;
                float x[kEach];
#pragma unroll
                for (int c = 0; c < PER; c++) {
                    uint4 q = held[tile][c];           // (opened anew each time: kept open, they take twice the registers)
                    asm volatile("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w));
                    Chunks::open(q, x + c * Chunks::VEC);
                }
                f(tile, x);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            // Eight chunks of a thread at once: a CU has a microsecond's way to memory, and one or two
            // chunks of each thread on it are a tenth of what it could have.
            constexpr int BATCH = 8 / PER;
            for (int tile0 = from; tile0 < to; tile0 += BATCH) {
                uint4 q[BATCH][PER];
                const int lo = tile0 * kTile - this->first;
                if (lo >= 0 && lo + BATCH * kTile <= this->V && tile0 + BATCH <= to) {
#pragma unroll
                    for (int i = 0; i < BATCH; i++)
#pragma unroll
                        for (int c = 0; c < PER; c++) q[i][c] = this->whole(index(tile0 + i) + c * Chunks::VEC);
                } else {
#pragma unroll
                    for (int i = 0; i < BATCH; i++)
                        if (tile0 + i < to) raw(tile0 + i, q[i]);
                }
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    if (tile0 + i >= to) break;
                    float x[kEach];
#pragma unroll
                    for (int c = 0; c < PER; c++) Chunks::open(q[i][c], x + c * Chunks::VEC);
                    f(tile0 + i, x);
                }
            }
        }
    }
};

// Draws among the logits whose rank is at least `border` and that pass min-p, from the tiles' weights.
template <int DT, int NT, class ROW> __device__ __forceinline__ void draw_tile(const SampleArgs& a, int64_t row, const ROW& r, const Settings& g, const Weights& w,
                                                               u64 border, float least, Histograms<NT>& s) {
    u64 all = 0, total;
    for (int i = 0; i < r.tiles; i++) all += s.tile_mass[i];
    u64 target = draw_target(a, row, all);
    int tile = 0;
    for (; tile + 1 < r.tiles && target >= s.tile_mass[tile]; tile++) target -= s.tile_mass[tile];
    float x[kEach];
    u64 v[kEach], mine = 0;
    r.load(tile, x);
#pragma unroll
    for (int e = 0; e < kEach; e++) {
        const double y = w.log2_of(x[e]);
        v[e] = x[e] >= least && rank_of(x[e], r.index(tile) + e) >= border && g.passes(y) ? w.of_log2(y) : 0;
        mine += v[e];
    }
    u64 from = Block<NT>::before(mine, s.waves, total);
    if (from <= target && target < from + mine) {
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            if (from <= target && target < from + v[e]) put_drawn(a, row, r.index(tile) + e, w.log2_of(x[e]), all);
            from += v[e];
        }
    }
}

// Kept are the values above some border value and the first few equal to it.  The border is found
// digit by digit from the highest values down, in histograms of counts (top-k) or weights (top-p).
template <int DT, int NT, class ROW> __device__ __forceinline__ void draw_any(const SampleArgs& a, int64_t row, const ROW& r, const Settings& g, const Weights& wt,
                                                              Histograms<NT>& s) {
    constexpr int kRounds = DT == kF32 ? 3 : 2;        // digits of 11, 11 and 10 bits; 16-bit logits differ in the first two
    const int tid = (int)threadIdx.x;
    uint32_t border = 0;                               // (no key: everything is kept)
    u64 ties = 0, equal = 0;                           // equal: keys that are the border's, of those ranked at all
    // The value at which the sums of amount(x) over the keys >= least pass want_of(their total), and
    // the sum above it; false: they do not.  less: what to take off the sum of least's own bin.
    auto search = [&](auto amount, uint32_t least, u64 less, auto want_of, u64& above) {
        uint32_t prefix = 0;
        u64 want = 0, within = 0;
        above = 0;
        for (int round = 0; round < kRounds; round++) {
            const int low = round == 0 ? 21 : round == 1 ? 10 : 0, width = round == 2 ? 10 : 11;
            __syncthreads();
            for (int i = tid; i < kBins; i += NT) s.bins[i] = 0;
            __syncthreads();
            r.each([&](int, const float (&x)[kEach]) {
#pragma unroll
                for (int e = 0; e < kEach; e++) {
                    const uint32_t key = key_of(x[e]);
                    if (x[e] == -INFINITY || key < least) continue;
                    if (round && (key >> (low + width)) != prefix) continue;
                    const u64 v = amount(x[e]);
                    if (v) atomicAdd(&s.bins[(key >> low) & ((1u << width) - 1)], v);
                }
            });
            __syncthreads();
            if (less && tid == 0 && (!round || (least >> (low + width)) == prefix))
                s.bins[(least >> low) & ((1u << width) - 1)] -= less;
            __syncthreads();
            if (round == 0) {
                u64 sum = 0;
                for (int i = tid; i < kBins; i += NT) sum += s.bins[i];
                const u64 total = Block<NT>::reduce(sum, s.waves, Add());
                want = want_of(total);
                if (!want || want > total) return false;
            }
            u64 over, total;
            const int bin = kBins - 1 - reach<NT, kBins / NT>([&](int i) { return s.bins[kBins - 1 - i]; }, want - above, s.waves, s.found, over, total);
            above += over;
            within = s.bins[bin];
            prefix = (prefix << width) | (uint32_t)bin;
        }
        if (kRounds == 2) prefix = prefix & (1u << 21) ? prefix << 10 : (prefix << 10) | 0x3FF;      // the digits all values share
        border = prefix;
        equal = within;
        return true;
    };

    if (g.by_k) {
        u64 above;
        if (search([](float) { return (u64)1; }, 0u, 0, [&](u64) { return (u64)g.k; }, above)) ties = (u64)g.k - above;
    }
    if (g.by_p) {
        // of border's equals only `ties` are there
        const uint32_t least = border;
        const u64 own = least ? wt.of(of_key(least)) : 0, gone = least ? (equal - ties) * own : 0;
        u64 above, want = 0;
        const bool some = search([&](float x) { return wt.of(x); }, least, gone, [&](u64 total) { return want = g.want(total); }, above);
        if (some) {
            const u64 each = wt.of(of_key(border)), n = equal / each;            // (each > 0: the sums pass want here)
            ties = (want - above + each - 1) / each;
            ties = ties < 1 ? 1 : ties > n ? n : ties;
            equal = border == least ? n + (gone / (own ? own : 1)) : n;
        }
    }
    const bool some_ties = border && ties < equal;     // the ties are told apart by index

    // ---- the kept weights, tile by tile in index order
    // Weights of this thread's logits; before: equals of the border in the tiles and threads before.
    auto weigh = [&](const float (&x)[kEach], u64 before, u64 (&v)[kEach]) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t key = key_of(x[e]);
            bool keep = x[e] > -INFINITY && key >= border;
            if (some_ties && key == border) keep = keep && before++ < ties;
            const double y = wt.log2_of(x[e]);
            v[e] = keep && g.passes(y) ? wt.of_log2(y) : 0;
            sum += v[e];
        }
        return sum;
    };
    auto count_ties = [&](const float (&x)[kEach]) {
        u64 n = 0;
#pragma unroll
        for (int e = 0; e < kEach; e++) n += x[e] > -INFINITY && key_of(x[e]) == border;
        return n;
    };
    u64 all = 0, met = 0;
    __syncthreads();
    r.each([&](int tile, const float (&x)[kEach]) {
        u64 v[kEach], before = 0, total;
        if (tid == 0) s.tile_ties[tile] = (uint32_t)met;
        if (some_ties) {
            before = met + Block<NT>::before(count_ties(x), s.waves, total);
            met += total;
        }
        total = Block<NT>::reduce(weigh(x, before, v), s.waves, Add());
        if (tid == 0) s.tile_mass[tile] = total;
        all += total;
    });
    __syncthreads();

    // ---- the draw
    u64 target = draw_target(a, row, all);
    int tile = 0;
    for (; tile + 1 < r.tiles && target >= s.tile_mass[tile]; tile++) target -= s.tile_mass[tile];
    float x[kEach];
    u64 v[kEach], before = 0, total;
    r.load(tile, x);
    if (some_ties) before = s.tile_ties[tile] + Block<NT>::before(count_ties(x), s.waves, total);
    const u64 mine = weigh(x, before, v);
    u64 from = Block<NT>::before(mine, s.waves, total);
    if (from <= target && target < from + mine) {
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            if (from <= target && target < from + v[e]) put_drawn(a, row, r.index(tile) + e, wt.log2_of(x[e]), all);
            from += v[e];
        }
    }
}

// A value that at least k logits are no less than, from the largest logits of some groups of them
// (visit(f) calls f with the thread's): counted in bins between the least and the largest of these,
// lo and top.  -inf: there are fewer groups.  (Where these are equal or so near that scale is past
// float32, the bins' edges say nothing and it is lo.)
template <int NT, class V> __device__ __forceinline__ float kth_bound(V visit, u64 k, float lo, float top, Histograms<NT>& s) {
    const float scale = (float)(kBins - 1) / (top - lo);
    __syncthreads();
    for (int i = (int)threadIdx.x; i < kBins; i += NT) s.bins[i] = 0;
    __syncthreads();
    visit([&](float x) {
        if (x == -INFINITY) return;
        const float f = (top - x) * scale;             // (NaN of equal or infinite ones: bin 0)
        atomicAdd(&s.bins[f > 0.0f ? (int)fminf(f, kBins - 1) : 0], (u64)1);
    });
    __syncthreads();
    u64 before, total;
    const int bin = reach<NT, kBins / NT>([&](int i) { return s.bins[i]; }, k, s.waves, s.found, before, total);
    if (bin < 0) return -INFINITY;
    if (!(scale < INFINITY)) return top < INFINITY ? lo : -INFINITY;
    const float edge = top - (float)(bin + 1) / scale;                 // (rounded: down by more than its own errors)
    const float least = edge - 1e-5f * (__builtin_fabsf(top) + __builtin_fabsf(lo));
    return least == least && top < INFINITY ? least : -INFINITY;
}

// Among the `count` ranks of the border's bin (weights above it: `above`) the last that top-p keeps;
// kept(rank, weight), for every lane of a wave, with the weight 0 where it is not kept.  bins: LDS of
// kBins.  Logits of 16 bits have few values, so many may be equal there: then as many are kept as
// their weight goes into what is wanted, and the last one's index is found by counting.
template <int NT, class F> __device__ __forceinline__ u64 border_in(u64* list, int count, u64 above, u64 want, const Settings& g, const Weights& w, u64* waves,
                                                     u64* found, unsigned* bins, int V, F kept) {
    const int tid = (int)threadIdx.x;
    constexpr int E = kMost / NT;
    float lo = INFINITY, hi = -INFINITY;
    for (int i = tid; i < count; i += NT) {
        const float x = value_of(list[i]);
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
    }
    lo = Block<NT>::reduce(lo, waves, Min());
    hi = Block<NT>::reduce(hi, waves, Max());
    u64 total, before;
    if (lo == hi && count > kFew) {
        const u64 each = w.of(hi);
        const int n = (int)min((want - above + each - 1) / each, (u64)count);        // (each > 0: the bin's weights pass want)
        // the n-th smallest index: its bin of indices, then among that bin's
        const int per = (V + kBins - 1) / kBins;
        for (int i = tid; i < kBins; i += NT) bins[i] = 0;
        __syncthreads();
        for (int i = tid; i < count; i += NT) atomicAdd(&bins[index_of(list[i]) / per], 1u);
        __syncthreads();
        const int bin = reach<NT, kBins / NT>([&](int i) { return (u64)bins[i]; }, (u64)n, waves, found, before, total);
        __syncthreads();
        unsigned* some_ = (unsigned*)(found + 1);
        if (tid == 0) *some_ = 0;
        __syncthreads();
        for (int i = tid; i < count; i += NT)          // (at most kBins: in the bins' place)
            if (index_of(list[i]) / per == bin) bins[atomicAdd(some_, 1u)] = (unsigned)index_of(list[i]);
        __syncthreads();
        const int some = (int)*some_, nth = n - (int)before;
        for (int i = tid; i < some; i += NT) {
            int less = 0;
            for (int j = 0; j < some; j++) less += bins[j] < bins[i];
            if (less == nth - 1) found[0] = rank_of(hi, (int)bins[i]);
        }
        __syncthreads();
    } else if (count <= kFew) {
        // (behind the list is room)
        const u64 b = border_of<NT>(list, count, lo, hi, above, want, [&](u64 rank) { return w.of(value_of(rank)); }, list, list + kMost / 2, nullptr, waves, found);
        if (tid == 0) found[0] = b;
        __syncthreads();
    } else {
        int n = 64;
        while (n < count) n *= 2;
        for (int i = count + tid; i < n; i += NT) list[i] = 0;
        sort_falling<NT>(list, n);
        u64 v[E], sum = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            v[e] = E * tid + e < count ? w.of(value_of(list[E * tid + e])) : 0;
            sum += v[e];
        }
        if (tid == 0) found[0] = ~0ull;
        before = above + Block<NT>::before(sum, waves, total);
#pragma unroll
        for (int e = 0; e < E; e++) {
            if (E * tid + e < count && before < want) atomicMin(&found[0], list[E * tid + e]);
            before += v[e];
        }
        __syncthreads();
    }
    const u64 border = found[0];
    for (int i = tid; i < (count + 63) / 64 * 64; i += NT) {
        const u64 rank = i < count ? list[i] : 0;
        const float x = value_of(rank);
        kept(rank, rank && rank >= border && g.passes(w.log2_of(x)) ? w.of(x) : 0);
    }
    __syncthreads();
    return border;
}

// The smallest key whose value holds(value) is true of, which it is of all larger ones: sixty-four
// keys at a time.  (That of a NaN above all values: there is none.)
template <class F> __device__ __forceinline__ uint32_t first_key(F holds) {
    const uint32_t lane = threadIdx.x & 63, top = 0xFF800000u, bottom = 0x007FFFFFu;      // +inf, -inf
    uint32_t not_yet = 0;
#pragma unroll
    for (int shift = 26; shift >= -4; shift -= 6) {
        const int s = shift < 0 ? 0 : shift;
        const uint32_t key = not_yet + (lane << s);
        const bool yes = (shift < 0 && lane > 3) || key > top || (key > bottom && holds(of_key(key)));
        const unsigned long long no = ~__ballot(yes);              // (lane 0's among them)
        not_yet += (uint32_t)(63 - __builtin_clzll(no | 1)) << s;
    }
    return not_yet + 1;
}

// Bins of a weight's logarithm from the largest down.
__device__ __forceinline__ int log_bin(double y) { return min((int)(y * -51.0), kBins - 1); }      // (51 to a factor of two: 40 of them)

// A block per row.  HELD: the row is read once, into registers.  Bound by one CU's double products and
// LDS atomics where top-p weighs the whole row (32000 logits: 42 us, of them 9 for the histogram,
// 6 .. 10 for the second pass), else by its chain of barriers (top-k of 50: 16 us, greedy 6).  Where
// the row is read again for each pass (HELD false) the compiler spills 60 .. 160 bytes a thread of 1024
// (131072 bfloat16 by top-p: 100 us one row, 117 64 rows; by temperature 42).
template <int DT, int NT, bool HELD> __global__ __launch_bounds__(NT) void k_sample_row(SampleArgs a) {
    __shared__ SampleShared<NT> s;
    typedef Block<NT> B;
    const int64_t row = blockIdx.x;
    const int tid = (int)threadIdx.x;
    const SampleRow<DT, NT, HELD> r(a, row);
    const Settings g(a, row);

    // ---- the largest value
    float most = -INFINITY;
    auto largest = [](const float (&x)[kEach]) {
        float v = x[0];
#pragma unroll
        for (int e = 1; e < kEach; e++) v = fmaxf(v, x[e]);
        return v;
    };
    r.each([&](int, const float (&x)[kEach]) { most = fmaxf(most, largest(x)); });
    const float top = B::reduce(most, s.h.waves, Max());
    if (top == -INFINITY) {
        if (tid == 0) put_token(a, row, -1, -INFINITY);
        return;
    }
    if (g.greedy) {                                    // and where it is first
        int at = 0x7FFFFFFF;
        r.each([&](int tile, const float (&x)[kEach]) {
#pragma unroll
            for (int e = kEach - 1; e >= 0; e--) at = x[e] == top ? min(at, r.index(tile) + e) : at;
        });
        at = B::reduce(at, s.h.waves, Min());
        if (tid == 0) put_token(a, row, at, 0.0f);
        return;
    }
    const Weights w = {finite(top), g.per, a.shift};

    do {
        // ---- top-k, or min-p alone: few candidates, where few are above what none kept is below
        if (g.by_k || (!g.by_p && g.m > 0.0)) {
            float least = -INFINITY;
            if (g.by_k) {
                // (groups: a thread's logits of a tile)
                float lo = top;
                r.each([&](int, const float (&x)[kEach]) {
                    const float v = largest(x);
                    lo = v > -INFINITY ? fminf(lo, v) : lo;
                });
                lo = B::reduce(lo, s.h.waves, Min());
                least = kth_bound<NT>([&](auto f) { r.each([&](int, const float (&x)[kEach]) { f(largest(x)); }); }, (u64)g.k, lo, top, s.h);
            }
            if (g.m > 0.0 && !g.by_p) least = fmaxf(least, g.least(top));
            __syncthreads();
            if (tid == 0) s.c.count = 0;
            __syncthreads();
            r.each([&](int tile, const float (&x)[kEach]) {
                unsigned in = 0;
#pragma unroll
                for (int e = 0; e < kEach; e++) in |= x[e] >= least && x[e] > -INFINITY ? 1u << e : 0;
                add_candidates(s.c.rank, &s.c.count, kMost, in, x, [&](int e) { return r.index(tile) + e; });
            });
            __syncthreads();
            if (s.c.count <= kMost) {
                draw_candidates<NT>(a, row, g, w, least, top, s.c);
                return;
            }
            break;
        }
        // ---- no filter, or top-p: the weights by their logarithm, then those above the border's bin by
        // tile, and the bin's own one by one
        Histograms<NT>& h = s.h;
        u64 border = 0;
        int bin = kBins;
        u64 above = 0, want = 0;
        if (g.by_p) {
            __syncthreads();
            for (int i = tid; i < kBins; i += NT) h.bins[i] = 0;
            __syncthreads();
            r.each([&](int, const float (&x)[kEach]) {
#pragma unroll
                for (int e = 0; e < kEach; e++) {
                    const double y = w.log2_of(x[e]);
                    const u64 v = w.of_log2(y);
                    if (v) atomicAdd(&h.bins[log_bin(y)], v);
                }
            });
            __syncthreads();
            u64 sum = 0, total;
            for (int i = tid; i < kBins; i += NT) sum += h.bins[i];
            sum = B::reduce(sum, h.waves, Add());
            want = g.want(sum);
            bin = reach<NT, kBins / NT>([&](int i) { return h.bins[i]; }, want, h.waves, h.found, above, total);
            if (bin == kBins - 1) break;                   // (among weights below 2^-40)
            __syncthreads();
            if (tid == 0) h.tile_ties[0] = 0;              // the bin's count; its ranks go where the bins were
            __syncthreads();
        }
        const int lane = tid & 63;
        for (int i = tid; i < r.tiles; i += NT) h.tile_mass[i] = 0;
        __syncthreads();
        // (the bin's logits are those from lo on and below hi)
        float lo = 0.0f, hi = 0.0f;
        if (g.by_p) {
            lo = of_key(first_key([&](float x) { return log_bin(w.log2_of(x)) <= bin; }));
            hi = of_key(first_key([&](float x) { return log_bin(w.log2_of(x)) < bin; }));
            if (!(hi == hi)) hi = INFINITY;                // (none is above: the first bin, in which a +inf is)
        }
        r.each([&](int tile, const float (&x)[kEach]) {
            u64 sum = 0;
            if (!g.by_p) {
                sum = w.sum(x);
            } else {
                unsigned in = 0, over = 0;
#pragma unroll
                for (int e = 0; e < kEach; e++) {
                    const bool above_bin = bin > 0 && x[e] >= hi;
                    over |= above_bin ? 1u << e : 0;
                    in |= x[e] >= lo && !above_bin ? 1u << e : 0;
                }
                if (__ballot(over != 0)) {                 // (all of a wave's or none: eight branches take twice as long)
#pragma unroll
                    for (int e = 0; e < kEach; e++) {
                        const double y = w.log2_of(x[e]);
                        const u64 v = w.of_log2(y);
                        sum += (over >> e & 1) && g.passes(y) ? v : 0;
                    }
                }
                add_candidates(h.bins, &h.tile_ties[0], kBins, in, x, [&](int e) { return r.index(tile) + e; });
            }
            sum = wave_allreduce(sum, Add());
            if (lane == 0 && sum) atomicAdd(&h.tile_mass[tile], sum);
        });
        __syncthreads();
        if (g.by_p) {
            const int count = (int)h.tile_ties[0];
            if (count > kBins) break;                  // (many equal ones)
            border = border_in<NT>(h.bins, count, above, want, g, w, h.waves, h.found, h.tile_ties, a.V, [&](u64 rank, u64 v) {
                if (v) atomicAdd(&h.tile_mass[(index_of(rank) + r.first) / r.kTile], v);
            });
        }
        draw_tile<DT, NT>(a, row, r, g, w, border, -FLT_MAX, h);
        return;
    } while (false);
    // ---- too many candidates
    __syncthreads();
    draw_any<DT, NT>(a, row, r, g, w, s.h);
}

// ---- a row spread over blocks -----------------------------------------------------------------
// Few long rows would leave most of the GPU idle, and many are read more often than need be by a
// block each.  So one launch reads all logits once and leaves, of every 4096 of a row (a span), the
// largest value, the sum of the weights against it, and, where top-p or min-p may need them, these sums
// by the weights' logarithm; of every 16 the largest value.  A block per row goes on from those:
// with top-k the few logits that can be kept, else the span that the draw falls into, and for a
// border the logits whose logarithm is the border's.
// (64 x 131072 bfloat16 by top-p: 18 us for the spans and 60 for the rows, a block per row 117;
// 256 x 131072 float32 by temperature: 39 us, 3.4 TB/s with 34 M weights in double on the way, which keep
// the vector units busy for 78 % of it, and 8, a block per row 62.  A row with a border: 25 us to find the logits in its bins, four operations
// for each of 131072 on one CU, so of few rows several blocks do that, and the last one that is done
// goes on; 10 for the finer bins, 5 for the border.)
constexpr int kSpanThreads = 256, kSpan = 16 * kSpanThreads;
constexpr int kPickThreads = 512;                      // (1024 have half the registers: spills cost every row 6 us)
constexpr int kSpans = 512;                            // of a row at most
constexpr int kLogBins = 128;                          // four to a factor of two, from a span's largest down
constexpr int kNear = 12288;                           // logits of the border's bins

struct Spread {
    float *largest, *group;            // of each span, and of each 16 logits
    u64 *mass, *bins;                  // of each span
    u64* near;                         // of each row, with several parts: the logits of its border's bins
    unsigned *count, *done;            // how many those are, and parts that have added theirs
    int spans;                         // of a row
    int parts;                         // blocks that look for a row's border's logits
};
// Parts of a row: no more blocks than CUs, and of many rows enough logits each to be worth the fences
// between their blocks (by top-p, us with one part and with these: 1 x 250000 106 and 64; 16 x 131072
// 77 and 62; 33 x 131072 79 and 65; 64 x 131072 85 and 78, 64 x 40000 41 and, with four, 47; 100 x
// 131072 91 and 89, 100 x 40000 43 and, with two, 48; sixteen parts 60 and 64 for the first two).
inline int parts_of(int64_t rows, int64_t V) {
    if (rows <= 32) return 8;
    if (rows <= 64) return (int)std::max<int64_t>(1, std::min<int64_t>(4, V / 24576));
    return rows <= 128 && V >= 131072 ? 2 : 1;
}

// A logit's logarithm in bins, downwards, from that of 0 on: the same for all spans and launches.
__device__ __forceinline__ double grid_of(float x, double per) { return -__builtin_floor(finite(x) * (per * 4.0)); }

// Chunk i of a lane's 16 logits of a span: its first index.
template <int DT> __device__ __forceinline__ int span_index(const RowChunks<DT>& r, int span, int group, int i) {
    return span * kSpan + (group >> 6) * 1024 + i * 64 * RowChunks<DT>::VEC + (group & 63) * RowChunks<DT>::VEC - r.first;
}

template <int DT> __global__ __launch_bounds__(kSpanThreads) void k_sample_spans(SampleArgs a, Spread w) {
    __shared__ u64 bins[kLogBins], waves[kSpanThreads / 64];
    typedef Block<kSpanThreads> B;
    constexpr int N = 16 / RowChunks<DT>::VEC;
    const int64_t row = blockIdx.x / (unsigned)w.spans;
    const int span = (int)(blockIdx.x % (unsigned)w.spans), tid = (int)threadIdx.x;
    const RowChunks<DT> r(a, row);
    uint4 q[N];
    const int lo = span * kSpan + __builtin_amdgcn_readfirstlane(tid >> 6) * 1024 - r.first;
    r.chunks(lo, lo + 1024, [&](int i) { return span_index<DT>(r, span, tid, i); }, q);
    const Settings g(a, row);
    const bool logs = !g.greedy && !g.by_k && g.filters(), sums = !g.greedy && !g.by_k && (g.by_p || !logs);
    if (logs && tid < kLogBins) bins[tid] = 0;
    float x[16];
#pragma unroll
    for (int i = 0; i < N; i++) RowChunks<DT>::open(q[i], x + i * RowChunks<DT>::VEC);
    float most = x[0];
#pragma unroll
    for (int e = 1; e < 16; e++) most = fmaxf(most, x[e]);
    const int64_t at = row * w.spans + span;
    if (g.by_k) w.group[at * kSpanThreads + tid] = most;
    const float top = B::reduce(most, waves, Max());
    if (tid == 0) {
        w.largest[at] = top;
        if (span == 0) w.count[row] = w.done[row] = 0;
    }
    if (!logs && !sums) return;
    u64 sum = 0;
    if (top > -INFINITY) {
        const Weights wt = {finite(top), g.per, a.shift};
        const double from = logs ? grid_of(top, g.per) : 0.0;
#pragma unroll
        for (int e0 = 0; e0 < 16; e0 += 4) {           // (four at a time: eight waves' registers on a SIMD)
            float z[4] = {x[e0], x[e0 + 1], x[e0 + 2], x[e0 + 3]};
            if (!logs) {
                sum += wt.sum(z);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const u64 v = wt.of(z[e]);
                    const double b = __builtin_fmin(grid_of(z[e], g.per) - from, kLogBins - 1);
                    if (v) atomicAdd(&bins[(int)b], v);
                    sum += v;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    sum = B::reduce(sum, waves, Add());                // (and the bins are filled)
    if (tid == 0) w.mass[at] = sum;
    if (logs && tid < kLogBins) w.bins[at * kLogBins + tid] = bins[tid];
}

// The span in which the sums of mass(span) pass the target, and the target within it.
template <class M> __device__ __forceinline__ int pick_span(const SampleArgs& a, int64_t row, int spans, u64* waves, u64* found, M mass, u64& target, u64& all) {
    const int i = 2 * (int)threadIdx.x;                // (at most 2 kPickThreads)
    const u64 p = i < spans ? mass(i) : 0, q = i + 1 < spans ? mass(i + 1) : 0;
    const u64 before = Block<kPickThreads>::before(p + q, waves, all);
    target = draw_target(a, row, all);
    if (before <= target && target < before + p) { found[0] = (u64)i; found[1] = target - before; }
    else if (before + p <= target && target < before + p + q) { found[0] = (u64)i + 1; found[1] = target - before - p; }
    __syncthreads();
    target = found[1];
    return (int)found[0];
}

struct PickShared {
    union {
        SampleShared<kPickThreads> s;
        struct {
            u64 waves[kPickThreads / 64], fine[kBins], row_bins[kLogBins];
            u64 near[kNear];
        };
    };
    u64 kept[kSpans], found[2];
    unsigned count, count2, base, turn;
};
constexpr int kOwn = 8;                                // logits of a thread in the drawn span
static_assert(kSpan == kOwn * kPickThreads, "the drawn span");

template <int DT> __global__ __launch_bounds__(kPickThreads) void k_sample_pick(SampleArgs a, Spread w) {
    __shared__ PickShared s;
    typedef Block<kPickThreads> B;
    constexpr int NT = kPickThreads, VEC = RowChunks<DT>::VEC;
    const int64_t row = blockIdx.x / (unsigned)w.parts;
    const int part = (int)(blockIdx.x % (unsigned)w.parts);
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const float* largest = w.largest + row * w.spans;
    const u64* mass = w.mass + row * w.spans;
    const Settings g(a, row);
    if (part && (g.greedy || g.by_k || !g.filters())) return;      // (the first does these)
    float top = -INFINITY;
    for (int i = tid; i < w.spans; i += NT) top = fmaxf(top, largest[i]);
    top = B::reduce(top, s.waves, Max());
    if (top == -INFINITY) {
        if (tid == 0 && !part) put_token(a, row, -1, -INFINITY);
        return;
    }
    const RowChunks<DT> r(a, row);
    // A thread's neighbouring logits of a span, and the first one's index.
    auto logits = [&](int span, float (&x)[kOwn]) {
        const int i = span * kSpan + kOwn * tid - r.first, lo = span * kSpan + kOwn * (tid & ~63) - r.first;
        uint4 q[kOwn / VEC];
        r.chunks(__builtin_amdgcn_readfirstlane(lo), __builtin_amdgcn_readfirstlane(lo) + 64 * kOwn, [&](int c) { return i + c * VEC; }, q);
#pragma unroll
        for (int c = 0; c < kOwn / VEC; c++) RowChunks<DT>::open(q[c], x + c * VEC);
        return i;
    };
    if (g.greedy) {
        int at = 0x7FFFFFFF;
        for (int i = tid; i < w.spans; i += NT) at = largest[i] == top ? min(at, i) : at;
        float x[kOwn];
        const int i = logits(B::reduce(at, s.waves, Min()), x);
        at = 0x7FFFFFFF;
#pragma unroll
        for (int e = kOwn - 1; e >= 0; e--) at = x[e] == top ? i + e : at;
        at = B::reduce(at, s.waves, Min());
        if (tid == 0) put_token(a, row, at, 0.0f);
        return;
    }
    const Weights wt = {finite(top), g.per, a.shift};
    // A sum of weights against a span's largest value (y: log2 of this one's weight), against the row's.
    // (Nothing where the largest itself weighs nothing: no draw could end there.)
    auto factor_of = [&](double y) { return y >= -(double)a.shift ? exp2(y) : 0.0; };
    auto against_top = [&](u64 v, double factor) { return (u64)__builtin_rint((double)v * factor); };
    // Draws in a span among what keep(x, index, log2 of the weight) says.
    auto draw_span = [&](int span, u64 target, u64 all, auto keep) {
        float x[kOwn];
        u64 v[kOwn], mine = 0, total;
        const int i = logits(span, x);
#pragma unroll
        for (int e = 0; e < kOwn; e++) {
            const double y = wt.log2_of(x[e]);
            v[e] = x[e] > -INFINITY && keep(x[e], i + e, y) ? wt.of_log2(y) : 0;
            mine += v[e];
        }
        u64 before = B::before(mine, s.waves, total);
        if (target >= total) target = total - 1;       // (its sum against its own largest value was rounded once more)
#pragma unroll
        for (int e = 0; e < kOwn; e++) {
            if (before <= target && target < before + v[e]) put_drawn(a, row, i + e, wt.log2_of(x[e]), all);
            before += v[e];
        }
    };
    if (!g.filters()) {
        u64 target, all;
        const int span = pick_span(a, row, w.spans, s.waves, s.found,
                                   [&](int i) { return against_top(mass[i], factor_of(wt.log2_of(largest[i]))); }, target, all);
        draw_span(span, target, all, [](float, int, double) { return true; });
        return;
    }
    do {
        const SampleRow<DT, NT, false> whole(a, row);
        if (g.by_k) {
            // ---- the few logits that can be among the k largest
            const float* group = w.group + row * w.spans * kSpanThreads;
            const int groups = w.spans * kSpanThreads;
            float lo = top;
            for (int i = tid; i < groups; i += NT) lo = group[i] > -INFINITY ? fminf(lo, group[i]) : lo;
            lo = B::reduce(lo, s.waves, Min());
            float least = kth_bound<NT>([&](auto f) {
                for (int i = tid; i < groups; i += NT) f(group[i]);
            }, (u64)g.k, lo, top, s.s.h);
            if (g.m > 0.0 && !g.by_p) least = fmaxf(least, g.least(top));
            __syncthreads();
            if (tid == 0) s.s.c.count = 0;
            __syncthreads();
            for (int i0 = 0; i0 < groups && s.s.c.count <= kMost; i0 += NT) {
                const int i = i0 + tid;
                const bool near = i < groups && group[i] >= least && group[i] > -INFINITY;
                if (!__ballot(near)) continue;
                float x[16];
                unsigned in = 0;
                const int span = i / kSpanThreads, of = i % kSpanThreads;
                if (near) {
                    uint4 q[16 / VEC];
                    r.chunks(span_index<DT>(r, span, of, 0), span_index<DT>(r, span, of, 16 / VEC - 1) + VEC, [&](int c) { return span_index<DT>(r, span, of, c); }, q);
#pragma unroll
                    for (int c = 0; c < 16 / VEC; c++) RowChunks<DT>::open(q[c], x + c * VEC);
#pragma unroll
                    for (int e = 0; e < 16; e++) in |= x[e] >= least && x[e] > -INFINITY ? 1u << e : 0;
                }
                add_candidates(s.s.c.rank, &s.s.c.count, kMost, in, x, [&](int e) { return span_index<DT>(r, span, of, e / VEC) + e % VEC; });
            }
            __syncthreads();
            if (s.s.c.count <= kMost) {
                draw_candidates<NT>(a, row, g, wt, least, top, s.s.c);
                return;
            }
            break;
        }

        // ---- top-p, min-p: the row's weights by their logarithm
        const double from = grid_of(top, g.per);
        __syncthreads();
        if (tid < kLogBins) s.row_bins[tid] = 0;
        if (tid == 0) s.count = s.count2 = 0;
        __syncthreads();
        auto each_bin = [&](auto f) {                      // f(span, bin of the row, weight): a wave per span
            for (int i = tid >> 6; i < w.spans; i += B::kWaves) {
                const double y = wt.log2_of(largest[i]), below = grid_of(largest[i], g.per) - from;
                const double factor = factor_of(y);
                if (!(factor > 0.0 && below < kLogBins)) continue;
                const u64* b = w.bins + (row * w.spans + i) * kLogBins;
                f(i, (int)below + lane, against_top(b[lane], factor), (int)below + 64 + lane, against_top(b[lane + 64], factor));
            }
        };
        u64 weights = 0;
        each_bin([&](int, int i, u64 p, int j, u64 q) {
            // (the last bin of a span holds all that is below: no less than the row's last)
            if (p) atomicAdd(&s.row_bins[min(i, kLogBins - 1)], p);
            if (q) atomicAdd(&s.row_bins[min(j, kLogBins - 1)], q);
            weights += p + q;
        });
        if (g.by_p) {                                      // and the spans that lie below the bins as a whole
            for (int i = tid; i < w.spans; i += NT) {
                if (grid_of(largest[i], g.per) - from < kLogBins) continue;
                const u64 v = against_top(mass[i], factor_of(wt.log2_of(largest[i])));
                if (v) atomicAdd(&s.row_bins[kLogBins - 1], v);
                weights += v;
            }
        }
        weights = B::reduce(weights, s.waves, Add());
        const u64 want = g.by_p ? g.want(weights) : ~0ull;
        u64 above = 0, total;
        int first = kLogBins, last = -1;                   // bins that a border may lie in
        if (g.by_p) {
            first = reach<NT, 1>([&](int i) { return i < kLogBins ? s.row_bins[i] : 0; }, want, s.waves, s.found, above, total);
            if (first < 0) first = kLogBins - 1;
            last = first;
        }
        if (g.m > 0.0) {
            const double b = __builtin_fmin(-__builtin_floor(wt.top * (g.per * 4.0) + 4.0 * log2(g.m)) - from, kLogBins);
            if ((int)b - 1 <= last || !g.by_p) first = min(first, max((int)b - 1, 0));
            if (!g.by_p || (int)b - 1 <= last) last = max((int)b + 1, first);      // (min-p's, unless top-p's is well above)
            if (g.by_p && (int)b - 1 > first) last = first;
            // weights above the first bin
            u64 sum = tid < kLogBins && tid < first ? s.row_bins[tid] : 0;
            above = B::reduce(sum, s.waves, Add());
        }
        if (last >= kLogBins - 1) {                // (among weights below 2^-31 of the largest)
            if (part) return;
            break;
        }
        // the logits in those bins, by the values that bound these; a wave finds the places of a tile's
        // all at once.  Each part's block looks through its tiles, and the last one that is done goes on
        // with what all have found.
        const float lo = of_key(first_key([&](float x) { return grid_of(x, g.per) - from <= last; }));
        const float hi = of_key(first_key([&](float x) { return grid_of(x, g.per) - from < first; }));
        const bool open_end = !(hi == hi);                 // (none is above)
        whole.each([&](int tile, const float (&x)[kEach]) {
            unsigned in = 0;
#pragma unroll
            for (int e = 0; e < kEach; e++) in |= x[e] >= lo && (open_end || x[e] < hi) ? 1u << e : 0;
            add_candidates(s.near, &s.count, kNear, in, x, [&](int e) { return whole.index(tile) + e; });
        }, part * ((whole.tiles + w.parts - 1) / w.parts), min((part + 1) * ((whole.tiles + w.parts - 1) / w.parts), whole.tiles));
        __syncthreads();
        if (w.parts > 1) {
            u64* all = w.near + row * kNear;
            if (tid == 0) s.base = atomicAdd(&w.count[row], s.count);
            __syncthreads();
            const unsigned base = s.base, n = min(s.count, base < kNear ? kNear - base : 0u);
            for (unsigned i = tid; i < n; i += NT) all[base + i] = s.near[i];
            // Each wave's stores are in this XCD's L2 before the barrier, which by itself waits for none
            // that are on their way; then the fence of one thread writes that L2 back before `done`
            // says so, and the last block's drops what its own caches hold from before.  (Fences of
            // every wave took 45 us more, as each writes a cache back.)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                __threadfence();
                s.turn = atomicAdd(&w.done[row], 1u);
                __threadfence();
                s.count = atomicAdd(&w.count[row], 0u);
            }
            __syncthreads();
            if (s.turn + 1 < (unsigned)w.parts) return;
            for (unsigned i = tid; i < min(s.count, (unsigned)kNear); i += NT) s.near[i] = all[i];
            __syncthreads();
        }
        if (s.count > kNear) break;
        // the spans' weights above the bins
        for (int i = tid; i < w.spans; i += NT) s.kept[i] = 0;
        __syncthreads();
        each_bin([&](int span, int i, u64 p, int j, u64 q) {
            const u64 sum = wave_allreduce((i < first ? p : 0) + (j < first ? q : 0), Add());
            if (lane == 0) s.kept[span] = sum;
        });
        __syncthreads();
        const int near = (int)s.count;
        u64 border = 0;
        auto span_of = [&](u64 rank) { return (index_of(rank) + r.first) / kSpan; };
        // Adds a wave's weights to their spans, mostly one or two (lanes adding to one place wait for each other).
        auto keep = [&](u64 rank, u64 v) {
            const int span = v ? span_of(rank) : -1;
            for (unsigned long long todo = __ballot(v != 0); todo;) {
                const int of = __builtin_amdgcn_readlane(span, __builtin_ctzll(todo));
                const u64 sum = wave_allreduce(span == of ? v : 0, Add());
                if (lane == 0) atomicAdd(&s.kept[of], sum);
                todo &= ~__ballot(span == of);
            }
        };
        const int near_all = (near + NT - 1) / NT * NT;    // (whole waves)
        if (g.by_p) {
            // the same once more in finer bins, by the logarithm's place between the first and the last
            const double y0 = -(from + first - 1) - wt.top * (g.per * 4.0), per_bin = kBins / (double)(last - first + 1);      // (4 log2 at the upper end)
            auto fine_bin = [&](double y) {
                const double b = (y0 - 4.0 * y) * per_bin;
                return b <= 0.0 ? 0 : b >= kBins - 1 ? kBins - 1 : (int)b;
            };
            for (int i = tid; i < kBins; i += NT) s.fine[i] = 0;
            __syncthreads();
            for (int i = tid; i < near; i += NT) {
                const double y = wt.log2_of(value_of(s.near[i]));
                atomicAdd(&s.fine[fine_bin(y)], wt.of_log2(y));
            }
            __syncthreads();
            u64 over;
            int bin = reach<NT, kBins / NT>([&](int i) { return s.fine[i]; }, want - above, s.waves, s.found, over, total);
            if (bin < 0) bin = kBins;                      // (the sums were rounded: all of them)
            __syncthreads();
            for (int i = tid; i < near_all; i += NT) {
                const u64 rank = i < near ? s.near[i] : 0;
                const double y = rank ? wt.log2_of(value_of(rank)) : -100.0;
                const int b = rank ? fine_bin(y) : kBins + 1;
                keep(rank, b < bin && g.passes(y) ? wt.of_log2(y) : 0);
                const float x[1] = {value_of(rank)};
                add_candidates(s.fine, &s.count2, kBins, b == bin ? 1u : 0, x, [&](int) { return index_of(rank); });      // (in the bins' place)
            }
            __syncthreads();
            if (s.count2 > kBins) break;           // (many equal ones)
            if (s.count2) border = border_in<NT>(s.fine, (int)s.count2, above + over, want, g, wt, s.waves, s.found, (unsigned*)s.near, a.V, keep);
        } else {
            for (int i = tid; i < near_all; i += NT) {
                const u64 rank = i < near ? s.near[i] : 0;
                const double y = rank ? wt.log2_of(value_of(rank)) : -100.0;
                keep(rank, rank && g.passes(y) ? wt.of_log2(y) : 0);
            }
        }
        __syncthreads();
        u64 target, all;
        const int span = pick_span(a, row, w.spans, s.waves, s.found, [&](int i) { return s.kept[i]; }, target, all);
        draw_span(span, target, all, [&](float x, int i, double y) {
            return x >= lo && rank_of(x, i) >= border && g.passes(y);
        });
        return;
    } while (false);
    // ---- too many candidates
    __syncthreads();
    const SampleRow<DT, NT, false> whole(a, row);
    draw_any<DT, NT>(a, row, whole, g, wt, s.s.h);
}

// Memory of a spread call: its parts for `rows` rows at base, and its size.
size_t spread_layout(Spread& w, void* base, int64_t rows, int64_t V) {
    w.spans = (int)((V + 7 + kSpan - 1) / kSpan);
    char* p = (char*)base;
    auto take = [&](auto*& to, int64_t n) {
        to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(p);
        p += (n * (int64_t)sizeof(*to) + 255) / 256 * 256;
    };
    take(w.largest, rows * w.spans);
    take(w.group, rows * w.spans * kSpanThreads);
    take(w.mass, rows * w.spans);
    take(w.bins, rows * w.spans * kLogBins);
    w.parts = parts_of(rows, V);
    take(w.near, w.parts > 1 ? rows * kNear : 0);
    take(w.count, rows);
    take(w.done, rows);
    return (size_t)(p - (char*)base);
}

constexpr int kShort = kHeld * kShortThreads * kEach - 8, kLong = kHeld * kRowThreads * kEach - 8;

// Rows of up to kLong logits stay in a block's registers: one launch where two take 4 us more (32000
// logits by top-k: 13.5 .. 16 us, spread 19; but by temperature alone 17 and 10, by top-p 42 and 34,
// which the host cannot know).  Short ones take a small block, whose barriers are cheaper.
template <int DT> void launch_sample(const SampleArgs& a, const Spread* w, hipStream_t s) {
    const unsigned rows = (unsigned)a.rows;
    if (w) {
        hipLaunchKernelGGL(k_sample_spans<DT>, dim3(rows * (unsigned)w->spans), dim3(kSpanThreads), 0, s, a, *w);
        hipLaunchKernelGGL(k_sample_pick<DT>, dim3(rows * (unsigned)w->parts), dim3(kPickThreads), 0, s, a, *w);
    } else if (a.V <= kShort) {
        hipLaunchKernelGGL((k_sample_row<DT, kShortThreads, true>), dim3(rows), dim3(kShortThreads), 0, s, a);
    } else if (a.V <= kLong) {
        hipLaunchKernelGGL((k_sample_row<DT, kRowThreads, true>), dim3(rows), dim3(kRowThreads), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_sample_row<DT, kRowThreads, false>), dim3(rows), dim3(kRowThreads), 0, s, a);
    }
}

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" {

size_t sample_workspace_bytes(int rows, int columns) {
    if (rows < 1 || columns <= kLong || columns > kSpans * kSpan - 8 ||
        (int64_t)rows * ((columns + 7) / kSpan + 1) * kSpanThreads >= (int64_t(1) << 32))
        return 0;
    Spread w;
    return spread_layout(w, nullptr, rows, columns);
}

void sample_forward(const Tensor* Logits, const Tensor* Uniform, const Tensor* Temperature,
                               const Tensor* TopK, const Tensor* TopP, const Tensor* MinP, Tensor* Token,
                               Tensor* LogProb, const SampleParams* params, Tensor* Workspace) {
    const char* name = "sample_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    const Tensor* needed[] = {Logits, Uniform, Token};
    for (const Tensor* t : needed)
        if (!tensor_sane(t, name)) return;
    const Tensor* all[] = {Logits, Uniform, Token, Temperature, TopK, TopP, MinP, LogProb, Workspace};
    for (const Tensor* t : all) {
        if (!t) continue;
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
    }
    const int dt = (int)Logits->dtype;
    if (dt != kF16 && dt != kBF16 && dt != kF32) {
        set_error("%s: Logits must be float16, bfloat16 or float32", name);
        return;
    }
    if (Logits->ndim != 2 || Logits->shape[1] < 1) { set_error("%s: Logits must be [rows, columns]", name); return; }
    SampleArgs a = {};
    a.rows = Logits->shape[0];
    a.ld = Logits->shape[1];
    if (params->vocab < 0 || params->vocab > a.ld) {
        set_error("%s: vocab must be 0 or at most the columns of Logits, got %d", name, params->vocab);
        return;
    }
    a.V = params->vocab ? params->vocab : (int)a.ld;
    if (a.V > kMaxTiles * kRowThreads * kEach - 16) { set_error("%s: more than %d columns", name, kMaxTiles * kRowThreads * kEach - 16); return; }
    if ((uintptr_t)Logits->data % dt_bytes(dt)) { set_error("%s: Logits must be aligned to their type", name); return; }
    auto vector = [&](const Tensor* t, int d0, int d1, const char* what) {
        if (!t || (t->ndim == 1 && t->shape[0] == a.rows && ((int)t->dtype == d0 || (int)t->dtype == d1))) return true;
        set_error("%s: %s", name, what);
        return false;
    };
    if (!vector(Uniform, kF32, kF64, "Uniform must be float32 or float64 [rows]") ||
        !vector(Token, kI32, kI64, "Token must be int32 or int64 [rows]") ||
        !vector(TopK, kI32, kI64, "TopK must be int32 or int64 [rows]") ||
        !vector(Temperature, kF32, kF32, "Temperature, TopP, MinP and LogProb must be float32 [rows]") ||
        !vector(TopP, kF32, kF32, "Temperature, TopP, MinP and LogProb must be float32 [rows]") ||
        !vector(MinP, kF32, kF32, "Temperature, TopP, MinP and LogProb must be float32 [rows]") ||
        !vector(LogProb, kF32, kF32, "Temperature, TopP, MinP and LogProb must be float32 [rows]"))
        return;
    const Tensor* outs[] = {Token, LogProb, Workspace};
    for (int i = 0; i < 3; i++) {
        for (const Tensor* in : {Logits, Uniform, Temperature, TopK, TopP, MinP})
            if (overlaps(in, outs[i])) { set_error("%s: an output or Workspace overlaps an input", name); return; }
        for (int j = 0; j < i; j++)
            if (overlaps(outs[i], outs[j])) { set_error("%s: Token, LogProb and Workspace must not overlap", name); return; }
    }
    if (a.rows >= (1 << 22)) { set_error("%s: more than %d rows", name, (1 << 22) - 1); return; }
    if (!ensure_device()) return;
    if (!a.rows) return;
    a.x = Logits->data;
    a.u = Uniform->data;
    a.u64 = (int)Uniform->dtype == kF64;
    a.temperature = Temperature ? (const float*)Temperature->data : nullptr;
    a.top_p = TopP ? (const float*)TopP->data : nullptr;
    a.min_p = MinP ? (const float*)MinP->data : nullptr;
    if (TopK) a.top_k = {TopK->data, (int)TopK->dtype == kI64};
    a.token = Token->data;
    a.token64 = (int)Token->dtype == kI64;
    a.logprob = LogProb ? (float*)LogProb->data : nullptr;
    int bits = 0;
    while ((int64_t(1) << bits) < a.V) bits++;
    a.shift = std::min(51, 62 - bits);
    DeviceScope scope;
    // Rows that a block holds in registers are done by it in one launch; longer ones are spread.
    Spread w = {};
    const size_t bytes = sample_workspace_bytes(a.rows, a.V);
    void* part = nullptr;
    if (bytes) {
        if (Workspace && tensor_bytes(Workspace) >= bytes && !((uintptr_t)Workspace->data & 15)) {
            spread_layout(w, Workspace->data, a.rows, a.V);
        } else if ((part = pool_alloc(bytes, true))) {
            spread_layout(w, part, a.rows, a.V);
        }
    }
    const Spread* spread = w.largest ? &w : nullptr;
    if (dt == kF16) launch_sample<kF16>(a, spread, stream());
    else if (dt == kBF16) launch_sample<kBF16>(a, spread, stream());
    else launch_sample<kF32>(a, spread, stream());
    check_launch(name);
    if (part) pool_free(part);
}

}  // extern "C"
