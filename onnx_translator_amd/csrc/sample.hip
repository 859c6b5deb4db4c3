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
// beside a border would depend on the order: of 131072 tokens one row in some thousands.)
#include "attention.h"

#include <algorithm>
#include <cmath>

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
// Order-preserving key of a logit: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = f2u(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return u2f(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// log2 of x's weight against the row's largest value (x <= top; equal infinities weigh 1).
__device__ __forceinline__ double log2_weight(float x, float top, double per) {
    return x == top ? 0.0 : x == -INFINITY || top == INFINITY ? -INFINITY : ((double)x - (double)top) * per;
}
// 2^y for y <= 0: 2^f by its Taylor series, |f| <= 1/2 (12 terms: 2^-52 of the result).
__device__ __forceinline__ double pow2(double y) {
    const double n = __builtin_rint(y), f = y - n;
    double p = 2.5678435993488206e-11;                // ln2^12 / 12!, ...
    p = __builtin_fma(p, f, 4.4455382718708116e-10);
    p = __builtin_fma(p, f, 7.054911620801123e-09);
    p = __builtin_fma(p, f, 1.01780860092397e-07);
    p = __builtin_fma(p, f, 1.321548679014431e-06);
    p = __builtin_fma(p, f, 1.5252733804059841e-05);
    p = __builtin_fma(p, f, 0.0001540353039338161);
    p = __builtin_fma(p, f, 0.0013333558146428443);
    p = __builtin_fma(p, f, 0.009618129107628477);
    p = __builtin_fma(p, f, 0.05550410866482158);
    p = __builtin_fma(p, f, 0.24022650695910072);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// The weight 2^y in whole numbers of 2^-shift (shift <= 51), rounded to the nearest: the low bits
// of the sum with 2^52.
__device__ __forceinline__ u64 fixed_weight(double y, int shift) {
    if (!(y >= -54.0)) return 0;
    const double v = __builtin_ldexp(pow2(y), shift) + 0x1p52;
    return __builtin_bit_cast(u64, v) & 0xFFFFFFFFFFFFFull;
}

// ---- a block's sums ---------------------------------------------------------------------
constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kEach = 8;                               // logits of a thread in a tile, in index order
constexpr int kTile = kThreads * kEach;
constexpr int kBins = 2048, kMaxTiles = 2048;          // (16 M columns)

__device__ __forceinline__ u64 shfl_up64(u64 v, int o) { return (u64)__shfl_up((long long)v, o); }

// Sums of all threads before this one, and of all.
__device__ __forceinline__ u64 scan_before(u64 v, u64* waves, u64& total) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
    u64 s = v;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const u64 x = shfl_up64(s, o);
        if (lane >= o) s += x;
    }
    __syncthreads();                                   // (the last call's are read)
    if (lane == 63) waves[w] = s;
    __syncthreads();
    u64 before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        const u64 x = waves[i];
        before += i < w ? x : 0;
        total += x;
    }
    return before + s - v;
}

struct SampleShared {
    u64 waves[kWaves];
    u64 bins[kBins];
    u64 tile_mass[kMaxTiles];
    uint32_t tile_ties[kMaxTiles];
    u64 found[3];
};

// The bin, from the highest down, in which the sums pass `want` (1 <= want <= the sum of all): the
// bin and the sum of the bins above it.
__device__ __forceinline__ void pick_bin(SampleShared& s, u64 want, int& bin, u64& above) {
    const int hi = kBins - 1 - 2 * (int)threadIdx.x;
    const u64 a = s.bins[hi], b = s.bins[hi - 1];
    u64 total;
    const u64 before = scan_before(a + b, s.waves, total);
    if (before < want && want <= before + a) { s.found[0] = (u64)hi; s.found[1] = before; }
    else if (before + a < want && want <= before + a + b) { s.found[0] = (u64)hi - 1; s.found[1] = before + a; }
    __syncthreads();
    bin = (int)s.found[0];
    above = s.found[1];
}

// ---- a row ---------------------------------------------------------------------------------
// Tiles begin at the 16-byte chunk that holds the row's first logit; places outside the row give
// -inf.
template <int DT> struct SampleRow {
    static constexpr int ES = DT == kF32 ? 4 : 2, VEC = 16 / ES;
    const char* base;
    int first, V, tiles;

    __device__ __forceinline__ SampleRow(const SampleArgs& a, int64_t row) {
        const uintptr_t p = (uintptr_t)a.x + (uintptr_t)(row * a.ld * ES);
        base = (const char*)(p & ~(uintptr_t)15);
        first = (int)((p & 15) / ES);
        V = a.V;
        tiles = (first + V + kTile - 1) / kTile;
    }
    __device__ __forceinline__ int index(int tile) const { return tile * kTile + (int)threadIdx.x * kEach - first; }
    __device__ __forceinline__ void load(int tile, float (&x)[kEach]) const {
        const int i0 = index(tile);
#pragma unroll
        for (int c = 0; c < kEach; c += VEC) {
            const int i = i0 + c;
            const char* p = base + (int64_t)(i + first) * ES;
            if (i >= 0 && i + VEC <= V) {
                const uint4 q = *reinterpret_cast<const uint4*>(p);
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (DT == kF32) {
                        x[c + e] = u2f(w[e]);
                    } else if constexpr (DT == kBF16) {
                        x[c + 2 * e] = u2f(w[e] << 16);
                        x[c + 2 * e + 1] = u2f(w[e] & 0xFFFF0000u);
                    } else {
                        x[c + 2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
                        x[c + 2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; e++)
                    x[c + e] = i + e >= 0 && i + e < V ? (float)ld_d<DT>(p, e) : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < kEach; e++) x[e] = x[e] != x[e] ? -INFINITY : x[e];
    }
};

__device__ __forceinline__ void put_token(const SampleArgs& a, int64_t row, int64_t token, float logprob) {
    if (a.token64) ((int64_t*)a.token)[row] = token;
    else ((int32_t*)a.token)[row] = (int32_t)token;
    if (a.logprob) a.logprob[row] = logprob;
}

// A block per row, any filters, any logits.
template <int DT> __global__ __launch_bounds__(kThreads) void k_sample_row(SampleArgs a) {
    __shared__ SampleShared s;
    constexpr int kRounds = DT == kF32 ? 3 : 2;        // digits of 11, 11 and 10 bits; 16-bit logits differ in the first two
    const int64_t row = blockIdx.x;
    const int tid = (int)threadIdx.x;
    const SampleRow<DT> r(a, row);
    const double t = a.temperature ? (double)a.temperature[row] : 1.0;
    const double p = a.top_p ? (double)a.top_p[row] : 1.0, m = a.min_p ? (double)a.min_p[row] : 0.0;
    const int64_t k = a.top_k.p ? a.top_k[row] : 0;

    // ---- the largest value, and where it is first: (key, ~index) as one number
    u64 best = 0;
    for (int tile = 0; tile < r.tiles; tile++) {
        float x[kEach];
        r.load(tile, x);
        const int i = r.index(tile);
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const u64 v = ((u64)key_of(x[e]) << 32) | (uint32_t)~(i + e);
            best = x[e] > -INFINITY && v > best ? v : best;
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const u64 v = (u64)__shfl_xor((long long)best, o);
        best = v > best ? v : best;
    }
    if ((tid & 63) == 0) s.waves[tid >> 6] = best;
    __syncthreads();
    best = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) best = s.waves[i] > best ? s.waves[i] : best;
    if (best == 0) {
        if (tid == 0) put_token(a, row, -1, -INFINITY);
        return;
    }
    if (!(t > 0.0)) {
        if (tid == 0) put_token(a, row, (int)~(uint32_t)best, 0.0f);
        return;
    }
    const float top = of_key((uint32_t)(best >> 32));
    const double per = 1.4426950408889634 / t;
    auto weight = [&](float x) { return fixed_weight(log2_weight(x, top, per), a.shift); };

    // ---- the border: kept are keys above `border`, and the first `ties` equal to it
    uint32_t border = 0;                               // (no key: everything is kept)
    u64 ties = 0, equal = 0;                           // equal: keys that are the border's, of those ranked at all
    // A digit search from the highest key down: the value at which the sums of amount(x) over the
    // keys >= least pass want.  less: what to take off the sum of least's own bin.
    auto search = [&](auto amount, uint32_t least, u64 less, auto want_of, u64& above) {
        uint32_t prefix = 0;
        u64 want = 0, within = 0;
        above = 0;
        for (int round = 0; round < kRounds; round++) {
            const int low = round == 0 ? 21 : round == 1 ? 10 : 0, width = round == 2 ? 10 : 11;
            for (int i = tid; i < kBins; i += kThreads) s.bins[i] = 0;
            __syncthreads();
            for (int tile = 0; tile < r.tiles; tile++) {
                float x[kEach];
                r.load(tile, x);
#pragma unroll
                for (int e = 0; e < kEach; e++) {
                    const uint32_t key = key_of(x[e]);
                    if (x[e] == -INFINITY || key < least) continue;
                    if (round && (key >> (low + width)) != prefix) continue;
                    const u64 v = amount(x[e]);
                    if (v) atomicAdd(&s.bins[(key >> low) & (kBins - 1) & ((1u << width) - 1)], v);
                }
            }
            __syncthreads();
            if (less && tid == 0 && (!round || (least >> (low + width)) == prefix))
                s.bins[(least >> low) & ((1u << width) - 1)] -= less;
            __syncthreads();
            if (round == 0) {
                u64 total;
                (void)scan_before(s.bins[2 * tid] + s.bins[2 * tid + 1], s.waves, total);
                want = want_of(total);
                if (!want || want > total) return false;               // all of them
            }
            int bin;
            u64 over;
            pick_bin(s, want - above, bin, over);
            above += over;
            within = s.bins[bin];
            prefix = (prefix << width) | (uint32_t)bin;
            __syncthreads();
        }
        if (kRounds == 2) prefix = prefix & (1u << 21) ? prefix << 10 : (prefix << 10) | 0x3FF;      // the digits all values share
        border = prefix;
        equal = within;
        return true;
    };

    if (k > 0 && k < a.V) {
        u64 above;
        if (search([](float) { return (u64)1; }, 0u, 0, [&](u64) { return (u64)k; }, above)) ties = (u64)k - above;
    }
    if (p < 1.0) {
        // of border's equals only `ties` are there
        const uint32_t least = border;
        const u64 own = least ? weight(of_key(least)) : 0, gone = least ? (equal - ties) * own : 0, had = ties;
        u64 above, want = 0;
        const bool some = search(weight, least, gone, [&](u64 total) {
            const double w = __builtin_ceil(p * (double)total);
            want = !(w >= 1.0) ? 1 : w >= (double)total ? total : (u64)w;
            return want;
        }, above);
        if (some) {
            const u64 each = weight(of_key(border)), n = equal / each;            // (each > 0: the sums pass want here)
            ties = (want - above + each - 1) / each;
            ties = ties < 1 ? 1 : ties > n ? n : ties;
            equal = border == least ? n + (gone / (own ? own : 1)) : n;
        } else {
            ties = had;
        }
    }
    const double least_weight = m >= 1.0 ? 1.0 : m > 0.0 ? m : 0.0;
    const bool some_ties = border && ties < equal;     // the ties are told apart by index

    // ---- the kept weights, tile by tile in index order
    // Weights of this thread's logits; before: equals of the border in the tiles and threads before.
    auto weigh = [&](const float (&x)[kEach], u64 before, u64 (&w)[kEach]) {
        u64 sum = 0;
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t key = key_of(x[e]);
            bool keep = x[e] > -INFINITY && key >= border;
            if (some_ties && key == border) keep = keep && before++ < ties;
            w[e] = 0;
            if (keep) {
                const double y = log2_weight(x[e], top, per);
                if (!(least_weight > 0.0) || pow2(y < -1000.0 ? -1000.0 : y) >= least_weight) w[e] = fixed_weight(y, a.shift);
            }
            sum += w[e];
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
    for (int tile = 0; tile < r.tiles; tile++) {
        float x[kEach];
        u64 w[kEach], before = 0, total;
        r.load(tile, x);
        if (tid == 0) s.tile_ties[tile] = (uint32_t)met;
        if (some_ties) {
            before = met + scan_before(count_ties(x), s.waves, total);
            met += total;
        }
        (void)scan_before(weigh(x, before, w), s.waves, total);
        if (tid == 0) s.tile_mass[tile] = total;
        all += total;
    }
    __syncthreads();

    // ---- the draw
    const double u = a.u64 ? ((const double*)a.u)[row] : (double)((const float*)a.u)[row];
    const double at = u * (double)all;
    u64 target = !(at > 0.0) ? 0 : at >= (double)all ? all - 1 : (u64)at;
    if (target >= all) target = all - 1;
    int tile = 0;
    for (; tile + 1 < r.tiles && target >= s.tile_mass[tile]; tile++) target -= s.tile_mass[tile];
    float x[kEach];
    u64 w[kEach], before = 0, total;
    r.load(tile, x);
    if (some_ties) before = s.tile_ties[tile] + scan_before(count_ties(x), s.waves, total);
    const u64 mine = weigh(x, before, w);
    u64 from = scan_before(mine, s.waves, total);
    if (from <= target && target < from + mine) {
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            if (from <= target && target < from + w[e])
                put_token(a, row, r.index(tile) + e,
                          (float)(log2_weight(x[e], top, per) * 0.6931471805599453 + (double)a.shift * 0.6931471805599453 - log((double)all)));
            from += w[e];
        }
    }
}

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" void sample_forward(const Tensor* Logits, const Tensor* Uniform, const Tensor* Temperature,
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
    if (a.V > kMaxTiles * kTile - 16) { set_error("%s: more than %d columns", name, kMaxTiles * kTile - 16); return; }
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
    const dim3 grid((unsigned)a.rows);
    if (dt == kF16) hipLaunchKernelGGL(k_sample_row<kF16>, grid, dim3(kThreads), 0, stream(), a);
    else if (dt == kBF16) hipLaunchKernelGGL(k_sample_row<kBF16>, grid, dim3(kThreads), 0, stream(), a);
    else hipLaunchKernelGGL(k_sample_row<kF32>, grid, dim3(kThreads), 0, stream(), a);
    check_launch(name);
}
