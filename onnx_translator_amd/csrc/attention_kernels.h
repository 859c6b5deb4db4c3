// attention_kernels.h — the attention kernels for gfx950, by element type (one source
// file instantiates each).
//
//   y = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j + bias_j - max_j)
//
// over the keys a query sees.  One pass over the keys: a running maximum and sum,
// the output rescaled where the maximum grows.  Scores, statistics and sums are
// held in 32 bits or more.  Two roundings to a 16-bit type: each weight p_j for its
// product with V (and for the sum of the weights: AttnWave::pack), and the result.
//
// Keys that are not seen (past the length, later than the query, outside the
// window, closed by the mask, or on a page that the cache does not have) add
// nothing, whatever K and V hold there; a row that sees none gives zeros.
#pragma once

#include <cmath>
#include <type_traits>

#include "attention.h"

namespace tohip {
namespace {

template <int DT> __device__ __forceinline__ float ld_f(const void* p, int64_t i) { return (float)ld_d<DT>(p, i); }

__device__ __forceinline__ double lane_value(double v, int lane) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, lane);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(u >> 32), lane);
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}

// ---- one row per wave ---------------------------------------------------------------
// Any head size, alignment and content.  Lanes take 64 keys at a time for the scores,
// then 64 columns of V for the sums, in double: nothing overflows on the way to a
// finite result, and a key that is not seen is never multiplied.  Bound by its double
// products and one dependent pass after the other: what the matrix kernels do in 540 us
// (4096 queries over 8192 keys, 32 heads of 128) takes it 0.29 s, so it takes what they do
// not: odd head sizes, unaligned tensors, and single rows that they hand over.
constexpr int kRowCols = 4;        // columns of V per lane and pass over the keys

// Partial result of the keys [ks, ke) for query head h of token i: the maximum (of
// scaled scores), the sum and, by store(d, value), the normalised output.
template <int DT, int KEYS, class ST>
__device__ __forceinline__ void attn_row(const AttnArgs& a, const AttnSeq& s, int h, int i, int ks, int ke, float& m_out,
                                         float& l_out, ST store) {
    constexpr bool PAGED = KEYS != kDense;
    const int lane = (int)(threadIdx.x & 63), hk = (int)a.fd_g.div((uint32_t)h);
    const int shared = KEYS == kPrefixed ? attn_shared(a) : 0;      // all of them are seen
    const int lo = max(ks, attn_lo(a, s, i)), hi = min(ke, shared + (shared ? max(attn_hi(a, s, i), 0) : attn_hi(a, s, i)));
    const int64_t qo = PAGED ? (s.tok0 + i) * a.qt + h * a.qh : s.b * a.qb + i * a.qt + h * a.qh;
    const int64_t mo = s.b * a.mb + h * a.mh + i * a.mq;
    for (int d0 = 0; d0 < a.Dv; d0 += 64 * kRowCols) {
        float m = -INFINITY;
        double l = 0.0, acc[kRowCols] = {};
        for (int j0 = lo; j0 < hi; j0 += 64) {
            const int j = j0 + lane;
            bool seen = j < hi;
            const int page = PAGED && seen ? attn_page<KEYS>(a, s.b, j, shared) : 0;
            seen = seen && page >= 0;
            float t = -INFINITY;
            KeyRow row = {0, 0};
            if (seen) {
                row = attn_key_row<PAGED>(a, s.b, page, j < shared ? j : j - shared);
                float bias = 0.0f;
                if (a.mask) {
                    const int64_t o = mo + (int64_t)j * a.mk;
                    if (a.mask_dt == kU8 || a.mask_dt == kI8) {
                        seen = ((const uint8_t*)a.mask)[o] != 0;
                    } else {
                        bias = a.mask_dt == kF32 ? ((const float*)a.mask)[o] : ld_f<DT>(a.mask, o);
                        seen = !(bias == -INFINITY);
                    }
                }
                if (seen) {
                    double dot = 0.0;
                    for (int d = 0; d < a.Dk; d++)
                        dot += (double)ld_f<DT>(a.q, qo + d) * (double)ld_f<DT>(a.k, row.k + hk * a.kh + d);
                    t = (float)(dot * (double)a.scale + (double)bias);
                }
            }
            const unsigned long long sees = __ballot(seen);
            if (!sees) continue;
            const bool bad = __ballot(seen && t != t) != 0;
            const float top = wave_allreduce(t != t ? -INFINITY : t, [](float x, float y) { return x > y ? x : y; });
            const float mn = bad ? NAN : (top > m ? top : m);
            if (mn == -INFINITY) continue;
            const float alpha = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * kLog2e);
            const double p = seen ? (double)__builtin_amdgcn_exp2f((t - mn) * kLog2e) : 0.0;
            l = l * (double)alpha + wave_allreduce(p, [](double x, double y) { return x + y; });
#pragma unroll
            for (int c = 0; c < kRowCols; c++) acc[c] *= (double)alpha;
            m = mn;
            for (int jj = 0; jj < 64; jj++) {
                if (!((sees >> jj) & 1)) continue;
                const double pj = lane_value(p, jj);
                const int64_t ro = (int64_t)__builtin_bit_cast(long long, lane_value(__builtin_bit_cast(double, (long long)row.v), jj));
#pragma unroll
                for (int c = 0; c < kRowCols; c++) {
                    const int d = d0 + c * 64 + lane;
                    if (d < a.Dv) acc[c] += pj * (double)ld_f<DT>(a.v, ro + hk * a.vh + d);
                }
            }
        }
#pragma unroll
        for (int c = 0; c < kRowCols; c++) {
            const int d = d0 + c * 64 + lane;
            if (d < a.Dv) store(d, l == 0.0 ? 0.0f : (float)(acc[c] / l));
        }
        m_out = m;
        l_out = (float)l;
    }
}

template <int DT, int KEYS> __device__ __forceinline__ void attn_rows(const AttnArgs& a, int64_t rows) {
    constexpr bool PAGED = KEYS != kDense;
    const int64_t step = (int64_t)gridDim.x * 4;
    for (int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); r < rows; r += step) {
        const int64_t t = r / a.Hq;
        const int h = (int)(r - t * a.Hq);
        int b, i;
        if constexpr (PAGED) {
            // the last sequence that starts at or before the token
            int lo = 0, hi = a.B;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (a.qstart[mid] <= t) lo = mid + 1;
                else hi = mid;
            }
            b = lo - 1;
            if (b < 0) continue;
        } else {
            b = (int)(t / a.Sq);
        }
        const AttnSeq s = attn_seq<PAGED>(a, b);
        const int64_t at = PAGED ? t - s.tok0 : t - (int64_t)b * a.Sq;
        if (at < 0 || at >= s.n) continue;             // behind the last sequence: left as it is
        i = (int)at;
        const int64_t yo = PAGED ? t * a.yt + h * a.yh : b * a.yb + i * a.yt + h * a.yh;
        float m, l;
        attn_row<DT, KEYS>(a, s, h, i, 0, KEYS == kPrefixed ? 0x7FFFFFFF : s.len, m, l, [&](int d, float v) { st_code<DT>(a.y, yo + d, v); });
    }
}

template <int DT, bool PAGED> __global__ __launch_bounds__(256) void k_attn_rows(AttnArgs a, int64_t rows) {
    attn_rows<DT, PAGED ? kPaged : kDense>(a, rows);
}
// Behind a shared prefix, in one pass over both.
template <int DT> __global__ __launch_bounds__(256) void k_prefix_rows(AttnArgs a, int64_t rows) {
    attn_rows<DT, kPrefixed>(a, rows);
}

// ---- tiles on the matrix cores ------------------------------------------------------
// A wave owns MR rows (query heads of tokens) and walks over the keys, 32 at a time:
//   S' = K Q'    32 keys x MR rows: a lane holds a part of one row's keys (MR = 32: half of
//                them, MR = 16: a quarter), so maximum and sum of a row are a few register
//                operations and one or two exchanges inside the wave;
//   O' += V' P'  head size x MR rows: the rescaling factor of a row is one lane's value,
//                and P goes from the accumulators of S' straight into the operand: the
//                product sums over keys in any order, so V's rows are simply read in the
//                order in which the lanes hold their keys.
// Tiles of K and V go from memory to LDS directly (no registers) in 16-byte chunks whose
// place in a row is turned by the row's number, so that fragment reads spread over the
// banks; V's columns are read by the transposing LDS loads (16-bit types).
//   k_attn_tiles   prompts: four waves of 32 rows share the tiles, two deep;
//   k_attn_few     few rows, where reading the keys is the work: a block is one wave.
//
// What a closed key holds does not matter as long as it is finite: its weight is zero.
// Where a result comes out infinite or NaN (a closed key's value was, or values near the
// type's largest overflowed a sum on the way), or a page of the sequence is missing, the
// row is computed again by attn_row above, which looks at open keys only.  A q.k that falls
// below float32's range before the scale is -inf, a key of no weight.
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfloatx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));

#define TOHIP_INLINE __attribute__((always_inline))

template <int DT> constexpr int kElem = DT == kF32 ? 4 : 2;

// One product step.  16 bits: operands of eight values per lane (a 16-byte chunk); 32 bits:
// one value per lane.  MR = 32: 32x32 results, two lanes' values per column and step;
// MR = 16: 16x16, four lanes'.
template <int MR> struct AttnAcc { typedef floatx16 type; };
template <> struct AttnAcc<16> { typedef floatx4 type; };
template <int DT, int MR, class ACC> __device__ __forceinline__ ACC mfma16(uint4 a, uint4 b, ACC c) {
    if constexpr (DT == kF16) {
        const halfx8 x = __builtin_bit_cast(halfx8, a), y = __builtin_bit_cast(halfx8, b);
        if constexpr (MR == 32) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    } else {
        const bfloatx8 x = __builtin_bit_cast(bfloatx8, a), y = __builtin_bit_cast(bfloatx8, b);
        if constexpr (MR == 32) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
}
template <int MR, class ACC> __device__ __forceinline__ ACC mfma32(float a, float b, ACC c) {
    if constexpr (MR == 32) return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Values rounded to the nearest of the 16-bit type.
template <int DT, int N> __device__ __forceinline__ auto round16(const float* p) {
    typedef std::conditional_t<DT == kF16, _Float16, __bf16> T;
    typedef T vec __attribute__((ext_vector_type(N)));
    vec h;
#pragma unroll
    for (int i = 0; i < N; i++) h[i] = (T)p[i];
    return h;
}

// s and the two 16-bit values of a register (the pair's product with ones: exact, subnormal values
// too, and off by at most three float32 half steps in the sum).
template <int DT> __device__ __forceinline__ float add_pair(uint32_t v, float s) {
    if constexpr (DT == kF16) {
        typedef _Float16 pair __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(pair, v), pair{(_Float16)1.0f, (_Float16)1.0f}, s, false);
    } else {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, v), pair{(__bf16)1.0f, (__bf16)1.0f}, s, false);
    }
}

// 16 bytes per lane from its own address into LDS, lane l to the l-th 16 bytes of `to`.
__device__ __forceinline__ void load_lds16(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
// Four rows x 16 columns of 16-bit values in LDS, read by 16 lanes (8 bytes each, lane i
// at row i / 4, columns 4 (i % 4) ..): lane i receives column i of the four rows.
__device__ __forceinline__ uint2 read_turned(const char* p) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4*)p));
}
// Several LDS reads and the wait for them in one go.  The loads that write LDS are waited for by
// count (wait_loads); where the compiler sees the reads it adds a wait of its own, inside a loop
// for everything in flight, the next tiles' loads among them.
__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
__device__ __forceinline__ void read_keys4(const uint32_t (&at)[4], uint4 (&v)[4]) {
    asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]) : "memory");
}
__device__ __forceinline__ void read_keys8(const uint32_t (&at)[8], uint4 (&v)[8]) {
    asm volatile("ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
                 "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\tds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7]) : "memory");
}
// read_turned at four addresses, and STEP bytes further on.
template <int STEP> __device__ __forceinline__ void read_values(const uint32_t (&at)[4], uint2 (&x)[4], uint2 (&y)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %6, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %3, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(STEP) : "memory");
}
// Eight 32-bit values of one column: rows 0 .. 3 and G .. G + 3 of RB bytes each.
template <int RB, int G> __device__ __forceinline__ void read_column8(uint32_t at, float (&v)[8]) {
    asm volatile("ds_read_b32 %0, %8\n\tds_read_b32 %1, %8 offset:%9\n\tds_read_b32 %2, %8 offset:%10\n\t"
                 "ds_read_b32 %3, %8 offset:%11\n\tds_read_b32 %4, %8 offset:%12\n\tds_read_b32 %5, %8 offset:%13\n\t"
                 "ds_read_b32 %6, %8 offset:%14\n\tds_read_b32 %7, %8 offset:%15\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(at), "n"(RB), "n"(2 * RB), "n"(3 * RB), "n"(G * RB), "n"((G + 1) * RB), "n"((G + 2) * RB), "n"((G + 3) * RB)
                 : "memory");
}
// At most N of this wave's loads are in flight (they land in order), and its LDS reads have
// returned.
template <int N> __device__ __forceinline__ void wait_loads() {
    constexpr int n = N > 63 ? 63 : N;
    __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | ((n >> 4) << 14));
}
// A value that all lanes hold, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Place of chunk c in row r of a tile of CH chunks per row.  Keys are read by 16 or 32 rows
// of one chunk.  Values of 16 bits: by four (MR = 32) or eight rows (MR = 16) of four or
// two neighbouring chunks; of 32 bits: by rows four apart, two of eight chunks or four of four.
template <int CH> __device__ __forceinline__ int key_place(int r, int c) {
    return c ^ (CH == 8 ? (r >> 1) & 7 : r & 15);
}
template <int DT, int CH, int MR> __device__ __forceinline__ int value_place(int r, int c) {
    if constexpr (DT == kF32) return c ^ (MR == 32 ? ((r >> 2) & 1) << 3 : ((r >> 2) & 3) << 2);
    else if constexpr (MR == 32) return c ^ (CH == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2);
    else return c ^ (CH == 8 ? ((r >> 1) & 3) << 1 : (r & 7) << 1);
}

// log2 units that a row's maximum may grow by before its sums are rescaled: weights stay
// below 2^8 (and the float16 ones, raised by 2^6 out of its subnormal range, below 2^14).
constexpr float kLazy = 8.0f;
template <int DT> constexpr float kRaise = DT == kF16 ? 6.0f : 0.0f;
template <int DT> constexpr float kLower = DT == kF16 ? 0x1p-6f : 1.0f;        // 2^-kRaise

// ---- blocks, rows, keys -----------------------------------------------------------------
// The sequence whose tiles hold slot t: the last b with floor(start_b * G / BM) + b <= t.
// (The slots of a sequence, one more than its whole tiles may need, follow from the starts
// alone, so no list of tiles has to be made.)  64 sequences are tried at a time.
template <int BM> __device__ __forceinline__ int64_t slot_base(const AttnArgs& a, int b) {
    int64_t t0 = a.qstart[b];
    t0 = t0 < 0 ? 0 : t0 > a.T ? a.T : t0;
    return t0 * a.G / BM + b;
}
template <int BM> __device__ __forceinline__ AttnSeq slot_sequence(const AttnArgs& a, int64_t t) {
    int lo = 0, n = a.B;                       // the answer is in [lo, lo + n)
    const int lane = (int)(threadIdx.x & 63);
    if (n < 64) {                              // all starts in one load
        const int64_t v = IndexVec{lane < n ? a.qstart.p : a.qend, a.qstart.is64}[lane < n ? lane : n - 1];
        const int start = (int)(v < 0 ? 0 : v > a.T ? a.T : v);
        const bool le = lane < n && (int64_t)start * a.G / BM + lane <= t;
        const int b = max(0, (int)__popcll(__ballot(le)) - 1);
        return attn_seq_at(a, b, __builtin_amdgcn_readlane(start, b), __builtin_amdgcn_readlane(start, b + 1));
    }
    while (n > 1) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const bool le = lane * step < n && slot_base<BM>(a, b) <= t;
        const int k = __popcll(__ballot(le));
        if (k > 1) lo += (k - 1) * step;
        n = min(step, a.B - lo);
    }
    return attn_seq<true>(a, uniform(lo));
}

// A block's part of the call: `rows` rows from row0 of its sequence on (of key head hk), over
// the keys [klo, khi); klo is a multiple of 32.
struct AttnBlock {
    AttnSeq s;
    int hk, split, row0, rows, klo, khi;
    int table, from;                           // pages from .. from + 63 of the sequence, one per lane
};
// One of its rows.
struct AttnRow {
    int tok, head;
    int64_t y, out;                            // element of Y, row among all rows of Y
};
template <bool PAGED> __device__ __forceinline__ AttnRow attn_row_at(const AttnArgs& a, const AttnBlock& k, int r) {
    AttnRow w;
    const uint32_t row = (uint32_t)(k.row0 + r);
    w.tok = (int)a.fd_g.div(row);
    w.head = k.hk * a.G + (int)(row - (uint32_t)w.tok * (uint32_t)a.G);
    const int64_t token = PAGED ? k.s.tok0 + w.tok : (int64_t)k.s.b * a.Sq + w.tok;
    w.out = token * a.Hq + w.head;
    w.y = PAGED ? token * a.yt + w.head * a.yh : k.s.b * a.yb + w.tok * a.yt + w.head * a.yh;
    return w;
}

// Block `bid` of the call, of which this is thread `thread` of `threads`.  false: nothing to do for it.
template <bool PAGED, int BM> __device__ __forceinline__ bool attn_block(const AttnArgs& a, uint32_t bid, int thread, int threads, AttnBlock& k) {
    k.hk = (int)(bid % (uint32_t)a.Hkv);
    bid /= (uint32_t)a.Hkv;
    k.split = (int)(bid % (uint32_t)a.nsplit);
    bid /= (uint32_t)a.nsplit;
    int tile;
    if constexpr (PAGED) {
        // the last slots first: the later tokens of a prompt have the most keys
        const int64_t slot = (int64_t)a.tiles - 1 - bid;
        k.s = slot_sequence<BM>(a, slot);
        const int64_t tl = slot - (k.s.tok0 * a.G / BM + k.s.b);
        // without a window the first page follows from the split alone: its number is on its way
        // together with the length
        k.from = -64;
        k.table = -1;
        if (!a.window && a.max_pages > 0) {
            const int64_t j = a.nsplit > 1 ? (int64_t)k.split * a.share : 0;
            k.from = min((int)a.fd_ps.div((uint32_t)min(j, (int64_t)0x7FFFFFFF)), a.max_pages - 1);
            const int64_t p = a.pages[(int64_t)k.s.b * a.max_pages + min(k.from + (int)(threadIdx.x & 63), a.max_pages - 1)];
            k.table = p >= 0 && p < a.npages ? (int)p : -1;
        }
        tile = uniform(tl < 0 || tl > 0x7FFFFFFF / BM ? -1 : (int)tl);
        if (tile < 0) return false;
    } else {
        const uint32_t tl = bid % (uint32_t)a.tiles;
        tile = a.tiles - 1 - (int)tl;
        k.s = attn_seq<PAGED>(a, (int)(bid / (uint32_t)a.tiles));
    }
    k.s.n = uniform(k.s.n);
    k.s.len = uniform(k.s.len);
    k.s.first = uniform(k.s.first);
    const int nrows = k.s.n * a.G;             // below 2^31: the host sees to it
    k.row0 = tile * BM;
    if (k.row0 >= nrows) return false;
    k.rows = min(BM, nrows - k.row0);
    const int tok0 = (int)a.fd_g.div((uint32_t)k.row0), tok1 = (int)a.fd_g.div((uint32_t)(k.row0 + k.rows - 1));
    k.klo = attn_lo(a, k.s, tok0) & ~31;
    k.khi = attn_hi(a, k.s, tok1);
    if (a.nsplit > 1) {                        // this split's share
        const int64_t at = (int64_t)k.klo + (int64_t)k.split * a.share;
        if (k.split + 1 < a.nsplit) k.khi = (int)min((int64_t)k.khi, at + a.share);      // the last one takes what is left
        if (at >= k.khi) {                     // no keys: it weighs nothing
            for (int r = thread; r < k.rows; r += threads)
                a.part_ml[(int64_t)k.split * a.rows + attn_row_at<PAGED>(a, k, r).out] = make_float2(-INFINITY, 0.0f);
            return false;
        }
        k.klo = (int)at;
    }
    return true;
}

// ---- a wave's sums ------------------------------------------------------------------------
// EARLY: LDS fragments are read ahead of a group of products.
template <int DT, int D, bool PAGED, bool MASK, int MR, bool EARLY> struct AttnWave {
    typedef typename AttnAcc<MR>::type Acc;
    static constexpr int ES = kElem<DT>, VEC = 16 / ES, CH = D / VEC, RB = D * ES;
    static constexpr int GR = 64 / MR;         // lanes of a row
    static constexpr int NP = 32 / GR;         // keys of a lane, of 32
    static constexpr int NS = CH / GR;         // chunks of a row of Q in a lane
    static constexpr int NO = D / MR, NR = MR * MR / 64;       // result blocks, registers of each

    uint4 q[NS];
    Acc o[NO];
    float m, l, c;                             // maximum so far, this lane's part of the sum, exp2's factor
    int lr, h;                                 // the lane's row, and which of the row's lanes it is
    int lo, hi;                                // keys that the row sees
    int any_lo, any_hi, all_lo, all_hi;        // that some row of the wave sees, and all of them
    int64_t mo;                                // the row's mask
    bool live;

    // key i of this lane's, of 32; and column i of a result block's registers
    TOHIP_INLINE __device__ int key(int i) const { return 4 * GR * (i >> 2) + 4 * h + (i & 3); }

    // Rows [r0, r0 + MR) of the block; those past its end repeat the last and are not stored.
    TOHIP_INLINE __device__ AttnRow begin(const AttnArgs& a, const AttnBlock& k, int r0) {
        const int lane = (int)(threadIdx.x & 63);
        lr = lane & (MR - 1);
        h = lane / MR;
        live = r0 + lr < k.rows;
        const AttnRow w = attn_row_at<PAGED>(a, k, min(r0 + lr, k.rows - 1));
        lo = max(k.klo, attn_lo(a, k.s, w.tok));
        hi = min(k.khi, attn_hi(a, k.s, w.tok));
        const int tok0 = (int)a.fd_g.div((uint32_t)(k.row0 + min(r0, k.rows - 1)));
        const int tok1 = (int)a.fd_g.div((uint32_t)(k.row0 + min(r0 + MR - 1, k.rows - 1)));
        any_lo = max(k.klo, attn_lo(a, k.s, tok0));
        any_hi = r0 < k.rows ? min(k.khi, attn_hi(a, k.s, tok1)) : 0;
        all_lo = max(k.klo, attn_lo(a, k.s, tok1));
        all_hi = min(k.khi, attn_hi(a, k.s, tok0));
        const int64_t qo = PAGED ? (k.s.tok0 + w.tok) * a.qt + w.head * a.qh : k.s.b * a.qb + w.tok * a.qt + w.head * a.qh;
        const uint4* qp = reinterpret_cast<const uint4*>((const char*)a.q + qo * ES);
        const int qch = a.Dk / VEC;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int ch = GR * i + h;
            q[i] = live && ch < qch ? qp[ch] : uint4{0, 0, 0, 0};
        }
        mo = MASK ? k.s.b * a.mb + w.head * a.mh + w.tok * a.mq : 0;
#pragma unroll
        for (int d = 0; d < NO; d++)
#pragma unroll
            for (int i = 0; i < NR; i++) o[d][i] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
        c = MASK ? kLog2e : a.scale * kLog2e;
        return w;
    }

    // Waits for Q here: waited for at its first use, inside the walk, the compiler would wait for
    // every load in flight there, each time round.
    TOHIP_INLINE __device__ void have_q() {
#pragma unroll
        for (int i = 0; i < NS; i++) asm volatile("" : "+v"(q[i].x), "+v"(q[i].y), "+v"(q[i].z), "+v"(q[i].w));
    }

    // q.k of the 32 keys in rows sub .. of a tile.
    TOHIP_INLINE __device__ void products(const char* kt, int sub, float (&x)[NP]) {
        Acc s[NP / NR];
#pragma unroll
        for (int u = 0; u < NP / NR; u++) {
#pragma unroll
            for (int i = 0; i < NR; i++) s[u][i] = 0.0f;
        }
        constexpr int U = NP / NR, NF = NS * U, G = !EARLY ? 1 : NF < 8 ? NF : 8;
#pragma unroll
        for (int g = 0; g < NF; g += G) {
            uint4 kf[G];
            uint32_t at[G];
#pragma unroll
            for (int f = 0; f < G; f++) {
                const int i = (g + f) / U, r = (g + f) % U * MR + lr;
                const char* p = kt + (sub + r) * RB + key_place<CH>(r, GR * i + h) * 16;
                if constexpr (EARLY) at[f] = lds_address(p);
                else kf[f] = *reinterpret_cast<const uint4*>(p);
            }
            if constexpr (G == 4) read_keys4(at, kf);
            if constexpr (G == 8) read_keys8(at, kf);
#pragma unroll
            for (int f = 0; f < G; f++) {
                const int i = (g + f) / U, u = (g + f) % U;
                if constexpr (DT == kF32) {
                    s[u] = mfma32<MR>(u2f(kf[f].x), u2f(q[i].x), s[u]);
                    s[u] = mfma32<MR>(u2f(kf[f].y), u2f(q[i].y), s[u]);
                    s[u] = mfma32<MR>(u2f(kf[f].z), u2f(q[i].z), s[u]);
                    s[u] = mfma32<MR>(u2f(kf[f].w), u2f(q[i].w), s[u]);
                } else {
                    s[u] = mfma16<DT, MR>(kf[f], q[i], s[u]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NP; i++) x[i] = s[i / NR][i % NR];
    }

    // Scores of the 32 keys from jb on (without a mask still unscaled), -inf where not seen.
    TOHIP_INLINE __device__ void close(const AttnArgs& a, int jb, float (&x)[NP]) {
        const bool inside = jb >= all_lo && jb + 32 <= all_hi;
        if constexpr (MASK) {
            float bias[NP];
            if (inside && a.mk) {              // four keys at a time
#pragma unroll
                for (int i = 0; i < NP; i += 4) {
                    const int64_t at = mo + jb + key(i);
                    if (a.mask_dt == kU8 || a.mask_dt == kI8) {
                        uint32_t w;
                        __builtin_memcpy(&w, (const uint8_t*)a.mask + at, 4);
#pragma unroll
                        for (int e = 0; e < 4; e++) bias[i + e] = (w >> (8 * e)) & 0xFF ? 0.0f : -INFINITY;
                    } else if (DT == kF32 || a.mask_dt == kF32) {
                        __builtin_memcpy(bias + i, (const float*)a.mask + at, 16);
                    } else {
                        uint16_t w[4];
                        __builtin_memcpy(w, (const uint16_t*)a.mask + at, 8);
#pragma unroll
                        for (int e = 0; e < 4; e++) bias[i + e] = ld_f<DT>(w, e);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int j = jb + key(i);
                    bias[i] = -INFINITY;
                    if (j >= lo && j < hi) {
                        const int64_t at = mo + (int64_t)j * a.mk;
                        if (a.mask_dt == kU8 || a.mask_dt == kI8) bias[i] = ((const uint8_t*)a.mask)[at] ? 0.0f : -INFINITY;
                        else if (a.mask_dt == kF32) bias[i] = ((const float*)a.mask)[at];
                        else bias[i] = ld_f<DT>(a.mask, at);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < NP; i++) x[i] = bias[i] == -INFINITY ? -INFINITY : __builtin_fmaf(x[i], a.scale, bias[i]);
        } else if (!inside) {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int j = jb + key(i);
                x[i] = j >= lo && j < hi ? x[i] : -INFINITY;
            }
        }
    }

    // The largest of a row's scores.
    TOHIP_INLINE __device__ float top_of(const float (&x)[NP]) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i < NP; i++) top = fmaxf(top, x[i]);
        float ta, tb;
        if constexpr (GR == 4) {
            permlane_pair<16>(top, ta, tb);
            top = fmaxf(ta, tb);
        }
        permlane_pair<32>(top, ta, tb);
        return fmaxf(ta, tb);
    }
    // Scores to weights against the maximum m.
    TOHIP_INLINE __device__ void weights(float (&x)[NP]) {
        const float base = m == -INFINITY ? 0.0f : m;
        if constexpr (MASK) {
            // the difference first: a mask of the type's lowest value times log2 e would overflow
#pragma unroll
            for (int i = 0; i < NP; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i] - base, c, kRaise<DT>));
        } else {
            const float off = kRaise<DT> - base * c;
#pragma unroll
            for (int i = 0; i < NP; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, off));
        }
    }
    // The sums, which stand against the maximum `was`, against m.
    TOHIP_INLINE __device__ void rescale(float was) {
        const float f = m == was ? 1.0f : __builtin_amdgcn_exp2f((was - m) * c);
        l *= f;
#pragma unroll
        for (int d = 0; d < NO; d++)
#pragma unroll
            for (int i = 0; i < NR; i++) o[d][i] *= f;
    }
    TOHIP_INLINE __device__ void weigh(float (&x)[NP]) {
        const float top = top_of(x);
        if (__ballot((top - m) * c > kLazy)) {
            const float was = m;
            m = fmaxf(m, top);
            rescale(was);
        }
        weights(x);
    }

    // A lane's weights: 16-bit types rounded to the type and packed as the product's operand, since
    // the matrix unit takes both operands in one type (values in two parts would double the work).
    // Off by half a step each.  The sum is that of the rounded ones, so that such an error moves the
    // mean between the values but never scales it, and a weight that takes nearly everything has
    // none.  (With the sum of the unrounded ones the error of one float16 token over 1500 keys was up
    // to 2.1 times that of float32 weights, in 10000 draws, now 1.7; bfloat16 over 1025 keys 2.0 and
    // 1.45; on average 1.25 either way.  It costs 34.0 -> 36.2 us for 448 queries over 300 .. 1500
    // keys of 16 heads of 64, eight batches; nothing measurable over pages, where heads are longer
    // or rows few.)
    static constexpr int NPV = DT == kF32 ? NP : 1, NKK = DT == kF32 ? 1 : NP / 8;
    struct Weights {
        uint4 h[NKK];
        float f[NPV];
    };
    TOHIP_INLINE __device__ void pack(const float (&x)[NP], Weights& p) {
        float sum[2] = {0.0f, 0.0f};
        if constexpr (DT == kF32) {
#pragma unroll
            for (int i = 0; i < NP; i++) {
                p.f[i] = x[i];
                sum[i & 1] += x[i];
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < NKK; kk++) {
                p.h[kk] = __builtin_bit_cast(uint4, round16<DT, 8>(x + 8 * kk));
                sum[0] = add_pair<DT>(p.h[kk].x, sum[0]);
                sum[1] = add_pair<DT>(p.h[kk].y, sum[1]);
                sum[0] = add_pair<DT>(p.h[kk].z, sum[0]);
                sum[1] = add_pair<DT>(p.h[kk].w, sum[1]);
            }
        }
        l += sum[0] + sum[1];
    }
    // The weighted values of the 32 keys in rows sub .. of a tile.
    TOHIP_INLINE __device__ void add(const char* vt, int sub, const Weights& p) {
        if constexpr (DT == kF32) {
#pragma unroll
            for (int d = 0; d < NO; d++) {
                // (a lane's rows are turned by the same amount)
                const char* at = vt + (sub + 4 * h) * RB + value_place<DT, CH, MR>(4 * h, d * (MR / 4) + (lr >> 2)) * 16 + (lr & 3) * 4;
#pragma unroll
                for (int g = 0; g < NP; g += 8) {
                    float vf[8];
                    if constexpr (EARLY) {
                        read_column8<RB, 4 * GR>(lds_address(at + GR * g * RB), vf);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            vf[i] = *reinterpret_cast<const float*>(at + (4 * GR * ((g + i) >> 2) + (i & 3)) * RB);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) o[d] = mfma32<MR>(vf[i], p.f[g + i], o[d]);
                }
            }
        } else {
            const int lane = (int)(threadIdx.x & 63), r4 = (lane & 15) >> 2;
            const int cc = (MR == 32 ? ((lane >> 4) & 1) * 2 : 0) + ((lane & 3) >> 1), in = (lane & 1) * 8;
            constexpr int G = EARLY ? (NO < 4 ? NO : 4) : 1;
            static_assert(G == 1 || G == 4 || NO == 2, "groups");
#pragma unroll
            for (int kk = 0; kk < NP / 8; kk++) {
                const uint4 pf = p.h[kk];
                const int r = sub + 8 * GR * kk + 4 * h + r4;
#pragma unroll
                for (int g = 0; g < NO; g += G) {
                    uint2 x[G], y[G];
                    uint32_t at[G];
#pragma unroll
                    for (int f = 0; f < G; f++) {
                        // (row r + 4 GR is turned by the same amount as row r)
                        const char* v = vt + r * RB + value_place<DT, CH, MR>(r, (g + f) * (MR / 8) + cc) * 16 + in;
                        if constexpr (G == 4) {
                            at[f] = lds_address(v);
                        } else {
                            x[f] = read_turned(v);
                            y[f] = read_turned(v + 4 * GR * RB);
                        }
                    }
                    if constexpr (G == 4) read_values<4 * GR * RB>(at, x, y);
#pragma unroll
                    for (int f = 0; f < G; f++) o[g + f] = mfma16<DT, MR>(uint4{x[f].x, x[f].y, y[f].x, y[f].y}, pf, o[g + f]);
                }
            }
        }
    }

    // Divides, stores, and has rows whose result is not finite (or all: again) computed again.
    TOHIP_INLINE __device__ void end(const AttnArgs& a, const AttnBlock& k, int r0, const AttnRow& w, bool again) {
        float la, lb;
        if constexpr (GR == 4) {
            permlane_pair<16>(l, la, lb);
            l = la + lb;
        }
        permlane_pair<32>(l, la, lb);
        l = la + lb;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const bool parts = a.parts;
        // (no weight although a key was seen: the scores are past what float32 holds in log2 units)
        bool bad = again || (l == 0.0f && m > -INFINITY);
#pragma unroll
        for (int d = 0; d < NO; d++) {
#pragma unroll
            for (int g = 0; g < NR / 4; g++) {
                const int col = d * MR + key(4 * g);
                if (col >= a.Dv) continue;
                float r[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    r[e] = l == 0.0f ? 0.0f : o[d][4 * g + e] * inv;
                    bad |= !(__builtin_fabsf(r[e]) <= 3.402823466e38f);
                }
                if (!live) continue;
                if (parts) {
                    *reinterpret_cast<float4*>(a.part_o + ((int64_t)k.split * a.rows + w.out) * a.Dv + col) = make_float4(r[0], r[1], r[2], r[3]);
                } else if constexpr (DT == kF32) {
                    *reinterpret_cast<float4*>((float*)a.y + w.y + col) = make_float4(r[0], r[1], r[2], r[3]);
                } else {
                    *reinterpret_cast<uint2*>((uint16_t*)a.y + w.y + col) = __builtin_bit_cast(uint2, round16<DT, 4>(r));
                }
            }
        }
        // The maximum as a score: times log2 e it would overflow where scores are near float32's
        // largest, and splits of other maxima would count as equal.  (1 / 2^kRaise is exact.)
        if (parts && live && h == 0)
            a.part_ml[(int64_t)k.split * a.rows + w.out] = make_float2(MASK || m == -INFINITY ? m : m * a.scale, l * kLower<DT>);
        unsigned long long rows = __ballot(bad && live);
        rows |= rows >> 32;
        if constexpr (GR == 4) rows |= rows >> 16;
        rows &= (1ull << MR) - 1;
        for (; rows; rows &= rows - 1) {
            const AttnRow x = attn_row_at<PAGED>(a, k, r0 + __builtin_ctzll(rows));
            float rm = -INFINITY, rl = 0.0f;
            attn_row<DT, PAGED>(a, k.s, x.head, x.tok, k.klo, k.khi, rm, rl, [&](int d, float v) {
                if (parts) a.part_o[((int64_t)k.split * a.rows + x.out) * a.Dv + d] = v;
                else st_code<DT>(a.y, x.y + d, v);
            });
            if (parts && (threadIdx.x & 63) == 0) a.part_ml[(int64_t)k.split * a.rows + x.out] = make_float2(rm, rl);
        }
    }
};

// ---- loads of a tile ------------------------------------------------------------------------
// A tile of keys starts at a multiple of 32.  Instruction i of wave w fills the rows
// (i W + w) RPI .. of K's or V's tile.  The first rows' offsets are worked out by one lane each,
// all at once; a lane's offset from them is kept in a register: worked out per lane and
// instruction, the addresses of paged keys took longer than the loads themselves.  Rows past the last key
// repeat it.  Pages whose size an instruction's rows do not divide are looked up row by row.
// A wave holds 64 of the sequence's page numbers in a register: looked up in memory for each
// tile, they were a second trip to it per tile (32 keys of one wave: 1.4 us).  A tile's pages are
// all among them: a tile has at most 64 keys, or 128 that begin at an even one where pages have two
// keys or more (the host sees to it).
// Columns past the head size repeat the last chunk: Q is zero there, and where the product of
// a value that is not finite is not either, the row is computed again.
template <int DT, int D, bool PAGED, int MR, int W> struct AttnLoads {
    static constexpr int ES = kElem<DT>, VEC = 16 / ES, CH = D / VEC, RB = D * ES, RPI = 1024 / RB;
    const char *kbase, *vbase;
    int table;                                 // lane n: page from + n of the sequence
    int wave, lane, lrow, lslot, kch, vch, kstep, vstep, last, b;
    int from;
    int64_t koff, voff;                        // of the found tile: lane n has its row n RPI's
    bool even;
    int worst;                                 // < 0: some key's page was none of the cache's

    TOHIP_INLINE __device__ void begin(const AttnArgs& a, const AttnBlock& k, int w) {
        lane = (int)(threadIdx.x & 63);
        kbase = (const char*)a.k + k.hk * a.kh * ES;
        vbase = (const char*)a.v + k.hk * a.vh * ES;
        wave = w;
        lrow = lane / CH;
        lslot = lane % CH;
        kch = a.Dk / VEC;
        vch = a.Dv / VEC;
        kstep = (int)a.kt * ES;
        vstep = (int)a.vt * ES;
        last = k.s.len - 1;
        b = k.s.b;
        even = !PAGED || (a.ps & (RPI - 1)) == 0;
        worst = 0;
        koff = voff = 0;
        table = PAGED ? k.table : -1;
        from = PAGED ? k.from : -64;           // (-64: nothing in it yet)
    }
    TOHIP_INLINE __device__ int entry(const AttnArgs& a, int j) const { return __shfl(table, (int)a.fd_ps.div((uint32_t)j) - from); }
    // Looks up the pages of the tile of KEYS keys at j0, and where its instructions' rows begin.
    template <int KEYS> TOHIP_INLINE __device__ void find(const AttnArgs& a, int j0) {
        static_assert(KEYS <= kTablePages || KEYS == kKeys256, "pages of a tile");
        const int end = min(j0 + KEYS - 1, last), j = min(j0 + lane * RPI, end);
        int pg = 0;
        if constexpr (PAGED) {
            if ((int)a.fd_ps.div((uint32_t)end) >= from + 64) {
                from = (int)a.fd_ps.div((uint32_t)min(j0, last));
                const int i = min(from + lane, (int)a.fd_ps.div((uint32_t)last));
                const int64_t p = a.pages[(int64_t)b * a.max_pages + i];
                table = p >= 0 && p < a.npages ? (int)p : -1;
            }
            if (!even) return;
            pg = entry(a, j);
            if (__ballot(pg < 0)) worst = -1;
            pg = max(pg, 0);
        }
        const KeyRow at = attn_key_row<PAGED>(a, b, pg, j);
        koff = at.k * ES;
        voff = at.v * ES;
    }
    // One operand's tile (V: the values').
    template <bool V, int NI> TOHIP_INLINE __device__ void load(const AttnArgs& a, char* to, int j0) {
        const char* base = V ? vbase : kbase;
        const int step = V ? vstep : kstep, ch = (V ? vch : kch) - 1;
        auto chunk = [&](int r) TOHIP_INLINE {
            return (uint32_t)min(V ? value_place<DT, CH, MR>(r, lslot) : key_place<CH>(r, lslot), ch) * 16u;
        };
        auto first = [&](int i) TOHIP_INLINE {                 // the address of the instruction's first row
            const uint64_t off = (uint64_t)(V ? voff : koff);
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)off, i * W + wave);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(off >> 32), i * W + wave);
            return base + (((uint64_t)hi << 32) | lo);
        };
        if (even && j0 + NI * W * RPI - 1 <= last) {
#pragma unroll
            for (int i = 0; i < NI; i++)
                load_lds16(first(i) + ((uint32_t)(lrow * step) + chunk((i * W + wave) * RPI + lrow)), to + (i * W + wave) * 1024);
        } else if (even) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int r0 = (i * W + wave) * RPI, j = min(j0 + r0, last);
                load_lds16(first(i) + ((uint32_t)(min(lrow, last - j) * step) + chunk(r0 + lrow)), to + (i * W + wave) * 1024);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < NI; i++) {
                const int r = (i * W + wave) * RPI + lrow, j = min(j0 + r, last);
                int pg = 0;
                if constexpr (PAGED) {
                    pg = entry(a, j);
                    if (__ballot(pg < 0)) worst = -1;
                    pg = max(pg, 0);
                }
                const KeyRow at = attn_key_row<PAGED>(a, b, pg, j);
                load_lds16(base + (V ? at.v : at.k) * ES + chunk(r), to + (i * W + wave) * 1024);
            }
        }
    }
};

// The four tiles that a kernel keeps in LDS, N bytes each.  As variables of their own: as parts of one
// array, or as a function's arguments, the compiler waits for loads into one tile before it reads
// another and checks each address that a load writes to (cache attention, single tokens over up to
// 300 keys: 55 us, else 59).
template <int N> struct Tiles {
    template <int I> TOHIP_INLINE __device__ char* at() const {
        __shared__ __attribute__((aligned(1024))) char t[N];
        return t;
    }
};
// One behind the other in an array, for the kernels behind a prefix, whose code for two parts is as fast
// with one as with the other (4 tokens behind 2000 keys 15.0 us, as variables 15.6; 3 in float16 behind
// 4915 15.3 and 14.7) and whose waves divide it otherwise.
template <int N> struct TilesAt {
    char* lds;
    template <int I> TOHIP_INLINE __device__ char* at() const { return lds + I * N; }
};

// Prompts: W waves of 32 rows share tiles of BN keys, two deep: while tile n is worked on, tile
// n + 1 is on its way.  S' = K Q' leaves a query's scores in one lane pair, in the order in
// which O' += V' P' takes its weights, so they never leave the registers; 32 rows per wave are
// what the products' largest form takes with the sums of 128 columns still in registers.
// Bound by the matrix and vector units together (32 keys of 32 rows: 512 cycles of products at
// 128 values per head, about as many for the 16 exponentials per lane and what surrounds them)
// and, at full length, by power: 4096 queries over 8192 keys, 32 heads of 128 in bf16, 538 .. 557 us
// by card or 1.0 PFLOP/s; the last 4096 of 16384 keys in pages of 16, 980 .. 1020 us (630 and
// 1080 in the first hundred calls of an idle card, whose clock rises meanwhile).  With 64 values per head the
// exponentials weigh twice as much.
template <int DT, int D, bool PAGED, bool MASK, int W, int BN, class TILES>
TOHIP_INLINE __device__ void attn_tiles(const AttnArgs& a, uint32_t bid, TILES tiles) {
    typedef AttnWave<DT, D, PAGED, MASK, 32, (D <= 128)> Wave;      // (as far as registers go)
    constexpr int RB = Wave::RB, NI = BN * RB / (1024 * W);
    static_assert(NI >= 1, "tile");
    char *k0_ = tiles.template at<0>(), *k1_ = tiles.template at<1>(), *v0_ = tiles.template at<2>(), *v1_ = tiles.template at<3>();
    __shared__ int missing;                    // a key's page was none of the cache's
    const int t = (int)threadIdx.x, wave = uniform(t >> 6);
    AttnBlock k;
    if (!attn_block<PAGED, 32 * W>(a, bid, t, 64 * W, k)) return;
    Wave w;
    const AttnRow row = w.begin(a, k, wave * 32);
    AttnLoads<DT, D, PAGED, 32, W> ld;
    ld.begin(a, k, wave);
    if (t == 0) missing = 0;
    __syncthreads();
    auto step = [&](int j0, const char* kt, const char* vt, char* kn, char* vn) TOHIP_INLINE {
        wait_loads<0>();
        __builtin_amdgcn_s_barrier();          // every wave's part of this tile is there, and the other buffer is free
        __builtin_amdgcn_sched_barrier(0);
        if (j0 + BN < k.khi) {
            ld.template load<false, NI>(a, kn, j0 + BN);
            ld.template load<true, NI>(a, vn, j0 + BN);
            ld.template find<BN>(a, j0 + 2 * BN);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int sub = 0; sub < BN; sub += 32) {
            const int jb = j0 + sub;
            if (jb >= w.any_hi || jb + 32 <= w.any_lo) continue;
            float x[Wave::NP];
            typename Wave::Weights p;
            w.products(kt, sub, x);
            w.close(a, jb, x);
            w.weigh(x);
            w.pack(x, p);
            w.add(vt, sub, p);
        }
    };
    if (k.klo < k.khi) {
        ld.template find<BN>(a, k.klo);
        if (PAGED) w.have_q();
        ld.template load<false, NI>(a, k0_, k.klo);
        ld.template load<true, NI>(a, v0_, k.klo);
        ld.template find<BN>(a, k.klo + BN);
        if (!PAGED) w.have_q();
        for (int j0 = k.klo; j0 < k.khi; j0 += 2 * BN) {
            step(j0, k0_, v0_, k1_, v1_);
            if (j0 + BN < k.khi) step(j0 + BN, k1_, v1_, k0_, v0_);
        }
    }
    if (PAGED && ld.worst < 0) missing = 1;
    __syncthreads();
    if (wave * 32 < k.rows) w.end(a, k, wave * 32, row, missing != 0);
}
template <int DT, int D, bool PAGED, bool MASK, int W, int BN>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(D * kElem<DT> <= 128 && W == 4 && !MASK ? 3 : D * kElem<DT> <= 256 ? 2 : 1))) void k_attn_tiles(AttnArgs a) {
    attn_tiles<DT, D, PAGED, MASK, W, BN>(a, blockIdx.x, Tiles<BN * D * kElem<DT>>());
}

// Few rows: a block is one wave, so nothing waits for another.  K and V have two buffers of
// 32 keys each; K's is filled again as soon as its scores are made and V's as soon as it is
// added, so three of the four are in flight while one is worked on.  Bound by memory: 64
// tokens of 32 heads over 130 .. 8192 keys of 8 heads of 128 in bf16 take 220 us, 5.0 TB/s
// (filled a whole tile at a time 261); one token over 1025 keys 12.3 us, of which 4 are the
// join's launch and the rest a chain of loads: starts, length, pages, keys.  float32 heads of more
// than 64 values take 64 or 128 KB of LDS per wave and, for 256 values and 32 rows, more than 512
// registers, so two waves or one run on a CU: 16 tokens of 16 heads over 130 .. 4096 keys of 4
// heads reach 2.0 TB/s with 64 values, 2.2 with 128, 1.5 with 256.
template <int DT, int D, bool PAGED, bool MASK, int MR, class TILES> TOHIP_INLINE __device__ void attn_few(const AttnArgs& a, uint32_t bid, TILES tiles) {
    typedef AttnWave<DT, D, PAGED, MASK, MR, (MR == 16 || D <= 128)> Wave;      // (as far as registers go)
    constexpr int RB = Wave::RB, NI = 32 * RB / 1024;
    char *k0_ = tiles.template at<0>(), *k1_ = tiles.template at<1>(), *v0_ = tiles.template at<2>(), *v1_ = tiles.template at<3>();
    AttnBlock k;
    if (!attn_block<PAGED, MR>(a, bid, (int)threadIdx.x, 64, k)) return;
    Wave w;
    const AttnRow row = w.begin(a, k, 0);
    AttnLoads<DT, D, PAGED, MR, 1> ld;
    ld.begin(a, k, 0);
    // In flight behind a tile's K: its V, and K and V of the next tile if there is one; behind
    // its V: those, and K of the tile after that.
    auto step = [&](int j0, char* kt, char* vt, bool next, bool third) TOHIP_INLINE {
        float x[Wave::NP];
        if (next) wait_loads<3 * NI>();
        else wait_loads<NI>();
        __builtin_amdgcn_sched_barrier(0);
        w.products(kt, 0, x);
        if (third) ld.template load<false, NI>(a, kt, j0 + 64);
        __builtin_amdgcn_sched_barrier(0);
        w.close(a, j0, x);
        w.weigh(x);
        if (third) wait_loads<3 * NI>();
        else if (next) wait_loads<2 * NI>();
        else wait_loads<0>();
        __builtin_amdgcn_sched_barrier(0);
        typename Wave::Weights p;
        w.pack(x, p);
        w.add(vt, 0, p);
        if (third) {
            ld.template load<true, NI>(a, vt, j0 + 64);
            ld.template find<32>(a, j0 + 96);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (k.klo < k.khi) {
        ld.template find<32>(a, k.klo);
        if (PAGED) w.have_q();
        ld.template load<false, NI>(a, k0_, k.klo);
        ld.template load<true, NI>(a, v0_, k.klo);
        if (k.klo + 32 < k.khi) {
            ld.template find<32>(a, k.klo + 32);
            ld.template load<false, NI>(a, k1_, k.klo + 32);
            ld.template load<true, NI>(a, v1_, k.klo + 32);
            ld.template find<32>(a, k.klo + 64);
        }
        if (!PAGED) w.have_q();
        // (a loop of its own for the steps with nothing conditional about their loads, or the
        // compiler, which does not see which waits belong to which loads, waits for all of them)
        int j0 = k.klo;
        for (; j0 + 96 < k.khi; j0 += 64) {
            step(j0, k0_, v0_, true, true);
            step(j0 + 32, k1_, v1_, true, true);
        }
        for (; j0 < k.khi; j0 += 64) {
            step(j0, k0_, v0_, j0 + 32 < k.khi, j0 + 64 < k.khi);
            if (j0 + 32 < k.khi) step(j0 + 32, k1_, v1_, j0 + 64 < k.khi, false);
        }
    }
    w.end(a, k, 0, row, PAGED && ld.worst < 0);
}
template <int DT, int D, bool PAGED, bool MASK, int MR>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(D * kElem<DT> <= 256 ? 2 : 1))) void k_attn_few(AttnArgs a) {
    attn_few<DT, D, PAGED, MASK, MR>(a, blockIdx.x, Tiles<32 * D * kElem<DT>>());
}

// ---- behind a shared prefix --------------------------------------------------------------
// The rows of all sequences over the prefix (pre) and each sequence's over its own keys (own), in one
// launch where both are cut into blocks of one size: the first `first` blocks are the prefix's.
// One after the other, the second part would wait for the first one's last block; and where the
// prefix is bound by its products and single tokens by their keys' bytes, they run beside each other.
template <int DT, int D, int MR>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(2))) void k_prefix_few(AttnArgs pre, AttnArgs own, unsigned first) {
    __shared__ __attribute__((aligned(1024))) char lds[128 * D * kElem<DT>];
    if (blockIdx.x < first) attn_few<DT, D, true, false, MR>(pre, blockIdx.x, TilesAt<32 * D * kElem<DT>>{lds});
    else attn_few<DT, D, true, false, MR>(own, blockIdx.x - first, TilesAt<32 * D * kElem<DT>>{lds});
}
template <int DT, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D * kElem<DT> <= 128 ? 3 : 2))) void k_prefix_tiles(AttnArgs pre, AttnArgs own, unsigned first) {
    __shared__ __attribute__((aligned(1024))) char lds[256 * D * kElem<DT>];
    if (blockIdx.x < first) attn_tiles<DT, D, true, false, 4, 64>(pre, blockIdx.x, TilesAt<64 * D * kElem<DT>>{lds});
    else attn_tiles<DT, D, true, false, 4, 64>(own, blockIdx.x - first, TilesAt<64 * D * kElem<DT>>{lds});
}
// Few rows as one of a block's four waves that know nothing of each other, in a quarter of the LDS of
// its tiles: one buffer for K and one for V, filled again as soon as they are read.  (Eight such waves
// on a CU have as many bytes on their way as five with four buffers.)
template <int DT, int D, int MR> TOHIP_INLINE __device__ void attn_few_wave(const AttnArgs& a, uint32_t bid, char* lds) {
    typedef AttnWave<DT, D, true, false, MR, (MR == 16 || D <= 128)> Wave;
    constexpr int RB = Wave::RB, NI = 32 * RB / 1024;
    char *kt = lds, *vt = lds + 32 * RB;
    AttnBlock k;
    if (!attn_block<true, MR>(a, bid, (int)(threadIdx.x & 63), 64, k)) return;
    Wave w;
    const AttnRow row = w.begin(a, k, 0);
    AttnLoads<DT, D, true, MR, 1> ld;
    ld.begin(a, k, 0);
    auto step = [&](int j0, bool next) TOHIP_INLINE {
        float x[Wave::NP];
        wait_loads<NI>();                      // (V's are on their way)
        __builtin_amdgcn_sched_barrier(0);
        w.products(kt, 0, x);
        __builtin_amdgcn_sched_barrier(0);     // (the tile is read before it is filled again)
        if (next) ld.template load<false, NI>(a, kt, j0 + 32);
        __builtin_amdgcn_sched_barrier(0);
        w.close(a, j0, x);
        w.weigh(x);
        if (next) wait_loads<NI>();
        else wait_loads<0>();
        __builtin_amdgcn_sched_barrier(0);
        typename Wave::Weights p;
        w.pack(x, p);
        w.add(vt, 0, p);
        __builtin_amdgcn_sched_barrier(0);
        if (next) {
            ld.template load<true, NI>(a, vt, j0 + 32);
            ld.template find<32>(a, j0 + 64);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (k.klo < k.khi) {
        ld.template find<32>(a, k.klo);
        w.have_q();
        ld.template load<false, NI>(a, kt, k.klo);
        ld.template load<true, NI>(a, vt, k.klo);
        ld.template find<32>(a, k.klo + 32);
        int j0 = k.klo;
        for (; j0 + 32 < k.khi; j0 += 32) step(j0, true);
        step(j0, false);
    }
    w.end(a, k, 0, row, ld.worst < 0);
}
template <int DT, int D, int MR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void k_prefix_both(AttnArgs pre, AttnArgs own, unsigned first, unsigned own_blocks) {
    __shared__ __attribute__((aligned(1024))) char lds[256 * D * kElem<DT>];
    if (blockIdx.x < first) {
        attn_tiles<DT, D, true, false, 4, 64>(pre, blockIdx.x, TilesAt<64 * D * kElem<DT>>{lds});
    } else {
        const int wave = uniform((int)threadIdx.x >> 6);
        const unsigned bid = (blockIdx.x - first) * 4 + (unsigned)wave;
        if (bid < own_blocks) attn_few_wave<DT, D, MR>(own, bid, lds + wave * 64 * D * kElem<DT>);
    }
}

// ---- the splits of a row together -----------------------------------------------------
// y = sum_s w_s o_s, w_s = l_s exp(m_s - max) / sum: a wave per row.  Lanes hold the splits'
// weights, two each; then groups of Dv / 4 lanes add every group's share of the splits, four
// columns per lane, kJoin splits at a time (one split after the other, by a thread per four
// columns, took 38 us for 47 splits of 16 rows).
constexpr int kJoin = 4;
template <int DT, bool PAGED> __global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    const int lane = (int)threadIdx.x & 63, quads = a.Dv / 4, groups = 64 / quads;
    const int grp = lane / quads, col = (lane - grp * quads) * 4;      // (lanes past the last group repeat the last split)
    const int64_t step = (int64_t)gridDim.x * 4;
    for (int64_t row = (int64_t)blockIdx.x * 4 + uniform((int)(threadIdx.x >> 6)); row < a.rows; row += step) {
        const int64_t token = row / a.Hq;
        const int head = (int)(row - token * a.Hq);
        int64_t yo;
        if constexpr (PAGED) {
            if (token < a.qstart[0] || token >= a.qstart[a.B]) continue;      // behind the last sequence
            yo = token * a.yt + head * a.yh;
        } else {
            const int64_t b = token / a.Sq;
            yo = b * a.yb + (token - b * a.Sq) * a.yt + head * a.yh;
        }
        const float2 none = make_float2(-INFINITY, 0.0f);
        const float2 ml0 = lane < a.nsplit ? a.part_ml[lane * a.rows + row] : none;
        const float2 ml1 = lane + 64 < a.nsplit ? a.part_ml[(lane + 64) * a.rows + row] : none;
        float4 v[kJoin];
        auto read = [&](int s0) TOHIP_INLINE {
#pragma unroll
            for (int i = 0; i < kJoin; i++) {
                const int s = min(s0 + i * groups + grp, a.nsplit - 1);
                v[i] = *reinterpret_cast<const float4*>(a.part_o + (s * a.rows + row) * a.Dv + col);
            }
        };
        // Few rows: on their way while the weights are worked out (9.5 -> 9.0 us for one token
        // over 1500 keys).  Many: only what weighs something is read.
        const bool ahead = a.rows <= 4096;
        if (ahead) read(0);
        const float m = wave_allreduce(fmaxf(ml0.x, ml1.x), [](float x, float y) { return fmaxf(x, y); });
        auto weight = [&](float2 ml) {         // 0 for a split that saw no key
            return ml.y == 0.0f ? 0.0f : ml.y * (ml.x == m ? 1.0f : __builtin_amdgcn_exp2f((ml.x - m) * kLog2e));
        };
        const float w0 = weight(ml0), w1 = weight(ml1);
        const float total = wave_allreduce(w0 + w1, [](float x, float y) { return x + y; });
        // divided before the sum, which then cannot leave the range of its terms
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        float r[4] = {};
        for (int s0 = 0; s0 < a.nsplit; s0 += kJoin * groups) {
            if (ahead && s0) read(s0);
            float f[kJoin];
#pragma unroll
            for (int i = 0; i < kJoin; i++) {
                const int s = s0 + i * groups + grp;
                const float wa = __shfl(w0, s & 63), wb = __shfl(w1, s & 63);
                f[i] = s < a.nsplit && grp < groups ? (s < 64 ? wa : wb) * inv : 0.0f;
                if (!ahead && f[i] != 0.0f) v[i] = *reinterpret_cast<const float4*>(a.part_o + (s * a.rows + row) * a.Dv + col);
            }
#pragma unroll
            for (int i = 0; i < kJoin; i++) {
                if (f[i] == 0.0f) continue;    // weighs nothing: it may have stored nothing
                r[0] = __builtin_fmaf(f[i], v[i].x, r[0]);
                r[1] = __builtin_fmaf(f[i], v[i].y, r[1]);
                r[2] = __builtin_fmaf(f[i], v[i].z, r[2]);
                r[3] = __builtin_fmaf(f[i], v[i].w, r[3]);
            }
        }
        for (int g = 1; g < groups; g++) {     // the groups' parts, in order
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float o = __shfl(r[e], (lane + g * quads) & 63);
                if (grp == 0) r[e] += o;
            }
        }
        if (grp == 0) {
            if constexpr (DT == kF32) *reinterpret_cast<float4*>((float*)a.y + yo + col) = make_float4(r[0], r[1], r[2], r[3]);
            else *reinterpret_cast<uint2*>((uint16_t*)a.y + yo + col) = __builtin_bit_cast(uint2, round16<DT, 4>(r));
        }
    }
}

// Many rows, and no more splits than the L lanes of a row: 64 / L rows per wave, a lane having
// one split's weight and four columns of the sum.  (22560 rows of 64 values, six splits: 7.2 us
// at 2.7 TB/s, with a wave per row 13.5, both bound by the latency of two loads in a row;
// 9456 rows, five splits: 5.0 and 7.4.)
template <int DT, bool PAGED, int L> __global__ __launch_bounds__(256) void k_attn_join_rows(AttnArgs a) {
    const int lane = (int)threadIdx.x & (L - 1), col = lane * 4;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + (int)threadIdx.x / L;
    bool there = row < a.rows;
    int64_t yo = 0;
    if (there) {
        const int64_t token = row / a.Hq;
        const int head = (int)(row - token * a.Hq);
        if constexpr (PAGED) {
            there = token >= a.qstart[0] && token < a.qstart[a.B];            // not behind the last sequence
            yo = token * a.yt + head * a.yh;
        } else {
            const int64_t b = token / a.Sq;
            yo = b * a.yb + (token - b * a.Sq) * a.yt + head * a.yh;
        }
    }
    const float2 ml = there && lane < a.nsplit ? a.part_ml[lane * a.rows + row] : make_float2(-INFINITY, 0.0f);
    float m = ml.x;
#pragma unroll
    for (int o = 1; o < L; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
    const float w = ml.y == 0.0f ? 0.0f : ml.y * (ml.x == m ? 1.0f : __builtin_amdgcn_exp2f((ml.x - m) * kLog2e));
    float total = w;
#pragma unroll
    for (int o = 1; o < L; o *= 2) total += __shfl_xor(total, o);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const float* at = a.part_o + row * a.Dv + col;
    float r[4] = {};
    for (int s0 = 0; s0 < a.nsplit; s0 += kJoin) {
        float f[kJoin];
        float4 v[kJoin];
#pragma unroll
        for (int i = 0; i < kJoin; i++) {
            const int s = s0 + i;
            f[i] = __shfl(w, s & (L - 1), L) * inv;
            if (s >= a.nsplit || col >= a.Dv) f[i] = 0.0f;
            if (f[i] != 0.0f) v[i] = *reinterpret_cast<const float4*>(at + s * a.rows * a.Dv);
        }
#pragma unroll
        for (int i = 0; i < kJoin; i++) {
            if (f[i] == 0.0f) continue;        // weighs nothing: it may have stored nothing
            r[0] = __builtin_fmaf(f[i], v[i].x, r[0]);
            r[1] = __builtin_fmaf(f[i], v[i].y, r[1]);
            r[2] = __builtin_fmaf(f[i], v[i].z, r[2]);
            r[3] = __builtin_fmaf(f[i], v[i].w, r[3]);
        }
    }
    if (!there || col >= a.Dv) return;
    if constexpr (DT == kF32) *reinterpret_cast<float4*>((float*)a.y + yo + col) = make_float4(r[0], r[1], r[2], r[3]);
    else *reinterpret_cast<uint2*>((uint16_t*)a.y + yo + col) = __builtin_bit_cast(uint2, round16<DT, 4>(r));
}

// ---- launches -------------------------------------------------------------------------
// How a call is cut into blocks is worked out on the host (attention.hip), from sizes alone.
template <int DT, int D, bool PAGED, bool MASK> void launch_tiles_of(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (p.rows == 16) hipLaunchKernelGGL((k_attn_few<DT, D, PAGED, MASK, 16>), dim3(p.blocks), dim3(64), 0, s, a);
    else if (p.rows == 32) hipLaunchKernelGGL((k_attn_few<DT, D, PAGED, MASK, 32>), dim3(p.blocks), dim3(64), 0, s, a);
    else if (p.rows == 128) hipLaunchKernelGGL((k_attn_tiles<DT, D, PAGED, MASK, 4, D * kElem<DT> <= 256 ? 64 : 32>), dim3(p.blocks), dim3(256), 0, s, a);
    else if constexpr (kElem<DT> == 2 && D <= 128) hipLaunchKernelGGL((k_attn_tiles<DT, D, PAGED, MASK, 8, kKeys256>), dim3(p.blocks), dim3(512), 0, s, a);
}
template <int DT, int D> void launch_tiles_d(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (p.keys == kPaged) launch_tiles_of<DT, D, true, false>(a, p, s);
    else if (a.mask) launch_tiles_of<DT, D, false, true>(a, p, s);
    else launch_tiles_of<DT, D, false, false>(a, p, s);
}
template <int DT> void launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    const bool paged = p.keys != kDense;
    if (!p.d) {
        const unsigned grid = grid_for((size_t)a.rows, 4, 1u << 20);
        if (p.keys == kPrefixed) hipLaunchKernelGGL((k_prefix_rows<DT>), dim3(grid), dim3(256), 0, s, a, a.rows);
        else if (paged) hipLaunchKernelGGL((k_attn_rows<DT, true>), dim3(grid), dim3(256), 0, s, a, a.rows);
        else hipLaunchKernelGGL((k_attn_rows<DT, false>), dim3(grid), dim3(256), 0, s, a, a.rows);
        return;
    }
    if (!p.blocks) {}
    else if (p.d == 64) launch_tiles_d<DT, 64>(a, p, s);
    else if (p.d == 128) launch_tiles_d<DT, 128>(a, p, s);
    else launch_tiles_d<DT, 256>(a, p, s);
    if (p.join && a.nsplit > 1) {
        const int lanes = a.Dv <= 64 ? 16 : a.Dv <= 128 ? 32 : 64;
        if (a.rows > 4096 && a.rows <= (1 << 24) && a.nsplit <= lanes) {
            const dim3 grid((unsigned)((a.rows + 256 / lanes - 1) / (256 / lanes)));
            auto join = [&](auto paged) {
                constexpr bool P = decltype(paged)::value;
                if (lanes == 16) hipLaunchKernelGGL((k_attn_join_rows<DT, P, 16>), grid, dim3(256), 0, s, a);
                else if (lanes == 32) hipLaunchKernelGGL((k_attn_join_rows<DT, P, 32>), grid, dim3(256), 0, s, a);
                else hipLaunchKernelGGL((k_attn_join_rows<DT, P, 64>), grid, dim3(256), 0, s, a);
            };
            if (paged) join(std::true_type());
            else join(std::false_type());
            return;
        }
        const unsigned grid = grid_for((size_t)a.rows, 4, 1u << 20);
        if (paged) hipLaunchKernelGGL((k_attn_join<DT, true>), dim3(grid), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_attn_join<DT, false>), dim3(grid), dim3(256), 0, s, a);
    }
}

// Both parts of a call behind a prefix (and not their join), in one launch where there is one for the
// shapes of their blocks.
template <int DT, int D> void launch_prefix_d(const AttnArgs& pre, const AttnPlan& p0, const AttnArgs& own, const AttnPlan& p1, hipStream_t s) {
    const unsigned n = p0.blocks + p1.blocks;
    if constexpr (D * kElem<DT> <= 256) {
        if (p0.rows <= 32 && p0.rows == p1.rows) {
            if (p0.rows == 16) hipLaunchKernelGGL((k_prefix_few<DT, D, 16>), dim3(n), dim3(64), 0, s, pre, own, p0.blocks);
            else hipLaunchKernelGGL((k_prefix_few<DT, D, 32>), dim3(n), dim3(64), 0, s, pre, own, p0.blocks);
            return;
        }
        if (p0.rows == 128) {
            const unsigned some = p0.blocks + (p1.blocks + 3) / 4;
            if (p1.rows == 128) hipLaunchKernelGGL((k_prefix_tiles<DT, D>), dim3(n), dim3(256), 0, s, pre, own, p0.blocks);
            else if (p1.rows == 16) hipLaunchKernelGGL((k_prefix_both<DT, D, 16>), dim3(some), dim3(256), 0, s, pre, own, p0.blocks, p1.blocks);
            else hipLaunchKernelGGL((k_prefix_both<DT, D, 32>), dim3(some), dim3(256), 0, s, pre, own, p0.blocks, p1.blocks);
            return;
        }
    }
    launch_tiles_of<DT, D, true, false>(pre, p0, s);
    launch_tiles_of<DT, D, true, false>(own, p1, s);
}
template <int DT> void launch_prefix(const AttnArgs& pre, const AttnPlan& p0, const AttnArgs& own, const AttnPlan& p1, hipStream_t s) {
    if (p0.d == 64) launch_prefix_d<DT, 64>(pre, p0, own, p1, s);
    else if (p0.d == 128) launch_prefix_d<DT, 128>(pre, p0, own, p1, s);
    else launch_prefix_d<DT, 256>(pre, p0, own, p1, s);
}

}  // namespace
}  // namespace tohip
