// attention_kernels.h — the attention kernels for gfx950, by element type (one source
// file instantiates each).
//
//   y = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j + bias_j - max_j)
//
// over the keys a query sees.  One pass over the keys: a running maximum and sum,
// the output rescaled where the maximum grows.  Scores, statistics and sums are
// held in 32 bits or more; the result is rounded once.
//
// Keys that are not seen (past the length, later than the query, outside the
// window, closed by the mask, or on a page that the cache does not have) add
// nothing, whatever K and V hold there; a row that sees none gives zeros.
#pragma once

#include <cmath>

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
// finite result, and a key that is not seen is never multiplied.
constexpr int kRowCols = 4;        // columns of V per lane and pass over the keys

// Partial result of the keys [ks, ke) for query head h of token i: the maximum (of
// scaled scores), the sum and, by store(d, value), the normalised output.
template <int DT, bool PAGED, class ST>
__device__ __forceinline__ void attn_row(const AttnArgs& a, const AttnSeq& s, int h, int i, int ks, int ke, float& m_out,
                                         float& l_out, ST store) {
    const int lane = (int)(threadIdx.x & 63), hk = (int)a.fd_g.div((uint32_t)h);
    const int lo = max(ks, attn_lo(a, s, i)), hi = min(ke, attn_hi(a, s, i));
    const int64_t qo = PAGED ? (s.tok0 + i) * a.qt + h * a.qh : s.b * a.qb + i * a.qt + h * a.qh;
    const int64_t mo = s.b * a.mb + h * a.mh + i * a.mq;
    for (int d0 = 0; d0 < a.Dv; d0 += 64 * kRowCols) {
        float m = -INFINITY;
        double l = 0.0, acc[kRowCols] = {};
        for (int j0 = lo; j0 < hi; j0 += 64) {
            const int j = j0 + lane;
            bool seen = j < hi;
            const int page = PAGED && seen ? attn_page(a, s.b, j) : 0;
            seen = seen && page >= 0;
            float t = -INFINITY;
            KeyRow row = {0, 0};
            if (seen) {
                row = attn_key_row<PAGED>(a, s.b, page, j);
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

template <int DT, bool PAGED> __global__ __launch_bounds__(256) void k_attn_rows(AttnArgs a, int64_t rows) {
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
        attn_row<DT, PAGED>(a, s, h, i, 0, s.len, m, l, [&](int d, float v) { st_code<DT>(a.y, yo + d, v); });
    }
}

// ---- tiles on the matrix cores ------------------------------------------------------
// A wave owns 32 rows (query heads of tokens) and walks over the keys 32 at a time:
//   S' = K Q'    32 keys x 32 rows: a lane holds 16 keys of one row, its other 16 are in
//                the lane 32 further on, so maximum and sum of a row are a few register
//                operations and one exchange between the halves of the wave;
//   O' += V' P'  head size x 32 rows: the rescaling factor of a row is one lane's value,
//                and P goes from the accumulators of S' straight into the operand: the
//                product sums over keys in any order, so V's rows are simply read in the
//                order in which the lanes hold their keys.
// RW waves share the keys and own different rows (prompts), or KW waves own the same rows
// and different keys (few rows, where reading the keys is the work) and join at the end.
// Key and value tiles go from memory to LDS directly (no registers), two buffers deep, in
// 16-byte chunks whose place in a row is turned by the row's number so that fragment
// reads spread over the banks.
//
// What a closed key holds does not matter as long as it is finite: its weight is zero.
// Where a result comes out infinite or NaN (a closed key's value was, or values near the
// type's largest overflowed a sum on the way), or a page of the sequence is missing, the
// row is computed again by attn_row above, which looks at open keys only.
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bfloatx8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <int DT> constexpr int kElem = DT == kF32 ? 4 : 2;

// One 16-byte chunk per lane of each operand: 8 values of 16 bits (one product), or 4 of
// 32 bits (four products, the chunk's j-th values of both wave halves in the j-th).
template <int DT> __device__ __forceinline__ floatx16 mfma_chunk(uint4 a, uint4 b, floatx16 c) {
    if constexpr (DT == kF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    } else if constexpr (DT == kBF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bfloatx8, a), __builtin_bit_cast(bfloatx8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(a.x), u2f(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(a.y), u2f(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(a.z), u2f(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(a.w), u2f(b.w), c, 0, 0, 0);
    }
}

// Eight weights as the product's operand, each rounded to the nearest 16-bit value.
template <int DT> __device__ __forceinline__ uint4 pack8(const float* p) {
    if constexpr (DT == kF16) {
        halfx8 h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (_Float16)p[i];
        return __builtin_bit_cast(uint4, h);
    } else {
        bfloatx8 h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (__bf16)p[i];
        return __builtin_bit_cast(uint4, h);
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
// All of this wave's loads have landed and its LDS reads have returned.
__device__ __forceinline__ void wait_all_loads() { __builtin_amdgcn_s_waitcnt(0x0070); }
// A value that all lanes hold, as a scalar.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Place of chunk c in row r of a tile of CH chunks per row.  Keys are read by 16 or 32 rows
// of one chunk; values by four rows of four neighbouring chunks (16 bits), or by rows r and
// r + 4 of eight (32 bits).
template <int CH> __device__ __forceinline__ int key_place(int r, int c) {
    return c ^ (CH == 8 ? (r >> 1) & 7 : r & 15);
}
template <int DT, int CH> __device__ __forceinline__ int value_place(int r, int c) {
    if constexpr (DT == kF32) return c ^ (((r >> 2) & 1) << 3);
    else return c ^ (CH == 8 ? ((r >> 1) & 1) << 2 : (r & 3) << 2);
}

// The sequence whose tiles hold slot t: the last b with floor(start_b * G / BM) + b <= t.
// (The slots of a sequence, one more than its whole tiles may need, follow from the starts
// alone, so no list of tiles has to be made.)  64 sequences are tried at a time.
template <int BM> __device__ __forceinline__ int64_t slot_base(const AttnArgs& a, int b) {
    int64_t t0 = a.qstart[b];
    t0 = t0 < 0 ? 0 : t0 > a.T ? a.T : t0;
    return t0 * a.G / BM + b;
}
template <int BM> __device__ __forceinline__ int slot_sequence(const AttnArgs& a, int64_t t) {
    int lo = 0, n = a.B;                       // the answer is in [lo, lo + n)
    const int lane = (int)(threadIdx.x & 63);
    while (n > 1) {
        const int step = (n + 63) / 64, b = lo + lane * step;
        const bool le = lane * step < n && slot_base<BM>(a, b) <= t;
        const int k = __popcll(__ballot(le));
        if (k > 1) lo += (k - 1) * step;
        n = min(step, a.B - lo);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// log2 units that a row's maximum may grow by before its sums are rescaled: weights stay
// below 2^8 (and the float16 ones, raised by 2^6 out of its subnormal range, below 2^14).
constexpr float kLazy = 8.0f;
template <int DT> constexpr float kRaise = DT == kF16 ? 6.0f : 0.0f;

template <int DT, int D, bool PAGED, bool MASK, int RW, int KW, int BN>
__global__ __launch_bounds__(64 * RW * KW, D * kElem<DT> <= 256 ? 2 : 1) void k_attn_tiles(AttnArgs a) {
    constexpr int ES = kElem<DT>, VEC = 16 / ES, CH = D / VEC, RB = D * ES, W = RW * KW;
    constexpr int BM = 32 * RW, NSUB = BN / (32 * KW), NI = BN * RB / (1024 * W), RPI = 1024 / RB;
    constexpr int NS = CH / 2;                 // chunk pairs of a head: products of S' per 32 keys
    constexpr int ND = D / 32;                 // 32-column blocks of the result
    static_assert(NSUB >= 1 && NI >= 1 && RPI >= 1, "tile");
    // distinct arrays: a read of one does not wait for the loads in flight to the other
    __shared__ __attribute__((aligned(1024))) char k0_[BN * RB], k1_[BN * RB], v0_[BN * RB], v1_[BN * RB];
    __shared__ int missing;                    // a key's page was none of the cache's
    const int t = (int)threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int lr = lane & 31, h = lane >> 5;

    // ---- this block's rows and keys
    uint32_t bid = blockIdx.x;
    const int hk = (int)(bid % (uint32_t)a.Hkv);
    bid /= (uint32_t)a.Hkv;
    const int split = (int)(bid % (uint32_t)a.nsplit);
    bid /= (uint32_t)a.nsplit;
    int b, tile;
    if constexpr (PAGED) {
        // the last slots first: the later tokens of a prompt have the most keys
        const int64_t slot = (int64_t)a.tiles - 1 - bid;
        b = slot_sequence<BM>(a, slot);
        const int64_t tl = slot - slot_base<BM>(a, b);
        tile = uniform(tl < 0 ? -1 : (int)tl);
        if (tile < 0) return;
    } else {
        const uint32_t tl = bid % (uint32_t)a.tiles;
        tile = a.tiles - 1 - (int)tl;
        b = (int)(bid / (uint32_t)a.tiles);
    }
    AttnSeq s = attn_seq<PAGED>(a, b);
    s.n = uniform(s.n);
    s.len = uniform(s.len);
    s.first = uniform(s.first);
    const int64_t nrows = (int64_t)s.n * a.G;
    const int64_t row0 = (int64_t)tile * BM;
    if (row0 >= nrows) return;
    const int rows = (int)min((int64_t)BM, nrows - row0);
    const int tok0 = (int)(row0 / a.G);                          // first and last token of the block
    const int tok1 = (int)((row0 + rows - 1) / a.G);
    // keys of the block, cut to this split's share (whole tiles)
    int klo = attn_lo(a, s, tok0), khi = attn_hi(a, s, tok1);
    if (a.nsplit > 1) {
        const int share = ((khi - klo + a.nsplit - 1) / a.nsplit + BN - 1) / BN * BN;
        const int64_t at = (int64_t)klo + (int64_t)split * share;
        khi = (int)min((int64_t)khi, at + share);
        klo = (int)min((int64_t)khi, at);
    }
    const int last = s.len - 1;

    // ---- this lane's row
    const int wrow = KW > 1 ? 0 : wave * 32;                     // the wave's first row in the block
    const int my = min(wrow + lr, rows - 1);
    const bool live = wrow + lr < rows;
    const int64_t row = row0 + my;
    const int tok = (int)(row / a.G), head = hk * a.G + (int)(row - (int64_t)tok * a.G);
    const int lo = max(klo, attn_lo(a, s, tok)), hi = min(khi, attn_hi(a, s, tok));
    // keys that some row of the wave sees, and those that all see
    const int wtok0 = (int)((row0 + min(wrow, rows - 1)) / a.G), wtok1 = (int)((row0 + min(wrow + 31, rows - 1)) / a.G);
    const int any_lo = max(klo, attn_lo(a, s, wtok0)), any_hi = min(khi, attn_hi(a, s, wtok1));
    const int all_lo = max(klo, attn_lo(a, s, wtok1)), all_hi = min(khi, attn_hi(a, s, wtok0));
    const bool wlive = wrow < rows;

    uint4 q[NS];
    {
        const int64_t qo = PAGED ? (s.tok0 + tok) * a.qt + head * a.qh : s.b * a.qb + tok * a.qt + head * a.qh;
        const uint4* qp = reinterpret_cast<const uint4*>((const char*)a.q + qo * ES);
        const int qch = a.Dk / VEC;
#pragma unroll
        for (int i = 0; i < NS; i++) {
            const int c = 2 * i + h;
            q[i] = live && c < qch ? qp[c] : uint4{0, 0, 0, 0};
        }
    }
    const int64_t mo = MASK ? s.b * a.mb + head * a.mh + tok * a.mq : 0;

    // ---- loads: instruction i of this wave fills rows (i W + wave) RPI ..
    const char* kbase = (const char*)a.k + hk * a.kh * ES;
    const char* vbase = (const char*)a.v + hk * a.vh * ES;
    const int lrow = lane / CH, lslot = lane % CH, kch = a.Dk / VEC, vch = a.Dv / VEC;
    int page[PAGED ? NI : 1];
    auto find_pages = [&](int j0) {
        if constexpr (PAGED) {
#pragma unroll
            for (int i = 0; i < NI; i++) page[i] = attn_page(a, b, min(j0 + (i * W + wave) * RPI + lrow, last));
        }
    };
    auto load = [&](char* kt, char* vt, int j0) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = (i * W + wave) * RPI + lrow, j = min(j0 + r, last);
            int pg = PAGED ? page[i] : 0;
            if (PAGED && pg < 0) {
                missing = 1;
                pg = 0;
            }
            const KeyRow at = attn_key_row<PAGED>(a, b, pg, j);
            const int kc = key_place<CH>(r, lslot), vc = value_place<DT, CH>(r, lslot);
            if (kc < kch) load_lds16(kbase + at.k * ES + kc * 16, kt + (i * W + wave) * 1024);
            if (vc < vch) load_lds16(vbase + at.v * ES + vc * 16, vt + (i * W + wave) * 1024);
        }
    };

    // ---- the sums
    floatx16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;             // the row's maximum so far; this lane's part of the sum
    const float c = MASK ? kLog2e : a.scale * kLog2e;

    auto work = [&](const char* kt, const char* vt, int j0) {
#pragma unroll
        for (int n = 0; n < NSUB; n++) {
            const int sub = KW > 1 ? (n * KW + wave) * 32 : n * 32, jb = j0 + sub;
            if (!wlive || jb >= any_hi || jb + 32 <= any_lo) continue;
            floatx16 x;
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = 0.0f;
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const uint4 kf = *reinterpret_cast<const uint4*>(kt + (sub + lr) * RB + key_place<CH>(lr, 2 * i + h) * 16);
                x = mfma_chunk<DT>(kf, q[i], x);
            }
            if constexpr (MASK) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int j = jb + 8 * (i >> 2) + 4 * h + (i & 3);
                    float bias = -INFINITY;
                    if (j >= lo && j < hi) {
                        const int64_t at = mo + (int64_t)j * a.mk;
                        if (a.mask_dt == kU8 || a.mask_dt == kI8) bias = ((const uint8_t*)a.mask)[at] ? 0.0f : -INFINITY;
                        else if (a.mask_dt == kF32) bias = ((const float*)a.mask)[at];
                        else bias = ld_f<DT>(a.mask, at);
                    }
                    x[i] = bias == -INFINITY ? -INFINITY : __builtin_fmaf(x[i], a.scale, bias);
                }
            } else if (jb < all_lo || jb + 32 > all_hi) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int j = jb + 8 * (i >> 2) + 4 * h + (i & 3);
                    x[i] = j >= lo && j < hi ? x[i] : -INFINITY;
                }
            }
            float top = x[0];
#pragma unroll
            for (int i = 1; i < 16; i++) top = fmaxf(top, x[i]);
            float ta, tb;
            permlane_pair<32>(top, ta, tb);
            top = fmaxf(ta, tb);
            if (__ballot((top - m) * c > kLazy)) {
                const float mn = fmaxf(m, top);
                const float f = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] *= f;
                m = mn;
            }
            const float base = m == -INFINITY ? 0.0f : m;
            float p[16];
            if constexpr (MASK) {
                // the difference first: a mask of the type's lowest value times log2 e would overflow
#pragma unroll
                for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i] - base, c, kRaise<DT>));
            } else {
                const float off = kRaise<DT> - base * c;
#pragma unroll
                for (int i = 0; i < 16; i++) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, off));
            }
#pragma unroll
            for (int i = 0; i < 16; i++) l += p[i];
            if constexpr (DT == kF32) {
                // weight i of both wave halves: keys 8 (i / 4) + i % 4 and 4 further on
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int r = sub + 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const float vf = *reinterpret_cast<const float*>(vt + r * RB + value_place<DT, CH>(r, d * 8 + (lr >> 2)) * 16 + (lr & 3) * 4);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf, p[i], o[d], 0, 0, 0);
                    }
                }
            } else {
                const int r4 = (lane & 15) >> 2, cc = (lane >> 4 & 1) * 2 + ((lane & 3) >> 1), in = (lane & 1) * 8;
#pragma unroll
                for (int kk = 0; kk < 2; kk++) {
                    const uint4 pf = pack8<DT>(p + 8 * kk);
                    const int r = sub + 16 * kk + 4 * h + r4;
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        const uint2 va = read_turned(vt + r * RB + value_place<DT, CH>(r, d * 4 + cc) * 16 + in);
                        const uint2 vb = read_turned(vt + (r + 8) * RB + value_place<DT, CH>(r + 8, d * 4 + cc) * 16 + in);
                        o[d] = mfma_chunk<DT>(uint4{va.x, va.y, vb.x, vb.y}, pf, o[d]);
                    }
                }
            }
        }
    };

    // ---- the walk: while tile n is worked on, tile n + 1 is on its way, and the pages of n + 2
    if (t == 0) missing = 0;
    if (kch < CH) {                            // columns past the head size: zeros that no load touches
        for (int i = t; i < BN * CH; i += 64 * W) {
            reinterpret_cast<uint4*>(k0_)[i] = uint4{0, 0, 0, 0};
            reinterpret_cast<uint4*>(k1_)[i] = uint4{0, 0, 0, 0};
        }
    }
    __syncthreads();
    const int jbeg = klo, jend = khi;
    if (jbeg < jend) {
        find_pages(jbeg);
        load(k0_, v0_, jbeg);
        find_pages(jbeg + BN);
        auto step = [&](int j0, const char* kt, const char* vt, char* kn, char* vn) {
            wait_all_loads();
            __builtin_amdgcn_s_barrier();      // every wave's part of this tile is there, and the other buffer is free
            __builtin_amdgcn_sched_barrier(0);
            if (j0 + BN < jend) {
                load(kn, vn, j0 + BN);
                find_pages(j0 + 2 * BN);
                __builtin_amdgcn_sched_barrier(0);
            }
            work(kt, vt, j0);
        };
        for (int j0 = jbeg; j0 < jend; j0 += 2 * BN) {
            step(j0, k0_, v0_, k1_, v1_);
            if (j0 + BN < jend) step(j0 + BN, k1_, v1_, k0_, v0_);
        }
    }
    __syncthreads();

    // ---- the end: join the waves' keys, divide, store
    {
        float la, lb;
        permlane_pair<32>(l, la, lb);
        l = la + lb;
    }
    float m2 = m == -INFINITY ? -INFINITY : m * c - kRaise<DT>;      // log2 units, as l is scaled
    if constexpr (KW > 1) {
        static_assert(2 * BN * RB >= KW * 32 * 8, "room for the statistics");
        float* st = reinterpret_cast<float*>(k0_);                 // [KW][32][2]
        if (h == 0) {
            st[(wave * 32 + lr) * 2] = m2;
            st[(wave * 32 + lr) * 2 + 1] = l;
        }
        __syncthreads();
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; w++) mm = fmaxf(mm, st[(w * 32 + lr) * 2]);
#pragma unroll
        for (int w = 0; w < KW; w++) {
            const float mw = st[(w * 32 + lr) * 2];
            ll += mw == -INFINITY ? st[(w * 32 + lr) * 2 + 1] : st[(w * 32 + lr) * 2 + 1] * __builtin_amdgcn_exp2f(mw - mm);
        }
        const float f = m2 == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m2 - mm);
        // one wave after another adds its part to the first one's
        float* sum = reinterpret_cast<float*>(v0_);                // [D][32], up to 32 KB
        static_assert(KW == 1 || BN * RB >= D * 32 * 4, "room for the sums");
        for (int w = 1; w < KW; w++) {
            __syncthreads();
            if (wave == w) {
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[(d * 16 + i) * 64 + lane] = o[d][i] * f;
            }
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] = (w == 1 ? o[d][i] * f : o[d][i]) + sum[(d * 16 + i) * 64 + lane];
            }
        }
        if (wave != 0) return;
        m2 = mm;
        l = ll;
    }
    if (!wlive) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t token = PAGED ? s.tok0 + tok : (int64_t)s.b * a.Sq + tok;
    const int64_t orow = token * a.Hq + head;                      // of the rows of Y
    const bool split_out = a.nsplit > 1;
    bool bad = missing != 0;
#pragma unroll
    for (int d = 0; d < ND; d++) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int col = d * 32 + 8 * g + 4 * h;
            if (col >= a.Dv) continue;
            float r[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                r[e] = l == 0.0f ? 0.0f : o[d][4 * g + e] * inv;
                bad |= !(__builtin_fabsf(r[e]) <= 3.402823466e38f);
            }
            if (!live) continue;
            if (split_out) {
                *reinterpret_cast<float4*>(a.part_o + ((int64_t)split * a.rows + orow) * a.Dv + col) = make_float4(r[0], r[1], r[2], r[3]);
            } else {
                const int64_t yo = PAGED ? token * a.yt + head * a.yh : s.b * a.yb + tok * a.yt + head * a.yh;
                if constexpr (DT == kF32) {
                    *reinterpret_cast<float4*>((float*)a.y + yo + col) = make_float4(r[0], r[1], r[2], r[3]);
                } else {
                    uint16_t e[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) e[i] = DT == kF16 ? enc_f16(r[i]) : enc_bf16(r[i]);
                    *reinterpret_cast<uint2*>((uint16_t*)a.y + yo + col) = uint2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
                }
            }
        }
    }
    if (split_out && live && h == 0) a.part_ml[(int64_t)split * a.rows + orow] = make_float2(m2, l);
    // rows to be computed again, one after the other by the whole wave
    unsigned long long again = __ballot(bad && live);
    again = (again | again >> 32) & 0xFFFFFFFFull;
    for (; again; again &= again - 1) {
        const int r = __builtin_ctzll(again);
        const int64_t rw = row0 + wrow + r;
        const int tk = (int)(rw / a.G), hd = hk * a.G + (int)(rw - (int64_t)tk * a.G);
        const int64_t tkn = PAGED ? s.tok0 + tk : (int64_t)s.b * a.Sq + tk, orw = tkn * a.Hq + hd;
        float rm = -INFINITY, rl = 0.0f;
        if (split_out) {
            float* po = a.part_o + ((int64_t)split * a.rows + orw) * a.Dv;
            attn_row<DT, PAGED>(a, s, hd, tk, klo, khi, rm, rl, [&](int d, float v) { po[d] = v; });
            if (lane == 0) a.part_ml[(int64_t)split * a.rows + orw] = make_float2(rm * kLog2e, rl);
        } else {
            const int64_t yo = PAGED ? tkn * a.yt + hd * a.yh : s.b * a.yb + tk * a.yt + hd * a.yh;
            attn_row<DT, PAGED>(a, s, hd, tk, klo, khi, rm, rl, [&](int d, float v) { st_code<DT>(a.y, yo + d, v); });
        }
    }
}

// ---- the splits of a row together -----------------------------------------------------
// y = sum_s w_s o_s / sum_s w_s, w_s = l_s 2^(m_s - max): four columns per thread.
template <int DT, bool PAGED> __global__ __launch_bounds__(256) void k_attn_join(AttnArgs a, int quads) {
    const int64_t n = a.rows * quads, step = (int64_t)gridDim.x * 256;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < n; u += step) {
        const int64_t row = u / quads;
        const int col = (int)(u - row * quads) * 4;
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
        float m = -INFINITY;
        for (int s = 0; s < a.nsplit; s++) m = fmaxf(m, a.part_ml[s * a.rows + row].x);
        auto weight = [&](float2 ml) { return ml.y * (ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m)); };
        float total = 0.0f, r[4] = {};
        for (int s = 0; s < a.nsplit; s++) {
            const float2 ml = a.part_ml[s * a.rows + row];
            if (ml.y != 0.0f) total += weight(ml);
        }
        // divided before the sum, which then cannot leave the range of its terms
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
        for (int s = 0; s < a.nsplit; s++) {
            const float2 ml = a.part_ml[s * a.rows + row];
            if (ml.y == 0.0f) continue;                      // saw no key
            const float w = weight(ml) * inv;
            if (w == 0.0f) continue;                         // weighs nothing
            const float4 v = *reinterpret_cast<const float4*>(a.part_o + (s * a.rows + row) * a.Dv + col);
            r[0] = __builtin_fmaf(w, v.x, r[0]);
            r[1] = __builtin_fmaf(w, v.y, r[1]);
            r[2] = __builtin_fmaf(w, v.z, r[2]);
            r[3] = __builtin_fmaf(w, v.w, r[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) st_code<DT>(a.y, yo + col + e, r[e]);
    }
}

// ---- launches -------------------------------------------------------------------------
// How a call is cut into blocks: worked out on the host (attention.hip) from sizes alone.
template <int DT, int D, int RW, int KW, int BN> void launch_tiles_of(const AttnArgs& a, bool paged, unsigned blocks, hipStream_t s) {
    constexpr int threads = 64 * RW * KW;
    if (paged) hipLaunchKernelGGL((k_attn_tiles<DT, D, true, false, RW, KW, BN>), dim3(blocks), dim3(threads), 0, s, a);
    else if (a.mask) hipLaunchKernelGGL((k_attn_tiles<DT, D, false, true, RW, KW, BN>), dim3(blocks), dim3(threads), 0, s, a);
    else hipLaunchKernelGGL((k_attn_tiles<DT, D, false, false, RW, KW, BN>), dim3(blocks), dim3(threads), 0, s, a);
}
template <int DT, int D> void launch_tiles_d(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    constexpr AttnTile big = attn_tile(D * kElem<DT>, false), few = attn_tile(D * kElem<DT>, true);
    if (p.few) launch_tiles_of<DT, D, few.rw, few.kw, few.bn>(a, p.paged, p.blocks, s);
    else launch_tiles_of<DT, D, big.rw, big.kw, big.bn>(a, p.paged, p.blocks, s);
}
template <int DT> void launch_attention(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
    if (!p.d) {
        const unsigned grid = grid_for((size_t)a.rows, 4, 1u << 20);
        if (p.paged) hipLaunchKernelGGL((k_attn_rows<DT, true>), dim3(grid), dim3(256), 0, s, a, a.rows);
        else hipLaunchKernelGGL((k_attn_rows<DT, false>), dim3(grid), dim3(256), 0, s, a, a.rows);
        return;
    }
    if (p.d == 64) launch_tiles_d<DT, 64>(a, p, s);
    else if (p.d == 128) launch_tiles_d<DT, 128>(a, p, s);
    else launch_tiles_d<DT, 256>(a, p, s);
    if (a.nsplit > 1) {
        const int quads = a.Dv / 4;
        const unsigned grid = grid_for((size_t)a.rows * quads, 256, 1u << 20);
        if (p.paged) hipLaunchKernelGGL((k_attn_join<DT, true>), dim3(grid), dim3(256), 0, s, a, quads);
        else hipLaunchKernelGGL((k_attn_join<DT, false>), dim3(grid), dim3(256), 0, s, a, quads);
    }
}

}  // namespace
}  // namespace tohip
