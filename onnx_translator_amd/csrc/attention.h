// attention.h — arguments and key addressing shared by the attention kernels.
//
// Both operators are the same sum over different memory:
//   y = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j + bias_j - max),
// over the keys lo <= j < hi that a query row sees.  attention_forward's keys lie
// at fixed strides; cache_attention_forward's in pages named by a table.
//
// A row of work is one query head of one token.  The query heads that share a key
// head (a group of G) are taken together, row r = token * G + head in group, so a
// tile of rows reads its keys once for all of them.
#pragma once

#include "runtime.h"

namespace tohip {

// An int32 or int64 vector in device memory (lengths, starts, page numbers).
struct IndexVec {
    const void* p;
    int is64;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
    }
};

struct AttnArgs {
    const void *q, *k, *v, *mask;
    void* y;
    // element strides: batch (dense) or page (paged), head, token
    int64_t qb, qh, qt, kb, kh, kt, vb, vh, vt, yb, yh, yt;
    int64_t mb, mh, mq;            // mask strides: batch, query head, query (0: broadcast)
    int mk;                        // mask stride of a key (0 or 1)
    int mask_dt;                   // kU8 / kI8: 0 closes a key; else added to the score
    IndexVec len;                  // keys in use per batch (dense: p may be null) or sequence
    IndexVec pages, qstart;        // paged only
    int B, Hq, Hkv, G, Sq, Skv, Dk, Dv;
    int T;                         // paged: tokens of Q
    int ps, max_pages, npages;     // page size, pages per sequence, pages of the cache
    FastDiv fd_g, fd_ps;
    float scale;
    int causal, window;
    // tiles: rows of tiles per batch (dense) or in all (paged), and the key splits of each
    int tiles, nsplit, share;      // share: keys of a split
    float* part_o;                 // [nsplit][rows][Dv]: normalised results of a split
    float2* part_ml;               // [nsplit][rows]: (maximum of the scores, sum against it)
    int64_t rows;                  // rows of Y: tokens x query heads
};

// A sequence's part of a call: n new tokens, len keys, token i at position first + i.
struct AttnSeq {
    int b, n, len, first;
    int64_t tok0;                  // paged: its first row of Q
};

// Sequence b of a paged call, from its first row of Q and the next one's.  Starts and lengths
// come from the device: whatever they hold, no token outside Q and no key outside the table's
// capacity is touched.
__device__ __forceinline__ AttnSeq attn_seq_at(const AttnArgs& a, int b, int64_t t0, int64_t t1) {
    const int64_t c0 = t0 < 0 ? 0 : t0 > a.T ? a.T : t0, c1 = t1 < c0 ? c0 : t1 > a.T ? a.T : t1;
    const int64_t cap = (int64_t)a.max_pages * a.ps, l = a.len[b];
    AttnSeq s;
    s.b = b;
    s.tok0 = c0;
    s.n = (int)(c1 - c0);
    s.len = (int)(l < 0 ? 0 : l > cap ? cap : l);
    s.first = s.len - s.n;
    return s;
}
template <bool PAGED> __device__ __forceinline__ AttnSeq attn_seq(const AttnArgs& a, int b) {
    if constexpr (PAGED) {
        return attn_seq_at(a, b, a.qstart[b], a.qstart[b + 1]);
    } else {
        AttnSeq s;
        s.b = b;
        s.tok0 = 0;
        s.n = a.Sq;
        s.len = a.Skv;
        if (a.len.p) {
            const int64_t l = a.len[b];
            s.len = (int)(l < 0 ? 0 : l > a.Skv ? a.Skv : l);
        }
        s.first = 0;
        return s;
    }
}

// Keys [lo, hi) that token i of a sequence sees before any mask tensor.
__device__ __forceinline__ int attn_hi(const AttnArgs& a, const AttnSeq& s, int i) {
    const int p = s.first + i + 1;
    return a.causal && p < s.len ? p : s.len;
}
__device__ __forceinline__ int attn_lo(const AttnArgs& a, const AttnSeq& s, int i) {
    const int64_t p = (int64_t)s.first + i + 1 - a.window;       // (first may be as low as -n)
    return a.window && p > 0 ? (int)p : 0;
}

// The page of key j of sequence b, or -1 where the table names none of the cache's.
__device__ __forceinline__ int attn_page(const AttnArgs& a, int b, int j) {
    const int64_t p = a.pages[(int64_t)b * a.max_pages + (int)a.fd_ps.div((uint32_t)j)];
    return p >= 0 && p < a.npages ? (int)p : -1;
}

// Element offsets of key j's row of K and V from the key head's base.
struct KeyRow { int64_t k, v; };
template <bool PAGED> __device__ __forceinline__ KeyRow attn_key_row(const AttnArgs& a, int b, int page, int j) {
    if constexpr (PAGED) {
        const int o = j - (int)a.fd_ps.div((uint32_t)j) * a.ps;
        return {page * a.kb + o * a.kt, page * a.vb + o * a.vt};
    } else {
        return {b * a.kb + j * a.kt, b * a.vb + j * a.vt};
    }
}

// Whether two tensors' memory overlaps.
inline bool overlaps(const Tensor* a, const Tensor* b) {
    if (!a || !b || !a->size || !b->size) return false;
    const char *x = (const char*)a->data, *y = (const char*)b->data;
    return x < y + tensor_bytes(b) && y < x + tensor_bytes(a);
}

// Device of the caller for the length of a call: launches go to the library's device.
class DeviceScope {
  public:
    DeviceScope() {
        if (hipGetDevice(&was_) == hipSuccess && was_ != device_id()) moved_ = hipSetDevice(device_id()) == hipSuccess;
    }
    ~DeviceScope() {
        if (moved_) (void)hipSetDevice(was_);
    }

  private:
    int was_ = 0;
    bool moved_ = false;
};

constexpr int kMaxSplits = 128;    // of the keys: two per lane of a joining wave
constexpr int kTablePages = 64;    // page numbers that a wave holds, one per lane: a tile of keys names no more
constexpr int kKeys256 = 128;      // keys of a tile under blocks of 256 rows (64 or 32 under the others)

struct AttnPlan {
    bool paged;
    int d;                         // padded head size of the tile kernels; 0: a wave per row
    int rows;                      // rows of a block: 16 or 32 (one wave), 128 (four) or 256 (eight)
    unsigned blocks;
};
void launch_attention_f16(const AttnArgs& a, const AttnPlan& p, hipStream_t s);
void launch_attention_bf16(const AttnArgs& a, const AttnPlan& p, hipStream_t s);
void launch_attention_f32(const AttnArgs& a, const AttnPlan& p, hipStream_t s);

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace tohip
