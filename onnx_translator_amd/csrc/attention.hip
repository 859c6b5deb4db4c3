// attention.hip — attention_forward (dense keys and values, masks, lengths),
// cache_attention_forward (new tokens over a paged cache) and prefix_cache_attention_forward
// (the same behind a shared prefix): argument checks and launches.
// The kernels are in attention_kernels.h.
#include "attention.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>

namespace tohip {
namespace {

bool float_type(const Tensor* t) {
    return (int)t->dtype == kF16 || (int)t->dtype == kBF16 || (int)t->dtype == kF32;
}
bool index_type(const Tensor* t) { return (int)t->dtype == kI32 || (int)t->dtype == kI64; }

bool good_scale(float s, const char* name) {
    if (std::isfinite(s) && s >= 0.0f) return true;
    set_error("%s: scale must be positive (0: 1 / sqrt of the head size), got %g", name, (double)s);
    return false;
}

constexpr int64_t kMaxKeys = 0x7FFFFFFF - 4096;      // key numbers past the last tile stay in 31 bits

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Y and Workspace share no memory with an input or with each other.
bool apart(std::initializer_list<const Tensor*> inputs, const Tensor* Y, const Tensor* Workspace, const char* name) {
    for (const Tensor* t : inputs) {
        if (overlaps(t, Y)) { set_error("%s: Y overlaps an input", name); return false; }
        if (overlaps(t, Workspace)) { set_error("%s: Workspace overlaps an input", name); return false; }
    }
    if (overlaps(Y, Workspace)) { set_error("%s: Workspace overlaps Y", name); return false; }
    return true;
}

bool good_workspace(const Tensor* ws, const char* name) {
    if (!ws || (tensor_sane(ws, name) && (!ws->size || is_dev(classify(ws->data))))) return true;
    if (!*tensor_ops_hip_last_error()) set_error("%s: Workspace must be a device tensor", name);
    return false;
}

// What the calls over a paged cache have in common.
bool cache_args(AttnArgs& a, const Tensor* Q, const Tensor* KCache, const Tensor* VCache, const Tensor* Pages,
                const Tensor* QStart, const Tensor* KVLen, const Tensor* Y, float scale, const char* name) {
    const Tensor* all[] = {Q, KCache, VCache, Pages, QStart, KVLen, Y};
    for (const Tensor* t : all) {
        if (!tensor_sane(t, name)) return false;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return false; }
    }
    if (!float_type(Q) || Q->dtype != KCache->dtype || Q->dtype != VCache->dtype || Q->dtype != Y->dtype) {
        set_error("%s: Q, the caches and Y must have one type: float16, bfloat16 or float32", name);
        return false;
    }
    if (Q->ndim != 3 || KCache->ndim != 4 || VCache->ndim != 4 || Y->ndim != 3) {
        set_error("%s: Q and Y must be [tokens, heads, size], the caches [pages, heads, page size, size]", name);
        return false;
    }
    a.T = Q->shape[0];
    a.Hq = Q->shape[1];
    a.Dk = Q->shape[2];
    a.npages = KCache->shape[0];
    a.Hkv = KCache->shape[1];
    a.ps = KCache->shape[2];
    a.Dv = VCache->shape[3];
    if (a.npages < 1 || a.ps < 1 || a.Dk < 1 || a.Dv < 1 || KCache->shape[3] != a.Dk || VCache->shape[0] != a.npages ||
        VCache->shape[1] != a.Hkv || VCache->shape[2] != a.ps) {
        set_error("%s: the shapes of Q and the caches do not belong together", name);
        return false;
    }
    if (a.Hq < 1 || a.Hkv < 1 || a.Hq % a.Hkv) {
        set_error("%s: the query heads must be a multiple of the key heads, got %d and %d", name, a.Hq, a.Hkv);
        return false;
    }
    if (Y->shape[0] != a.T || Y->shape[1] != a.Hq || Y->shape[2] != a.Dv) {
        set_error("%s: Y must have Q's shape with the values' head size", name);
        return false;
    }
    if (!index_type(Pages) || !index_type(QStart) || !index_type(KVLen) || Pages->ndim != 2 || QStart->ndim != 1 ||
        KVLen->ndim != 1 || KVLen->shape[0] != Pages->shape[0] || QStart->shape[0] != Pages->shape[0] + 1) {
        set_error("%s: Pages must be [sequences, pages], KVLen [sequences] and QStart [sequences + 1], int32 or int64", name);
        return false;
    }
    if (!good_scale(scale, name)) return false;
    a.B = Pages->shape[0];
    a.max_pages = Pages->shape[1];
    if ((int64_t)a.max_pages * a.ps > kMaxKeys) {
        set_error("%s: Pages hold 2^31 keys or more per sequence", name);
        return false;
    }
    a.G = a.Hq / a.Hkv;
    a.fd_g = make_fastdiv((uint32_t)a.G);
    a.fd_ps = make_fastdiv((uint32_t)a.ps);
    a.scale = scale != 0.0f ? scale : (float)(1.0 / std::sqrt((double)a.Dk));
    a.causal = 1;
    a.qh = a.Dk;
    a.qt = (int64_t)a.Hq * a.Dk;
    a.yh = a.Dv;
    a.yt = (int64_t)a.Hq * a.Dv;
    a.kt = a.Dk;
    a.kh = (int64_t)a.ps * a.Dk;
    a.kb = a.kh * a.Hkv;
    a.vt = a.Dv;
    a.vh = (int64_t)a.ps * a.Dv;
    a.vb = a.vh * a.Hkv;
    a.q = Q->data;
    a.k = KCache->data;
    a.v = VCache->data;
    a.y = Y->data;
    a.pages = {Pages->data, (int)Pages->dtype == kI64};
    a.qstart = {QStart->data, (int)QStart->dtype == kI64};
    a.qend = (const char*)QStart->data + dt_bytes((int)QStart->dtype);
    a.len = {KVLen->data, (int)KVLen->dtype == kI64};
    return true;
}

// The blocks that a call's rows make.
struct AttnBlocks {
    int64_t units, tiles;              // blocks of one split; row tiles of a batch (dense) or in all (paged)
    int resident;                      // blocks on the GPU at once
};

// Whether the matrix kernels take the call; its block shape in p.  rows: that the caller wants of a
// block (0: by the call's own).
bool attention_blocks(const AttnArgs& a, int es, bool paged, AttnPlan& p, AttnBlocks& k, int rows = 0) {
    const int vec = 16 / es, dm = a.Dk > a.Dv ? a.Dk : a.Dv;
    const int64_t per = paged ? (int64_t)a.T : (int64_t)a.Sq;      // tokens of a sequence at most
    if (!(dm <= 256 && a.Dk % vec == 0 && a.Dv % vec == 0 && per * a.G < 0x7FFFFF00 && a.kt * es < (1 << 26) &&
          a.vt * es < (1 << 26) && aligned(a.q) && aligned(a.k) && aligned(a.v) && aligned(a.y)))
        return false;
    p.d = dm <= 64 ? 64 : dm <= 128 ? 128 : 256;
    const int64_t mean = paged ? ((int64_t)a.T * a.G + a.B - 1) / a.B : per * a.G;      // rows of a sequence
    p.rows = rows ? rows : mean <= 16 ? 16 : mean <= 32 ? 32 : 128;
    auto units_of = [&](int rows) {
        const int64_t t = paged ? (int64_t)a.T * a.G / rows + a.B : (per * a.G + rows - 1) / rows;
        return t * (paged ? 1 : a.B) * a.Hkv;
    };
    // 256 rows per block where such blocks fill the GPU twice over (one fits a CU): K and V
    // pass through LDS half as often (1024 blocks of 128 rows over 8192 keys 589 us, 512 of
    // 256 538; of 64 values per head 120 and 100.  256 blocks over 300 .. 1500 keys: 35.6,
    // twice as many of 128 rows 33.7).  Not where a tile of their keys may lie on more pages
    // than a wave holds numbers of (pages of one key; tiles begin at multiples of 32).
    if (!rows && p.rows == 128 && p.d * es <= 256 && es == 2 && (!paged || kKeys256 <= kTablePages * (int64_t)a.ps) &&
        units_of(256) >= 2 * num_cus())
        p.rows = 256;
    k.units = units_of(p.rows);
    k.tiles = k.units / ((paged ? 1 : a.B) * (int64_t)a.Hkv);
    const int bn = p.rows == 128 && p.d * es <= 256 ? 64 : 32;
    const int lds = 4 * bn * p.d * es;
    // blocks on a CU at once (by registers: three of four waves for 64 values of 16 bits)
    const int most = p.rows == 128 ? (p.d * es <= 128 && !a.mask ? 3 : 2) : 8;
    k.resident = num_cus() * (p.rows == 256 ? 1 : std::min(160 * 1024 / lds, most));
    return true;
}

// Keys per split: four blocks for every place on the GPU, as lengths differ, and two tiles
// at least (64 tokens over 130 .. 8192 keys: 219 us with four, 231 with sixteen, 356 with
// two; one token over 1025: 12.4 us with two tiles, 13.2 with one, 14.0 with four, 18.2
// with eight; 96 blocks of 577 f32 keys: 39 with 128 keys, 45 with 64, 57 with 256).
// Prompts are split only where there are fewer blocks than two per CU (12 sequences of
// 2 .. 304 tokens, 376 blocks: 54 us with twelve per CU, 56 with eight, 69 with four, 78
// unsplit; 512 blocks over 300 .. 1500 keys: 33.7 unsplit, 42 in two; 1024 blocks of
// 128 rows over 8192: 589 and 634).
int64_t attention_share(const AttnPlan& p, const AttnBlocks& k, int64_t kv, int splits) {
    int64_t share = std::max<int64_t>({k.units * kv / ((int64_t)k.resident * 4), p.rows >= 128 ? 128 : 64,
                                       (kv + splits - 1) / splits});
    if (p.rows >= 128 && k.units >= std::min(k.resident, 2 * num_cus())) share = kv;
    return (share + 31) / 32 * 32;
}

// Whether the blocks of a launch stay within the runtime's work-items.
bool launchable(const AttnPlan& p, const AttnBlocks& k, int64_t split) {
    const int threads = p.rows >= 128 ? 2 * p.rows : 64;
    return k.tiles <= 0x7FFFFFFF && k.units * split * threads < (int64_t(1) << 32);
}

void launch(const AttnArgs& a, const AttnPlan& p, int dt) {
    (dt == kF16 ? launch_attention_f16 : dt == kBF16 ? launch_attention_bf16 : launch_attention_f32)(a, p, stream());
}

// Cuts the call into blocks and launches it.  kv: the most keys that a row may see, as far
// as the host knows.
void run_attention(AttnArgs& a, int dt, bool paged, int64_t kv, const Tensor* ws, const char* name) {
    a.rows = (paged ? (int64_t)a.T : (int64_t)a.B * a.Sq) * a.Hq;
    a.nsplit = 1;
    AttnPlan p = {paged ? kPaged : kDense, 0, 0, 0, true};
    AttnBlocks k;
    void* part = nullptr;
    if (attention_blocks(a, dt == kF32 ? 4 : 2, paged, p, k)) {
        int64_t share = attention_share(p, k, kv, kMaxSplits);
        int64_t split = kv > share ? (kv + share - 1) / share : 1;
        const int64_t each = a.rows * (a.Dv * 4 + 8);
        if (split > 1 && ws) {
            split = std::min<int64_t>(split, (int64_t)tensor_bytes(ws) / each);
            share = split ? ((kv + split - 1) / split + 31) / 32 * 32 : kv;
            part = ws->data;
            if (!aligned(part)) split = 1;
        } else if (split > 1) {
            part = pool_alloc((size_t)(split * each), true);
            if (!part) split = 1;
        }
        if (split > 1) {
            a.nsplit = (int)split;
            a.share = (int)share;
            a.parts = true;
            a.part_o = (float*)part;
            a.part_ml = (float2*)(a.part_o + split * a.rows * a.Dv);
        }
        if (!launchable(p, k, a.nsplit)) {
            p.d = 0;                                   // past the runtime's work-items per launch
            a.nsplit = 1;
        }
        a.tiles = (int)k.tiles;
        p.blocks = (unsigned)(k.units * a.nsplit);
    }
    launch(a, p, dt);
    check_launch(name);
    if (part && !ws) pool_free(part);
}

// A batch behind a shared prefix: the prefix's keys as those of one long sequence whose new
// tokens are all of the batch's (so a tile of rows is filled by many sequences, and the keys
// are read once per tile and not once per sequence), each sequence's own keys as ever, both as
// partial results, and one join.  own_kv, prefix_kv: the most keys, as far as the host knows.
void run_prefixed(AttnArgs& own, int dt, int64_t own_kv, int64_t prefix_kv, const Tensor* ws, const char* name) {
    const int es = dt == kF32 ? 4 : 2;
    own.rows = (int64_t)own.T * own.Hq;
    own.nsplit = 1;
    AttnArgs pre = own;
    pre.qend = (const char*)own.qstart.p + (size_t)own.B * (own.qstart.is64 ? 8 : 4);
    pre.B = 1;
    pre.pages = own.prefix;
    pre.len = own.plen;
    pre.max_pages = own.prefix_pages;
    pre.causal = 0;
    AttnPlan p0 = {kPaged, 0, 0, 0, false}, p1 = p0;
    AttnBlocks k0, k1;
    if (attention_blocks(pre, es, true, p0, k0) && attention_blocks(own, es, true, p1, k1)) {
        const int64_t rows = (int64_t)own.T * own.G;           // of a key head
        const int cus = num_cus();
        auto tiles_of = [&](int n) { return (rows + n - 1) / n * own.Hkv; };
        // Time on the whole GPU of the prefix's products (64 keys of a block of 128 rows: 1.7 us with
        // two blocks on a CU, at 128 values of 16 bits per head; float32 products take about seven times
        // as long, which is left out: longer blocks than their prefix would need) and of the own
        // keys' bytes, in us: lengths differ, so about half of the longest.
        const double step = 1.7 * p0.d / 128, pre_us = (double)tiles_of(128) * (double)prefix_kv / 64 * step / (2 * cus);
        const double own_us = 0.5 * own.B * own.Hkv * (double)own_kv * (own.Dk + own.Dv) * es / 4.5e6;
        // (three tiles at least: 4 tokens behind 2000 keys 14.9 us, 15.4 with two, 15.9 with four; 16
        // behind 4097 in float32 23.5, 27.4 and 22.7)
        int64_t share0 = std::max<int64_t>(attention_share(p0, k0, prefix_kv, kMaxSplits - 32), 96);
        if (p0.rows == 32 && p1.rows == 16) attention_blocks(own, es, true, p1, k1, 32);      // (one launch for both)
        int64_t share1 = attention_share(p1, k1, own_kv, 32);
        if (p0.rows >= 128) {
            p0.rows = 0;
            if (es == 2 && p0.d * es <= 256 && kKeys256 <= kTablePages * (int64_t)own.ps && pre_us > std::max(2 * own_us, 100.0)) {
                // Products are all there is: blocks of 256 rows, one to a CU, all of one length, in as
                // many splits as fill the last round of them best, and a launch for the own keys (2048
                // tokens of 32 heads behind 16384 keys: 591 us, 647 by 128 rows and one launch; 608
                // tokens of 24 behind 2501: 57 and 44).
                double best = 0.7;
                for (int n = 1; n <= 8; n++) {
                    const int64_t blocks = tiles_of(256) * n;
                    const double full = (double)blocks / (double)((blocks + cus - 1) / cus * cus) - 0.02 * n;
                    if (full <= best || prefix_kv < 512 * n) continue;
                    best = full;
                    p0.rows = 256;
                    share0 = (prefix_kv + n - 1) / n;
                }
            }
            if (p0.rows) {
                attention_blocks(pre, es, true, p0, k0, 256);
            } else {
                // Beside the own keys: blocks that take half of the time that both need, so that few
                // partial results are written (each split writes and reads a row of Dv float32), but
                // no more than fill the GPU where the prefix is all.  (64 tokens of 32 heads behind 8192
                // keys: 46 us with 768 keys a split, 49 with 512, 51 with 1024.)
                attention_blocks(pre, es, true, p0, k0, 128);
                if (p1.rows == 256) {
                    attention_blocks(own, es, true, p1, k1, 128);
                    share1 = attention_share(p1, k1, own_kv, 32);
                }
                share0 = (int64_t)(64 * (pre_us + own_us) / (2 * step));
                share0 = std::max<int64_t>({share0, prefix_kv * tiles_of(128) / (2 * cus), 256, (prefix_kv + 95) / 96});
            }
            share0 = (share0 + 127) / 128 * 128;
        }
        auto splits = [](int64_t kv, int64_t share) { return kv > share ? (kv + share - 1) / share : 1; };
        const int64_t each = own.rows * (own.Dv * 4 + 8);
        int64_t n0 = splits(prefix_kv, share0), n1 = splits(own_kv, share1);
        void* part = nullptr;
        if (ws && aligned(ws->data) && (int64_t)tensor_bytes(ws) / each >= 2) {
            const int64_t room = (int64_t)tensor_bytes(ws) / each;
            if (n0 + n1 > room) {                      // fewer of both
                n1 = std::max<int64_t>(1, n1 * room / (n0 + n1));
                n0 = std::max<int64_t>(1, room - n1);
                share0 = ((prefix_kv + n0 - 1) / n0 + 31) / 32 * 32;
                share1 = ((own_kv + n1 - 1) / n1 + 31) / 32 * 32;
            }
            part = ws->data;
        } else {
            ws = nullptr;
            if (stream_capturing(stream())) {
                set_error("%s: a captured call needs a workspace of two splits at least (%lld bytes, 16-byte aligned)", name,
                          (long long)(2 * each));
                return;
            }
            part = pool_alloc((size_t)((n0 + n1) * each), true);
        }
        if (part && launchable(p0, k0, n0 * 2) && launchable(p1, k1, n1 * 8)) {      // (both in one launch)
            AttnArgs all = own;
            all.nsplit = (int)(n0 + n1);
            all.parts = true;
            all.part_o = (float*)part;
            all.part_ml = (float2*)(all.part_o + all.nsplit * own.rows * own.Dv);
            auto cut = [&](AttnArgs& a, AttnPlan& p, const AttnBlocks& k, int64_t n, int64_t share, int64_t at) {
                a.nsplit = (int)n;
                a.share = (int)share;
                a.parts = true;
                a.tiles = (int)k.tiles;
                a.part_o = all.part_o + at * own.rows * own.Dv;
                a.part_ml = all.part_ml + at * own.rows;
                p.blocks = (unsigned)(k.units * n);
            };
            cut(pre, p0, k0, n0, share0, 0);
            cut(own, p1, k1, n1, share1, n0);
            (dt == kF16 ? launch_prefix_f16 : dt == kBF16 ? launch_prefix_bf16 : launch_prefix_f32)(pre, p0, own, p1, stream());
            p1.blocks = 0;
            p1.join = true;
            launch(all, p1, dt);
            check_launch(name);
            if (!ws) pool_free(part);
            return;
        }
        if (part && !ws) pool_free(part);
    }
    AttnPlan rows = {kPrefixed, 0, 0, 0, false};       // other sizes, and calls without memory
    launch(own, rows, dt);
    check_launch(name);
}

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" {

void attention_forward(const Tensor* Q, const Tensor* K, const Tensor* V, const Tensor* Mask, const Tensor* KVLen,
                       Tensor* Y, const AttentionParams* params, Tensor* Workspace) {
    const char* name = "attention_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    if (!tensor_sane(Q, name) || !tensor_sane(K, name) || !tensor_sane(V, name) || !tensor_sane(Y, name)) return;
    if (!float_type(Q) || Q->dtype != K->dtype || Q->dtype != V->dtype || Q->dtype != Y->dtype) {
        set_error("%s: Q, K, V and Y must have one type: float16, bfloat16 or float32", name);
        return;
    }
    if ((Q->ndim != 3 && Q->ndim != 4) || K->ndim != Q->ndim || V->ndim != Q->ndim || Y->ndim != Q->ndim) {
        set_error("%s: Q, K, V and Y must all be [batch, heads, length, size] or all [batch, length, heads * size]", name);
        return;
    }
    AttnArgs a = {};
    const bool packed = Q->ndim == 3;
    if (packed) {
        a.Hq = params->q_heads;
        a.Hkv = params->kv_heads;
        if (a.Hq < 1 || a.Hkv < 1 || Q->shape[2] % a.Hq || K->shape[2] % a.Hkv || V->shape[2] % a.Hkv) {
            set_error("%s: q_heads and kv_heads must divide the last dimensions of 3-D Q, K and V, got %d and %d", name,
                      a.Hq, a.Hkv);
            return;
        }
        a.Sq = Q->shape[1];
        a.Skv = K->shape[1];
        a.Dk = Q->shape[2] / a.Hq;
        a.Dv = V->shape[2] / a.Hkv;
    } else {
        a.Hq = Q->shape[1];
        a.Hkv = K->shape[1];
        a.Sq = Q->shape[2];
        a.Skv = K->shape[2];
        a.Dk = Q->shape[3];
        a.Dv = V->shape[3];
        if ((params->q_heads && params->q_heads != a.Hq) || (params->kv_heads && params->kv_heads != a.Hkv)) {
            set_error("%s: q_heads and kv_heads differ from the head dimensions of Q and K", name);
            return;
        }
    }
    a.B = Q->shape[0];
    const int kd = packed ? K->shape[2] / a.Hkv : K->shape[3];
    if (a.Hq < 1 || a.Hkv < 1 || a.Hq % a.Hkv) {
        set_error("%s: the query heads must be a multiple of the key heads, got %d and %d", name, a.Hq, a.Hkv);
        return;
    }
    if (kd != a.Dk || K->shape[0] != a.B || V->shape[0] != a.B || (packed ? V->shape[1] : V->shape[2]) != a.Skv ||
        (!packed && V->shape[1] != a.Hkv) || a.Dk < 1 || a.Dv < 1) {
        set_error("%s: the shapes of Q, K and V do not belong together", name);
        return;
    }
    if (Y->shape[0] != a.B || (packed ? Y->shape[1] != a.Sq || Y->shape[2] != a.Hq * a.Dv
                                      : Y->shape[1] != a.Hq || Y->shape[2] != a.Sq || Y->shape[3] != a.Dv)) {
        set_error("%s: Y must have Q's shape with V's head size", name);
        return;
    }
    if (a.Skv > kMaxKeys) { set_error("%s: K holds 2^31 keys or more per head", name); return; }
    if (!good_scale(params->scale, name)) return;
    a.G = a.Hq / a.Hkv;
    a.fd_g = make_fastdiv((uint32_t)a.G);
    a.scale = params->scale != 0.0f ? params->scale : (float)(1.0 / std::sqrt((double)a.Dk));
    a.causal = params->causal != 0;
    auto strides = [&](int heads, int len, int d, int64_t& sb, int64_t& sh, int64_t& st) {
        sb = (int64_t)heads * len * d;
        sh = packed ? d : (int64_t)len * d;
        st = packed ? (int64_t)heads * d : d;
    };
    strides(a.Hq, a.Sq, a.Dk, a.qb, a.qh, a.qt);
    strides(a.Hkv, a.Skv, a.Dk, a.kb, a.kh, a.kt);
    strides(a.Hkv, a.Skv, a.Dv, a.vb, a.vh, a.vt);
    strides(a.Hq, a.Sq, a.Dv, a.yb, a.yh, a.yt);
    if (Mask) {
        if (!tensor_sane(Mask, name)) return;
        a.mask_dt = (int)Mask->dtype;
        if (a.mask_dt != kU8 && a.mask_dt != kI8 && a.mask_dt != kF32 && a.mask_dt != (int)Q->dtype) {
            set_error("%s: Mask must be bool (uint8 / int8), float32 or of Q's type", name);
            return;
        }
        const int full[4] = {a.B, a.Hq, a.Sq, a.Skv};
        int64_t st[4] = {}, run = 1;
        bool ok = Mask->ndim >= 1 && Mask->ndim <= 4;
        for (int d = 3; ok && d >= 0; d--) {
            const int md = Mask->ndim - 4 + d, ext = md >= 0 ? Mask->shape[md] : 1;
            if (ext != full[d] && ext != 1) ok = false;
            st[d] = ext == 1 ? 0 : run;
            run *= ext;
        }
        if (!ok) { set_error("%s: Mask does not broadcast to [batch, heads, queries, keys]", name); return; }
        a.mb = st[0];
        a.mh = st[1];
        a.mq = st[2];
        a.mk = (int)st[3];
    }
    if (KVLen) {
        if (!tensor_sane(KVLen, name)) return;
        if (!index_type(KVLen) || KVLen->ndim != 1 || KVLen->shape[0] != a.B) {
            set_error("%s: KVLen must be int32 or int64 [batch]", name);
            return;
        }
    }
    if (!good_workspace(Workspace, name)) return;
    if (!apart({Q, K, V, Mask, KVLen}, Y, Workspace, name)) return;
    if (!ensure_device()) return;
    if (!Y->size) return;
    DeviceScope scope;
    Staging st;
    a.q = st.in(Q);
    a.k = st.in(K);
    a.v = st.in(V);
    a.mask = Mask && Mask->size ? st.in(Mask) : nullptr;
    a.len.p = KVLen ? st.in(KVLen) : nullptr;
    a.len.is64 = KVLen && (int)KVLen->dtype == kI64;
    a.y = st.out(Y, tensor_bytes(Y));
    if (*tensor_ops_hip_last_error()) return;
    run_attention(a, (int)Q->dtype, false, a.Skv, Workspace, name);
    st.finish();
}

void cache_attention_forward(const Tensor* Q, const Tensor* KCache, const Tensor* VCache, const Tensor* Pages,
                             const Tensor* QStart, const Tensor* KVLen, Tensor* Y, const CacheAttentionParams* params,
                             Tensor* Workspace) {
    const char* name = "cache_attention_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    AttnArgs a = {};
    if (!cache_args(a, Q, KCache, VCache, Pages, QStart, KVLen, Y, params->scale, name)) return;
    if (params->window < 0 || params->max_kv < 0) { set_error("%s: window and max_kv must not be negative", name); return; }
    if (!good_workspace(Workspace, name)) return;
    if (!apart({Q, KCache, VCache, Pages, QStart, KVLen}, Y, Workspace, name)) return;
    if (!ensure_device()) return;
    if (!Y->size || !a.B) return;
    const int64_t cap = (int64_t)a.max_pages * a.ps;
    a.window = params->window < cap ? params->window : 0;     // (one that long closes nothing)
    DeviceScope scope;
    run_attention(a, (int)Q->dtype, true, params->max_kv ? std::min<int64_t>(params->max_kv, cap) : cap, Workspace, name);
}

void prefix_cache_attention_forward(const Tensor* Q, const Tensor* KCache, const Tensor* VCache,
                                    const Tensor* PrefixPages, const Tensor* PrefixLen, const Tensor* Pages,
                                    const Tensor* QStart, const Tensor* KVLen, Tensor* Y,
                                    const PrefixAttentionParams* params, Tensor* Workspace) {
    const char* name = "prefix_cache_attention_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    AttnArgs a = {};
    if (!cache_args(a, Q, KCache, VCache, Pages, QStart, KVLen, Y, params->scale, name)) return;
    for (const Tensor* t : {PrefixPages, PrefixLen}) {
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
    }
    if (!index_type(PrefixPages) || !index_type(PrefixLen) || PrefixPages->ndim != 1 || PrefixLen->size != 1) {
        set_error("%s: PrefixPages must be [pages] and PrefixLen one number, int32 or int64", name);
        return;
    }
    if (params->max_prefix < 0 || params->max_kv < 0) { set_error("%s: max_prefix and max_kv must not be negative", name); return; }
    a.prefix_pages = PrefixPages->shape[0];
    const int64_t cap = (int64_t)a.max_pages * a.ps, prefix_cap = (int64_t)a.prefix_pages * a.ps;
    if (prefix_cap > kMaxKeys || cap + prefix_cap > kMaxKeys) {
        set_error("%s: PrefixPages and Pages hold 2^31 keys or more per sequence", name);
        return;
    }
    if (!good_workspace(Workspace, name)) return;
    if (!apart({Q, KCache, VCache, PrefixPages, PrefixLen, Pages, QStart, KVLen}, Y, Workspace, name)) return;
    if (!ensure_device()) return;
    if (!Y->size || !a.B) return;
    a.prefix = {PrefixPages->data, (int)PrefixPages->dtype == kI64};
    a.plen = {PrefixLen->data, (int)PrefixLen->dtype == kI64};
    DeviceScope scope;
    auto known = [](int most, int64_t cap) { return most ? std::min<int64_t>(most, cap) : cap; };
    run_prefixed(a, (int)Q->dtype, known(params->max_kv, cap), known(params->max_prefix, prefix_cap), Workspace, name);
}

}  // extern "C"
