// attention.hip — attention_forward (dense keys and values, masks, lengths) and
// cache_attention_forward (new tokens over a paged cache) for gfx950.
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
#include "attention.h"

#include <cmath>

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

// ---- host ---------------------------------------------------------------------------
bool float_type(const Tensor* t) {
    return (int)t->dtype == kF16 || (int)t->dtype == kBF16 || (int)t->dtype == kF32;
}
bool index_type(const Tensor* t) { return (int)t->dtype == kI32 || (int)t->dtype == kI64; }

bool good_scale(float s, const char* name) {
    if (std::isfinite(s) && s >= 0.0f) return true;
    set_error("%s: scale must be positive (0: 1 / sqrt of the head size), got %g", name, (double)s);
    return false;
}

template <bool PAGED> void launch_rows(const AttnArgs& a, int dt, const char* name) {
    const int64_t rows = (PAGED ? (int64_t)a.T : (int64_t)a.B * a.Sq) * a.Hq;
    const unsigned grid = grid_for((size_t)rows, 4, 1u << 20);
    if (dt == kF16) hipLaunchKernelGGL((k_attn_rows<kF16, PAGED>), dim3(grid), dim3(256), 0, stream(), a, rows);
    else if (dt == kBF16) hipLaunchKernelGGL((k_attn_rows<kBF16, PAGED>), dim3(grid), dim3(256), 0, stream(), a, rows);
    else hipLaunchKernelGGL((k_attn_rows<kF32, PAGED>), dim3(grid), dim3(256), 0, stream(), a, rows);
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
    if (Workspace && (!tensor_sane(Workspace, name) || (Workspace->size && !is_dev(classify(Workspace->data))))) {
        if (!*tensor_ops_hip_last_error()) set_error("%s: Workspace must be a device tensor", name);
        return;
    }
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
    launch_rows<false>(a, (int)Q->dtype, name);
    st.finish();
}

void cache_attention_forward(const Tensor* Q, const Tensor* KCache, const Tensor* VCache, const Tensor* Pages,
                             const Tensor* QStart, const Tensor* KVLen, Tensor* Y, const CacheAttentionParams* params,
                             Tensor* Workspace) {
    const char* name = "cache_attention_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    const Tensor* all[] = {Q, KCache, VCache, Pages, QStart, KVLen, Y};
    for (const Tensor* t : all) {
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
    }
    if (!float_type(Q) || Q->dtype != KCache->dtype || Q->dtype != VCache->dtype || Q->dtype != Y->dtype) {
        set_error("%s: Q, the caches and Y must have one type: float16, bfloat16 or float32", name);
        return;
    }
    if (Q->ndim != 3 || KCache->ndim != 4 || VCache->ndim != 4 || Y->ndim != 3) {
        set_error("%s: Q and Y must be [tokens, heads, size], the caches [pages, heads, page size, size]", name);
        return;
    }
    AttnArgs a = {};
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
        return;
    }
    if (a.Hq < 1 || a.Hkv < 1 || a.Hq % a.Hkv) {
        set_error("%s: the query heads must be a multiple of the key heads, got %d and %d", name, a.Hq, a.Hkv);
        return;
    }
    if (Y->shape[0] != a.T || Y->shape[1] != a.Hq || Y->shape[2] != a.Dv) {
        set_error("%s: Y must have Q's shape with the values' head size", name);
        return;
    }
    if (!index_type(Pages) || !index_type(QStart) || !index_type(KVLen) || Pages->ndim != 2 || QStart->ndim != 1 ||
        KVLen->ndim != 1 || KVLen->shape[0] != Pages->shape[0] || QStart->shape[0] != Pages->shape[0] + 1) {
        set_error("%s: Pages must be [sequences, pages], KVLen [sequences] and QStart [sequences + 1], int32 or int64", name);
        return;
    }
    if (!good_scale(params->scale, name)) return;
    if (params->window < 0 || params->max_kv < 0) { set_error("%s: window and max_kv must not be negative", name); return; }
    a.B = Pages->shape[0];
    a.max_pages = Pages->shape[1];
    if ((int64_t)a.max_pages * a.ps > 0x7FFFFFFF - 4096) {
        set_error("%s: Pages hold 2^31 keys or more per sequence", name);
        return;
    }
    if (Workspace && (!tensor_sane(Workspace, name) || (Workspace->size && !is_dev(classify(Workspace->data))))) {
        if (!*tensor_ops_hip_last_error()) set_error("%s: Workspace must be a device tensor", name);
        return;
    }
    if (!ensure_device()) return;
    if (!Y->size || !a.B) return;
    a.G = a.Hq / a.Hkv;
    a.fd_g = make_fastdiv((uint32_t)a.G);
    a.fd_ps = make_fastdiv((uint32_t)a.ps);
    a.scale = params->scale != 0.0f ? params->scale : (float)(1.0 / std::sqrt((double)a.Dk));
    a.causal = 1;
    a.window = params->window;
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
    a.len = {KVLen->data, (int)KVLen->dtype == kI64};
    DeviceScope scope;
    launch_rows<true>(a, (int)Q->dtype, name);
}

}  // extern "C"
