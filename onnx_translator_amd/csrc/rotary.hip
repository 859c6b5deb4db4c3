// rotary.hip — qk_norm_rotary_forward for gfx950: the packed projections of a decoder
// layer's queries, keys and values on their way to the attention.
//
// Per head of a token's queries and keys, x of D values:
//   y = x * rsqrt(mean(x^2) + epsilon) * w                       (w given)
//   (y_i, y_j) -> (y_i cos - y_j sin, y_i sin + y_j cos)         (the first R values)
// with the angles' cosines and sines from the tables' row of the token's position and
// pairs (i, i + R/2), or (2i, 2i + 1) when interleaved.  All in float32, rounded once.
// Values pass unchanged.  Keys and values go to dense tensors or into the pages of a
// cache, at the slot (page * page size + place in page) that the caller gives a token.
#include "attention.h"

#include <cmath>

namespace tohip {
namespace {

struct RotaryArgs {
    const void *x, *wq, *wk, *cos, *sin;
    void *q, *k, *v;
    IndexVec pos, slots;           // slots.p null: dense K and V
    int T, Hq, Hkv, H, D, R, rows; // H = Hq + 2 Hkv; rows of the tables
    int table_dt, weight_dt;
    int interleaved, norm_q, norm_k;
    int ps;                        // cache: page size
    int64_t slots_n;               // slots of the cache
    FastDiv fd_ps;
    float epsilon;
};

// Element offset of head g (of the keys or values) of a token in K or V, or -1: not stored.
__device__ __forceinline__ int64_t kv_offset(const RotaryArgs& a, int64_t t, int g) {
    if (!a.slots.p) return (t * a.Hkv + g) * a.D;
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.slots_n) return -1;
    const int64_t page = slot / a.ps, o = slot - page * a.ps;
    return ((page * a.Hkv + g) * a.ps + o) * a.D;
}

// ---- any head size and alignment: a wave per head -----------------------------------
template <int DT> __global__ __launch_bounds__(256) void k_rotary_any(RotaryArgs a, int64_t heads) {
    const int lane = (int)(threadIdx.x & 63);
    const int64_t step = (int64_t)gridDim.x * 4;
    for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < heads; u += step) {
        const int64_t t = u / a.H;
        const int h = (int)(u - t * a.H);
        const int kind = h < a.Hq ? 0 : h < a.Hq + a.Hkv ? 1 : 2;
        const int64_t pos = a.pos.p ? a.pos[t] : 0;
        if (pos < 0 || (a.cos && pos >= a.rows)) continue;      // a token to be left out
        const int64_t to = kind == 0 ? (t * a.Hq + h) * a.D : kv_offset(a, t, h - a.Hq - (kind == 2 ? a.Hkv : 0));
        if (to < 0) continue;
        const int64_t from = (t * a.H + h) * a.D;
        void* y = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
        if (kind == 2) {
            for (int d = lane; d < a.D; d += 64) {
                if constexpr (DT == kF32) ((uint32_t*)y)[to + d] = ((const uint32_t*)a.x)[from + d];
                else ((uint16_t*)y)[to + d] = ((const uint16_t*)a.x)[from + d];
            }
            continue;
        }
        const bool norm = kind == 0 ? a.norm_q : a.norm_k;
        const void* w = kind == 0 ? a.wq : a.wk;
        float r = 1.0f;
        if (norm) {
            float sum = 0.0f;
            for (int d = lane; d < a.D; d += 64) {
                const float v = (float)ld_d<DT>(a.x, from + d);
                sum = __builtin_fmaf(v, v, sum);
            }
            sum = wave_allreduce(sum, [](float x, float z) { return x + z; });
            r = 1.0f / __builtin_sqrtf(sum / (float)a.D + a.epsilon);
        }
        auto value = [&](int d) {
            const float v = (float)ld_d<DT>(a.x, from + d);
            return norm ? v * r * (float)ld_d_rt(a.weight_dt, w, d) : v;
        };
        const int half = a.R / 2;
        for (int i = lane; i < half; i += 64) {
            const int d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
            const float c = (float)ld_d_rt(a.table_dt, a.cos, pos * half + i), s = (float)ld_d_rt(a.table_dt, a.sin, pos * half + i);
            const float v0 = value(d0), v1 = value(d1);
            st_code<DT>(y, to + d0, v0 * c - v1 * s);
            st_code<DT>(y, to + d1, v0 * s + v1 * c);
        }
        for (int d = a.R + lane; d < a.D; d += 64) st_code<DT>(y, to + d, value(d));
    }
}

bool rotary_type(const Tensor* t) {
    return (int)t->dtype == kF16 || (int)t->dtype == kBF16 || (int)t->dtype == kF32;
}
bool index_type(const Tensor* t) { return (int)t->dtype == kI32 || (int)t->dtype == kI64; }

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" void qk_norm_rotary_forward(const Tensor* QKV, const Tensor* QWeight, const Tensor* KWeight,
                                       const Tensor* Cos, const Tensor* Sin, const Tensor* Positions,
                                       const Tensor* Slots, Tensor* Q, Tensor* K, Tensor* V,
                                       const QKNormRotaryParams* params) {
    const char* name = "qk_norm_rotary_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    const Tensor* needed[] = {QKV, Q, K, V};
    for (const Tensor* t : needed)
        if (!tensor_sane(t, name)) return;
    const Tensor* all[] = {QKV, Q, K, V, QWeight, KWeight, Cos, Sin, Positions, Slots};
    for (const Tensor* t : all) {
        if (!t) continue;
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
    }
    if (!rotary_type(QKV) || QKV->dtype != Q->dtype || QKV->dtype != K->dtype || QKV->dtype != V->dtype) {
        set_error("%s: QKV, Q, K and V must have one type: float16, bfloat16 or float32", name);
        return;
    }
    RotaryArgs a = {};
    a.Hq = params->q_heads;
    a.Hkv = params->kv_heads;
    if (a.Hq < 1 || a.Hkv < 1 || a.Hq > (1 << 20) || a.Hkv > (1 << 20)) {
        set_error("%s: q_heads and kv_heads must be positive, got %d and %d", name, a.Hq, a.Hkv);
        return;
    }
    a.H = a.Hq + 2 * a.Hkv;
    if (QKV->ndim != 2 || QKV->shape[1] < 1 || QKV->shape[1] % a.H) {
        set_error("%s: QKV must be [tokens, (q_heads + 2 kv_heads) * size]", name);
        return;
    }
    a.T = QKV->shape[0];
    a.D = QKV->shape[1] / a.H;
    if (Q->ndim != 3 || Q->shape[0] != a.T || Q->shape[1] != a.Hq || Q->shape[2] != a.D) {
        set_error("%s: Q must be [tokens, q_heads, size]", name);
        return;
    }
    if (Slots) {
        if (!index_type(Slots) || Slots->ndim != 1 || Slots->shape[0] != a.T) {
            set_error("%s: Slots must be int32 or int64 [tokens]", name);
            return;
        }
        if (K->ndim != 4 || V->ndim != 4 || K->shape[1] != a.Hkv || K->shape[3] != a.D || K->shape[2] < 1 ||
            V->shape[0] != K->shape[0] || V->shape[1] != a.Hkv || V->shape[2] != K->shape[2] || V->shape[3] != a.D) {
            set_error("%s: with Slots, K and V must be caches [pages, kv_heads, page size, size]", name);
            return;
        }
        a.ps = K->shape[2];
        a.slots_n = (int64_t)K->shape[0] * a.ps;
        a.fd_ps = make_fastdiv((uint32_t)a.ps);
    } else if (K->ndim != 3 || V->ndim != 3 || K->shape[0] != a.T || V->shape[0] != a.T || K->shape[1] != a.Hkv ||
               V->shape[1] != a.Hkv || K->shape[2] != a.D || V->shape[2] != a.D) {
        set_error("%s: without Slots, K and V must be [tokens, kv_heads, size]", name);
        return;
    }
    const Tensor* weights[] = {QWeight, KWeight};
    for (const Tensor* w : weights) {
        if (!w) continue;
        if (w->ndim != 1 || w->shape[0] != a.D || ((int)w->dtype != kF32 && w->dtype != QKV->dtype) ||
            (QWeight && KWeight && QWeight->dtype != KWeight->dtype)) {
            set_error("%s: QWeight and KWeight must be [size], both float32 or both of QKV's type", name);
            return;
        }
        a.weight_dt = (int)w->dtype;
    }
    if (!Cos != !Sin || (Cos && !Positions)) {
        set_error("%s: a rotation needs Cos, Sin and Positions", name);
        return;
    }
    if (Cos) {
        if (Cos->ndim != 2 || Sin->ndim != 2 || Cos->shape[0] != Sin->shape[0] || Cos->shape[1] != Sin->shape[1] ||
            Cos->dtype != Sin->dtype || ((int)Cos->dtype != kF32 && Cos->dtype != QKV->dtype) || Cos->shape[1] < 1 ||
            2 * (int64_t)Cos->shape[1] > a.D) {
            set_error("%s: Cos and Sin must be [positions, rotated / 2], both float32 or both of QKV's type, with at "
                      "most the head's size rotated", name);
            return;
        }
        a.R = 2 * Cos->shape[1];
        a.rows = Cos->shape[0];
        a.table_dt = (int)Cos->dtype;
    }
    if (Positions && (!index_type(Positions) || Positions->ndim != 1 || Positions->shape[0] != a.T)) {
        set_error("%s: Positions must be int32 or int64 [tokens]", name);
        return;
    }
    if (!(params->epsilon >= 0.0f) || !std::isfinite(params->epsilon)) {
        set_error("%s: epsilon must not be negative, got %g", name, (double)params->epsilon);
        return;
    }
    if (!ensure_device()) return;
    if (!QKV->size) return;
    a.epsilon = params->epsilon;
    a.interleaved = params->interleaved != 0;
    a.norm_q = QWeight != nullptr;
    a.norm_k = KWeight != nullptr;
    a.x = QKV->data;
    a.wq = QWeight ? QWeight->data : nullptr;
    a.wk = KWeight ? KWeight->data : nullptr;
    a.cos = Cos ? Cos->data : nullptr;
    a.sin = Sin ? Sin->data : nullptr;
    a.q = Q->data;
    a.k = K->data;
    a.v = V->data;
    if (Positions) a.pos = {Positions->data, (int)Positions->dtype == kI64};
    if (Slots) a.slots = {Slots->data, (int)Slots->dtype == kI64};
    DeviceScope scope;
    const int64_t heads = (int64_t)a.T * a.H;
    const unsigned grid = grid_for((size_t)heads, 4, 1u << 20);
    if ((int)QKV->dtype == kF16) hipLaunchKernelGGL((k_rotary_any<kF16>), dim3(grid), dim3(256), 0, stream(), a, heads);
    else if ((int)QKV->dtype == kBF16) hipLaunchKernelGGL((k_rotary_any<kBF16>), dim3(grid), dim3(256), 0, stream(), a, heads);
    else hipLaunchKernelGGL((k_rotary_any<kF32>), dim3(grid), dim3(256), 0, stream(), a, heads);
    check_launch(name);
}
