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

#include <algorithm>
#include <cmath>
#include <type_traits>

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
// ([8192, 48 x 128] bf16: 303 us, bound by its 2-byte accesses; the chunks below take 47.)
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

// ---- whole chunks: heads in registers --------------------------------------------------
// L lanes hold a head, two 16-byte chunks each: lane u of the first P chunk pairs has the
// chunks that the rotation turns together (u and u + P of the rotated part, or 2u and
// 2u + 1 when interleaved), the others the values behind the rotated part.  Squares are
// summed over the L lanes, so a head is read once and nothing passes through LDS.
// A group of lanes takes several heads of one token, one after the other, with the
// token's cosines and sines and the weights in registers: read for every head they would
// be three times the bytes of the head itself through L1.
template <int DT, int VEC> __device__ __forceinline__ void unpack(uint4 c, float (&v)[VEC]) {
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (DT == kF32) {
            v[i] = u2f(w[i]);
        } else if constexpr (DT == kBF16) {
            v[2 * i] = u2f(w[i] << 16);
            v[2 * i + 1] = u2f(w[i] & 0xFFFF0000u);
        } else {
            v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
            v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        }
    }
}
// Each value rounded to the nearest of the type (the conversion instructions).
template <int DT, int VEC> __device__ __forceinline__ uint4 repack(const float (&v)[VEC]) {
    if constexpr (DT == kF32) {
        return uint4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
    } else {
        typedef std::conditional_t<DT == kF16, _Float16, __bf16> T;
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = (T)v[i];
        return __builtin_bit_cast(uint4, h);
    }
}
// VEC values of the tables or weights at element i (float32, or of the data's type).
template <int DT, int VEC> __device__ __forceinline__ void load_params(const void* p, int dt, int64_t i, float (&v)[VEC]) {
    if (DT == kF32 || dt == kF32) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const float4 f = *reinterpret_cast<const float4*>((const float*)p + i + e);
            v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
        }
    } else {
        unpack<DT, VEC>(*reinterpret_cast<const uint4*>((const uint16_t*)p + i), v);
    }
}
// The sum over aligned groups of L lanes, in every lane of the group.
template <int L> __device__ __forceinline__ float lane_group_sum(float v) {
    v += dpp_mov<0xB1>(v);                       // quad_perm [1, 0, 3, 2]
    v += dpp_mov<0x4E>(v);                       // quad_perm [2, 3, 0, 1]
    if constexpr (L > 4) v += dpp_mov<0x141>(v); // row_half_mirror
    if constexpr (L > 8) v += dpp_mov<0x140>(v); // row_mirror
    float x, y;
    if constexpr (L > 16) {
        permlane_pair<16>(v, x, y);
        v = x + y;
    }
    if constexpr (L > 32) {
        permlane_pair<32>(v, x, y);
        v = x + y;
    }
    return v;
}

template <int DT, int L> __global__ __launch_bounds__(256) void k_rotary_chunks(RotaryArgs a, int groups, FastDiv fd_groups) {
    constexpr int ES = DT == kF32 ? 4 : 2, VEC = 16 / ES;
    const int u = (int)threadIdx.x & (L - 1);
    const int P = a.R / (2 * VEC), CH = a.D / VEC;         // turned chunk pairs, chunks of a head
    const bool inter = a.interleaved;
    // this lane's chunks (CH: none)
    const int c0 = u < P && !inter ? u : 2 * u < CH ? 2 * u : CH;
    const int c1 = u < P && !inter ? u + P : 2 * u + 1 < CH ? 2 * u + 1 : CH;
    const int64_t n = (int64_t)a.T * groups, step = (int64_t)gridDim.x * (256 / L);        // n < 2^32
    for (int64_t w = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; w < n; w += step) {
        const uint32_t tw = fd_groups.div((uint32_t)w);
        const int64_t t = tw;
        const int g = (int)((uint32_t)w - tw * (uint32_t)groups);
        const int64_t pos = a.pos.p ? a.pos[t] : 0;
        if (pos < 0 || (a.cos && pos >= a.rows)) continue;
        // cosines and sines of the pairs in the lane's first and second chunk
        float cs[VEC], sn[VEC];
        if (u < P) {
            // halves: pair e of both chunks is (i, i + R/2); interleaved: VEC/2 pairs in each
            load_params<DT, VEC>(a.cos, a.table_dt, pos * (a.R / 2) + (int64_t)u * VEC, cs);
            load_params<DT, VEC>(a.sin, a.table_dt, pos * (a.R / 2) + (int64_t)u * VEC, sn);
        }
        const int64_t slot = a.slots.p ? a.slots[t] : 0;
        const bool stored = !a.slots.p || (slot >= 0 && slot < a.slots_n);
        int64_t kv = t * a.Hkv * a.D, kvh = a.D;           // key head 0 of the token, and the step to the next
        if (a.slots.p) {
            const int64_t page = !stored ? 0 : a.slots_n <= 0xFFFFFFFFll ? (int64_t)a.fd_ps.div((uint32_t)slot) : slot / a.ps;
            kv = (page * a.Hkv * a.ps + (slot - page * a.ps)) * a.D;
            kvh = (int64_t)a.ps * a.D;
        }
        float w0[VEC] = {}, w1[VEC] = {};
        int have = -1;                                 // whose weights w0 and w1 are
        const uint4 zero = {0, 0, 0, 0};
        const char* x = (const char*)a.x + (t * a.H + g) * a.D * ES;
        const int64_t xstep = (int64_t)groups * a.D * ES;
        uint4 n0 = c0 < CH ? *reinterpret_cast<const uint4*>(x + c0 * 16) : zero;
        uint4 n1 = c1 < CH ? *reinterpret_cast<const uint4*>(x + c1 * 16) : zero;
        // neighbouring groups take neighbouring heads; the next head's chunks are on their way
        // while this one's are worked on
        for (int hd = g; hd < a.H; hd += groups) {
            uint4 r0 = n0, r1 = n1;
            x += xstep;
            if (hd + groups < a.H) {
                if (c0 < CH) n0 = *reinterpret_cast<const uint4*>(x + c0 * 16);
                if (c1 < CH) n1 = *reinterpret_cast<const uint4*>(x + c1 * 16);
            }
            const int kind = hd < a.Hq ? 0 : hd < a.Hq + a.Hkv ? 1 : 2;
            if (kind && !stored) continue;
            char* y = kind == 0 ? (char*)a.q + (t * a.Hq + hd) * a.D * ES
                                : (char*)(kind == 1 ? a.k : a.v) + (kv + (hd - a.Hq - (kind == 2 ? a.Hkv : 0)) * kvh) * ES;
            if (kind < 2) {
                float v0[VEC], v1[VEC];
                unpack<DT, VEC>(r0, v0);
                unpack<DT, VEC>(r1, v1);
                if (kind == 0 ? a.norm_q : a.norm_k) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < VEC; e++) sum = __builtin_fmaf(v0[e], v0[e], __builtin_fmaf(v1[e], v1[e], sum));
                    sum = lane_group_sum<L>(sum);
                    const float r = 1.0f / __builtin_sqrtf(sum / (float)a.D + a.epsilon);
                    const void* wt = kind == 0 ? a.wq : a.wk;
                    if (have != kind) {
                        have = kind;
                        if (c0 < CH) load_params<DT, VEC>(wt, a.weight_dt, c0 * VEC, w0);
                        if (c1 < CH) load_params<DT, VEC>(wt, a.weight_dt, c1 * VEC, w1);
                    }
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        v0[e] = v0[e] * r * w0[e];
                        v1[e] = v1[e] * r * w1[e];
                    }
                }
                if (u < P) {
                    if (!inter) {
#pragma unroll
                        for (int e = 0; e < VEC; e++) {
                            const float p = v0[e], q = v1[e];
                            v0[e] = p * cs[e] - q * sn[e];
                            v1[e] = p * sn[e] + q * cs[e];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC; e += 2) {
                            const float p = v0[e], q = v0[e + 1], s = v1[e], z = v1[e + 1];
                            const float ca = cs[e / 2], sa = sn[e / 2], cb = cs[VEC / 2 + e / 2], sb = sn[VEC / 2 + e / 2];
                            v0[e] = p * ca - q * sa;
                            v0[e + 1] = p * sa + q * ca;
                            v1[e] = s * cb - z * sb;
                            v1[e + 1] = s * sb + z * cb;
                        }
                    }
                }
                r0 = repack<DT, VEC>(v0);
                r1 = repack<DT, VEC>(v1);
            }
            if (c0 < CH) *reinterpret_cast<uint4*>(y + c0 * 16) = r0;
            if (c1 < CH) *reinterpret_cast<uint4*>(y + c1 * 16) = r1;
        }
    }
}

template <int DT> void launch_rotary(const RotaryArgs& a, hipStream_t s) {
    constexpr int VEC = DT == kF32 ? 4 : 8;
    auto aligned = [](const void* p) { return ((uintptr_t)p & 15) == 0; };
    const int lanes = (a.D / VEC + 1) / 2;
    if (a.D % VEC == 0 && a.R % (2 * VEC) == 0 && lanes <= 64 && aligned(a.x) && aligned(a.q) && aligned(a.k) &&
        aligned(a.v) && aligned(a.cos) && aligned(a.sin) && aligned(a.wq) && aligned(a.wk)) {
        const int L = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
        // heads per group: the more, the fewer times a token's angles are read, as long as there
        // are 8 waves per CU ([8192, 48 x 128] bf16: 75 us for one head per group, 50 for 4, 47
        // for 6, 49 for 12; [1023, 20 x 80] f32, 5115 waves: 7.4 for one, 6.8 for 2, 8.6 for 8)
        const int64_t waves = (int64_t)a.T * a.H * L / 64;
        int per = (int)std::min<int64_t>({6, a.H, std::max<int64_t>(1, waves / (num_cus() * 8))});
        if ((int64_t)a.T * a.H > 0xFFFFFFFFll) per = a.H;       // 32-bit group numbers
        const int groups = (a.H + per - 1) / per;
        const FastDiv fd = make_fastdiv((uint32_t)groups);
        const unsigned grid = grid_for((size_t)a.T * groups, 256 / L, 1u << 20);
        if (L == 4) hipLaunchKernelGGL((k_rotary_chunks<DT, 4>), dim3(grid), dim3(256), 0, s, a, groups, fd);
        else if (L == 8) hipLaunchKernelGGL((k_rotary_chunks<DT, 8>), dim3(grid), dim3(256), 0, s, a, groups, fd);
        else if (L == 16) hipLaunchKernelGGL((k_rotary_chunks<DT, 16>), dim3(grid), dim3(256), 0, s, a, groups, fd);
        else if (L == 32) hipLaunchKernelGGL((k_rotary_chunks<DT, 32>), dim3(grid), dim3(256), 0, s, a, groups, fd);
        else hipLaunchKernelGGL((k_rotary_chunks<DT, 64>), dim3(grid), dim3(256), 0, s, a, groups, fd);
        return;
    }
    const int64_t heads = (int64_t)a.T * a.H;
    hipLaunchKernelGGL((k_rotary_any<DT>), dim3(grid_for((size_t)heads, 4, 1u << 20)), dim3(256), 0, s, a, heads);
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
    if (overlaps(QKV, Q) || overlaps(QKV, K) || overlaps(QKV, V) || overlaps(Q, K) || overlaps(Q, V) || overlaps(K, V)) {
        set_error("%s: QKV, Q, K and V must not overlap", name);
        return;
    }
    for (const Tensor* out : {Q, K, V})
        for (const Tensor* in : {QWeight, KWeight, Cos, Sin, Positions, Slots})
            if (overlaps(in, out)) { set_error("%s: an output overlaps an input", name); return; }
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
    if ((int)QKV->dtype == kF16) launch_rotary<kF16>(a, stream());
    else if ((int)QKV->dtype == kBF16) launch_rotary<kBF16>(a, stream());
    else launch_rotary<kF32>(a, stream());
    check_launch(name);
}
