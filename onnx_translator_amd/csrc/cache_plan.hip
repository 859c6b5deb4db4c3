// cache_plan.hip — cache_plan_forward for gfx950: what a step's requests need of a paged
// cache, worked out on the device from their lengths.
//
// Request b holds past_b tokens on ceil(past_b / ps) pages and brings new_b more, or has
// ended (new_b < 0).  With exclusive sums over b:
//   back_b = ended ? ceil(past_b / ps) : 0                    pages given back
//   need_b = ceil((past_b + new_b) / ps) - ceil(past_b / ps)  pages taken
//   start_b = sum of new tokens before b                      its first row
// Free pages lie in a ring; the counts of pages ever taken from it and ever given back to it
// are the ends of what it holds.  Given back first, taken then, in the order of the requests:
// b is served if the needs up to and with its own are there, so a refused request lets none
// behind it take pages that it may get in the next step.
//
// Whole numbers throughout, a fixed order and no memory traffic to speak of: the time is the
// launch and a chain of dependent loads (lengths, free pages, the table).  So a block of 1024
// threads does it all, a request per thread, 1024 at a time; pages and tokens are spread over
// the threads by a search in the sums, which stay in LDS.
#include "attention.h"

#include <algorithm>

namespace tohip {
namespace {

struct IndexOut {
    void* p;
    int is64;
    __device__ __forceinline__ int64_t operator[](int64_t i) const { return IndexVec{p, is64}[i]; }
    __device__ __forceinline__ bool holds(int64_t v) const { return is64 || v <= 0x7FFFFFFF; }
    __device__ __forceinline__ void set(int64_t i, int64_t v) const {
        if (is64) ((int64_t*)p)[i] = v;
        else ((int32_t*)p)[i] = (int32_t)v;
    }
};

struct PlanArgs {
    IndexVec fresh, past, offset;      // offset.p may be null
    const int64_t* state;              // pages taken, given back (ever), requests refused
    int64_t* next;
    IndexVec pages, ring;
    IndexOut pages_to, ring_to, start, len, pos, slots;
    int B, cols, ps, T;
    int64_t cap, F;                    // tokens that a table's row can name; size of the ring
    FastDiv fd_ps;
};

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

__device__ __forceinline__ int64_t pages_of(const PlanArgs& a, int64_t tokens) {      // 0 <= tokens <= cap < 2^31
    return (int64_t)a.fd_ps.div((uint32_t)tokens + (uint32_t)a.ps - 1);
}
// Place k of the ring.
__device__ __forceinline__ int64_t ring_at(const PlanArgs& a, int64_t base, int64_t k) {
    const int64_t i = base + k;
    return i < a.F ? i : i % a.F;
}

// Inclusive sums over the block, the block's total in `total`.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* waves, int64_t& total) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int64_t u = __shfl_up((long long)v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();                   // (the last scan's waves[] are read)
    if (lane == 63) waves[w] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; i++) {
        const int64_t x = waves[i];
        before += i < w ? x : 0;
        total += x;
    }
    return v + before;
}
// The first of n entries of the rising sums that is above k.
__device__ __forceinline__ int first_above(const int* sums, int n, int k) {
    int lo = 0;
    for (int len = n; len > 0;) {
        const int half = len >> 1;
        if (sums[lo + half] <= k) {
            lo += half + 1;
            len -= half + 1;
        } else {
            len = half;
        }
    }
    return lo;
}

__device__ __forceinline__ int64_t offset_of(const PlanArgs& a) {
    const int64_t o = a.offset.p ? a.offset[0] : 0;
    return o < 0 ? 0 : min(o, int64_t(1) << 60);
}
// Row t: token `place` of request b, or none (place < 0).  A position that Positions does not
// hold counts as none, a slot on a page that is no page as -1.
__device__ __forceinline__ void place_token(const PlanArgs& a, int64_t t, int64_t b, int64_t place, int64_t offset) {
    int64_t pos = -1, slot = -1;
    if (place >= 0 && a.pos.holds(offset + place)) {
        pos = offset + place;
        const int64_t col = (int64_t)a.fd_ps.div((uint32_t)place), page = a.pages[b * a.cols + col];
        if (page >= 0 && page <= 0x7FFFFFFF) slot = page * a.ps + (place - col * a.ps);
        if (!a.slots.holds(slot)) slot = -1;
    }
    a.pos.set(t, pos);
    a.slots.set(t, slot);
}

// TOKENS: positions and slots of all rows too; otherwise each request's first row gets its
// position, or -1, and k_plan_tokens does the others from it.
template <bool TOKENS> __global__ __launch_bounds__(kPlanThreads) void k_plan(PlanArgs a) {
    __shared__ int64_t waves[kPlanWaves];
    __shared__ int sum_pages[kPlanThreads], sum_tokens[kPlanThreads], past_of[kPlanThreads], have_of[kPlanThreads];
    __shared__ unsigned long long cut_;
    __shared__ int refused_;
    const int tid = (int)threadIdx.x;
    const int64_t taken = a.state[0], given = a.state[1], offset = offset_of(a);
    // ends of the ring as places in it (a state that no ring has counts as an empty ring)
    const bool sane = taken >= 0 && given >= taken && given - taken <= a.F;
    const int64_t ring_from = sane ? taken % a.F : 0, ring_to = sane ? given % a.F : 0;
    if (tid == 0) refused_ = 0;
    auto lengths = [&](int s, int64_t& fresh, int64_t& past) {
        fresh = a.fresh[s];
        past = a.past[s];
    };
    auto held = [&](int64_t past) { return pages_of(a, past < 0 ? 0 : past > a.cap ? a.cap : past); };

    // ---- pages of ended requests go back
    int64_t back = 0;
    for (int s0 = 0; s0 < a.B; s0 += kPlanThreads) {
        const int s = s0 + tid, n = min(kPlanThreads, a.B - s0);
        int64_t fresh = 0, past = 0, total;
        if (s < a.B) lengths(s, fresh, past);
        if (!__syncthreads_or(fresh < 0)) continue;
        const int64_t mine = fresh < 0 ? held(past) : 0;
        const int64_t incl = block_scan(mine, waves, total);
        sum_pages[tid] = (int)min(incl, (int64_t)0x7FFFFFFF);
        __syncthreads();
        if (sane) {
            for (int k = tid; k < (int)min(total, a.F); k += kPlanThreads) {
                const int at = first_above(sum_pages, n, k);
                const int col = k - (at ? sum_pages[at - 1] : 0);
                a.ring_to.set(ring_at(a, ring_to, back + k), a.pages[(int64_t)(s0 + at) * a.cols + col]);
            }
        }
        back += total;
        __syncthreads();               // (sum_pages)
    }
    __syncthreads();                   // the ring is written
    const int64_t there = sane ? min(given + back - taken, a.F) : 0;

    // ---- pages for the new tokens
    int64_t tokens = 0, asked = 0, got = 0;
    for (int s0 = 0; s0 < a.B; s0 += kPlanThreads) {
        const int s = s0 + tid, n = min(kPlanThreads, a.B - s0);
        int64_t fresh = 0, past = 0, total;
        if (s < a.B) lengths(s, fresh, past);
        const bool ended = fresh < 0;
        const int64_t in = ended ? 0 : min(fresh, (int64_t)0x7FFFFFFF), was = past < 0 ? 0 : past;
        const int64_t end = tokens + block_scan(in, waves, total), begin = end - in;
        const int64_t tokens0 = tokens;
        tokens += total;
        const bool fits = !ended && end <= a.T && was <= a.cap && was + in <= a.cap;
        const int64_t have = held(past), need = fits ? pages_of(a, was + in) - have : 0;
        const int64_t upto = asked + block_scan(need, waves, total);
        asked += total;
        const bool served = fits && (need == 0 || upto <= there);
        if (tid == 0) cut_ = (unsigned long long)got;
        __syncthreads();
        if (served && need) atomicMax(&cut_, (unsigned long long)upto);
        if (s < a.B && !ended && !served) atomicAdd(&refused_, 1);
        __syncthreads();
        // what has been taken up to and with each request (those refused: what was there before)
        const int64_t cut = (int64_t)cut_, got0 = got;
        got = cut;
        sum_pages[tid] = (int)(min(upto, cut) - got0);
        sum_tokens[tid] = (int)min(end, (int64_t)a.T);
        past_of[tid] = served ? (int)was : -1;
        have_of[tid] = (int)have;
        if (s < a.B) {
            a.start.set(s, min(begin, (int64_t)a.T));
            a.len.set(s, ended ? 0 : served ? was + in : past);
            if (!TOKENS && in > 0 && begin < a.T)
                a.pos.set(begin, served && a.pos.holds(offset + was) ? offset + was : -1);
        }
        __syncthreads();
        for (int k = tid; k < (int)(cut - got0); k += kPlanThreads) {
            const int at = first_above(sum_pages, n, k);
            const int col = have_of[at] + k - (at ? sum_pages[at - 1] : 0);
            a.pages_to.set((int64_t)(s0 + at) * a.cols + col, a.ring[ring_at(a, ring_from, got0 + k)]);
        }
        if constexpr (TOKENS) {
            __syncthreads();           // the table is written
            const int from = (int)min(tokens0, (int64_t)a.T), to = (int)min(tokens, (int64_t)a.T);
            for (int t = from + tid; t < to; t += kPlanThreads) {
                const int at = first_above(sum_tokens, n, t);
                const int i = t - (at ? sum_tokens[at - 1] : from);
                place_token(a, t, s0 + at, past_of[at] < 0 ? -1 : (int64_t)past_of[at] + i, offset);
            }
        }
        __syncthreads();               // (the sums)
    }
    if constexpr (TOKENS) {            // rows behind the last request
        for (int64_t t = min(tokens, (int64_t)a.T) + tid; t < a.T; t += kPlanThreads) place_token(a, t, 0, -1, 0);
    }
    __syncthreads();
    if (tid == 0) {
        a.start.set(a.B, min(tokens, (int64_t)a.T));
        a.next[0] = taken + got;
        a.next[1] = given + (sane ? back : 0);
        a.next[2] = refused_;
    }
}

// Positions and slots of many rows: a lane per row.  The request of a row is the last one that
// starts at or before it; a wave looks for that of its first and last row among 64 starts at a
// time, and its lanes in between.
__global__ __launch_bounds__(256) void k_plan_tokens(PlanArgs a) {
    const int lane = (int)threadIdx.x & 63;
    const int64_t t0 = (int64_t)blockIdx.x * 256 + __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63), t = t0 + lane;
    if (t0 >= a.T) return;
    const int64_t rows = a.start[a.B], offset = offset_of(a);
    auto last_at = [&](int64_t row) {          // (row < rows: the answer is in [lo, lo + n))
        int lo = 0, n = a.B;
        while (n > 1) {
            const int step = (n + 63) / 64, b = lo + lane * step;
            const bool le = lane * step < n && a.start[b] <= row;
            const int k = __popcll(__ballot(le));
            if (k > 1) lo += (k - 1) * step;
            n = min(step, a.B - lo);
        }
        return lo;
    };
    int b = 0, hi = 0;
    if (t0 < rows) {
        b = last_at(t0);
        hi = last_at(min(t0 + 63, rows - 1));
    }
    if (t >= a.T) return;
    if (t >= rows) {
        place_token(a, t, 0, -1, 0);
        return;
    }
    while (b < hi) {                           // the last b with start <= t
        const int mid = (b + hi + 1) >> 1;
        if (a.start[mid] <= t) b = mid;
        else hi = mid - 1;
    }
    // (the first row's own position is written again as it is, whoever reads it meanwhile)
    const int64_t begin = a.start[b], first = a.pos[begin];
    place_token(a, t, b, first < 0 ? -1 : first - offset + (t - begin), offset);
}

bool index_type(const Tensor* t) { return (int)t->dtype == kI32 || (int)t->dtype == kI64; }
IndexVec reads(const Tensor* t) { return {t->data, (int)t->dtype == kI64}; }
IndexOut writes(const Tensor* t) { return {t->data, (int)t->dtype == kI64}; }

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" void cache_plan_forward(const Tensor* New, const Tensor* Past, const Tensor* Offset, const Tensor* State,
                                   Tensor* Pages, Tensor* Free, Tensor* QStart, Tensor* KVLen, Tensor* Positions,
                                   Tensor* Slots, Tensor* NextState, const CachePlanParams* params) {
    const char* name = "cache_plan_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    const Tensor* all[] = {New, Past, State, Pages, Free, QStart, KVLen, Positions, Slots, NextState, Offset};
    for (const Tensor* t : all) {
        if (!t && t == Offset) continue;
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
        if (!index_type(t)) { set_error("%s: every tensor must be int32 or int64", name); return; }
    }
    PlanArgs a = {};
    if (New->ndim != 1 || Past->ndim != 1 || Past->shape[0] != New->shape[0]) {
        set_error("%s: New and Past must be [requests]", name);
        return;
    }
    a.B = New->shape[0];
    if (Pages->ndim != 2 || Pages->shape[0] != a.B || Free->ndim != 1 || Free->shape[0] < 1) {
        set_error("%s: Pages must be [requests, pages] and Free [pages]", name);
        return;
    }
    if ((int)State->dtype != kI64 || (int)NextState->dtype != kI64 || State->ndim != 1 || State->shape[0] != 3 ||
        NextState->ndim != 1 || NextState->shape[0] != 3) {
        set_error("%s: State and NextState must be int64 [3]", name);
        return;
    }
    if (QStart->ndim != 1 || QStart->shape[0] != a.B + 1 || KVLen->ndim != 1 || KVLen->shape[0] != a.B) {
        set_error("%s: QStart must be [requests + 1] and KVLen [requests]", name);
        return;
    }
    if (Positions->ndim != 1 || Slots->ndim != 1 || Slots->shape[0] != Positions->shape[0]) {
        set_error("%s: Positions and Slots must be [tokens]", name);
        return;
    }
    if (Offset && Offset->size != 1) { set_error("%s: Offset must hold one number", name); return; }
    a.cols = Pages->shape[1];
    a.ps = params->page_size;
    a.F = Free->shape[0];
    a.T = Positions->shape[0];
    if (a.ps < 1) { set_error("%s: page_size must be positive, got %d", name, a.ps); return; }
    a.cap = (int64_t)a.cols * a.ps;
    if (a.cap + a.ps > 0x7FFFFFFF) { set_error("%s: Pages hold 2^31 tokens or more per request", name); return; }
    if ((int)Slots->dtype == kI32 && a.F * a.ps > 0x7FFFFFFF) {
        set_error("%s: int32 Slots do not hold the places of %lld pages of %d", name, (long long)a.F, a.ps);
        return;
    }
    // KVLen may be Past and NextState State, each as a whole; nothing else may share memory
    auto same = [](const Tensor* x, const Tensor* y) { return x->data == y->data && x->dtype == y->dtype; };
    const Tensor* outs[] = {Pages, Free, QStart, KVLen, Positions, Slots, NextState};
    const Tensor* ins[] = {New, Past, Offset, State};
    for (size_t i = 0; i < sizeof outs / sizeof *outs; i++) {
        for (const Tensor* in : ins) {
            if (!overlaps(in, outs[i]) || (outs[i] == KVLen && in == Past && same(in, KVLen)) ||
                (outs[i] == NextState && in == State && same(in, NextState)))
                continue;
            set_error("%s: an output overlaps an input", name);
            return;
        }
        for (size_t j = 0; j < i; j++)
            if (overlaps(outs[i], outs[j])) { set_error("%s: outputs must not overlap", name); return; }
    }
    if (!ensure_device()) return;
    a.fresh = reads(New);
    a.past = reads(Past);
    if (Offset) a.offset = reads(Offset);
    a.state = (const int64_t*)State->data;
    a.next = (int64_t*)NextState->data;
    a.pages = reads(Pages);
    a.pages_to = writes(Pages);
    a.ring = reads(Free);
    a.ring_to = writes(Free);
    a.start = writes(QStart);
    a.len = writes(KVLen);
    a.pos = writes(Positions);
    a.slots = writes(Slots);
    a.fd_ps = make_fastdiv((uint32_t)a.ps);
    DeviceScope scope;
    if (a.T <= 4096) {
        hipLaunchKernelGGL((k_plan<true>), dim3(1), dim3(kPlanThreads), 0, stream(), a);
    } else {
        hipLaunchKernelGGL((k_plan<false>), dim3(1), dim3(kPlanThreads), 0, stream(), a);
        hipLaunchKernelGGL(k_plan_tokens, dim3(grid_for((size_t)a.T, 256, 1u << 24)), dim3(256), 0, stream(), a);
    }
    check_launch(name);
}
