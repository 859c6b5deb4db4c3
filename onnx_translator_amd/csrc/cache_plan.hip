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
// launch and a chain of dependent loads (lengths, free pages, the table).  So one block does it
// all, a request per thread; pages and tokens are spread over the threads by a search in the
// sums, which stay in LDS.
#include "attention.h"

#include <algorithm>

namespace tohip {
namespace {

// int32 or int64 numbers, read and written; ALL32: the call's are all int32.  (Told apart at every
// read, loads that could go out together wait for each other, each in a branch of its own.)
template <bool ALL32> struct Numbers {
    void* p;
    int is64;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return !ALL32 && is64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
    }
    __device__ __forceinline__ bool holds(int64_t v) const { return (!ALL32 && is64) || v <= 0x7FFFFFFF; }
    __device__ __forceinline__ void set(int64_t i, int64_t v) const {
        if (!ALL32 && is64) ((int64_t*)p)[i] = v;
        else ((int32_t*)p)[i] = (int32_t)v;
    }
};

template <bool ALL32> struct PlanArgs {
    typedef Numbers<ALL32> N;
    N fresh, past, offset;             // offset.p may be null
    const int64_t* state;              // pages taken, given back (ever), requests refused
    int64_t* next;
    N pages, ring, start, len, pos, slots;
    int B, cols, ps, T;
    int64_t cap, F;                    // tokens that a table's row can name; size of the ring
    FastDiv fd_ps;
};

template <bool I> __device__ __forceinline__ int64_t pages_of(const PlanArgs<I>& a, int64_t tokens) {      // 0 <= tokens <= cap < 2^31
    return (int64_t)a.fd_ps.div((uint32_t)tokens + (uint32_t)a.ps - 1);
}
template <bool I> __device__ __forceinline__ int64_t held_pages(const PlanArgs<I>& a, int64_t past) { return pages_of(a, past < 0 ? 0 : past > a.cap ? a.cap : past); }
// Place k of the ring.
template <bool I> __device__ __forceinline__ int64_t ring_at(const PlanArgs<I>& a, int64_t base, int64_t k) {
    const int64_t i = base + k;
    return i < a.F ? i : i % a.F;
}

// The lanes' numbers up to and with each, added: DPP moves within rows of 16 and from row to row.
template <int CTRL, int ROWS> __device__ __forceinline__ int64_t lanes_before(int64_t v) {      // (0 where there is none)
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xF, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)((uint64_t)v >> 32), CTRL, ROWS, 0xF, false);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {
    v += lanes_before<0x111, 0xF>(v);
    v += lanes_before<0x112, 0xF>(v);
    v += lanes_before<0x114, 0xF>(v);
    v += lanes_before<0x118, 0xF>(v);
    v += lanes_before<0x142, 0xA>(v);
    return v + lanes_before<0x143, 0xC>(v);
}
// N sums at once over the block, up to and with each thread's, and their totals.
template <int NT, int N> __device__ __forceinline__ void block_scan(int64_t (&v)[N], int64_t (*waves)[N], int64_t (&total)[N]) {
    const int lane = (int)threadIdx.x & 63, w = (int)threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = wave_scan(v[i]);
    __syncthreads();                   // (the last scan's waves[] are read)
    if (lane == 63) {
#pragma unroll
        for (int i = 0; i < N; i++) waves[w][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        int64_t before = 0;
        total[i] = 0;
#pragma unroll
        for (int j = 0; j < NT / 64; j++) {
            const int64_t x = waves[j][i];
            before += j < w ? x : 0;
            total[i] += x;
        }
        v[i] += before;
    }
}

// For each of the numbers from .. n - 1 the first of the NT rising sums that is above it: store(number,
// that entry, load(number, that entry)).  Four of a thread at a time, so that their searches and their
// loads go out together (512 requests, 7000 pages back: 11.1 us; sums, searches and loads one after
// the other 18).
template <int NT, class L, class S> __device__ __forceinline__ void spread(const int* sums, int from, int n, L load, S store) {
    // (unsigned: the last round of 2^31 - 2 pages goes past an int)
    for (unsigned k0 = (unsigned)from + threadIdx.x; k0 < (unsigned)n; k0 += 4 * NT) {
        int at[4] = {};
#pragma unroll
        for (int step = NT / 2; step > 0; step /= 2) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if ((unsigned)sums[at[i] + step - 1] <= k0 + i * NT) at[i] += step;
        }
        int64_t x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if ((unsigned)sums[at[i]] <= k0 + i * NT) at[i]++;       // (at < NT where k < n)
            x[i] = k0 + i * NT < (unsigned)n ? load((int)(k0 + i * NT), at[i]) : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (k0 + i * NT < (unsigned)n) store((int)(k0 + i * NT), at[i], x[i]);
    }
}

template <bool I> __device__ __forceinline__ int64_t offset_of(const PlanArgs<I>& a) {
    const int64_t o = a.offset.p ? a.offset[0] : 0;
    return o < 0 ? 0 : min(o, int64_t(1) << 60);
}
// Row t: token `place` of a request, on `page`, or none (place < 0).  A position that Positions does
// not hold counts as none, a slot on a page that is no page as -1.
template <bool I> __device__ __forceinline__ void place_token(const PlanArgs<I>& a, int64_t t, int64_t place, int64_t page, int64_t offset) {
    int64_t pos = -1, slot = -1;
    if (place >= 0 && a.pos.holds(offset + place)) {
        pos = offset + place;
        const int64_t col = (int64_t)a.fd_ps.div((uint32_t)place);
        if (page >= 0 && page <= 0x7FFFFFFF) slot = page * a.ps + (place - col * a.ps);
        if (!a.slots.holds(slot)) slot = -1;
    }
    a.pos.set(t, pos);
    a.slots.set(t, slot);
}

// A block does all requests, NT at a time.  TOKENS: positions and slots of all rows too; otherwise each
// request's first row gets its position, or -1, and k_plan_tokens does the others from it.
template <int NT, bool TOKENS, bool I> __global__ __launch_bounds__(NT) void k_plan(PlanArgs<I> a) {
    __shared__ int64_t waves[NT / 64][3];
    __shared__ int sum_back[NT], sum_pages[NT], sum_tokens[NT], past_of[NT], have_of[NT];
    __shared__ unsigned long long cut_;
    __shared__ int refused_;
    const int tid = (int)threadIdx.x;
    const int64_t taken = a.state[0], given = a.state[1], offset = offset_of(a);
    // ends of the ring as places in it (a state that no ring has counts as an empty ring)
    const bool sane = taken >= 0 && given >= taken && given - taken <= a.F;
    if (tid == 0) { refused_ = 0; cut_ = 0; }
    const int64_t ring_from = sane ? taken % a.F : 0, ring_to = sane ? given % a.F : 0;
    // Pages of ended requests s0 .. s0 + NT - 1 go back to the ring, behind the `before` of others.
    auto give = [&](int s0, int64_t before, int64_t total) {
        if (!sane) return;
        spread<NT>(sum_back, 0, (int)min(total, a.F),
                   [&](int k, int at) { return a.pages[(int64_t)(s0 + at) * a.cols + (k - (at ? sum_back[at - 1] : 0))]; },
                   [&](int k, int, int64_t page) { a.ring.set(ring_at(a, ring_to, before + k), page); });
    };
    int64_t back = 0;
    if (a.B > NT) {                    // all of them before the first page is taken
        for (int s0 = 0; s0 < a.B; s0 += NT) {
            const int s = s0 + tid;
            const bool ended = s < a.B && a.fresh[s] < 0;
            int64_t sum[1] = {ended ? held_pages(a, a.past[s]) : 0}, total[1];
            if (!__syncthreads_or(ended)) continue;
            block_scan<NT>(sum, (int64_t(*)[1])waves, total);
            sum_back[tid] = (int)min(sum[0], (int64_t)0x7FFFFFFF);
            __syncthreads();
            give(s0, back, total[0]);
            back += total[0];
            __syncthreads();           // (sum_back, and the ring is written)
        }
    }

    int64_t tokens = 0, asked = 0, got = 0;
    for (int s0 = 0; s0 < a.B; s0 += NT) {
        const int s = s0 + tid;
        int64_t fresh = 0, past = 0;
        if (s < a.B) {
            fresh = a.fresh[s];
            past = a.past[s];
        }
        const bool ended = fresh < 0;
        const int64_t in = ended ? 0 : min(fresh, (int64_t)0x7FFFFFFF), was = past < 0 ? 0 : past, have = held_pages(a, past);
        // (Needs of requests whose rows are past Positions' end are added too: those behind them
        // are past it as well.)
        const bool fits = !ended && was <= a.cap && was + in <= a.cap;
        const int64_t need = fits ? pages_of(a, was + in) - have : 0;
        int64_t sum[3] = {in, need, ended ? have : 0}, total[3];
        block_scan<NT>(sum, waves, total);
        const int64_t end = tokens + sum[0], begin = end - in, upto = asked + sum[1], tokens0 = tokens, got0 = got;
        if (a.B <= NT) back = total[2];
        const int64_t there = sane ? min(given + back - taken, a.F) : 0;
        const bool served = fits && end <= a.T && (need == 0 || upto <= there);
        tokens += total[0];
        asked += total[1];
        if (served && need) atomicMax(&cut_, (unsigned long long)upto);      // (whose pages are there)
        if (s < a.B && !ended && !served) atomicAdd(&refused_, 1);
        sum_back[tid] = (int)min(sum[2], (int64_t)0x7FFFFFFF);
        sum_pages[tid] = (int)min(upto - got0, (int64_t)0x7FFFFFFF);
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
        got = max((int64_t)cut_, got0);
        if (a.B <= NT && total[2]) {
            give(s0, 0, total[2]);
            __syncthreads();           // (the ring is written)
        }
        spread<NT>(sum_pages, 0, (int)(got - got0), [&](int k, int) { return a.ring[ring_at(a, ring_from, got0 + k)]; },
                   [&](int k, int at, int64_t page) {
                       a.pages.set((int64_t)(s0 + at) * a.cols + have_of[at] + k - (at ? sum_pages[at - 1] : 0), page);
                   });
        if constexpr (TOKENS) {
            // (pages that the step has taken come from the ring, so that nothing waits for the table)
            const int from = (int)min(tokens0, (int64_t)a.T), to = (int)min(tokens, (int64_t)a.T);
            auto place_of = [&](int t, int at) { return past_of[at] < 0 ? (int64_t)-1 : (int64_t)past_of[at] + t - (at ? sum_tokens[at - 1] : from); };
            spread<NT>(sum_tokens, from, to,
                       [&](int t, int at) {
                           const int64_t place = place_of(t, at);
                           if (place < 0) return (int64_t)-1;
                           const int64_t col = (int64_t)a.fd_ps.div((uint32_t)place), more = col - have_of[at];
                           return more < 0 ? a.pages[(int64_t)(s0 + at) * a.cols + col]
                                           : a.ring[ring_at(a, ring_from, got0 + (at ? sum_pages[at - 1] : 0) + more)];
                       },
                       [&](int t, int at, int64_t page) { place_token(a, t, place_of(t, at), page, offset); });
        }
        __syncthreads();               // (the sums, cut_)
    }
    if constexpr (TOKENS) {            // rows behind the last request
        for (int64_t t = min(tokens, (int64_t)a.T) + tid; t < a.T; t += NT) place_token(a, t, -1, -1, 0);
    }
    if (a.B == 0) __syncthreads();     // (refused_)
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
template <bool I> __global__ __launch_bounds__(256) void k_plan_tokens(PlanArgs<I> a) {
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
        place_token(a, t, -1, -1, 0);
        return;
    }
    while (b < hi) {                           // the last b with start <= t
        const int mid = (b + hi + 1) >> 1;
        if (a.start[mid] <= t) b = mid;
        else hi = mid - 1;
    }
    // (the first row's own position is written again as it is, whoever reads it meanwhile)
    const int64_t begin = a.start[b], first = a.pos[begin];
    const int64_t place = first < 0 ? -1 : first - offset + (t - begin);
    place_token(a, t, place, place < 0 ? -1 : a.pages[(int64_t)b * a.cols + (int64_t)a.fd_ps.div((uint32_t)place)], offset);
}

bool index_type(const Tensor* t) { return (int)t->dtype == kI32 || (int)t->dtype == kI64; }

template <bool I> void launch_plan(PlanArgs<I>& a, const Tensor* New, const Tensor* Past, const Tensor* Offset, const Tensor* State, Tensor* Pages,
                                   Tensor* Free, Tensor* QStart, Tensor* KVLen, Tensor* Positions, Tensor* Slots, Tensor* NextState, hipStream_t s) {
    auto of = [](const Tensor* t) { return t ? Numbers<I>{t->data, (int)t->dtype == kI64} : Numbers<I>{nullptr, 0}; };
    a.fresh = of(New);
    a.past = of(Past);
    a.offset = of(Offset);
    a.state = (const int64_t*)State->data;
    a.next = (int64_t*)NextState->data;
    a.pages = of(Pages);
    a.ring = of(Free);
    a.start = of(QStart);
    a.len = of(KVLen);
    a.pos = of(Positions);
    a.slots = of(Slots);
    // Up to 4096 rows one launch does (8 requests of a token: 4.5 us; two launches take 4 more), in a
    // small block where that is enough (1024 threads: 7.9).
    if (a.T > 4096) {
        hipLaunchKernelGGL((k_plan<512, false, I>), dim3(1), dim3(512), 0, s, a);
        hipLaunchKernelGGL(k_plan_tokens<I>, dim3(grid_for((size_t)a.T, 256, 1u << 24)), dim3(256), 0, s, a);
    } else if (a.B <= 256 && a.T <= 1024) {
        hipLaunchKernelGGL((k_plan<256, true, I>), dim3(1), dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((k_plan<512, true, I>), dim3(1), dim3(512), 0, s, a);
    }
}

}  // namespace
}  // namespace tohip

using namespace tohip;

extern "C" void cache_plan_forward(const Tensor* New, const Tensor* Past, const Tensor* Offset, const Tensor* State,
                                   Tensor* Pages, Tensor* Free, Tensor* QStart, Tensor* KVLen, Tensor* Positions,
                                   Tensor* Slots, Tensor* NextState, const CachePlanParams* params) {
    const char* name = "cache_plan_forward";
    tensor_ops_hip_clear_error();
    if (!params) { set_error("%s: NULL params", name); return; }
    const Tensor* needed[] = {New, Past, State, Pages, Free, QStart, KVLen, Positions, Slots, NextState};
    for (const Tensor* t : needed)
        if (!tensor_sane(t, name)) return;
    const Tensor* all[] = {New, Past, State, Pages, Free, QStart, KVLen, Positions, Slots, NextState, Offset};
    for (const Tensor* t : all) {
        if (!t) continue;              // (Offset)
        if (!tensor_sane(t, name)) return;
        if (t->size && !is_dev(classify(t->data))) { set_error("%s: every tensor must be device-resident", name); return; }
        if (!index_type(t)) { set_error("%s: every tensor must be int32 or int64", name); return; }
    }
    PlanArgs<true> a = {};
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
    a.fd_ps = make_fastdiv((uint32_t)a.ps);
    DeviceScope scope;
    bool all32 = true;
    for (const Tensor* t : all) all32 = all32 && (!t || t == State || t == NextState || (int)t->dtype == kI32);
    if (all32) {
        launch_plan<true>(a, New, Past, Offset, State, Pages, Free, QStart, KVLen, Positions, Slots, NextState, stream());
    } else {
        PlanArgs<false> b = {};
        b.B = a.B;
        b.cols = a.cols;
        b.ps = a.ps;
        b.T = a.T;
        b.cap = a.cap;
        b.F = a.F;
        b.fd_ps = a.fd_ps;
        launch_plan<false>(b, New, Past, Offset, State, Pages, Free, QStart, KVLen, Positions, Slots, NextState, stream());
    }
    check_launch(name);
}
