"""Plain restatements of the decoding loop's operators: page plans in whole numbers, attention
behind a shared prefix and sampling in float64 (attention's tolerance: tests/attention_ref.py)."""
import ctypes
import math

import numpy as np

from oracle import oracle as O
from tests import attention_ref
from tests.attention_ref import U, attend, cast, check


class Dev(attention_ref.Dev):
    """Device tensors of one test, freed with it."""

    def __init__(self, hip):
        super().__init__(hip)
        P, V = O.PT, ctypes.c_void_p
        for name, args in (("prefix_cache_attention_forward", [P] * 9 + [V, P]), ("cache_plan_forward", [P] * 11 + [V]),
                           ("sample_forward", [P] * 8 + [V, P])):
            f = getattr(self.lib, name)
            f.argtypes, f.restype = args, None
        self.lib.sample_workspace_bytes.argtypes, self.lib.sample_workspace_bytes.restype = [ctypes.c_int] * 2, ctypes.c_size_t


# ------------------------------------------------------------------------ plans ---
def plan(new, past, pages, free, state, rows, page, offset=0):
    """[q_start, kv_len, positions, slots, pages, free, state] after a step, request by request."""
    pages, free, past = pages.astype(np.int64).copy(), free.astype(np.int64).copy(), np.maximum(past.astype(np.int64), 0)
    taken, given = int(state[0]), int(state[1])
    cols, size = pages.shape[1], len(free)
    before = np.asarray(past)
    for b in np.flatnonzero(new < 0):
        for c in range(-(-int(past[b]) // page)):
            free[given % size] = pages[b, c]
            given += 1
    there, asked, refused = given - taken, 0, 0
    start, length = [0], []
    positions, slots = np.full(rows, -1, np.int64), np.full(rows, -1, np.int64)
    total = 0
    for b, n in enumerate(int(x) for x in new):
        begin, total = total, total + max(n, 0)
        start.append(min(total, rows))
        if n < 0:
            length.append(0)
            continue
        have, most = -(-int(past[b]) // page), -(-(int(past[b]) + n) // page)
        fits = total <= rows and most <= cols
        asked += most - have if fits else 0
        if not fits or (most > have and asked > there):
            refused += 1
            length.append(int(before[b]))
            continue
        for c in range(have, most):
            pages[b, c] = free[taken % size]
            taken += 1
        for i in range(n):
            j = int(past[b]) + i
            positions[begin + i] = j + offset
            at = pages[b, j // page]
            slots[begin + i] = at * page + j % page if at >= 0 else -1
        length.append(int(past[b]) + n)
    return [np.array(x, np.int64) for x in (start, length, positions, slots, pages, free, [taken, given, refused])]


class PlanProblem:
    """Requests (new, past) with tables, and a ring that holds the pages that no table names."""

    def __init__(self, requests, page, spare=50, cols=None, rows=None, offset=0, seed=0, taken=None):
        rng = np.random.default_rng(seed)
        self.new, self.past = (np.array([r[i] for r in requests], np.int64) for i in (0, 1))
        have = -(-self.past // page)
        need = -(-(self.past + np.maximum(self.new, 0)) // page)
        cols = int(max(need.max(initial=0), 1)) if cols is None else cols
        used = int(have.sum())
        total = used + max(spare, 1)
        order = rng.permutation(total)
        self.pages = np.full((len(requests), cols), -7, np.int64)
        at = 0
        for b, n in enumerate(have):
            n = min(int(n), cols)
            self.pages[b, :n] = order[at:at + n]
            at += n
        taken = int(rng.integers(0, 3 * total)) if taken is None else taken
        self.free = np.full(total, -9, np.int64)
        self.free[(taken + np.arange(spare)) % total] = order[used:used + spare]
        self.state = np.array([taken, taken + spare, 4], np.int64)
        self.page, self.offset = page, offset
        self.rows = int(np.maximum(self.new, 0).sum()) if rows is None else rows

    def run(self, hip, index="int32", in_place=False, out=None):
        from onnx_translator_amd.nn.Operators import CCachePlanParams
        out = out or index
        with Dev(hip) as dev:
            put = lambda x, dt=index: dev.put(np.asarray(x).astype(dt))      # noqa: E731
            new, past, state = put(self.new), put(self.past), put(self.state, "int64")
            pages, free = put(self.pages), put(self.free)
            b = len(self.new)
            start, slots, pos = (put(np.full(n, 99), out) for n in (b + 1, self.rows, self.rows))
            length = past if in_place else put(np.full(b, 99), out)
            after = state if in_place else put(np.full(3, 99), "int64")
            p = CCachePlanParams(self.page)
            dev.call("cache_plan_forward", new, past, put([self.offset]) if self.offset else O.PT(), state, pages, free,
                     start, length, pos, slots, after, ctypes.byref(p))
            kinds = (out, index if in_place else out, out, out, index, index, "int64")
            got = [hip.dev_read(t, O.dtype_code(k)).astype(np.int64)
                   for t, k in zip((start, length, pos, slots, pages, free, after), kinds)]
            if not in_place:
                assert (hip.dev_read(past, O.dtype_code(index)) == self.past).all()
                assert (hip.dev_read(state, O.I64) == self.state).all()
            return got

    def reference(self):
        return plan(self.new, self.past, self.pages, self.free, self.state, self.rows, self.page, self.offset)

    def check(self, hip, **kw):
        got = self.run(hip, **kw)
        for name, g, w in zip(("q_start", "kv_len", "positions", "slots", "pages", "free", "state"), got, self.reference()):
            assert g.shape == w.shape and (g == w).all(), (name, kw, np.flatnonzero((g != w).reshape(-1))[:8], g.reshape(-1)[:20], w.reshape(-1)[:20])
        return got


# ----------------------------------------------------------------------- prefix ---
class PrefixProblem:
    """Sequences of (new tokens, own length) behind a prefix, on one cache; every place that nobody
    owns holds NaN, and so do pad_rows rows of q behind the last sequence."""

    def __init__(self, seqs, shared, hq, hkv, d, page, dtype, dv=None, scale=None, seed=0, pad_rows=0, spare_columns=1,
                 spare_prefix=1, std=1.0, skip_rows=0):
        rng = np.random.default_rng(seed)
        dv = dv or d
        self.seqs, self.shared, self.hq, self.hkv, self.d, self.dv, self.page, self.dtype = seqs, shared, hq, hkv, d, dv, page, dtype
        self.scale = scale
        need = [-(-l // page) for _, l in seqs]
        first = -(-shared // page)
        total = sum(need) + first + 2
        order = rng.permutation(total)
        k, v = np.full((total, hkv, page, d), np.nan), np.full((total, hkv, page, dv), np.nan)

        def fill(which, n):
            j = np.arange(n)
            k[which[j // page], :, j % page] = rng.normal(0, std, (n, hkv, d))
            v[which[j // page], :, j % page] = rng.normal(0, 1, (n, hkv, dv))

        self.prefix_pages = np.full(first + spare_prefix, total + 3, np.int32)
        self.prefix_pages[:first] = order[:first]
        fill(self.prefix_pages, shared)
        self.pages = np.full((len(seqs), max(need + [0]) + spare_columns), -1, np.int32)
        at = first
        for b, (_, l) in enumerate(seqs):
            self.pages[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            fill(self.pages[b], l)
        self.start = (skip_rows + np.concatenate([[0], np.cumsum([n for n, _ in seqs])])).astype(np.int32)
        self.len = np.array([l for _, l in seqs], np.int32)
        t = int(self.start[-1])
        q = np.full((t + pad_rows, hq, d), np.nan)
        q[skip_rows:t] = rng.normal(0, 1.5 * std, (t - skip_rows, hq, d))
        (self.q, self.q64), (self.k, self.k64), (self.v, self.v64) = (cast(x, dtype) for x in (q, k, v))

    def reference(self, heads=None):
        t = self.q64.shape[0]
        out, tol = np.zeros((t, self.hq, self.dv)), np.zeros((t, self.hq, self.dv))
        if heads is not None:
            tol[:] = np.inf
        scale, group = self.scale or 1 / math.sqrt(self.d), self.hq // self.hkv
        shared = min(self.shared, len(self.prefix_pages) * self.page)
        for b, (n, _) in enumerate(self.seqs):
            if not n:
                continue
            l = int(min(max(self.len[b], 0), self.pages.shape[1] * self.page))
            page = np.concatenate([self.prefix_pages[np.arange(shared) // self.page], self.pages[b, np.arange(l) // self.page]])
            place = np.concatenate([np.arange(shared), np.arange(l)]) % self.page
            good = (page >= 0) & (page < self.k64.shape[0])
            safe = np.where(good, page, 0)
            pos = l - n + np.arange(n)[:, None]
            seen = np.concatenate([np.ones((n, shared), bool), np.arange(l) <= pos], 1) & good
            rows = slice(self.start[b], self.start[b] + n)
            for h in range(self.hq) if heads is None else heads:
                out[rows, h], tol[rows, h] = attend(self.q64[rows, h], self.k64[safe, h // group, place],
                                                    self.v64[safe, h // group, place], scale, seen, dtype=self.dtype)
        return out, tol

    def run(self, hip, index="int32", fill=7.0, workspace=0, max_kv=0, max_prefix=0):
        from onnx_translator_amd.nn.Operators import CPrefixAttentionParams
        with Dev(hip) as dev:
            q, k, v = dev.put(self.q), dev.put(self.k), dev.put(self.v)
            ix = [dev.put(np.asarray(x).astype(index)) for x in
                  (self.prefix_pages, [self.shared], self.pages, self.start, self.len)]
            y = dev.full(self.q.shape[:2] + (self.dv,), fill, self.dtype)
            ws = dev.put(np.full(workspace, 255, np.uint8)) if workspace else O.PT()
            p = CPrefixAttentionParams(self.scale or 0.0, max_prefix, max_kv)
            dev.call("prefix_cache_attention_forward", q, k, v, *ix, y, ctypes.byref(p), ws)
            return dev.get(y, self.dtype)

    def check(self, hip, fill=7.0, heads=None, **kw):
        got = self.run(hip, fill=fill, **kw)
        assert np.isfinite(got).all()
        ref, tol = self.reference(heads)
        a, t = int(self.start[0]), int(self.start[-1])
        check(got[a:t], ref[a:t], tol[a:t], f"{self.seqs} behind {self.shared}, {self.hq}/{self.hkv} {self.d} page {self.page} {self.dtype}")
        assert (got[t:] == fill).all() and (got[:a] == fill).all(), "rows of no sequence were written"
        return got


# ---------------------------------------------------------------------- sampling ---
def sample(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(tokens that may be drawn, the log of the first one's probability) of one row of float64
    logits.  Sums of n weights in fixed point of 2^-s, s = min(51, 62 - ceil(log2 n)), are off by at
    most n 2^-s / 2 and float64 ones by less: a draw nearer than n 2^-s to a border may fall on
    either side of it.  The p border must not be that near (the inputs are chosen so)."""
    x = np.where(np.isnan(x), -np.inf, x)
    n = len(x)
    near = n * 2.0 ** -min(51, 62 - math.ceil(math.log2(max(n, 2))))
    top = x.max()
    if top == -np.inf:
        return [-1], -np.inf
    if not t > 0:
        return [int(np.argmax(x))], 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.where((x == -np.inf) | (top == np.inf), 0.0, np.exp((x - top) / t)))
    order = np.lexsort((np.arange(n), -np.where(np.isinf(x), np.sign(x) * 1e300, x)))
    order = order[x[order] > -np.inf]
    if k > 0:
        order = order[:k]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        want = p * w[order].sum()
        assert p <= 0 or np.abs(before[1:] - want).min(initial=np.inf) > near, "a border of top-p"
        order = order[:max(1, int((before < want).sum()))]
    low = min(m, 1.0) if m == m else 0.0
    order = np.sort(order[w[order] >= low])
    upto = np.cumsum(w[order])
    total = upto[-1]
    target = min(max(u, 0.0), 1.0) * total if u == u else 0.0
    lo, hi = np.concatenate([[0.0], upto[:-1]]) - near, upto + near
    may = order[(w[order] > 0) & (lo <= target) & (target < hi)]
    first = int(np.searchsorted(upto, target, side="right"))
    first = order[min(first, len(order) - 1)] if u < 1 or u != u else order[np.flatnonzero(w[order] > 2.0 ** -50)[-1]]
    may = [int(first)] + [int(i) for i in may if i != first]
    return may, None


def log_chance(x, token, t=1.0, k=0, p=1.0, m=0.0):
    """The log of the probability with which the row's token is drawn."""
    may, fixed = sample(x, 0.0, t, k, p, m)
    if fixed is not None:
        return fixed
    x = np.where(np.isnan(x), -np.inf, x)
    top, n = x.max(), len(x)
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(x == top, 0.0, np.where((x == -np.inf) | (top == np.inf), -np.inf, (x - top) / t))
    w = np.exp(y)
    order = np.lexsort((np.arange(n), -np.where(np.isinf(x), np.sign(x) * 1e300, x)))
    order = order[x[order] > -np.inf]
    order = order[:k] if k > 0 else order
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w[order])[:-1]])
        order = order[:max(1, int((before < p * w[order].sum()).sum()))]
    order = order[w[order] >= (min(m, 1.0) if m == m else 0.0)]
    assert token in order
    return y[token] - math.log(w[order].sum())


class SampleProblem:
    """Rows of logits with a setting of its own for each (None: not given)."""

    def __init__(self, x, u, dtype="float32", t=None, k=None, p=None, m=None, vocab=0, u_type="float32"):
        self.x, self.x64 = cast(x, dtype)
        rows = len(self.x64)
        self.dtype, self.vocab, self.u_type = dtype, vocab, u_type
        spread = lambda v, dt: None if v is None else np.broadcast_to(np.asarray(v, dt), (rows,)).copy()      # noqa: E731
        self.u = spread(u, u_type)
        self.t, self.k, self.p, self.m = spread(t, np.float32), spread(k, np.int64), spread(p, np.float32), spread(m, np.float32)

    def run(self, hip, token="int32", index="int32", logprob=True, workspace=0):
        from onnx_translator_amd.nn.Operators import CSampleParams
        with Dev(hip) as dev:
            put = lambda v: dev.put(v) if v is not None else O.PT()      # noqa: E731
            rows = len(self.x64)
            out = dev.put(np.full(rows, 77, token))
            lp = dev.put(np.full(rows, 77, np.float32)) if logprob else O.PT()
            ws = dev.put(np.full(workspace, 255, np.uint8)) if workspace else O.PT()
            k = None if self.k is None else self.k.astype(index)
            p = CSampleParams(self.vocab)
            dev.call("sample_forward", dev.put(self.x), put(self.u), put(self.t), put(k), put(self.p), put(self.m), out, lp,
                     ctypes.byref(p), ws)
            return (hip.dev_read(out, O.dtype_code(token)).astype(np.int64),
                    hip.dev_read(lp, O.F32).astype(np.float64) if logprob else None)

    def settings(self, row):
        at = lambda v, none: none if v is None else float(v[row])      # noqa: E731
        return at(self.t, 1.0), int(at(self.k, 0)), at(self.p, 1.0), at(self.m, 0.0)

    def check(self, hip, **kw):
        tokens, lps = self.run(hip, **kw)
        for row, token in enumerate(tokens):
            x = self.x64[row, :self.vocab or None]
            s = self.settings(row)
            may, _ = sample(x, float(self.u[row]), *s)
            assert token in may, (row, token, may, s, float(self.u[row]))
            if lps is not None:
                want = log_chance(x, token, *s)
                # rounded once; the sum of the weights is off by n 2^-s / 2 <= 2^-27 of 1 or more
                assert lps[row] == want or abs(lps[row] - want) <= U * abs(want) + 2.0 ** -26, (row, token, lps[row], want, s)
        return tokens, lps
