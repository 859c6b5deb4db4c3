"""Plain float64 restatements of the attention operators, with the error that their
arithmetic allows, and helpers that call the library on device tensors.

Tolerance of a result o = sum p v / sum p, from its roundings alone (u = 2^-24 the float32
half step, h the half step of a 16-bit type, 0 for float32; A = sum p |v| / sum p):

* the result is rounded once: (h or u) |o|;
* a weight is rounded to the 16-bit type before the product with V: h A;
* a score is a float32 sum of D products: off by at most (D + 2) u sum_d |q_d k_d| scale, plus
  3 u |s| for the scale, the bias and the subtraction of the maximum; that factor exp(error)
  appears in the weight and in the sum: 2 A times it;
* exp2 of a float32 argument (1 ulp, and half an ulp of the argument's own rounding, |arg| <=
  |s| log2 e + the bias of 16): 2 A (2 + 2 (|s| + 16)) u;
* the sums of n products and weights: 2 n u A;
* float16 weights below 2^-14 are spaced 2^-24 with a row's largest weight at 1 or more:
  n 2^-25 max |v|.
"""
import ctypes
import math

import numpy as np
import torch

from oracle import oracle as O

TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
U = 2.0 ** -24


def attend(q, k, v, scale, seen, bias=None, dtype="float32"):
    """One head: q [n, D], k [m, D], v [m, Dv] (float64, of values of dtype), seen [n, m].  Keys
    not seen add nothing, whatever they hold; a row that sees none is zero.  Returns (o, tol)."""
    n, m = seen.shape
    out, tol = np.zeros((n, v.shape[1])), np.zeros((n, v.shape[1]))
    step = HALF_STEP[dtype]
    h = 0.0 if dtype == "float32" else step
    with np.errstate(all="ignore"):
        for i in range(n):
            w = np.flatnonzero(seen[i])
            if not len(w):
                continue
            prod = q[i] * k[w]
            s = prod.sum(1) * scale
            size = np.abs(s)
            if bias is not None:
                s = s + bias[i, w]
                size = np.maximum(size, np.abs(s))
            top = s.max()
            if top == -math.inf:
                continue
            p = np.exp(s - top)
            total = p.sum()
            o = p @ v[w] / total
            a = p @ np.abs(v[w]) / total
            # keys of no weight have no part in the error
            live = p > 1e-30
            largest = size[live].max(initial=0.0)
            arg = min(largest, 120.0)
            ds = (q.shape[1] + 2) * U * np.abs(prod[live]).sum(1).max(initial=0.0) * scale + 3 * U * largest
            rel = h + 2 * ds + 2 * (2 + 2 * (arg + 16)) * U + 2 * len(w) * U
            out[i] = o
            tol[i] = step * np.abs(o) + rel * a * (1 + rel)
            if dtype == "float16":
                tol[i] += len(w) * 2.0 ** -25 * np.abs(v[w]).max(0) + 2.0 ** -25
    return out, tol


def check(got, ref, tol, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    nan = np.isnan(ref)
    with np.errstate(invalid="ignore"):
        bad = np.where(nan, ~np.isnan(got), ~(np.abs(got - ref) <= tol) & ~(got == ref))
    if bad.any():
        at = [tuple(int(x) for x in i) for i in np.argwhere(bad)[:6]]
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside tolerance; first "
                             f"{[(i, got[i], ref[i], tol[i]) for i in at]}")


def cast(x, dtype):
    """float64 values -> (torch CPU tensor of dtype, the float64 values it holds)."""
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float64)).to(TORCH[dtype])
    return t, t.double().numpy()


def bits(t):
    """Storage array of a torch CPU tensor as the library's codecs have it."""
    if t.dtype == torch.bfloat16:
        return t.view(torch.int16).numpy().view(np.uint16)
    return t.numpy()


class Dev:
    """Device tensors of one test, freed with it."""

    def __init__(self, hip):
        self.hip, self.lib, self.held = hip, hip.lib, []
        P, V = O.PT, ctypes.c_void_p
        for name, args in (("attention_forward", [P] * 6 + [V, P]), ("cache_attention_forward", [P] * 7 + [V, P]),
                           ("qk_norm_rotary_forward", [P] * 10 + [V])):
            f = getattr(self.lib, name)
            f.argtypes, f.restype = args, None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for t in self.held:
            self.lib.free_tensor(t)

    def put(self, x, dtype=None):
        """A device tensor of a torch CPU tensor or of a numpy array (with its dtype's name)."""
        if x is None:
            return O.PT()
        if isinstance(x, torch.Tensor):
            dtype = {v: k for k, v in TORCH.items()}[x.dtype]
            x = bits(x)
        elif dtype is None:
            dtype = str(x.dtype)
        self.held.append(self.hip.dev_from(x, O.dtype_code(dtype)))
        return self.held[-1]

    def get(self, t, dtype):
        raw = self.hip.dev_read(t, O.dtype_code(dtype))
        if dtype == "bfloat16":
            raw = torch.from_numpy(raw.view(np.int16)).view(torch.bfloat16).double().numpy()
        elif dtype == "float16":
            raw = raw.view(np.float16)
        return raw.astype(np.float64)

    def full(self, shape, value, dtype):
        return self.put(torch.full(tuple(shape), value, dtype=TORCH[dtype]))

    def call(self, fn, *args):
        self.lib.tensor_ops_hip_clear_error()
        getattr(self.lib, fn)(*args)
        err = self.hip.last_error()
        assert not err, err


# ---- problems -------------------------------------------------------------------------
class CacheProblem:
    """Sequences of (new tokens, length) over a paged cache; every place of the cache that no
    sequence owns holds NaN, and so do pad_rows rows of q behind the last sequence."""

    def __init__(self, seqs, hq, hkv, d, page, dtype, dv=None, window=0, scale=None, seed=0, pad_rows=0, extra_pages=2,
                 spare_columns=1, std=1.0):
        rng = np.random.default_rng(seed)
        dv = dv or d
        self.seqs, self.hq, self.hkv, self.d, self.dv, self.page, self.dtype = seqs, hq, hkv, d, dv, page, dtype
        self.window, self.scale = window, scale
        need = [-(-l // page) for _, l in seqs]
        total = sum(need) + extra_pages
        order = rng.permutation(total)
        cols = max(need + [0]) + spare_columns
        self.pages = np.full((len(seqs), cols), total + 3, np.int32)      # unused entries name no page
        k = np.full((total, hkv, page, d), np.nan)
        v = np.full((total, hkv, page, dv), np.nan)
        at = 0
        for b, (_, l) in enumerate(seqs):
            self.pages[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            for j in range(l):
                k[self.pages[b, j // page], :, j % page] = rng.normal(0, std, (hkv, d))
                v[self.pages[b, j // page], :, j % page] = rng.normal(0, 1, (hkv, dv))
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.len = np.array([l for _, l in seqs], np.int32)
        t = int(self.start[-1])
        q = np.full((t + pad_rows, hq, d), np.nan)
        q[:t] = rng.normal(0, 1.5 * std, (t, hq, d))
        (self.q, self.q64), (self.k, self.k64), (self.v, self.v64) = (cast(x, dtype) for x in (q, k, v))

    def reference(self, heads=None):
        """(result, tolerance); of some heads only if asked (no check elsewhere)."""
        t = self.q64.shape[0]
        out, tol = np.zeros((t, self.hq, self.dv)), np.zeros((t, self.hq, self.dv))
        if heads is not None:
            tol[:] = np.inf
        scale = self.scale or 1 / math.sqrt(self.d)
        group = self.hq // self.hkv
        for b, (n, l) in enumerate(self.seqs):
            if not n:
                continue
            l = min(l, self.pages.shape[1] * self.page)
            j = np.arange(l)
            page = self.pages[b, j // self.page]
            good = (page >= 0) & (page < self.k64.shape[0])
            safe = np.where(good, page, 0)
            pos = l - n + np.arange(n)[:, None]
            seen = (j <= pos) & good
            if self.window:
                seen &= j > pos - self.window
            rows = slice(self.start[b], self.start[b] + n)
            for h in range(self.hq) if heads is None else heads:
                out[rows, h], tol[rows, h] = attend(self.q64[rows, h], self.k64[safe, h // group, j % self.page],
                                                    self.v64[safe, h // group, j % self.page], scale, seen,
                                                    dtype=self.dtype)
        return out, tol

    def run(self, hip, index="int32", fill=7.0, workspace=0, max_kv=0):
        from onnx_translator_amd.nn.Operators import CCacheAttentionParams
        with Dev(hip) as dev:
            q, k, v = dev.put(self.q), dev.put(self.k), dev.put(self.v)
            ix = [dev.put(x.astype(index)) for x in (self.pages, self.start, self.len)]
            y = dev.full(self.q.shape[:2] + (self.dv,), fill, self.dtype)
            ws = dev.put(np.zeros(workspace, np.uint8)) if workspace else O.PT()
            p = CCacheAttentionParams(self.scale or 0.0, self.window, max_kv)
            dev.call("cache_attention_forward", q, k, v, *ix, y, ctypes.byref(p), ws)
            return dev.get(y, self.dtype)

    def check(self, hip, fill=7.0, heads=None, **kw):
        got = self.run(hip, fill=fill, **kw)
        assert np.isfinite(got).all()
        ref, tol = self.reference(heads)
        t = int(self.start[-1])
        check(got[:t], ref[:t], tol[:t], f"{self.seqs} {self.hq}/{self.hkv} {self.d} page {self.page} {self.dtype}")
        assert (got[t:] == fill).all(), "rows behind the last sequence were written"
        return got


class DenseProblem:
    def __init__(self, b, hq, hkv, sq, skv, d, dtype, dv=None, mask=None, mask_dtype=None, lengths=None, causal=False,
                 packed=False, scale=None, seed=0, std=1.0):
        """mask: float64 values (added; of mask_dtype, 'float32' or dtype) or truth values."""
        rng = np.random.default_rng(seed)
        dv = dv or d
        self.b, self.hq, self.hkv, self.sq, self.skv, self.d, self.dv, self.dtype = b, hq, hkv, sq, skv, d, dv, dtype
        self.causal, self.packed, self.scale = causal, packed, scale
        self.lengths = None if lengths is None else np.asarray(lengths)
        self.q, self.q64 = cast(rng.normal(0, 1.5 * std, (b, hq, sq, d)), dtype)
        self.k, self.k64 = cast(rng.normal(0, std, (b, hkv, skv, d)), dtype)
        self.v, self.v64 = cast(rng.normal(0, 1, (b, hkv, skv, dv)), dtype)
        self.mask, self.mask64 = None, None
        if mask is not None and mask.dtype == bool:
            self.mask, self.mask64 = mask.astype(np.uint8), np.where(mask, 0.0, -np.inf)
        elif mask is not None:
            self.mask, self.mask64 = cast(mask, mask_dtype or dtype)

    def set_v(self, at, value):
        self.v[at] = value
        self.v64[at] = value

    def set_k(self, at, value):
        self.k[at] = value
        self.k64[at] = value

    def reference(self, heads=None):
        """(result, tolerance); of some heads only if asked (no check elsewhere)."""
        out, tol = np.zeros((self.b, self.hq, self.sq, self.dv)), np.zeros((self.b, self.hq, self.sq, self.dv))
        if heads is not None:
            tol[:] = np.inf
        scale, group = self.scale or 1 / math.sqrt(self.d), self.hq // self.hkv
        mask = None if self.mask64 is None else np.broadcast_to(self.mask64, (self.b, self.hq, self.sq, self.skv))
        for b in range(self.b):
            seen = np.ones((self.sq, self.skv), bool)
            if self.lengths is not None:
                seen &= np.arange(self.skv) < self.lengths[b]
            if self.causal:
                seen &= np.tri(self.sq, self.skv, dtype=bool)
            for h in range(self.hq) if heads is None else heads:
                see, bias = seen, None
                if mask is not None:
                    bias = mask[b, h]
                    see = seen & (bias != -np.inf)
                out[b, h], tol[b, h] = attend(self.q64[b, h], self.k64[b, h // group], self.v64[b, h // group], scale,
                                              see, bias, self.dtype)
        return out, tol

    def _laid(self, t):
        return t.permute(0, 2, 1, 3).reshape(t.shape[0], t.shape[2], -1).contiguous() if self.packed else t

    def run(self, hip, workspace=0, index="int32"):
        from onnx_translator_amd.nn.Operators import CAttentionParams
        with Dev(hip) as dev:
            q, k, v = (dev.put(self._laid(t)) for t in (self.q, self.k, self.v))
            mask = dev.put(self.mask)
            length = dev.put(None if self.lengths is None else self.lengths.astype(index))
            shape = (self.b, self.sq, self.hq * self.dv) if self.packed else (self.b, self.hq, self.sq, self.dv)
            y = dev.full(shape, math.nan, self.dtype)
            ws = dev.put(np.zeros(workspace, np.uint8)) if workspace else O.PT()
            p = CAttentionParams(self.hq if self.packed else 0, self.hkv if self.packed else 0, self.scale or 0.0,
                                 int(self.causal))
            dev.call("attention_forward", q, k, v, mask, length, y, ctypes.byref(p), ws)
            got = dev.get(y, self.dtype)
            if self.packed:
                got = got.reshape(self.b, self.sq, self.hq, self.dv).transpose(0, 2, 1, 3)
            return got

    def check(self, hip, heads=None, **kw):
        got = self.run(hip, **kw)
        assert not np.isnan(got).any()
        ref, tol = self.reference(heads)
        check(got, ref, tol, f"b{self.b} h{self.hq}/{self.hkv} {self.sq}x{self.skv} d{self.d} {self.dtype}")
        return got
