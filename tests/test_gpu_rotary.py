"""qk_norm_rotary_forward on the GPU against a float64 restatement.

Tolerance: the result is rounded once (half a step h of the type, u = 2^-24 for float32).  Before
that, in float32: x * x and its sum of D terms, the division, the epsilon, the square root and
the reciprocal put at most (D / 2 + 6) u on the norm's factor (half of the sum's relative error,
which is at most D u as all terms are positive); two products make 2 u more, and the rotation's two
products and their sum 3 u of |a c| + |b s|.  Together (D / 2 + 12) u of (|a| |c| + |b| |s|)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import oracle as O
from onnx_translator_amd.nn.Operators import CQKNormRotaryParams
from tests.attention_ref import HALF_STEP, U, Dev, cast, check

pytestmark = pytest.mark.gpu
TYPES = ("float16", "bfloat16", "float32")


class Rotary:
    def __init__(self, t, hq, hkv, d, r, dtype, interleaved=False, norm="qk", tables="float32", weights=None, page=0,
                 rows=200, epsilon=1e-6, seed=0, std=2.0):
        rng = np.random.default_rng(seed)
        self.t, self.hq, self.hkv, self.d, self.r, self.dtype = t, hq, hkv, d, r, dtype
        self.interleaved, self.epsilon, self.page, self.rows = interleaved, epsilon, page, rows
        self.x, self.x64 = cast(rng.normal(0, std, (t, (hq + 2 * hkv) * d)), dtype)
        self.wq = cast(1 + rng.normal(0, 0.2, d), weights or dtype) if "q" in norm else (None, None)
        self.wk = cast(1 + rng.normal(0, 0.2, d), weights or dtype) if "k" in norm else (None, None)
        self.cos = self.sin = (None, None)
        if r:
            angle = np.arange(rows)[:, None] * 100.0 ** (-np.arange(0, r, 2) / r)
            self.cos, self.sin = cast(np.cos(angle), tables), cast(np.sin(angle), tables)
        self.pos = rng.integers(0, rows, t).astype(np.int32)
        if page:
            self.pages = -(-t // page) + 3
            self.slots = rng.permutation(self.pages * page)[:t].astype(np.int32)

    def reference(self):
        x = self.x64.reshape(self.t, -1, self.d)
        out, tol = x.copy(), np.zeros_like(x)
        half = self.r // 2
        a = np.arange(0, self.r, 2) if self.interleaved else np.arange(half)
        b = a + 1 if self.interleaved else a + half
        for lo, hi, (_, w) in ((0, self.hq, self.wq), (self.hq, self.hq + self.hkv, self.wk)):
            y = x[:, lo:hi]
            if w is not None:
                y = y / np.sqrt((y * y).mean(-1, keepdims=True) + self.epsilon) * w
            z, size = y.copy(), np.abs(y)
            if self.r:
                ok = (self.pos >= 0) & (self.pos < self.rows)
                c, s = (t[1][np.where(ok, self.pos, 0)][:, None] for t in (self.cos, self.sin))
                z[..., a], z[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
                size[..., a] = np.abs(y[..., a] * c) + np.abs(y[..., b] * s)
                size[..., b] = np.abs(y[..., a] * s) + np.abs(y[..., b] * c)
            out[:, lo:hi] = z
            tol[:, lo:hi] = HALF_STEP[self.dtype] * np.abs(z) + (self.d / 2 + 12) * U * size * (1 + 2.0 ** -7)
            if self.dtype == "float16":
                tol[:, lo:hi] += 2.0 ** -24          # below the normal range
        return out, tol

    def run(self, hip, index="int32", fill=5.0):
        with Dev(hip) as dev:
            q = dev.full((self.t, self.hq, self.d), fill, self.dtype)
            kv = (self.pages, self.hkv, self.page, self.d) if self.page else (self.t, self.hkv, self.d)
            k, v = dev.full(kv, fill, self.dtype), dev.full(kv, fill, self.dtype)
            ix = lambda a: dev.put(a.astype(index))      # noqa: E731
            p = CQKNormRotaryParams(self.hq, self.hkv, self.epsilon, int(self.interleaved))
            dev.call("qk_norm_rotary_forward", dev.put(self.x), dev.put(self.wq[0]), dev.put(self.wk[0]),
                     dev.put(self.cos[0]), dev.put(self.sin[0]), ix(self.pos), ix(self.slots) if self.page else O.PT(),
                     q, k, v, ctypes.byref(p))
            return [dev.get(t, self.dtype) for t in (q, k, v)]

    def check(self, hip, fill=5.0, **kw):
        q, k, v = self.run(hip, fill=fill, **kw)
        ref, tol = self.reference()
        what = f"t{self.t} {self.hq}/{self.hkv} d{self.d} r{self.r} {self.dtype}"
        ok = (self.pos >= 0) & (self.pos < self.rows) if self.r else self.pos >= 0
        check(q[ok], ref[ok, :self.hq], tol[ok, :self.hq], what)
        assert (q[~ok] == fill).all()
        want = {"k": ref[:, self.hq:self.hq + self.hkv], "v": ref[:, self.hq + self.hkv:]}
        band = {"k": tol[:, self.hq:self.hq + self.hkv], "v": tol[:, self.hq + self.hkv:]}
        for name, got in (("k", k), ("v", v)):
            if not self.page:
                check(got[ok], want[name][ok], band[name][ok], what + name)
                assert (got[~ok] == fill).all()
                continue
            got = got.transpose(0, 2, 1, 3).reshape(-1, self.hkv, self.d)
            in_ = ok & (self.slots >= 0) & (self.slots < len(got))
            check(got[self.slots[in_]], want[name][in_], band[name][in_], what + name)
            rest = np.ones(len(got), bool)
            rest[self.slots[in_]] = False
            assert (got[rest] == fill).all(), "slots that no token names were written"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(64, 64), (128, 128), (128, 64), (80, 40), (256, 256), (96, 32), (40, 8), (66, 66), (20, 6),
                                 (33, 32), (128, 2), (512, 128), (8, 8), (1, 0), (192, 192), (64, 48)])
def test_sizes(hip, d, r, interleaved, dtype):
    Rotary(5, 6, 2, d, r, dtype, interleaved, page=16, seed=d + r).check(hip)
    Rotary(3, 3, 1, d, r, dtype, interleaved, seed=d + r).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1, 2, 7, 64, 333])
def test_tokens(hip, t, dtype):
    Rotary(t, 8, 2, 128, 128, dtype, page=16, rows=5000, seed=t).check(hip)
    Rotary(t, 5, 5, 64, 64, dtype, rows=5000, seed=t).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", ["", "q", "k", "qk"])
@pytest.mark.parametrize("r", [0, 64])
def test_norms(hip, norm, r, dtype):
    Rotary(9, 4, 2, 64, r, dtype, norm=norm, weights="float32" if norm == "q" else None, page=3, seed=1).check(hip)


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("tables", ["float32", "own"])
def test_table_types(hip, tables, dtype):
    Rotary(17, 4, 2, 128, 128, dtype, tables=dtype if tables == "own" else "float32", seed=2).check(hip)


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_that_are_left_out(hip, dtype, index):
    """Negative positions and ones past the tables; slots outside the cache."""
    p = Rotary(40, 4, 2, 64, 64, dtype, page=8, seed=3)
    p.pos[[0, 7, 39]] = [-1, -2 ** 31, p.rows]
    p.slots[[1, 8, 38]] = [-1, p.pages * 8, 2 ** 31 - 1]
    p.check(hip, index=index)
    p = Rotary(40, 4, 2, 64, 64, dtype, seed=3)
    p.pos[[0, 7, 39]] = [-1, -2 ** 31, 2 ** 31 - 1]
    p.check(hip, index=index)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_heads_and_large_values(hip, dtype):
    """A head of zeros stays zero (the epsilon), large values keep their norm."""
    p = Rotary(4, 2, 1, 64, 64, dtype, seed=4, std=100.0)
    p.x[1], p.x64[1] = 0, 0
    p.check(hip)
