"""sample_forward on the GPU against a float64 restatement (tests/decode_ref.py)."""
import math

import numpy as np
import pytest

from tests.decode_ref import Dev, SampleProblem

pytestmark = pytest.mark.gpu

TYPES = ("float16", "bfloat16", "float32")
FILTERS = {"none": {}, "k": dict(k=20), "k1": dict(k=1), "p": dict(p=0.8), "m": dict(m=0.05), "kp": dict(k=40, p=0.9),
           "kpm": dict(k=50, p=0.95, m=0.02), "pm": dict(p=0.7, m=0.1)}


def logits(rows, v, seed=0, std=2.0, tall=8):
    """A bulk, and a few that stand out."""
    rng = np.random.default_rng(seed)
    x = rng.normal(0, std, (rows, v))
    for r in range(rows):
        at = rng.integers(0, v, min(tall, v))
        x[r, at] += rng.uniform(0, 12, len(at))
    return x, rng.random(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", list(FILTERS))
@pytest.mark.parametrize("v", [1, 2, 7, 100, 1000, 8191, 8192, 8193, 32003])
def test_filters(hip, v, filters, dtype):
    x, u = logits(5, v, seed=v)
    SampleProblem(x, u, dtype, t=[1.0, 0.7, 1.3, 0.3, 2.0], **FILTERS[filters]).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", ["none", "p", "kp"])
@pytest.mark.parametrize("v", [50021, 131072, 262144])
def test_large_vocabularies(hip, v, filters, dtype):
    x, u = logits(3, v, seed=v)
    SampleProblem(x, u, dtype, t=[1.0, 0.6, 1.5], **FILTERS[filters]).check(hip)


@pytest.mark.parametrize("rows,v", [(1, 60000), (32, 40000), (33, 50021), (64, 98304), (65, 131072), (129, 131080)])
def test_rows_in_parts(hip, rows, v):
    """However many blocks look through a row; of every kind of row some, flat ones among them."""
    x, u = logits(rows, v, seed=rows)
    x[::5] *= 0.1
    kind = np.arange(rows) % 6
    of = lambda *values: np.asarray(values)[kind]        # noqa: E731
    SampleProblem(x, u, "bfloat16", t=of(1.0, 1.0, 1.0, 1.0, 0.0, 1.0), k=of(0, 0, 0, 30, 0, 0),
                  p=of(0.95, 0.5, 0.99, 1.0, 1.0, 1.0), m=of(0.0, 0.01, 0.0, 0.0, 0.0, 0.2)).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
def test_flat_rows(hip, dtype):
    """Nothing stands out: top-p keeps tens of thousands, top-k thousands."""
    x, u = logits(6, 40000, tall=0, std=0.5)
    SampleProblem(x, u, dtype, p=[0.5, 0.9, 0.99, 0.999, 0.2, 0.01], t=1.0).check(hip)
    SampleProblem(x, u, dtype, k=[4000, 4096, 4097, 5000, 20000, 39999]).check(hip)
    SampleProblem(x, u, dtype, k=[4000, 20000, 30000, 39999, 40000, 50000], p=[0.9, 0.95, 0.5, 0.99, 0.3, 0.999]).check(hip)
    SampleProblem(x, u, dtype, m=[0.001, 0.01, 0.1, 0.2, 0.3, 0.9]).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [10, 5000, 20011, 40013])
def test_equal_logits(hip, v, dtype):
    """Ties rank by index, at the top-k and the top-p border alike."""
    rng = np.random.default_rng(v)
    x = rng.integers(-2, 3, (8, v)).astype(np.float64)
    x[0] = 1.0
    u = rng.random(8).astype(np.float32)
    SampleProblem(x, u, dtype, k=[3, 3, 1, 2, v // 2, v // 3, v - 1, v]).check(hip)
    SampleProblem(x, u, dtype, p=[0.313, 0.771, 0.2077, 0.55, 0.931, 0.1017, 0.0501, 0.99]).check(hip)
    SampleProblem(x, u, dtype, k=[5, 9, v // 2, v // 2, v // 4, v // 4, v - 1, v], p=[0.313, 0.771, 0.2077, 0.55, 0.931, 0.1017, 0.6001, 0.97]).check(hip)


def test_both_zeros_are_equal(hip):
    x = np.array([[-1.0, -0.0, 0.0, -0.0, 0.0]])
    for k, may in ((1, {1}), (2, {1, 2}), (3, {1, 2, 3})):
        seen = set()
        for u in np.linspace(0, 0.999, 13):
            tokens, _ = SampleProblem(x, [u], k=k).check(hip)
            seen.add(int(tokens[0]))
        assert seen == may
    assert SampleProblem(x, [0.5], t=0.0).check(hip)[0][0] == 1


@pytest.mark.parametrize("t", [0.0, -1.0, math.nan])
@pytest.mark.parametrize("dtype", TYPES)
def test_greedy(hip, dtype, t):
    x, u = logits(6, 9000, seed=3)
    x[1, [70, 8500]] = 40.0                          # equal: the first
    x[2, 8999] = 50.0
    x[3, 0] = 50.0
    tokens, lps = SampleProblem(x, u, dtype, t=t, k=5, p=0.5, m=0.1).check(hip)
    assert tokens[1:4].tolist() == [70, 8999, 0] and not lps.any()
    wide = np.full((6, 70001), -5.0)
    wide[:, 30000:39000] = x
    tokens, lps = SampleProblem(wide, u, dtype, t=t, k=5, p=0.5, m=0.1).check(hip)
    assert tokens[1:4].tolist() == [30070, 38999, 30000] and not lps.any()


@pytest.mark.parametrize("v", [3001, 40003])
@pytest.mark.parametrize("t", [1e-30, 1e-3, 50.0, 1e30, math.inf])
def test_temperatures(hip, t, v):
    x, u = logits(4, v, seed=4)
    SampleProblem(x, u, t=t).check(hip)
    SampleProblem(x, u, t=t, k=17).check(hip)
    SampleProblem(x, u, t=t, p=0.8317).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", list(FILTERS))
@pytest.mark.parametrize("v", [5003, 50003])
def test_masked_logits(hip, v, dtype, filters):
    """-inf and NaN are never drawn; a row of nothing else gives -1."""
    x, u = logits(6, v, seed=5)
    rng = np.random.default_rng(6)
    x[0, rng.random(v) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3] = -np.inf
    x[3, 4321] = -3.0                                # one left
    x[4, rng.random(v) < 0.5] = np.nan
    x[5, :5000] = -np.inf
    u[:] = [0.999, 0.5, 0.5, 0.9, 0.99, 0.9]
    tokens, lps = SampleProblem(x, u, dtype, t=[1.0, 1.0, 0.0, 0.7, 1.0, 1.0], **FILTERS[filters]).check(hip)
    assert tokens[1] == tokens[2] == -1 and lps[1] == lps[2] == -np.inf and tokens[3] == 4321 and tokens[5] >= 5000
    assert SampleProblem(x, u, dtype, t=0.0).check(hip)[0][[1, 2, 3]].tolist() == [-1, -1, 4321]


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_logits(hip, dtype):
    """+inf takes everything, several share alike."""
    for v in (2000, 40001):
        x, u = logits(4, v, seed=7)
        x[:, [17, 900, 1500]] = np.inf
        _infinite(hip, x, u, dtype)
    low = np.full((2, 50), float(np.finfo(np.float16).min) if dtype == "float16" else -3e38)
    SampleProblem(low, [0.3, 0.9], dtype, p=[1.0, 0.517]).check(hip)


def _infinite(hip, x, u, dtype):
    for u0, want in ((0.0, 17), (0.4, 900), (0.9, 1500)):
        u[:] = u0
        for f in ({}, dict(p=0.99), dict(m=0.3), dict(k=3)):
            assert (SampleProblem(x, u, dtype, **f).check(hip)[0] == want).all()
        assert (SampleProblem(x, u, dtype, k=1).check(hip)[0] == 17).all()


@pytest.mark.parametrize("u_type", ["float32", "float64"])
def test_uniform_numbers_outside(hip, u_type):
    """Below 0 (or NaN) the first kept token, 1 or more the last."""
    x, _ = logits(1, 500, seed=8)
    kept = np.sort(np.argsort(-x[0])[:10])
    for u, want in ((0.0, kept[0]), (-1.0, kept[0]), (-math.inf, kept[0]), (math.nan, kept[0]), (1.0, kept[-1]), (7.0, kept[-1]), (math.inf, kept[-1])):
        got = SampleProblem(x, [u], k=10, t=5.0, u_type=u_type).run(hip)[0]
        assert got[0] == want, u


def test_settings_out_of_range(hip):
    """k below 1: all; p of 0 or less: the largest alone; p of 1 and more, NaN: all; m above 1: the largest."""
    for v in (3000, 12000, 40000):
        _out_of_range(hip, *logits(6, v, seed=9))


def _out_of_range(hip, x, u):
    v = x.shape[1]
    SampleProblem(x, u, k=[0, -5, v, v + 1, 1 << 30, 2]).check(hip)
    tokens, _ = SampleProblem(x, u, p=[0.0, -1.0, -math.inf, 1.0, 3.0, math.nan]).check(hip)
    assert (tokens[:3] == x[:3].argmax(1)).all()
    tokens, _ = SampleProblem(x, u, m=[1.0, 2.0, math.inf, 0.0, -1.0, math.nan]).check(hip)
    assert (tokens[:3] == x[:3].argmax(1)).all()
    SampleProblem(x, u, k=np.full(6, 1 << 40)).check(hip, index="int64")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns,vocab", [(100, 99), (1001, 1), (9000, 8191), (8200, 8199), (40000, 32761), (50000, 32760), (50001, 49999)])
def test_part_of_the_columns(hip, dtype, columns, vocab):
    """Columns behind the vocabulary are no tokens, whatever they hold."""
    x, u = logits(4, columns, seed=columns)
    x[:, vocab:] = [[np.nan], [np.inf], [1e4], [-np.inf]]
    for f in ({}, dict(k=3), dict(p=0.5), dict(t=0.0)):
        SampleProblem(x, u, dtype, vocab=vocab, **f).check(hip)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257, 600])
def test_rows(hip, rows):
    x, u = logits(rows, 701, seed=rows)
    rng = np.random.default_rng(rows)
    SampleProblem(x, u, "float16", t=rng.uniform(0.3, 1.5, rows) * (rng.random(rows) < 0.9), k=rng.integers(0, 60, rows),
                  p=rng.uniform(0.3, 1.2, rows), m=rng.uniform(0, 0.1, rows)).check(hip)


def test_types_and_absent_results(hip):
    x, u = logits(4, 900, seed=11)
    p = SampleProblem(x, u, k=[3, 0, 9, 1], u_type="float64")
    a = p.check(hip, token="int64", index="int64")
    b = p.check(hip, logprob=False)
    assert (a[0] == b[0]).all()


def test_logits_off_their_alignment(hip):
    """Rows that begin in the middle of a 16-byte chunk, and a tensor that does."""
    import ctypes
    import torch
    from oracle import oracle as O
    from onnx_translator_amd.nn.Operators import CSampleParams
    for dtype, code in ((torch.float16, O.F16), (torch.bfloat16, O.BF16), (torch.float32, O.F32)):
        name = str(dtype).replace("torch.", "")
        for v, skip in ((997, 0), (997, 1), (8193, 3), (20001, 5), (32757, 7), (33001, 1), (50021, 3)):
            x, u = logits(3, v, seed=v + skip)
            p = SampleProblem(x, u, name, k=[0, 30, 7], p=[0.9, 1.0, 0.8])
            flat = torch.full((skip + 3 * v,), float("inf"), dtype=dtype, device="cuda")
            flat[skip:] = p.x.cuda().reshape(-1)
            torch.cuda.synchronize()
            with Dev(hip) as dev:
                xt = hip.lib.tensor_wrap_device(ctypes.c_void_p(flat.data_ptr() + skip * flat.element_size()), (ctypes.c_int * 2)(3, v), 2, code)
                out = dev.put(np.zeros(3, np.int32))
                dev.call("sample_forward", xt, dev.put(p.u), O.PT(), dev.put(p.k), dev.put(p.p), O.PT(), out, O.PT(),
                         ctypes.byref(CSampleParams(0)), O.PT())
                got = hip.dev_read(out, O.I32)
                dev.held.append(xt)
            assert (got == p.run(hip)[0]).all(), (name, v, skip)
            p.check(hip)


@pytest.mark.parametrize("dtype", TYPES)
def test_very_many_columns(hip, dtype):
    """More than a spread row may have: a block per row."""
    v = 2100001
    Dev(hip)
    assert not hip.lib.sample_workspace_bytes(2, v)
    x, u = logits(2, v, seed=13)
    SampleProblem(x, u, dtype, k=[30, 0], p=[0.9, 0.8], t=[1.0, 0.9]).check(hip)


@pytest.mark.parametrize("rows,v", [(3, 40000), (40, 33000)])
def test_workspaces(hip, rows, v):
    """The caller's, one too small (the pool serves) and the pool's: the same tokens."""
    x, u = logits(rows, v, seed=14, tall=4)
    p = SampleProblem(x, u, "bfloat16", p=np.linspace(0.5, 1.1, rows), m=np.linspace(0, 0.01, rows))
    a = p.check(hip)
    need = hip.lib.sample_workspace_bytes(rows, v)
    assert need and not hip.lib.sample_workspace_bytes(rows, 32000)
    for size in (need, need - 1, need + 1000):
        b = p.run(hip, workspace=size)
        assert (a[0] == b[0]).all() and (a[1] == b[1]).all(), size


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_without_a_workspace(hip, dtype):
    """A block per row that reads it again: the tokens of the eager call, replay after replay."""
    import ctypes
    import torch
    from oracle import oracle as O
    from onnx_translator_amd.nn.Operators import CSampleParams
    x, u = logits(7, 45001, seed=15)
    x[5] = np.round(x[5])                            # many equal ones
    x[6, 100:] = -np.inf
    p = SampleProblem(x, u, dtype, t=[1.0, 0.0, 0.8, 1.2, 1.0, 1.0, 1.0], k=[0, 0, 50, 3000, 0, 0, 0], p=[1.0, 1.0, 0.9, 0.9, 0.7, 0.7117, 0.9],
                      m=[0.0, 0.0, 0.0, 0.0, 0.05, 0.0, 0.0])
    want = p.check(hip)[0]
    t = [p.x.cuda(), *(torch.from_numpy(v).cuda() for v in (p.u, p.t, p.k, p.p, p.m)), torch.zeros(7, dtype=torch.int32, device="cuda")]
    code = {torch.float16: O.F16, torch.bfloat16: O.BF16, torch.float32: O.F32, torch.int64: O.I64, torch.int32: O.I32}
    side = torch.cuda.Stream()
    with Dev(hip) as dev:
        w = [hip.lib.tensor_wrap_device(ctypes.c_void_p(v.data_ptr()), (ctypes.c_int * v.dim())(*v.shape), v.dim(), code[v.dtype]) for v in t]
        dev.held += w
        prm = CSampleParams(0)
        hip.lib.tensor_ops_hip_set_stream(ctypes.c_void_p(side.cuda_stream))
        try:
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                dev.call("sample_forward", *w, O.PT(), ctypes.byref(prm), O.PT())
            for _ in range(4):
                t[-1].fill_(-9)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                assert (t[-1].cpu().numpy() == want).all()
        finally:
            torch.cuda.synchronize()
            hip.lib.tensor_ops_hip_set_stream(None)


def test_the_distribution(hip):
    """Evenly spaced numbers draw each token as often as its probability says (within one)."""
    n = 4000
    x = np.broadcast_to(np.log([0.5, 0.2, 0.05, 0.15, 0.1]), (n, 5)).copy()
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for f, p in (({}, [0.5, 0.2, 0.05, 0.15, 0.1]), (dict(k=3), np.array([0.5, 0.2, 0, 0.15, 0]) / 0.85),
                 (dict(p=0.6), np.array([0.5, 0.2, 0, 0, 0]) / 0.7), (dict(m=0.25), np.array([0.5, 0.2, 0, 0.15, 0]) / 0.85)):
        tokens, _ = SampleProblem(x, u, **f).run(hip)
        assert np.abs(np.bincount(tokens, minlength=5) - n * np.array(p)).max() <= 1


def test_repeatable(hip):
    x, u = logits(64, 50000, seed=12, tall=2)
    p = SampleProblem(x, u, "float16", p=0.97)
    a = p.run(hip)
    for _ in range(5):
        b = p.run(hip)
        assert (a[0] == b[0]).all() and (a[1] == b[1]).all()


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("v", [1000, 9000, 40000, 131072])
@pytest.mark.parametrize("high,low", [(1e-37, 0.0), (1e-39, 0.0), (0.0, -1e-37), (1e-37, -1e-37), (5e-36, 1e-36), (2e-35, 0.0), (1e-40, 1e-40)])
def test_logits_that_differ_by_next_to_nothing(hip, high, low, v, dtype):
    """Nearly equal logits around zero, down to subnormal ones: top-k keeps k of them, by value and index."""
    x = np.full((6, v), low)
    x[0, v // 2] = x[1, [3, v - 1]] = x[2, ::v // 9] = high
    x[3, 5:15] = high
    x[4, ::2] = high
    u = np.array([0.02, 0.31, 0.52, 0.77, 0.93, 0.99], np.float32)
    SampleProblem(x, u, dtype, k=[20, 20, 15, 7, 300, 1]).check(hip)
    SampleProblem(x, u, dtype, k=[20, 1, 500, 11, 64, 600], p=[0.523, 0.9, 0.313, 0.771, 0.657, 0.41]).check(hip)


@pytest.mark.parametrize("rows,v,k", [(1, 200003, 8), (20, 131072, 8), (64, 98304, 4), (100, 131072, 2)])
def test_parts_of_a_row_hand_over_what_they_found(hip, rows, v, k):
    """Blocks that look through one row each leave logits for the last of them in a workspace that holds an
    earlier call's: two batches in turn, whose borders lie elsewhere, give the same results every time."""
    import ctypes
    from oracle import oracle as O
    from onnx_translator_amd.nn.Operators import CSampleParams
    with Dev(hip) as dev:
        ws = dev.put(np.full(hip.lib.sample_workspace_bytes(rows, v), 255, np.uint8))
        prm, calls = CSampleParams(0), []
        for seed in range(2):
            x, u = logits(rows, v, seed=seed, std=0.4 + 0.3 * seed, tall=2)
            p = SampleProblem(x, u, "bfloat16", p=np.linspace(0.3 + 0.2 * seed, 0.9, rows), m=np.where(np.arange(rows) % k == 1, 0.05, 0.0))
            want = p.check(hip)
            out, lp = dev.put(np.full(rows, 77, np.int32)), dev.put(np.full(rows, 77, np.float32))
            calls.append((want, out, lp, [dev.put(p.x), dev.put(p.u), O.PT(), O.PT(), dev.put(p.p), dev.put(p.m), out, lp, ctypes.byref(prm), ws]))
        for i in range(40):
            want, out, lp, args = calls[i % 2]
            dev.call("sample_forward", *args)
            assert (hip.dev_read(out, O.I32) == want[0]).all() and (hip.dev_read(lp, O.F32) == want[1]).all(), i


def _captured(hip, p, replays=2):
    """Tokens of a call that is captured without a workspace (a block per row)."""
    import ctypes
    import torch
    from oracle import oracle as O
    from onnx_translator_amd.nn.Operators import CSampleParams
    rows = len(p.x64)
    code = {torch.float16: O.F16, torch.bfloat16: O.BF16, torch.float32: O.F32, torch.float64: O.F64, torch.int64: O.I64, torch.int32: O.I32}
    t = [p.x.cuda() if isinstance(p.x, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(p.x)).cuda()]
    t += [torch.from_numpy(v).cuda() if v is not None else None for v in (p.u, p.t, p.k, p.p, p.m)]
    t += [torch.full((rows,), -9, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")]
    side = torch.cuda.Stream()
    with Dev(hip) as dev:
        w = [O.PT() if v is None else hip.lib.tensor_wrap_device(ctypes.c_void_p(v.data_ptr()), (ctypes.c_int * v.dim())(*v.shape), v.dim(), code[v.dtype])
             for v in t]
        dev.held += [x for x, v in zip(w, t) if v is not None]
        prm = CSampleParams(p.vocab)
        hip.lib.tensor_ops_hip_set_stream(ctypes.c_void_p(side.cuda_stream))
        try:
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                dev.call("sample_forward", *w, ctypes.byref(prm), O.PT())
            for _ in range(replays):
                t[-2].fill_(-9)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
        finally:
            torch.cuda.synchronize()
            hip.lib.tensor_ops_hip_set_stream(None)
        return t[-2].cpu().numpy().astype(np.int64), t[-1].cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("v", [40000, 131072, 2000003])
def test_a_border_far_below_the_largest(hip, v, dtype):
    """A peak and a tail 2^-32 of it and less that top-p keeps in part: the tail counts, whichever blocks
    its logits lie in."""
    rng = np.random.default_rng(v)
    x = np.full((4, v), -22.2)
    x[1] = rng.uniform(-23.5, -22.2, v)
    x[2, :3000] = -20.5
    x[3, ::2] = -24.0
    x[:, 0], x[3, 0], x[3, 777] = 0.0, -22.2, 0.0
    p = SampleProblem(x, np.zeros(4), dtype, p=np.ones(4), u_type="float64")
    w = np.exp(p.x64 - p.x64.max(1, keepdims=True))
    tail = w.sum(1) - 1
    p.p = np.float32(1 - 0.4 * tail)
    p.u = 1 - 0.3 * tail
    tokens, lps = p.run(hip)
    whole = _captured(hip, p)
    assert (tokens == whole[0]).all() and (lps == whole[1]).all()
    # Weights are rounded to 2^-s: a sum of theirs is off by n 2^-s / 2 at most, so what is kept by n 2^-s and a
    # weight, on either side, and with it the sums over it and their share u.
    step = v * 2.0 ** -min(51, 62 - math.ceil(math.log2(v)))
    for r in range(4):
        order = np.lexsort((np.arange(v), -p.x64[r]))
        upto = np.cumsum(w[r, order])
        kept = np.sort(order[:1 + int((upto[:-1] < float(p.p[r]) * upto[-1]).sum())])
        before, total = np.concatenate([[0.0], np.cumsum(w[r, kept])]), w[r, kept].sum()
        off = 6 * step + 4 * w[r, order[1]]
        at = int(np.searchsorted(kept, tokens[r]))
        low, high = before[at], before[min(at + 1, len(kept))]
        assert low - off <= p.u[r] * total <= high + off, (r, tokens[r], low, high, p.u[r] * total, off)
        want = p.x64[r, tokens[r]] - p.x64[r].max() - math.log(total)
        assert abs(lps[r] - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -26 + off
        assert w[r, tokens[r]] < 0.5, "the peak's share is what the draw is past"


@pytest.mark.parametrize("v", [2000, 40001])
@pytest.mark.parametrize("t", [1e-30, 1e-9, 1e-3, math.inf])
def test_infinite_logits_at_any_temperature(hip, t, v):
    """+inf keeps its share where the others' distance from it, over the temperature, is past float64."""
    x, u = logits(4, v, seed=17)
    x[:, [17, 1500]] = np.inf
    u[:] = [0.0, 0.49, 0.51, 0.99]
    for f in ({}, dict(p=0.99), dict(m=0.3), dict(p=0.9, m=0.3), dict(k=3), dict(k=3, p=0.99)):
        tokens, _ = SampleProblem(x, u, "float32", t=t, **f).run(hip)
        assert tokens.tolist() == [17, 17, 1500, 1500], (f, tokens)
