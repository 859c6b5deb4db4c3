"""What the decoding loop's operators refuse, without a GPU: the arguments are checked before any
device work, so each call here ends with its own message (a call that passes the checks launches
under the recording runtime of tests/launches)."""
import ctypes

import numpy as np
import pytest

from oracle import oracle as O
from onnx_translator_amd.nn import Tensor, Tensor_
from onnx_translator_amd.nn import Operators as Op


@pytest.fixture(scope="module")
def rec():
    from tests.launches.recorder import Recorder
    r = Recorder()
    P, V = O.PT, ctypes.c_void_p
    r.lib.prefix_cache_attention_forward.argtypes = [P] * 9 + [V, P]
    r.lib.cache_plan_forward.argtypes = [P] * 11 + [V]
    r.lib.sample_forward.argtypes = [P] * 8 + [V, P]
    r.lib.create_tensor.restype = P
    r.lib.create_tensor.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_int, ctypes.c_int]
    return r


def _on_host(rec, args, at):
    c = args[at].contents
    shape = [int(c.shape[i]) for i in range(c.ndim)]
    args[at] = rec.lib.create_tensor(O._ints(shape), len(shape), c.dtype)


def _share(args, at):
    """Argument `to` over the memory of argument `of`."""
    of, to = at
    args[to].contents.data = args[of].contents.data


# ------------------------------------------------------------------------ plans ---
NEW, PAST, OFFSET, STATE, PAGES, FREE, START, LENGTH, POS, SLOTS, NEXT = range(11)


def plan(rec, new=(5,), past=(5,), offset=(1,), state=(3,), pages=(5, 7), free=(40,), start=(6,), length=(5,), pos=(12,),
         slots=None, after=(3,), ix=O.I32, state_dt=O.I64, types=None, page=16, params=True, host=None, share=None):
    shapes = [new, past, offset, state, pages, free, start, length, pos, pos if slots is None else slots, after]
    kinds = [ix] * 11
    kinds[STATE] = kinds[NEXT] = state_dt
    for i, dt in (types or {}).items():
        kinds[i] = dt
    args = [rec.tensor(s, dt) if s is not None else O.PT() for s, dt in zip(shapes, kinds)]
    if host is not None:
        _on_host(rec, args, host)
    if share is not None:
        _share(args, share)
    p = Op.CCachePlanParams(page)
    return rec.call("cache_plan_forward", *args, ctypes.byref(p) if params else None)


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"), (dict(new=None), "NULL tensor"), (dict(after=None), "NULL tensor"),
    (dict(ix=O.F32), "int32 or int64"), (dict(types={SLOTS: O.I16}), "int32 or int64"), (dict(types={PAGES: O.U8}), "int32 or int64"),
    (dict(new=(5, 1)), "New and Past must be"), (dict(past=(4,)), "New and Past must be"),
    (dict(pages=(5,)), "Pages must be"), (dict(pages=(4, 7)), "Pages must be"), (dict(free=(0,)), "Pages must be"),
    (dict(free=(4, 4)), "Pages must be"), (dict(state=(2,)), "State and NextState"), (dict(state_dt=O.I32), "State and NextState"),
    (dict(after=(3, 1)), "State and NextState"), (dict(start=(5,)), "QStart must be"), (dict(length=(6,)), "QStart must be"),
    (dict(slots=(11,)), "Positions and Slots"), (dict(pos=(3, 4)), "Positions and Slots"), (dict(offset=(2,)), "Offset must hold"),
    (dict(offset=(0,)), "Offset must hold"), (dict(page=0), "page_size must be"), (dict(page=-1), "page_size must be"),
    (dict(pages=(5, 1 << 27)), "2^31 tokens"), (dict(page=1 << 29), "2^31 tokens"), (dict(free=(1 << 28,)), "int32 Slots"),
    (dict(share=(NEW, LENGTH)), "overlaps an input"), (dict(share=(PAST, START)), "overlaps an input"),
    (dict(share=(PAST, LENGTH), types={LENGTH: O.I64}), "overlaps an input"), (dict(share=(OFFSET, POS)), "overlaps an input"),
    (dict(share=(STATE, POS)), "overlaps an input"), (dict(share=(PAGES, FREE)), "must not overlap"),
    (dict(share=(POS, SLOTS)), "must not overlap"), (dict(share=(START, LENGTH)), "must not overlap"),
] + [(dict(host=i), "device-resident") for i in range(11)], ids=lambda v: str(v)[:60])
def test_plan_refuses(rec, kw, message):
    launches, err = plan(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("absent", [i for i in range(11) if i != OFFSET])
def test_plan_refuses_null_without_an_offset(rec, absent):
    """An absent Offset makes no other tensor absent."""
    shapes = [(5,), (5,), None, (3,), (5, 7), (40,), (6,), (5,), (12,), (12,), (3,)]
    args = [rec.tensor(s, O.I64 if i in (STATE, NEXT) else O.I32) if s and i != absent else O.PT() for i, s in enumerate(shapes)]
    launches, err = rec.call("cache_plan_forward", *args, ctypes.byref(Op.CCachePlanParams(16)))
    assert "NULL tensor" in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(offset=None), dict(ix=O.I64), dict(types={PAGES: O.I64, POS: O.I64}),
                                dict(share=(PAST, LENGTH)), dict(share=(STATE, NEXT)), dict(new=(0,), past=(0,), pages=(0, 7), start=(1,), length=(0,)),
                                dict(pos=(0,)), dict(pages=(5, 0)), dict(free=(1 << 28,), types={SLOTS: O.I64}), dict(page=1)],
                         ids=lambda v: str(v)[:60])
def test_plan_takes(rec, kw):
    launches, err = plan(rec, **kw)
    assert not err and len(launches) == 1


def test_plan_of_many_tokens(rec):
    """Positions and slots of many rows are a launch of their own, within the runtime's work-items."""
    for rows in (4097, (1 << 31) - 1):
        launches, err = plan(rec, pos=(rows,))
        assert not err and [l.kernel for l in launches] == ["k_plan<512, false, true>", "k_plan_tokens<true>"]
        assert launches[1].grid[0] * launches[1].block >= rows


# ----------------------------------------------------------------------- prefix ---
def prefix(rec, q=(10, 8, 64), k=(12, 2, 16, 64), v=(12, 2, 16, 64), ppages=(5,), plen=(1,), pages=(3, 4), start=(4,), length=(3,),
           y=None, dt=O.BF16, kdt=None, ydt=None, ix=O.I32, pix=None, scale=0.0, max_prefix=0, max_kv=0, params=True, host=None,
           share=None, ws=None):
    t = rec.tensor
    pix = ix if pix is None else pix
    args = [t(q, dt), t(k, dt if kdt is None else kdt), t(v, dt), t(ppages, pix) if ppages is not None else O.PT(), t(plen, pix),
            t(pages, ix), t(start, ix), t(length, ix), t(y or q[:2] + (v[3],), dt if ydt is None else ydt)]
    if host is not None:
        _on_host(rec, args, host)
    if share is not None:
        _share(args, share)
    p = Op.CPrefixAttentionParams(scale, max_prefix, max_kv)
    return rec.call("prefix_cache_attention_forward", *args, ctypes.byref(p) if params else None,
                    t((ws,), O.U8) if ws is not None else O.PT())


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"), (dict(ppages=None), "NULL tensor"),
    (dict(dt=O.F64), "one type"), (dict(kdt=O.F16), "one type"), (dict(ydt=O.F32), "one type"),
    (dict(q=(10, 512), y=(10, 512)), "Q and Y must be"), (dict(k=(12, 2, 16, 32)), "belong together"),
    (dict(q=(10, 7, 64)), "multiple of the key heads"), (dict(y=(10, 8, 32)), "Y must have"),
    (dict(start=(3,)), "Pages must be"), (dict(length=(4,)), "Pages must be"), (dict(ix=O.F32), "Pages must be"),
    (dict(ppages=(5, 1)), "PrefixPages must be"), (dict(plen=(2,)), "PrefixPages must be"), (dict(plen=(0,)), "PrefixPages must be"),
    (dict(pix=O.F32), "PrefixPages must be"), (dict(scale=-1.0), "scale must be positive"),
    (dict(max_prefix=-1), "must not be negative"), (dict(max_kv=-1), "must not be negative"),
    (dict(pages=(3, 1 << 27)), "2^31 keys"), (dict(ppages=(1 << 27,)), "2^31 keys"),
    (dict(ppages=(1 << 26,), pages=(3, 1 << 26)), "2^31 keys"),
    (dict(share=(0, 8)), "Y overlaps an input"), (dict(share=(3, 8)), "Y overlaps an input"), (dict(share=(4, 8)), "Y overlaps an input"),
] + [(dict(host=i), "device-resident") for i in range(9)], ids=lambda v: str(v)[:60])
def test_prefix_refuses(rec, kw, message):
    launches, err = prefix(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(dt=O.F32), dict(ix=O.I64), dict(pix=O.I64), dict(ppages=(0,)), dict(pages=(3, 0)),
                                dict(v=(12, 2, 16, 40)), dict(max_prefix=60, max_kv=9, scale=0.1)], ids=lambda v: str(v)[:60])
def test_prefix_takes(rec, kw):
    """Prefix and own keys in one launch, and their join."""
    launches, err = prefix(rec, **kw)
    assert not err and len(launches) == 2 and launches[0].kernel.startswith("k_prefix") and launches[1].kernel.startswith("k_attn_join")


@pytest.mark.parametrize("tokens,b,d,dt,kernels", [
    (4, 4, 128, O.BF16, ["k_prefix_few<3, 128, 16>"]), (8, 8, 64, O.F32, ["k_prefix_few<4, 64, 32>"]),
    (7, 1, 64, O.F16, ["k_prefix_few<2, 64, 32>"]), (64, 64, 128, O.BF16, ["k_prefix_both<3, 128, 16>"]),
    (64, 10, 64, O.F16, ["k_prefix_both<2, 64, 32>"]), (300, 10, 64, O.F32, ["k_prefix_tiles<4, 64>"]),
    (4096, 16, 128, O.BF16, ["k_attn_tiles<3, 128, true, false, 8, 128>"] * 2), (704, 12, 64, O.F16, ["k_prefix_tiles<2, 64>"]),
    (64, 64, 128, O.F32, ["k_attn_tiles<4, 128, true, false, 4, 32>", "k_attn_few<4, 128, true, false, 16>"]),
    (4, 4, 256, O.F16, ["k_attn_few<2, 256, true, false, 16>"] * 2)], ids=str)
def test_prefix_kernels(rec, tokens, b, d, dt, kernels):
    launches, err = prefix(rec, q=(tokens, 32, d), k=(2000, 8, 16, d), v=(2000, 8, 16, d), ppages=(512,), pages=(b, 8), start=(b + 1,),
                           length=(b,), dt=dt)
    assert not err and [l.kernel for l in launches[:-1]] == kernels and launches[-1].kernel.startswith("k_attn_join")


@pytest.mark.parametrize("kw", [dict(q=(0, 8, 64)), dict(pages=(0, 4), start=(1,), length=(0,))], ids=["no tokens", "no sequences"])
def test_prefix_of_nothing(rec, kw):
    assert prefix(rec, **kw) == ([], "")


def test_prefix_under_capture(rec):
    """The partial results of both parts need memory: a captured call without it is refused, one with
    two splits of it runs, and sizes that a wave per row takes need none."""
    two = 2 * 10 * 8 * (64 * 4 + 8)
    rec.capturing(True)
    try:
        for ws in (None, two - 1):
            launches, err = prefix(rec, ws=ws)
            assert "needs a workspace" in err and not launches
        launches, err = prefix(rec, ws=two, ppages=(1000,))
        assert not err and len(launches) == 2
        launches, err = prefix(rec, q=(10, 8, 63), k=(12, 2, 16, 63), v=(12, 2, 16, 63))
        assert not err and [l.kernel for l in launches] == ["k_prefix_rows<3>"]
    finally:
        rec.capturing(False)


def test_prefix_without_memory(rec):
    rec.no_memory(True)
    try:
        launches, err = prefix(rec)
    finally:
        rec.no_memory(False)
    assert not err and [l.kernel for l in launches] == ["k_prefix_rows<3>"]


# ---------------------------------------------------------------------- sampling ---
def sample(rec, x=(6, 100), u=(6,), t=(6,), k=(6,), p=(6,), m=(6,), token=(6,), lp=(6,), dt=O.F16, udt=O.F32, tdt=O.F32, kdt=O.I32,
           pdt=O.F32, mdt=O.F32, odt=O.I32, ldt=O.F32, vocab=0, params=True, host=None, share=None, ws=None, offset=0):
    arg = lambda s, d: rec.tensor(s, d) if s is not None else O.PT()      # noqa: E731
    args = [rec.tensor(x, dt, offset) if x is not None else O.PT(), arg(u, udt), arg(t, tdt), arg(k, kdt), arg(p, pdt), arg(m, mdt),
            arg(token, odt), arg(lp, ldt)]
    if host is not None:
        _on_host(rec, args, host)
    if share is not None:
        _share(args, share)
    prm = Op.CSampleParams(vocab)
    return rec.call("sample_forward", *args, ctypes.byref(prm) if params else None, arg(ws, O.U8))


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"), (dict(x=None), "NULL tensor"), (dict(u=None), "NULL tensor"), (dict(token=None), "NULL tensor"),
    (dict(dt=O.F64), "Logits must be float16"), (dict(dt=O.I8), "Logits must be float16"), (dict(x=(600,)), "Logits must be [rows"),
    (dict(x=(6, 0)), "Logits must be [rows"), (dict(x=(6, 10, 10)), "Logits must be [rows"), (dict(vocab=101), "vocab must be"),
    (dict(vocab=-1), "vocab must be"), (dict(x=(6, 1 << 24)), "columns"), (dict(offset=1), "aligned"),
    (dict(u=(5,)), "Uniform must be"), (dict(u=(6, 1)), "Uniform must be"), (dict(udt=O.F16), "Uniform must be"),
    (dict(token=(7,)), "Token must be"), (dict(odt=O.F32), "Token must be"), (dict(odt=O.I16), "Token must be"),
    (dict(k=(1,)), "TopK must be"), (dict(kdt=O.F32), "TopK must be"), (dict(t=(1,)), "Temperature, TopP"), (dict(tdt=O.F16), "Temperature, TopP"),
    (dict(p=(2,)), "Temperature, TopP"), (dict(pdt=O.F64), "Temperature, TopP"), (dict(m=(2,)), "Temperature, TopP"),
    (dict(mdt=O.BF16), "Temperature, TopP"), (dict(lp=(2,)), "Temperature, TopP"), (dict(ldt=O.F16), "Temperature, TopP"),
    (dict(share=(0, 6)), "overlaps an input"), (dict(share=(1, 6)), "overlaps an input"), (dict(share=(4, 7)), "overlaps an input"),
    (dict(share=(6, 7)), "must not overlap"),
] + [(dict(host=i), "device-resident") for i in range(8)], ids=lambda v: str(v)[:60])
def test_sample_refuses(rec, kw, message):
    launches, err = sample(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(dt=O.F32), dict(dt=O.BF16), dict(t=None, k=None, p=None, m=None, lp=None), dict(vocab=99),
                                dict(udt=O.F64, kdt=O.I64, odt=O.I64), dict(x=(6, 1)), dict(offset=2), dict(x=(6, 131072))],
                         ids=lambda v: str(v)[:60])
def test_sample_takes(rec, kw):
    launches, err = sample(rec, **kw)
    assert not err and launches


def _kernels(r):
    launches, err = r
    assert not err
    return [l.kernel for l in launches]


@pytest.mark.parametrize("v,kernels", [
    (1, ["k_sample_row<2, 256, true>"]), (8184, ["k_sample_row<2, 256, true>"]), (8185, ["k_sample_row<2, 1024, true>"]),
    (32760, ["k_sample_row<2, 1024, true>"]), (32761, ["k_sample_spans<2>", "k_sample_pick<2>"]),
    (2097144, ["k_sample_spans<2>", "k_sample_pick<2>"]), (2097145, ["k_sample_row<2, 1024, false>"])], ids=str)
def test_sample_kernels(rec, v, kernels):
    """Rows in a block's registers, spread over blocks, or a block's that reads them again."""
    assert _kernels(sample(rec, x=(6, v))) == kernels


def test_sample_without_memory(rec):
    """Without a workspace captured calls, and calls that get no memory, keep a row in a block."""
    whole = ["k_sample_row<3, 1024, false>"]
    x = dict(x=(6, 131072), dt=O.BF16)
    rec.no_memory(True)
    try:
        assert _kernels(sample(rec, **x)) == whole
    finally:
        rec.no_memory(False)
    rec.lib.sample_workspace_bytes.restype = ctypes.c_size_t
    need = rec.lib.sample_workspace_bytes(6, 131072)
    rec.capturing(True)
    try:
        assert _kernels(sample(rec, **x)) == whole
        assert _kernels(sample(rec, ws=(need - 1,), **x)) == whole
        assert _kernels(sample(rec, ws=(need,), **x)) == ["k_sample_spans<3>", "k_sample_pick<3>"]
    finally:
        rec.capturing(False)


def test_sample_of_many_rows(rec):
    n = (1 << 22) - 1
    rows = lambda m: {k: (m,) for k in ("u", "t", "k", "p", "m", "token", "lp")}      # noqa: E731
    assert _kernels(sample(rec, x=(n, 9), **rows(n))) == ["k_sample_row<2, 256, true>"]
    launches, err = sample(rec, x=(n + 1, 9), **rows(n + 1))
    assert "rows" in err and not launches
    # (a launch of its spans would be past the runtime's work-items)
    assert _kernels(sample(rec, x=(1 << 20, 100000), **rows(1 << 20))) == ["k_sample_row<2, 1024, false>"]


def test_sample_of_nothing(rec):
    assert sample(rec, **{n: (0,) for n in ("u", "t", "k", "p", "m", "token", "lp")}, x=(0, 100)) == ([], "")


# ----------------------------------------------------------------- Python layer ---
def test_shapes():
    y = Op.PrefixCacheAttention([], []).forward_(Tensor_(7, 8, 64), Tensor_(3, 2, 16, 64), Tensor_(3, 2, 16, 48))["tensor"]
    assert y.size == (7, 8, 48)
    outs = Op.CachePlan([], [], 16).forward_(Tensor_(5, dtype="int32"), tokens=9)["tensor"]
    assert [t.size for t in outs] == [(6,), (5,), (9,), (9,)] and {t.dtype for t in outs} == {"int32"}
    token, lp = Op.Sample([], [], dtype="int64").forward_(Tensor_(5, 100))["tensor"]
    assert (token.size, token.dtype, lp.size, lp.dtype) == ((5,), "int64", (5,), "float32")


def test_python_refusals():
    x = Tensor(5, 512, dtype="float32")
    with pytest.raises(ValueError, match="scale must be positive"):
        Op._scale(-1.0)
    with pytest.raises(ValueError, match="q must be on the device"):
        Op.PrefixCacheAttention([], []).forward(*[x] * 8)
    with pytest.raises(ValueError, match="new must be on the device"):
        Op.CachePlan([], [], 16).forward(*[x] * 5, tokens=3)
    with pytest.raises(ValueError, match="logits must be on the device"):
        Op.Sample([], []).forward(x, x)


def test_the_plain_plan():
    """The restatement that the GPU tests go by, on a step worked out by hand."""
    from tests.decode_ref import plan as by_hand
    free = np.array([9, 8, 7, 6, 5])
    pages = np.array([[1, -1, -1], [2, 3, -1], [4, -1, -1]])
    out = by_hand(np.array([3, -1, 20]), np.array([15, 17, 0]), pages, free, np.array([3, 5, 0]), 25, 16, offset=100)
    start, length, pos, slots, table, ring, state = [x.tolist() for x in out]
    assert start == [0, 3, 3, 23] and length == [18, 0, 20] and state == [6, 7, 0]
    assert ring == [2, 3, 7, 6, 5] and table == [[1, 6, -1], [2, 3, -1], [5, 2, -1]]
    assert pos == [115, 116, 117] + list(range(100, 120)) + [-1, -1]
    assert slots == [31, 96, 97] + [80 + i for i in range(16)] + [32, 33, 34, 35] + [-1, -1]
