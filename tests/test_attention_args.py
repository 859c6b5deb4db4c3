"""What the attention operators refuse, without a GPU: the arguments are checked before any
device work, so each call here ends with its own message (a call that passes the checks ends
with the missing device's, or launches under the recording runtime of tests/launches)."""
import ctypes
import itertools
import re
import subprocess

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
    r.lib.attention_forward.argtypes = [P] * 6 + [V, P]
    r.lib.cache_attention_forward.argtypes = [P] * 7 + [V, P]
    r.lib.qk_norm_rotary_forward.argtypes = [P] * 10 + [V]
    r.lib.create_tensor.restype = P
    r.lib.create_tensor.argtypes = [ctypes.POINTER(ctypes.c_int), ctypes.c_int, ctypes.c_int]
    return r


def attn(rec, q=(2, 4, 5, 64), k=(2, 2, 7, 64), v=(2, 2, 7, 64), y=None, mask=None, mask_dt=O.U8, length=None, len_dt=O.I32,
         dt=O.F16, kdt=None, vdt=None, ydt=None, heads=(0, 0), scale=0.0, causal=0, params=True):
    t = rec.tensor
    y = y or q[:-1] + (v[-1],)
    p = Op.CAttentionParams(*heads, scale, causal)
    return rec.call("attention_forward", t(q, dt), t(k, dt if kdt is None else kdt), t(v, dt if vdt is None else vdt),
                    t(mask, mask_dt) if mask is not None else O.PT(),
                    t(length, len_dt) if length is not None else O.PT(), t(y, dt if ydt is None else ydt),
                    ctypes.byref(p) if params else None, O.PT())


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"),
    (dict(dt=O.F64), "one type"), (dict(kdt=O.F32), "one type"), (dict(vdt=O.BF16), "one type"), (dict(ydt=O.F32), "one type"),
    (dict(dt=O.I8), "one type"), (dict(dt=O.E4M3), "one type"),
    (dict(q=(2, 5, 64), y=(2, 5, 64)), "must all be"), (dict(q=(4, 5), k=(4, 5), v=(4, 5)), "must all be"),
    (dict(q=(2, 3, 5, 64)), "multiple of the key heads"), (dict(q=(2, 0, 5, 64)), "multiple of the key heads"),
    (dict(k=(2, 2, 7, 32)), "belong together"), (dict(k=(1, 2, 7, 64)), "belong together"),
    (dict(v=(2, 2, 8, 64)), "belong together"), (dict(v=(2, 1, 7, 64)), "belong together"),
    (dict(q=(2, 4, 5, 0), k=(2, 2, 7, 0)), "belong together"),
    (dict(y=(2, 4, 5, 32)), "Y must have"), (dict(y=(2, 4, 6, 64)), "Y must have"),
    (dict(heads=(8, 2)), "differ from the head dimensions"), (dict(heads=(4, 4)), "differ from the head dimensions"),
    (dict(scale=-1.0), "scale must be positive"), (dict(scale=float("nan")), "scale must be positive"),
    (dict(scale=float("inf")), "scale must be positive"),
    (dict(mask=(3, 1, 5, 7)), "does not broadcast"), (dict(mask=(5, 8)), "does not broadcast"),
    (dict(mask=(1, 2, 4, 5, 7)), "does not broadcast"), (dict(mask=(5, 7), mask_dt=O.F64), "Mask must be"),
    (dict(mask=(5, 7), mask_dt=O.BF16), "Mask must be"), (dict(mask=(5, 7), mask_dt=O.I32), "Mask must be"),
    (dict(length=(3,)), "KVLen must be"), (dict(length=(2, 1)), "KVLen must be"), (dict(length=(2,), len_dt=O.F32), "KVLen must be"),
    (dict(q=(2, 5, 256), k=(2, 7, 128), v=(2, 7, 128), y=(2, 5, 256)), "q_heads and kv_heads must divide"),
    (dict(q=(2, 5, 256), k=(2, 7, 128), v=(2, 7, 128), y=(2, 5, 256), heads=(3, 1)), "q_heads and kv_heads must divide"),
    (dict(q=(2, 5, 256), k=(2, 7, 128), v=(2, 7, 128), y=(2, 5, 128), heads=(4, 2)), "Y must have"),
], ids=lambda v: str(v)[:60])
def test_attention_refuses(rec, kw, message):
    launches, err = attn(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(q=(2, 5, 256), k=(2, 7, 128), v=(2, 7, 128), heads=(4, 2), y=(2, 5, 256)),
                                dict(mask=(1, 7)), dict(mask=(7,), mask_dt=O.F16), dict(mask=(2, 1, 5, 1), mask_dt=O.F32),
                                dict(length=(2,), len_dt=O.I64), dict(k=(2, 2, 0, 64), v=(2, 2, 0, 64)),
                                dict(v=(2, 2, 7, 24), y=(2, 4, 5, 24)), dict(dt=O.F32, causal=1), dict(dt=O.BF16)],
                         ids=lambda v: str(v)[:60])
def test_attention_takes(rec, kw):
    launches, err = attn(rec, **kw)
    assert not err and launches


@pytest.mark.parametrize("kw", [dict(q=(0, 4, 5, 64), k=(0, 2, 7, 64), v=(0, 2, 7, 64)), dict(q=(2, 4, 0, 64))],
                         ids=["no batch", "no queries"])
def test_attention_of_nothing(rec, kw):
    assert attn(rec, **kw) == ([], "")


def cache(rec, q=(10, 8, 64), k=(12, 2, 16, 64), v=(12, 2, 16, 64), pages=(3, 4), start=(4,), length=(3,), y=None, dt=O.BF16,
          kdt=None, ydt=None, ix=O.I32, start_dt=None, scale=0.0, window=0, max_kv=0, params=True, host=None):
    t = rec.tensor
    args = [t(q, dt), t(k, dt if kdt is None else kdt), t(v, dt), t(pages, ix), t(start, ix if start_dt is None else start_dt),
            t(length, ix), t(y or q[:2] + (v[3],), dt if ydt is None else ydt)]
    if host is not None:
        shape = [int(args[host].contents.shape[i]) for i in range(args[host].contents.ndim)]
        dtype = args[host].contents.dtype
        args[host] = rec.lib.create_tensor(O._ints(shape), len(shape), dtype)
    p = Op.CCacheAttentionParams(scale, window, max_kv)
    return rec.call("cache_attention_forward", *args, ctypes.byref(p) if params else None, O.PT())


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"),
    (dict(dt=O.F64), "one type"), (dict(kdt=O.F16), "one type"), (dict(ydt=O.F32), "one type"), (dict(kdt=O.E4M3), "one type"),
    (dict(q=(10, 512), y=(10, 512)), "Q and Y must be"), (dict(k=(12, 2, 1024)), "Q and Y must be"),
    (dict(k=(12, 2, 16, 32)), "belong together"), (dict(k=(11, 2, 16, 64)), "belong together"),
    (dict(v=(12, 4, 16, 64)), "belong together"), (dict(v=(12, 2, 8, 64)), "belong together"),
    (dict(k=(0, 2, 16, 64), v=(0, 2, 16, 64)), "belong together"),
    (dict(q=(10, 7, 64)), "multiple of the key heads"), (dict(y=(10, 8, 32)), "Y must have"), (dict(y=(9, 8, 64)), "Y must have"),
    (dict(start=(3,)), "Pages must be"), (dict(length=(4,)), "Pages must be"), (dict(pages=(12,)), "Pages must be"),
    (dict(ix=O.F32), "Pages must be"), (dict(start_dt=O.U8), "Pages must be"),
    (dict(scale=-0.5), "scale must be positive"), (dict(window=-1), "must not be negative"), (dict(max_kv=-1), "must not be negative"),
    (dict(pages=(3, 1 << 27)), "2^31 keys"),
] + [(dict(host=i), "device-resident") for i in range(7)], ids=lambda v: str(v)[:60])
def test_cache_attention_refuses(rec, kw, message):
    launches, err = cache(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(dt=O.F32), dict(ix=O.I64), dict(start_dt=O.I64), dict(window=5, max_kv=100, scale=0.1),
                                dict(v=(12, 2, 16, 40)), dict(k=(12, 2, 17, 64), v=(12, 2, 17, 64))], ids=lambda v: str(v)[:60])
def test_cache_attention_takes(rec, kw):
    launches, err = cache(rec, **kw)
    assert not err and launches


@pytest.mark.parametrize("kw", [dict(q=(0, 8, 64)), dict(pages=(0, 4), start=(1,), length=(0,))], ids=["no tokens", "no sequences"])
def test_cache_attention_of_nothing(rec, kw):
    assert cache(rec, **kw) == ([], "")


def rotary(rec, x=(5, 8 * 64), wq=(64,), wk=(64,), cos=(100, 32), sin=(100, 32), pos=(5,), slots=None, q=(5, 4, 64),
           k=(5, 2, 64), v=(5, 2, 64), dt=O.F16, wdt=None, kwdt=None, tdt=O.F32, ix=O.I32, kdt=None, heads=(4, 2), eps=1e-6,
           params=True, host=None):
    t = lambda s, d: rec.tensor(s, d) if s is not None else O.PT()      # noqa: E731
    wdt = dt if wdt is None else wdt
    args = [t(x, dt), t(wq, wdt), t(wk, wdt if kwdt is None else kwdt), t(cos, tdt), t(sin, tdt), t(pos, ix), t(slots, ix),
            t(q, dt), t(k, dt if kdt is None else kdt), t(v, dt)]
    if host is not None:
        shape = [int(args[host].contents.shape[i]) for i in range(args[host].contents.ndim)]
        args[host] = rec.lib.create_tensor(O._ints(shape), len(shape), args[host].contents.dtype)
    p = Op.CQKNormRotaryParams(*heads, eps, 0)
    return rec.call("qk_norm_rotary_forward", *args, ctypes.byref(p) if params else None)


CACHE = (7, 2, 16, 64)


@pytest.mark.parametrize("kw,message", [
    (dict(params=False), "NULL params"), (dict(x=None), "NULL tensor"), (dict(q=None), "NULL tensor"),
    (dict(dt=O.F64), "one type"), (dict(kdt=O.F32), "one type"),
    (dict(heads=(0, 2)), "must be positive"), (dict(heads=(4, -1)), "must be positive"),
    (dict(x=(5, 8 * 64 + 1)), "QKV must be"), (dict(x=(5, 8, 64)), "QKV must be"), (dict(x=(5, 0)), "QKV must be"),
    (dict(q=(5, 4, 32)), "Q must be"), (dict(q=(4, 4, 64)), "Q must be"),
    (dict(k=(5, 4, 64)), "without Slots"), (dict(v=CACHE), "without Slots"),
    (dict(slots=(5,)), "with Slots"), (dict(slots=(5,), k=CACHE, v=(7, 2, 8, 64)), "with Slots"),
    (dict(slots=(5,), k=(7, 4, 16, 64), v=(7, 4, 16, 64)), "with Slots"), (dict(slots=(4,), k=CACHE, v=CACHE), "Slots must be"),
    (dict(wq=(32,)), "QWeight and KWeight"), (dict(wdt=O.BF16), "QWeight and KWeight"), (dict(kwdt=O.F32), "QWeight and KWeight"),
    (dict(sin=None), "needs Cos, Sin and Positions"), (dict(cos=None), "needs Cos, Sin and Positions"),
    (dict(pos=None), "needs Cos, Sin and Positions"), (dict(sin=(100, 16)), "Cos and Sin"), (dict(cos=(100, 33), sin=(100, 33)), "Cos and Sin"),
    (dict(tdt=O.BF16), "Cos and Sin"), (dict(cos=(100, 0), sin=(100, 0)), "Cos and Sin"),
    (dict(pos=(4,)), "Positions must be"), (dict(ix=O.F32), "Positions must be"),
    (dict(eps=-1.0), "epsilon"), (dict(eps=float("nan")), "epsilon"), (dict(eps=float("inf")), "epsilon"),
] + [(dict(host=i), "device-resident") for i in (0, 1, 2, 3, 4, 5, 7, 8, 9)], ids=lambda v: str(v)[:60])
def test_rotary_refuses(rec, kw, message):
    launches, err = rotary(rec, **kw)
    assert message in err and not launches


@pytest.mark.parametrize("kw", [dict(), dict(slots=(5,), k=CACHE, v=CACHE), dict(wq=None), dict(wq=None, wk=None),
                                dict(cos=None, sin=None, pos=None), dict(cos=None, sin=None), dict(ix=O.I64), dict(dt=O.F32),
                                dict(wdt=O.F32), dict(tdt=O.F16), dict(cos=(100, 8), sin=(100, 8))], ids=lambda v: str(v)[:60])
def test_rotary_takes(rec, kw):
    launches, err = rotary(rec, **kw)
    assert not err and launches


def test_rotary_of_nothing(rec):
    assert rotary(rec, x=(0, 512), pos=(0,), q=(0, 4, 64), k=(0, 2, 64), v=(0, 2, 64)) == ([], "")


# ----------------------------------------------------------------- Python layer ---
def test_shapes():
    a = Op.Attention([], [], dtype="float16")
    assert a.forward_(Tensor_(2, 8, 5, 64), Tensor_(2, 2, 9, 64), Tensor_(2, 2, 9, 32))["tensor"].size == (2, 8, 5, 32)
    a = Op.Attention([], [], q_num_heads=8, kv_num_heads=2)
    y = a.forward_(Tensor_(2, 5, 512, dtype="bfloat16"), Tensor_(2, 9, 128), Tensor_(2, 9, 64))["tensor"]
    assert y.size == (2, 5, 256) and y.dtype == "bfloat16"
    with pytest.raises(ValueError, match="q_num_heads"):
        Op.Attention([], []).forward_(Tensor_(2, 5, 512), Tensor_(2, 9, 128), Tensor_(2, 9, 128))
    c = Op.CacheAttention([], []).forward_(Tensor_(7, 8, 64), Tensor_(3, 2, 16, 64), Tensor_(3, 2, 16, 48))["tensor"]
    assert c.size == (7, 8, 48)
    r = Op.QKNormRotary([], [], 4, 2).forward_(Tensor_(5, 8 * 64))["tensor"]
    assert [t.size for t in r] == [(5, 4, 64), (5, 2, 64), (5, 2, 64)]
    kc = Tensor_(3, 2, 16, 64)
    r = Op.QKNormRotary([], [], 4, 2).forward_(Tensor_(5, 8 * 64), key_cache=kc, value_cache=kc, slots=Tensor_(5))["tensor"]
    assert [t.size for t in r] == [(5, 4, 64), (3, 2, 16, 64), (3, 2, 16, 64)]


def test_python_refusals():
    x = Tensor(5, 512, dtype="float32")
    for scale in (0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale must be positive"):
            Op.Attention([], [], scale=scale).forward(*[Tensor(1, 1, 1, 8, dtype="float32")] * 3)
    with pytest.raises(ValueError, match="qkv must be on the device"):
        Op.QKNormRotary([], [], 4, 2).forward(x)
    with pytest.raises(ValueError, match="q must be on the device"):
        Op.CacheAttention([], []).forward(x, x, x, x, x, x)


def _node(ins, attrs, outs=("y",)):
    from onnx_translator_amd.onnx import proto as P
    return P.NodeProto("Attention", list(ins), list(outs), attributes=[P.make_attribute(k, v) for k, v in attrs.items()])


def test_onnx_attention_node():
    from onnx_translator_amd.nn.ONNXImport import make_op
    op = make_op(_node(["q", "k", "v"], {}), {"y": "float16"}, {})
    assert isinstance(op, Op.Attention) and op.inputs == ["q", "k", "v", ""] and op.scale is None and op.dtype == "float16"
    op = make_op(_node(["q", "k", "v", "m", "", "", "n"], {"q_num_heads": 8, "kv_num_heads": 2, "scale": 0.25}), {}, {})
    assert op.inputs == ["q", "k", "v", "m", "n"] and (op.q_num_heads, op.kv_num_heads, op.scale) == (8, 2, 0.25)
    for ins, attrs, outs in ((["q", "k", "v", "", "pk"], {}, ["y"]), (["q", "k", "v"], {"softcap": 30.0}, ["y"]),
                             (["q", "k", "v"], {}, ["y", "present"]), (["q", "k", "v", "", "", "", "n"], {"is_causal": 1}, ["y"])):
        with pytest.raises(NotImplementedError):
            make_op(_node(ins, attrs, outs), {}, {})


def test_onnx_attention_of_another_domain():
    """The operator of that name in another domain has other inputs (packed weights, say)."""
    from onnx_translator_amd.nn.ONNXImport import ONNXImport, make_op
    from onnx_translator_amd.onnx import proto as P
    node = _node(["x", "w", "b"], {"num_heads": 8})
    node.domain = "com.microsoft"
    with pytest.raises(NotImplementedError, match="com.microsoft"):
        make_op(node, {}, {})
    g = P.GraphProto(nodes=[node], name="g", inputs=[P.ValueInfoProto("x", P.FLOAT, [1, 4, 64])],
                     outputs=[P.ValueInfoProto("y", P.FLOAT, [1, 4, 64])], initializers=[])
    with pytest.raises(NotImplementedError, match="com.microsoft"):
        ONNXImport(P.ModelProto.parse(P.ModelProto(graph=g).serialize()))
    for domain in ("", "ai.onnx"):
        node = _node(["q", "k", "v"], {})
        node.domain = domain
        assert isinstance(make_op(node, {}, {}), Op.Attention)


def test_onnx_attention_softmax_precision():
    """The softmax is float32: float32 and less may be asked for, float64 (11) is refused."""
    from onnx_translator_amd.nn.ONNXImport import make_op
    for precision in (1, 10, 16):
        assert isinstance(make_op(_node(["q", "k", "v"], {"softmax_precision": precision}), {}, {}), Op.Attention)
    with pytest.raises(NotImplementedError, match="float64"):
        make_op(_node(["q", "k", "v"], {"softmax_precision": 11}), {}, {})


# ------------------------------------------------------------------ dispatch -----
def names(result):
    launches, err = result
    assert not err, err
    return [l.kernel.split("<")[0] for l in launches]


def variant(result):
    """Rows of a block of the tile kernel that a call launches."""
    k = result[0][0].kernel
    assert not result[1]
    args = k[k.index("<") + 1:k.rindex(">")].replace(" ", "").split(",")
    return int(args[4]) if k.startswith("k_attn_few") else 32 * int(args[4]) if k.startswith("k_attn_tiles") else 0


@pytest.mark.parametrize("q,k,dt,rows", [
    ((1, 8, 1, 64), (1, 2, 500, 64), O.F16, 16), ((1, 8, 4, 128), (1, 2, 500, 128), O.BF16, 16), ((1, 8, 5, 64), (1, 2, 500, 64), O.F32, 32),
    ((1, 8, 8, 64), (1, 2, 500, 64), O.F16, 32), ((1, 8, 9, 64), (1, 2, 500, 64), O.F16, 128), ((64, 8, 64, 64), (64, 8, 500, 64), O.F16, 256),
    ((64, 8, 64, 64), (64, 8, 500, 64), O.F32, 128), ((64, 8, 64, 256), (64, 8, 500, 256), O.F16, 128),
    ((64, 8, 64, 256), (64, 8, 500, 256), O.F32, 128),
    ((1, 8, 40, 20), (1, 2, 500, 20), O.F16, 0), ((1, 8, 40, 20), (1, 2, 500, 20), O.F32, 128), ((1, 8, 40, 264), (1, 2, 500, 264), O.F16, 0),
    ((1, 8, 1, 30), (1, 2, 500, 30), O.F32, 0)], ids=lambda v: str(v))
def test_rows_of_a_block(rec, q, k, dt, rows):
    r = attn(rec, q=q, k=k, v=k, dt=dt)
    assert variant(r) == rows and (rows or names(r) == ["k_attn_rows"])


@pytest.mark.parametrize("dt", [O.F16, O.BF16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,rows", [(1, 128), (2, 256), (3, 256), (16, 256)])
def test_a_tile_of_keys_names_64_pages_at_most(rec, page, rows, d, dt):
    """Blocks of 256 rows have tiles of 128 keys, and a wave holds 64 page numbers."""
    caches = (16384 // page, 8, page, d)
    r = cache(rec, q=(4096, 32, d), k=caches, v=caches, pages=(1, 16384 // page), start=(2,), length=(1,), dt=dt)
    assert variant(r) == rows


def test_keys_split_where_blocks_are_few(rec):
    few, many = ((1, 8, 1, 64), (1, 8, 1500, 64)), ((512, 8, 64, 64), (512, 8, 1500, 64))
    assert names(attn(rec, q=few[0], k=few[1], v=few[1])) == ["k_attn_few", "k_attn_join"]
    assert names(attn(rec, q=many[0], k=many[1], v=many[1])) == ["k_attn_tiles"]
    short = (1, 8, 64, 64)
    assert names(attn(rec, q=few[0], k=short, v=short)) == ["k_attn_few"]
    # neither memory nor a capture: one pass over the keys
    rec.no_memory(True)
    try:
        assert names(attn(rec, q=few[0], k=few[1], v=few[1])) == ["k_attn_few"]
        assert names(cache(rec, pages=(3, 400))) == ["k_attn_few"]
    finally:
        rec.no_memory(False)
    rec.capturing(True)
    try:
        assert names(attn(rec, q=few[0], k=few[1], v=few[1])) == ["k_attn_few"]
        assert names(cache(rec, pages=(3, 400))) == ["k_attn_few"]
        assert names(rotary(rec, slots=(5,), k=CACHE, v=CACHE)) == ["k_rotary_chunks"]
    finally:
        rec.capturing(False)
    assert names(cache(rec, pages=(3, 400))) == ["k_attn_few", "k_attn_join"]
    # what the caller says of the lengths shapes the launch
    assert names(cache(rec, pages=(3, 400), max_kv=64)) == ["k_attn_few"]


def test_a_workspace_splits_under_capture(rec):
    t = rec.tensor
    p = Op.CAttentionParams(0, 0, 0.0, 0)
    rec.capturing(True)
    try:
        for size, kernels in ((1 << 20, ["k_attn_few", "k_attn_join"]), (8 * 264 * 2, ["k_attn_few", "k_attn_join"]), (8 * 264 * 2 - 1, ["k_attn_few"])):
            r = rec.call("attention_forward", t((1, 8, 1, 64), O.F16), t((1, 8, 1500, 64), O.F16), t((1, 8, 1500, 64), O.F16), O.PT(),
                         O.PT(), t((1, 8, 1, 64), O.F16), ctypes.byref(p), t((size,), O.U8))
            assert names(r) == kernels, size
        r = rec.call("attention_forward", t((1, 8, 1, 64), O.F16), t((1, 8, 1500, 64), O.F16), t((1, 8, 1500, 64), O.F16), O.PT(),
                     O.PT(), t((1, 8, 1, 64), O.F16), ctypes.byref(p), t((1 << 20,), O.U8, offset=8))
        assert names(r) == ["k_attn_few"]       # not aligned
    finally:
        rec.capturing(False)


@pytest.mark.parametrize("offset", [2, 8])
def test_operands_off_their_alignment(rec, offset):
    t = rec.tensor
    p = Op.CAttentionParams(0, 0, 0.0, 0)
    for which in range(4):
        ops = [t((1, 8, 40, 64), O.F16, offset=offset if i == which else 0) for i in range(4)]
        assert names(rec.call("attention_forward", *ops[:3], O.PT(), O.PT(), ops[3], ctypes.byref(p), O.PT())) == ["k_attn_rows"]


def test_launches_within_the_runtimes_limit(rec):
    """Blocks past 2^32 work-items: a wave per row instead (the recorder refuses what the runtime would)."""
    big = (1 << 20, 64, 1, 64)
    r = attn(rec, q=big, k=big, v=big)
    assert names(r) == ["k_attn_rows"]
    assert names(attn(rec, q=(1 << 18, 64, 1, 64), k=(1 << 18, 64, 1, 64), v=(1 << 18, 64, 1, 64))) == ["k_attn_few"]
    assert names(rotary(rec, x=(1 << 24, 512), pos=(1 << 24,), q=(1 << 24, 4, 64), k=(1 << 24, 2, 64), v=(1 << 24, 2, 64))) == ["k_rotary_chunks"]


def test_rotary_kernels(rec):
    assert names(rotary(rec)) == ["k_rotary_chunks"]
    assert names(rotary(rec, cos=(100, 12), sin=(100, 12))) == ["k_rotary_any"]           # 24 rotated: no whole chunk pairs
    assert names(rotary(rec, x=(5, 8 * 20), wq=(20,), wk=(20,), cos=None, sin=None, pos=None, q=(5, 4, 20), k=(5, 2, 20), v=(5, 2, 20))) == ["k_rotary_any"]


def test_every_instance_is_reached(rec):
    """The attention kernels in the library are those that some call launches."""
    from tests.launches import recorder
    out = subprocess.run(["nm", "-C", recorder.OUT], capture_output=True, text=True, check=True).stdout
    built = {m.replace(" ", "") for m in re.findall(r"__device_stub__(k_attn_\w+<[^>]*>)", out)}
    launched = set()
    for dt, d, n in itertools.product((O.F16, O.BF16, O.F32), (64, 128, 256), (1, 4, 5, 1000)):
        # one row, up to 16 and 32, and tiles, each with keys to split and without; more heads fill the GPU
        for hkv, skv in ((1, 1500), (2, 64), (128, 300), (16, 1024)):
            q, kv, page = (1, 5 * hkv, n, d), (1, hkv, skv, d), (skv // 4, hkv, 4, d)
            for r in (attn(rec, q=q, k=kv, v=kv, dt=dt), attn(rec, q=q, k=kv, v=kv, dt=dt, mask=(n, skv)),
                      cache(rec, q=(n, 5 * hkv, d), k=page, v=page, pages=(1, skv // 4), start=(2,), length=(1,), dt=dt)):
                assert not r[1]
                launched |= {l.kernel.replace(" ", "") for l in r[0]}
        # a wave per row
        for r in (attn(rec, q=(1, 2, n, d), k=(1, 2, 9, d), v=(1, 2, 9, 33), dt=dt),
                  cache(rec, q=(n, 2, d), k=(3, 2, 4, d), v=(3, 2, 4, 33), pages=(1, 3), start=(2,), length=(1,), dt=dt)):
            launched |= {l.kernel.replace(" ", "") for l in r[0]}
    assert built == launched, (sorted(built - launched), sorted(launched - built))


def test_outputs_overlap_no_input(rec):
    t = rec.tensor
    P = O.PT()
    at = t((2, 2, 5, 64), O.F16)
    same = rec.lib.tensor_wrap_device(at.contents.data + 64, O._ints((2, 2, 5, 64)), 4, O.F16)
    other = [t((2, 2, 5, 64), O.F16) for _ in range(2)]
    p = Op.CAttentionParams(0, 0, 0.0, 0)
    for ops in ((at, other[0], other[1]), (other[0], at, other[1]), (other[0], other[1], at)):
        rec.lib.tensor_ops_hip_clear_error()
        rec.lib.attention_forward(*ops, P, P, same, ctypes.byref(p), P)
        assert b"overlaps" in rec.lib.tensor_ops_hip_last_error()
    q, cache_ = t((4, 2, 64), O.F16), t((3, 2, 4, 64), O.F16)
    rec.lib.cache_attention_forward(q, cache_, cache_, t((1, 3), O.I32), t((2,), O.I32), t((1,), O.I32), q,
                                    ctypes.byref(Op.CCacheAttentionParams(0.0, 0, 0)), P)
    assert b"overlaps" in rec.lib.tensor_ops_hip_last_error()
    x, y, kv = t((4, 6 * 64), O.F16), t((4, 2, 64), O.F16), t((4, 2, 64), O.F16)
    rec.lib.qk_norm_rotary_forward(x, P, P, P, P, P, P, y, kv, kv, ctypes.byref(Op.CQKNormRotaryParams(2, 2, 0.0, 0)))
    assert b"must not overlap" in rec.lib.tensor_ops_hip_last_error()


def test_indices_tables_and_workspaces_overlap_nothing(rec):
    t, P = rec.tensor, O.PT()

    def alias(x, shape, dt):
        return rec.lib.tensor_wrap_device(x.contents.data, O._ints(shape), len(shape), dt)

    def refused(fn, *a):
        rec.lib.tensor_ops_hip_clear_error()
        getattr(rec.lib, fn)(*a)
        return b"overlap" in rec.lib.tensor_ops_hip_last_error()
    q, k, v, y = (t((2, 2, 5, 64), O.F16) for _ in range(4))
    p = ctypes.byref(Op.CAttentionParams(0, 0, 0.0, 0))
    assert refused("attention_forward", q, k, v, P, alias(y, (2,), O.I32), y, p, P)
    for x in (q, k, v, y):
        assert refused("attention_forward", q, k, v, P, P, y, p, alias(x, (64,), O.U8))
    assert not refused("attention_forward", q, k, v, P, P, y, p, t((64,), O.U8))
    q, kc, vc, y = t((4, 2, 64), O.F16), t((3, 2, 4, 64), O.F16), t((3, 2, 4, 64), O.F16), t((4, 2, 64), O.F16)
    ix = [t((1, 3), O.I32), t((2,), O.I32), t((1,), O.I32)]
    p = ctypes.byref(Op.CCacheAttentionParams(0.0, 0, 0))
    for i, shape in enumerate(((1, 3), (2,), (1,))):
        on = list(ix)
        on[i] = alias(y, shape, O.I32)
        assert refused("cache_attention_forward", q, kc, vc, *on, y, p, P)
    for x in (q, kc, vc, *ix, y):
        assert refused("cache_attention_forward", q, kc, vc, *ix, y, p, alias(x, (4,), O.U8))
    assert not refused("cache_attention_forward", q, kc, vc, *ix, y, p, t((64,), O.U8))
    x, y, k, v = t((4, 6 * 64), O.F16), t((4, 2, 64), O.F16), t((4, 2, 64), O.F16), t((4, 2, 64), O.F16)
    w, cos, sin, pos = t((64,), O.F16), t((9, 32), O.F16), t((9, 32), O.F16), t((4,), O.I32)
    p = ctypes.byref(Op.CQKNormRotaryParams(2, 2, 0.0, 0))
    assert not refused("qk_norm_rotary_forward", x, w, w, cos, sin, pos, P, y, k, v, p)
    for out in (y, k, v):
        for i, (shape, dt) in enumerate((((64,), O.F16), ((64,), O.F16), ((2, 32), O.F16), ((2, 32), O.F16), ((4,), O.I32))):
            ins = [w, w, cos, sin, pos]
            ins[i] = alias(out, shape, dt)
            if i in (2, 3):                    # both tables of one shape
                ins[5 - i] = t(shape, dt)
            assert refused("qk_norm_rotary_forward", x, *ins, P, y, k, v, p)


def test_too_many_keys(rec):
    big = (1, 1, (1 << 31) - 100, 8)
    launches, err = attn(rec, q=(1, 1, 1, 8), k=big, v=big)
    assert "2^31 keys" in err and not launches
