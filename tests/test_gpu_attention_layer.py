"""The attention operators as a program runs them: one after the other with the Gemm before them,
from an ONNX model, on host tensors, captured into graphs, on several streams and threads."""
import ctypes
import threading

import numpy as np
import pytest
import torch

from oracle import oracle as O
from onnx_translator_amd.nn import DeviceArray, Ops, Tensor
from onnx_translator_amd.nn import Operators as Op
from tests.attention_ref import HALF_STEP, U, CacheProblem, DenseProblem, Dev, attend, cast, check

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    a = np.asarray(a)
    return Tensor(*a.shape, dtype=dtype or str(a.dtype), data=np.ascontiguousarray(a)).to_device()


@pytest.mark.parametrize("dtype", ("float16", "float32"))
def test_a_layer_over_a_cache(hip, dtype):
    """Gemm -> QKNormRotary -> CacheAttention, a prompt in two chunks beside another sequence's
    single tokens, then single tokens of both: every call against float64 on its own inputs, and
    the cache in the end what one pass over all tokens gives."""
    rng = np.random.default_rng(0)
    hidden, hq, hkv, d, page = 96, 6, 2, 64, 16
    heads = hq + 2 * hkv
    np_dt = np.float16 if dtype == "float16" else np.float32
    w = dev(rng.normal(0, 0.1, (heads * d, hidden)).astype(np_dt))
    wq, wk = (dev((1 + rng.normal(0, 0.1, d)).astype(np_dt)) for _ in range(2))
    angle = np.arange(128)[:, None] * 100.0 ** (-np.arange(0, d, 2) / d)
    cos, sin = dev(np.cos(angle).astype(np.float32)), dev(np.sin(angle).astype(np.float32))
    kc, vc = (dev(np.full((12, hkv, page, d), np.nan, np_dt)) for _ in range(2))
    pages = np.array([[7, 2, 11, 0], [4, 9, 1, 5]], np.int32)
    x = [rng.normal(0, 1, (n, hidden)).astype(np_dt) for n in (45, 6)]       # both sequences' tokens
    gemm = Op.Gemm([], [], 1.0, 0.0, 0, 1, dtype)
    rotary, attention = Op.QKNormRotary([], [], hq, hkv), Op.CacheAttention([], [], max_kv=64)
    done, outs, qkvs = [0, 0], [[], []], [[], []]
    for take in ((30, 1), (13, 1), (1, 1), (1, 1), (0, 2)):
        rows = np.concatenate([x[b][done[b]:done[b] + n] for b, n in enumerate(take)])
        pos = np.concatenate([np.arange(done[b], done[b] + n) for b, n in enumerate(take)]).astype(np.int32)
        seq = np.repeat([0, 1], take)
        slots = (pages[seq, pos // page] * page + pos % page).astype(np.int32)
        qkv = gemm.forward(dev(rows), w)["tensor"]
        q, k2, v2 = rotary.forward(qkv, wq, wk, cos, sin, dev(pos), kc, vc, dev(slots))["tensor"]
        assert k2 is kc and v2 is vc
        done = [a + n for a, n in zip(done, take)]
        start = np.array([0, take[0], sum(take)], np.int32)
        y = attention.forward(q, kc, vc, dev(pages), dev(start), dev(np.array(done, np.int32)))["tensor"].numpy().astype(np.float64)
        q64, k64, v64 = (t.numpy().astype(np.float64) for t in (q, kc, vc))
        for b, n in enumerate(take):
            if not n:
                continue
            j = np.arange(done[b])
            seen = j <= done[b] - n + np.arange(n)[:, None]
            for h in range(hq):
                at = (pages[b, j // page], h // 3, j % page)
                ref, tol = attend(q64[start[b]:start[b + 1], h], k64[at], v64[at], d ** -0.5, seen, dtype=dtype)
                check(y[start[b]:start[b + 1], h], ref, tol, f"{take} {b} {h}")
            outs[b].append(y[start[b]:start[b + 1]])
            qkvs[b].append(qkv.numpy().astype(np.float64)[start[b]:start[b + 1]])
    assert done == [45, 6]
    # the cache: keys normed and rotated, values as they were, nothing else touched
    k64, v64 = kc.numpy().astype(np.float64), vc.numpy().astype(np.float64)
    wk64, c, s = (t.numpy().astype(np.float64) for t in (wk, cos, sin))
    for b in range(2):
        all_ = np.concatenate(qkvs[b]).reshape(-1, heads, d)
        j = np.arange(done[b])
        key = all_[:, hq:hq + hkv]
        key = key / np.sqrt((key ** 2).mean(-1, keepdims=True) + 1e-6) * wk64
        lo, hi = key[..., :d // 2], key[..., d // 2:]
        cc, ss = c[j][:, None], s[j][:, None]
        want = np.concatenate([lo * cc - hi * ss, lo * ss + hi * cc], -1)
        size = np.concatenate([np.abs(lo * cc) + np.abs(hi * ss), np.abs(lo * ss) + np.abs(hi * cc)], -1)
        tol = HALF_STEP[dtype] * np.abs(want) + (d / 2 + 12) * U * size * (1 + 2.0 ** -7) + (2.0 ** -24 if dtype == "float16" else 0)
        check(k64[pages[b, j // page], :, j % page], want, tol, "keys")
        assert (v64[pages[b, j // page], :, j % page] == all_[:, hq + hkv:]).all()
    assert np.isnan(k64).sum() == (12 * page - 51) * hkv * d == np.isnan(v64).sum()


def test_onnx_model(hip):
    """An Attention node with a bool mask and shared heads, its queries from a graph's Relu: on the
    device, on the host, and by shape propagation."""
    from onnx_translator_amd.nn.ONNXImport import load_graph
    from onnx_translator_amd.onnx import proto as P
    p = DenseProblem(2, 4, 2, 9, 33, 64, "float32", mask=np.random.default_rng(1).random((2, 1, 9, 33)) < 0.7, packed=True)
    p.q64 = np.maximum(p.q64, 0)
    ins = [p._laid(t).numpy() for t in (p.q, p.k, p.v)]
    names = ["q", "k", "v"]
    nodes = [P.NodeProto("Relu", ["q"], ["r"]),
             P.NodeProto("Attention", ["r", "k", "v", "m"], ["y"], attributes=[P.make_attribute("q_num_heads", 4), P.make_attribute("kv_num_heads", 2)])]
    g = P.GraphProto(nodes=nodes, name="g", inputs=[P.ValueInfoProto(n, P.FLOAT, list(a.shape)) for n, a in zip(names, ins)],
                     outputs=[P.ValueInfoProto("y", P.FLOAT, [2, 9, 256])], initializers=[P.TensorProto.from_numpy(p.mask, "m", 2)])
    model = P.ModelProto(graph=g)
    ref, tol = p.reference()
    for device in (True, False):
        y = load_graph(model, device=device).forward(*ins)
        assert y.on_device == device
        check(y.numpy().reshape(2, 9, 4, 64).transpose(0, 2, 1, 3), ref, tol, str(device))


@pytest.mark.parametrize("dtype", ("float16", "float32"))
def test_host_tensors(hip, dtype):
    p = DenseProblem(2, 4, 2, 5, 70, 64, dtype, lengths=[70, 12], seed=2)
    ins = [Tensor(*t.shape, dtype=dtype, data=t.numpy()) for t in (p.q, p.k, p.v)]
    y = Op.Attention([], []).forward(*ins, None, Tensor(2, dtype="int64", data=p.lengths.astype(np.int64)))["tensor"]
    assert not y.on_device
    ref, tol = p.reference()
    check(y.data, ref, tol)


def test_bool_mask_of_numpy(hip):
    m = np.random.default_rng(3).random((5, 40)) < 0.5
    p = DenseProblem(1, 2, 2, 5, 40, 64, "float32", mask=m, seed=3)
    ins = [Tensor(*t.shape, dtype="float32", data=t.numpy()).to_device() for t in (p.q, p.k, p.v)]
    y = Op.Attention([], []).forward(*ins, Tensor(5, 40, dtype="bool", data=m).to_device())["tensor"]
    ref, tol = p.reference()
    check(y.numpy(), ref, tol)


class Step:
    """A decode step on torch memory: rotary into the cache, attention over it."""

    def __init__(self, lib, b, workspace, seed=0, cap=512):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lib, self.held, self.b = lib, [], b
        hq, hkv, d, page = 8, 2, 64, 16
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()      # noqa: E731
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")        # noqa: E731
        per = cap // page
        self.t = dict(qkv=rand(b, (hq + 2 * hkv) * d), q=rand(b, hq, d), k=rand(b * per, hkv, page, d), v=rand(b * per, hkv, page, d),
                      cos=torch.rand(cap, d // 2, generator=g, device="cuda"), sin=torch.rand(cap, d // 2, generator=g, device="cuda"),
                      pos=ints([100 + 30 * i for i in range(b)]), slots=ints([0] * b),
                      pages=torch.arange(b * per, dtype=torch.int32, device="cuda").reshape(b, per), start=ints(list(range(b + 1))),
                      len=ints([0] * b), y=rand(b, hq, d))
        if workspace:
            self.t["ws"] = torch.empty(workspace, dtype=torch.uint8, device="cuda")
        self.cap, self.g = cap, g
        self.p1, self.p2 = Op.CQKNormRotaryParams(hq, hkv, 1e-6, 0), Op.CCacheAttentionParams(0.0, 0, cap)
        name = {torch.float16: O.F16, torch.float32: O.F32, torch.int32: O.I32, torch.uint8: O.U8}
        self.w = {}
        for k, x in self.t.items():
            self.w[k] = lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * x.dim())(*x.shape), x.dim(), name[x.dtype])
        self.set_positions()

    def set_positions(self):
        t = self.t
        t["slots"].copy_(t["pages"].gather(1, (t["pos"] // 16).long()[:, None])[:, 0] * 16 + t["pos"] % 16)
        t["len"].copy_(t["pos"] + 1)

    def advance(self):
        self.t["pos"].add_(1)
        self.t["qkv"].copy_(torch.randn(self.t["qkv"].shape, generator=self.g, device="cuda"))
        self.set_positions()

    def run(self):
        w, none = self.w, O.PT()
        self.lib.qk_norm_rotary_forward(w["qkv"], none, none, w["cos"], w["sin"], w["pos"], w["slots"], w["q"], w["k"], w["v"], ctypes.byref(self.p1))
        assert not self.lib.tensor_ops_hip_last_error(), self.lib.tensor_ops_hip_last_error()
        self.lib.cache_attention_forward(w["q"], w["k"], w["v"], w["pages"], w["start"], w["len"], w["y"], ctypes.byref(self.p2), w.get("ws", none))
        assert not self.lib.tensor_ops_hip_last_error(), self.lib.tensor_ops_hip_last_error()

    def free(self):
        for p in self.w.values():
            self.lib.free_tensor(p)


def _lib(hip):
    with Dev(hip):
        pass                                    # the signatures
    return hip.lib


@pytest.mark.parametrize("workspace", [0, 1 << 22])
def test_captured_steps(hip, workspace):
    """A decode step captured once and replayed with positions, lengths and projections rewritten
    on the device: every replay equals the eager step on the same state.  (Without a workspace
    the captured attention does not split the keys, another order of the same sums.)"""
    lib = _lib(hip)
    side = torch.cuda.Stream()
    lib.tensor_ops_hip_set_stream(ctypes.c_void_p(side.cuda_stream))
    s = Step(lib, 3, workspace)
    try:
        with torch.cuda.stream(side):
            s.run()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                s.run()
            for r in range(5):
                s.advance()
                s.t["y"].fill_(float("nan"))
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                replayed = {k: s.t[k].clone() for k in ("q", "k", "v", "y")}
                s.run()                          # eager, on the same state
                torch.cuda.synchronize()
                for k in ("q", "k", "v"):
                    assert torch.equal(replayed[k], s.t[k]), (r, k)
                if workspace:
                    assert torch.equal(replayed["y"], s.t["y"]), r
                else:                            # one half step of each side, and of each side's weights
                    assert torch.allclose(replayed["y"].float(), s.t["y"].float(), rtol=2.0 ** -9, atol=2.0 ** -9), r
                assert torch.isfinite(replayed["y"]).all()
    finally:
        torch.cuda.synchronize()
        s.free()
        lib.tensor_ops_hip_set_stream(None)


def test_two_graphs_with_their_own_workspaces(hip):
    """Two captured steps replayed at once on two streams: each keeps its own workspace."""
    lib = _lib(hip)
    streams = [torch.cuda.Stream() for _ in range(2)]
    steps = [Step(lib, 4, 1 << 22, seed=i) for i in range(2)]
    graphs = []
    try:
        for st, s in zip(streams, steps):
            lib.tensor_ops_hip_set_stream(ctypes.c_void_p(st.cuda_stream))
            with torch.cuda.stream(st):
                s.run()
                torch.cuda.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    s.run()
                graphs.append(g)
        want = [s.t["y"].clone() for s in steps]
        torch.cuda.synchronize()
        for _ in range(10):
            for s in steps:
                s.t["y"].zero_()
            torch.cuda.synchronize()
            for st, g in zip(streams, graphs):
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for s, w in zip(steps, want):
                assert torch.equal(s.t["y"], w)
    finally:
        torch.cuda.synchronize()
        for s in steps:
            s.free()
        lib.tensor_ops_hip_set_stream(None)


def test_threads_on_their_own_streams(hip):
    """Two threads, a stream each, the library's pool for their workspaces."""
    lib = _lib(hip)
    steps = [Step(lib, 4, 0, seed=i) for i in range(2)]
    for s in steps:
        s.run()
    torch.cuda.synchronize()
    lib.tensor_ops_hip_sync()
    want = [s.t["y"].clone() for s in steps]
    torch.cuda.synchronize()
    failed = []

    def work(s, w):
        try:
            st = torch.cuda.Stream()
            lib.tensor_ops_hip_set_thread_stream(ctypes.c_void_p(st.cuda_stream))
            for _ in range(30):
                with torch.cuda.stream(st):
                    s.t["y"].zero_()
                    s.run()
                st.synchronize()
                if not torch.equal(s.t["y"], w):
                    failed.append(s)
                    break
            lib.tensor_ops_hip_set_thread_stream(None)
        except Exception as e:                  # noqa: BLE001
            failed.append(e)

    lib.tensor_ops_hip_set_thread_stream.argtypes = [ctypes.c_void_p]
    threads = [threading.Thread(target=work, args=a) for a in zip(steps, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for s in steps:
        s.free()
    assert not failed, failed


def test_repeatable(hip):
    """The same call gives the same bits: sums are joined in a fixed order."""
    for p in (DenseProblem(2, 4, 2, 1, 1500, 64, "float16"), DenseProblem(1, 4, 2, 100, 900, 64, "float32")):
        a = p.run(hip)
        for _ in range(5):
            assert (p.run(hip) == a).all()
    c = CacheProblem([(1, 1500), (60, 300)], 8, 2, 64, 16, "bfloat16")
    a = c.run(hip)
    for _ in range(5):
        assert (c.run(hip) == a).all()
