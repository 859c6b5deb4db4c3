"""cache_plan_forward on the GPU against a restatement that goes request by request."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import oracle as O
from tests.decode_ref import Dev, PlanProblem

pytestmark = pytest.mark.gpu


def requests(b, n_hi, past_hi, ended=0, seed=0):
    rng = np.random.default_rng(seed)
    new = rng.integers(0, n_hi + 1, b)
    if ended:
        new[rng.random(b) < ended] = -1
    return list(zip(new.tolist(), rng.integers(0, past_hi + 1, b).tolist()))


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("b", [1, 2, 63, 64, 65, 500])
def test_sizes(hip, b, page, index):
    PlanProblem(requests(b, 5, 200, ended=0.2, seed=b), page, spare=3000, seed=b, offset=17).check(hip, index=index)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,n", [(1023, 1), (1024, 2), (1025, 3), (2500, 2), (3000, 9)])
def test_more_requests_than_threads(hip, b, n, in_place):
    PlanProblem(requests(b, n, 60, ended=0.1, seed=n), 8, spare=6000, seed=b).check(hip, in_place=in_place)


@pytest.mark.parametrize("new", [[9000], [0, 5000, 0], [4096, 0, 1], [4097], [1] * 70 + [5000] + [0, 1] * 50, [300] * 40])
def test_many_tokens(hip, new):
    """Prompts of one launch and of two, among single tokens and requests without any."""
    rng = np.random.default_rng(len(new))
    p = PlanProblem([(n, int(rng.integers(0, 40))) for n in new], 16, spare=sum(new) // 16 + 2 * len(new), seed=1, offset=1000,
                    rows=sum(new) + 77)
    p.check(hip)


@pytest.mark.parametrize("spare", [0, 1, 7, 8, 30, 31, 32])
@pytest.mark.parametrize("big", [False, True])
def test_too_few_pages(hip, spare, big):
    """The first request whose pages are not all there and those behind it that need some take none."""
    new = [16, 33, 0, 100, 1, 5, -1, 64, 3]
    past = [0, 15, 7, 16, 16, 12, 40, 0, 13]
    p = PlanProblem(list(zip(new, past)), 16, spare=spare, seed=spare, rows=6000 if big else 400)
    got = p.check(hip)
    # needs, added up: 1, 3, 3, 10, 11, 12, -, 16, 16, of the ring's and three that come back
    assert got[6][2] == {0: 4, 1: 4, 7: 3, 8: 2}.get(spare, 0)


def test_returned_pages_are_taken_in_the_same_step(hip):
    """An empty ring: what ended requests give back is all there is, a later one's pages too."""
    p = PlanProblem([(40, 0), (-1, 100), (1, 16), (-1, 33), (16, 16)], 16, spare=0, seed=3)
    got = p.check(hip)
    assert got[6][2] == 0 and got[6][0] - p.state[0] == 5


def test_rows_that_are_short(hip):
    """Requests whose table row or whose rows of tokens end too soon are refused."""
    p = PlanProblem([(5, 10), (40, 10), (3, 31), (2, 0), (50, 0)], 16, cols=2, spare=20, rows=49)
    got = p.check(hip)
    assert got[6][2] == 4                            # all but the first


def test_many_refused_over_several_rounds(hip):
    """More requests than threads and pages for some of them only."""
    PlanProblem([(16, 0)] * 3000, 16, spare=1500, rows=48000).check(hip)
    PlanProblem([(1, 16 * (i % 3)) for i in range(3000)], 16, spare=1200, seed=1).check(hip)


@pytest.mark.parametrize("pad", [0, 1, 100, 9000])
def test_rows_behind_the_last_request(hip, pad):
    reqs = requests(20, 4, 50, seed=4)
    PlanProblem(reqs, 16, rows=sum(max(n, 0) for n, _ in reqs) + pad).check(hip)


def test_no_requests(hip):
    got = PlanProblem([], 16, rows=5).check(hip)
    assert (got[2] == -1).all() and got[0].tolist() == [0]


def test_types_of_their_own(hip):
    p = PlanProblem(requests(30, 6, 50, ended=0.2, seed=5), 16, spare=100, offset=5)
    for index in ("int32", "int64"):
        for out in ("int32", "int64"):
            p.check(hip, index=index, out=out)


def test_places_that_the_type_does_not_hold(hip):
    """A position past int32 makes the token one to be left out; int64 holds it."""
    p = PlanProblem([(3, 5)], 16, offset=(1 << 31) - 7)
    with Dev(hip) as dev:
        from onnx_translator_amd.nn.Operators import CCachePlanParams
        put = lambda x, dt="int64": dev.put(np.asarray(x).astype(dt))      # noqa: E731
        outs = [put([0, 0], "int32"), put([0], "int32"), put([9] * 3, "int32"), put([9] * 3, "int32")]
        state = put(p.state)
        dev.call("cache_plan_forward", put(p.new), put(p.past), put([p.offset]), state, put(p.pages), put(p.free), *outs, state,
                 ctypes.byref(CCachePlanParams(16)))
        pos, slots = (hip.dev_read(t, O.I32) for t in outs[2:])
    assert pos.tolist() == [(1 << 31) - 2, (1 << 31) - 1, -1] and slots[2] == -1 and (slots[:2] >= 0).all()
    got = p.check(hip, index="int64")
    assert got[2].tolist() == [(1 << 31) - 2, (1 << 31) - 1, 1 << 31]


def test_a_state_that_no_ring_has(hip):
    """Counts the wrong way round, negative, or more than the ring holds: nothing is taken, nothing
    is given back, the lengths of requests that need no page grow."""
    for state in ((9, 5), (-3, 2), (0, 1000)):
        p = PlanProblem([(1, 3), (20, 3), (-1, 40)], 16, spare=10)
        p.state[:2] = state
        got = p.run(hip)
        assert got[1].tolist() == [4, 3, 0] and got[6].tolist() == [*state, 1]
        assert (got[4] == p.pages).all() and (got[5] == p.free).all()


def test_lengths_that_no_request_has(hip):
    """Past tokens below zero count as none, more than the table's row as refused; a count of new
    tokens past any length is refused."""
    p = PlanProblem([(4, 0), (2, 0), (1, 0), (3, 0)], 16, cols=4, spare=10, rows=20)
    p.past[:] = [-5, 1000, 0, 0]
    p.new[:] = [4, 2, 1 << 40, 3]
    got = p.run(hip, index="int64")
    assert got[1].tolist() == [4, 1000, 0, 0] and got[6][2] == 3
    assert got[0].tolist() == [0, 4, 6, 20, 20] and got[2].tolist() == [0, 1, 2, 3] + [-1] * 16


def test_a_service(hip):
    """Steps of a service with its lengths, table, ring and state on the device all along, as a
    captured step replayed: requests come, grow and end, no page is ever in two hands, and the ring
    holds the rest."""
    lib = hip.lib
    with Dev(hip):
        pass
    from onnx_translator_amd.nn.Operators import CCachePlanParams
    rng = np.random.default_rng(0)
    b, cols, page, rows, pages = 24, 8, 4, 256, 90
    side = torch.cuda.Stream()
    ints = lambda v: torch.as_tensor(np.asarray(v), dtype=torch.int32, device="cuda")      # noqa: E731
    t = dict(new=ints(np.zeros(b)), past=ints(np.zeros(b)), state=torch.tensor([0, pages, 0], device="cuda"),
             pages=ints(np.full((b, cols), -1)), free=ints(np.arange(pages)), start=ints(np.zeros(b + 1)),
             pos=ints(np.zeros(rows)), slots=ints(np.zeros(rows)))
    code = {torch.int32: O.I32, torch.int64: O.I64}
    w = {k: lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * x.dim())(*x.shape), x.dim(), code[x.dtype])
         for k, x in t.items()}
    prm = CCachePlanParams(page)

    def call():
        lib.cache_plan_forward(w["new"], w["past"], O.PT(), w["state"], w["pages"], w["free"], w["start"], w["past"], w["pos"],
                               w["slots"], w["state"], ctypes.byref(prm))
        assert not lib.tensor_ops_hip_last_error()

    lib.tensor_ops_hip_set_stream(ctypes.c_void_p(side.cuda_stream))
    try:
        with torch.cuda.stream(side):
            call()                                   # nobody brings anything
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call()
            from tests.decode_ref import plan
            refused = 0
            for step in range(60):
                past, table, free, state = (t[k].cpu().numpy() for k in ("past", "pages", "free", "state"))
                new = np.where(past == 0, rng.integers(0, 20, b) * (rng.random(b) < 0.3), rng.integers(0, 3, b))
                new[(rng.random(b) < 0.08) & (past > 0)] = -1
                t["new"].copy_(ints(new))
                torch.cuda.synchronize()
                g.replay() if step % 3 else call()
                torch.cuda.synchronize()
                want = plan(new, past, table, free, state, rows, page)
                for k, x in zip(("start", "past", "pos", "slots", "pages", "free", "state"), want):
                    assert (t[k].cpu().numpy() == x).all(), (step, k)
                refused += int(want[6][2])
                # each page in one hand
                past, table, free, state = (t[k].cpu().numpy() for k in ("past", "pages", "free", "state"))
                held = [int(table[i, c]) for i in range(b) for c in range(-(-int(past[i]) // page))]
                held += [int(free[i % pages]) for i in range(int(state[0]), int(state[1]))]
                assert sorted(held) == list(range(pages)), step
            assert refused > 0
    finally:
        torch.cuda.synchronize()
        for p in w.values():
            lib.free_tensor(p)
        lib.tensor_ops_hip_set_stream(None)


def test_nearly_all_that_an_int32_counts_comes_back(hip):
    """One request gives 2^31 - 2 pages back: the places behind the last do not wrap around."""
    from onnx_translator_amd.nn.Operators import CCachePlanParams
    n, taken = (1 << 31) - 2, 5
    pages = torch.arange(n, dtype=torch.int32, device="cuda")
    free = torch.full((n + 1,), -3, dtype=torch.int32, device="cuda")
    small = [torch.tensor(x, dtype=dt, device="cuda") for x, dt in
             (([-1], torch.int32), ([n], torch.int32), ([taken, taken, 0], torch.int64), ([7, 7], torch.int32), ([7], torch.int32),
              ([7, 7], torch.int32), ([7, 7], torch.int64), ([0, 0, 0], torch.int64))]
    torch.cuda.synchronize()
    new, past, state, start, length, pos, slots, after = small
    with Dev(hip) as dev:
        def wrap(x, shape=None):
            shape = shape or tuple(x.shape)
            dev.held.append(hip.lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * len(shape))(*shape), len(shape),
                                                       O.I32 if x.dtype == torch.int32 else O.I64))
            return dev.held[-1]
        dev.call("cache_plan_forward", wrap(new), wrap(past), O.PT(), wrap(state), wrap(pages, (1, n)), wrap(free), wrap(start), wrap(length),
                 wrap(pos), wrap(slots), wrap(after), ctypes.byref(CCachePlanParams(1)))
        torch.cuda.synchronize()
    assert after.tolist() == [taken, taken + n, 0] and length.tolist() == [0] and start.tolist() == [0, 0]
    assert pos.tolist() == slots.tolist() == [-1, -1]
    assert torch.equal(free[taken:], pages[:n + 1 - taken]) and torch.equal(free[:taken - 1], pages[n + 1 - taken:]) and int(free[taken - 1]) == -3
