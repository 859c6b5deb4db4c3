"""prefix_cache_attention_forward on the GPU against float64 (tests/decode_ref.py)."""
import numpy as np
import pytest

from tests.attention_ref import HALF_STEP, CacheProblem
from tests.decode_ref import PrefixProblem

pytestmark = pytest.mark.gpu

TYPES = ("float16", "bfloat16", "float32")
SEQS = [(1, 1), (1, 37), (3, 3), (20, 45), (1, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 20, 33, 40, 64, 80, 96, 128, 192, 256, 300])
def test_head_sizes(hip, d, dtype):
    PrefixProblem(SEQS, 75, 4, 2, d, 16, dtype, seed=d).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,dv", [(64, 128), (128, 64), (96, 40), (33, 8)])
def test_value_size_of_its_own(hip, d, dv, dtype):
    PrefixProblem(SEQS, 50, 2, 1, d, 16, dtype, dv=dv, seed=d).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shared", [0, 1, 15, 16, 17, 31, 32, 33, 64, 127, 129, 500, 1500])
def test_prefix_lengths(hip, shared, dtype):
    PrefixProblem(SEQS, shared, 4, 2, 64, 16, dtype, seed=shared).check(hip)


@pytest.mark.parametrize("dtype", ("float16", "float32"))
@pytest.mark.parametrize("seqs", [[(1, 1)], [(1, 1500)], [(1, 1)] * 70, [(64, 64)], [(0, 0), (1, 5), (0, 9), (2, 2), (0, 0)],
                                  [(130, 600), (1, 1), (7, 300)], [(300, 300)]], ids=lambda s: str(s)[:30])
def test_sequences(hip, seqs, dtype):
    PrefixProblem(seqs, 333, 4, 2, 64, 16, dtype, seed=len(seqs)).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (7, 1), (12, 4), (40, 1)])
def test_shared_heads(hip, hq, hkv, dtype):
    PrefixProblem(SEQS, 70, hq, hkv, 64, 16, dtype, seed=hq).check(hip)


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("page", [1, 2, 3, 8, 24, 64, 128])
def test_page_sizes(hip, page, dtype):
    PrefixProblem(SEQS, 200, 4, 2, 64, page, dtype, seed=page).check(hip)


@pytest.mark.parametrize("tokens", [1, 5, 16, 33, 63, 64, 65, 127, 128, 200, 520])
def test_batches_of_single_tokens(hip, tokens):
    """From a wave's rows to several tiles of the batch's rows, whatever sequences they are of."""
    PrefixProblem([(1, 1 + i % 40) for i in range(tokens)], 700, 4, 1, 64, 16, "bfloat16", seed=tokens).check(hip, heads=(0, 3))


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
def test_blocks_of_256_rows(hip, dtype):
    """Enough rows that the prefix is read by blocks of eight waves."""
    PrefixProblem([(128, 128 + i) for i in range(16)], 4001, 64, 16, 64, 16, dtype, std=0.7).check(hip, heads=(37,))


@pytest.mark.parametrize("index", ["int32", "int64"])
def test_index_types(hip, index):
    PrefixProblem(SEQS, 90, 4, 2, 64, 16, "float16").check(hip, index=index)


@pytest.mark.parametrize("said", [dict(max_kv=1, max_prefix=1), dict(max_kv=45, max_prefix=1300), dict(max_kv=1 << 30, max_prefix=1 << 30)])
def test_what_the_caller_knows_shapes_only_the_launch(hip, said):
    PrefixProblem(SEQS, 1300, 4, 2, 64, 16, "float16", spare_columns=100, spare_prefix=300).check(hip, **said)


@pytest.mark.parametrize("dtype", ("float16", "float32"))
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 1000])
def test_workspaces(hip, splits, dtype):
    """Of one split (too small, the pool serves), of some, of more than are used."""
    p = PrefixProblem(SEQS, 1300, 4, 2, 64, 16, dtype)
    p.check(hip, workspace=splits * 26 * 4 * (64 * 4 + 8))


def test_rows_of_no_sequence(hip):
    """Rows before the first and behind the last sequence hold NaN and are left as they were."""
    for d in (64, 20):
        PrefixProblem(SEQS, 80, 4, 2, d, 16, "float16", pad_rows=9, skip_rows=5).check(hip)


@pytest.mark.parametrize("d", [64, 20])
def test_lengths_past_the_tables(hip, d):
    """Lengths are cut to what the tables can name, and below zero to none."""
    p = PrefixProblem([(1, 40), (2, 20), (1, 9)], 90, 4, 2, d, 16, "float16", spare_columns=0, spare_prefix=0)
    p.len[0] = 10000
    p.shared = 96                                    # the last page's places behind the prefix: NaN unless filled
    last = p.prefix_pages[-1]
    for c, c64 in ((p.k, p.k64), (p.v, p.v64)):
        c[last] = 1.0
        c64[last] = 1.0
        for b in (0,):
            c[p.pages[b, -1]] = 0.5
            c64[p.pages[b, -1]] = 0.5
    p.check(hip)
    more = PrefixProblem([(1, 40), (2, 20), (1, 9)], 96, 4, 2, d, 16, "float16", spare_prefix=0)
    want = more.check(hip)
    more.shared = 1 << 30
    assert (more.run(hip) == want).all()
    none = PrefixProblem([(1, 40), (2, 20)], 0, 4, 2, d, 16, "float16")
    want = none.check(hip)
    none.shared = -5
    assert (none.run(hip) == want).all()


@pytest.mark.parametrize("d", [64, 20])
def test_tokens_before_their_sequence(hip, d):
    """More new tokens than keys (a refused request's): those in front see the prefix alone."""
    p = PrefixProblem([(3, 5), (4, 6)], 50, 4, 2, d, 16, "float16")
    p.len[:] = [1, 0]
    p.check(hip)
    p = PrefixProblem([(3, 5)], 0, 4, 2, d, 16, "float16")
    p.len[:] = [1]
    got = p.check(hip)
    assert not got[:2].any() and got[2].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_missing_pages(hip, dtype):
    """Keys on pages that the cache does not have are not seen, of the prefix or of a sequence."""
    p = PrefixProblem(SEQS + [(2, 70)], 150, 4, 2, 64, 16, dtype)
    p.prefix_pages[[0, 5]] = [-1, 10 ** 6]
    p.pages[3, 1] = 10 ** 6
    p.pages[5, 0] = -4
    p.check(hip)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(hip, dtype):
    """One part's weights may all vanish beside the other's."""
    p = PrefixProblem([(2, 30), (1, 1)], 64, 2, 2, 64, 16, dtype, std=4.0)
    p.check(hip)


@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_value_nobody_sees(hip, dtype):
    p = PrefixProblem([(2, 30), (5, 5)], 40, 2, 1, 64, 16, dtype)
    v = p.pages[1, 0]
    p.v[v, :, 5:] = np.inf                           # behind the second sequence's keys
    p.k[v, :, 5:] = np.inf
    p.check(hip)


def test_equal_to_a_cache_without_sharing(hip):
    """The same keys as sequences of their own through cache_attention_forward: within the half steps
    of both."""
    dtype, d = "float16", 64
    p = PrefixProblem([(3, 20), (1, 48)], 64, 4, 2, d, 16, dtype)
    a = p.check(hip)
    c = CacheProblem([(3, 84), (1, 112)], 4, 2, d, 16, dtype)
    for b in range(2):
        own = [p.pages[b, i] for i in range(-(-p.seqs[b][1] // 16))]
        for i, page in enumerate(list(p.prefix_pages[:4]) + own):
            c.k[c.pages[b, i]], c.v[c.pages[b, i]] = p.k[page], p.v[page]
    c.q = p.q
    e = c.run(hip)
    assert np.abs(a - e).max() <= 4 * HALF_STEP[dtype] * np.abs(e).max()


def test_repeatable(hip):
    p = PrefixProblem([(1, 30 + i) for i in range(40)], 1500, 8, 2, 64, 16, "bfloat16")
    a = p.run(hip)
    for _ in range(5):
        assert (p.run(hip) == a).all()


def test_past_32_bits(hip):
    """Pages whose elements lie past 2^31 in the cache."""
    import ctypes
    import torch
    from oracle import oracle as O
    from onnx_translator_amd.nn.Operators import CPrefixAttentionParams
    from tests.decode_ref import Dev
    hq, hkv, d, page = 4, 2, 128, 64
    p = PrefixProblem([(1, 70), (2, 130)], 200, hq, hkv, d, page, "float16")
    ref, tol = p.reference()
    pages = (1 << 31) // (hkv * page * d) + p.k.shape[0]
    k, v = (torch.zeros(pages, hkv, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    at = pages - p.k.shape[0]
    k[at:], v[at:] = p.k.cuda(), p.v.cuda()
    q, y = p.q.cuda(), torch.zeros(3, hq, d, dtype=torch.float16, device="cuda")
    ints = [torch.from_numpy(np.asarray(x, np.int32)).cuda() for x in
            (np.where(p.prefix_pages < p.k.shape[0], p.prefix_pages + at, -1), [200], np.where(p.pages >= 0, p.pages + at, -1), p.start, p.len)]
    torch.cuda.synchronize()
    with Dev(hip) as dev:
        w = [hip.lib.tensor_wrap_device(ctypes.c_void_p(x.data_ptr()), (ctypes.c_int * x.dim())(*x.shape), x.dim(),
                                        O.I32 if x.dtype == torch.int32 else O.F16) for x in (q, k, v, *ints, y)]
        dev.held += w
        dev.call("prefix_cache_attention_forward", *w, ctypes.byref(CPrefixAttentionParams(0.0, 0, 0)), O.PT())
        got = dev.get(w[-1], "float16")
    from tests.attention_ref import check
    check(got, ref, tol)
