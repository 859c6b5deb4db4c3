"""attention_forward and cache_attention_forward on the GPU against a float64 restatement
(tests/attention_ref.py, which derives the tolerance)."""
import numpy as np
import pytest

from tests.attention_ref import CacheProblem, DenseProblem

pytestmark = pytest.mark.gpu

TYPES = ("float16", "bfloat16", "float32")
SIZES = (8, 20, 33, 40, 64, 80, 96, 128, 192, 256, 300)


# ------------------------------------------------------------------- dense -------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", SIZES)
def test_head_sizes(hip, d, dtype):
    DenseProblem(2, 4, 2, 37, 75, d, dtype, seed=d).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,dv", [(64, 128), (128, 64), (96, 40), (16, 256), (33, 8)])
def test_value_size_of_its_own(hip, d, dv, dtype):
    DenseProblem(2, 2, 1, 19, 66, d, dtype, dv=dv, seed=d).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 2, 31, 32, 33, 130])
@pytest.mark.parametrize("skv", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 257])
def test_lengths(hip, sq, skv, dtype):
    DenseProblem(1, 2, 2, sq, skv, 64, dtype, seed=sq * 1000 + skv).check(hip)


@pytest.mark.parametrize("dtype", ("float16", "float32"))
@pytest.mark.parametrize("sq,skv", [(1, 1500), (1, 4099), (3, 1500), (17, 1025), (200, 700)])
def test_long_keys(hip, sq, skv, dtype):
    DenseProblem(2, 4, 2, sq, skv, 64, dtype, seed=skv).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 5), (6, 2), (7, 1), (12, 4), (40, 1)])
def test_shared_heads(hip, hq, hkv, dtype):
    DenseProblem(2, hq, hkv, 9, 70, 64, dtype, seed=hq).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq,skv", [(1, 5), (64, 64), (70, 33), (33, 140), (130, 130)])
def test_causal(hip, sq, skv, dtype):
    DenseProblem(2, 4, 2, sq, skv, 64, dtype, causal=True, seed=sq).check(hip)


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("sq", [1, 40])
def test_key_lengths(hip, sq, index):
    """Lengths of zero and one among them, and ones past the tensor (cut to it)."""
    p = DenseProblem(6, 4, 2, sq, 100, 64, "bfloat16", lengths=[0, 1, 64, 65, 100, 1000], seed=1)
    p.set_v((slice(1, 2), slice(None), slice(1, None)), np.nan)       # past the length: not seen
    p.set_k((slice(1, 2), slice(None), slice(1, None)), np.inf)
    got = p.check(hip, index=index)
    assert not got[0].any()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_packed_heads(hip, dtype, packed):
    DenseProblem(3, 6, 2, 21, 70, 40, dtype, packed=packed, lengths=[70, 3, 41], seed=2).check(hip)


MASKS = {"full": (3, 4, 37, 75), "heads": (3, 1, 37, 75), "batch": (1, 4, 37, 75), "keys": (1, 75), "one": (1,),
         "queries": (3, 1, 37, 1), "two": (37, 75)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["bool", "own", "float32"])
@pytest.mark.parametrize("shape", list(MASKS))
def test_masks(hip, shape, kind, dtype):
    rng = np.random.default_rng(len(shape))
    s = MASKS[shape]
    if kind == "bool":
        mask = rng.random(s) < 0.7
    else:
        mask = rng.normal(0, 1, s)
        mask[rng.random(s) < 0.3] = -np.inf
    DenseProblem(3, 4, 2, 37, 75, 64, dtype, mask=mask, mask_dtype=dtype if kind == "own" else "float32",
                 seed=3).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 33])
def test_rows_that_see_nothing(hip, sq, dtype):
    rng = np.random.default_rng(5)
    mask = rng.random((2, 1, sq, 130)) < 0.5
    mask[0, :, 0] = False
    mask[1, :, sq // 2] = False
    got = DenseProblem(2, 2, 1, sq, 130, 64, dtype, mask=mask, seed=4).check(hip)
    assert not got[0, :, 0].any() and not got[1, :, sq // 2].any()
    add = np.where(mask, 0.0, -np.inf)
    got = DenseProblem(2, 2, 1, sq, 130, 64, dtype, mask=add, seed=4).check(hip)
    assert not got[0, :, 0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_of_the_lowest_value(hip, dtype):
    """The type's lowest value closes a key next to open ones; a row of nothing else is the mean."""
    import torch
    from tests.attention_ref import TORCH
    low = torch.finfo(TORCH[dtype]).min
    rng = np.random.default_rng(6)
    mask = np.where(rng.random((1, 1, 34, 70)) < 0.5, 0.0, low)
    mask[0, 0, 3] = low
    # scores far below a step of the lowest value: a row of it alone has equal scores
    p = DenseProblem(1, 2, 1, 34, 70, 64, dtype, mask=mask, std=0.01 if dtype == "float16" else 1.0, seed=7)
    if dtype != "float16":
        p.mask64 = np.where(p.mask64 < -1e30, -1e30, p.mask64)     # the same weights, finite in float64
        ref, tol = p.reference()
        ref[0, :, 3], tol[0, :, 3] = p.v64[0, 0].mean(0), 2.0 ** -6 * np.abs(p.v64[0, 0]).mean(0)
    else:
        ref, tol = p.reference()
    from tests.attention_ref import check
    check(p.run(hip), ref, tol, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_masked_may_hold_anything(hip, value, dtype):
    """A key that is closed to some queries holds NaN or infinity: those rows do not notice."""
    mask = np.ones((1, 1, 40, 90), bool)
    mask[..., 17] = False
    mask[..., 20:, 71] = False
    p = DenseProblem(1, 2, 1, 40, 90, 64, dtype, mask=mask, seed=8)
    for set_ in (p.set_v, p.set_k):
        set_((0, 0, 17), value)
    p.set_v((0, 0, 71, slice(0, 5)), value)
    got = p.run(hip)
    ref, tol = p.reference()
    assert np.isfinite(got[0, :, 20:]).all()
    from tests.attention_ref import check
    check(got, ref, tol, f"{value} {dtype}")
    # later keys of a causal chunk
    p = DenseProblem(1, 2, 2, 70, 70, 64, dtype, causal=True, seed=9)
    p.set_v((0, slice(None), slice(40, None)), value)
    got = p.run(hip)
    assert np.isfinite(got[0, :, :40]).all() and not np.isfinite(got[0, :, 40:]).any()


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
def test_large_values_do_not_overflow(hip, dtype):
    """Values near the type's largest: their weighted mean is finite."""
    p = DenseProblem(1, 2, 1, 33, 200, 64, dtype, seed=10)
    p.v64[:] = np.sign(p.v64) * 3e38
    import torch
    from tests.attention_ref import TORCH, check
    p.v = torch.from_numpy(p.v64).to(TORCH[dtype])
    p.v64 = p.v.double().numpy()
    check(p.run(hip), *p.reference(), dtype)


def test_large_scores(hip):
    """Scores of thousands: one key takes everything, none overflows."""
    DenseProblem(1, 2, 1, 33, 200, 64, "float16", std=20.0, seed=11).check(hip)
    DenseProblem(1, 2, 1, 33, 200, 64, "bfloat16", std=1000.0, scale=1e-3, seed=12).check(hip)


# Enough blocks of 256 rows to fill the GPU twice over.
@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,skv,kw", [(40, 300, {}), (257, 129, dict(causal=True)), (40, 1, {}), (33, 70, dict(lengths=[0, 1, 70, 33, 64, 65, 2, 69])),
                                       (40, 131, dict(mask=True))], ids=["plain", "causal", "one key", "lengths", "mask"])
def test_many_blocks(hip, sq, skv, kw, d, dtype):
    kw = dict(kw)
    if kw.pop("mask", None):
        kw["mask"] = np.random.default_rng(1).random((8, 1, sq, skv)) < 0.6
    DenseProblem(8, 64, 64, sq, skv, d, dtype, seed=sq, **kw).check(hip, heads=[0, 31, 63])


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("page,window", [(16, 0), (3, 0), (64, 40)])
def test_cache_many_blocks(hip, page, window, dtype):
    seqs = [(40, 90), (1, 700), (257, 257), (3, 3), (130, 400), (0, 9), (64, 65), (33, 128)]
    CacheProblem(seqs, 64, 64, 128 if page == 16 else 64, page, dtype, window=window, seed=page, pad_rows=2).check(hip, heads=[0, 40, 63])


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page,window", [(1, 0), (1, 150), (2, 0)])
def test_cache_many_blocks_over_tiny_pages(hip, page, window, d, dtype):
    """A tile of keys on more pages than a wave holds numbers of, or just as many."""
    seqs = [(40, 90), (1, 700), (257, 257), (3, 3), (130, 400), (0, 9), (64, 65), (33, 128)]
    CacheProblem(seqs, 64, 64, d, page, dtype, window=window, seed=d, pad_rows=2).check(hip, heads=[0, 40, 63])


# More keys than a row has splits of two tiles, and than one register of page numbers.
@pytest.mark.parametrize("dtype,d", [("float16", 64), ("float32", 64), ("bfloat16", 256), ("float32", 256)])
def test_very_long_keys(hip, dtype, d):
    DenseProblem(1, 1, 1, 1, 20011, d, dtype, seed=1).check(hip)
    CacheProblem([(1, 9001), (1, 5)], 2, 1, d, 4, dtype, seed=2).check(hip)
    CacheProblem([(40, 5000)], 1, 1, d, 1, dtype, seed=2).check(hip)


# Rows and splits for each join: up to 16, 32 and 64 splits of heads up to 64, 128 and 256, and more.
@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("d,dv", [(64, 64), (64, 40), (128, 96), (128, 128), (256, 136), (256, 256)])
@pytest.mark.parametrize("skv", [300, 2500])
def test_joins_of_many_rows(hip, skv, d, dv, dtype):
    DenseProblem(1, 16, 16, 300, skv, d, dtype, dv=dv, lengths=[skv - 40], seed=d).check(hip, heads=[0, 15])
    seqs = [(200, skv), (1, 65), (0, 7), (100, 128)]
    CacheProblem(seqs, 16, 4, d, 16, dtype, dv=dv, pad_rows=5, seed=dv).check(hip, heads=[0, 15])


@pytest.mark.parametrize("dtype", TYPES)
def test_workspace(hip, dtype):
    """A workspace of any size: too small for a split, for some of them, and for all."""
    for sq, skv in ((1, 1500), (100, 900)):
        for size in (1, 5000, 40000, 1 << 24):
            DenseProblem(1, 4, 2, sq, skv, 64, dtype, seed=3).check(hip, workspace=size)
    for size in (1, 5000, 1 << 24):
        CacheProblem([(1, 1500), (3, 700)], 4, 2, 64, 16, dtype, seed=4).check(hip, workspace=size)


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
def test_scores_past_log2_units(hip, dtype):
    """Scores near float32's largest: one key still takes everything."""
    p = DenseProblem(1, 1, 1, 3, 40, 64, dtype, scale=1.0, seed=5)
    p.q64[:], p.k64[:] = 0.0, 0.0
    p.q64[..., 0], p.k64[..., 0] = 1e19, np.linspace(-2.9e19, 2.9e19, 40)
    import torch
    from tests.attention_ref import TORCH, check
    p.q, p.k = torch.from_numpy(p.q64).to(TORCH[dtype]), torch.from_numpy(p.k64).to(TORCH[dtype])
    got = p.run(hip)
    check(got, np.broadcast_to(p.v64[:, :, 39:40], got.shape), np.zeros_like(got), dtype)


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("b,hq,hkv,sq,skv", [(2, 4, 2, 1, 900), (2, 4, 2, 9, 900), (2, 4, 2, 70, 900), (8, 64, 64, 40, 90)],
                         ids=["few", "32 rows", "tiles", "many blocks"])
def test_mean_of_equal_values(hip, b, hq, hkv, sq, skv, d, dtype):
    """Keys whose values are all the same: their mean is that value, whatever the weights are and
    however they are rounded (what is added up is what is divided by).  Sums of n float32 terms
    are off by (2 n + 4) 2^-24 < 2^-12 of the value: it is still the nearest of the type."""
    from tests.attention_ref import cast
    rng = np.random.default_rng(d)
    for kw in (dict(), dict(mask=rng.random((b, 1, sq, skv)) < 0.8)):
        p = DenseProblem(b, hq, hkv, sq, skv, d, dtype, scale=0.25 if d == 64 else 0.1, seed=sq, **kw)
        p.v, p.v64 = cast(np.broadcast_to(rng.normal(0, 1, (b, hkv, 1, d)), p.v64.shape), dtype)
        got = p.run(hip)
        want = np.repeat(p.v64[:, :, :1], hq // hkv, axis=1)
        assert (got == want).all(), (kw.keys(), int((got != want).sum()), got.size)
    c = CacheProblem([(sq, skv), (1, 33)], hq, hkv, d, 16, dtype, scale=0.25, seed=sq)
    value, value64 = cast(rng.normal(0, 1, (hkv, 1, d)), dtype)
    c.v[:], c.v64[:] = value, value64
    assert (c.run(hip) == np.repeat(value64[None, :, 0], hq // hkv, axis=1)).all()


# Queries, keys and heads: splits of few rows and of tiles, and the join of many rows.
SPLIT = [(3, 1500, 1), (40, 1500, 1), (300, 300, 16)]


@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
@pytest.mark.parametrize("low,high", [(2.5e19, 2.9e19), (-2.9e19, -2.5e19)])
@pytest.mark.parametrize("sq,skv,heads", SPLIT)
def test_split_scores_past_log2_units(hip, sq, skv, heads, low, high, dtype):
    """Scores near float32's largest in every split of the keys: the largest of all takes
    everything (its weight is one and the others' zero, so the result is its value)."""
    from tests.attention_ref import cast, check
    p = DenseProblem(1, heads, heads, sq, skv, 64, dtype, scale=1.0, seed=5)
    p.q64[:], p.k64[:] = 0.0, 0.0
    p.q64[..., 0], p.k64[..., 0] = 1e19, low
    at = skv - 70
    p.k64[:, :, at, 0] = high
    (p.q, p.q64), (p.k, p.k64) = cast(p.q64, dtype), cast(p.k64, dtype)
    got = p.run(hip)
    check(got, np.broadcast_to(p.v64[:, :, at:at + 1], got.shape), np.zeros_like(got), dtype)
    # the same keys in the pages of a cache, for tokens that all see them
    c = CacheProblem([(3, skv), (1, skv)], 2, 1, 64, 16, dtype, scale=1.0, seed=6)
    c.q64[:], c.k64[:] = 0.0, 0.0
    c.q64[..., 0], c.k64[..., 0] = 1e19, low
    (c.q, c.q64) = cast(c.q64, dtype)
    want = np.empty_like(c.q64)
    for b, rows in enumerate((slice(0, 3), slice(3, 4))):
        c.k64[c.pages[b, at // 16], :, at % 16, 0] = high
        want[rows] = c.v64[c.pages[b, at // 16], 0, at % 16]
    (c.k, c.k64) = cast(c.k64, dtype)
    check(c.run(hip), want, np.zeros_like(want), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq,skv,heads", SPLIT)
def test_split_masks_near_the_lowest_value(hip, sq, skv, heads, dtype):
    """A float32 mask far below every score in every split: the key it closes least takes
    everything."""
    from tests.attention_ref import check
    mask = np.full((1, skv), -3.0e38)
    mask[:, skv - 70] = -2.6e38
    p = DenseProblem(1, heads, heads, sq, skv, 64, dtype, mask=mask, mask_dtype="float32", seed=7)
    got = p.run(hip)
    check(got, np.broadcast_to(p.v64[:, :, skv - 70:skv - 69], got.shape), np.zeros_like(got), dtype)


# ------------------------------------------------------------------- cache -------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", SIZES)
def test_cache_head_sizes(hip, d, dtype):
    CacheProblem([(1, 40), (5, 21), (34, 70)], 4, 2, d, 16, dtype, seed=d).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 32, 64, 100, 256])
def test_cache_page_sizes(hip, page, dtype):
    """Pages that end inside a tile, and pages longer than one."""
    CacheProblem([(1, 130), (40, 65), (3, 3)], 6, 2, 64, page, dtype, seed=page, pad_rows=3).check(hip)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 100, 1000])
def test_cache_windows(hip, window, dtype):
    CacheProblem([(1, 300), (70, 200), (1, 1), (33, 33)], 4, 2, 64, 16, dtype, window=window, seed=window).check(hip)


@pytest.mark.parametrize("dtype", ("float16", "float32"))
@pytest.mark.parametrize("hq", [2, 12, 40])
@pytest.mark.parametrize("count", [63, 64, 65, 130, 4097])
def test_cache_many_sequences(hip, count, hq, dtype):
    """More sequences than one load of starts holds, with some that have no token (the last ones
    among them), for each kind of block: 2, 12 and 40 rows of a key head per token."""
    rng = np.random.default_rng(count)
    new = rng.choice([0, 1, 1, 1, 2, 5], count)
    new[-2:] = 0
    seqs = [(int(n), int(n + e)) for n, e in zip(new, rng.integers(0, 12, count))]
    heads = None if count < 1000 else [0, hq - 1]
    CacheProblem(seqs, hq, 1, 64, 4, dtype, pad_rows=3, seed=count).check(hip, heads=heads)


@pytest.mark.parametrize("dtype", ("float16", "float32"))
@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("window", [95, 96, 97, 2 ** 31 - 1])
def test_cache_windows_of_all_keys(hip, window, d, dtype):
    """Windows about as long as what the table can name (96 keys), and the largest, with a length
    that leaves the first tokens of a sequence without a key."""
    p = CacheProblem([(90, 96), (40, 3), (1, 96)], 2, 1, d, 16, dtype, window=window, spare_columns=0, seed=7)
    got = p.check(hip)
    assert not got[90:127].any()


@pytest.mark.parametrize("index", ["int32", "int64"])
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_ragged_batches(hip, dtype, index):
    """Sequences without new tokens, of one key, whole prompts, and rows behind the last."""
    seqs = [(0, 10), (1, 1), (0, 0), (2, 2), (129, 129), (1, 500), (7, 64), (0, 5), (64, 65), (1, 64)]
    CacheProblem(seqs, 8, 2, 64, 16, dtype, pad_rows=9, seed=1).check(hip, index=index)
    CacheProblem([(0, 3), (0, 0)], 4, 2, 64, 16, dtype, pad_rows=4, seed=1).check(hip, index=index)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (10, 2), (16, 8), (36, 1)])
@pytest.mark.parametrize("n", [1, 4, 50])
def test_cache_shared_heads(hip, n, hq, hkv, dtype):
    CacheProblem([(n, 90), (n, 51), (n, 200)], hq, hkv, 64, 16, dtype, seed=hq + n).check(hip)


@pytest.mark.parametrize("max_kv", [0, 10, 5000, 100000])
@pytest.mark.parametrize("seqs", [[(1, 3000)], [(1, 1025), (1, 17), (1, 2048)], [(2, 4097), (30, 900)]])
@pytest.mark.parametrize("dtype", ("bfloat16", "float32"))
def test_cache_long(hip, dtype, seqs, max_kv):
    """Few rows over many keys; what the caller says of the longest changes nothing."""
    CacheProblem(seqs, 8, 2, 128, 16, dtype, seed=5).check(hip, max_kv=max_kv)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_cache_pages_out_of_range(hip, n, dtype):
    """Table entries that name no page of the cache: their keys are not seen.  (-1, one past the
    last, and far outside; the last sequence has no page at all.)"""
    p = CacheProblem([(n, 200), (n, 130), (n, 96), (n, 64)], 4, 2, 64, 16, dtype, seed=3)
    p.pages[0, 2] = -1
    p.pages[1, 0] = p.k.shape[0]
    p.pages[2, 5] = 2 ** 31 - 1
    p.pages[3, :] = -2 ** 31
    got = p.check(hip)
    assert not got[p.start[3]:].any()


@pytest.mark.parametrize("dtype", ("float16", "float32"))
def test_cache_lengths_out_of_range(hip, dtype):
    """Lengths past the table are cut to it; a length below the new tokens leaves the first of
    them without a key; a negative one leaves all."""
    p = CacheProblem([(4, 64), (6, 20), (3, 10)], 4, 2, 64, 16, dtype, spare_columns=0, seed=4)
    p.len[0], p.seqs[0] = 100000, (4, 64)
    p.len[1], p.seqs[1] = 4, (6, 4)
    p.len[2], p.seqs[2] = -5, (3, 0)
    got = p.check(hip)
    assert not got[4:6].any() and not got[10:13].any()


@pytest.mark.parametrize("dtype", ("float16", "float32"))
def test_cache_starts_out_of_range(hip, dtype):
    """Starts past the rows of q, negative or falling: nothing outside q is touched (the rows of
    sequences that are well formed are right)."""
    p = CacheProblem([(4, 64), (6, 20), (3, 10)], 4, 2, 64, 16, dtype, seed=4)
    ref, tol = p.reference()
    p.start = np.array([0, 4, 10, 10 ** 6], np.int32)          # the last one is cut to q's rows
    got = p.run(hip)
    from tests.attention_ref import check
    check(got, ref, tol, "past the end")
    p.start = np.array([-3, 4, 2, 1], np.int32)
    p.run(hip)


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_cache_later_tokens_may_hold_anything(hip, dtype, value):
    p = CacheProblem([(50, 80), (1, 33)], 4, 2, 64, 16, dtype, seed=6)
    for j in range(60, 80):
        page = p.pages[0, j // 16]
        p.k[page, :, j % 16], p.v[page, :, j % 16] = value, value
    ref, tol = p.reference()
    got = p.run(hip)
    from tests.attention_ref import check
    keep = np.r_[0:30, 50]                                     # tokens before the 60th, and the other sequence
    check(got[keep], ref[keep], tol[keep], str(value))
    assert not np.isfinite(got[30:50]).any()


def test_cache_past_32_bits(hip):
    """A cache of more than 2^32 bytes and 2^31 elements: pages at its end."""
    import torch
    import ctypes
    from onnx_translator_amd.nn.Operators import CCacheAttentionParams
    from tests.attention_ref import Dev, attend, bits, check
    from oracle import oracle as O
    pages, hkv, page, d = 70000, 4, 64, 128                    # 2.3e9 elements, 4.6 GB each
    with Dev(hip) as dev:
        held = [torch.empty(pages, hkv, page, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        g = torch.Generator().manual_seed(1)
        table = np.array([[69999, 5, 69998]], np.int32)
        vals = [torch.randn(3, hkv, page, d, generator=g).to(torch.bfloat16) for _ in range(2)]
        for t, v in zip(held, vals):
            t[table[0].tolist()] = v.cuda()
        torch.cuda.synchronize()
        wraps = []
        for t in held:
            wraps.append(dev.lib.tensor_wrap_device(ctypes.c_void_p(t.data_ptr()), (ctypes.c_int * 4)(*t.shape), 4, O.BF16))
        dev.held += wraps
        for n in (1, 40):
            q = torch.randn(n, 8, d, generator=g).to(torch.bfloat16)
            y = dev.full((n, 8, d), 0.0, "bfloat16")
            p = CCacheAttentionParams(0.0, 0, 0)
            dev.call("cache_attention_forward", dev.put(q), *wraps, dev.put(table), dev.put(np.array([0, n], np.int32)),
                     dev.put(np.array([170], np.int32)), y, ctypes.byref(p), O.PT())
            got = dev.get(y, "bfloat16")
            seen = np.arange(170) <= 170 - n + np.arange(n)[:, None]
            k, v = (x.double().numpy().transpose(1, 0, 2, 3).reshape(hkv, 3 * page, d)[:, :170] for x in vals)
            for h in range(8):
                ref, tol = attend(q[:, h].double().numpy(), k[h // 2], v[h // 2], d ** -0.5, seen, dtype="bfloat16")
                check(got[:, h], ref, tol, f"head {h} n {n}")
