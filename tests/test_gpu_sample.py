"""Draws from scores (sc_sample) against the definition: numpy in 64 bits,
sorting what the kernel selects.  Places are whole numbers and have to be
equal.  Weights are rounded to units of 2^-36 at most and cumulated weights
differ from numpy's by about 1e-13 of a typical weight, so a random number
would have to lie that near to a border for another place."""
import math

import numpy as np
import pytest
import torch

import surfcascade_amd as sc

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tr():
    return sc.Trainer()


def reference(scores, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, lens=None):
    """(index, kept) of [b, v] scores (float64 numpy) and [b, s] numbers."""
    index, kept = np.zeros(u.shape, np.int64), np.zeros(len(scores), np.int64)
    for i, s in enumerate(scores):
        s = s[:len(s) if lens is None else min(max(int(lens[i]), 0), len(s))]
        pool = np.flatnonzero(s > -np.inf)
        if not len(pool):
            index[i], kept[i] = -1, 0
            continue
        order = pool[np.lexsort((pool, -s[pool]))]
        best = s[order[0]]
        if temperature == 0:
            order = order[:1]
        if top_k > 0:
            order = order[:top_k]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(s[order] == best, 1.0, np.exp((s[order] - best) / (temperature or 1.0)))
        n = len(order)
        if top_p < 1:
            c = np.cumsum(w)
            n = 1 + int(np.searchsorted(c, top_p * c[-1], side="left"))
        n = max(min(n, int(np.count_nonzero(w >= min_p))), 1)
        chosen, w = order[:n], w[:n]
        by = np.argsort(chosen)
        c = np.cumsum(w[by])
        x = np.clip(np.nan_to_num(u[i], nan=0.0), 0.0, 1.0) * c[-1]
        at = np.searchsorted(c, x, side="right")
        last = int(np.flatnonzero(w[by] > 0)[-1])
        index[i], kept[i] = chosen[by][np.minimum(at, last)], n
    return index, kept


def _check(tr, scores, u, lens=None, **kw):
    """scores: CPU [b, v] tensor of a type; u: CPU float64 [b, s]."""
    want, wkept = reference(scores.double().numpy(), u.numpy(), lens=None if lens is None else lens.numpy(), **kw)
    idx, kept = tr.sample(scores.cuda(), u.cuda(), lens=None if lens is None else lens.cuda(), **kw)
    assert idx.dtype == torch.int32 and idx.shape == u.shape and kept.shape == (scores.shape[0],)
    np.testing.assert_array_equal(kept.cpu().numpy(), wkept)
    np.testing.assert_array_equal(idx.cpu().numpy(), want)


def _inputs(b, v, s, seed, dtype="f32"):
    g = torch.Generator().manual_seed(seed)
    return (2 * torch.randn(b, v, generator=g)).to(DT[dtype]), torch.rand(b, s, generator=g, dtype=torch.float64)


SIZES = [(1, 1, 1), (1, 2, 5), (3, 63, 7), (2, 64, 64), (1, 65, 3), (2, 1023, 33), (2, 1024, 32), (1, 1025, 31),
         (4, 2047, 9), (1, 2049, 1000), (64, 300, 1), (2, 20011, 128), (1, 32768, 17), (2, 32769, 40),
         (1, 70000, 5000), (3, 131071, 3)]
TRIMS = [dict(), dict(temperature=0.5), dict(top_k=1), dict(top_k=17), dict(top_p=0.9), dict(top_p=0.3, temperature=2.0),
         dict(min_p=0.05), dict(top_k=500, top_p=0.8, min_p=0.02, temperature=0.7), dict(temperature=0.0),
         dict(top_p=0.0), dict(min_p=1.0), dict(top_k=10**9, top_p=0.999)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("trim", TRIMS, ids=str)
def test_draws(tr, size, trim):
    scores, u = _inputs(*size, seed=size[1])
    _check(tr, scores, u, **trim)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("trim", TRIMS, ids=str)
def test_half_scores_tie(tr, dtype, trim):
    """8 or 11 bits of score: most places tie with others, also at the cut."""
    scores, u = _inputs(2, 9000, 200, 5, dtype)
    _check(tr, scores, u, **trim)


@pytest.mark.parametrize("v", [16, 4096, 40000])
@pytest.mark.parametrize("trim", [dict(top_k=5), dict(top_k=4095), dict(top_p=0.5), dict(top_k=13, top_p=0.5),
                                  dict(top_p=0.25, min_p=0.5), dict()], ids=str)
def test_equal_scores(tr, v, trim):
    """Every place ties: the lowest places are kept, and numbers that are
    exactly at a border belong to the place behind it."""
    scores = torch.full((2, v), 1.25)
    u = torch.cat([torch.arange(16).double() / 16, torch.rand(50, dtype=torch.float64,
                   generator=torch.Generator().manual_seed(1))])[None].repeat(2, 1)
    _check(tr, scores, u, **trim)


@pytest.mark.parametrize("trim", TRIMS, ids=str)
def test_masked_places(tr, trim):
    """Rows with masked places: -inf, the type's lowest value, NaN, nothing
    left at all, one place left, +inf and -0."""
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    v = 1500
    g = torch.Generator().manual_seed(3)
    scores = torch.randn(9, v, generator=g)
    scores[0] = -inf
    scores[1] = nan
    scores[2] = -inf
    scores[2, 777] = -3.0
    scores[3, ::2] = -inf
    scores[4, ::3] = nan
    scores[5] = low
    scores[6, 5:] = low
    scores[7, 100] = scores[7, 900] = inf
    scores[8] = torch.where(torch.rand(v, generator=g) < 0.5, 0.0, -0.0)
    u = torch.rand(9, 40, generator=g, dtype=torch.float64)
    _check(tr, scores, u, **trim)


@pytest.mark.parametrize("trim", [dict(), dict(top_k=40, top_p=0.9)], ids=str)
def test_lengths(tr, trim):
    """Rows of their own lengths; what lies behind them (NaN, +inf) is not read."""
    scores, u = _inputs(8, 5000, 20, 9)
    lens = torch.tensor([0, 1, 2, 4999, 5000, -3, 2**31 - 1, 1024], dtype=torch.int32)
    for i, n in enumerate(lens.tolist()):
        n = min(max(n, 0), 5000)
        scores[i, n:] = float("inf") if i % 2 else float("nan")
    _check(tr, scores, u, lens=lens, **trim)


def test_random_numbers_at_the_ends(tr):
    scores, _ = _inputs(1, 3000, 1, 2)
    scores[0, :3] = -float("inf")
    scores[0, -2:] = -float("inf")
    u = torch.tensor([[0.0, -1.0, float("nan"), 1.0 - 2.0**-53, 1.0, 5.0, float("inf"), -float("inf"), 2.0**-70]],
                     dtype=torch.float64)
    idx, _ = tr.sample(scores.cuda(), u.cuda())
    first, last = 3, 2997
    assert idx.cpu()[0].tolist() == [first, first, first, last, last, last, last, first, first]


def test_frequencies(tr):
    """A grid of numbers draws each place as often as its weight says, to one."""
    scores, _ = _inputs(1, 500, 1, 4)
    u = (torch.arange(100000, dtype=torch.float64) + 0.5)[None] / 100000
    idx, _ = tr.sample(scores.cuda(), u.cuda())
    got = np.bincount(idx.cpu().numpy()[0], minlength=500)
    w = np.exp(scores[0].double().numpy())
    assert np.abs(got - 100000 * w / w.sum()).max() <= 1.0


def test_wide_range_and_outliers(tr):
    """Keys of every exponent, and one far outlier over a narrow cluster."""
    g = torch.Generator().manual_seed(6)
    a = torch.randn(30000, generator=g).sign() * torch.exp(torch.empty(30000).uniform_(-80, 80, generator=g))
    b = 0.4 + 1e-4 * torch.randn(30000, generator=g)
    b[12345] = 1e30
    c = 0.4 + 1e-4 * torch.randn(30000, generator=g)
    c[54] = -1e30
    scores = torch.stack([a, b, c])
    u = torch.rand(3, 100, generator=g, dtype=torch.float64)
    for trim in (dict(), dict(top_k=7000), dict(top_p=0.5), dict(top_k=100, top_p=0.7), dict(temperature=1e-3, top_p=0.9),
                 dict(temperature=1e30, top_p=0.5)):
        _check(tr, scores, u, **trim)


def test_large_pool(tr):
    scores, u = _inputs(1, 1000003, 4000, 8)
    for trim in (dict(), dict(top_k=400000, top_p=0.97), dict(min_p=0.001, temperature=0.6)):
        _check(tr, scores, u, **trim)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [8193, 16384, 16385, 30000, 32768])
def test_long_rows_trimmed_first(tr, v, dtype):
    """Rows of which top_k keeps few, up to the border and past it."""
    scores, u = _inputs(3, v, 300, v, dtype)
    scores[1, ::3] = -float("inf")
    lens = torch.tensor([v, v - 5, 8100], dtype=torch.int32)
    for k in (1, 2, 63, 8191, 8192, 8193):
        _check(tr, scores, u, top_k=k)
        _check(tr, scores, u, lens=lens, top_k=k, top_p=0.9, min_p=1e-3, temperature=1.5)
    many, numbers = _inputs(40, v, 7, v + 1, dtype)  # (rows enough to be trimmed without top_p)
    _check(tr, many, numbers, top_k=700)
    _check(tr, many, numbers, temperature=0.0)
    equal = torch.full((1, v), 0.5).to(DT[dtype])
    for k in (5, 8192):
        _check(tr, equal, u[:1], top_k=k)
        _check(tr, equal, u[:1], top_k=k, top_p=0.5)


def test_larger_pools_and_many_rows(tr):
    """Past 2^22 scores a part's groups grow; past 128 rows each row has one
    workgroup again, however long it is."""
    scores, u = _inputs(1, 5000011, 300, 14, "bf16")
    for trim in (dict(top_p=0.9), dict(top_k=3000000, top_p=0.9, min_p=1e-4), dict(top_k=2)):
        _check(tr, scores, u, **trim)
    scores, u = _inputs(150, 9001, 5, 15)
    lens = torch.randint(0, 9002, (150,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    _check(tr, scores, u, lens=lens, top_k=2000, top_p=0.9)
    _check(tr, scores[:128].contiguous(), u[:128].contiguous(), lens=lens[:128], top_k=2000, top_p=0.9)


@pytest.mark.parametrize("trim", TRIMS, ids=str)
def test_masked_places_in_long_rows(tr, trim):
    inf, low = float("inf"), torch.finfo(torch.float32).min
    v = 40001
    g = torch.Generator().manual_seed(7)
    scores = torch.randn(8, v, generator=g)
    scores[0] = -inf
    scores[1] = float("nan")
    scores[2] = -inf
    scores[2, 31234] = -3.0
    scores[3, :30000] = -inf
    scores[4, ::3] = float("nan")
    scores[5] = low
    scores[6, 5:] = low
    scores[7, 100] = scores[7, 39000] = inf
    u = torch.rand(8, 70, generator=g, dtype=torch.float64)
    _check(tr, scores, u, **trim)


def test_strides(tr):
    """Rows of wider buffers, and offsets past 32 bits."""
    scores, u = _inputs(3, 700, 11, 10)
    wide = torch.full((3, 1001), float("inf"))
    wide[:, 5:705] = scores
    wu = torch.full((3, 20), 0.5, dtype=torch.float64)
    wu[:, 3:14] = u
    a = tr.sample(scores.cuda(), u.cuda(), top_p=0.9)
    b = tr.sample(wide.cuda()[:, 5:705], wu.cuda()[:, 3:14], top_p=0.9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ld = 2**31 + 7
    big = torch.empty(ld + 700, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((2, 700), (ld, 1))
    far.copy_(scores[:2])
    c = tr.sample(far, u[:2].cuda())
    d = tr.sample(scores[:2].bfloat16().cuda(), u[:2].cuda())
    assert torch.equal(c[0], d[0])


def test_one_row_and_empty_sizes(tr):
    scores, u = _inputs(1, 50, 6, 11)
    i1, k1 = tr.sample(scores[0].cuda(), u[0].cuda())
    i2, k2 = tr.sample(scores.cuda(), u.cuda())
    assert i1.shape == (6,) and torch.equal(i1, i2[0]) and torch.equal(k1, k2)
    e = dict(device="cuda")
    i, k = tr.sample(torch.zeros(3, 0, **e), torch.zeros(3, 4, dtype=torch.float64, **e))
    assert (i == -1).all() and not k.any()
    i, k = tr.sample(torch.zeros(3, 5, **e), torch.zeros(3, 0, dtype=torch.float64, **e))
    assert i.shape == (3, 0) and (k == 5).all()
    i, k = tr.sample(torch.zeros(0, 5, **e), torch.zeros(0, 2, dtype=torch.float64, **e))
    assert i.shape == (0, 2) and k.shape == (0,)


def test_refused_tensors(tr):
    s, u = _inputs(2, 10, 3, 12)
    S, Q = s.cuda(), u.cuda()
    for bad in (lambda: tr.sample(s, Q), lambda: tr.sample(S, u), lambda: tr.sample(S, Q.float()),
                lambda: tr.sample(S.double(), Q), lambda: tr.sample(S, Q[:1]), lambda: tr.sample(S[0], Q),
                lambda: tr.sample(S.t().contiguous().t(), Q), lambda: tr.sample(S[:, ::2], Q),
                lambda: tr.sample(S[:1].expand(2, 10), Q),
                lambda: tr.sample(S, Q, lens=torch.zeros(2, dtype=torch.int64).cuda()),
                lambda: tr.sample(S, Q, lens=torch.zeros(3, dtype=torch.int32).cuda())):
        with pytest.raises(ValueError):
            bad()
    for kw in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=-0.5), dict(min_p=2.0)):
        with pytest.raises(sc.SurfCascadeError) as e:
            tr.sample(S, Q, **kw)
        assert e.value.code == -1


def test_same_call_same_bits(tr):
    scores, u = _inputs(1, 200000, 3000, 13)
    S, Q = scores.cuda(), u.cuda()
    a = tr.sample(S, Q, top_k=90000, top_p=0.95)
    for _ in range(3):
        b = tr.sample(S, Q, top_k=90000, top_p=0.95)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("v", [700, 4000, 8192, 20000])
@pytest.mark.parametrize("trim", [dict(top_k=350), dict(top_p=0.5), dict(top_k=300, top_p=0.6)], ids=str)
def test_crowded_bins(tr, v, trim):
    """Rows whose descents end in a bin with more members than are ranked at
    once, several levels deep: most scores within a few hundred steps of 1, two
    far ones that make the range wide."""
    g = torch.Generator().manual_seed(v)
    near = 1.0 + torch.randint(0, 300, (300, v), generator=g).float() * 2.0 ** -20
    near[:, 0], near[:, 1] = -3.0e38, -1.0
    near[:, 600:] = -20.0 - torch.rand(300, v - 600, generator=g)
    near = near[:, torch.randperm(v, generator=g)].contiguous()
    _check(tr, near, torch.rand(300, 4, generator=g, dtype=torch.float64), **trim)


def test_more_rows_than_a_grid_has(tr):
    """2^21 rows are one launch; the rows behind them are a second."""
    b = 2**21 + 5
    scores = torch.rand(b, 3, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    u = torch.full((b, 1), 0.5, dtype=torch.float64, device="cuda")
    idx, kept = tr.sample(scores, u, temperature=0.0)
    assert torch.equal(idx[:, 0].long(), scores.argmax(1)) and bool((kept == 1).all())


def test_more_draws_than_a_grid_has(tr):
    """Past 2^28 draws a wave makes more than 16 of them."""
    v, reps = 8193, 2**28 // 8193 + 2
    place = torch.arange(v, device="cuda")
    u = ((place.double() + 0.5) / v).repeat(reps)[None]
    assert u.numel() > 2**28
    idx, kept = tr.sample(torch.zeros(1, v, device="cuda"), u)
    assert int(kept) == v
    assert bool((idx.view(reps, v) == place.int()).all())


@pytest.mark.parametrize("v", [700, 5000, 20000])
@pytest.mark.parametrize("temperature", [1e-3, 1.0, 1e4])
@pytest.mark.parametrize("at,scale", [(0.0, 2.0), (1.0e6, 2.0), (-3.0e7, 40.0), (0.0, 1.0e30), (0.0, 1.0e-30)])
def test_scores_far_from_zero(tr, at, scale, temperature, v):
    """Ranges from a few roundings of the scores to more than float32 holds, with
    a mask of the lowest value or without one, weights from all equal to one."""
    g = torch.Generator().manual_seed(v)
    scores = at + scale * torch.randn(4, v, generator=g)
    scores[1, ::3] = torch.finfo(torch.float32).min
    scores[2, 5::7] = torch.finfo(torch.float32).max
    scores[3, 11] = math.inf
    u = torch.rand(4, 9, generator=g, dtype=torch.float64)
    for trim in (dict(top_k=v // 3), dict(top_k=40), dict(top_p=0.7), dict(top_k=v // 3, top_p=0.9)):
        _check(tr, scores, u, temperature=temperature, **trim)
