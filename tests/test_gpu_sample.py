"""Sampling against the 64-bit definition: the same token, exactly."""
import numpy as np
import pytest
import torch

import _op_ref as ref
from _gpu import KEEP, P, S, call, dev, empty, host

pytestmark = pytest.mark.gpu


def draw(gpu, x, u, t=None, k=None, p=None, m=None, stride=None):
    r, n = x.shape
    if stride:
        x = np.concatenate([x, np.full((r, stride - n), 99, np.float32)], 1)
    d = [None if a is None else dev(np.asarray(a, ty))
         for a, ty in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    out, size = empty(r, torch.int32), gpu.load().tf_sample_ws_bytes(r, n)
    ws = empty(size, torch.uint8).fill_(0xA5)
    call("tf_sample", P(dev(x)), r, n, stride or n, *(P(a) for a in d),
         P(dev(np.asarray(u, np.float32))), P(out), P(ws), size, S())
    return host(out)


def want(x, u, t=None, k=None, p=None, m=None):
    r = x.shape[0]
    pick = lambda a, i, off: off if a is None else np.asarray(a)[i]  # noqa: E731
    return np.array([ref.sample(x[i], pick(t, i, 1.0), pick(k, i, 0), np.float32(pick(p, i, 1.0)),
                                np.float32(pick(m, i, 0.0)), u[i]) for i in range(r)])


def logits(rng, r, n, body=2.2):
    x = (body * rng.standard_normal((r, n))).astype(np.float32)
    for i in range(r):
        at = rng.integers(0, n, min(n, 30))
        x[i, at] += rng.uniform(2, 12, at.size).astype(np.float32)
    return x


SIZES = [(1, 1), (1, 2), (3, 7), (2, 63), (5, 64), (2, 65), (1, 1000), (3, 4097), (2, 8192),
         (2, 8193), (1, 32000), (2, 50257), (1, 151936), (2, 262145), (1, 524287)]


@pytest.mark.parametrize("r,n", SIZES)
@pytest.mark.parametrize("filters", ["none", "k", "p", "m", "all"])
def test_random(gpu, r, n, filters):
    rng = np.random.default_rng(r * n)
    for trial in range(3):
        x, u = logits(rng, r, n), rng.random(r).astype(np.float32)
        a = {"t": rng.uniform(0.3, 2.0, r).astype(np.float32)}
        if filters in ("k", "all"):
            a["k"] = rng.choice([0, 1, 2, 40, 1000, n, n + 5], r)
        if filters in ("p", "all"):
            a["p"] = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0], r)
        if filters in ("m", "all"):
            a["m"] = rng.choice([0.0, 0.001, 0.05, 0.3, 1.0, 7.0], r)
        got = draw(gpu, x, u, **a, stride=n + 3 if trial == 1 else None)
        assert np.array_equal(got, want(x, u, **a)), a


@pytest.mark.parametrize("n", [257, 20001, 151936])
def test_flat_and_hot(gpu, n):
    """Distributions whose cut lies among tens of thousands of near-equal tokens."""
    rng = np.random.default_rng(n)
    x = (0.01 * rng.standard_normal((6, n))).astype(np.float32)
    u = rng.random(6).astype(np.float32)
    for t in (1.0, 50.0, 1e-3):
        for p in (0.3, 0.95):
            a = dict(t=[t] * 6, p=[p] * 6, k=[0, 0, n // 2, n // 3, 17, 0], m=[0, 0.99, 0, 0, 0, 0.5])
            assert np.array_equal(draw(gpu, x, u, **a), want(x, u, **a)), (t, p)


@pytest.mark.parametrize("n", [5, 1030, 151936])
def test_ties(gpu, n):
    """Equal logits: the lowest indices are kept, -0 equals +0."""
    rng = np.random.default_rng(n)
    x = np.zeros((8, n), np.float32)
    x[1] = -3.5
    x[2, ::2] = -0.0
    x[3] = rng.integers(0, 2, n)
    x[4] = rng.integers(0, 5, n)
    x[5] = np.finfo(np.float32).min
    x[6] = np.finfo(np.float32).max
    x[7, n // 2] = 40.0
    u = np.array([0, 0.25, 0.5, 0.9, 0.75, 1 - 2.0**-24, 0.3, 0.999], np.float32)
    for a in ({}, {"k": [3] * 8}, {"p": [0.5] * 8}, {"k": [max(1, n // 2)] * 8, "p": [0.75] * 8},
              {"m": [0.5] * 8}, {"k": [n - 1] * 8, "m": [1.0] * 8, "p": [0.25] * 8}):
        assert np.array_equal(draw(gpu, x, u, **a), want(x, u, **a)), a


def test_masked_and_infinite(gpu):
    n = 9001
    rng = np.random.default_rng(4)
    x = logits(rng, 10, n)
    x[0] = -np.inf                     # nothing to draw
    x[1] = np.nan
    x[2, rng.random(n) < 0.9] = -np.inf
    x[3, rng.random(n) < 0.9] = np.nan
    x[4] = -np.inf
    x[4, 8000] = -1e38                 # one token left
    x[5, [7, 70, 700]] = np.inf        # shared by three
    x[6, rng.random(n) < 0.99] = np.finfo(np.float32).min
    x[7] = np.nan
    x[7, 3:6] = -np.inf
    x[8, :] = -np.inf
    x[8, [100, 200]] = np.inf
    x[9, ::2] = np.nan
    for u in (0.0, 0.4, 0.99):
        us = np.full(10, u, np.float32)
        for a in ({}, {"k": [2] * 10}, {"k": [8000] * 10}, {"p": [0.9] * 10}, {"m": [0.1] * 10},
                  {"t": [0.5] * 10, "k": [5000] * 10, "p": [0.99] * 10, "m": [0.01] * 10}):
            assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), (u, a)


def test_greedy_and_odd_settings(gpu):
    rng = np.random.default_rng(6)
    x = logits(rng, 6, 3001)
    x[0, [10, 20]] = 50
    u = np.full(6, 0.7, np.float32)
    t = np.array([0, -1, np.nan, 1e-30, np.inf, 1], np.float32)
    assert np.array_equal(draw(gpu, x, u, t=t), want(x, u, t=t))
    assert draw(gpu, x, u, t=t)[0] == 10
    nan = np.full(6, np.nan, np.float32)
    off = draw(gpu, x, u)
    assert np.array_equal(draw(gpu, x, u, p=nan, m=nan, k=[-4] * 6), off)
    assert np.array_equal(off, want(x, u))
    assert np.array_equal(draw(gpu, x, np.array([np.nan, -1, 1, 2, 0, 1], np.float32), k=[9] * 6),
                          want(x, np.array([0, 0, 1, 2, 0, 1], np.float32), k=[9] * 6))


def test_many_rows(gpu):
    rng = np.random.default_rng(8)
    x, u = logits(rng, 700, 1500), rng.random(700).astype(np.float32)
    a = dict(t=rng.uniform(0.5, 1.5, 700).astype(np.float32), k=rng.integers(0, 100, 700),
             p=rng.uniform(0.5, 1.05, 700).astype(np.float32),
             m=rng.uniform(-0.05, 0.1, 700).astype(np.float32))
    assert np.array_equal(draw(gpu, x, u, **a), want(x, u, **a))


def test_a_distribution(gpu):
    """Many draws of one row: each token as often as its weight says."""
    w = np.array([0.5, 0.25, 0.125, 0.0625, 0.0625])
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = draw(gpu, np.tile(np.log(w).astype(np.float32), (n, 1)), u)
    assert np.array_equal(np.bincount(got, minlength=5), (w * n).astype(int))


@pytest.mark.parametrize("n", [300, 9001, 40000])
@pytest.mark.parametrize("t", [np.inf, 1e36, 1e32, 1e-5, 1e-30, 1e-44])
def test_extreme_temperatures_with_filters(gpu, n, t):
    rng = np.random.default_rng(n)
    x = logits(rng, 6, n)
    x[1, ::3] = -np.inf
    x[2, ::2] = np.nan
    x[3] = rng.uniform(-3e38, 3e38, n)
    x[4, 5] = np.inf
    x[5] = rng.uniform(-3e38, -1e38, n)
    for u in (0.1, 0.8):
        us = np.full(6, u, np.float32)
        for a in ({"k": [n // 2] * 6}, {"p": [0.7] * 6}, {"m": [0.5] * 6},
                  {"k": [70] * 6, "p": [0.4] * 6, "m": [1e-30] * 6}):
            a = {"t": [t] * 6, **a}
            assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), (u, a)


def test_cut_far_below_among_both_signs(gpu):
    """The k-th element among keys that end within 2^24 of 2^32, 32 and more below the
    largest; u past the sum takes the last kept."""
    x = np.full((1, 400), -np.inf, np.float32)
    x[0, 100] = 3.3e38
    x[0, 101:201] = np.linspace(2.69e38, 2.6e38, 100)
    x[0, 201:301] = np.linspace(-1.5e38, -1.6e38, 100)
    for k, last in ((51, 150), (101, 200), (102, 201), (150, 249)):
        got = draw(gpu, x, [1.0], t=[1e36], k=[k])
        assert got[0] == last == ref.sample(x[0], np.float32(1e36), k, 1, 0, 1.0)


def test_min_p_alone_far_down(gpu):
    """Bounds of min-p from its least value to one, on rows of a wide and a narrow range."""
    rng = np.random.default_rng(12)
    x = (np.array([[40.], [0.5], [8.]]) * rng.standard_normal((3, 20000))).astype(np.float32)
    for m in (1e-45, 1e-38, 1e-20, 1e-7, 0.02, 0.999, 1.0):
        for u in (0.05, 0.5, 0.97):
            a = dict(m=[m] * 3, t=[1.0, 0.7, 3.0])
            us = np.full(3, u, np.float32)
            assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), (m, u)


def test_long_lists(gpu):
    """Bins that hold more than a chunk's list, a row's list, or just fewer."""
    rng = np.random.default_rng(13)
    n = 60000
    x = np.full((4, n), -9.0, np.float32)
    x[0, :2000] = 1 + 0.01 * rng.random(2000)      # within a chunk's list
    x[1, 5000:7100] = 1 + 0.01 * rng.random(2100)  # past it
    x[2, ::8] = 1 + 0.01 * rng.random(7500)        # of every chunk, within the row's
    x[3, ::7] = 1 + 0.01 * rng.random(8572)        # past it
    for u in (0.2, 0.9):
        us = np.full(4, u, np.float32)
        for a in ({"k": [1234] * 4}, {"p": [0.61] * 4}, {"k": [1999] * 4, "p": [0.37] * 4}):
            assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), (u, a)


@pytest.mark.parametrize("body,t", [(2.0, 1.0), (3.0, 4.0), (300.0, 150.0)])
def test_min_p_beside_the_other_cuts(gpu, body, t):
    """min-p's bound in, just before and just behind the bins that top-k or top-p cuts, on
    rows far from zero too (where a bin's bounds round)."""
    rng = np.random.default_rng(14)
    n = 30000
    x = (body * rng.standard_normal((5, n))).astype(np.float32)
    x[1] += 1e4
    x[2] -= 3e4
    x[3] += 2e5
    w = np.exp((x.astype(np.float64) - x.max(1, keepdims=True)) / t)
    for m in (0.5, 0.05, 1e-3):
        for near in (0.6, 0.98, 1.0, 1.02, 1.7):
            above = w >= m * near
            k, p = above.sum(1), np.minimum((w * above).sum(1) / w.sum(1), 0.9999)
            for a in ({"k": k}, {"p": p}, {"k": k + 3, "p": p * 0.999}):
                a = {**a, "t": [t] * 5, "m": [m] * 5}
                us = rng.random(5).astype(np.float32)
                assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), (m, near, a)


def test_chunks_of_many_spreads(gpu):
    """Parts of a row that are flat, wide, far below the rest, masked by the lowest value or
    empty, in one row."""
    rng = np.random.default_rng(15)
    n = 8192 * 7 + 100
    x = rng.standard_normal((8, n)).astype(np.float32)
    cut = np.arange(n) // 8192
    for i in range(8):
        for c in range(8):
            at, kind = cut == c, rng.integers(0, 6)
            x[i, at] *= np.float32([1e-4, 0.02, 1, 3, 40, 0][kind])
            x[i, at] += np.float32(rng.choice([0, -0.5, -20, -400]) if i % 2 else 0)
    x[2, cut == 3] = -np.inf
    x[3, cut == 1] = np.finfo(np.float32).min
    x[4, 15:] = np.finfo(np.float32).min
    x[5, ::3] = np.finfo(np.float32).min
    x[6] += 5e3
    for t in (0.8, 30.0, 3e-5, 1e-9, 1e-36):
        for a in ({"p": [0.3] * 8}, {"p": [0.97] * 8}, {"k": [40] * 8}, {"k": [30000] * 8},
                  {"k": [9000] * 8, "p": [0.8] * 8}, {"k": [40] * 8, "p": [0.9] * 8, "m": [0.02] * 8}):
            us = rng.random(8).astype(np.float32)
            a = {**a, "t": [t] * 8}
            assert np.array_equal(draw(gpu, x, us, **a), want(x, us, **a)), a


@pytest.mark.parametrize("n,top", [(1500, 1200), (20000, 9000)])
def test_small_u_with_filters(gpu, n, top):
    """Kept weights far below the largest, of which a small u draws one: every token but one
    has 4e-18 of its weight, the first of them 2e-15."""
    x = np.zeros((1, n), np.float32)
    x[0, top] = 40
    x[0, 700] = 6
    for u in (0.0, 1e-30, 2e-17, 1e-15, 3e-15, 1e-7, 9e-7, 1e-6, 0.5):
        for a in ({}, {"m": [1e-18]}, {"k": [n - 100]}, {"k": [n - 100], "m": [4e-18]},
                  {"k": [n - 100], "m": [1e-17]}, {"p": [0.5]}, {"k": [n - 1], "p": [0.99]}):
            assert np.array_equal(draw(gpu, x, [u], **a), want(x, np.float32([u]), **a)), (u, a)


def test_u_of_zero_among_weights_that_are_never_drawn(gpu):
    """Weights below 2^-1000 (index 10: 2^-1040) are never drawn, in a part of the row whose
    largest (index 2100: 2^-577) is far below the row's."""
    x = np.full((1, 16384), -np.inf, np.float32)
    x[0, 10], x[0, 2100], x[0, 9000] = -1040 * np.log(2), -577 * np.log(2), 0
    for a in ({}, {"m": [1e-45]}, {"k": [3]}):
        assert draw(gpu, x, [0.0], **a)[0] == (9000 if "m" in a else 2100), a
