"""Routing to experts on the GPU against the plain form in 64 bits: the ids and the load are equal, the weights within
fp32's roundings: an exponential's argument x - max is off by 2^-24 of itself, the sums of E and K terms by a rounding a
term, and each function by a few: 2^-23 (16 + |x - max| + E / 64 + K) of the weight, at the largest |x - max| of a chosen
expert (and no less than 2^-126, where fp32 has subnormal numbers)."""
import numpy as np
import pytest

from tests import ops_ref as ref
from tests.harness import moe
from tests.ops_dev import TYPES, hip

pytestmark = pytest.mark.gpu


def check(x, K, type="f32", sigmoid=False, bias=None, groups=0, kept=0, best=1, renorm=True, scale=1.0, extra=0):
    T, E = x.shape
    t, values = hip.rows(x, type, extra, 0 if T else 1, 99.0)
    b = None if bias is None else hip.put(np.asarray(bias, np.float32))
    ids, w = hip.full((T + 1, K), 77, np.int32), hip.full((T + 1, K), 77)
    load = hip.full(E + 1, 77, np.int32)
    r = moe.Router(E, K, moe.MOE_SCORE_SIGMOID if sigmoid else moe.MOE_SCORE_SOFTMAX, groups, kept, best, renorm, scale,
                   TYPES[type])
    r.route_async(t.ptr, T, ids.ptr, w.ptr, load.ptr, None if b is None else b.ptr, stride=E + extra)
    want_ids, want_w, want_load = ref.route(values, K, sigmoid, None if bias is None else np.asarray(bias, np.float32),
                                            groups, kept, best, renorm, scale)
    ids, w, load = ids.get(), w.get(), load.get()
    assert np.array_equal(ids[:T], want_ids)
    assert np.array_equal(load[:E], want_load)
    got = w[:T].astype(np.float64)
    top = np.where(values > -np.inf, values, -np.inf).max(-1, initial=-np.inf)
    for i in range(T):
        there = want_ids[i] >= 0
        far = np.abs(values[i, want_ids[i][there]] - (0.0 if sigmoid else top[i]))
        far = far[np.isfinite(far)].max(initial=0.0)
        bound = 2.0 ** -23 * (16 + far + E / 64 + K) * np.abs(want_w[i]) + 2.0 ** -126
        assert np.all(np.abs(got[i] - want_w[i]) <= bound), (i, got[i], want_w[i])
        assert np.all(got[i][~there] == 0.0)
    assert (ids[T:] == 77).all() and (w[T:] == 77.0).all() and load[E] == 77


def logits(T, E, seed, spread=1.5):
    return np.random.default_rng(seed).normal(size=(T, E)) * spread


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,extra", [(1, 1, 1, 0), (1, 512, 10, 0), (3, 8, 8, 1), (5, 60, 4, 3), (64, 64, 1, 0),
                                         (130, 511, 16, 1), (257, 384, 6, 0)])
def test_plain(T, E, K, extra, sigmoid, type):
    print("route", T, E, K, sigmoid, type, flush=True)
    x = logits(T, E, T + E)
    check(x, K, type, sigmoid, extra=extra)
    check(x, K, type, sigmoid, renorm=False, scale=2.5, extra=extra)
    check(x, K, type, sigmoid, bias=logits(1, E, 5, 0.05)[0], extra=extra)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,K,groups,kept,best", [(256, 8, 8, 4, 2), (160, 6, 8, 3, 1), (64, 4, 64, 8, 1), (64, 4, 64, 8, 2),
                                                  (96, 16, 4, 2, 2), (32, 8, 4, 1, 2), (512, 10, 2, 1, 1), (12, 3, 4, 4, 2),
                                                  (511, 7, 7, 3, 2)])
def test_groups(E, K, groups, kept, best, biased, sigmoid):
    print("groups", E, K, groups, kept, best, biased, sigmoid, flush=True)
    x = logits(70, E, E + K)
    x[3:50:3][np.random.default_rng(1).random((16, E)) < 0.7] = -np.inf
    x[60] = -np.inf
    x[61, 1:] = -np.inf
    check(x, K, "f32", sigmoid, logits(1, E, 6, 0.1)[0] if biased else None, groups, kept, best, scale=2.5)
    check(x, K, "bf16", sigmoid, logits(1, E, 6, 0.1)[0] if biased else None, groups, kept, best, renorm=False)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,kept,best", [(0, 0, 1), (4, 2, 1), (4, 2, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_ties(biased, groups, kept, best, sigmoid):
    """Equal scores: the lower id, the lower group, whatever lane holds it."""
    print("ties", biased, groups, kept, best, sigmoid, flush=True)
    r = np.random.default_rng(3)
    x = np.round(logits(90, 512, 2, 1.0) * 2) / 2
    x[0], x[1] = 0.0, -3.0
    x[2, ::2] = 5.0
    bias = np.round(r.normal(size=512) * 2) / 8 if biased else None
    check(x[:3] if biased else x, 10, "f32", sigmoid, np.zeros(512) if biased else None, groups, kept, best)
    if not biased:
        check(x, 16, "bf16", sigmoid, None, groups, kept, best)
    else:
        check(x, 16, "f32", sigmoid, bias, 0, 0, 1)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("biased", [False, True])
def test_near_ties(biased, sigmoid):
    """Scores that fp32 cannot tell apart: the order is the one of 64 bits."""
    print("near ties", biased, sigmoid, flush=True)
    r = np.random.default_rng(4)
    base = np.float32(r.normal(size=(40, 1)))
    x = (base * (1 + r.integers(0, 6, size=(40, 256)) * 2.0 ** -23)).astype(np.float32)
    bias = (np.float32(0.25) * (1 + r.integers(0, 4, size=256) * 2.0 ** -22)).astype(np.float32) if biased else None
    check(x, 16, "f32", sigmoid, bias)
    check(x, 16, "f32", sigmoid, bias, 8, 4, 2)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups", [0, 4])
def test_masked(groups, sigmoid):
    """Rows with nothing left, few experts left, NaNs, the lowest float, infinities, masked biases."""
    print("masked", groups, sigmoid, flush=True)
    E, K = 64, 8
    low = np.finfo(np.float32).min
    x = logits(16, E, 9)
    x[0] = -np.inf
    x[1] = np.nan
    x[2], x[2, 40] = -np.inf, 1.0
    x[3, 5:60] = -np.inf
    x[4, ::2] = np.nan
    x[5] = low
    x[6, 3:] = low
    x[7, 10], x[7, 50] = np.inf, np.inf
    x[8], x[8, 63] = -np.inf, low
    x[9] = 80.0 + x[9]
    x[10] = -85.0 + x[10]
    x[11, 7] = 120.0
    kw = dict(groups=groups, kept=2 if groups else 0)
    check(x, K, "f32", sigmoid, best=1, **kw)
    rows = [0, 1, 2, 3, 4, 7, 8, 12, 13]  # (scores that underflow are all equal: by id, as in 64 bits)
    check(x[rows], K, "f32", sigmoid, best=2 if groups else 1, **kw)
    b = np.zeros(E)
    b[3], b[9], b[40] = -np.inf, np.nan, -np.inf
    check(x[rows], K, "f32", sigmoid, bias=b, best=1, **kw)
    check(x[rows], K, "f32", sigmoid, bias=b, best=2 if groups else 1, renorm=False, **kw)


def test_large():
    print("large", flush=True)
    check(logits(5000, 512, 11), 10)
    check(logits(4097, 24, 14), 4)
    check(logits(70000, 8, 15), 1, "bf16")
    check(logits(5000, 256, 12), 8, "bf16", True, logits(1, 256, 13, 0.1)[0], 8, 4, 2, True, 2.5)


@pytest.mark.parametrize("T", [2, 9, 15, 16, 17, 33])
def test_few(T):
    """Around the number of tokens whose load one work-group counts."""
    x = logits(T, 96, T)
    check(x, 6)
    check(x, 16, "f16", True, logits(1, 96, 3, 0.1)[0], 8, 4, 2)


def test_no_load_and_no_tokens():
    x = logits(4, 32, 1)
    b = hip.put(x.astype(np.float32))
    ids, w = hip.full((4, 2), 0, np.int32), hip.full((4, 2), 0)
    moe.Router(32, 2).route_async(b.ptr, 4, ids.ptr, w.ptr)
    assert np.array_equal(ids.get(), np.argsort(-x, axis=1)[:, :2])
    check(np.zeros((0, 32)), 2)


def test_graph():
    """Captured, replayed on new logits between other work; load is that call's alone."""
    print("graph", flush=True)
    T, E, K = 300, 128, 6
    x = hip.full((T, E), 0)
    out = [[hip.full((T, K), 0, np.int32), hip.full((T, K), 0), hip.full(E, 0, np.int32)] for _ in range(2)]
    r = moe.Router(E, K, moe.MOE_SCORE_SIGMOID)
    s, q = hip.stream(), hip.stream()

    def call(o, stream):
        r.route_async(x.ptr, T, o[0].ptr, o[1].ptr, o[2].ptr, stream=stream)

    launch = hip.capture(s, lambda: call(out[0], s))
    for i in range(4):
        x.put(logits(T, E, i))
        launch()
        call(out[1], q)
        for a, b in zip(*out):
            assert np.array_equal(a.get(), b.get())
        assert np.array_equal(out[0][0].get(), ref.route(x.get(), K, True)[0])
        assert int(out[0][2].get().sum()) == T * K


@pytest.mark.parametrize("E", [64, 100, 256, 512])
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_equal_at_the_last_rank(sigmoid, grouped, E):
    """Equal experts at the last rank and behind it, and, further behind in 32 bits, one that is larger in 64: from one such
    expert more than the ranks to all of them, more than a wave's candidates."""
    print("equal at the last rank", sigmoid, grouped, E, flush=True)
    K, n = 4, (3, 4, 5, 7, 9, 40, E - 3)
    x = np.full((4 * len(n), E), -6.0)
    for i, m in enumerate(n):
        for j, at in enumerate((E - 1, E // 2, 0, E - 2)):
            x[4 * i + j, :m] = 20.0
            x[4 * i + j, at] = 25.0 if j < 3 else 19.5
    bias = np.zeros(E)
    if not sigmoid:  # scores far below the bias that all have: e^(20 - 60)
        x[:, E - 3] = 60.0
        bias += 1.0
        bias[E - 3] = -2.0
    groups = dict(groups=4, kept=3, best=2) if grouped else {}
    check(x, K, "f32", sigmoid, bias, **groups)
    check(x, K, "bf16", sigmoid, bias, renorm=False, **groups)
    if sigmoid and grouped:
        check(x, K, "f32", sigmoid, None, **groups)
    check(np.full((3, E), 20.0), K, "f32", sigmoid, np.zeros(E), **groups)


@pytest.mark.parametrize("E,groups", [(32, 8), (60, 4), (128, 16), (256, 8), (512, 64), (500, 5)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_groups_whose_biases_cancel(sigmoid, E, groups):
    """A group's worth of one large and one as small value: its roundings are those of the values, not of their sum."""
    print("cancelling biases", sigmoid, E, groups, flush=True)
    x = logits(40, E, E)
    n = E // groups
    bias = np.zeros(E)
    for g in range(0, groups, 2):
        bias[g * n:(g + 1) * n] = -2.0 ** 26
        bias[g * n], bias[g * n + 1] = 2.0 ** 24, -2.0 ** 24
    for kept in (1, groups // 2, groups - 1):
        check(x, 4, "f32", sigmoid, bias, groups, kept, 2)
    bias[:] = 0.0
    bias[:n], bias[n], bias[-1] = -1e9, 1e30, -3e38  # masked by a large number; one that is always chosen
    check(x, 4, "f32", sigmoid, bias, groups, groups // 2, 2)


@pytest.mark.parametrize("E,groups", [(8, 2), (64, 8), (96, 3), (256, 8), (512, 4)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_all_groups_kept(sigmoid, E, groups):
    """A group's worth of two values: the order is the scores' in 64 bits, also where no group is left out."""
    print("all groups kept", sigmoid, E, groups, flush=True)
    x = logits(60, E, E + groups)
    x[::3] += 40.0  # sigmoids that are all 1 in 64 bits
    x[1::3] *= 1e-18  # exponentials and sigmoids that are all equal
    check(x, 4, "f32", sigmoid, None, groups, groups, 2)
    check(x, 4, "bf16", sigmoid, None, groups, groups, 2, renorm=False)
    check(x, 4, "f32", sigmoid, None, groups, groups, 1)  # the logits' own order


@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_tiny_scores(sigmoid, biased, renorm):
    """Tokens whose chosen scores are all far below what fp32 holds: over the renormaliser's floor of 1e-20 their weights are
    ordinary numbers, down to scores of 1e-57; beside a larger one they are as small as they are."""
    print("tiny scores", sigmoid, biased, renorm, flush=True)
    T, E, K = 64, 128, 6
    r = np.random.default_rng(8)
    x = -2.2 * np.arange(T)[:, None] - 10.0 * r.random((T, E))  # down to e^-150
    x[::4, 7] = -45.0
    bias = np.zeros(E) if biased else None
    if not sigmoid:
        x[:, 90] = 0.0  # the softmax's largest logit
        if biased:
            bias[90] = -2.0  # never chosen
    check(x, K, "f32", sigmoid, bias, renorm=renorm)
    check(x, K, "f32", sigmoid, bias, 8, 5, 2, renorm=renorm)
