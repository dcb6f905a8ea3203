"""The choice of experts against its definition in f64.

Weights: f64 throughout and one rounding to f32, half a step (2^-24), and what
f64's exp and sums leave, under 1e-12."""
import numpy as np
import pytest

import ggml_hip as G
import moe_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOL = R.U + 1e-12


def _check(logits, k, **kw):
    bias = kw.pop("bias", None)
    ids, w = G.route(torch.from_numpy(logits).cuda(), k, bias=None if bias is None else torch.from_numpy(bias).cuda(), **kw)
    want_ids, want = R.route(logits, k, bias=bias, **kw)
    ids, w = ids.cpu().numpy(), w.cpu().numpy().astype(np.float64)
    assert np.array_equal(ids, want_ids)
    assert np.array_equal(np.isnan(w), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.all(np.abs(w - want)[fine] <= TOL * np.abs(want)[fine] + 2.0 ** -149)
    return ids, w


def _logits(n, e, seed=0, spread=2.0):
    return (np.random.RandomState(seed).randn(n, e) * spread).astype(np.float32)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("n,e,k", [(1, 1, 1), (3, 2, 2), (5, 8, 2), (1, 60, 4), (7, 64, 64), (9, 65, 6), (1, 128, 8),
                                   (130, 128, 8), (33, 160, 6), (17, 256, 8), (4, 511, 10), (6, 1024, 32)])
def test_choice(gating, biased, n, e, k):
    bias = (np.random.RandomState(9).randn(e) * 0.2).astype(np.float32) if biased else None
    for renormalize, scale in ((False, 1.0), (True, 2.5)):
        _check(_logits(n, e), k, gating=gating, bias=bias, renormalize=renormalize, scale=scale)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("e,groups,keep,top,k", [(256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (64, 64, 5, 2, 5), (64, 4, 4, 2, 8),
                                                 (1024, 16, 1, 2, 20), (36, 6, 2, 2, 20), (96, 2, 1, 1, 48),
                                                 (15, 5, 3, 2, 9), (448, 7, 2, 1, 3)])
def test_groups(gating, biased, e, groups, keep, top, k):
    bias = (np.random.RandomState(8).randn(e) * 0.2).astype(np.float32) if biased else None
    _check(_logits(23, e, 3), k, gating=gating, bias=bias, groups=groups, keep=keep, top=top, renormalize=True)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_take_the_lowest_index(gating, groups):
    logits = np.random.RandomState(1).randint(-1, 2, (40, 128)).astype(np.float32)
    logits[0] = 0.0
    logits[1] = -0.0
    logits[2, ::2] = -0.0
    logits[2, 1::2] = 0.0
    for bias in (None, np.zeros(128, np.float32), (np.arange(128) % 3 == 0).astype(np.float32)):
        _check(logits, 9, gating=gating, bias=bias, groups=groups, keep=min(groups, 2), top=2)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("groups,top", [(1, 1), (8, 1), (8, 2)])
def test_hidden_experts(gating, groups, top):
    r = np.random.RandomState(5)
    logits = _logits(64, 64, 4)
    logits[r.rand(64, 64) < 0.6] = -np.inf
    logits[0] = -np.inf                  # none
    logits[1, 1:] = -np.inf              # one
    logits[2, :8] = -np.inf              # a whole group
    logits[3] = np.finfo(np.float32).min  # the type's lowest value hides nothing
    logits[4, 5:] = np.finfo(np.float32).min
    bias = (r.randn(64) * 0.1).astype(np.float32)
    bias[r.rand(64) < 0.3] = -np.inf
    for b in (None, bias):
        ids, w = _check(logits, 7, gating=gating, bias=b, groups=groups, keep=min(groups, 3), top=top, renormalize=True)
        assert (ids[0] == -1).all() and (w[0] == 0).all()


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("biased", [False, True])
def test_values_that_are_not_finite(gating, biased):
    logits = _logits(5, 96, 6)
    logits[0, 17] = np.nan
    logits[1, [3, 50]] = np.nan, np.inf
    logits[2, 80] = np.inf
    logits[3, [4, 5]] = np.inf
    logits[4, 7] = -np.inf
    bias = (np.random.RandomState(2).randn(96) * 0.1).astype(np.float32) if biased else None
    for groups in (1, 4):
        _check(logits, 6, gating=gating, bias=bias, groups=groups, keep=2 if groups > 1 else 1, top=2, renormalize=True)
    if biased:
        bias[11] = np.nan
        bias[12] = np.inf
        _check(_logits(5, 96, 6), 6, gating=gating, bias=bias)


def test_far_and_close_scores():
    # p differs by less than f32 tells apart: the order is that of f64, and without a bias that of the logits.
    logits = np.full((4, 64), -20.0, np.float32)
    logits[0, 30:40] = np.nextafter(np.float32(15.0), np.float32(16.0)) + np.arange(10, dtype=np.float32) * np.spacing(np.float32(15.0))
    logits[1] = np.linspace(-200, -100, 64, dtype=np.float32)
    logits[2] = np.linspace(90, 300, 64, dtype=np.float32)
    logits[3] = np.linspace(-1e30, 1e30, 64, dtype=np.float32)
    for gating in ("softmax", "sigmoid", "softmax_chosen"):
        _check(logits, 5, gating=gating, renormalize=True)
        _check(logits[:1], 5, gating=gating, bias=np.full(64, 0.125, np.float32), renormalize=True)


def test_the_smallest_sum():
    logits = np.full((2, 8), -60.0, np.float32)
    logits[1] = -800.0
    for min_sum in (2.0 ** -14, 1e-30, 0.5):
        _check(logits, 3, gating="sigmoid", renormalize=True, min_sum=min_sum)


def test_strides_and_given_results():
    wide = torch.randn(37, 300, device="cuda")
    logits = wide[:, 3:203]
    ids = torch.full((37, 20), -7, dtype=torch.int32, device="cuda")
    w = torch.full((37, 11), 5.0, device="cuda")
    G.route(logits, 6, renormalize=True, ids=ids[:, 2:8], weights=w[:, :6])
    want = G.route(logits.contiguous(), 6, renormalize=True)
    assert torch.equal(ids[:, 2:8], want[0]) and torch.equal(w[:, :6], want[1])
    assert (ids[:, :2] == -7).all() and (ids[:, 8:] == -7).all() and (w[:, 6:] == 5).all()
    assert np.array_equal(want[0].cpu().numpy(), R.route(logits.cpu().numpy(), 6, renormalize=True)[0])


def test_many_tokens():
    _check(_logits(4099, 40, 12), 4, gating="sigmoid", renormalize=True)


def test_no_tokens():
    ids, w = G.route(torch.empty(0, 16, device="cuda"), 4)
    assert ids.shape == w.shape == (0, 4)


def _balanced_groups(gating, n, groups, size, large, seed):
    """Logits and a bias for which each group's two best are `large` above and below, and the sums of two nearly the
    same for all groups: f32 scores of that size do not tell them apart."""
    r = np.random.RandomState(seed)
    p = r.uniform(0.1, 0.9, (n, groups, 1))
    near = r.choice([-1, 1], (n, groups, 1)) * 10 ** r.uniform(-6, -4, (n, groups, 1))
    rest = np.full((n, groups, size - 2), 0.01)
    p = np.concatenate([p, 1 + near - p, rest], -1)
    logits = {"softmax": np.log, "sigmoid": lambda x: np.log(x / (1 - x)), "softmax_chosen": lambda x: x}[gating](p)
    bias = np.full((groups, size), -3.0 * large)
    bias[:, 0], bias[:, 1] = large, -large
    return logits.reshape(n, -1).astype(np.float32), bias.ravel().astype(np.float32)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("large", [30, 300, 1000, 4096, 1e5])
@pytest.mark.parametrize("groups,size,keep", [(2, 2, 1), (8, 2, 4), (4, 3, 2), (8, 32, 4)])
def test_groups_whose_two_best_cancel(gating, large, groups, size, keep):
    logits, bias = _balanced_groups(gating, 500, groups, size, large, groups)
    _check(logits, keep, gating=gating, bias=bias, groups=groups, keep=keep, top=2)


@pytest.mark.parametrize("logits,large", [([0.47, 3.82, 2.17, 0.83], 1024), ([-0.6627474, -1.0630597, -1.5472649, -0.31719202], 300)])
def test_the_better_of_two_groups(logits, large):
    _check(np.array([logits], np.float32), 1, gating="sigmoid", bias=np.array([large, -large] * 2, np.float32), groups=2, top=2)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
def test_groups_far_below_the_others(gating):
    """Scores of a mask's size beside ordinary ones, and as many of them kept as there have to be."""
    logits = _logits(40, 64, 7)
    bias = (np.random.RandomState(3).randn(64) * 0.2).astype(np.float32)
    bias[16:40] = -1e9
    bias[40:44] = 1e9, -1e9, 1e4, -1e4
    for keep in (1, 3, 5, 7, 8):
        _check(logits, 6, gating=gating, bias=bias, groups=8, keep=keep, top=2)


@pytest.mark.parametrize("gating", ["softmax", "sigmoid", "softmax_chosen"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,size", [(2, 8), (4, 16), (6, 6), (8, 32)])
def test_sums_beyond_f32_are_not_hidden(gating, biased, groups, size):
    """Groups whose two best sum to less than f32 holds come before those without an expert."""
    least = np.finfo(np.float32).min
    logits = _logits(7, groups * size, 5).reshape(7, groups, size)
    logits[:6, 0] = -np.inf
    logits[1:, 1:] = least
    logits[2, -1] = -0.9e38
    logits[3, 1:, :2] = least / 2          # a sum that is just held
    logits[4, 1:, 1:] = -np.inf            # one expert a group
    logits[5, 1:] = np.abs(logits[5, 1:])  # and above what f32 holds
    bias = None
    if biased:
        bias = np.full((groups, size), -3e38, np.float32)
        bias[1, 1] = -2e38
        if gating == "softmax_chosen":
            logits[np.isfinite(logits)] /= 8  # some scores themselves are beyond f32, others their sums alone
        bias = bias.ravel()
    for keep in range(1, groups):
        ids, _ = _check(logits.reshape(7, -1), 2, gating=gating, bias=bias, groups=groups, keep=keep, top=2)
        if gating == "softmax_chosen":
            assert (ids[:6, 0] >= size).all()
