"""Weighted sums of experts' rows against f64: n + 1 terms summed by fused
multiply-adds, each off by half a step of a partial sum, which is at most the sum
of magnitudes."""
import math

import numpy as np
import pytest

import ggml_hip as G
import moe_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _check(y, w, ids=None, add=None, got=None):
    n = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    if got is None:
        got = G.combine(y, w, ids=ids, add=add)
    want, size = R.combine(n(y), n(w), n(ids), n(add))
    off = np.abs(got.cpu().numpy().astype(np.float64) - want)
    assert np.all(off <= (y.shape[1] + 1) * R.U * size * (1 + 1e-6) + 2.0 ** -140)


@pytest.mark.parametrize("n,k,rows", [(1, 1, 1), (1, 8, 2048), (7, 8, 2048), (3, 2, 5), (5, 3, 127), (2, 16, 4096), (33, 6, 1030),
                                      (300, 8, 768), (1000, 4, 2049), (1, 64, 100), (9, 1, 8192), (4, 9, 40000), (70000, 1, 4)])
@pytest.mark.parametrize("add", [False, True])
def test_sums(n, k, rows, add):
    torch.manual_seed(n + rows)
    y, w = torch.randn(n, k, rows, device="cuda"), torch.randn(n, k, device="cuda")
    _check(y, w, add=torch.randn(n, rows, device="cuda") if add else None)


def test_slots_left_out():
    torch.manual_seed(0)
    y, w = torch.randn(50, 8, 260, device="cuda"), torch.rand(50, 8, device="cuda")
    ids = torch.randint(-3, 5, (50, 8), dtype=torch.int32, device="cuda")
    ids[3] = -1
    ids[4] = 2 ** 31 - 1
    _check(y, w, ids=ids)
    y[ids < 0] = float("nan")
    w[ids < 0] = float("inf")
    got = G.combine(y, w, ids=ids)
    y[ids < 0] = 0
    w[ids < 0] = 0
    _check(y, w, ids=ids, got=got)
    assert (got[3] == 0).all()


def test_no_slots():
    add = torch.randn(5, 33, device="cuda")
    assert torch.equal(G.combine(torch.empty(5, 0, 33, device="cuda"), torch.empty(5, 0, device="cuda"), add=add), add)
    assert (G.combine(torch.empty(5, 0, 33, device="cuda"), torch.empty(5, 0, device="cuda")) == 0).all()
    assert G.combine(torch.empty(0, 4, 33, device="cuda"), torch.empty(0, 4, device="cuda")).shape == (0, 33)


@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strides_and_in_place(shift):
    torch.manual_seed(shift)
    y = torch.randn(20, 3, 600, device="cuda")[..., shift:shift + 512]
    w = torch.randn(20, 9, device="cuda")[:, 2:5]
    add = torch.randn(20, 700, device="cuda")
    was = add.clone()
    here = add[:, shift:shift + 512]
    G.combine(y, w, add=here, out=here)
    _check(y, w, add=was[:, shift:shift + 512], got=here)
    here.copy_(was[:, shift:shift + 512])
    assert torch.equal(add, was)
    one = torch.randn(20, 1, 512, device="cuda").expand(20, 3, 512)  # the same row in every slot
    _check(one, w)


def test_what_is_not_finite():
    y, w = torch.ones(3, 2, 8, device="cuda"), torch.ones(3, 2, device="cuda")
    y[0, 1, 2] = float("nan")
    y[1, 0, 3] = float("inf")
    w[1, 1] = 0.0
    w[2, 0] = float("inf")
    got = G.combine(y, w).cpu()
    assert torch.isnan(got[0, 2]) and (got[0, [0, 1, 3, 4, 5, 6, 7]] == 2).all()
    assert got[1, 3] == float("inf") and (got[1, :3] == 1).all() and torch.isinf(got[2]).all()


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 6, 7, 514, 1031])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_ends_of_rows(rows, off):
    """Rows of any length from any multiple of four bytes; nothing before or behind them is written."""
    torch.manual_seed(rows)
    y = torch.randn(9, 4, rows + 5, device="cuda")[..., off:off + rows]
    w = torch.randn(9, 4, device="cuda")
    add = torch.randn(9, rows + 6, device="cuda")[:, 1:1 + rows]
    out = torch.full((9, rows + 5), 7.0, device="cuda")
    got = G.combine(y, w, add=add, out=out[:, off:off + rows])
    _check(y, w, add=add, got=got)
    assert (out[:, :off] == 7).all() and (out[:, off + rows:] == 7).all()


@pytest.mark.parametrize("n,k,rows", [(3, 1, 50), (5, 8, 130), (4, 16, 70), (2, 64, 41)])
@pytest.mark.parametrize("add", [False, True])
def test_one_rounding(n, k, rows, add):
    """Sums that nearly cancel, against the exact ones: half a step of the result, and what k f64 terms and the
    reference's own rounding leave of their magnitudes."""
    r = np.random.RandomState(k + rows)
    y, w = r.randn(n, k, rows).astype(np.float32), r.randn(n, k).astype(np.float32)
    terms = y.astype(np.float64) * w[..., None].astype(np.float64)  # exact
    base = np.zeros((n, rows))
    if add:
        base = (-terms.sum(1) * (1 + r.randn(n, rows) * 1e-4)).astype(np.float32).astype(np.float64)
    elif k > 1:
        y[:, -1] = -(terms[:, :-1].sum(1) / w[:, -1:]) * (1 + r.randn(n, rows) * 1e-4)
        terms = y.astype(np.float64) * w[..., None].astype(np.float64)
    want = np.array([[math.fsum([base[t, m], *terms[t, :, m]]) for m in range(rows)] for t in range(n)])
    bound = R.U * np.abs(want) + (k + 2) * 2.0 ** -53 * (np.abs(base) + np.abs(terms).sum(1)) + 2.0 ** -150
    got = G.combine(torch.from_numpy(y).cuda(), torch.from_numpy(w).cuda(),
                    add=torch.from_numpy(base.astype(np.float32)).cuda() if add else None).cpu().numpy()
    assert np.all(np.abs(got.astype(np.float64) - want) <= bound)
    # What the bound is for: sums in f32 would not keep it.
    f32 = base.astype(np.float32)
    for s in range(k):
        f32 = f32 + y[:, s] * w[:, s:s + 1]
    if k > 1 or add:
        assert np.any(np.abs(f32.astype(np.float64) - want) > bound)
