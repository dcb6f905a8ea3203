"""Attention over the paged cache (hip_qmm_attn_paged) where queries, keys or
values are not finite: only the results that they belong to are touched, in
every kernel form, type and head size, whichever tile holds them."""
import math

import pytest

import attn_ref as R
from test_gpu_attn import FORMS, _case, _hold, _run

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DIMS = [64, 80, 96, 128, 256]


def _plan(c):
    import ggml_hip as G
    return G.attn_paged_plan(G.PagedKV(c["k"], c["v"]), c["q"].shape[1], len(c["new"]), c["q"].shape[0], max(c["new"]),
                             c["table"].shape[1] * c["k"].shape[2])


def _at(c, seq, token):
    page = c["k"].shape[2]
    return int(c["table"][seq, token // page]), token % page


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("n,new", [(700, 300), (764, 300), (3000, 15), (3064, 13)])
def test_other_rows_keep_their_results(n, new, dim, dtype):
    """Workgroups of 64 rows: a NaN query row, and a NaN value in the first tile (every block), in the middle and in the
    last tile.  Every row and dimension that they do not belong to is what it was, bit for bit."""
    c = _case(dtype, 32, 8, dim, page=32, lens=(n, n - 37), new=[new, new])
    assert _plan(c)[0] == 64
    clean = _run(c)
    q, v = c["q"].clone(), c["v"].clone()
    for token in (0, n // 2, n - 1, None):
        c["q"], c["v"] = q.clone(), v.clone()
        want = clean.clone()
        if token is not None:
            page, slot = _at(c, 0, token)
            c["v"][page, 5, slot, dim - 3] = math.nan
            want[max(0, token - (n - new)):new, 20:24, dim - 3] = math.nan
        c["q"][2, 9, 7] = c["q"][new + 3, 31, 0] = math.nan
        want[2, 9] = want[new + 3, 31] = math.nan
        for _ in range(3):
            got = _run(c)
            assert torch.equal(torch.isnan(got), torch.isnan(want))
            assert torch.equal(got.nan_to_num(), want.nan_to_num())


def _definition(c, window=0, sinks=0, scale=None):
    """dst = sum w v / sum w over what is seen, w = exp(scale q.k), in f64 with infinities and NaN as IEEE has them; a zero
    row where the weights' sum is 0.  The result and the largest |score| that is finite."""
    q, out, top = c["q"].double(), torch.zeros(c["q"].shape, dtype=torch.float64, device="cuda"), 0.0
    group = q.shape[1] // c["k"].shape[1]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for s, n in enumerate(c["lens"].tolist()):
        lo, m = int(c["starts"][s]), c["new"][s]
        if n == 0:
            continue
        ks, ok = R.rows_of(c["k"], c["table"][s], n)
        vs, _ = R.rows_of(c["v"], c["table"][s], n)
        see = R.seen(m, n, ok, window, sinks)
        for h in range(q.shape[1]):
            k, v = ks[:, h // group].double(), vs[:, h // group].double()
            rows = q[lo:lo + m, h]
            odd = ~torch.isfinite(k).all(1)
            sc = rows @ torch.where(odd[:, None], 0.0, k).T
            for j in odd.nonzero()[:, 0].tolist():
                sc[:, j] = (rows * k[j]).sum(1)
            sc = (sc * scale).masked_fill(~see, -math.inf)
            most = sc.amax(1, keepdim=True)
            w = torch.exp(sc - torch.where(most == -math.inf, 0.0, most)).masked_fill(~see, 0.0)
            o = w @ torch.where(torch.isfinite(v), v, 0.0)
            for j in (~torch.isfinite(v).all(1)).nonzero()[:, 0].tolist():
                o += torch.where(see[:, j:j + 1] & ~torch.isfinite(v[j]), w[:, j:j + 1] * v[j], 0.0)
            total = w.sum(1, keepdim=True)
            out[lo:lo + m, h] = torch.where(total == 0, 0.0, o / total)
            fin = sc[torch.isfinite(sc)]
            top = max(top, float(fin.abs().max())) if fin.numel() else top
    return out, top


def _check(c, **kw):
    got, (want, top) = _run(c, decode=False, **kw), _definition(c, **kw)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    _hold(got, want, top, c["q"].shape[2])
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("form", FORMS)
def test_infinite_keys(form, dim, dtype):
    """A score of -inf is a weight of 0, of +inf or NaN a row of NaN: each head of keys has another kind of them."""
    _, _, seqs, new, n = form
    heads, kv_heads = 16, 8
    c = _case(dtype, heads, kv_heads, dim, page=32, lens=[n] * seqs, new=[new] * seqs)
    clean = _run(c, decode=False)
    q, k, v, inf = c["q"], c["k"], c["v"], math.inf
    first, last, mid = _at(c, 0, 1), _at(c, 0, n - 1), _at(c, 0, n - 1 - new // 2)

    def key(at, h, **elements):
        for d, x in elements.items():
            k[at[0], h, at[1], int(d[1:])] = x

    key(first, 0, d3=inf)                      # by the query's sign: weight 0, or NaN
    q[:, 2:4, 3].abs_().neg_()
    key(first, 1, d3=inf), key(last, 1, d3=inf)  # weight 0 in every row
    q[:, 4:6, 3] = torch.where(q[:, 4:6, 3] > 0, 2.0 ** -40, -2.0 ** -40)  # less than a part of the row's 22 bits
    key(first, 2, d3=-inf)
    q[:, 6:8, 3].abs_()
    q[0, 6, 3] = 0.0                           # 0 times infinity
    key(first, 3, d3=-inf)
    q[:, 8:10, 3].abs_(), q[:, 8:10, 5].abs_()
    key(first, 4, d3=-inf, d5=-inf), key(mid, 4, d3=-inf, d5=inf)  # the middle one: inf - inf
    q[:, 10:12, 3].abs_()
    key(mid, 5, d3=-inf)                       # weight 0, times an infinite value
    v[mid[0], 5, mid[1], 9] = inf
    q[:, 12:14].abs_()
    k[first[0], 6, first[1]] = -inf            # every element
    got = _check(c)
    assert torch.equal(got[:, 14:], clean[:, 14:])  # the head of keys with none
    assert bool(torch.isfinite(got[:, 2:4]).all() and torch.isfinite(got[:, 12:14]).all())
    _check(c, scale=-0.2)
    _check(c, window=max(1, n // 3), sinks=2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_rows_whose_scores_are_all_minus_infinity(new, dtype):
    """Weights of 0 alone: zeros, as where nothing is seen, whatever the values; but NaN for a query that is not finite."""
    c = _case(dtype, 8, 2, 128, lens=(300, 50), new=[new, 1])
    c["q"][:, :, 7].abs_()
    used = c["table"][0][c["table"][0] >= 0].long()
    c["k"][used, 1, :, 7] = -math.inf
    c["v"][int(used[0]), 1, 0, 3] = math.inf
    got = _check(c)
    assert float(got[:new, 4:].abs().max()) == 0.0 and bool((got[:new, :4].abs().amax(2) > 0).all())
    c["q"][0, 5, 0], c["q"][0, 1, 7], c["q"][-1, 0, 3] = math.inf, math.nan, -math.inf
    got = _run(c)
    assert bool(torch.isnan(got[0, 5]).all() and torch.isnan(got[0, 1]).all() and torch.isnan(got[-1, 0]).all())


def test_a_stored_key_over_the_types_range():
    """rope_kv_store rounds a key of 1e6 to infinity in f16: where the query is of the other sign it weighs nothing."""
    import ggml_hip as G
    c = _case("f16", 8, 2, 64, page=16, lens=(100,), new=[1])
    kv, (page, slot) = G.PagedKV(c["k"], c["v"]), _at(c, 0, 40)
    new = torch.randn((1, 2, 64), generator=torch.Generator("cuda").manual_seed(5), device="cuda")
    new[0, :, 11] = 1e6
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    G.rope_kv_store(None, new, new, i32(0), G.rope_steps(64)[0], kv, i32(page * 16 + slot))
    assert bool((c["k"][page, :, slot, 11] == math.inf).all())
    c["v"][page, :, slot, 11] = 0.0
    c["q"][:, :, 11].abs_().neg_()
    assert bool(torch.isfinite(_check(c)).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("form", FORMS)
def test_infinite_values(form, dim, dtype):
    """In the first, a middle and the last tile, alone and where an infinity of the other sign follows."""
    _, _, seqs, new, n = form
    c = _case(dtype, 8, 4, dim, page=32, lens=[n] * seqs, new=[new] * seqs)
    clean, v, inf = _run(c, decode=False), c["v"], math.inf
    for token, h, d, x in ((0, 0, 3, inf), (n // 2, 0, 5, -inf), (n - 1, 0, 7, inf), (1, 1, 3, inf), (n - 1, 1, 3, -inf),
                           (n - 1 - new // 2, 2, dim - 1, math.nan), (n - 1 - new // 3, 2, dim - 2, inf)):
        page, slot = _at(c, 0, token)
        v[page, h, slot, d] = x
    got = _check(c)
    assert torch.equal(got[:, 6:], clean[:, 6:]) and torch.equal(got[new:], clean[new:])
    _check(c, window=max(1, n // 3), sinks=2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("most", [30, 380])
def test_many_short_sequences(most, dim, dtype):
    """A wave for each: keys and values that are not finite in some of them."""
    lens = [most, 0, 1, most - 1] + [(37 * i) % most for i in range(13)]
    c = _case(dtype, 64, 64, dim, page=16, lens=lens)
    clean = _run(c)
    for s, h, token, where, x in ((0, 1, most - 1, "k", math.inf), (0, 2, 0, "k", -math.inf), (0, 3, 0, "v", math.inf),
                                  (2, 4, 0, "k", -math.inf), (2, 4, 0, "v", math.nan), (3, 5, most - 2, "k", math.nan)):
        page, slot = _at(c, s, token)
        c[where][page, h, slot, 6] = x
    got = _check(c)
    assert torch.equal(got[4:], clean[4:]) and torch.equal(got[:, 6:], clean[:, 6:])
