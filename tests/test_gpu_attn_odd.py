"""Attention over the paged cache (hip_qmm_attn_paged) where queries, keys or
values are not finite: only the results that they belong to are touched, in
every kernel form, type and head size, whichever tile holds them."""
import math

import pytest

import attn_ref as R
from test_gpu_attn import _case, _run

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
