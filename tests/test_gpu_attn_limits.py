"""Attention over the paged cache (hip_qmm_attn_paged) at the ends of what its
arguments may hold."""
import pytest

import attn_ref as R
from test_gpu_attn import _case, _check, _hold, _run

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,up", [("bf16", 121), ("f16", 13)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,new", [((300, 77), 1), ((5000,), 1), ((300, 77), 40), ((3000,), 15), ((700, 400), 300)])
def test_large_queries(lens, new, dim, dtype, up):
    """Queries far over 1 that small keys meet, some keys all zeros: scores of a few units, and 0."""
    c = _case(dtype, dim=dim, lens=lens, new=[new] * len(lens))
    c["q"] *= 2.0 ** up
    gen = torch.Generator("cuda").manual_seed(3)
    size = 0.5 + torch.rand(c["k"].shape, generator=gen, device="cuda")  # normal numbers of the type
    c["k"].copy_(torch.copysign(size, c["k"].float()) * 2.0 ** -up)
    c["k"][:, :, 5] = 0.0
    assert torch.isfinite(c["q"]).all() and bool((c["k"][:, :, 4] != 0).all())
    _check(c)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40, 300])
def test_the_largest_queries_on_keys_of_zero(new, dtype):
    c = _case(dtype, lens=(700, 300), new=[new, new])
    c["q"].copy_(torch.copysign(torch.full_like(c["q"], 3.4e38), c["q"]))
    c["k"].zero_()
    _check(c)


def test_planned_for_more_workgroups_than_a_launch_has():
    """2048 sequences of 64 heads planned for 2^20 tokens: fewer splits than such a length would have alone."""
    import ggml_hip as G
    c = _case("f16", 64, 64, 64, lens=[40000] + [1 + i % 16 for i in range(2047)])
    c["table"] = torch.nn.functional.pad(c["table"], (0, 65536 - c["table"].shape[1]), value=-1)
    rows, splits = G.attn_paged_plan(G.PagedKV(c["k"], c["v"]), 64, 2048, 2048, 1, 1 << 20)
    assert rows == 16 and splits > 2 and splits * 64 * 2048 <= 1 << 23
    got = _run(c)
    exact = _run(c, max_kv=40000)
    for s in (slice(0, 1), slice(1, 40), slice(2000, 2048)):
        want, top = R.attention(c["q"][s], c["k"], c["v"], c["table"][s], c["lens"][s], c["starts"][:s.stop - s.start + 1],
                                64 ** -0.5)
        _hold(got[s], want, top, 64)
        _hold(exact[s], want, top, 64)


@pytest.mark.parametrize("pages", [40, 9000])
def test_compaction_of_tables_without_entries(pages):
    """No table, no lengths: no page is in use, in one launch and in two."""
    import ctypes as C

    import ggml_hip as G
    from ggml_hip import attn as A
    k = torch.randn((pages, 1, 16, 8), device="cuda").half()
    kv, want = G.PagedKV(k, k.clone()), k.clone()
    size = A._lib().hip_qmm_kv_compact_workspace_size(kv._p)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    live = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert A._lib().hip_qmm_kv_compact(kv._p, None, 0, 0, None, 5, None, 0, live.data_ptr(), ws.data_ptr(), size, stream) == 0
    assert live.tolist() == [0]
    table, n = G.compact_pages(kv, torch.zeros((5, 0), dtype=torch.int32, device="cuda"),
                               torch.full((5,), 100, dtype=torch.int32, device="cuda"))
    assert table.shape == (5, 0) and n.tolist() == [0]
    table, n = G.compact_pages(kv, torch.zeros((0, 4), dtype=torch.int32, device="cuda"),
                               torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert table.shape == (0, 4) and n.tolist() == [0] and torch.equal(kv.k, want)
