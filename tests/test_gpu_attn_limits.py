"""Attention over the paged cache (hip_qmm_attn_paged) at the ends of what its
arguments may hold."""
import pytest

from test_gpu_attn import _case, _check

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
