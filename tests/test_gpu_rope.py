"""Rotary positions and the store into the paged cache (hip_qmm_rope_f32,
hip_qmm_rope_kv_store) against their f64 definition."""
import math

import pytest

import attn_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# The turn's rounding to f32 (2^-25 of half a turn at most), sin and cos to 2 ulp,
# three f32 operations: under 8 * 2^-24 of the pair's length.
TOL = 8 * 2.0 ** -24


def _freqs(n_dims, base=10000.0):
    return base ** (-torch.arange(0, n_dims, 2, dtype=torch.float64) / n_dims)


def _hold(got, want, x, mscale=1.0):
    # a pair's length is at most sqrt(2) times the largest of its elements' sizes
    size = x.double().abs().amax(-1, keepdim=True) * math.sqrt(2) * mscale + 1e-300
    assert float(((got.double() - want).abs() / size).max()) <= TOL


def _x(*shape, seed=1):
    return torch.randn(shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda")


def _pos(n, lo=0, hi=131072, seed=2):
    return torch.randint(lo, hi, (n,), generator=torch.Generator("cuda").manual_seed(seed), device="cuda").int()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 128, 64), (7, 2, 80, 32),
                                                  (65, 4, 64, 64), (9, 3, 96, 20), (5, 2, 100, 50), (4, 3, 256, 256),
                                                  (2, 2, 1024, 256), (300, 8, 128, 128), (6, 3, 12, 8), (5, 71, 64, 16)])
def test_rope(layout, tokens, heads, dim, rot):
    import ggml_hip as G
    x, pos = _x(tokens, heads, dim), _pos(tokens)
    steps, mscale = G.rope_steps(rot)
    assert mscale == 1.0
    got = G.rope(x, pos, steps, layout)
    _hold(got, R.rope(x, pos, _freqs(rot), layout), x)
    assert torch.equal(got[..., rot:], x[..., rot:])
    same = G.rope(x, pos, steps, layout, out=x)  # in place
    assert same.data_ptr() == x.data_ptr() and torch.equal(same, got)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions(layout):
    """Zero, negative and the largest positions; turning back gives what was there."""
    import ggml_hip as G
    pos = torch.tensor([0, -1, -5000, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1], dtype=torch.int32, device="cuda")
    x = _x(6, 2, 128)
    steps, _ = G.rope_steps(128, 500000.0)
    got = G.rope(x, pos, steps, layout)
    # the f64 angle is exact to 2^-53 of itself: up to 2^31 * 2^-53 radians
    _hold(got, R.rope(x, pos, _freqs(128, 500000.0), layout), x)
    assert torch.equal(got[0], x[0])
    pos[4] = 0  # its negative does not exist
    back = G.rope(G.rope(x, pos, steps, layout), -pos, steps, layout)
    assert float((back - x).abs().max()) <= 2 * TOL * 2 ** 0.5 * float(x.abs().max())


def test_scores_depend_on_the_distance_alone():
    import ggml_hip as G
    x, y = _x(1, 1, 128), _x(1, 1, 128, seed=3)
    steps, _ = G.rope_steps(128, 500000.0)
    at = lambda t, p: G.rope(t, torch.tensor([p], dtype=torch.int32, device="cuda"), steps).double().flatten()  # noqa: E731
    want = float(at(x, 37) @ at(y, 0))
    for p in (1, 999, 131072, 2 ** 24 + 5):
        assert abs(float(at(x, 37 + p) @ at(y, p)) - want) <= 128 * 4 * TOL


def test_scaled_frequencies():
    """Linear scaling, frequency factors and the mixed (YaRN) form, against their formulas."""
    import ggml_hip as G
    f = _freqs(64, 500000.0)
    unit = 2 * math.pi / 2.0 ** 64

    def freq(*a, **kw):
        steps, mscale = G.rope_steps(64, 500000.0, *a, device="cpu", **kw)
        return steps.double() * unit, mscale

    got, _ = freq()
    torch.testing.assert_close(got, f, rtol=1e-15, atol=1e-18)
    got, m = freq(0.25)
    torch.testing.assert_close(got, f / 4, rtol=1e-15, atol=1e-18)
    assert m == 1.0
    factors = torch.linspace(1, 8, 32)
    got, _ = freq(freq_factors=factors)
    torch.testing.assert_close(got, f / factors.double(), rtol=1e-15, atol=1e-18)
    got, m = freq(1 / 8, 1.0, 1.5, n_ctx_orig=8192)
    pair = lambda turns: 64 * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))  # noqa: E731
    low, high = max(0, math.floor(pair(32))), min(63, math.ceil(pair(1)))
    keep = 1 - ((torch.arange(32).double() - low) / (high - low)).clamp(0, 1)
    torch.testing.assert_close(got, f * keep + f / 8 * (1 - keep), rtol=1e-14, atol=1e-18)
    assert m == pytest.approx(1.5 * (1 + 0.1 * math.log(8)), rel=1e-6)
    x, pos = _x(40, 3, 96), _pos(40)
    steps, m = G.rope_steps(64, 500000.0, 1 / 8, 1.0, n_ctx_orig=8192)
    got = G.rope(x, pos, steps, "interleaved", m)
    want = R.rope(x, pos, f * keep + f / 8 * (1 - keep), "interleaved", m)
    _hold(got, want, x, m)


def _store(dtype="f16", tokens=50, heads=8, kv_heads=2, dim=128, rot=128, page=16, layout="half", order="heads"):
    gen = torch.Generator("cuda").manual_seed(5)
    pages = -(-tokens // page) + 2
    k_cache, v_cache = R.make_cache(gen, R.DTYPES[dtype], pages, kv_heads, page, dim, order=order)
    slots = torch.randperm(pages * page, generator=gen, device="cuda")[:tokens].int()
    return (_x(tokens, heads, dim), _x(tokens, kv_heads, dim, seed=6), _x(tokens, kv_heads, dim, seed=7), _pos(tokens),
            slots, k_cache, v_cache)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot,page,order", [
    (1, 32, 8, 128, 128, 64, "heads"), (1, 1, 1, 8, 2, 16, "heads"), (77, 8, 2, 128, 64, 16, "tokens"),
    (33, 6, 6, 80, 32, 32, "heads"), (20, 5, 1, 72, 20, 16, "heads"), (600, 4, 2, 64, 64, 128, "heads"),
    (9, 3, 3, 256, 256, 16, "tokens")])
def test_store(layout, dtype, tokens, heads, kv_heads, dim, rot, page, order):
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store(dtype, tokens, heads, kv_heads, dim, rot, page, layout, order)
    steps, _ = G.rope_steps(rot)
    kw, vw = kc.clone(), vc.clone()
    at, off = slots.long() // page, slots.long() % page
    rk = G.rope(k, pos, steps, layout)
    kw[at, :, off], vw[at, :, off] = rk.to(kc.dtype), v.to(vc.dtype)
    got = G.rope_kv_store(q, k, v, pos, steps, G.PagedKV(kc, vc), slots, layout)
    assert torch.equal(got, G.rope(q, pos, steps, layout))
    assert torch.equal(kc, kw) and torch.equal(vc, vw)
    # keys and values alone
    kc.zero_()
    vc.zero_()
    assert G.rope_kv_store(None, k, v, pos, steps, G.PagedKV(kc, vc), slots, layout) is None
    assert torch.equal(kc[at, :, off], rk.to(kc.dtype)) and torch.equal(vc[at, :, off], v.to(vc.dtype))


def test_slots_outside_the_cache_store_nothing():
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store()
    steps, _ = G.rope_steps(128)
    total = kc.shape[0] * 16
    kw, vw = kc.clone(), vc.clone()
    bad = torch.tensor([-1, total, 2 ** 31 - 1, -2 ** 31, -17] * 10, dtype=torch.int32, device="cuda")
    got = G.rope_kv_store(q, k, v, pos, steps, G.PagedKV(kc, vc), bad)
    assert torch.equal(kc, kw) and torch.equal(vc, vw) and torch.equal(got, G.rope(q, pos, steps))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_what_the_cache_cannot_hold(dtype):
    """Over the type's range becomes infinite, NaN stays, zeros and signs too, ties round to even: as torch converts."""
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store(dtype)
    v[0, 0, :8] = torch.tensor([1e6, -1e6, math.nan, math.inf, -0.0, 1e-9, 65519.9, 1.00048828125])
    v[1, 1, :2] = torch.tensor([3.3e38, 1.00390625])
    steps, _ = G.rope_steps(128)
    G.rope_kv_store(q, k, v, pos, steps, G.PagedKV(kc, vc), slots)
    got = vc[slots.long() // 16, :, slots.long() % 16]
    want = v.to(vc.dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float(), 7.0), torch.nan_to_num(want.float(), 7.0))
    assert torch.signbit(got[0, 0, 4])


def test_parts_of_a_fused_projection_and_strided_results():
    """q, k and v as views of one [tokens, (heads + 2 kv_heads) * dim] row, the result in a wider one; any alignment."""
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store()
    steps, _ = G.rope_steps(128)
    want = G.rope(q, pos, steps)
    G.rope_kv_store(None, k, v, pos, steps, G.PagedKV(kc, vc), slots)
    for pad in (0, 1, 4):
        row = torch.full((50, 12 * 128 + 2 * pad), math.nan, device="cuda")[:, pad:pad + 12 * 128]
        row[:, :1024], row[:, 1024:1280], row[:, 1280:] = q.flatten(1), k.flatten(1), v.flatten(1)
        parts = [row[:, a:b].unflatten(1, (-1, 128)) for a, b in ((0, 1024), (1024, 1280), (1280, 1536))]
        out = torch.full((50, 9, 128 + pad), 5.0, device="cuda")
        kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
        G.rope_kv_store(*parts, pos, steps, G.PagedKV(kc2, vc2), slots, out=out[:, :8, pad:])
        assert torch.equal(out[:, :8, pad:], want)
        out[:, :8, pad:] = 5.0
        assert bool((out == 5.0).all())
        at = (slots.long() // 16, slice(None), slots.long() % 16)
        assert torch.equal(kc2[at], kc[at]) and torch.equal(vc2[at], vc[at])


def test_in_a_graph_and_on_another_stream():
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store()
    steps, _ = G.rope_steps(128)
    kv = G.PagedKV(kc, vc)
    out = torch.empty_like(q)
    G.rope_kv_store(q, k, v, pos, steps, kv, slots, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        G.rope_kv_store(q, k, v, pos, steps, kv, slots, out=out)
    for _ in range(3):
        q.normal_()
        pos += 11
        want = G.rope(q, pos, steps)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = G.rope(q, pos, steps)
    side.synchronize()
    assert torch.equal(got, want)


def test_offsets_past_32_bits():
    import ggml_hip as G
    q, k, v, pos, slots, kc, vc = _store()
    steps, _ = G.rope_steps(128)
    pages = (2 ** 31 + 2 ** 27) // (2 * 16 * 128)
    far_k = torch.empty((pages, 2, 16, 128), dtype=torch.float16, device="cuda")
    far_v = torch.empty_like(far_k)
    G.rope_kv_store(None, k, v, pos, steps, G.PagedKV(kc, vc), slots)
    move = (pages - kc.shape[0]) * 16
    G.rope_kv_store(None, k, v, pos, steps, G.PagedKV(far_k, far_v), slots + move)
    at = (slots.long() // 16, slice(None), slots.long() % 16)
    far = (at[0] + move // 16, slice(None), at[2])
    assert torch.equal(far_k[far], kc[at]) and torch.equal(far_v[far], vc[at])
