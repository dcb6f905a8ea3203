"""A mixture-of-experts layer on the operators together: router's scores to
experts and weights, 8-bit gate and up products, SwiGLU, the down product, the
weighted sum with a shared expert; and the router's choice in front of the
block-quantized experts.  Every stage is checked from what the one before it
gave, with that operator's own bound."""
import numpy as np
import pytest

import ggml_hip as G
import moe_ref as R
import oracle_lib as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E, K_EXPERTS, WIDTH, INNER = 32, 4, 512, 192


class Layer:
    def __init__(self, seed=1):
        gen = torch.Generator("cuda").manual_seed(seed)
        def weights(*shape):
            return G.quantize_i8(torch.randn(shape, generator=gen, device="cuda") * shape[-1] ** -0.5)
        self.router = torch.randn(E, WIDTH, generator=gen, device="cuda") * WIDTH ** -0.5
        self.bias = torch.randn(E, generator=gen, device="cuda") * 0.1
        self.up, self.down = weights(E, 2 * INNER, WIDTH), weights(E, WIDTH, INNER)
        self.shared_up, self.shared_down = weights(2 * INNER, WIDTH), weights(WIDTH, INNER)

    def __call__(self, x):
        n = x.shape[0]
        logits = x @ self.router.T.contiguous()
        ids, weights = G.route(logits, K_EXPERTS, gating="sigmoid", bias=self.bias, groups=8, keep=4, renormalize=True,
                               scale=2.5)
        both = G.mul_mat_id_i8(*self.up, x[:, None], ids)
        rows = both.view(-1, 2 * INNER)
        h = G.glu_f32(rows[:, :INNER], rows[:, INNER:]).view(n, K_EXPERTS, INNER)
        y = G.mul_mat_id_i8(*self.down, h, ids)
        own = G.mul_mat_i8(*self.shared_up, x)
        own_h = G.glu_f32(own[:, :INNER], own[:, INNER:])
        shared = G.mul_mat_i8(*self.shared_down, own_h)
        out = G.combine(y, weights, ids=ids, add=shared)
        return dict(logits=logits, ids=ids, weights=weights, both=both, h=h, y=y, own=own, own_h=own_h, shared=shared, out=out)


def _close(got, want, tol=3 * R.U * (1 + 1e-6)):
    got = got.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= tol * np.abs(want) + 2.0 ** -149)


def _check(layer, x, s):
    n = lambda t: t.cpu().numpy()  # noqa: E731
    ids, weights = R.route(n(s["logits"]), K_EXPERTS, "sigmoid", n(layer.bias), 8, 4, renormalize=True, scale=2.5)
    assert np.array_equal(n(s["ids"]), ids)
    _close(s["weights"], weights, R.U + 1e-12)
    for name, w, x_of in (("both", layer.up, x[:, None]), ("y", layer.down, s["h"])):
        q, d = R.quantize(n(x_of))
        _close(s[name], R.product_id(n(w[0]), n(w[1]), q, d, ids))
    for name, w, x_of in (("own", layer.shared_up, x), ("shared", layer.shared_down, s["own_h"])):
        _close(s[name], R.product(n(w[0]), n(w[1]), *R.quantize(n(x_of))))
    want, size = R.combine(n(s["y"]), n(s["weights"]), ids, n(s["shared"]))
    off = np.abs(s["out"].double().cpu().numpy() - want)
    assert np.all(off <= (K_EXPERTS + 1) * R.U * size * (1 + 1e-6))


@pytest.mark.parametrize("n", [1, 2, 9, 150, 1300])
def test_layer(n):
    layer = Layer()
    x = torch.randn(n, WIDTH, device="cuda")
    _check(layer, x, layer(x))


@pytest.mark.parametrize("n", [1, 7, 300])
def test_captured_layer(n):
    """Replays with new tokens, the program's own calls between them."""
    layer = Layer(2)
    x = torch.randn(n, WIDTH, device="cuda")
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer(x)
    for i in range(4):
        x.copy_(torch.randn(n, WIDTH, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        eager = layer(x)
        for name, t in got.items():
            if name != "logits":  # a library product
                assert torch.equal(t, eager[name]) or not torch.equal(got["logits"], eager["logits"]), (i, name)
        _check(layer, x, got)


@pytest.mark.parametrize("n", [1, 20, 100])
def test_choice_before_block_quantized_experts(n):
    """Ids and -1 as hip_qmm_mul_mat_id takes them: hidden experts, places with none left."""
    rows, K, e, k = 64, 256, 8, 3
    w = O.fill_normal(7, e * rows * K, 0.0, 0.05).reshape(e * rows, K)
    wq = O.quantize_rows(O.TYPE_Q8_0, w)
    x = torch.randn(n, 1, K, device="cuda")
    logits = torch.randn(n, e, device="cuda")
    logits[:, 2] = -float("inf")
    logits[n // 2, 1:] = -float("inf")
    ids, weights = G.route(logits, k, renormalize=True)
    assert (ids != 2).all() and ids[n // 2].tolist() == [0, -1, -1]
    y = G.mul_mat_id("Q8_0", torch.from_numpy(wq).cuda().view(e, rows, -1), x, ids)
    assert (y[n // 2, 1:] == 0).all()
    want = O.mul_mat_id(O.TYPE_Q8_0, wq, e, rows, K, x.cpu().numpy(), ids.cpu().numpy()).reshape(n, k, rows)
    off = (y.cpu().numpy().astype(np.float64) - want) ** 2
    assert off.sum() < 5e-4 * (want.astype(np.float64) ** 2).sum()  # that operator's bound
    total, size = R.combine(y.cpu().numpy(), weights.cpu().numpy(), ids.cpu().numpy())
    got = G.combine(y, weights, ids=ids).double().cpu().numpy()
    assert np.all(np.abs(got - total) <= (k + 1) * R.U * size * (1 + 1e-6))
