"""A mixture-of-experts layer from given router scores in captured graphs: every
stage of every replay has the bits of the eager layer."""
import pytest

import ggml_hip as G
from test_gpu_moe_layer import E, INNER, K_EXPERTS, WIDTH, Layer

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _stages(layer, x, logits):
    n = x.shape[0]
    ids, weights = G.route(logits, K_EXPERTS, gating="sigmoid", bias=layer.bias, groups=8, keep=4, renormalize=True, scale=2.5)
    both = G.mul_mat_id_i8(*layer.up, x[:, None], ids)
    rows = both.view(-1, 2 * INNER)
    h = G.glu_f32(rows[:, :INNER], rows[:, INNER:]).view(n, K_EXPERTS, INNER)
    y = G.mul_mat_id_i8(*layer.down, h, ids)
    q, scale = G.quantize_i8(x)
    own = G.mul_mat_i8(*layer.shared_up, q, scale)
    own_h = G.glu_f32(own[:, :INNER], own[:, INNER:])
    shared = G.mul_mat_i8(*layer.shared_down, own_h)
    return dict(ids=ids, weights=weights, both=both, h=h, y=y, q=q, scale=scale, own=own, shared=shared,
                out=G.combine(y, weights, ids=ids, add=shared))


def _random(n, *into):
    new = (torch.randn(n, WIDTH, device="cuda"), torch.randn(n, E, device="cuda") * 2)
    new[1][torch.rand(n, E, device="cuda") < 0.1] = -float("inf")
    for to, t in zip(into, new):
        to.copy_(t)
    return new


class Captured:
    def __init__(self, layer, n):
        self.layer, self.given = layer, _random(n)
        _stages(layer, *self.given)
        torch.cuda.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.got = _stages(layer, *self.given)

    def check(self):
        want = _stages(self.layer, *self.given)
        for name, t in self.got.items():
            assert torch.equal(t, want[name]), name


@pytest.mark.parametrize("n", [1, 7, 300, 2500])
def test_replays(n):
    layer = Captured(Layer(2), n)
    for _ in range(4):
        _random(n, *layer.given)
        layer.graph.replay()
        torch.cuda.synchronize()
        layer.check()


def test_two_graphs_in_turn():
    """Each with workspaces of its own."""
    both = [Captured(Layer(s), n) for s, n in ((3, 40), (4, 1100))]
    for i in range(4):
        for one in both:
            _random(one.given[0].shape[0], *one.given)
            one.graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        for one in both:
            one.check()
