"""The entry points of include/ggml_hip_moe.h on the CPU: every declared one is
exported, and what they do not take is refused before anything is launched."""
import math
import re

import pytest

import ggml_hip as G
from ggml_hip import moe as M

HEADER = G.PKG_DIR.parent / "include" / "ggml_hip_moe.h"
BAD = 1  # hipErrorInvalidValue
P = 1 << 20  # an aligned address that nothing reads: every call here is refused or empty


def test_declared_entry_points_are_exported():
    names = set(re.findall(r"\b(hip_qmm_\w+)\(", HEADER.read_text())) - {"hip_qmm_mul_mat_id"}
    assert {"hip_qmm_moe_route", "hip_qmm_quantize_i8", "hip_qmm_mul_mat_i8", "hip_qmm_mul_mat_id_i8",
            "hip_qmm_moe_combine", "hip_qmm_mul_mat_i8_workspace_size", "hip_qmm_mul_mat_id_i8_workspace_size"} <= names
    L = M._lib()
    assert all(hasattr(L, n) for n in names)


def _route(**kw):
    f = dict(logits=P, n=1, e=64, ls=64, bias=None, gating=0, groups=1, keep=1, top=1, k=4, renorm=0, min_sum=0.0, scale=1.0,
             ids=P, si=4, w=P, sw=4)
    f.update(kw)
    return M._lib().hip_qmm_moe_route(*f.values(), None)


def test_route_refusals():
    assert _route(n=0) == 0 and _route(n=0, logits=None, ids=None, w=None) == 0
    for kw in (dict(n=-1), dict(n=(1 << 24) + 1), dict(e=0), dict(e=1025, ls=1025), dict(gating=-1), dict(gating=3), dict(k=0),
               dict(k=65, e=128, ls=128, si=65, sw=65), dict(k=5, e=4), dict(groups=0), dict(groups=65, e=130, ls=130),
               dict(groups=3), dict(keep=0), dict(groups=4, keep=5), dict(top=0), dict(top=3), dict(min_sum=-1.0),
               dict(min_sum=math.nan), dict(min_sum=math.inf), dict(scale=math.nan), dict(scale=math.inf), dict(logits=None),
               dict(ids=None), dict(w=None), dict(ls=63), dict(si=3), dict(sw=3), dict(ls=1 << 50), dict(ls=-64)):
        assert _route(**kw) == BAD, kw


def _quantize(**kw):
    f = dict(x=P, K=64, n=1, xs=64, q=P, qs=64, scale=P)
    f.update(kw)
    return M._lib().hip_qmm_quantize_i8(*f.values(), None)


def test_quantize_refusals():
    assert _quantize(n=0) == 0
    for kw in (dict(K=0), dict(K=131072, xs=131072, qs=131072), dict(n=-1), dict(n=(1 << 24) + 1), dict(x=None), dict(q=None),
               dict(scale=None), dict(xs=63), dict(qs=63), dict(xs=1 << 50), dict(qs=-1)):
        assert _quantize(**kw) == BAD, kw


def _product(**kw):
    f = dict(w=P, ws=P, K=64, rows=32, stride=64, x=P, xs=P, n=4, x_stride=64, dst=P, dst_stride=32, workspace=P, size=1 << 40)
    f.update(kw)
    return M._lib().hip_qmm_mul_mat_i8(*f.values(), None)


def test_product_refusals():
    assert _product(n=0) == 0
    for kw in (dict(K=0), dict(K=131072, stride=131072, x_stride=131072), dict(rows=0), dict(rows=(1 << 22) + 1), dict(n=-1),
               dict(n=(1 << 22) + 1), dict(w=None), dict(ws=None), dict(x=None), dict(dst=None), dict(stride=63), dict(stride=72),
               dict(stride=48), dict(w=P + 8), dict(x=P + 4), dict(x_stride=72), dict(x_stride=48), dict(dst_stride=31),
               dict(xs=None, x_stride=63), dict(xs=None, x=P + 2), dict(stride=1 << 50), dict(x_stride=1 << 50),
               dict(dst_stride=1 << 50)):
        assert _product(**kw) == BAD, kw
    need = M._lib().hip_qmm_mul_mat_i8_workspace_size(64, 32, 400, 0)
    assert need >= 400 * 68
    for kw in (dict(size=need - 1), dict(workspace=None), dict(workspace=P + 128)):
        assert _product(**kw, xs=None, n=400) == BAD, kw
    f = M._lib().hip_qmm_mul_mat_i8_workspace_size
    for K in (1, 127, 128, 129, 4096, 131071):
        for n in (1, 2, 16, 17, 33, 1000, 1 << 22):
            assert f(K, 500, n, 0) <= n * (K + 131) + 512 and f(K, 500, n, 1) == 0
    assert f(0, 32, 4, 0) == f(64, 0, 4, 0) == f(64, 32, 0, 0) == f(64, 32, -1, 1) == 0


def _by_experts(**kw):
    f = dict(w=P, ws=P, K=64, rows=32, stride=64, es=2048, e=8, x=P, xs=P, ne11=1, n=4, x_stride=64, ids=P, n_ids=2, si=2,
             dst=P, dst_stride=32, workspace=P, size=1 << 40)
    f.update(kw)
    return M._lib().hip_qmm_mul_mat_id_i8(*f.values(), None)


def test_product_by_experts_refusals():
    assert _by_experts(n=0) == 0 and _by_experts(n_ids=0) == 0
    for kw in (dict(K=0), dict(K=131072, stride=131072, es=1 << 30, x_stride=131072), dict(rows=0), dict(e=0), dict(e=1025),
               dict(n=-1), dict(n_ids=-1), dict(n=1 << 22, n_ids=2), dict(n=1 << 40), dict(ne11=3), dict(ne11=0), dict(w=None),
               dict(ws=None), dict(x=None), dict(ids=None), dict(dst=None), dict(si=1), dict(dst_stride=31), dict(stride=72),
               dict(stride=48), dict(es=2047), dict(es=1024), dict(es=0), dict(es=-2048), dict(w=P + 1), dict(x=P + 8),
               dict(x_stride=63), dict(si=1 << 50), dict(es=1 << 50)):
        assert _by_experts(**kw) == BAD, kw
    for quantized in (0, 1):
        need = M._lib().hip_qmm_mul_mat_id_i8_workspace_size(64, 32, 8, 1, 400, 2, quantized)
        assert need >= 800 * 8
        for kw in (dict(size=need - 1), dict(workspace=None), dict(workspace=P + 128)):
            assert _by_experts(**kw, n=400, xs=P if quantized else None) == BAD, kw
    f = M._lib().hip_qmm_mul_mat_id_i8_workspace_size
    assert f(64, 32, 8, 3, 400, 2, 1) == f(64, 32, 0, 1, 400, 2, 1) == f(64, 32, 8, 1, 0, 2, 1) == 0


def _combine(**kw):
    f = dict(y=P, n=2, n_ids=4, rows=16, yt=64, ys=16, w=P, sw=4, ids=P, si=4, add=P, sa=16, dst=P + 4096, so=16)
    f.update(kw)
    return M._lib().hip_qmm_moe_combine(*f.values(), None)


def test_combine_refusals():
    assert _combine(n=0) == 0 and _combine(rows=0) == 0
    for kw in (dict(n=-1), dict(n=1 << 31), dict(n_ids=-1), dict(n_ids=65536), dict(rows=-1), dict(rows=1 << 31), dict(y=None),
               dict(w=None), dict(dst=None), dict(sw=3), dict(si=3), dict(sa=15), dict(so=15), dict(yt=-1), dict(ys=-16),
               dict(add=P + 4096, sa=20), dict(so=1 << 50), dict(yt=1 << 50)):
        assert _combine(**kw) == BAD, kw


def test_python_refusals_without_a_gpu():
    torch = pytest.importorskip("torch")
    f, b, i = torch.zeros(2, 16), torch.zeros((2, 16), dtype=torch.int8), torch.zeros((2, 1), dtype=torch.int32)
    for call in (lambda: G.route(f, 2), lambda: G.quantize_i8(f), lambda: G.mul_mat_i8(b, f[:, 0], f),
                 lambda: G.mul_mat_id_i8(b[None], f[:1, :2], f[:, None], i), lambda: G.combine(f[:, None], f[:, :1])):
        with pytest.raises(G.HipQmmError):
            call()


@pytest.mark.parametrize("call,names", [(_route, ("logits", "bias", "ids", "w")), (_quantize, ("x", "scale")),
                                        (_product, ("ws", "xs", "dst")), (_by_experts, ("ws", "xs", "ids", "dst")),
                                        (_combine, ("y", "w", "ids", "add", "dst"))])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_tensors_at_odd_bytes(call, names, off):
    for name in names:
        assert call(**{name: P + off}) == BAD, name
