"""The 8-bit products in workspaces of exactly the size that they ask for: the
same bits as with their own, and nothing before or behind is written."""
import numpy as np
import pytest

import ggml_hip as G
from ggml_hip import moe as M

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

GUARD = 1 << 16


def _exactly(need, call):
    guarded = torch.full((2 * GUARD + need,), 0x5A, dtype=torch.uint8, device="cuda")
    got = call(guarded[GUARD:GUARD + need])
    torch.cuda.synchronize()
    assert (guarded[:GUARD] == 0x5A).all() and (guarded[GUARD + need:] == 0x5A).all()
    if need:
        with pytest.raises(G.HipQmmError):
            call(guarded[GUARD:GUARD + need - 1])
    return got


def _weights(r, *shape):
    q = torch.from_numpy(r.randint(-127, 128, (*shape[:-1], -(-shape[-1] // 16) * 16)).astype(np.int8)).cuda()
    return q[..., :shape[-1]], torch.from_numpy(r.rand(*shape[:-1]).astype(np.float32)).cuda()


def _by_experts(ids, e, rows, K, slots, f32):
    r = np.random.RandomState(rows)
    n, k = ids.shape
    w, ws = _weights(r, e, rows, K)
    x, scale = torch.randn(n, k if slots else 1, K, device="cuda"), None
    if not f32:
        x, scale = G.quantize_i8(x)
    need = M._lib().hip_qmm_mul_mat_id_i8_workspace_size(K, rows, e, x.shape[1], n, k, int(not f32))
    ids = torch.from_numpy(ids.astype(np.int32)).cuda()
    want = G.mul_mat_id_i8(w, ws, x, ids, scale)
    assert torch.equal(_exactly(need, lambda space: G.mul_mat_id_i8(w, ws, x, ids, scale, workspace=space)), want)
    return need


# Experts whose columns are one more than whole tiles, so that there are as many tiles as there can be: of 64 x 64,
# 128 x 64, 128 x 128 and 256 x 256, in one chunk of 4096 pairs and in several.
@pytest.mark.parametrize("e,columns,rows,K", [(16, 65, 100, 70), (100, 65, 40, 33), (16, 65, 2048, 130), (64, 65, 700, 48),
                                              (16, 129, 4096, 200), (40, 129, 4000, 100), (24, 513, 4096, 1030)])
@pytest.mark.parametrize("f32", [False, True])
def test_as_many_tiles_as_there_can_be(e, columns, rows, K, f32):
    ids = np.random.RandomState(e).permutation(np.repeat(np.arange(e), columns))[:, None]
    assert _by_experts(ids, e, rows, K, False, f32) > 0


@pytest.mark.parametrize("n,k,e", [(1, 8, 128), (1, 2, 3), (9, 8, 128), (48, 8, 128), (64, 8, 60), (65, 8, 1024), (513, 1, 7), (513, 8, 1024),
                                   (2048, 2, 2), (2049, 2, 300)])
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_pairs(n, k, e, slots, f32):
    _by_experts(np.random.RandomState(n).randint(-1, e + 1, (n, k)), e, 50, 129, slots, f32)


@pytest.mark.parametrize("rows,K,n", [(300, 1, 1), (300, 2061, 1), (300, 2061, 16), (300, 16384, 2), (300, 2061, 17), (40, 129, 33),
                                      (9000, 127, 40), (5003, 128, 333), (300, 20001, 100), (4096, 300, 2100)])
@pytest.mark.parametrize("f32", [False, True])
def test_columns(rows, K, n, f32):
    r = np.random.RandomState(K)
    w, ws = _weights(r, rows, K)
    x, scale = torch.randn(n, K, device="cuda"), None
    if not f32:
        x, scale = G.quantize_i8(x)
    need = M._lib().hip_qmm_mul_mat_i8_workspace_size(K, rows, n, int(not f32))
    want = G.mul_mat_i8(w, ws, x, scale)
    assert torch.equal(_exactly(need, lambda space: G.mul_mat_i8(w, ws, x, scale, workspace=space)), want)
