"""8-bit integer products against exact sums scaled in f64.

A result is a whole number converted to f32 and two products: three roundings of
half a step (2^-24) each, (1 + u)^3 - 1 < 3 u (1 + 1e-6).  Quantizing gives the definition's integers and scales
exactly."""
import numpy as np
import pytest

import ggml_hip as G
import moe_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TOL = 3 * R.U * (1 + 1e-6)


def _near(got, want):
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    want = np.where(np.abs(want) >= np.finfo(np.float32).max * (1 + R.U), np.copysign(np.inf, want), want)
    assert np.array_equal(np.isinf(got), np.isinf(want)) and np.array_equal(got[np.isinf(got)], want[np.isinf(got)])
    fine &= np.isfinite(want)
    off = np.abs(got[fine] - want[fine])
    assert np.all(off <= TOL * np.abs(want)[fine] + 2.0 ** -149)


def _rows(r, *shape, full=False):
    """int8 on the GPU in rows as the products take them, garbage in their padding, and on the CPU."""
    lo = -128 if full else -127
    q = r.randint(lo, 128, (*shape[:-1], (shape[-1] + 15) // 16 * 16)).astype(np.int8)
    return torch.from_numpy(q).cuda()[..., :shape[-1]], q[..., :shape[-1]]


def _scales(r, *shape):
    s = (r.rand(*shape) + 0.5).astype(np.float32) * np.float32(1e-3)
    return torch.from_numpy(s).cuda(), s


INNER = [1, 15, 16, 17, 63, 64, 100, 127, 128, 129, 200, 256, 383, 1000, 1024, 2061, 4096]


@pytest.mark.parametrize("K", INNER)
@pytest.mark.parametrize("rows,n", [(1, 1), (17, 3), (64, 16), (100, 33), (257, 130)])
def test_product_of_integers(K, rows, n):
    r = np.random.RandomState(K + rows)
    w, wn = _rows(r, rows, K, full=True)
    x, xn = _rows(r, n, K, full=True)
    (ws, wsn), (xs, xsn) = _scales(r, rows), _scales(r, n)
    _near(G.mul_mat_i8(w, ws, x, xs), R.product(wn, wsn, xn, xsn))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 192, 255, 256,
                               257, 300, 511, 513, 1100])
@pytest.mark.parametrize("rows,K", [(513, 300), (256, 1024)])
def test_numbers_of_columns(n, rows, K):
    r = np.random.RandomState(n)
    w, wn = _rows(r, rows, K)
    (ws, wsn), x = _scales(r, rows), r.randn(n, K).astype(np.float32)
    q, s = R.quantize(x)
    _near(G.mul_mat_i8(w, ws, torch.from_numpy(x).cuda()), R.product(wn, wsn, q, s))


@pytest.mark.parametrize("rows,K,n", [(4096, 14336, 1), (14336, 4096, 24), (5003, 2720, 333), (1024, 131071, 2),
                                      (300, 131071, 300), (40, 131071, 1), (2048, 768, 1), (1000, 4096, 700), (2304, 4096, 2100)])
def test_large_products(rows, K, n):
    r = np.random.RandomState(1)
    w, wn = _rows(r, rows, K)
    (ws, wsn), x = _scales(r, rows), r.randn(n, K).astype(np.float32)
    q, s = R.quantize(x)
    want = R.product(wn, wsn, q, s)
    _near(G.mul_mat_i8(w, ws, torch.from_numpy(x).cuda()), want)
    qd, sd = G.quantize_i8(torch.from_numpy(x).cuda())
    _near(G.mul_mat_i8(w, ws, qd, sd), want)


@pytest.mark.parametrize("n", [1, 20, 200])
def test_largest_sums(n):
    w = torch.full((40, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
    x = torch.full((n, 131072), -128, dtype=torch.int8, device="cuda")[:, :131071]
    one = torch.ones(40, device="cuda")
    got = G.mul_mat_i8(w, one, x, torch.ones(n, device="cuda"))
    assert (got == float(np.float32(131071 * 16384))).all()


@pytest.mark.parametrize("K", [1, 3, 4, 16, 63, 64, 65, 100, 768, 1023, 1024, 2049, 4096, 14336, 20001, 131071])
@pytest.mark.parametrize("n", [1, 5])
def test_quantize(K, n):
    r = np.random.RandomState(K)
    x = (r.randn(n, K) * np.exp(r.randn(n, 1) * 5)).astype(np.float32)
    q, s = G.quantize_i8(torch.from_numpy(x).cuda())
    wq, wsc = R.quantize(x)
    assert q.shape == x.shape and (q.stride(0) % 16 == 0 or n == 1)
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), wsc)


def test_quantize_what_it_can_meet():
    K = 300
    x = np.random.RandomState(3).randn(12, K).astype(np.float32)
    x[0] = 0.0
    x[1, 299] = np.nan
    x[2, 0] = np.inf
    x[3, 5] = -np.inf
    x[4] *= np.float32(1e-44) / 4          # below 127 of the smallest steps: the scale is 0
    x[5] = np.linspace(-1, 1, K) * 1e-43   # a scale of few bits
    x[6] = np.arange(K) % 255 - 127        # whole numbers
    x[7] = (np.arange(K) % 254 - 127) + 0.5  # halves: to even
    x[7, 0] = 127
    x[8] *= np.float32(3e38) / np.abs(x[8]).max()
    x[9, 1:] = 0.0
    x[10] = -0.0
    wq, ws = R.quantize(x)
    q, s = G.quantize_i8(torch.from_numpy(x).cuda())
    assert np.array_equal(q.cpu().numpy(), wq) and np.array_equal(s.cpu().numpy(), ws, equal_nan=True)
    # and through products of few and of many columns
    r = np.random.RandomState(4)
    w, wn = _rows(r, 70, K)
    wsc, wscn = _scales(r, 70)
    for n in (1, 2, 4, 6, 12, 120):
        for at in range(0, 12, n) if n < 12 else (0,):
            part = np.tile(x, (10, 1))[at:at + n]
            want = R.product(wn, wscn, *R.quantize(part))
            _near(G.mul_mat_i8(w, wsc, torch.from_numpy(part).cuda()), want)


def test_quantize_given_results_and_strides():
    x = torch.randn(9, 130, device="cuda")[:, 5:95]
    out = torch.full((9, 112), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(9, device="cuda")
    q, s = G.quantize_i8(x, out=out[:, :90], scale=scale)
    wq, ws = R.quantize(x.cpu().numpy())
    assert np.array_equal(out[:, :90].cpu().numpy(), wq) and np.array_equal(scale.cpu().numpy(), ws)
    assert (out[:, 90:] == 77).all()  # what lies behind the rows stays
    tight = torch.empty(9, 90, dtype=torch.int8, device="cuda")
    assert torch.equal(G.quantize_i8(x, out=tight)[0], q)
    w3 = torch.randn(3, 7, 33, device="cuda")
    q3, s3 = G.quantize_i8(w3)
    wq3, ws3 = R.quantize(w3.cpu().numpy())
    assert q3.shape == w3.shape and s3.shape == (3, 7)
    assert np.array_equal(q3.cpu().numpy(), wq3) and np.array_equal(s3.cpu().numpy(), ws3)


@pytest.mark.parametrize("n", [1, 3, 40, 300])
def test_strides(n):
    r = np.random.RandomState(n)
    K, rows = 333, 200
    w, wn = _rows(r, rows, K)
    big = torch.zeros(rows, 400, dtype=torch.int8, device="cuda")
    big[:, 16:16 + K] = w
    x = torch.randn(n, 700, device="cuda")[:, 1:1 + K]
    ws, wsn = _scales(r, rows)
    out = torch.full((n, 210), 9.0, device="cuda")
    G.mul_mat_i8(big[:, 16:16 + K], ws, x, out=out[:, 3:203])
    q, s = R.quantize(x.cpu().numpy())
    _near(out[:, 3:203], R.product(wn, wsn, q, s))
    assert (out[:, :3] == 9).all() and (out[:, 203:] == 9).all()
    xq = torch.zeros(n, 512, dtype=torch.int8, device="cuda")
    xq[:, 32:32 + K] = torch.from_numpy(q).cuda()
    out2 = G.mul_mat_i8(big[:, 16:16 + K], ws, xq[:, 32:32 + K], torch.from_numpy(s).cuda())
    assert torch.equal(out2, out[:, 3:203])


# ---- by experts


def _experts(r, e, rows, K):
    w, wn = _rows(r, e, rows, K)
    ws, wsn = _scales(r, e, rows)
    return w, wn, ws, wsn


@pytest.mark.parametrize("n,k,e", [(1, 1, 1), (1, 2, 4), (1, 8, 128), (2, 8, 128), (3, 5, 16), (7, 8, 16), (8, 8, 128), (16, 8, 128),
                                   (48, 8, 128), (130, 2, 8), (40, 4, 1024), (300, 8, 8), (1000, 4, 16), (2100, 8, 16)])
@pytest.mark.parametrize("slots", [False, True])
def test_products_by_experts(n, k, e, slots):
    r = np.random.RandomState(n + k)
    rows, K = 150, 200
    w, wn, ws, wsn = _experts(r, e, rows, K)
    ids = np.stack([r.permutation(max(e, k))[:k] for _ in range(n)]).astype(np.int32)
    ids[r.rand(n, k) < 0.1] = -1
    ids[ids >= e] = e + 5
    x = r.randn(n, k if slots else 1, K).astype(np.float32)
    q, s = R.quantize(x)
    want = R.product_id(wn, wsn, q, s, ids)
    ids_d, x_d = torch.from_numpy(ids).cuda(), torch.from_numpy(x).cuda()
    _near(G.mul_mat_id_i8(w, ws, x_d, ids_d), want)
    qd, sd = G.quantize_i8(x_d)
    _near(G.mul_mat_id_i8(w, ws, qd, ids_d, sd), want)


@pytest.mark.parametrize("rows,K", [(1, 1), (16, 16), (17, 129), (257, 768), (1536, 2048), (2048, 768)])
@pytest.mark.parametrize("n", [1, 5, 60, 700])
def test_expert_sizes(rows, K, n):
    r = np.random.RandomState(rows)
    e, k = 12, 4
    w, wn, ws, wsn = _experts(r, e, rows, K)
    ids = np.stack([r.permutation(e)[:k] for _ in range(n)]).astype(np.int32)
    x = r.randn(n, 1, K).astype(np.float32)
    q, s = R.quantize(x)
    _near(G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda()), R.product_id(wn, wsn, q, s, ids))


@pytest.mark.parametrize("n", [1, 4, 90, 1500])
@pytest.mark.parametrize("how", ["one", "none", "same slot twice", "far"])
def test_uneven_experts(n, how):
    r = np.random.RandomState(n)
    e, k, rows, K = 32, 3, 96, 160
    w, wn, ws, wsn = _experts(r, e, rows, K)
    ids = np.full((n, k), {"one": 31, "none": -1, "same slot twice": 4, "far": 2 ** 31 - 1}[how], np.int32)
    if how == "same slot twice":
        ids[:, 2] = r.randint(0, e, n)
    if how == "far":
        ids[:, 1] = -2 ** 31
        ids[::2, 0] = 0
    x = r.randn(n, k, K).astype(np.float32)
    q, s = R.quantize(x)
    out = torch.full((n, k, rows), np.nan, device="cuda")
    G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), out=out)
    _near(out, R.product_id(wn, wsn, q, s, ids))


@pytest.mark.parametrize("n", [2, 70, 600])
def test_expert_strides(n):
    r = np.random.RandomState(n)
    e, k, rows, K = 6, 2, 50, 90
    w, wn, ws, wsn = _experts(r, e, rows, K)
    big = torch.zeros(e, rows + 3, 128, dtype=torch.int8, device="cuda")
    big[:, 2:2 + rows, 16:16 + K] = w
    ids = torch.from_numpy(r.randint(-1, e, (n, 5)).astype(np.int32)).cuda()
    x = torch.randn(n, k, 128, device="cuda")[..., 6:6 + K]
    out = torch.full((n, k, 64), 3.0, device="cuda")
    G.mul_mat_id_i8(big[:, 2:2 + rows, 16:16 + K], ws, x, ids[:, 1:3], out=out[..., 5:55])
    q, s = R.quantize(x.cpu().numpy())
    _near(out[..., 5:55], R.product_id(wn, wsn, q, s, ids[:, 1:3].cpu().numpy()))
    assert (out[..., :5] == 3).all() and (out[..., 55:] == 3).all()


def test_rows_that_are_not_finite_stay_by_themselves():
    r = np.random.RandomState(2)
    e, k, rows, K, n = 8, 2, 64, 256, 200
    w, wn, ws, wsn = _experts(r, e, rows, K)
    x = r.randn(n, 1, K).astype(np.float32)
    x[17, 0, 3] = np.nan
    x[90, 0, 200] = np.inf
    ids = np.stack([r.permutation(e)[:k] for _ in range(n)]).astype(np.int32)
    ids[90, 1] = -1
    q, s = R.quantize(x)
    want = R.product_id(wn, wsn, q, s, ids)
    got = G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda())
    _near(got, want)
    assert np.isnan(want[17]).all() and np.isnan(want[90, 0]).all() and (want[90, 1] == 0).all()


# ---- streams, graphs, workspaces


def _calls(n):
    r = np.random.RandomState(n)
    w, _, ws, _ = _experts(r, 16, 300, 400)
    x = torch.randn(n, 1, 400, device="cuda")
    ids = torch.from_numpy(np.stack([r.permutation(16)[:4] for _ in range(n)]).astype(np.int32)).cuda()
    return [lambda out=None, workspace=None: G.mul_mat_i8(w[3], ws[3], x[:, 0], out=out, workspace=workspace),
            lambda out=None, workspace=None: G.mul_mat_id_i8(w, ws, x, ids, out=out, workspace=workspace)], x


@pytest.mark.parametrize("n", [1, 3, 50, 400])
def test_captured(n):
    calls, x = _calls(n)
    for call in calls:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for i in range(4):
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, call()), i


@pytest.mark.parametrize("n", [1, 3, 50, 400])
def test_two_streams_and_dirty_workspaces(n):
    calls, _ = _calls(n)
    for call in calls:
        want = call()
        dirty = torch.full((64 << 20,), 0xA5, dtype=torch.uint8, device="cuda")
        assert torch.equal(call(workspace=dirty), want)
        assert torch.equal(call(workspace=dirty), want)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for _ in range(3):
            for s in streams:
                with torch.cuda.stream(s):
                    outs.append(call())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("K", [1, 2, 3, 5, 127, 1001, 2048, 4096])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_tokens_of_any_alignment(K, shift):
    """f32 rows of one and a few tokens that start at any float."""
    r = np.random.RandomState(K)
    w, wn, ws, wsn = _experts(r, 5, 40, K)
    for n in (1, 2, 3):
        x = torch.randn(n, K + 5, device="cuda")[:, shift:shift + K]
        q, s = R.quantize(x.cpu().numpy())
        _near(G.mul_mat_i8(w[1], ws[1], x), R.product(wn[1], wsn[1], q, s))
        ids = torch.from_numpy(r.randint(-1, 6, (n, 3)).astype(np.int32)).cuda()
        _near(G.mul_mat_id_i8(w, ws, x[:, None], ids), R.product_id(wn, wsn, q[:, None], s[:, None], ids.cpu().numpy()))


def test_one_row_of_any_length():
    q = torch.randint(-127, 128, (32,), dtype=torch.int8, device="cuda")
    one = torch.ones(1, device="cuda")
    got = G.mul_mat_i8(q[None, :21], one, q[None, :21], one)
    assert got.item() == float((q[:21].double() ** 2).sum())


@pytest.mark.parametrize("rows,K,n", [(300, 256, 17), (9000, 640, 20), (9000, 160, 40), (260, 300, 520), (4100, 200, 600),
                                      (2050, 130, 2100), (30000, 100, 300), (30000, 96, 1)])
def test_every_form(rows, K, n):
    """Sizes at which each kernel and tile is chosen, with ragged ends."""
    r = np.random.RandomState(K)
    w, wn = _rows(r, rows, K)
    (ws, wsn), x = _scales(r, rows), r.randn(n, K).astype(np.float32)
    q, s = R.quantize(x)
    _near(G.mul_mat_i8(w, ws, torch.from_numpy(x).cuda()), R.product(wn, wsn, q, s))


@pytest.mark.parametrize("K,n,k,e", [(4096, 40, 8, 64), (9000, 30, 4, 40), (20000, 30, 4, 40), (40000, 3, 2, 6), (100000, 1, 2, 3),
                                     (100000, 4, 2, 3)])
def test_experts_of_long_rows(K, n, k, e):
    """Columns that do not fit in LDS together, or not at all."""
    r = np.random.RandomState(K)
    w, wn, ws, wsn = _experts(r, e, 20, K)
    ids = r.randint(0, e, (n, k)).astype(np.int32)
    x = r.randn(n, 1, K).astype(np.float32)
    q, s = R.quantize(x)
    _near(G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda()), R.product_id(wn, wsn, q, s, ids))


@pytest.mark.parametrize("n,e,k", [(4200, 3, 1), (9000, 2, 1), (2500, 70, 2), (1100, 300, 8)])
def test_pairs_in_several_chunks(n, e, k):
    """More pairs than one grouping workgroup takes, some without an expert."""
    r = np.random.RandomState(n)
    w, wn, ws, wsn = _experts(r, e, 33, 48)
    ids = r.randint(-1, e + 1, (n, k)).astype(np.int32)
    x = r.randn(n, 1, 48).astype(np.float32)
    q, s = R.quantize(x)
    out = torch.full((n, k, 33), np.nan, device="cuda")
    G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), out=out)
    _near(out, R.product_id(wn, wsn, q, s, ids))


@pytest.mark.parametrize("rows,K,n,k,e", [(282, 842, 272, 5, 8), (2100, 130, 500, 2, 8), (300, 200, 3750, 4, 32), (4100, 1030, 1250, 4, 32),
                                          (4100, 1030, 1400, 4, 32), (4100, 65, 1400, 4, 32), (4100, 1600, 1400, 4, 32), (4100, 2061, 1400, 4, 32),
                                          (1540, 2061, 900, 8, 56)])
def test_tiles_of_each_size_by_experts(rows, K, n, k, e):
    """Some experts with few columns, some with many, and some pairs without one."""
    r = np.random.RandomState(rows)
    w, wn, ws, wsn = _experts(r, e, rows, K)
    liked = r.rand(e) ** 2 + 0.01
    ids = r.choice(e, (n, k), p=liked / liked.sum()).astype(np.int32)
    ids[r.rand(n, k) < 0.02] = -1
    x = r.randn(n, 1, K).astype(np.float32)
    q, s = R.quantize(x)
    out = torch.full((n, k, rows), np.nan, device="cuda")
    G.mul_mat_id_i8(w, ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda(), out=out)
    _near(out, R.product_id(wn, wsn, q, s, ids))


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 7, 1021, 4099, 8193, 20002])
@pytest.mark.parametrize("off", [0, 1, 2, 3])
def test_quantized_rows_at_any_byte(K, off):
    """Values from any multiple of four bytes, results to any byte, and nothing behind a row is written."""
    r = np.random.RandomState(K)
    n = 7
    x = np.zeros((n, K + 9), np.float32)
    x[:, off:off + K] = r.randn(n, K)
    q, s = R.quantize(x[:, off:off + K])
    xd = torch.from_numpy(x).cuda()
    out = torch.full((n, K + 6), 99, dtype=torch.int8, device="cuda")
    got, scale = G.quantize_i8(xd[:, off:off + K], out=out[:, off:off + K])
    assert np.array_equal(got.cpu().numpy(), q) and np.array_equal(scale.cpu().numpy(), s)
    assert (out[:, :off] == 99).all() and (out[:, off + K:] == 99).all()


@pytest.mark.parametrize("rows,K,n", [(269, 16070, 469), (16, 131071, 33), (4096, 129, 64), (4090, 2061, 37), (1, 300, 5000), (33, 4097, 2700),
                                      (1000, 20001, 128)])
@pytest.mark.parametrize("f32", [False, True])
def test_more_columns_than_one_workgroup_takes(rows, K, n, f32):
    """Few weight rows or few columns, so that the inner axis is shared by waves."""
    r = np.random.RandomState(n)
    w, wn = _rows(r, rows, K)
    ws, wsn = _scales(r, rows)
    x = r.randn(n, K).astype(np.float32)
    q, s = R.quantize(x)
    xd = torch.from_numpy(x).cuda()
    out = torch.full((n, rows + 3), np.nan, device="cuda")
    x8, scale = (xd, None) if f32 else G.quantize_i8(xd)
    got = G.mul_mat_i8(w, ws, x8, scale, out=out[:, 1:1 + rows])
    _near(got, R.product(wn, wsn, q, s))
    assert out[:, 0].isnan().all() and out[:, 1 + rows:].isnan().all()


@pytest.mark.parametrize("K", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 200, 700])
def test_many_tiles_along_a_short_axis(K):
    """Checked where the rows and columns of tiles begin and end."""
    r = np.random.RandomState(K)
    rows, n = 5003, 7710
    w, wn = _rows(r, rows, K, full=True)
    ws, wsn = _scales(r, rows)
    x, xn = _rows(r, n, K)
    xs, xsn = _scales(r, n)
    got = G.mul_mat_i8(w, ws, x, xs)
    assert got.isfinite().all()
    m = np.unique(np.concatenate([np.arange(b, b + 3) for b in range(0, rows - 2, 125)] + [np.arange(4864, rows)]))
    c = np.unique(np.concatenate([np.arange(b, b + 3) for b in range(0, n - 2, 127)] + [np.arange(7680, n)]))
    _near(got[torch.from_numpy(c).cuda()][:, torch.from_numpy(m).cuda()],
          R.product(wn[m], wsn[m], np.ascontiguousarray(xn[c]), xsn[c]))


def _rounded_thrice(w, w_scale, q, scale):
    """The definition's bits: the sum to f32, the first product to 24 bits of any exponent, the second to f32."""
    acc = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32).astype(np.float64)
    mantissa, exponent = np.frexp(acc * scale.astype(np.float64)[:, None])  # products of two f32 are exact in f64
    with np.errstate(all="ignore"):
        return (np.ldexp(mantissa.astype(np.float32).astype(np.float64), exponent) * w_scale.astype(np.float64)).astype(np.float32)


@pytest.mark.parametrize("n", [1, 3, 20, 60, 400])
@pytest.mark.parametrize("w_power,x_power", [(-70, -68), (-140, 0), (0, -143), (-100, -47), (100, -110), (3, 5), (110, 6)])
def test_bits_of_results(n, w_power, x_power):
    """Subnormal results among them: of the fewer bits that they have, rounded once."""
    r = np.random.RandomState(n)
    rows, K = 300, 90
    w, wn = _rows(r, rows, K)
    x, xn = _rows(r, n, K)
    wsn = np.ldexp(r.rand(rows) + 0.5, w_power).astype(np.float32)
    xsn = np.ldexp(r.rand(n) + 0.5, x_power).astype(np.float32)
    ws, xs = torch.from_numpy(wsn).cuda(), torch.from_numpy(xsn).cuda()
    want = _rounded_thrice(wn, wsn, xn, xsn)
    got = G.mul_mat_i8(w, ws, x, xs).cpu().numpy()
    assert np.array_equal(got, want), (np.argwhere(got != want)[:3], (got != want).sum())
    ids = torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    by_experts = G.mul_mat_id_i8(w[None], ws[None], x[:, None], ids, xs[:, None]).cpu().numpy()
    assert np.array_equal(by_experts[:, 0], want) and np.array_equal(by_experts[:, 1], want)


@pytest.mark.parametrize("n", [1, 30, 700])
def test_one_row_an_expert(n):
    r = np.random.RandomState(n)
    e, k, K = 6, 2, 90
    w, wn = _rows(r, e, K)
    ws, wsn = _scales(r, e, 1)
    ids = r.randint(-1, e, (n, k)).astype(np.int32)
    x = r.randn(n, 1, K).astype(np.float32)
    got = G.mul_mat_id_i8(w[:, None], ws, torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda())
    _near(got, R.product_id(wn[:, None], wsn, *R.quantize(x), ids))
