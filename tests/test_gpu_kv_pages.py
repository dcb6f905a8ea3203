"""Page copies and the compaction of the paged cache (hip_qmm_kv_copy_pages,
hip_qmm_kv_compact) against plain host code."""
import random

import pytest

import attn_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _cache(dtype="f16", pages=40, kv_heads=3, page=16, dim=64, order="heads", seed=1):
    gen = torch.Generator("cuda").manual_seed(seed)
    return R.make_cache(gen, R.DTYPES[dtype], pages, kv_heads, page, dim, order=order)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("order", ["heads", "tokens"])
@pytest.mark.parametrize("dtype,kv_heads,page,dim", [("f16", 8, 16, 128), ("bf16", 1, 64, 8), ("f16", 3, 32, 80),
                                                     ("bf16", 5, 128, 256)])
@pytest.mark.parametrize("n", [1, 7, 20])
def test_copy(order, dtype, kv_heads, page, dim, n):
    import ggml_hip as G
    k, v = _cache(dtype, 40, kv_heads, page, dim, order)
    perm = torch.randperm(40, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = perm[:n], perm[n:2 * n]
    counts = [random.Random(i).choice((1, 2, page - 1, page, page + 5, 0, -3)) for i in range(n)]
    for cut in (None, counts):
        wk, wv = k.clone(), v.clone()
        for i in range(n):
            m = page if cut is None else max(0, min(page, cut[i]))
            wk[dst[i], :, :m], wv[dst[i], :, :m] = wk[src[i], :, :m], wv[src[i], :, :m]
        G.copy_pages(G.PagedKV(k, v), _i32(src), _i32(dst), None if cut is None else _i32(cut))
        assert torch.equal(k, wk) and torch.equal(v, wv)


def test_one_page_forked_many_times_and_pairs_outside_the_pool():
    import ggml_hip as G
    k, v = _cache()
    wk, wv = k.clone(), v.clone()
    for d in (1, 5, 39):
        wk[d], wv[d] = k[3], v[3]
    G.copy_pages(G.PagedKV(k, v), _i32([3, -1, 3, 40, 3, 7, 3]), _i32([1, 2, 5, 8, 39, 40, -2 ** 31]))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    G.copy_pages(G.PagedKV(k, v), _i32([]), _i32([]))
    assert torch.equal(k, wk)


def _compact_plain(table, lens, pages, page):
    """(new table, pages in use, {page: new page}) by the definition."""
    keep = [[0 <= e < pages and i * page < n for i, e in enumerate(row)] for row, n in zip(table, lens)]
    used = sorted({e for row, ok in zip(table, keep) for e, k in zip(row, ok) if k})
    live = len(used)
    holes = [p for p in range(live) if p not in set(used)]
    moves = dict(zip([p for p in used if p >= live], holes))
    new = [[moves.get(e, e) if k else -1 for e, k in zip(row, ok)] for row, ok in zip(table, keep)]
    return new, live, moves


def _check_compact(k, v, table, lens, page, **kw):
    import ggml_hip as G
    pages = k.shape[0]
    want, live, moves = _compact_plain(table, lens, pages, page)
    wk, wv = k.clone(), v.clone()
    if moves:
        src, dst = list(moves), list(moves.values())
        wk[dst], wv[dst] = k[src], v[src]
    got, n = G.compact_pages(G.PagedKV(k, v), kw.pop("tensor", None) if "tensor" in kw else _i32(table), _i32(lens), **kw)
    assert got.tolist() == want and n.tolist() == [live]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    return got


@pytest.mark.parametrize("pages,seqs,width,share", [(40, 3, 5, 0), (40, 4, 9, 2), (33, 1, 33, 0), (64, 8, 8, 0), (1, 1, 1, 0),
                                                    (100, 50, 1, 0), (1000, 7, 100, 3), (5000, 60, 70, 10), (32, 5, 3, 0)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_compact(pages, seqs, width, share, seed):
    rng = random.Random(seed * 1000 + pages)
    k, v = _cache(pages=pages, kv_heads=2, dim=8, seed=seed)
    free = rng.sample(range(pages), pages)
    table, lens = [], []
    for s in range(seqs):
        n = rng.choice((0, 1, 16, rng.randint(0, 16 * width), 16 * width))
        row = []
        for i in range(width):
            if i < share and table and i * 16 < n and lens[0] > i * 16:
                row.append(table[0][i])
            elif i * 16 < n and free:
                row.append(free.pop())
            else:  # stale or hidden entries, which need not be in the pool
                row.append(rng.choice((-1, -7, pages, 2 ** 31 - 1, rng.randrange(pages) if i * 16 >= n else -1)))
        table.append(row)
        lens.append(n)
    _check_compact(k, v, table, lens, 16)


@pytest.mark.parametrize("dtype,kv_heads,page,dim,order", [("bf16", 8, 32, 128, "heads"), ("f16", 3, 16, 80, "tokens"),
                                                           ("f16", 1, 128, 256, "heads")])
def test_compact_cache_layouts(dtype, kv_heads, page, dim, order):
    k, v = _cache(dtype, 50, kv_heads, page, dim, order)
    _check_compact(k, v, [[49, 3, 20], [48, 0, -1], [30, 31, 3]], [3 * page, page + 1, 3 * page - 5], page)


def test_compact_nothing_and_everything():
    k, v = _cache(pages=16)
    _check_compact(k, v, [[3, 4], [5, 6]], [0, -4], 16)
    _check_compact(k, v, [list(range(15, -1, -1))], [16 * 16], 16)
    got = _check_compact(k, v, [[15, 0], [14, 2]], [32, 32], 16)
    again = _check_compact(k, v, got.tolist(), [32, 32], 16)  # together already: nothing moves
    assert torch.equal(again, got)


def test_compact_in_place_strided_and_in_a_graph():
    import ggml_hip as G
    k, v = _cache(pages=64)
    wide = torch.full((3, 9), 63, dtype=torch.int32, device="cuda")
    table = wide[:, 2:6]
    table.copy_(_i32([[60, 50, 40, 30], [61, 50, 41, -1], [1, 0, 35, 36]]))
    lens = [64, 40, 64]
    _check_compact(k, v, table.tolist(), lens, 16, tensor=table, out=table)
    assert bool((wide[:, :2] == 63).all()) and bool((wide[:, 6:] == 63).all())

    static, n = _i32([[0] * 4] * 3), _i32(lens)
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(static)
    kv = G.PagedKV(k, v)
    G.compact_pages(kv, static, n, out=out, workspace=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, live = G.compact_pages(kv, static, n, out=out, workspace=ws)
    for seed in range(4):
        rows = random.Random(seed).sample(range(64), 12)
        static.copy_(_i32(rows).view(3, 4))
        want, count, moves = _compact_plain(static.tolist(), lens, 64, 16)
        wk = k.clone()
        if moves:
            wk[list(moves.values())] = k[list(moves)]
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == want and live.tolist() == [count] and torch.equal(k, wk)


def test_compact_the_largest_pool():
    """2^20 pages: the bitmap of the plan is at its largest."""
    import ggml_hip as G
    pages = 1 << 20
    k = torch.zeros((pages, 1, 16, 8), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    k[:, 0, 0, 0] = (torch.arange(pages, device="cuda") % 2048).half()
    v[:, 0, 0, 0] = (torch.arange(pages, device="cuda") // 2048).half()
    table = torch.randperm(pages, generator=torch.Generator("cuda").manual_seed(1), device="cuda")[:600000].int().view(600, 1000)
    lens = torch.full((600,), 16000, dtype=torch.int32, device="cuda")
    got, n = G.compact_pages(G.PagedKV(k, v), table, lens)
    assert n.tolist() == [600000]
    flat = got.long().flatten()
    assert int(flat.unique().numel()) == 600000 and int(flat.max()) == 599999
    here = k[flat, 0, 0, 0].long() + 2048 * v[flat, 0, 0, 0].long()
    assert torch.equal(here, table.long().flatten())
    stay = table.flatten() < 600000
    assert torch.equal(got.flatten()[stay], table.flatten()[stay])


def test_fork_compact_and_attend():
    """A fork's attention is its parent's until they part, before and after the pool is compacted."""
    import ggml_hip as G
    gen = torch.Generator("cuda").manual_seed(3)
    k, v = R.make_cache(gen, torch.float16, 80, 8, 16, 128)
    kv = G.PagedKV(k, v)
    table = _i32([[70, 61, 52, 43, -1]] * 2)
    table[1, 3] = 77
    G.copy_pages(kv, table[0, 3:4].contiguous(), table[1, 3:4].contiguous(), _i32([7]))
    lens = _i32([55, 55])
    q = torch.randn((1, 32, 128), generator=gen, device="cuda").repeat(2, 1, 1)
    first = G.attn_paged(q, kv, table, lens)
    assert torch.equal(first[0], first[1])
    table, live = G.compact_pages(kv, table, lens)
    assert live.tolist() == [5] and int(table[:, :4].max()) == 4
    assert torch.equal(G.attn_paged(q, kv, table, lens), first)
    steps, _ = G.rope_steps(128)
    new = [torch.randn((2, h, 128), generator=gen, device="cuda") for h in (32, 8, 8)]
    slots = table[:, 3] * 16 + 7
    r = G.rope_kv_store(*new, lens, steps, kv, slots.int())
    got = G.attn_paged(r, kv, table, lens + 1)
    want, top = R.attention(r, k, v, table, lens + 1, torch.arange(3), 128 ** -0.5)
    assert float((got.double() - want).norm() / want.norm()) <= R.tolerance(128, top)
    assert not torch.equal(got[0], got[1])


@pytest.mark.parametrize("pages,width", [(8192, 60), (8193, 60), (300, 16384 // 3), (300, 16384 // 3 + 1)])
def test_compact_at_the_limits_of_one_launch(pages, width):
    """Up to 8192 pages and 16384 table entries it is one launch, above two."""
    rng = random.Random(pages + width)
    k, v = _cache(pages=pages, kv_heads=1, dim=8)
    free = rng.sample(range(pages), pages)
    lens = [16 * 60, 16 * 37 + 3, 16 * 50]
    table = [[free.pop() if i * 16 < n else rng.choice((-1, 5, pages)) for i in range(width)] for n in lens]
    got = _check_compact(k, v, table, lens, 16)
    # the same in place, which takes two launches
    k, v = _cache(pages=pages, kv_heads=1, dim=8)
    t = _i32(table)
    assert torch.equal(_check_compact(k, v, table, lens, 16, tensor=t, out=t), got)
