"""Attention over the paged cache (hip_qmm_attn_paged) against its f64
definition: types, head layouts, lengths from none to long ones, windows and
first tokens that stay visible, pages that end inside a tile, hidden tokens
that hold NaN, rows that see nothing, strides, streams, graphs."""
import math

import pytest

import attn_ref as R

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _case(dtype="f16", heads=32, kv_heads=8, dim=128, page=16, lens=(333,), new=None, order="heads", seed=1,
          spread=1.0, width=None):
    gen = torch.Generator("cuda").manual_seed(seed)
    table, pool = R.make_table(gen, lens, page, width=width)
    k, v = R.make_cache(gen, R.DTYPES[dtype], pool, kv_heads, page, dim, order=order)
    new = [1] * len(lens) if new is None else new
    starts = R.starts_of(new)
    q = torch.randn((int(starts[-1]), heads, dim), generator=gen, device="cuda") * spread
    return dict(q=q, k=k, v=v, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), starts=starts,
                new=new)


def _run(c, window=0, sinks=0, scale=None, decode=None, **kw):
    import ggml_hip as G
    decode = all(m == 1 for m in c["new"]) if decode is None else decode
    return G.attn_paged(c["q"], G.PagedKV(c["k"], c["v"]), c["table"], c["lens"],
                        q_starts=None if decode else c["starts"], max_q=max(c["new"]), window=window, sinks=sinks,
                        scale=scale, **kw)


def _hold(got, want, top, dim, vmax=None):
    tol = R.tolerance(dim, top)
    assert got.dtype == torch.float32
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got))
    d = torch.where(fin, got.double() - want, 0.0)
    w = torch.where(fin, want, 0.0)
    norm = float(w.norm())
    assert float(d.norm()) <= tol * norm + 1e-300, (float(d.norm()) / max(norm, 1e-300), tol)
    # one element is off by no more than what the whole may be off, times the largest value of v
    assert float(d.abs().max()) <= 8 * tol * (5.5 if vmax is None else vmax)


def _check(c, window=0, sinks=0, scale=None, vmax=None, **kw):
    dim = c["q"].shape[2]
    got = _run(c, window, sinks, scale, **kw)
    want, top = R.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"],
                            dim ** -0.5 if scale is None else scale, window, sinks)
    _hold(got, want, top, dim, vmax)
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (8, 2), (32, 4), (14, 2), (16, 1), (17, 1), (40, 1), (71, 1)])
def test_one_token_head_layouts(dtype, heads, kv_heads):
    _check(_case(dtype, heads, kv_heads, lens=(333, 1, 64, 1000)))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [8, 16, 40, 64, 72, 80, 96, 104, 112, 128, 136, 192, 200, 248, 256])
def test_head_dims(dtype, dim):
    _check(_case(dtype, 8, 2, dim, lens=(1, 33, 300)))
    _check(_case(dtype, 8, 2, dim, lens=(40, 33, 300), new=[40, 5, 100]))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("order", ["heads", "tokens"])
def test_page_sizes_and_cache_layouts(page, order):
    _check(_case(page=page, order=order, lens=(5, 333, 1025, 130)))
    _check(_case("bf16", page=page, order=order, lens=(5, 333, 700), new=[3, 100, 64]))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 511, 512, 513, 4097, 20001])
def test_one_token_lengths(n):
    _check(_case(lens=(n,)))


def test_empty_sequences_and_rows_that_see_nothing():
    c = _case(lens=(0, 7, 0, 64), new=[1, 1, 1, 1])
    got = _check(c)
    assert float(got[0].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0
    # more queries than tokens: the first ones sit before the sequence
    c = _case(lens=(3, 0, 100), new=[8, 4, 60])
    got = _check(c)
    assert float(got[:5].abs().max()) == 0.0 and float(got[5].abs().max()) > 0.0
    assert float(got[8:12].abs().max()) == 0.0
    # a table whose pages are all hidden
    c = _case(lens=(70, 70), new=[1, 1])
    c["table"][0] = -1
    got = _check(c)
    assert float(got[0].abs().max()) == 0.0
    c["lens"].fill_(-5)
    assert float(_run(c).abs().max()) == 0.0


def test_empty_calls():
    c = _case(lens=(40, 9), new=[0, 0])
    import ggml_hip as G
    out = G.attn_paged(c["q"], G.PagedKV(c["k"], c["v"]), c["table"], c["lens"], q_starts=c["starts"], max_q=0)
    assert out.shape == (0, 32, 128)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 4), (64, 100), (100, 0), (333, 16), (5000, 4)])
def test_windows_and_first_tokens(dtype, window, sinks):
    _check(_case(dtype, lens=(500, 64, 1, 90), page=32), window, sinks)
    _check(_case(dtype, lens=(500, 64, 1, 300), new=[300, 64, 1, 2]), window, sinks)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,new", [((13,), (13,)), ((1000,), (13,)), ((129, 128, 127, 1), (129, 128, 127, 1)),
                                      ((700, 300), (1, 300)), ((2500, 2049), (16, 33)), ((511,), (257,)),
                                      ((40,) * 9, (2,) * 9), ((4100,), (4,)), ((6000,), (9,))])
def test_many_tokens(dtype, lens, new):
    _check(_case(dtype, lens=lens, new=list(new)))
    _check(_case(dtype, heads=6, kv_heads=2, dim=64, lens=lens, new=list(new)))


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_prompt(dim):
    _check(_case(heads=4, kv_heads=2, dim=dim, page=64, lens=(1500, 1111), new=[1500, 1000]))
    _check(_case("bf16", heads=4, kv_heads=2, dim=dim, page=64, lens=(1500, 1111), new=[1500, 1000]), 256, 4)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 100])
def test_what_hidden_tokens_hold_does_not_matter(bad, dtype, new):
    """Unused pages, the rest of the last page, tokens behind the window and entries outside the pool."""
    window, sinks = 50, 3
    c = _case(dtype, lens=(333, 120), new=[new, 1], page=16)
    want = _run(c, window, sinks, decode=False)
    used = torch.zeros(c["k"].shape[0], 16, dtype=torch.bool, device="cuda")
    for s, n in enumerate(c["lens"].tolist()):
        first = n - c["new"][s]  # the first query's position
        for j in range(n):
            if j < sinks or first - j < window:
                used[int(c["table"][s, j // 16]), j % 16] = True
    for x in (c["k"], c["v"]):
        x.copy_(torch.where(used[:, None, :, None], x, torch.tensor(bad, dtype=x.dtype, device="cuda")))
    got = _run(c, window, sinks, decode=False)
    assert torch.equal(got, want)
    # pages that fell out of the window are gone from the table
    for s, n in enumerate(c["lens"].tolist()):
        low = (n - c["new"][s] - window) // 16
        c["table"][s, 1:max(1, low)] = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31] * 40, dtype=torch.int32)[:max(0, low - 1)]
    assert torch.equal(_run(c, window, sinks, decode=False), want)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [6, 100])
def test_a_later_tokens_value_does_not_reach_earlier_rows(bad, dtype, new):
    """The value (and key) of one token is not finite: only the rows that see it are touched, and there as IEEE has it."""
    c = _case(dtype, heads=8, kv_heads=2, lens=(200, 90), new=[new, 3])
    at = 200 - new // 2
    clean = _run(c)
    page = int(c["table"][0, at // 16])
    c["v"][page, 1, at % 16, 5] = bad
    got = _run(c)
    row = at - (200 - new)
    assert torch.equal(got[:row], clean[:row]) and torch.equal(got[new:], clean[new:])
    assert torch.equal(got[:, :4], clean[:, :4])  # the other key-value head
    hit = got[row:new, 4:, 5]
    assert bool((torch.isnan(hit) if math.isnan(bad) else hit == bad).all())
    keep = torch.ones(128, dtype=torch.bool, device="cuda")
    keep[5] = False
    assert torch.equal(got[:, :, keep], clean[:, :, keep])
    c["k"][page, 1, at % 16, 7] = math.nan
    got = _run(c)
    assert torch.equal(got[:row], clean[:row]) and torch.equal(got[:, :4], clean[:, :4])
    assert bool(torch.isnan(got[row:new, 4:]).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_extreme_queries(dtype, new):
    c = _case(dtype, lens=(300, 77), new=[new, 1])
    c["q"][0] *= 2.0 ** 40    # far over f16's range: the largest score takes all
    c["q"][-1] *= 2.0 ** -60  # all scores alike
    got = _run(c, decode=False)
    want, _ = R.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], 128 ** -0.5)
    # a winner's margin is far over its rounding except by chance: rows are compared where it is
    assert torch.isfinite(got).all()
    _hold(got[-1:], want[-1:], 0.0, 128)
    close = (got[0].double() - want[0]).abs().amax(1) < 1e-3
    assert int(close.sum()) >= 30
    c["q"].zero_()
    _check(c, decode=False)
    c = _case(dtype, lens=(300, 77), new=[new, 1], spread=6.0)
    _check(c, decode=False)
    _check(c, scale=-0.3, decode=False)
    _check(c, scale=0.0, decode=False)


@pytest.mark.parametrize("dtype,up", [("f16", 13), ("bf16", 100)])
@pytest.mark.parametrize("lens,new", [((300, 77), 1), ((300, 77), 40), ((5000,), 1), ((700, 400), 300), ((9000,), 150)])
def test_large_cached_values(dtype, up, lens, new):
    """Keys far over 1 that small queries meet, values up to the type's largest."""
    c = _case(dtype, lens=lens, new=[new] * len(lens))
    c["q"] *= 2.0 ** -up
    c["k"] *= 2.0 ** up
    most = torch.finfo(c["v"].dtype).max
    gen = torch.Generator("cuda").manual_seed(3)
    size = 0.5 + 0.5 * torch.rand(c["v"].shape, generator=gen, device="cuda")
    c["v"].copy_(torch.copysign(size, c["v"].float()) * most)
    assert torch.isfinite(c["k"]).all() and torch.isfinite(c["v"]).all()
    _check(c, vmax=most)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,new", [(300, 1), (20000, 1), (900, 20), (3000, 7), (3000, 15), (700, 300), (9000, 150)])
def test_an_infinite_value_of_tiny_weight(dtype, n, new):
    """A probability that f32 holds as 0 is above 0 all the same: times infinity it is infinity, not NaN."""
    c = _case(dtype, lens=(n,), new=[new])
    c["q"].abs_()
    page = int(c["table"][0, 0])
    c["k"][page, 3, 0] = -60.0  # scores near -500
    c["v"][page, 3, 0, 77] = math.inf
    got = _check(c)
    assert bool((got[:, 12:16, 77] == math.inf).all())


def test_longest_planning_length():
    """The longest length that can be planned for, over a short table and over one as long."""
    c = _case(lens=(333,))
    want = _check(c)
    _hold(_run(c, max_kv=1 << 30), want.double(), 8.0, 128)
    wide = torch.full((1, (1 << 26) + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, :c["table"].shape[1]] = c["table"]
    _hold(_run(dict(c, table=wide)), want.double(), 8.0, 128)
    _hold(_run(dict(c, table=wide), max_kv=2 ** 31 - 1), want.double(), 8.0, 128)


def test_nan_query_is_its_own_rows_matter():
    c = _case(lens=(100, 50), new=[20, 20])
    clean = _run(c)
    c["q"][3, 2, 5] = math.nan
    c["q"][25, 1, 0] = math.inf
    got = _run(c)
    keep = torch.ones(40, 32, dtype=torch.bool, device="cuda")
    keep[3, 2] = keep[25, 1] = False
    assert torch.equal(got[keep], clean[keep])
    assert bool(torch.isnan(got[3, 2]).all()) and bool(torch.isnan(got[25, 1]).all())


def test_strided_queries_and_results():
    c = _case(lens=(300, 77, 20), new=[50, 1, 20])
    want = _run(c)
    wide = torch.full((71, 64, 192), math.nan, device="cuda")
    wide[:, ::2, 32:160] = c["q"]
    out = torch.full((71, 40, 256), 7.0, device="cuda")
    c["q"] = wide[:, ::2, 32:160]
    view = out[:, 4:36, 64:192]
    got = _run(c, out=view)
    assert torch.equal(view, want) and got.data_ptr() == view.data_ptr()
    rest = out.clone()
    rest[:, 4:36, 64:192] = 7.0
    assert bool((rest == 7.0).all())


def test_rows_of_no_sequence_are_left_alone():
    """q_starts need not begin at the first row or end at the last."""
    c = _case(lens=(90, 40), new=[10, 5])
    want = _run(c)
    c["q"] = torch.cat([c["q"][:3] * 0 + math.nan, c["q"], c["q"][:2] * 0 + math.nan])
    c["starts"] += 3
    out = torch.full_like(c["q"], 3.0)
    _run(c, out=out)
    assert torch.equal(out[3:18], want) and bool((out[:3] == 3.0).all()) and bool((out[18:] == 3.0).all())


def test_planning_lengths_do_not_change_what_is_computed():
    """max_kv only plans: too small or too large, the result is the same to rounding."""
    c = _case(lens=(3000, 40, 700))
    want, top = R.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], 128 ** -0.5)
    for most in (1, 100, 3000, 3008):
        _hold(_run(c, max_kv=most), want, top, 128)
    c = _case(lens=(3000, 40, 700), new=[70, 2, 1])
    want, top = R.attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["starts"], 128 ** -0.5)
    for most in (1, 100, 3000, 3008):
        _hold(_run(c, max_kv=most), want, top, 128)


@pytest.mark.parametrize("new", [None, [20, 1]])
def test_repeatable_on_any_scratch(new):
    import ggml_hip as G
    c = _case(lens=(9000, 700), new=new)
    size = G.attn_paged_workspace_size(G.PagedKV(c["k"], c["v"]), 32, 2, c["q"].shape[0], max(c["new"]),
                                       c["table"].shape[1] * 16)
    first = None
    for fill in (0, 255, 127, 0):
        ws = torch.full((max(size, 1),), fill, dtype=torch.uint8, device="cuda")
        got = _run(c, workspace=ws, out=torch.full_like(c["q"], math.nan))
        first = got if first is None else first
        assert torch.equal(got, first)
    with pytest.raises(G.HipQmmError):
        _run(c, workspace=torch.empty(max(size - 1, 0), dtype=torch.uint8, device="cuda"))


@pytest.mark.parametrize("new", [None, [20, 1]])
def test_on_another_stream(new):
    c = _case(lens=(5000, 700), new=new)
    want = _run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(c)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [None, [20, 1]])
def test_in_a_graph(new):
    """Captured once, replayed with other contents and lengths, eager work in between."""
    c = _case(lens=(5000, 700), new=new)
    out = torch.empty_like(c["q"])
    import ggml_hip as G
    size = G.attn_paged_workspace_size(G.PagedKV(c["k"], c["v"]), 32, 2, c["q"].shape[0], max(c["new"]), 5008)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    _run(c, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(c, out=out, workspace=ws)
    for n in (5000, 33, 4097):
        c["lens"][0] = n
        c["q"].normal_()
        want = _run(c)
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_offsets_past_32_bits():
    """A pool of over 2^32 bytes and 2^31 elements in each of keys and values."""
    pages = (2 ** 31 + 2 ** 27) // (8 * 16 * 128)
    k = torch.empty((pages, 8, 16, 128), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    c = _case(lens=(333, 40))
    hold = torch.tensor([pages - 1 - i for i in range(c["k"].shape[0])], device="cuda")
    k[hold], v[hold] = c["k"], c["v"]
    far = dict(c, k=k, v=v, table=torch.where(c["table"] >= 0, pages - 1 - c["table"], -1).int())
    assert torch.equal(_run(far), _run(c))
    d = _case(lens=(333, 40), new=[50, 3])
    k[hold], v[hold] = d["k"], d["v"]
    far = dict(d, k=k, v=v, table=torch.where(d["table"] >= 0, pages - 1 - d["table"], -1).int())
    assert torch.equal(_run(far), _run(d))


FORMS = [  # rows of a workgroup, whether the tokens are split, sequences, new tokens, length
    (16, False, 2, 1, 300), (16, True, 2, 1, 3000), (16, False, 2, 40, 300), (16, True, 1, 20, 900),
    (32, True, 2, 7, 3000), (64, False, 2, 300, 700), (64, True, 2, 15, 3000), (128, False, 5, 1000, 1100),
    (128, True, 1, 150, 9000)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128, 192, 248, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (900, 5)])
@pytest.mark.parametrize("form", FORMS)
def test_every_kernel_form(form, window, sinks, dim, dtype):
    import ggml_hip as G
    rows, split, seqs, new, n = form
    lens = [n] + [max(new, n * 2 // 3 + 7 * i) for i in range(1, seqs)]
    c = _case(dtype, 32, 8, dim, page=32, lens=lens, new=[new] * seqs)
    kv = G.PagedKV(c["k"], c["v"])
    got, splits = G.attn_paged_plan(kv, 32, seqs, c["q"].shape[0], new, c["table"].shape[1] * 32, window, sinks)
    if not window and dim <= 128:
        assert (got, splits > 1) == (rows, split)
    _check(c, window, sinks)


@pytest.mark.parametrize("kv_heads,seqs", [(1, 1), (1, 8), (2, 3), (2, 4), (3, 3), (4, 1), (4, 3), (4, 6), (6, 2),
                                           (12, 3), (16, 1), (24, 2)])
@pytest.mark.parametrize("new,n", [(1, 3000), (40, 300), (300, 700), (200, 1500)])
def test_every_block_and_split_is_done_once(kv_heads, seqs, new, n):
    """Workgroups are dealt out by head, sequence and split: every order of them, with sequences of unlike lengths."""
    lens = [n if i == 0 else (n * (3 * i + 1)) // (4 * i + 2) for i in range(seqs)]
    c = _case("f16", 2 * kv_heads, kv_heads, 64, page=32, lens=lens, new=[min(new, m) for m in lens])
    _check(c)
    _check(c, max_kv=max(lens) // 2)  # planned as a prompt


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("most,window,sinks", [(30, 0, 0), (380, 0, 0), (380, 100, 5)])
def test_many_short_sequences(dtype, dim, most, window, sinks):
    """A wave for each: from empty ones to the longest, values that are hidden or seen and not finite among them."""
    lens = [most, 0, 1, most - 1] + [(37 * i) % most for i in range(13)]
    c = _case(dtype, 64, 64, dim, page=16, lens=lens)
    clean = _check(c, window, sinks)
    last = int(c["table"][0, (most - 1) // 16])
    c["v"][last, 5, most % 16:, :] = math.nan  # behind the end (most is no multiple of 16)
    c["v"][last, 7, (most - 1) % 16, 11] = math.inf
    got = _run(c, window, sinks)
    assert float(got[0, 7, 11]) == math.inf
    got[0, 7, 11] = clean[0, 7, 11]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("form", FORMS)
def test_values_that_are_not_finite_in_every_kernel_form(form, bad):
    """One bad value of a late token of the first sequence: its dimension of the rows that see it, nothing else."""
    rows, split, seqs, new, n = form
    c = _case("f16", 32, 8, 128, page=32, lens=[n] * seqs, new=[new] * seqs)
    clean = _run(c, decode=False)
    at = n - 1 - new // 3
    c["v"][int(c["table"][0, at // 32]), 3, at % 32, 77] = bad
    got = _run(c, decode=False)
    first = new - 1 - new // 3
    hit = got[first:new, 12:16, 77]
    assert bool((torch.isnan(hit) if math.isnan(bad) else hit == bad).all())
    got[first:new, 12:16, 77] = clean[first:new, 12:16, 77]
    assert torch.equal(got, clean)
