"""The entry points of include/ggml_hip_attn.h on the CPU: every declared one is
exported, what they do not take is refused before anything is launched, and the
host-side parts (rotation steps, workspace sizes) are what the header says."""
import ctypes as C
import math
import re

import pytest

import ggml_hip as G
from ggml_hip import attn as A

HEADER = G.PKG_DIR.parent / "include" / "ggml_hip_attn.h"
BAD = 1  # hipErrorInvalidValue
P = 1 << 20  # an aligned address that nothing reads: every call here is refused or empty


def _cache(**kw):
    f = dict(k=P, v=P, type=1, n_kv_heads=8, page_size=16, head_dim=128, n_pages=100, page_stride=16384,
             head_stride=2048, token_stride=128)
    f.update(kw)
    return A._KVCache(*[f[n] for n, _ in A._KVCache._fields_])


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(type=0), dict(type=8), dict(n_kv_heads=0),
              dict(n_kv_heads=-1), dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(page_size=131072),
              dict(head_dim=0), dict(head_dim=4), dict(head_dim=100), dict(head_dim=264), dict(n_pages=0),
              dict(n_pages=1 << 28), dict(page_stride=16380), dict(page_stride=8192), dict(page_stride=-16384),
              dict(head_stride=2044), dict(head_stride=1024), dict(token_stride=120), dict(token_stride=64),
              dict(head_stride=1 << 50), dict(page_stride=1 << 62)]


def test_declared_entry_points_are_exported():
    names = set(re.findall(r"\b(hip_qmm_\w+)\(", HEADER.read_text()))
    assert len(names) == 9
    L = A._lib()
    assert all(hasattr(L, n) for n in names)


def test_structure_layout():
    assert C.sizeof(A._KVCache) == 64 and A._KVCache.n_pages.offset == 32


def _rope(cache=None, **kw):
    f = dict(q=P, n_heads=32, q_token=4096, q_head=128, k=P, v=P, kv_token=1024, kv_head=128, n=0, pos=P, steps=P,
             n_dims=128, layout=2, mscale=1.0, dst=P, dst_token=4096, dst_head=128, slots=P)
    f.update(kw)
    c = _cache() if cache is None else cache
    return A._lib().hip_qmm_rope_kv_store(f["q"], f["n_heads"], f["q_token"], f["q_head"], f["k"], f["v"], f["kv_token"],
                                          f["kv_head"], f["n"], f["pos"], f["steps"], f["n_dims"], f["layout"],
                                          f["mscale"], f["dst"], f["dst_token"], f["dst_head"], C.addressof(c),
                                          f["slots"], None)


def test_rope_refusals():
    assert _rope() == 0  # no tokens: nothing to do
    assert _rope(n_heads=0, q=None, dst=None) == 0
    for kw in (dict(n=-1), dict(n=(1 << 23) + 1), dict(n_heads=-1), dict(q=None), dict(dst=None), dict(k=None),
               dict(v=None), dict(pos=None), dict(steps=None), dict(slots=None), dict(n_dims=0), dict(n_dims=3),
               dict(n_dims=130), dict(n_dims=-2), dict(layout=1), dict(layout=-1), dict(mscale=math.nan), dict(n=2, q_head=64),
               dict(n=2, q_token=100), dict(n=2, dst_token=4000), dict(n=2, kv_token=-1), dict(n=2, kv_head=100)):
        assert _rope(**kw) == BAD, kw
    for kw in BAD_CACHES:
        assert _rope(_cache(**kw), n=1) == BAD, kw
    assert A._lib().hip_qmm_rope_kv_store(P, 0, 0, 0, P, P, 0, 0, 0, P, P, 128, 2, 1.0, P, 0, 0, None, P, None) == BAD
    f = A._lib().hip_qmm_rope_f32
    assert f(P, 0, 4, 128, 512, 128, P, P, 128, 2, 1.0, P, 512, 128, None) == 0
    assert f(P, 5, 0, 128, 512, 128, P, P, 128, 2, 1.0, P, 512, 128, None) == 0
    for a in ((None, 1, 4, 128, 512, 128, P, P, 128, 2), (P, 1, 4, 1025, 5000, 1025, P, P, 128, 2),
              (P, 1, 4, 64, 512, 128, P, P, 128, 2), (P, 2, 4, 128, 500, 128, P, P, 128, 2),
              (P, 1, 4, 128, 512, 128, P, P, 128, 3)):
        assert f(*a, 1.0, P, 5000, 1025, None) == BAD, a


def test_rope_steps():
    L = A._lib()
    steps, m = (C.c_int64 * 128)(), C.c_float()

    def call(n=128, base=1e4, scale=1.0, ext=0.0, att=1.0, fast=32.0, slow=1.0, ctx=0, fac=None):
        return L.hip_qmm_rope_steps(n, base, scale, ext, att, fast, slow, ctx, fac, C.addressof(steps), C.addressof(m))

    assert call() == 0 and m.value == 1.0
    for i in (0, 1, 17, 63):
        want = 1e4 ** (-2 * i / 128) / (2 * math.pi) * 2.0 ** 64
        assert abs(steps[i] - want) <= want * 2.0 ** -49
    # over half a turn a position wraps to a negative step: the same turns
    fac = (C.c_float * 64)(*([0.25] * 64))
    assert call(fac=C.addressof(fac)) == 0
    assert abs(steps[0] - (4 / (2 * math.pi) - 1) * 2.0 ** 64) <= 2.0 ** 14
    for kw in (dict(n=0), dict(n=3), dict(n=258), dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(scale=0.0),
               dict(scale=-1.0), dict(ext=-1.0), dict(ext=math.nan), dict(att=math.inf), dict(ext=1.0), dict(ext=1.0, ctx=100, fast=0.0)):
        assert call(**kw) == BAD, kw
    for bad in (0.0, -1.0, math.nan, math.inf):
        fac[5] = bad
        assert call(fac=C.addressof(fac)) == BAD


def _attn(cache=None, **kw):
    f = dict(q=P, n_heads=32, q_token=4096, q_head=128, starts=P, n_seqs=0, n=0, max_q=0, table=P, width=10, lens=P,
             max_kv=160, scale=0.1, window=0, sinks=0, dst=P, dst_token=4096, dst_head=128, ws=P, ws_size=1 << 40)
    f.update(kw)
    c = _cache() if cache is None else cache
    return A._lib().hip_qmm_attn_paged(C.addressof(c), f["q"], f["n_heads"], f["q_token"], f["q_head"], f["starts"],
                                       f["n_seqs"], f["n"], f["max_q"], f["table"], f["width"], f["lens"], f["max_kv"],
                                       f["scale"], f["window"], f["sinks"], f["dst"], f["dst_token"], f["dst_head"],
                                       f["ws"], f["ws_size"], None)


def test_attention_refusals():
    assert _attn() == 0
    one = dict(n_seqs=1, n=4, max_q=4)
    for kw in (dict(n_heads=0), dict(n_heads=31), dict(n_heads=-32), dict(n_seqs=-1), dict(n_seqs=70000), dict(n=-1),
               dict(n=(1 << 23) + 1), dict(max_q=-1), dict(max_q=5), dict(max_kv=-1), dict(max_kv=(1 << 30) + 1), dict(scale=math.nan),
               dict(scale=3e38),
               dict(scale=math.inf), dict(window=-1), dict(sinks=-1), dict(window=1 << 31), dict(sinks=1 << 31),
               dict(width=-1), dict(width=1 << 31), dict(starts=None), dict(q=None), dict(dst=None), dict(lens=None),
               dict(table=None), dict(q=P + 4), dict(dst=P + 8), dict(q_token=4098), dict(q_head=126),
               dict(dst_token=4095), dict(dst_head=64), dict(dst_token=2048), dict(q_token=-4), dict(dst_head=-128),
               dict(q_token=1 << 50)):
        assert _attn(**{**one, **kw}) == BAD, kw
    for kw in BAD_CACHES:
        assert _attn(_cache(**kw), **one) == BAD, kw
    need = A._lib().hip_qmm_attn_paged_workspace_size(C.addressof(_cache()), 32, 1, 1, 1, 100000, 0, 0)
    far = dict(n_seqs=1, n=1, max_q=1, starts=None, width=10000, max_kv=100000)
    if need:
        assert _attn(**far, ws_size=need - 1) == BAD and _attn(**far, ws=None) == BAD and _attn(**far, ws=P + 4) == BAD


def test_workspace_size_of_what_is_refused():
    f = A._lib().hip_qmm_attn_paged_workspace_size
    assert f(None, 32, 1, 1, 1, 100, 0, 0) == 0
    assert f(C.addressof(_cache()), 31, 1, 1, 1, 100, 0, 0) == 0
    assert f(C.addressof(_cache()), 32, -1, 1, 1, 100, 0, 0) == 0


def test_plan():
    """Every kernel form is reached, and what is refused has no plan."""
    f = A._lib().hip_qmm_attn_paged_rows
    splits = C.c_int()

    def plan(n_seqs, new, kv, window=0, sinks=0, heads=32, **cache):
        c = _cache(**cache)
        rows = f(C.addressof(c), heads, n_seqs, n_seqs * new, new, kv, window, sinks, C.addressof(splits))
        need = A._lib().hip_qmm_attn_paged_workspace_size(C.addressof(c), heads, n_seqs, n_seqs * new, new, kv, window, sinks)
        assert (need > 0) == (splits.value > 1)
        assert need == 0 or need == splits.value * n_seqs * new * heads * (c.head_dim + 2) * 4
        assert 1 <= splits.value <= 256
        return rows, splits.value

    assert plan(1, 1, 333) == (16, 1)
    assert plan(1, 1, 131072) == (16, 32)
    assert plan(1, 1, 131072, 1024, 4)[1] < 16
    assert plan(64, 1, 4096)[0] == 16
    assert plan(1, 50, 50) == (16, 1)
    assert plan(1, 7, 4000)[0] == 32
    assert plan(2, 13, 20000)[0] == 64 and splits.value > 1
    assert plan(1, 1000, 1000) == (64, 1)
    assert plan(1, 4096, 4096) == (128, 1)
    assert plan(1, 512, 32768)[0] == 128 and splits.value > 1
    assert plan(1, 1, 1 << 30) == (16, 32)
    wide = dict(head_dim=256, token_stride=256, head_stride=4096, page_stride=32768)
    assert plan(1, 7, 4000, **wide)[0] == plan(1, 1000, 1000, **wide)[0] == plan(1, 9000, 9000, **wide)[0] == 64
    assert plan(1, 4, 4000, **wide)[0] == plan(1, 100, 100, **wide)[0] == 16 and plan(1, 200, 200, **wide)[0] == 64
    assert plan(1, 1, 1 << 20, heads=1, n_kv_heads=1) == (16, 256)
    assert f(None, 32, 1, 1, 1, 100, 0, 0, None) == 0
    c = _cache()
    assert f(C.addressof(c), 31, 1, 1, 1, 100, 0, 0, None) == 0 and f(C.addressof(c), 32, 1, 1, 0, 100, 0, 0, None) == 0


def _compact(cache=None, **kw):
    f = dict(table=P, stride=10, width=10, lens=P, n_seqs=1, out=P, out_stride=10, live=P, ws=P, size=1 << 30)
    f.update(kw)
    c = _cache() if cache is None else cache
    return A._lib().hip_qmm_kv_compact(C.addressof(c), f["table"], f["stride"], f["width"], f["lens"], f["n_seqs"],
                                       f["out"], f["out_stride"], f["live"], f["ws"], f["size"], None)


def test_page_refusals():
    L = A._lib()
    good = _cache()
    at = C.addressof(good)
    assert L.hip_qmm_kv_copy_pages(at, P, P, None, 0, None) == 0 and L.hip_qmm_kv_copy_pages(at, None, None, None, 0, None) == 0
    for a in ((None, P, P, None, 1), (at, None, P, None, 1), (at, P, None, None, 1), (at, P, P, None, -1)):
        assert L.hip_qmm_kv_copy_pages(*a, None) == BAD, a
    need = L.hip_qmm_kv_compact_workspace_size(at)
    assert need >= 100 * 4
    big = dict(head_dim=8, page_stride=1024, head_stride=128, token_stride=8)
    for kw in (dict(stride=9), dict(out_stride=9), dict(width=-1), dict(n_seqs=-1), dict(live=None), dict(ws=None), dict(ws=P + 2),
               dict(size=need - 1), dict(table=None), dict(lens=None), dict(out=None), dict(stride=11)):
        assert _compact(**kw) == BAD, kw
    assert _compact(_cache(n_pages=(1 << 20) + 1, **big)) == BAD
    assert L.hip_qmm_kv_compact_workspace_size(C.addressof(_cache(n_pages=(1 << 20) + 1, **big))) == 0
    for kw in BAD_CACHES:
        c = _cache(**kw)
        assert L.hip_qmm_kv_copy_pages(C.addressof(c), P, P, None, 1, None) == BAD, kw
        assert _compact(c) == BAD and L.hip_qmm_kv_compact_workspace_size(C.addressof(c)) == 0, kw


def test_python_refusals_without_a_gpu():
    torch = pytest.importorskip("torch")
    cpu = torch.zeros((4, 2, 16, 64), dtype=torch.float16)
    for k, v in ((cpu, cpu), (cpu.float(), cpu.float()), (cpu, cpu[:2]), (cpu[0], cpu[0])):
        with pytest.raises(G.HipQmmError):
            G.PagedKV(k, v)
    with pytest.raises(G.HipQmmError):
        G.rope_steps(3, device="cpu")
    with pytest.raises(G.HipQmmError):
        G.rope_steps(64, freq_factors=[1.0] * 3, device="cpu")
    x = torch.zeros((2, 2, 64))
    with pytest.raises(G.HipQmmError):
        G.rope(x, torch.zeros(2, dtype=torch.int32), torch.zeros(32, dtype=torch.int64))
