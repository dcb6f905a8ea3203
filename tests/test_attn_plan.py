"""The limits of hip_qmm_attn_paged and what its queries say of them, on the CPU."""
import ctypes as C

import pytest

from ggml_hip import attn as A
from test_attn_abi import BAD, _attn, _cache

MOST = 1 << 23  # workgroups


def _plan(n_seqs, n, max_q, max_kv, heads=32, window=0, sinks=0, **cache):
    c, splits = _cache(**cache), C.c_int(-1)
    args = (C.addressof(c), heads, n_seqs, n, max_q, max_kv, window, sinks)
    rows = A._lib().hip_qmm_attn_paged_rows(*args, C.addressof(splits))
    return rows, splits.value, A._lib().hip_qmm_attn_paged_workspace_size(*args)


@pytest.mark.parametrize("n_seqs", [256, 4096, 4097, 30000, 65535])
@pytest.mark.parametrize("max_kv", [1, 333, 131072, 1 << 20, 1 << 30])
@pytest.mark.parametrize("new", [1, 7, 100])
def test_planning_lengths_are_never_refused(n_seqs, max_kv, new):
    """max_kv only plans: where the splits it asks for are too many workgroups there are fewer of them."""
    rows, splits, size = _plan(n_seqs, n_seqs * new, new, max_kv)
    assert rows in (16, 32, 64, 128)
    assert 1 <= splits <= 256 and splits * -(-new * 4 // rows) * 8 * n_seqs <= MOST
    assert size == (splits * n_seqs * new * 32 * 130 * 4 if splits > 1 else 0)


def test_too_many_workgroups_have_no_plan():
    for n_seqs, n, max_q in ((128, 524288, 524288), (65535, 1 << 23, 5000)):
        assert _plan(n_seqs, n, max_q, 4096) == (0, -1, 0)
        assert _attn(n_seqs=n_seqs, n=n, max_q=max_q, max_kv=4096) == BAD
    assert _plan(128, 524288, 4096, 4096)[0] == 128
    # 2^16 workgroups of a key-value head at 128 rows, times 128 heads: the last that fits
    most = dict(n_kv_heads=128, page_stride=2048 * 128)
    assert _plan(1, 1 << 23, 1 << 23, 1, heads=128, **most)[0] == 128
    assert _plan(2, 1 << 23, 1 << 23, 1, heads=128, **most) == (0, -1, 0)
