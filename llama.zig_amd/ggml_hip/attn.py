"""Host-side mirror of the operators between the quantized projections
(include/ggml_hip_attn.h): rotary positions with the store into a paged
key-value cache, attention over that cache, and the upkeep of its pages.

A cache is a pair of f16 or bf16 tensors [n_pages, n_kv_heads, page_size,
head_dim] (`PagedKV`); a sequence's token j lies in page
page_table[s, j // page_size].  Activations are f32.
"""
from __future__ import annotations

import ctypes

import torch

from . import HipQmmError, _check
from . import lib as _base_lib

ROPE_LAYOUTS = {"interleaved": 0, "half": 2}
_KV_TYPES = {torch.float16: 1, torch.bfloat16: 30}

_bound = None


class _KVCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("type", ctypes.c_int32),
                ("n_kv_heads", ctypes.c_int32), ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("n_pages", ctypes.c_int64), ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
                ("token_stride", ctypes.c_int64)]


def _lib():
    global _bound
    if _bound is None:
        L = _base_lib()
        vp, i64, i32, f32, f64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_double
        size = ctypes.c_size_t
        L.hip_qmm_rope_steps.argtypes = [i32, f64, f64, f64, f64, f64, f64, i64, vp, vp, vp]
        L.hip_qmm_rope_f32.argtypes = [vp, i64, i64, i64, i64, i64, vp, vp, i32, i32, f32, vp, i64, i64, vp]
        L.hip_qmm_rope_kv_store.argtypes = [vp, i64, i64, i64, vp, vp, i64, i64, i64, vp, vp, i32, i32, f32, vp, i64,
                                            i64, vp, vp, vp]
        L.hip_qmm_attn_paged_workspace_size.restype = size
        L.hip_qmm_attn_paged_workspace_size.argtypes = [vp, i64, i64, i64, i64, i64, i64, i64]
        L.hip_qmm_attn_paged.argtypes = [vp, vp, i64, i64, i64, vp, i64, i64, i64, vp, i64, vp, i64, f32, i64, i64, vp,
                                         i64, i64, vp, size, vp]
        L.hip_qmm_attn_paged_rows.argtypes = [vp, i64, i64, i64, i64, i64, i64, i64, vp]
        L.hip_qmm_kv_copy_pages.argtypes = [vp, vp, vp, vp, i64, vp]
        L.hip_qmm_kv_compact_workspace_size.restype = size
        L.hip_qmm_kv_compact_workspace_size.argtypes = [vp]
        L.hip_qmm_kv_compact.argtypes = [vp, vp, i64, i64, vp, i64, vp, i64, vp, vp, size, vp]
        _bound = L
    return _bound


# The checks build their messages only when they refuse, and look up little: a step's call lasts a few microseconds.
_C, _I32, _I64, _F32 = torch._C, torch.int32, torch.int64, torch.float32


def _need(ok, what):
    if not ok:
        raise HipQmmError(what)


def _raw_stream(device):
    # A launch goes to the current device, whatever its stream's.
    if device != _C._cuda_getDevice():
        raise HipQmmError("tensors must live on the current GPU")
    return _C._cuda_getCurrentRawStream(device)


def _int32(t, n, name, device):
    if not (t.dtype is _I32 and t.get_device() == device and t.numel() == n and t.is_contiguous()):
        raise HipQmmError(f"{name} must be {n} contiguous int32 values on the GPU of the others")


def _scratch(workspace, need, device):
    """A caller's scratch, checked: its address and bytes."""
    have = workspace.numel() * workspace.element_size()
    if have < need:
        raise HipQmmError(f"workspace too small: {have} < {need}")
    if need and not (workspace.get_device() == device and workspace.is_contiguous()):
        raise HipQmmError("workspace must be contiguous, on the GPU of the others")
    return workspace.data_ptr(), have


class PagedKV:
    """One layer's cache: k and v f16 or bf16 [n_pages, n_kv_heads, page_size,
    head_dim], of equal strides with contiguous head_dim (a view with heads and
    tokens, or k and v, interleaved will do)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in _KV_TYPES,
              "k and v must be f16 or bf16 [n_pages, n_kv_heads, page_size, head_dim], alike")
        _need(k.is_cuda and v.device == k.device, "tensors must live on the GPU")
        _need(k.stride(3) == 1 and k.stride() == v.stride(), "k and v must have the same strides, head_dim contiguous")
        self.k, self.v, self._device = k, v, k.get_device()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self._c = _KVCache(k.data_ptr(), v.data_ptr(), _KV_TYPES[k.dtype], self.n_kv_heads, self.page_size,
                           self.head_dim, self.n_pages, k.stride(0), k.stride(1), k.stride(2))
        self._p = ctypes.addressof(self._c)


def rope_steps(n_dims: int, freq_base=10000.0, freq_scale=1.0, ext_factor=0.0, attn_factor=1.0, beta_fast=32.0,
               beta_slow=1.0, n_ctx_orig=0, freq_factors=None, device="cuda"):
    """A model's rotations: (steps int64 [n_dims / 2] on the device, in units of
    2^-64 turns per position; the magnitude scale).  freq_scale interpolates
    positions, ext_factor > 0 mixes it with the plain frequencies (YaRN)."""
    steps = torch.zeros(max(n_dims // 2, 1), dtype=torch.int64)
    mscale = ctypes.c_float()
    if freq_factors is not None:
        freq_factors = torch.as_tensor(freq_factors, dtype=torch.float32).cpu().contiguous()
        _need(freq_factors.numel() == n_dims // 2, "freq_factors must hold n_dims / 2 values")
    _check(_lib().hip_qmm_rope_steps(n_dims, freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow,
                                     n_ctx_orig, None if freq_factors is None else freq_factors.data_ptr(),
                                     steps.data_ptr(), ctypes.addressof(mscale)), "hip_qmm_rope_steps")
    return steps.to(device), mscale.value


def _heads(t, name, device):
    """Token and head stride of f32 [n_tokens, n_heads, head_dim]."""
    if not (t.get_device() == device >= 0 and t.dtype is _F32 and t.dim() == 3):
        raise HipQmmError(f"{name} must be f32 [n_tokens, n_heads, head_dim] on the GPU (of the others)")
    st, sh, sd = t.stride()
    if sd != 1:
        raise HipQmmError(f"{name}'s head_dim must be contiguous")
    return st, sh


def _result(out, x):
    """out, checked, or a new tensor of x's shape; with its strides."""
    if out is None:
        n, h, d = x.shape
        return x.new_empty((n, h, d)), h * d, d
    st, sh = _heads(out, "out", x.get_device())
    _need(out.shape == x.shape, "out must have the shape of its input")
    return out, st, sh


def _rotation(pos, steps, n, layout, device):
    _int32(pos, n, "pos", device)
    if not (steps.dtype is _I64 and steps.get_device() == device and steps.dim() == 1 and steps.is_contiguous()):
        raise HipQmmError("steps must be what rope_steps returns, on the GPU of the others")
    mode = ROPE_LAYOUTS.get(layout)
    if mode is None:
        raise HipQmmError(f"layout must be one of {sorted(ROPE_LAYOUTS)}")
    return mode, 2 * steps.numel()


def rope(x: torch.Tensor, pos: torch.Tensor, steps: torch.Tensor, layout="half", mscale=1.0, out=None):
    """x f32 [n_tokens, n_heads, head_dim] with the first 2 * len(steps)
    elements of each head rotated by pos int32 [n_tokens]; out may be x."""
    device = x.get_device()
    xt, xh = _heads(x, "x", device)
    n, h, d = x.shape
    mode, n_dims = _rotation(pos, steps, n, layout, device)
    out, ot, oh = _result(out, x)
    if n * h == 0:  # empty tensors have no address
        return out
    _check(_lib().hip_qmm_rope_f32(x.data_ptr(), n, h, d, xt, xh, pos.data_ptr(), steps.data_ptr(), n_dims, mode, mscale,
                                   out.data_ptr(), ot, oh, _raw_stream(device)), "hip_qmm_rope_f32")
    return out


def rope_kv_store(q, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, steps: torch.Tensor, kv: PagedKV,
                  slots: torch.Tensor, layout="half", mscale=1.0, out=None):
    """Rotates q and k f32 [n_tokens, heads, head_dim], stores the rotated k and
    the plain v at cache slots int32 [n_tokens] (page * page_size + token;
    outside the cache: not stored) and returns the rotated q.  q may be None."""
    device = kv._device
    kt, kh = _heads(k, "k", device)
    n, h, d = k.shape
    if _heads(v, "v", device) != (kt, kh) or v.shape != k.shape:
        raise HipQmmError("k and v must have the same shape and strides")
    if h != kv.n_kv_heads or d != kv.head_dim:
        raise HipQmmError("k and v must have the cache's heads and head_dim")
    mode, n_dims = _rotation(pos, steps, n, layout, device)
    _int32(slots, n, "slots", device)
    qp = op = None
    heads = qt = qh = ot = oh = 0
    if q is not None:
        qt, qh = _heads(q, "q", device)
        nq, heads, dq = q.shape
        if nq != n or dq != d:
            raise HipQmmError("q and k disagree on the tokens or head_dim")
        out, ot, oh = _result(out, q)
        qp, op = q.data_ptr(), out.data_ptr()
    else:
        out = None
    if n == 0:
        return out
    _check(_lib().hip_qmm_rope_kv_store(qp, heads, qt, qh, k.data_ptr(), v.data_ptr(), kt, kh, n, pos.data_ptr(),
                                        steps.data_ptr(), n_dims, mode, mscale, op, ot, oh, kv._p, slots.data_ptr(),
                                        _raw_stream(device)), "hip_qmm_rope_kv_store")
    return out


def attn_paged_workspace_size(kv: PagedKV, n_heads: int, n_seqs: int, n_tokens: int, max_q: int, max_kv: int,
                              window=0, sinks=0) -> int:
    return int(_lib().hip_qmm_attn_paged_workspace_size(kv._p, n_heads, n_seqs, n_tokens, max_q, max_kv, window,
                                                        sinks))


def attn_paged_plan(kv: PagedKV, n_heads: int, n_seqs: int, n_tokens: int, max_q: int, max_kv: int, window=0, sinks=0):
    """(rows of a workgroup, splits of a row's tokens at most) that attn_paged runs, for measurement and tests."""
    splits = ctypes.c_int()
    rows = _lib().hip_qmm_attn_paged_rows(kv._p, n_heads, n_seqs, n_tokens, max_q, max_kv, window, sinks,
                                          ctypes.addressof(splits))
    return rows, splits.value


def _table(t, device):
    if not (t.dtype is _I32 and t.get_device() == device and t.dim() == 2 and t.stride(1) == 1
            and t.stride(0) >= t.shape[1]):
        raise HipQmmError("page_table must be int32 [n_seqs, width] on the GPU of the others, its rows contiguous and apart")
    return t.shape


def attn_paged(q: torch.Tensor, kv: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts=None,
               max_q=None, max_kv=None, scale=None, window=0, sinks=0, out=None, workspace=None):
    """Attention of the newest tokens over the paged cache, causal: q f32
    [n_tokens, n_heads, head_dim]; page_table int32 [n_seqs, width]; kv_lens
    int32 [n_seqs], the new tokens included; q_starts int32 [n_seqs + 1] of
    ragged batches (None: one token per sequence), then with max_q, the most
    new tokens of a sequence.  A query at position p sees token j <= p if
    window is 0, p - j < window or j < sinks; entries outside the pool hide
    their tokens; nothing seen gives zeros.  max_kv: the longest length that
    the host knows of.  scale: head_dim ** -0.5 by default.  out does not
    overlap q."""
    device = kv._device
    qt, qh = _heads(q, "q", device)
    n, h, d = q.shape
    if d != kv.head_dim:
        raise HipQmmError("q must have the cache's head_dim")
    n_seqs, width = _table(page_table, device)
    _int32(kv_lens, n_seqs, "kv_lens", device)
    starts = None
    if q_starts is None:
        if n != n_seqs:
            raise HipQmmError("one token per sequence without q_starts")
        max_q = 1 if n else 0
    else:
        _int32(q_starts, n_seqs + 1, "q_starts", device)
        starts = q_starts.data_ptr()
        max_q = n if max_q is None else max_q
    if not page_table.is_contiguous():  # the row stride is the width that lengths are cut to
        page_table = page_table.contiguous()
    most = min(width * kv.page_size, 1 << 30)
    max_kv = most if max_kv is None or max_kv > most else max_kv
    out, ot, oh = _result(out, q)
    L = _lib()
    need = L.hip_qmm_attn_paged_workspace_size(kv._p, h, n_seqs, n, max_q, max_kv, window, sinks)
    if workspace is None:
        have, wp = need, None
        if need:
            workspace = q.new_empty(need, dtype=torch.uint8)
            wp = workspace.data_ptr()
    else:
        wp, have = _scratch(workspace, need, device)
    _check(L.hip_qmm_attn_paged(kv._p, q.data_ptr(), h, qt, qh, starts, n_seqs, n, max_q, page_table.data_ptr(), width,
                                kv_lens.data_ptr(), max_kv, d ** -0.5 if scale is None else scale, window, sinks,
                                out.data_ptr(), ot, oh, wp, have, _raw_stream(device)), "hip_qmm_attn_paged")
    return out


def copy_pages(kv: PagedKV, src: torch.Tensor, dst: torch.Tensor, n_tokens=None):
    """Copies the first n_tokens[i] tokens (None: all) of page src[i] into page
    dst[i], keys and values: what a fork does with the partly filled last page."""
    n = src.numel()
    device = kv._device
    _int32(src, n, "src", device)
    _int32(dst, n, "dst", device)
    if n_tokens is not None:
        _int32(n_tokens, n, "n_tokens", device)
    _check(_lib().hip_qmm_kv_copy_pages(kv._p, src.data_ptr(), dst.data_ptr(),
                                        None if n_tokens is None else n_tokens.data_ptr(), n, _raw_stream(device)),
           "hip_qmm_kv_copy_pages")


def compact_pages(kv: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, out=None, workspace=None):
    """Moves the pages in use (those that kv_lens' tokens need) to the front of
    the pool: (the table with their new numbers and -1 elsewhere, int32; the
    count of pages in use, int32 [1]), both on the device.  out may be
    page_table."""
    device = kv._device
    n_seqs, width = _table(page_table, device)
    _int32(kv_lens, n_seqs, "kv_lens", device)
    if out is None:
        out = page_table.new_empty((n_seqs, width))
    _need(_table(out, device) == page_table.shape, "out must have page_table's shape")
    n_live = page_table.new_empty(1)
    L = _lib()
    need = L.hip_qmm_kv_compact_workspace_size(kv._p)
    if workspace is None:
        workspace = page_table.new_empty(max(need, 1), dtype=torch.uint8)
    wp, have = _scratch(workspace, need, device)
    _check(L.hip_qmm_kv_compact(kv._p, page_table.data_ptr(), page_table.stride(0), width, kv_lens.data_ptr(), n_seqs,
                                out.data_ptr(), out.stride(0), n_live.data_ptr(), wp, have, _raw_stream(device)),
           "hip_qmm_kv_compact")
    return out, n_live
