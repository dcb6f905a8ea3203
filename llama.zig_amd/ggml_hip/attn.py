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

from . import HipQmmError, _check, _stream
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
        L.hip_qmm_kv_copy_pages.argtypes = [vp, vp, vp, vp, i64, vp]
        L.hip_qmm_kv_compact_workspace_size.restype = size
        L.hip_qmm_kv_compact_workspace_size.argtypes = [vp]
        L.hip_qmm_kv_compact.argtypes = [vp, vp, i64, i64, vp, i64, vp, i64, vp, vp, size, vp]
        _bound = L
    return _bound


def _need(ok, what):
    if not ok:
        raise HipQmmError(what)


def _int32(t, n, name):
    _need(t.dtype == torch.int32 and t.is_cuda and t.is_contiguous() and t.numel() == n,
          f"{name} must be {n} contiguous int32 values on the GPU")


class PagedKV:
    """One layer's cache: k and v f16 or bf16 [n_pages, n_kv_heads, page_size,
    head_dim], of equal strides with contiguous head_dim (a view with heads and
    tokens, or k and v, interleaved will do)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in _KV_TYPES,
              "k and v must be f16 or bf16 [n_pages, n_kv_heads, page_size, head_dim], alike")
        _need(k.is_cuda and v.device == k.device, "tensors must live on the GPU")
        _need(k.stride(3) == 1 and k.stride() == v.stride(), "k and v must have the same strides, head_dim contiguous")
        self.k, self.v = k, v
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


def _heads(t, name):
    _need(t.is_cuda and t.dtype == torch.float32 and t.dim() == 3 and t.stride(2) == 1,
          f"{name} must be f32 [n_tokens, n_heads, head_dim] on the GPU, head_dim contiguous")


def _rotation(pos, steps, n, layout):
    _int32(pos, n, "pos")
    _need(steps.dtype == torch.int64 and steps.is_cuda and steps.dim() == 1 and steps.is_contiguous(),
          "steps must be what rope_steps returns")
    _need(layout in ROPE_LAYOUTS, f"layout must be one of {sorted(ROPE_LAYOUTS)}")
    return ROPE_LAYOUTS[layout]


def rope(x: torch.Tensor, pos: torch.Tensor, steps: torch.Tensor, layout="half", mscale=1.0, out=None):
    """x f32 [n_tokens, n_heads, head_dim] with the first 2 * len(steps)
    elements of each head rotated by pos int32 [n_tokens]; out may be x."""
    _heads(x, "x")
    mode = _rotation(pos, steps, x.shape[0], layout)
    out = torch.empty(x.shape, dtype=torch.float32, device=x.device) if out is None else out
    _heads(out, "out")
    _need(out.shape == x.shape, "out must have x's shape")
    n, h, d = x.shape
    _check(_lib().hip_qmm_rope_f32(x.data_ptr(), n, h, d, x.stride(0), x.stride(1), pos.data_ptr(), steps.data_ptr(),
                                   2 * steps.numel(), mode, mscale, out.data_ptr(), out.stride(0), out.stride(1),
                                   _stream()), "hip_qmm_rope_f32")
    return out


def rope_kv_store(q, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, steps: torch.Tensor, kv: PagedKV,
                  slots: torch.Tensor, layout="half", mscale=1.0, out=None):
    """Rotates q and k f32 [n_tokens, heads, head_dim], stores the rotated k and
    the plain v at cache slots int32 [n_tokens] (page * page_size + token;
    outside the cache: not stored) and returns the rotated q.  q may be None."""
    _heads(k, "k")
    _heads(v, "v")
    n, h, d = k.shape
    _need(v.shape == k.shape and v.stride() == k.stride(), "k and v must have the same shape and strides")
    _need((h, d) == (kv.n_kv_heads, kv.head_dim), "k and v must have the cache's heads and head_dim")
    mode = _rotation(pos, steps, n, layout)
    _int32(slots, n, "slots")
    if q is None:
        _check(_lib().hip_qmm_rope_kv_store(None, 0, 0, 0, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), n,
                                            pos.data_ptr(), steps.data_ptr(), 2 * steps.numel(), mode, mscale, None, 0,
                                            0, kv._p, slots.data_ptr(), _stream()), "hip_qmm_rope_kv_store")
        return None
    _heads(q, "q")
    _need(q.shape[0] == n and q.shape[2] == d, "q and k disagree on the tokens or head_dim")
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device) if out is None else out
    _heads(out, "out")
    _need(out.shape == q.shape, "out must have q's shape")
    _check(_lib().hip_qmm_rope_kv_store(q.data_ptr(), q.shape[1], q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(),
                                        k.stride(0), k.stride(1), n, pos.data_ptr(), steps.data_ptr(),
                                        2 * steps.numel(), mode, mscale, out.data_ptr(), out.stride(0), out.stride(1),
                                        kv._p, slots.data_ptr(), _stream()), "hip_qmm_rope_kv_store")
    return out


def attn_paged_workspace_size(kv: PagedKV, n_heads: int, n_seqs: int, n_tokens: int, max_q: int, max_kv: int,
                              window=0, sinks=0) -> int:
    return int(_lib().hip_qmm_attn_paged_workspace_size(kv._p, n_heads, n_seqs, n_tokens, max_q, max_kv, window,
                                                        sinks))


def attn_paged(q: torch.Tensor, kv: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts=None,
               max_q=None, max_kv=None, scale=None, window=0, sinks=0, out=None, workspace=None):
    """Attention of the newest tokens over the paged cache, causal: q f32
    [n_tokens, n_heads, head_dim]; page_table int32 [n_seqs, width]; kv_lens
    int32 [n_seqs], the new tokens included; q_starts int32 [n_seqs + 1] of
    ragged batches (None: one token per sequence), then with max_q, the most
    new tokens of a sequence.  A query at position p sees token j <= p if
    window is 0, p - j < window or j < sinks; entries outside the pool hide
    their tokens; nothing seen gives zeros.  max_kv: the longest length that
    the host knows of.  scale: head_dim ** -0.5 by default."""
    _heads(q, "q")
    n, h, d = q.shape
    _need(d == kv.head_dim, "q must have the cache's head_dim")
    _need(page_table.dtype == torch.int32 and page_table.is_cuda and page_table.dim() == 2 and
          page_table.stride(1) == 1 and page_table.stride(0) >= page_table.shape[1],
          "page_table must be int32 [n_seqs, width] on the GPU")
    n_seqs, width = page_table.shape
    _int32(kv_lens, n_seqs, "kv_lens")
    if q_starts is None:
        _need(n == n_seqs, "one token per sequence without q_starts")
        max_q = 1 if n else 0
    else:
        _int32(q_starts, n_seqs + 1, "q_starts")
        max_q = n if max_q is None else max_q
    if page_table.stride(0) != width:  # the row stride is the width that lengths are cut to
        page_table = page_table.contiguous()
    if max_kv is None or max_kv > width * kv.page_size:
        max_kv = width * kv.page_size
    scale = d ** -0.5 if scale is None else scale
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device) if out is None else out
    _heads(out, "out")
    _need(out.shape == q.shape, "out must have q's shape")
    L = _lib()
    need = L.hip_qmm_attn_paged_workspace_size(kv._p, h, n_seqs, n, max_q, max_kv, window, sinks)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    elif workspace.numel() < need:
        raise HipQmmError(f"workspace too small: {workspace.numel()} < {need}")
    _check(L.hip_qmm_attn_paged(kv._p, q.data_ptr(), h, q.stride(0), q.stride(1),
                                None if q_starts is None else q_starts.data_ptr(), n_seqs, n, max_q,
                                page_table.data_ptr(), width, kv_lens.data_ptr(), max_kv, scale, window, sinks,
                                out.data_ptr(), out.stride(0), out.stride(1), workspace.data_ptr(),
                                workspace.numel(), _stream()), "hip_qmm_attn_paged")
    return out


def copy_pages(kv: PagedKV, src: torch.Tensor, dst: torch.Tensor, n_tokens=None):
    """Copies the first n_tokens[i] tokens (None: all) of page src[i] into page
    dst[i], keys and values: what a fork does with the partly filled last page."""
    n = src.numel()
    _int32(src, n, "src")
    _int32(dst, n, "dst")
    if n_tokens is not None:
        _int32(n_tokens, n, "n_tokens")
    _check(_lib().hip_qmm_kv_copy_pages(kv._p, src.data_ptr(), dst.data_ptr(),
                                        None if n_tokens is None else n_tokens.data_ptr(), n, _stream()),
           "hip_qmm_kv_copy_pages")


def compact_pages(kv: PagedKV, page_table: torch.Tensor, kv_lens: torch.Tensor, out=None, workspace=None):
    """Moves the pages in use (those that kv_lens' tokens need) to the front of
    the pool: (the table with their new numbers and -1 elsewhere, int32; the
    count of pages in use, int32 [1]), both on the device.  out may be
    page_table."""
    _need(page_table.dtype == torch.int32 and page_table.is_cuda and page_table.dim() == 2 and
          page_table.stride(1) == 1, "page_table must be int32 [n_seqs, width] on the GPU")
    n_seqs, width = page_table.shape
    _int32(kv_lens, n_seqs, "kv_lens")
    out = torch.empty((n_seqs, width), dtype=torch.int32, device=page_table.device) if out is None else out
    _need(out.dtype == torch.int32 and out.is_cuda and out.shape == page_table.shape and out.stride(1) == 1,
          "out must be int32 of page_table's shape")
    n_live = torch.empty(1, dtype=torch.int32, device=page_table.device)
    L = _lib()
    need = L.hip_qmm_kv_compact_workspace_size(kv._p)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=page_table.device)
    elif workspace.numel() < need:
        raise HipQmmError(f"workspace too small: {workspace.numel()} < {need}")
    _check(L.hip_qmm_kv_compact(kv._p, page_table.data_ptr(), page_table.stride(0), width, kv_lens.data_ptr(), n_seqs,
                                out.data_ptr(), out.stride(0), n_live.data_ptr(), workspace.data_ptr(),
                                workspace.numel(), _stream()), "hip_qmm_kv_compact")
    return out, n_live
