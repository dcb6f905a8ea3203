"""Host-side mirror of a mixture-of-experts layer's operators
(include/ggml_hip_moe.h): the choice of each token's experts, matrix products in
8-bit integers with a scale for each token and each channel, dense and by
experts, and the weighted sum of the experts' rows.

8-bit tensors are int8 with rows 16-byte aligned, a multiple of 16 bytes apart;
`quantize_i8` makes them, of tokens and of weights alike.  Activations are f32.
"""
from __future__ import annotations

import ctypes

import torch

from . import HipQmmError, _check
from . import lib as _base_lib
from .attn import _raw_stream, _scratch

GATINGS = {"softmax": 0, "sigmoid": 1, "softmax_chosen": 2}
_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32

_bound = None


def _lib():
    global _bound
    if _bound is None:
        L = _base_lib()
        vp, i64, i32, f32, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
        L.hip_qmm_moe_route.argtypes = [vp, i64, i64, i64, vp, i32, i64, i64, i32, i64, i32, f32, f32, vp, i64, vp, i64,
                                        vp]
        L.hip_qmm_quantize_i8.argtypes = [vp, i64, i64, i64, vp, i64, vp, vp]
        L.hip_qmm_mul_mat_i8_workspace_size.restype = size
        L.hip_qmm_mul_mat_i8_workspace_size.argtypes = [i64, i64, i64, i32]
        L.hip_qmm_mul_mat_i8.argtypes = [vp, vp, i64, i64, i64, vp, vp, i64, i64, vp, i64, vp, size, vp]
        L.hip_qmm_mul_mat_id_i8_workspace_size.restype = size
        L.hip_qmm_mul_mat_id_i8_workspace_size.argtypes = [i64, i64, i64, i64, i64, i64, i32]
        L.hip_qmm_mul_mat_id_i8.argtypes = [vp, vp, i64, i64, i64, i64, i64, vp, vp, i64, i64, i64, vp, i64, i64, vp,
                                            i64, vp, size, vp]
        L.hip_qmm_moe_combine.argtypes = [vp, i64, i64, i64, i64, i64, vp, i64, vp, i64, vp, i64, vp, i64, vp]
        _bound = L
    return _bound


# The checks build their messages only when they refuse, and ask little of a contiguous tensor: a step's call lasts a few
# microseconds.
def _rows(t, shape, dtype, name, device):
    """The stride between rows of a [.., n] tensor of the shape, its last dimension contiguous."""
    if t.dtype is not dtype or t.get_device() != device or t.shape != shape or device < 0:
        raise HipQmmError(f"{name} must be {dtype} {list(shape)} on the GPU (of the others), not {t.dtype} {list(t.shape)}")
    n = shape[-1]
    if t.is_contiguous():
        return n
    stride = t.stride(-2)
    if n > 1 and t.stride(-1) != 1:
        raise HipQmmError(f"{name}'s last dimension must be contiguous")
    if shape[-2] <= 1:
        return max(stride, n)
    if stride < n:
        raise HipQmmError(f"{name}'s rows must not overlap")
    return stride


def _flat(t, n, dtype, name, device):
    if t.dtype is not dtype or t.get_device() != device or t.numel() != n or not t.is_contiguous():
        raise HipQmmError(f"{name} must be {n} contiguous {dtype} values on the GPU of the others")
    return t.data_ptr()


def _rows3(t, shape, dtype, name, device):
    """The stride between rows of a 3-D tensor whose first two dimensions run on as one."""
    stride = _rows(t, shape, dtype, name, device)
    if t.is_contiguous():
        return stride
    a, b, n = shape
    sa, sb, _ = t.stride()
    if a > 1 and b > 1 and sa != b * sb:
        raise HipQmmError(f"{name}'s first two dimensions must be evenly spaced")
    return sb if b > 1 else sa if a > 1 else max(sb, n)


def _i8_rows(t, stride, name):
    """The stride of 8-bit rows, 2-D or 3-D, as the products take them; the last one's chunk of 16 bytes may end behind the
    row, but not behind the tensor's memory."""
    size = t.shape
    n = size[-1]
    if n % 16:
        if not t.numel():
            return stride
        whole = (n + 15) // 16 * 16
        last = t.storage_offset() + (size[-2] - 1) * stride
        if len(size) == 3:
            last += (size[0] - 1) * t.stride(0)
        if last + whole > t.untyped_storage().nbytes():
            raise HipQmmError(f"{name}'s last row must end in memory of the tensor's up to 16 bytes")
        if t.numel() == n:  # one row
            stride = whole
    if (stride % 16 or t.data_ptr() % 16) and t.numel():
        raise HipQmmError(f"{name}'s rows must be 16-byte aligned (quantize_i8 lays them so)")
    return stride


def route(logits: torch.Tensor, k: int, gating="softmax", bias=None, groups=1, keep=1, top=2, renormalize=False,
          min_sum=2.0 ** -14, scale=1.0, ids=None, weights=None):
    """The k experts of each token and their weights: (ids int32 [n_tokens, k],
    weights f32 [n_tokens, k]), best first.  logits f32 [n_tokens, n_experts];
    gating "softmax", "sigmoid" or "softmax_chosen" (softmax over the chosen
    ones); bias f32 [n_experts] is added to what is compared, not to the weights.
    Only the `keep` of `groups` groups of neighbouring experts whose `top` (1 or
    2) best scores sum highest are chosen from.  renormalize divides the
    weights by their sum, at least min_sum; scale multiplies them.  An expert
    whose logit or bias is -inf is never chosen; where none is left the id is
    -1 and the weight 0."""
    device, size = logits.get_device(), logits.shape
    if len(size) != 2:
        raise HipQmmError("logits must be f32 [n_tokens, n_experts]")
    n, e = size
    ls = _rows(logits, size, _F32, "logits", device)
    bp = None if bias is None else _flat(bias, e, _F32, "bias", device)
    mode = GATINGS.get(gating)
    if mode is None:
        raise HipQmmError(f"gating must be one of {sorted(GATINGS)}")
    if k < 1:
        raise HipQmmError("k must be at least 1")
    shape = (n, k)
    if ids is None:
        ids, si = logits.new_empty(shape, dtype=_I32), k
    else:
        si = _rows(ids, shape, _I32, "ids", device)
    if weights is None:
        weights, sw = logits.new_empty(n, k), k
    else:
        sw = _rows(weights, shape, _F32, "weights", device)
    _check(_lib().hip_qmm_moe_route(logits.data_ptr(), n, e, ls, bp, mode, groups, keep, top, k, bool(renormalize),
                                    min_sum, scale, ids.data_ptr(), si, weights.data_ptr(), sw, _raw_stream(device)),
           "hip_qmm_moe_route")
    return ids, weights


def quantize_i8(x: torch.Tensor, out=None, scale=None):
    """f32 [.., K] to 8-bit rows: (int8 [.., K], scale f32 [..]) with x near
    q * scale, scale = max|x| * (1/127) of each row; of tokens, or of weights with a
    row per channel.  The result's rows are 16-byte aligned."""
    device, K = x.get_device(), x.shape[-1] if x.dim() else 0
    if device < 0 or x.dtype is not _F32 or x.dim() < 2:
        raise HipQmmError("x must be f32 [.., K] on the GPU")
    lead = x.shape[:-1]
    if x.dim() > 2:
        if not x.is_contiguous():
            raise HipQmmError("x of more than two dimensions must be contiguous")
        flat = x.view(lead.numel(), K)
    else:
        flat = x
    n = flat.shape[0]
    xs = _rows(flat, flat.shape, _F32, "x", device)
    if out is None:
        qs = (K + 15) // 16 * 16
        out = x.new_empty((*lead, qs), dtype=_I8)[..., :K]
    else:
        if out.shape != x.shape or out.dtype is not _I8 or out.get_device() != device or (K > 1 and out.stride(-1) != 1):
            raise HipQmmError("out must be int8 of x's shape on its GPU, its last dimension contiguous")
        if out.dim() > 3:
            raise HipQmmError("out of more than three dimensions")
        qs = (_rows3 if out.dim() == 3 else _rows)(out, out.shape, _I8, "out", device)
        if n > 1 and qs < K:
            raise HipQmmError("out's rows must not overlap")
    if scale is None:
        scale = x.new_empty(lead)
    sp = _flat(scale, n, _F32, "scale", device)
    if n:
        _check(_lib().hip_qmm_quantize_i8(flat.data_ptr(), K, n, xs, out.data_ptr(), qs, sp, _raw_stream(device)),
               "hip_qmm_quantize_i8")
    return out, scale


def mul_mat_i8(w: torch.Tensor, w_scale: torch.Tensor, x: torch.Tensor, x_scale=None, out=None, workspace=None):
    """f32 [n, rows]: (x . w) * x_scale[n] * w_scale[row], summed in integers.
    w int8 [rows, K], w_scale f32 [rows]; x int8 [n, K] with x_scale f32 [n], or
    f32 [n, K], quantized in the call."""
    device, size, xsize = w.get_device(), w.shape, x.shape
    if len(size) != 2 or len(xsize) != 2:
        raise HipQmmError("w and x must be 2-D")
    rows, K = size
    n = xsize[0]
    ws = _i8_rows(w, _rows(w, size, _I8, "w", device), "w")
    sp = _flat(w_scale, rows, _F32, "w_scale", device)
    if x_scale is None:
        xs, xp = _rows(x, (n, K), _F32, "x", device), None
    else:
        xs = _i8_rows(x, _rows(x, (n, K), _I8, "x", device), "x")
        xp = _flat(x_scale, n, _F32, "x_scale", device)
    if out is None:
        out, os_ = w_scale.new_empty(n, rows), rows
    else:
        os_ = _rows(out, (n, rows), _F32, "out", device)
    L = _lib()
    if n == 0:
        return out
    if workspace is None:
        # What the header promises of int8 tokens and of many: cheaper than to ask.
        have = 0 if xp is not None else n * (K + 131) + 512 if n > 32 else L.hip_qmm_mul_mat_i8_workspace_size(K, rows, n, 0)
        wp = None
        if have:
            workspace = w_scale.new_empty(have, dtype=torch.uint8)
            wp = workspace.data_ptr()
    else:
        wp, have = _scratch(workspace, L.hip_qmm_mul_mat_i8_workspace_size(K, rows, n, xp is not None), device)
    _check(L.hip_qmm_mul_mat_i8(w.data_ptr(), sp, K, rows, ws, x.data_ptr(), xp, n, xs, out.data_ptr(), os_, wp, have,
                                _raw_stream(device)), "hip_qmm_mul_mat_i8")
    return out


def mul_mat_id_i8(w: torch.Tensor, w_scale: torch.Tensor, x: torch.Tensor, ids: torch.Tensor, x_scale=None, out=None,
                  workspace=None):
    """f32 [n_tokens, n_ids, rows]: row (t, s) is the product of expert
    ids[t, s] with x[t, s], or x[t, 0]; zeros for an id outside [0, n_experts).
    w int8 [n_experts, rows, K], w_scale f32 [n_experts, rows]; x int8 [n_tokens,
    1 or n_ids, K] with x_scale f32 of its first two dimensions, or f32,
    quantized in the call; ids int32 [n_tokens, n_ids]."""
    device, size, xsize, isize = w.get_device(), w.shape, x.shape, ids.shape
    if len(size) != 3 or len(xsize) != 3 or len(isize) != 2:
        raise HipQmmError("w and x must be 3-D, ids 2-D")
    e, rows, K = size
    n, ne11, _ = xsize
    n_ids = isize[1]
    ws = _rows(w, size, _I8, "w", device)
    # One row an expert: what lies between two is the experts' stride (w[:, None]'s own is the row's length).
    ws = _i8_rows(w, w.stride(0) if rows == 1 and e > 1 else ws, "w")
    es = w.stride(0) if e > 1 else rows * ws
    sp = _flat(w_scale, e * rows, _F32, "w_scale", device)
    if x_scale is None:
        xs, xp = _rows3(x, (n, ne11, K), _F32, "x", device), None
    else:
        xs = _i8_rows(x, _rows3(x, (n, ne11, K), _I8, "x", device), "x")
        xp = _flat(x_scale, n * ne11, _F32, "x_scale", device)
    si = _rows(ids, (n, n_ids), _I32, "ids", device)
    if out is None:
        out, os_ = w_scale.new_empty(n, n_ids, rows), rows
    else:
        os_ = _rows3(out, (n, n_ids, rows), _F32, "out", device)
    L = _lib()
    if n * n_ids == 0:
        return out
    need = L.hip_qmm_mul_mat_id_i8_workspace_size(K, rows, e, ne11, n, n_ids, xp is not None)
    if workspace is None:
        wp, have = None, need
        if need:
            workspace = w_scale.new_empty(need, dtype=torch.uint8)
            wp = workspace.data_ptr()
    else:
        wp, have = _scratch(workspace, need, device)
    _check(L.hip_qmm_mul_mat_id_i8(w.data_ptr(), sp, K, rows, ws, es, e, x.data_ptr(), xp, ne11, n, xs, ids.data_ptr(),
                                   n_ids, si, out.data_ptr(), os_, wp, have, _raw_stream(device)), "hip_qmm_mul_mat_id_i8")
    return out


def combine(y: torch.Tensor, weights: torch.Tensor, ids=None, add=None, out=None):
    """f32 [n_tokens, rows]: the sum of y[t, s] * weights[t, s] over the slots,
    and add[t].  y f32 [n_tokens, n_ids, rows], weights f32 [n_tokens, n_ids];
    with ids int32 [n_tokens, n_ids], slots of negative ids are left out.  out
    may be add."""
    device, size = y.get_device(), y.shape
    if len(size) != 3 or y.dtype is not _F32 or device < 0:
        raise HipQmmError("y must be f32 [n_tokens, n_ids, rows] on the GPU")
    n, n_ids, rows = size
    yt, ys, yc = y.stride()
    if yc != 1 and rows > 1:
        raise HipQmmError("y's rows must be contiguous")
    sw = _rows(weights, (n, n_ids), _F32, "weights", device)
    ip, si = (None, 0) if ids is None else (ids.data_ptr(), _rows(ids, (n, n_ids), _I32, "ids", device))
    ap, sa = (None, 0) if add is None else (add.data_ptr(), _rows(add, (n, rows), _F32, "add", device))
    if out is None:
        out, so = y.new_empty(n, rows), rows
    else:
        so = _rows(out, (n, rows), _F32, "out", device)
    if n * rows == 0:
        return out
    _check(_lib().hip_qmm_moe_combine(y.data_ptr(), n, n_ids, rows, yt, ys, weights.data_ptr(), sw, ip, si, ap, sa,
                                      out.data_ptr(), so, _raw_stream(device)), "hip_qmm_moe_combine")
    return out
