"""Thin wrappers that call the C ABI on torch device tensors.

torch only supplies device memory and the current HIP stream; every
computation below is one call into libghostflow_hip.so.  Each wrapper checks
dtype / contiguity / device on the host and raises GhostFlowError with the
library's status code and thread-local message when a call fails.
"""
from __future__ import annotations

import struct
from functools import lru_cache

import torch

from . import _lib


class GhostFlowError(RuntimeError):
    """A non-zero status from the C ABI (GhostFlowError codes)."""

    def __init__(self, status: int, message: str):
        self.status = status
        name = _lib.STATUS_NAMES.get(status, str(status))
        super().__init__(f"{name}: {message}")


def _check(rc: int) -> None:
    if rc != _lib.SUCCESS:
        msg = _lib.load().gfh_last_error()
        raise GhostFlowError(rc, msg.decode() if msg else "")


def _stream(dev=None) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace_bytes(ws):
    """Bytes a caller workspace holds, whatever its dtype: numel times the
    element size.  The workspace must be a contiguous device tensor."""
    if ws is None:
        return 0
    if not ws.is_cuda:
        raise GhostFlowError(_lib.INVALID_DATA, "workspace must be a device tensor")
    if not ws.is_contiguous():
        raise GhostFlowError(_lib.INVALID_DATA, "workspace must be contiguous")
    return ws.numel() * ws.element_size()


def _workspace(ws):
    """(pointer, bytes) of a caller workspace, (None, 0) without one."""
    return (None, 0) if ws is None else (ws.data_ptr(), _workspace_bytes(ws))


def _need(t, dtype, name):
    if t is None:
        return
    if not t.is_cuda:
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be contiguous")


_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _dtype(t, name):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return d


def _same_device(dev, *tensors):
    for t in tensors:
        if t is not None and t.device != dev:
            raise GhostFlowError(_lib.INVALID_DATA, f"all tensors must be on {dev}, one is on {t.device}")


def _call(dev, fn, *args):
    """fn(*args, stream) on dev's current stream, with dev the current device
    (a launch goes to the current one).  A call costs about as much host time
    as a decode step's kernels take: the device is only switched where it has
    to be, and the stream comes as its handle."""
    index = dev.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != _lib.SUCCESS:
        _check(rc)


def lib():
    return _lib.load()


def init() -> None:
    _check(lib().gfh_init())


def set_pointer_checks(enabled: bool) -> None:
    _check(lib().gfh_set_pointer_checks(1 if enabled else 0))


# ---- fp32 GEMM --------------------------------------------------------------

def sgemm(a, b, *, trans_a=False, trans_b=False, alpha=1.0, beta=0.0, bias=None, out=None):
    """out = alpha * op(a) @ op(b) + beta * out (+ bias), 2-D row-major."""
    _need(a, torch.float32, "a")
    _need(b, torch.float32, "b")
    _need(bias, torch.float32, "bias")
    m, k = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    k2, n = (b.shape[1], b.shape[0]) if trans_b else (b.shape[0], b.shape[1])
    if k != k2:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{m}, {k}] got [{k2}, {n}]")
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    _need(out, torch.float32, "out")
    _check(lib().gfh_sgemm(int(trans_a), int(trans_b), m, n, k, float(alpha), a.data_ptr(),
                           max(a.shape[1], 1), b.data_ptr(), max(b.shape[1], 1),
                           float(beta), out.data_ptr(), max(n, 1), _ptr(bias), _stream(a.device)))
    return out


def matmul(a, b):
    """Tensor::matmul (ghostflow-core/src/ops/matmul.rs:13-42): 2-D -> GEMM,
    otherwise the batched form with modulo batch indexing (:122-170)."""
    _need(a, torch.float32, "a")
    _need(b, torch.float32, "b")
    if a.dim() < 2 or b.dim() < 2:
        raise GhostFlowError(_lib.INVALID_SHAPE, "matmul requires at least 2D tensors")
    m, k = a.shape[-2:]
    k2, n = b.shape[-2:]
    if k != k2:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{m}, {k}] got [{k2}, {n}]")
    if a.dim() == 2 and b.dim() == 2:
        return sgemm(a, b)
    batch_shape = torch.broadcast_shapes(a.shape[:-2], b.shape[:-2])
    batch = 1
    for s in batch_shape:
        batch *= s
    ba = 1
    for s in a.shape[:-2]:
        ba *= s
    bb = 1
    for s in b.shape[:-2]:
        bb *= s
    out = torch.empty(tuple(batch_shape) + (m, n), dtype=torch.float32, device=a.device)
    _check(lib().gfh_sgemm_strided_batched(0, 0, m, n, k, 1.0, a.data_ptr(), k, m * k, max(ba, 1),
                                           b.data_ptr(), n, k * n, max(bb, 1), 0.0, out.data_ptr(),
                                           n, m * n, batch, None, _stream(a.device)))
    return out


def linear(x, weight, bias=None):
    """Linear::forward (ghostflow-nn/src/linear.rs:56-69): x @ W^T + b."""
    return sgemm(x, weight, trans_b=True, bias=bias)


# ---- int8 quantization ---------------------------------------------------------

def matmul_backward(grad, a, b, *, need_a=True, need_b=True):
    """matmul_backward (ghostflow-autograd/src/backward.rs:131-160) for
    C = a @ b: returns (grad @ b^T, a^T @ grad); a part not needed is None."""
    for t, n in ((grad, "grad"), (a, "a"), (b, "b")):
        _need(t, torch.float32, n)
    m, k = a.shape
    n = b.shape[1]
    if b.shape[0] != k or tuple(grad.shape) != (m, n):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch a {list(a.shape)} b {list(b.shape)} "
                             f"grad {list(grad.shape)}")
    ga = torch.empty((m, k), dtype=torch.float32, device=a.device) if need_a else None
    gb = torch.empty((k, n), dtype=torch.float32, device=a.device) if need_b else None
    _check(lib().gfh_matmul_backward_f32(grad.data_ptr(), a.data_ptr(), b.data_ptr(), m, k, n, _ptr(ga), _ptr(gb),
                                         _stream(a.device)))
    return ga, gb


def quantize_per_channel(x, symmetric=True):
    _need(x, torch.float32, "x")
    rows = x.shape[0]
    cols = x.numel() // rows if rows else 0
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    z = torch.empty(rows, dtype=torch.int8, device=x.device)
    _check(lib().gfh_quantize_i8_per_channel(x.data_ptr(), rows, cols, int(bool(symmetric)),
                                             q.data_ptr(), s.data_ptr(), z.data_ptr(),
                                             _stream(x.device)))
    return q, s, z


def quantize_per_tensor(x, symmetric=False, workspace=None):
    _need(x, torch.float32, "x")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    s = torch.empty(1, dtype=torch.float32, device=x.device)
    z = torch.empty(1, dtype=torch.int8, device=x.device)
    ws_ptr, ws_bytes = _workspace(workspace)
    _check(lib().gfh_quantize_i8_per_tensor(x.data_ptr(), x.numel(), int(bool(symmetric)),
                                            q.data_ptr(), s.data_ptr(), z.data_ptr(),
                                            ws_ptr, ws_bytes, _stream(x.device)))
    return q, s, z


def quantize_per_tensor_workspace_size(n: int) -> int:
    return int(lib().gfh_quantize_i8_per_tensor_workspace_size(n))


def dequantize(q, scales, zero_points):
    _need(q, torch.int8, "q")
    _need(scales, torch.float32, "scales")
    _need(zero_points, torch.int8, "zero_points")
    rows = q.shape[0] if q.dim() else 1
    cols = q.numel() // rows if rows else 0
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    _check(lib().gfh_dequantize_i8(q.data_ptr(), rows, cols, scales.data_ptr(), zero_points.data_ptr(),
                                   scales.numel(), out.data_ptr(), _stream(q.device)))
    return out


def qweight_rowsum(qw):
    _need(qw, torch.int8, "qw")
    n, k = qw.shape
    out = torch.empty(n, dtype=torch.int32, device=qw.device)
    _check(lib().gfh_qweight_rowsum(qw.data_ptr(), n, k, out.data_ptr(), _stream(qw.device)))
    return out


def qlinear(qx, sx, zx, qw, sw, *, x_per_row=False, w_rowsum=None, bias=None, want_y=True,
            want_acc=False):
    _need(qx, torch.int8, "qx")
    _need(qw, torch.int8, "qw")
    _need(sx, torch.float32, "sx")
    _need(sw, torch.float32, "sw")
    _need(zx, torch.int8, "zx")
    _need(w_rowsum, torch.int32, "w_rowsum")
    _need(bias, torch.float32, "bias")
    m, k = qx.shape
    n = qw.shape[0]
    if qw.shape[1] != k:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{m}, {k}] got [{qw.shape[1]}, {n}]")
    if zx is not None and w_rowsum is None:
        w_rowsum = qweight_rowsum(qw)
    y = torch.empty((m, n), dtype=torch.float32, device=qx.device) if want_y else None
    acc = torch.empty((m, n), dtype=torch.int32, device=qx.device) if want_acc else None
    _check(lib().gfh_qlinear_i8(qx.data_ptr(), _ptr(sx), _ptr(zx), int(bool(x_per_row)), qw.data_ptr(),
                                _ptr(sw), _ptr(w_rowsum), _ptr(bias), _ptr(y), _ptr(acc), m, n, k,
                                _stream(qx.device)))
    return y, acc


def qlinear_dynamic(x, qw, sw, w_rowsum, *, bias=None, out=None, workspace=None):
    """The INT8 linear on fp32 activations x [m, k]: quantize_activation
    (per tensor, asymmetric, quantization.rs:280-287) then qlinear with the
    per-channel weight codes qw [n, k]; y [m, n].  Same codes and outputs as
    quantize_per_tensor followed by qlinear, in one launch for m <= 4."""
    _need(x, torch.float32, "x")
    _need(qw, torch.int8, "qw")
    _need(sw, torch.float32, "sw")
    _need(w_rowsum, torch.int32, "w_rowsum")
    _need(bias, torch.float32, "bias")
    m, k = x.shape
    n = qw.shape[0]
    if qw.shape[1] != k:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{m}, {k}] got [{qw.shape[1]}, {n}]")
    y = torch.empty((m, n), dtype=torch.float32, device=x.device) if out is None else out
    ws_ptr, ws_bytes = _workspace(workspace)
    _check(lib().gfh_qlinear_dynamic_i8(x.data_ptr(), qw.data_ptr(), sw.data_ptr(), w_rowsum.data_ptr(),
                                        _ptr(bias), y.data_ptr(), m, n, k, ws_ptr, ws_bytes, _stream(x.device)))
    return y


# ---- 4-bit weights in groups ------------------------------------------------------

def _groups(k, group_size):
    return -(-k // group_size) if group_size > 0 else 0


def quantize_grouped_i4(w, group_size=128, symmetric=True):
    """4-bit codes [n, k / 2] (two per byte, even column low), fp32 scales
    [n, groups] and zero points [n, groups] (bytes; None if symmetric) of a
    Linear weight w [n, k], a scale per group of group_size columns; k and
    group_size are multiples of 32.  gfh_quantize_i4_grouped in
    ghostflow_hip.h has the formulas."""
    _need(w, torch.float32, "w")
    if w.dim() != 2:
        raise GhostFlowError(_lib.INVALID_SHAPE, "w must be [n, k]")
    n, k = w.shape
    groups = _groups(k, group_size)
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((n, groups), dtype=torch.float32, device=w.device)
    zps = None if symmetric else torch.empty((n, groups), dtype=torch.uint8, device=w.device)
    _call(w.device, lib().gfh_quantize_i4_grouped, w.data_ptr(), n, k, group_size, codes.data_ptr(), scales.data_ptr(),
          _ptr(zps))
    return codes, scales, zps


def _need_w4(codes, scales, zero_points, group_size):
    _need(codes, torch.uint8, "codes")
    _need(scales, torch.float32, "scales")
    _need(zero_points, torch.uint8, "zero_points")
    if codes.dim() != 2:
        raise GhostFlowError(_lib.INVALID_SHAPE, "codes must be [n, k / 2]")
    n, k = codes.shape[0], 2 * codes.shape[1]
    want = (n, _groups(k, group_size))
    for t, name in ((scales, "scales"), (zero_points, "zero_points")):
        if t is not None and t.shape != want:
            raise GhostFlowError(_lib.INVALID_SHAPE, f"{name} must be {list(want)} for groups of {group_size}, got "
                                 f"{list(t.shape)}")
    return n, k


def dequantize_grouped_i4(codes, scales, zero_points=None, group_size=128):
    """The weight [n, k] in fp32 that quantize_grouped_i4's result stands for."""
    n, k = _need_w4(codes, scales, zero_points, group_size)
    _same_device(codes.device, scales, zero_points)
    out = torch.empty((n, k), dtype=torch.float32, device=codes.device)
    _call(codes.device, lib().gfh_dequantize_i4_grouped, codes.data_ptr(), scales.data_ptr(), _ptr(zero_points), n, k,
          group_size, out.data_ptr())
    return out


def linear_w4_workspace_size(m: int, n: int, k: int, group_size: int = 128, dtype=torch.float32) -> int:
    """Bytes of linear_w4's workspace for x [m, k] and a weight [n, k]."""
    return int(lib().gfh_linear_w4_workspace_size(_DTYPES.get(dtype, -1), m, n, k, group_size))


def linear_w4(x, codes, scales, zero_points=None, bias=None, *, group_size=128, out=None, workspace=None):
    """Linear::forward (linear.rs:56-69) on a 4-bit weight: y = x . W'^T + bias
    for x [m, k] (rows may be strided), of float32, bfloat16 or float16 like
    bias and y."""
    n, k = _need_w4(codes, scales, zero_points, group_size)
    if not x.is_cuda:
        raise GhostFlowError(_lib.INVALID_DATA, "x must be a device tensor")
    dt = _dtype(x, "x")
    if x.dim() != 2 or x.shape[1] != k:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"x must be [m, {k}], got {list(x.shape)}")
    m = x.shape[0]
    if k > 1 and x.stride(1) != 1:
        raise GhostFlowError(_lib.INVALID_DATA, "the columns of x must be contiguous")
    _need(bias, x.dtype, "bias")
    if bias is not None and tuple(bias.shape) != (n,):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"bias must be [{n}], got {list(bias.shape)}")
    y = torch.empty((m, n), dtype=x.dtype, device=x.device) if out is None else out
    _need(y, x.dtype, "out")
    if tuple(y.shape) != (m, n):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"out must be [{m}, {n}], got {list(y.shape)}")
    _same_device(x.device, codes, scales, zero_points, bias, y, workspace)
    ws, ws_bytes = _workspace(workspace)
    _call(x.device, lib().gfh_linear_w4, dt, x.data_ptr(), x.stride(0) if m > 1 else k, codes.data_ptr(),
          scales.data_ptr(), _ptr(zero_points), _ptr(bias), y.data_ptr(), n, m, n, k, group_size, ws, ws_bytes)
    return y


# ---- GEMV ---------------------------------------------------------------------

def gemv_f32(x, w, out=None):
    _need(x, torch.float32, "x")
    _need(w, torch.float32, "w")
    b, k = x.shape
    n = w.shape[1]
    if w.shape[0] != k:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{b}, {k}] got [{w.shape[0]}, {n}]")
    y = torch.empty((b, n), dtype=torch.float32, device=x.device) if out is None else out
    _check(lib().gfh_gemv_f32(x.data_ptr(), w.data_ptr(), y.data_ptr(), b, k, n, _stream(x.device)))
    return y


def gemv_w8(x, qw, scales, zero_points=None, out=None):
    _need(x, torch.float32, "x")
    _need(qw, torch.int8, "qw")
    _need(scales, torch.float32, "scales")
    _need(zero_points, torch.int8, "zero_points")
    b, k = x.shape
    n = qw.shape[1]
    if qw.shape[0] != k:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch expected [{b}, {k}] got [{qw.shape[0]}, {n}]")
    y = torch.empty((b, n), dtype=torch.float32, device=x.device) if out is None else out
    _check(lib().gfh_gemv_w8(x.data_ptr(), qw.data_ptr(), scales.data_ptr(), _ptr(zero_points),
                             y.data_ptr(), b, k, n, _stream(x.device)))
    return y


# ---- attention ------------------------------------------------------------------

def softmax_lastdim(x, out=None):
    _need(x, torch.float32, "x")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    y = torch.empty_like(x) if out is None else out
    _check(lib().gfh_softmax_lastdim_f32(x.data_ptr(), y.data_ptr(), rows, cols, _stream(x.device)))
    return y


_SAMPLING = struct.Struct("@PPPPfiff")  # gfh_sampling


def sample_workspace_size(rows: int, vocab: int) -> int:
    """Bytes of sample's workspace for logits [rows, vocab]."""
    return int(lib().gfh_sample_workspace_size(rows, vocab))


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, want_logprobs=False, out=None, workspace=None):
    """A token (int32) per row of logits [rows, vocab] (rows may be strided), of
    float32, bfloat16 or float16, drawn with the uniform numbers u [rows] in
    [0, 1): temperature (0: the largest logit), then top_k (0: all), top_p (1:
    all) and min_p (0: all), each a number or a tensor [rows] (float32, top_k
    int32).  With want_logprobs also the logarithm of the token's probability
    among those that were left.  gfh_sample in ghostflow_hip.h has the rules;
    a row of which nothing can be drawn gets -1."""
    if not logits.is_cuda:
        raise GhostFlowError(_lib.INVALID_DATA, "logits must be a device tensor")
    dt, dev = _dtype(logits, "logits"), logits.device
    if logits.dim() != 2:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"logits must be [rows, vocab], got {list(logits.shape)}")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise GhostFlowError(_lib.INVALID_DATA, "the entries of a row of logits must be contiguous")
    ptrs, values = [], []
    for name, x, dtype, kind in (("temperature", temperature, torch.float32, float), ("top_k", top_k, torch.int32, int),
                                 ("top_p", top_p, torch.float32, float), ("min_p", min_p, torch.float32, float)):
        if torch.is_tensor(x):
            _need_rows(x, dtype, name, rows, dev)
            ptrs.append(x.data_ptr())
            values.append(0)
        else:
            ptrs.append(0)
            values.append(kind(x))
    if not -2 ** 31 <= values[1] < 2 ** 31:
        values[1] = 0  # more than there are
    _need_rows(u, torch.float32, "u", rows, dev)
    tokens = torch.empty(rows, dtype=torch.int32, device=dev) if out is None else out
    _need_rows(tokens, torch.int32, "out", rows, dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev) if want_logprobs else None
    ws, ws_bytes = None, 0
    if workspace is not None:
        _same_device(dev, workspace)
        ws, ws_bytes = _workspace(workspace)
    _call(dev, lib().gfh_sample, dt, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, u.data_ptr(),
          _SAMPLING.pack(*ptrs, *values), tokens.data_ptr(), _ptr(logprobs), ws, ws_bytes)
    return (tokens, logprobs) if want_logprobs else tokens


def _need_rows(t, dtype, name, rows, dev):
    if t.dtype is not dtype or t.get_device() != dev.index or not t.is_contiguous():
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be a contiguous {dtype} tensor on {dev}")
    if t.shape != (rows,):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"{name} must be [{rows}], got {list(t.shape)}")


def sdpa(q, k, v, *, scale=None, causal=False, mask=None, want_weights=False, out=None):
    """Fused scaled_dot_product_attention on [B, H, S, D] tensors."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, torch.float32, nm)
    _need(mask, torch.float32, "mask")
    b, h, sq, d = q.shape
    skv = k.shape[2]
    if scale is None:
        scale = _inv_sqrt(d)
    o = torch.empty_like(q) if out is None else out
    w = torch.empty((b, h, sq, skv), dtype=torch.float32, device=q.device) if want_weights else None
    _check(lib().gfh_sdpa_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(w), b, h, sq,
                              skv, d, float(scale), int(bool(causal)), _ptr(mask),
                              0 if mask is None else mask.numel(), _stream(q.device)))
    return (o, w) if want_weights else o


def flash_attention_blockwise(q, k, v, *, block_size_m=64, block_size_n=64, causal=False, scale=1.0,
                              out=None, workspace=None):
    """FlashAttention::forward (ghostflow-nn/src/flash_attention.rs:81-250)
    on q [B, Sq, d], k / v [B, Sk, d]: the reference's blockwise recurrence
    with its block sizes, causal flag (top-left j > i) and scale, including
    its once-per-key correction (softmax attention only at block_size_n ==
    1).  Errors as the reference: non-3-D inputs, a d_model mismatch."""
    for t, nm in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, torch.float32, nm)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise GhostFlowError(_lib.INVALID_SHAPE, "Expected 3D tensors [batch, seq_len, d_model]")
    b, sq, d = q.shape
    sk = k.shape[1]
    if k.shape[2] != d or v.shape[2] != d:
        raise GhostFlowError(_lib.INVALID_SHAPE, "Key and Value must have same d_model as Query")
    if k.shape[0] != b or v.shape[0] != b or v.shape[1] != sk:
        raise GhostFlowError(_lib.INVALID_SHAPE, "key / value must be [batch, seq_len_k, d_model] like query")
    o = torch.empty_like(q) if out is None else out
    _check(lib().gfh_flash_attention_f32(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), b, sq, sk, d,
                                         int(block_size_m), int(block_size_n), int(bool(causal)), float(scale),
                                         _ptr(workspace), _workspace_bytes(workspace), _stream(q.device)))
    return o


def kv_attention(q, k_cache, v_cache, kv_len, num_heads, *, scale=None, causal=False, mask=None,
                 want_weights=False, out=None):
    """Attention of q [B, Sq, E] over the first kv_len rows of the caches
    [B, C, E] (head h = columns h*D .. h*D+D-1, D = E / num_heads): the
    scaled_dot_product_attention step of MultiHeadAttention::
    forward_with_cache (ghostflow-nn/src/attention.rs:100-144) with the
    concatenated keys read in place.  Returns out [B, Sq, E] (and the
    [B, H, Sq, kv_len] weights)."""
    for t, nm in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(t, torch.float32, nm)
    _need(mask, torch.float32, "mask")
    b, sq, e = q.shape
    cap = k_cache.shape[1]
    if tuple(k_cache.shape) != (b, cap, e) or tuple(v_cache.shape) != (b, cap, e):
        raise GhostFlowError(_lib.INVALID_SHAPE, "k_cache / v_cache must be [B, C, E] like q")
    if e % num_heads:
        raise GhostFlowError(_lib.INVALID_SHAPE, "embed_dim must be divisible by num_heads")
    d = e // num_heads
    if scale is None:
        scale = _inv_sqrt(d)
    o = torch.empty_like(q) if out is None else out
    w = torch.empty((b, num_heads, sq, kv_len), dtype=torch.float32, device=q.device) if want_weights else None
    _check(lib().gfh_kv_attention_f32(q.data_ptr(), e, k_cache.data_ptr(), v_cache.data_ptr(), cap, e,
                                      o.data_ptr(), e, _ptr(w), b, num_heads, sq, kv_len, d, float(scale),
                                      int(bool(causal)), _ptr(mask), 0 if mask is None else mask.numel(),
                                      _stream(q.device)))
    return (o, w) if want_weights else o


@lru_cache(maxsize=None)
def _inv_sqrt(d):
    """1.0f32 / (d as f32).sqrt() (attention.rs:19-20), in float32."""
    return float(torch.tensor(1.0, dtype=torch.float32) / torch.sqrt(torch.tensor(float(d), dtype=torch.float32)))


# ---- multi-head attention with a key/value cache ------------------------------------

def mha_workspace_size(b: int, sq: int, e: int) -> int:
    return int(lib().gfh_mha_workspace_size(b, sq, e))


def mha_forward_cached(query, key, value, wq, bq, wk, bk, wv, bv, wo, bo, num_heads, k_cache, v_cache,
                       past_len, *, mask=None, causal=False, want_weights=False, out=None, workspace=None):
    """MultiHeadAttention::forward_with_cache on an in-place cache: writes
    the projected key/value rows into k_cache / v_cache [B, C, E] at
    [past_len, past_len + Sk) and attends over rows [0, past_len + Sk).
    Returns out [B, Sq, E] (and the [B, H, Sq, past_len + Sk] weights)."""
    for t, nm in ((query, "query"), (key, "key"), (value, "value"), (wq, "wq"), (wk, "wk"), (wv, "wv"),
                  (wo, "wo"), (bq, "bq"), (bk, "bk"), (bv, "bv"), (bo, "bo"), (k_cache, "k_cache"),
                  (v_cache, "v_cache"), (mask, "mask")):
        _need(t, torch.float32, nm)
    b, sq, e = query.shape
    sk = key.shape[1]
    if tuple(key.shape) != (b, sk, e) or tuple(value.shape) != (b, sk, e):
        raise GhostFlowError(_lib.INVALID_SHAPE, "key / value must be [B, Sk, E] like query")
    cap = k_cache.shape[1]
    if tuple(k_cache.shape) != (b, cap, e) or tuple(v_cache.shape) != (b, cap, e):
        raise GhostFlowError(_lib.INVALID_SHAPE, "k_cache / v_cache must be [B, C, E]")
    kv_len = past_len + sk
    o = torch.empty_like(query) if out is None else out
    w = (torch.empty((b, num_heads, sq, kv_len), dtype=torch.float32, device=query.device)
         if want_weights else None)
    ws_ptr, ws_bytes = _workspace(workspace)
    _check(lib().gfh_mha_forward_with_cache_f32(
        query.data_ptr(), key.data_ptr(), value.data_ptr(), wq.data_ptr(), _ptr(bq), wk.data_ptr(), _ptr(bk),
        wv.data_ptr(), _ptr(bv), wo.data_ptr(), _ptr(bo), k_cache.data_ptr(), v_cache.data_ptr(), cap, past_len,
        _ptr(mask), 0 if mask is None else mask.numel(), int(bool(causal)), o.data_ptr(), _ptr(w), b, sq, sk, e,
        num_heads, ws_ptr, ws_bytes, _stream(query.device)))
    return (o, w) if want_weights else o


def mha_forward_with_cache(query, key, value, wq, bq, wk, bk, wv, bv, wo, bo, num_heads, mask=None,
                           past_key=None, past_value=None):
    """The reference's signature and results (attention.rs:100-144):
    past_key / past_value [B, P, E] are concatenated before the new keys
    along dim 1; returns (output [B, Sq, E], attn_weights
    [B, H, Sq, P + Sk], k_cache, v_cache), the last two being the new
    projected keys / values as [B, H, Sk, D] views, like
    reshape_for_attention's (:146-150)."""
    b, sq, e = query.shape
    sk = key.shape[1]
    have_past = past_key is not None and past_value is not None
    p = past_key.shape[1] if have_past else 0
    kc = torch.empty((b, p + sk, e), dtype=torch.float32, device=query.device)
    vc = torch.empty_like(kc)
    if p:
        kc[:, :p].copy_(past_key)
        vc[:, :p].copy_(past_value)
    out, w = mha_forward_cached(query, key, value, wq, bq, wk, bk, wv, bv, wo, bo, num_heads, kc, vc, p,
                                mask=mask, want_weights=True)
    d = e // num_heads
    k_new = kc[:, p:].reshape(b, sk, num_heads, d).transpose(1, 2)
    v_new = vc[:, p:].reshape(b, sk, num_heads, d).transpose(1, 2)
    return out, w, k_new, v_new


# ---- key/value cache in pages ---------------------------------------------------

def _rows(t, name, like, tokens, heads, d):
    """Elements between the tokens of t [tokens, heads, d] (heads and dims
    contiguous), of like's type and on its device."""
    if t.dtype is not like.dtype or t.get_device() != like.get_device() or not t.is_cuda:
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be {like.dtype} on {like.device} (a GPU), got {t.dtype} on "
                             f"{t.device}")
    if t.shape != (tokens, heads, d):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"{name} must be [{tokens}, {heads}, {d}], got {list(t.shape)}")
    ld, hs, ds = t.stride()
    if (ds != 1 and d > 1) or (hs != d and heads > 1):
        raise GhostFlowError(_lib.INVALID_DATA, f"{name}: the heads of a token must be contiguous")
    return ld if tokens > 1 else heads * d


def _need_f32(t, name, dev):
    if t.dtype is not torch.float32 or t.get_device() != dev.index or not t.is_contiguous():
        raise GhostFlowError(_lib.INVALID_DATA, f"{name} must be a contiguous float32 tensor on {dev}")


_PAGED_KV = struct.Struct("@PPi7qP3qPPP")  # gfh_paged_kv; packed by hand, a ctypes Structure costs 3 us more
_PAGED_SCALES = struct.Struct("@PP2q")  # gfh_paged_scales
_PAGE_DTYPES = {**_DTYPES, torch.uint8: _lib.U8}


def _paged_kv(k_pages, v_pages, page_table, q_offsets, kv_lens, status, dev):
    """(gfh_paged_kv, kv_heads, head_dim) of checked arguments."""
    shape, stride = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.stride() != stride or v_pages.dtype != k_pages.dtype:
        raise GhostFlowError(_lib.INVALID_SHAPE, "k_pages and v_pages must be [pages, page_size, kv_heads, head_dim], of "
                             "one type and with one layout")
    dt = _PAGE_DTYPES.get(k_pages.dtype)
    if dt is None:
        raise GhostFlowError(_lib.INVALID_DATA, f"k_pages must be float32, bfloat16, float16 or uint8, got {k_pages.dtype}")
    pages, page_size, hkv, d = shape
    sp, sr, sh, sd = stride
    if sd != 1 and d > 1:
        raise GhostFlowError(_lib.INVALID_DATA, "the dims of k_pages must be contiguous")
    index = dev.index  # (device numbers compare faster than devices; of a host tensor -1)
    if dev.type != "cuda" or k_pages.get_device() != index or v_pages.get_device() != index:
        raise GhostFlowError(_lib.INVALID_DATA, f"k_pages and v_pages must be on {dev}, a GPU")
    tshape, tstride = page_table.shape, page_table.stride()
    seqs = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    if len(tshape) != 2 or tshape[0] != seqs or q_offsets.shape != (seqs + 1,):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"page_table [seqs, pages], q_offsets [seqs + 1] and kv_lens [seqs], "
                             f"got {list(tshape)}, {list(q_offsets.shape)}, {list(kv_lens.shape)}")
    width = tshape[1]
    i32 = torch.int32
    if (page_table.dtype is not i32 or q_offsets.dtype is not i32 or kv_lens.dtype is not i32
            or page_table.get_device() != index or q_offsets.get_device() != index or kv_lens.get_device() != index
            or not (tstride[1] == 1 or page_table.is_contiguous()) or not q_offsets.is_contiguous()
            or not kv_lens.is_contiguous()):
        bad = next(n for t, n in ((page_table, "page_table"), (q_offsets, "q_offsets"), (kv_lens, "kv_lens"))
                   if t.dtype is not i32 or t.get_device() != index
                   or not (t.is_contiguous() or (t is page_table and tstride[1] == 1)))
        raise GhostFlowError(_lib.INVALID_DATA, f"{bad} must be a contiguous int32 tensor on {dev}")
    if status is not None and (status.dtype is not i32 or status.get_device() != index or status.numel() < 1):
        raise GhostFlowError(_lib.INVALID_DATA, f"status must be an int32 tensor on {dev}")
    # (a stride over a single element says nothing)
    kv = _PAGED_KV.pack(k_pages.data_ptr(), v_pages.data_ptr(), dt, pages, page_size, hkv, d, sp if pages > 1 else 0,
                        sr if page_size > 1 else 0, sh if hkv > 1 else 0, page_table.data_ptr(), width,
                        tstride[0] if seqs > 1 else width, seqs, kv_lens.data_ptr(), q_offsets.data_ptr(),
                        0 if status is None else status.data_ptr())
    return kv, hkv, d


def _paged_scales(k_scales, v_scales, k_pages):
    """gfh_paged_scales of the step bytes [pages, kv_heads, page_size] that go
    with pages of 8 bits, None for others."""
    codes = k_pages.dtype is torch.uint8
    if k_scales is None and v_scales is None and not codes:
        return None
    if k_scales is None or v_scales is None or not codes:
        raise GhostFlowError(_lib.INVALID_DATA, "k_scales and v_scales go with pages of uint8, and those with both")
    pages, page_size, hkv, _ = k_pages.shape
    shape, stride = k_scales.shape, k_scales.stride()
    if shape != (pages, hkv, page_size) or v_scales.shape != shape or v_scales.stride() != stride:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"k_scales and v_scales must be [{pages}, {hkv}, {page_size}] with one "
                             f"layout, got {list(shape)} and {list(v_scales.shape)}")
    if k_scales.dtype is not torch.uint8 or v_scales.dtype is not torch.uint8 or (page_size > 1 and stride[2] != 1):
        raise GhostFlowError(_lib.INVALID_DATA, "k_scales and v_scales must be uint8, the rows of a page contiguous")
    index = k_pages.get_device()
    if k_scales.get_device() != index or v_scales.get_device() != index:
        raise GhostFlowError(_lib.INVALID_DATA, f"k_scales and v_scales must be on {k_pages.device}")
    return _PAGED_SCALES.pack(k_scales.data_ptr(), v_scales.data_ptr(), stride[0] if pages > 1 else 0,
                              stride[1] if hkv > 1 else 0)


def paged_append(k_pages, v_pages, page_table, q_offsets, kv_lens, k, v, *, q=None, q_out=None, cos=None, sin=None,
                 interleaved=False, status=None, k_scales=None, v_scales=None, q_norm=None, k_norm=None, norm_eps=1e-6):
    """Writes the new tokens' k and v [tokens, kv_heads, head_dim] into their
    sequences' pages [pages, page_size, kv_heads, head_dim], k turned by the
    rotary tables cos / sin [positions, rotary_dim / 2] (fp32) at the tokens'
    positions, and returns q [tokens, heads, head_dim] turned the same way
    (into q_out, which may be q; None without q).  gfh_paged_kv in
    ghostflow_hip.h says what page_table [seqs, pages], q_offsets [seqs + 1],
    kv_lens [seqs] (the new tokens included) and status (all int32) are.

    q_norm and k_norm [head_dim] (fp32): queries and keys are first normed per
    head, x / sqrt(mean(x^2) + norm_eps) * weight.  k_scales and v_scales
    [pages, kv_heads, page_size] with pages, all uint8: rows are written in 8
    bits, with the byte of their step (gfh_paged_scales)."""
    dev = k.device
    kv, hkv, d = _paged_kv(k_pages, v_pages, page_table, q_offsets, kv_lens, status, dev)
    scales = _paged_scales(k_scales, v_scales, k_pages)
    dt = _dtype(k, "k")
    tokens = k.shape[0] if k.dim() else 0
    ldk = _rows(k, "k", k, tokens, hkv, d)
    ldv = _rows(v, "v", k, tokens, hkv, d)
    heads, ldq, ldqo, qp, qop = hkv, 0, 0, None, None
    if q is not None:
        heads = q.shape[1] if q.dim() == 3 else 0
        ldq = _rows(q, "q", k, tokens, heads, d)
        if q_out is None:
            q_out = torch.empty((tokens, heads, d), dtype=q.dtype, device=dev)
        ldqo = _rows(q_out, "q_out", k, tokens, heads, d)
        qp, qop = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise GhostFlowError(_lib.INVALID_DATA, "q_out without q")
    rows, half, cp, sp = 0, 0, None, None
    if (cos is None) != (sin is None):
        raise GhostFlowError(_lib.INVALID_DATA, "cos and sin are given together")
    if cos is not None:
        _need_f32(cos, "cos", dev)
        _need_f32(sin, "sin", dev)
        shape = cos.shape
        if len(shape) != 2 or sin.shape != shape:
            raise GhostFlowError(_lib.INVALID_SHAPE, "cos and sin must be [positions, rotary_dim / 2]")
        rows, half = shape
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if scales is None and q_norm is None and k_norm is None:
        _call(dev, lib().gfh_paged_append, kv, dt, tokens, heads, qp, ldq, qop, ldqo, k.data_ptr(), ldk, v.data_ptr(),
              ldv, cp, sp, rows, 2 * half, 1 if interleaved else 0)
        return q_out
    wq = None if q_norm is None else _norm_weights(q_norm, "q_norm", d, dev)
    wk = None if k_norm is None else _norm_weights(k_norm, "k_norm", d, dev)
    _call(dev, lib().gfh_paged_append_norm, kv, scales, dt, tokens, heads, qp, ldq, qop, ldqo, k.data_ptr(), ldk,
          v.data_ptr(), ldv, cp, sp, rows, 2 * half, 1 if interleaved else 0, wq, wk, float(norm_eps))
    return q_out


def _norm_weights(w, name, d, dev):
    _need_f32(w, name, dev)
    if w.shape != (d,):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"{name} must be [{d}], got {list(w.shape)}")
    return w.data_ptr()


def paged_read(k_pages, v_pages, page_table, q_offsets, kv_lens, *, tokens=None, dtype=torch.float32, k_out=None,
               v_out=None, status=None, k_scales=None, v_scales=None):
    """What the pages hold at the batch's new positions, as dense k and v
    [tokens, kv_heads, head_dim] (into k_out and v_out, else of dtype): the
    inverse of paged_append.  A batch with as many new tokens as positions
    reads its sequences whole.  Arguments as paged_append's; without k_out and
    v_out, tokens is the last of q_offsets where the caller does not give it
    (which waits for the device).  Rows behind the last sequence are left as
    they are, and zero in tensors made here."""
    dev = k_pages.device
    kv, hkv, d = _paged_kv(k_pages, v_pages, page_table, q_offsets, kv_lens, status, dev)
    scales = _paged_scales(k_scales, v_scales, k_pages)
    if (k_out is None) != (v_out is None):
        raise GhostFlowError(_lib.INVALID_DATA, "k_out and v_out are given together")
    if k_out is None:
        if tokens is None:
            tokens = int(q_offsets[-1])
        k_out = torch.zeros((tokens, hkv, d), dtype=dtype, device=dev)
        v_out = torch.zeros_like(k_out)
    dt = _dtype(k_out, "k_out")
    tokens = k_out.shape[0] if k_out.dim() else 0
    _same_device(dev, k_out)
    ldk = _rows(k_out, "k_out", k_out, tokens, hkv, d)
    ldv = _rows(v_out, "v_out", k_out, tokens, hkv, d)
    _call(dev, lib().gfh_paged_read, kv, scales, dt, tokens, k_out.data_ptr(), ldk, v_out.data_ptr(), ldv)
    return k_out, v_out


def paged_attention(q, k_pages, v_pages, page_table, q_offsets, kv_lens, *, scale=None, causal=True, window=0,
                    max_kv_len=None, out=None, workspace=None, status=None, k_scales=None, v_scales=None):
    """Attention of the new tokens q [tokens, heads, head_dim] over their
    sequences' pages (arguments as paged_append's): token at position p sees
    the keys j < kv_len, j <= p if causal, j > p - window if window.  Returns
    out like q (which may be q); rows behind the last sequence are left as
    they are, and zero in an out made here.  max_kv_len: the batch's longest
    length where the caller knows it.  k_scales and v_scales go with pages of
    uint8; q is then of any type."""
    dev = q.device
    kv, _, d = _paged_kv(k_pages, v_pages, page_table, q_offsets, kv_lens, status, dev)
    scales = _paged_scales(k_scales, v_scales, k_pages)
    dt = _dtype(q, "q")
    if q.dim() != 3:
        raise GhostFlowError(_lib.INVALID_SHAPE, "q must be [tokens, heads, head_dim]")
    tokens, heads = q.shape[:2]
    ldq = _rows(q, "q", q, tokens, heads, d)
    if out is None:
        out = torch.zeros((tokens, heads, d), dtype=q.dtype, device=dev)
    ldo = _rows(out, "out", q, tokens, heads, d)
    if scale is None:
        scale = _inv_sqrt(d)
    ws, ws_bytes = None, 0
    if workspace is not None:
        _same_device(dev, workspace)
        ws, ws_bytes = _workspace(workspace)
    rest = (dt, tokens, heads, q.data_ptr(), ldq, out.data_ptr(), ldo, float(scale), 1 if causal else 0, int(window),
            int(max_kv_len or 0), ws, ws_bytes)
    if scales is None:
        _call(dev, lib().gfh_paged_attention, kv, *rest)
    else:
        _call(dev, lib().gfh_paged_attention_q8, kv, scales, *rest)
    return out


def paged_attention_workspace_size(q, k_pages, v_pages, page_table, q_offsets, kv_lens, window=0,
                                   max_kv_len=None) -> int:
    """Bytes of paged_attention's workspace for these arguments."""
    kv, _, _ = _paged_kv(k_pages, v_pages, page_table, q_offsets, kv_lens, None, q.device)
    size = (lib().gfh_paged_attention_q8_workspace_size if k_pages.dtype == torch.uint8
            else lib().gfh_paged_attention_workspace_size)
    return int(size(kv, q.shape[0], q.shape[1], int(window), int(max_kv_len or 0)))


# ---- SwiGLU feed-forward block (ghostflow-nn/src/llama.rs:259-287) -------------

def silu_mul(gate, up, out=None):
    """gate.silu().mul(&up): silu(v) = v / (1 + exp(-v)) (activation.rs:117-122)."""
    _need(gate, torch.float32, "gate")
    _need(up, torch.float32, "up")
    if gate.shape != up.shape:
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch {list(gate.shape)} vs {list(up.shape)}")
    if out is None:
        out = torch.empty_like(gate)
    _need(out, torch.float32, "out")
    _check(lib().gfh_silu_mul_f32(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(),
                                  _stream(gate.device)))
    return out


def _swiglu_dims(x, w_gate, w_down):
    if x.dim() != 2:
        raise GhostFlowError(_lib.INVALID_SHAPE, "x must be [m, hidden]")
    m, hidden = x.shape
    inter = w_gate.shape[0]
    if w_gate.shape[1] != hidden or tuple(w_down.shape) != (hidden, inter):
        raise GhostFlowError(_lib.INVALID_SHAPE, f"ShapeMismatch x [{m}, {hidden}] with gate "
                             f"{list(w_gate.shape)} and down {list(w_down.shape)}")
    return m, hidden, inter


def swiglu(x, wg, bg, wu, bu, wd, bd, *, want_h=False):
    """SwiGLU::forward (llama.rs:276-286) in fp32; returns y, or (y, h) with
    h = silu(gate) * up when want_h."""
    for t, n in ((x, "x"), (wg, "wg"), (bg, "bg"), (wu, "wu"), (bu, "bu"), (wd, "wd"), (bd, "bd")):
        _need(t, torch.float32, n)
    m, hidden, inter = _swiglu_dims(x, wg, wd)
    y = torch.empty((m, hidden), dtype=torch.float32, device=x.device)
    h = torch.empty((m, inter), dtype=torch.float32, device=x.device) if want_h else None
    _check(lib().gfh_swiglu_f32(x.data_ptr(), m, hidden, inter, wg.data_ptr(), _ptr(bg), wu.data_ptr(),
                                _ptr(bu), wd.data_ptr(), _ptr(bd), y.data_ptr(), _ptr(h), None, 0,
                                _stream(x.device)))
    return (y, h) if want_h else y


def qswiglu(x, gate, up, down, *, want_h=False):
    """SwiGLU::forward with each Linear as the INT8 linear on
    DynamicQuantization's scheme (quantization.rs:251-288).  gate / up / down
    are (codes, scales, rowsums, bias-or-None) of per-channel symmetric
    weights [out, in]; x and h are quantized per tensor (asymmetric) on the
    device."""
    _need(x, torch.float32, "x")
    for name, (q, s, r, b) in (("gate", gate), ("up", up), ("down", down)):
        _need(q, torch.int8, name + " codes")
        _need(s, torch.float32, name + " scales")
        _need(r, torch.int32, name + " rowsums")
        _need(b, torch.float32, name + " bias")
    m, hidden, inter = _swiglu_dims(x, gate[0], down[0])
    y = torch.empty((m, hidden), dtype=torch.float32, device=x.device)
    h = torch.empty((m, inter), dtype=torch.float32, device=x.device) if want_h else None
    args = []
    for q, s, r, b in (gate, up, down):
        args += [q.data_ptr(), s.data_ptr(), r.data_ptr(), _ptr(b)]
    _check(lib().gfh_swiglu_i8(x.data_ptr(), m, hidden, inter, *args, y.data_ptr(), _ptr(h), None, 0,
                               _stream(x.device)))
    return (y, h) if want_h else y


# ---- state dict files (ghostflow-core/src/serialize.rs) -------------------------

class StateDict:
    """An opened GHOSTFLW / GHOSTFLQ file (gfh_state_dict_open): names,
    shapes and kinds from the mapped header; tensors copied to the device on
    request.  Use as a context manager or call close()."""

    def __init__(self, path: str):
        import ctypes as C
        h = C.c_void_p()
        _check(lib().gfh_state_dict_open(str(path).encode(), C.byref(h)))
        self._h = h
        self._keys = []
        self._info = {}
        for i in range(int(lib().gfh_state_dict_count(h))):
            name, kind, dtype, ndim, nsc = C.c_char_p(), C.c_int(), C.c_int(), C.c_int(), C.c_int64()
            _check(lib().gfh_state_dict_entry(h, i, C.byref(name), C.byref(kind), C.byref(dtype), C.byref(ndim),
                                              None, 0, C.byref(nsc)))
            dims = (C.c_int64 * max(ndim.value, 1))()
            _check(lib().gfh_state_dict_entry(h, i, None, None, None, None, dims, ndim.value, None))
            key = name.value.decode("utf-8")
            self._keys.append(key)
            self._info[key] = (i, kind.value, dtype.value, tuple(dims[d] for d in range(ndim.value)), nsc.value)

    def close(self):
        if self._h:
            lib().gfh_state_dict_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def keys(self):
        return list(self._keys)

    def __contains__(self, key):
        return key in self._info

    def info(self, key):
        """(kind, dtype byte or scheme, shape, nscales)."""
        return self._info[key][1:]

    def tensor(self, key, device="cuda"):
        """A kind-0 entry as a float32 device tensor of its stored shape, or a
        kind-1 entry as (codes int8, scales f32, zero points int8)."""
        idx, kind, _dtype, shape, nsc = self._info[key]
        if kind == 0:
            out = torch.empty(shape, dtype=torch.float32, device=device)
            _check(lib().gfh_state_dict_read_f32(self._h, idx, out.data_ptr(), _stream(out.device)))
            return out
        codes = torch.empty(shape, dtype=torch.int8, device=device)
        scales = torch.empty(nsc, dtype=torch.float32, device=device)
        zps = torch.empty(nsc, dtype=torch.int8, device=device)
        _check(lib().gfh_state_dict_read_q8(self._h, idx, codes.data_ptr(), scales.data_ptr(), zps.data_ptr(),
                                            _stream(codes.device)))
        return codes, scales, zps


def load_state_dict(path, device="cuda"):
    """load_state_dict (serialize.rs:48-88) straight into device memory:
    name -> float32 tensor (GHOSTFLW), or name -> (codes, scales, zero
    points) for the quantized entries of a GHOSTFLQ file."""
    with StateDict(path) as sd:
        return {k: sd.tensor(k, device) for k in sd.keys()}


def save_state_dict(path, state, *, quantized_format=False, dtypes=None):
    """save_state_dict (serialize.rs:20-45) from device tensors, in the
    dict's order.  Values are float32 device tensors, or -- in a GHOSTFLQ
    file -- (codes, scales, zero points) tuples of a QuantizedTensor.
    dtypes optionally maps a name to the dtype byte (or scheme) recorded."""
    import ctypes as C
    entries = (_lib.TensorEntry * max(len(state), 1))()
    keep = []
    dev = None
    for i, (name, v) in enumerate(state.items()):
        e = entries[i]
        nb = str(name).encode("utf-8")
        keep.append(nb)
        e.name = nb
        quant = isinstance(v, (tuple, list))
        t = v[0] if quant else v
        if quant and not quantized_format:
            raise GhostFlowError(_lib.INVALID_DATA, f"{name}: quantized entries need quantized_format=True")
        _need(t, torch.int8 if quant else torch.float32, str(name))
        dev = t.device
        dims = (C.c_int64 * max(t.dim(), 1))(*t.shape)
        keep.append(dims)
        e.kind = 1 if quant else 0
        e.dtype = (dtypes or {}).get(name, 0 if quant else 2)
        e.ndim = t.dim()
        e.dims = C.cast(dims, C.POINTER(C.c_int64))
        e.data = t.data_ptr()
        if quant:
            _need(v[1], torch.float32, f"{name} scales")
            _need(v[2], torch.int8, f"{name} zero points")
            e.scales = v[1].data_ptr()
            e.zero_points = v[2].data_ptr()
            e.nscales = v[1].numel()
    _check(lib().gfh_state_dict_save(str(path).encode(), int(bool(quantized_format)), C.addressof(entries),
                                     len(state), _stream(dev) if dev is not None else None))
