"""Operators of the model's own forward and backward pass, as autograd functions over the C ABI: layer norm, causal
attention over sequences of different lengths, and the loss of distilling from a teacher's highest logits.

They are what runs between the hooked Linear modules of a collection step (the reference leaves it to the library:
bergson/collector/collector.py:926-985).  `fused_model_ops(model)` puts the first two into a transformers model;
`IndexConfig.fused_model_ops` does so for a collection run and `IndexConfig.loss_fn = "topk_kl"` makes the third the
run's loss.  Everything is enqueued on torch's current stream of the tensors' device, allocates through torch
(so that graph captures own their memory), and can be captured; gradients are not differentiable again.
"""
from __future__ import annotations

import ctypes as C
import math
import threading
from contextlib import contextmanager, nullcontext

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import AttentionRows, AttentionShape
from .ops import _need_gpu, _ptr, dtype_code

MAX_NORM_WIDTH = 16384    # elements of a row the layer norm kernels hold
MAX_HEAD_DIM = 128
MAX_TEACHER_ENTRIES = 1024


def _on(device: torch.device):
    """The device's context when it is not the current one already."""
    return nullcontext() if device.index in (None, torch.cuda.current_device()) else torch.cuda.device(device)


def _stream_of(device: torch.device) -> C.c_void_p:
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _same_device(ref: Tensor, **others: Tensor | None) -> None:
    for name, t in others.items():
        if t is not None and t.device != ref.device:
            raise ValueError(f"{name} lives on {t.device}, the input on {ref.device}")


# ---- layer norm ---------------------------------------------------------------------------------------------------

def _norm_rows(x: Tensor, d: int) -> Tensor:
    """[rows, d] with rows at least d elements apart and contiguous elements, copied only where x is not that."""
    rows = x.reshape(-1, d)
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < d):
        rows = rows.contiguous()
    return rows


def _row_stride(rows: Tensor) -> int:
    return max(rows.stride(0), rows.shape[1])


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, bias: Tensor | None, eps: float) -> Tensor:
        lib = _lib.load()
        d = x.shape[-1]
        rows = _norm_rows(x, d)
        weight = weight.contiguous()
        if bias is not None:
            bias = bias.contiguous()
        keep = any(ctx.needs_input_grad)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((2, rows.shape[0]), dtype=torch.float32, device=x.device) if keep else None
        with _on(x.device):
            rc = lib.bgx_layernorm_forward(
                _ptr(rows), _row_stride(rows), _ptr(weight), _ptr(bias), dtype_code(weight.dtype), rows.shape[0], d,
                dtype_code(x.dtype), eps, _ptr(y), d, None if stats is None else _ptr(stats[0]),
                None if stats is None else _ptr(stats[1]), _stream_of(x.device))
        _lib.check(rc, "bgx_layernorm_forward")
        if keep:
            ctx.save_for_backward(rows, weight, stats)
            ctx.shape = x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        lib = _lib.load()
        rows, weight, stats = ctx.saved_tensors
        n, d = rows.shape
        grad = _norm_rows(dy, d)
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        dx = torch.empty(ctx.shape, dtype=rows.dtype, device=rows.device) if want_x else None
        dw = torch.empty((d,), dtype=weight.dtype, device=rows.device) if want_w else None
        db = torch.empty((d,), dtype=weight.dtype, device=rows.device) if want_b else None
        ws = None
        if want_w or want_b:
            nbytes = lib.bgx_layernorm_backward_workspace_bytes(n, d)
            ws = torch.empty((nbytes,), dtype=torch.uint8, device=rows.device)
        with _on(rows.device):
            rc = lib.bgx_layernorm_backward(
                _ptr(grad), _row_stride(grad), _ptr(rows), _row_stride(rows), _ptr(weight), dtype_code(weight.dtype),
                _ptr(stats[0]), _ptr(stats[1]), n, d, dtype_code(rows.dtype), _ptr(dx), d, _ptr(dw), _ptr(db), _ptr(ws),
                0 if ws is None else ws.numel(), _stream_of(rows.device))
        _lib.check(rc, "bgx_layernorm_backward")
        return dx, dw, db, None


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (at most 16384 elements).

    x float32, float16 or bfloat16, any strides (an x whose rows are not contiguous is copied); weight and bias [d]
    in x's dtype or both in float32.  Statistics and the weight's and bias' gradients are summed in fp32, the
    latter in a fixed order."""
    dtype_code(x.dtype)
    d = x.shape[-1] if x.dim() else 0
    if d < 1 or d > MAX_NORM_WIDTH:
        raise ValueError(f"layer_norm takes rows of 1 to {MAX_NORM_WIDTH} elements, got {tuple(x.shape)}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            if name == "weight":
                raise ValueError("layer_norm needs a weight")
            continue
        if tuple(t.shape) != (d,):
            raise ValueError(f"{name} {tuple(t.shape)} does not match rows of {d} elements")
        if t.dtype not in (x.dtype, torch.float32) or t.dtype != weight.dtype:
            raise TypeError(f"{name} is {t.dtype}; weight and bias share x's dtype ({x.dtype}) or float32")
    if not eps >= 0.0 or eps == math.inf:
        raise ValueError(f"eps={eps} must be finite and not negative")
    _need_gpu(x, "x")
    _same_device(x, weight=weight, bias=bias)
    return _LayerNorm.apply(x, weight, bias, float(eps))


# ---- causal attention ---------------------------------------------------------------------------------------------

def _operand(t: Tensor) -> Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows_of(t: Tensor) -> AttentionRows:
    if t.dim() == 4:
        return AttentionRows(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))
    return AttentionRows(t.data_ptr(), 0, t.stride(0), t.stride(1))


def _gradient_like(t: Tensor) -> Tensor:
    """A gradient's buffer in the layout of its input, where that has every element once."""
    g = torch.empty_like(t)
    return g if g.stride(-1) == 1 or g.shape[-1] == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _attention_shape(q: Tensor, k: Tensor, plan: Tensor | None, lengths: Tensor | None, n_seqs: int, scale: float
                     ) -> AttentionShape:
    rows = q.shape[0] * q.shape[1] if q.dim() == 4 else q.shape[0]
    return AttentionShape(None if plan is None else plan.data_ptr(), None if lengths is None else lengths.data_ptr(),
                          rows, n_seqs, q.shape[-2], k.shape[-2], q.shape[-1], dtype_code(q.dtype), scale)


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Tensor, v: Tensor, cu_seqlens: Tensor | None, lengths: Tensor | None, scale: float
                ) -> Tensor:
        lib = _lib.load()
        q, k, v = _operand(q), _operand(k), _operand(v)
        device, keep = q.device, any(ctx.needs_input_grad)
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
        if q.numel() == 0:
            ctx.empty = True
            ctx.save_for_backward(q, k, v)
            return out
        ctx.empty = False
        with _on(device):
            stream = _stream_of(device)
            plan = None
            n_seqs = q.shape[0]
            if q.dim() == 3:
                n_seqs = cu_seqlens.shape[0] - 1
                nbytes = lib.bgx_attention_plan_bytes(q.shape[0], n_seqs)
                plan = torch.empty((nbytes,), dtype=torch.uint8, device=device)
                _lib.check(lib.bgx_attention_plan(_ptr(cu_seqlens), n_seqs, q.shape[0], _ptr(plan), nbytes, stream),
                           "bgx_attention_plan")
            shape = _attention_shape(q, k, plan, lengths, n_seqs, scale)
            lse = torch.empty((shape.heads, shape.rows), dtype=torch.float32, device=device) if keep else None
            rc = lib.bgx_attention_forward(C.byref(shape), C.byref(_rows_of(q)), C.byref(_rows_of(k)),
                                           C.byref(_rows_of(v)), C.byref(_rows_of(out)), _ptr(lse), stream)
        _lib.check(rc, "bgx_attention_forward")
        if keep:
            ctx.save_for_backward(q, k, v, out, lse, plan, lengths)
            ctx.n_seqs, ctx.scale = n_seqs, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        if ctx.empty:
            return *(torch.zeros_like(t) for t in ctx.saved_tensors), None, None, None
        lib = _lib.load()
        q, k, v, out, lse, plan, lengths = ctx.saved_tensors
        grad = _operand(grad)
        shape = _attention_shape(q, k, plan, lengths, ctx.n_seqs, ctx.scale)
        dq, dk, dv = _gradient_like(q), _gradient_like(k), _gradient_like(v)
        nbytes = lib.bgx_attention_backward_workspace_bytes(C.byref(shape))
        ws = torch.empty((nbytes,), dtype=torch.uint8, device=q.device)
        with _on(q.device):
            rc = lib.bgx_attention_backward(
                C.byref(shape), C.byref(_rows_of(q)), C.byref(_rows_of(k)), C.byref(_rows_of(v)),
                C.byref(_rows_of(out)), _ptr(lse), C.byref(_rows_of(grad)), C.byref(_rows_of(dq)),
                C.byref(_rows_of(dk)), C.byref(_rows_of(dv)), _ptr(ws), nbytes, _stream_of(q.device))
        _lib.check(rc, "bgx_attention_backward")
        return dq, dk, dv, None, None, None


def _index_vector(t: Tensor, name: str, size: int | None, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or (size is not None and t.numel() != size):
        raise ValueError(f"{name} must be a contiguous int32 vector"
                         + ("" if size is None else f" of {size} elements")
                         + f", got {str(t.dtype).removeprefix('torch.')} {tuple(t.shape)}")
    _need_gpu(t, name)
    if t.device != device:
        raise ValueError(f"{name} lives on {t.device}, the queries on {device}")


def causal_attention(q: Tensor, k: Tensor, v: Tensor, *, cu_seqlens: Tensor | None = None,
                     lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """softmax(scale q k^T + causal mask) v within every sequence, in the layout of q.

    Batch layout: q [N, S, H, D], k and v [N, S, Hk, D]; `lengths` int32 [N] (on the GPU) cuts sequence n to its first
    lengths[n] positions.  Packed: q [T, H, D], k and v [T, Hk, D]; sequence n is rows cu_seqlens[n] up to
    cu_seqlens[n + 1] (`cu_seqlens` int32 [N + 1] on the GPU, ascending; its values are not read back).
    H is a multiple of Hk and query head h uses key/value head h // (H // Hk).  D from 1 to 128, one dtype of float32,
    float16, bfloat16; any strides (only a non-contiguous last dimension is copied).  scale (default D ** -0.5) must
    be positive.  Positions and rows that belong to no sequence are not read: their output and gradients are 0."""
    dtype_code(q.dtype)
    if q.dim() not in (3, 4) or k.dim() != q.dim() or v.dim() != q.dim():
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} must all be [N, S, heads, D] or "
                         "all [T, heads, D]")
    if k.shape != v.shape or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v share one dtype; got {q.dtype}, {k.dtype}, {v.dtype}")
    heads, kv_heads, dim = q.shape[-2], k.shape[-2], q.shape[-1]
    if kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} query heads on {kv_heads} key/value heads")
    if not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head dimension {dim}; supported are 1 to {MAX_HEAD_DIM}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale={scale} must be positive and finite")
    if q.dim() == 3:
        if cu_seqlens is None or lengths is not None:
            raise ValueError("packed sequences come with cu_seqlens (and without lengths)")
    elif cu_seqlens is not None:
        raise ValueError("cu_seqlens go with packed [T, heads, D] inputs; a batch [N, S, heads, D] takes lengths")
    _need_gpu(q, "q")
    _same_device(q, k=k, v=v)
    if cu_seqlens is not None:
        _index_vector(cu_seqlens, "cu_seqlens", None, q.device)
        if cu_seqlens.numel() < 1:
            raise ValueError("cu_seqlens needs at least one element")
    if lengths is not None:
        _index_vector(lengths, "lengths", q.shape[0], q.device)
    return _CausalAttention.apply(q, k, v, cu_seqlens, lengths, scale)


# ---- distillation -------------------------------------------------------------------------------------------------

class _TopkDistillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, ids: Tensor, teacher: Tensor, valid: Tensor | None, temperature: float) -> Tensor:
        lib = _lib.load()
        V, K = logits.shape[-1], ids.shape[-1]
        rows = _norm_rows(logits, V)
        ids, teacher = ids.reshape(-1, K).contiguous(), teacher.reshape(-1, K).contiguous()
        if valid is not None:
            valid = valid.reshape(-1).contiguous()
        keep = ctx.needs_input_grad[0]
        losses = torch.empty(logits.shape[:-1], dtype=torch.float32, device=logits.device)
        stats = torch.empty((rows.shape[0], 2), dtype=torch.float32, device=logits.device) if keep else None
        with _on(logits.device):
            rc = lib.bgx_distill_forward(
                _ptr(rows), _row_stride(rows), rows.shape[0], V, dtype_code(rows.dtype), _ptr(ids), _ptr(teacher),
                dtype_code(teacher.dtype), K, _ptr(valid), temperature, _ptr(losses), _ptr(stats),
                _stream_of(logits.device))
        _lib.check(rc, "bgx_distill_forward")
        if keep:
            ctx.save_for_backward(rows, ids, teacher, stats)
            ctx.temperature, ctx.shape = temperature, logits.shape
        return losses

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        lib = _lib.load()
        rows, ids, teacher, stats = ctx.saved_tensors
        V = rows.shape[1]
        grad = grad.reshape(-1).contiguous()
        dlogits = torch.empty(ctx.shape, dtype=rows.dtype, device=rows.device)
        with _on(rows.device):
            rc = lib.bgx_distill_backward(
                _ptr(rows), _row_stride(rows), rows.shape[0], V, dtype_code(rows.dtype), _ptr(ids), _ptr(teacher),
                dtype_code(teacher.dtype), ids.shape[1], ctx.temperature, _ptr(stats), _ptr(grad), _ptr(dlogits), V,
                _stream_of(rows.device))
        _lib.check(rc, "bgx_distill_backward")
        return dlogits, None, None, None, None


def topk_distillation(logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, *, temperature: float = 1.0,
                      valid: Tensor | None = None) -> Tensor:
    """Per-token loss of a student's logits against a teacher's K highest ones, float32 [...].

    With p = softmax(teacher_logits / temperature) over the K entries and q = softmax(logits / temperature) over the
    whole vocabulary: temperature^2 * sum_k p_k (log p_k - log q[teacher_ids_k]).
    logits [..., V] float32, float16 or bfloat16; teacher_ids [..., K] int64 and teacher_logits [..., K] of any of those
    dtypes, K up to 1024.  An id outside 0..V-1 (by convention -1) is no entry, an id may come more than once (its
    probabilities add up).  Tokens without an entry, and those `valid` (bool [...]) excludes, have loss 0 and gradient
    0 whatever their logits hold.  The teacher's logits are constants."""
    dtype_code(logits.dtype)
    dtype_code(teacher_logits.dtype)
    if logits.dim() < 1 or teacher_ids.dim() != logits.dim() or logits.shape[-1] < 1:
        raise ValueError(f"logits {tuple(logits.shape)} and teacher_ids {tuple(teacher_ids.shape)} must be [..., V] and "
                         "[..., K]")
    if teacher_ids.shape != teacher_logits.shape or teacher_ids.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"teacher_ids {tuple(teacher_ids.shape)} and teacher_logits {tuple(teacher_logits.shape)} do not "
                         f"match logits {tuple(logits.shape)}")
    if not 1 <= teacher_ids.shape[-1] <= MAX_TEACHER_ENTRIES:
        raise ValueError(f"{teacher_ids.shape[-1]} teacher entries per token; supported are 1 to {MAX_TEACHER_ENTRIES}")
    if teacher_ids.dtype != torch.int64:
        raise TypeError(f"teacher_ids must be int64, got {teacher_ids.dtype}")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("teacher_logits are constants of the loss: detach them")
    if not 0.0 < temperature < math.inf:
        raise ValueError(f"temperature={temperature} must be positive and finite")
    if valid is not None and (valid.dtype != torch.bool or valid.shape != logits.shape[:-1]):
        raise ValueError(f"valid must be bool {tuple(logits.shape[:-1])}, got {valid.dtype} {tuple(valid.shape)}")
    _need_gpu(logits, "logits")
    _same_device(logits, teacher_ids=teacher_ids, teacher_logits=teacher_logits, valid=valid)
    return _TopkDistillation.apply(logits, teacher_ids, teacher_logits, valid, float(temperature))
