"""Operators of the model's own forward and backward pass: layer norm, causal attention over sequences of different
lengths, and the loss of distilling from a teacher's highest logits.

They are what runs between the hooked Linear modules of a collection step (the reference leaves it to the library:
bergson/collector/collector.py:926-985).  The arithmetic is the library's (include/bergson_amd.h); argument checks,
allocation and the autograd nodes are native too (csrc/torch_ops.cpp).  Everything is enqueued on torch's current
stream of the tensors' device, allocates through torch only (so that a graph capture owns its memory), keeps nothing
between calls and can be captured (a backward pass as torch has it: into leaves that no graph built before the
capture still holds); gradients are not differentiable again, and inputs with forward-mode tangents are refused.
"""
from __future__ import annotations

from torch import Tensor

_module = None


def _native():
    """The native module; it is linked against libbergson_amd.so, so that is loaded (and checked) first."""
    global _module
    if _module is None:
        from . import _lib

        _lib.load()
        try:
            from . import _model_ops
        except ImportError as e:
            raise ImportError(f"the native module of the model operators cannot be loaded ({e}): build the extension with "
                              "`python -m bergson_amd.build_ext` (there is no fallback)") from e
        _module = _model_ops
    return _module


def layer_norm(x: Tensor, weight: Tensor, bias: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (at most 16384 elements).

    x float32, float16 or bfloat16, any strides (an x whose rows are not contiguous is copied); weight and bias [d]
    in x's dtype or both in float32.  Statistics and the weight's and bias' gradients are summed in fp32, the
    latter in a fixed order."""
    return (_module or _native()).layer_norm(x, weight, bias, eps)


def causal_attention(q: Tensor, k: Tensor, v: Tensor, *, cu_seqlens: Tensor | None = None,
                     lengths: Tensor | None = None, scale: float | None = None) -> Tensor:
    """softmax(scale q k^T + causal mask) v within every sequence, as a contiguous tensor of q's shape.

    Batch layout: q [N, S, H, D], k and v [N, S, Hk, D]; `lengths` int32 [N] (on the GPU) cuts sequence n to its first
    lengths[n] positions.  Packed: q [T, H, D], k and v [T, Hk, D]; sequence n is rows cu_seqlens[n] up to
    cu_seqlens[n + 1] (`cu_seqlens` int32 [N + 1] on the GPU, ascending; its values are not read back).
    H is a multiple of Hk and query head h uses key/value head h // (H // Hk).  D from 1 to 128, one dtype of float32,
    float16, bfloat16; any strides (only a non-contiguous last dimension is copied).  scale (default D ** -0.5) must
    be positive.  Positions and rows that belong to no sequence are not read: their output and gradients are 0.

    Scores, softmax statistics and sums are fp32.  With 16-bit inputs the probabilities, and in the backward pass their
    gradients, are operands rounded to that type -- for sequences of up to 64 positions with a second operand for what the
    rounding cut off.  The output is the same with and without a gradient recorded."""
    return (_module or _native()).causal_attention(q, k, v, cu_seqlens, lengths, scale)


def topk_distillation(logits: Tensor, teacher_ids: Tensor, teacher_logits: Tensor, *, temperature: float = 1.0,
                      valid: Tensor | None = None) -> Tensor:
    """Per-token loss of a student's logits against a teacher's K highest ones, float32 [...].

    With p = softmax(teacher_logits / temperature) over the K entries and q = softmax(logits / temperature) over the
    whole vocabulary: temperature^2 * sum_k p_k (log p_k - log q[teacher_ids_k]).
    logits [..., V] float32, float16 or bfloat16; teacher_ids [..., K] int64 and teacher_logits [..., K] of any of those
    dtypes, K up to 1024.  An id outside 0..V-1 (by convention -1) is no entry, an id may come more than once (its
    probabilities add up).  Tokens without an entry, and those `valid` (bool [...]) excludes, have loss 0 and gradient
    0 whatever their logits hold.  The teacher's logits are constants."""
    return (_module or _native()).topk_distillation(logits, teacher_ids, teacher_logits, temperature, valid)
