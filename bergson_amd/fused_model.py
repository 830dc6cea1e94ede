"""A transformers model's layer norms and causal attention on this package's kernels.

`with fused_model_ops(model):` replaces, for the calls inside, the forward of every affine `nn.LayerNorm` and the
model's attention implementation (through transformers' public registries); what was there comes back at the end.
`IndexConfig.fused_model_ops` does this around a collection run.  The hooked Linear modules are not touched: a collector
sees the same modules with inputs and output gradients that differ by rounding.

Right-padded batches need no attention mask here: attention is causal, and with `sequence_lengths(lengths)` around a
forward pass the padding is not computed at all (its attention output is 0).  A mask that says anything else than
"causal" is refused, and so is an attention that takes anything beside queries, keys and values (sparse selections,
biases on the scores, sinks, windows).
"""
from __future__ import annotations

import functools
import threading
import warnings
from contextlib import contextmanager

import torch
import torch.nn as nn
from torch import Tensor

from .model_ops import causal_attention, layer_norm

IMPLEMENTATION = "bergson_amd"
# Keywords transformers hands through to attention that change none of its values: positions (the embeddings are in q and
# k by then, and packed positions are refused with their mask) and what a model is asked to return or count.
_WITHOUT_EFFECT = {"position_ids", "cache_position", "use_cache", "output_hidden_states", "output_router_logits",
                   "return_dict", "logits_to_keep", "num_items_in_batch"}
_current = threading.local()


@contextmanager
def sequence_lengths(lengths: Tensor | None):
    """Document lengths (int32 [N] on the GPU) of the right-padded batch whose forward pass runs inside: fused
    attention then skips the padding.  Per thread; None changes nothing.

    Not with activation checkpointing: a checkpointed block runs again on the backward pass' threads, outside this
    context, and torch refuses what it then saves (CheckpointError).  Without the lengths it is right, too: attention is
    causal, the padding only costs its time."""
    before = getattr(_current, "lengths", None)
    _current.lengths = lengths
    try:
        yield
    finally:
        _current.lengths = before


def _mask(*args, attention_mask=None, mask_function=None, q_length=None, kv_length=None, **kwargs):
    """What transformers asks a mask of: nothing is built, and nothing but a plain causal mask is accepted."""
    from transformers.masking_utils import causal_mask_function

    if attention_mask is not None:
        raise ValueError("fused attention takes no attention_mask: leave it out for right-padded batches (labels of -100 "
                         "on the padding) and give the documents' lengths with sequence_lengths(...)")
    if mask_function is not None and mask_function is not causal_mask_function:
        raise ValueError("fused attention is causal over whole sequences; this model asks for another mask "
                         "(sliding window, packed positions, bidirectional)")
    if q_length is not None and kv_length is not None and int(q_length) != int(kv_length):
        raise ValueError(f"fused attention has no key/value cache: {int(q_length)} queries against {int(kv_length)} keys")
    return None


def _attention(module: nn.Module, query: Tensor, key: Tensor, value: Tensor, attention_mask: Tensor | None,
               scaling: float | None = None, dropout: float = 0.0, **kwargs):
    """transformers' attention interface: [N, heads, S, D] in, [N, S, heads, D] out, no weights.  A keyword that is not
    known to leave the values alone is refused."""
    if attention_mask is not None:
        raise ValueError("fused attention takes no attention mask")
    if dropout:
        raise ValueError(f"fused attention has no dropout (got {dropout})")
    causal = kwargs.pop("is_causal", None)
    if (getattr(module, "is_causal", True) if causal is None else causal) is False:
        raise ValueError("fused attention is causal")
    if kwargs.pop("output_attentions", None):
        raise ValueError("fused attention has no weights to return (output_attentions)")
    # a window, sinks, a selection of keys, a bias on the scores ...: dropped, any of them would be a wrong result
    for name, given in kwargs.items():
        if given is not None and name not in _WITHOUT_EFFECT:
            raise ValueError(f"fused attention does not know {name}=" + (f"a tensor {tuple(given.shape)}" if
                             isinstance(given, Tensor) else repr(given)) + ": this model's attention is another one")
    if query.shape[2] != key.shape[2]:
        raise ValueError(f"fused attention has no key/value cache: {query.shape[2]} queries against {key.shape[2]} keys")
    lengths = getattr(_current, "lengths", None)
    if lengths is not None and lengths.shape[0] != query.shape[0]:
        raise ValueError(f"sequence_lengths of {lengths.shape[0]} documents around a batch of {query.shape[0]}")
    out = causal_attention(query.transpose(1, 2), key.transpose(1, 2), value.transpose(1, 2), lengths=lengths,
                           scale=scaling)
    return out, None


def _norm_forward(module: nn.LayerNorm, x: Tensor) -> Tensor:
    return layer_norm(x, module.weight, module.bias, module.eps)


def _fusable(module: nn.Module) -> bool:
    return (isinstance(module, nn.LayerNorm) and type(module).forward is nn.LayerNorm.forward
            and "forward" not in vars(module) and module.weight is not None and len(module.normalized_shape) == 1)


def _register() -> None:
    from transformers import AttentionInterface, AttentionMaskInterface

    AttentionInterface.register(IMPLEMENTATION, _attention)
    AttentionMaskInterface.register(IMPLEMENTATION, _mask)


def _attention_settings(model: nn.Module) -> list[tuple[object, str | None]]:
    """(configuration, attention implementation) of the model and of every part that has its own, outer ones first."""
    configs = {id(c): c for c in (getattr(m, "config", None) for m in model.modules()) if hasattr(c, "_attn_implementation")}
    return [(c, c._attn_implementation) for c in configs.values()]


def _name_what_is_left(model: nn.Module) -> None:
    """transformers leaves alone what does not go through its registry."""
    left = {id(c) for c, implementation in _attention_settings(model) if implementation not in (IMPLEMENTATION, None)}
    names = []
    for m in model.modules():
        config = getattr(m, "config", None)
        if id(config) in left:
            left.discard(id(config))
            names.append(type(m).__name__)
    if names:
        warnings.warn(f"{', '.join(names)} keeps its own attention: it cannot be replaced through transformers' registry, "
                      "only layer norms run on this package's kernels there", stacklevel=4)


@contextmanager
def fused_model_ops(model: nn.Module):
    """Layer norms and causal attention of `model` through `layer_norm` and `causal_attention` within the context.

    Attention is replaced in transformers models (`set_attn_implementation`; a warning names a model that does not take
    it); any other module keeps its own and only its layer norms change.  Not for two threads at once on one model."""
    norms = [m for m in model.modules() if _fusable(m)]
    swap = callable(getattr(model, "set_attn_implementation", None))
    # parts of a composite model have configurations of their own, which the outer one's setting overwrites
    before = _attention_settings(model) if swap else []
    try:
        for m in norms:
            m.forward = functools.partial(_norm_forward, m)
        if swap:
            _register()
            model.set_attn_implementation(IMPLEMENTATION)
            _name_what_is_left(model)
        yield model
    finally:
        for m in norms:
            vars(m).pop("forward", None)
        if swap:
            if before and before[0][1] is not None:
                model.set_attn_implementation(before[0][1])
            for config, implementation in before:
                config._attn_implementation = implementation
