"""Fused model operators around a model: what is replaced and put back, what is refused, and the teacher's columns."""
import warnings

import pytest
import torch
import torch.nn as nn

import bergson_amd as B
from bergson_amd import fused_model
from bergson_amd.collector import forward_loss_factory
from bergson_amd.data import pad_teacher
from bergson_amd.synthetic import make_gpt_neox, make_llama


def test_replaced_and_put_back():
    model = make_gpt_neox("pythia-14m", torch.float32, "cpu", layers=2)
    x = torch.randint(0, 100, (2, 9))
    want, before = model(x).logits, model.config._attn_implementation
    with B.fused_model_ops(model):
        assert model.config._attn_implementation == "bergson_amd"
        with pytest.raises(RuntimeError, match="no CPU path"):   # the kernels are reached, not the library
            model(x)
    assert model.config._attn_implementation == before
    assert not any("forward" in vars(m) for m in model.modules())
    assert torch.equal(model(x).logits, want)
    with pytest.raises(KeyError):
        with B.fused_model_ops(model):
            raise KeyError("inside")
    assert model.config._attn_implementation == before and torch.equal(model(x).logits, want)


def test_norms_of_other_modules():
    class Shifted(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x) + 1

    m = nn.Sequential(nn.LayerNorm(8), Shifted(8), nn.LayerNorm((2, 8)), nn.LayerNorm(8, elementwise_affine=False))
    with B.fused_model_ops(m):
        assert ["forward" in vars(l) for l in m] == [True, False, False, False]
    assert not any("forward" in vars(l) for l in m)


def test_masks_and_options_are_refused():
    model = make_llama(torch.float32, "cpu", layers=1, d=32, heads=4, kv_heads=2, mlp=64, vocab=50)
    x = torch.randint(0, 50, (2, 6))
    with B.fused_model_ops(model):
        with pytest.raises(ValueError, match="attention_mask"):
            model(x, attention_mask=torch.ones_like(x))
        with pytest.raises(ValueError, match="another mask|no key/value cache"):
            model(x, position_ids=torch.tensor([[0, 1, 2, 0, 1, 2]]))    # packed documents by position
    q = torch.zeros(2, 4, 5, 16)
    mod = nn.Module()
    with pytest.raises(ValueError, match="dropout"):
        fused_model._attention(mod, q, q, q, None, dropout=0.1)
    with pytest.raises(ValueError, match="sliding_window"):
        fused_model._attention(mod, q, q, q, None, sliding_window=4)
    with pytest.raises(ValueError, match="cache"):
        fused_model._attention(mod, q[:, :, :1], q, q, None)
    with pytest.raises(ValueError, match="causal"):
        fused_model._attention(mod, q, q, q, None, is_causal=False)
    with pytest.raises(ValueError, match="attention mask"):
        fused_model._attention(mod, q, q, q, torch.zeros(1))
    with B.sequence_lengths(torch.ones(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="3 documents"):
            fused_model._attention(mod, q, q, q, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fused_model._attention(mod, q, q, q, None)     # the lengths are gone with their context


def test_pad_teacher():
    batch = {"input_ids": [[1, 2, 3], [4]], "teacher_ids": [[[5, 6], [7]], [[8, 9]]],
             "teacher_logits": [[[0.5, 0.25], [2.0]], [[1.0, -1.0]]]}
    ids, logits = pad_teacher(batch, 4)
    assert ids.tolist() == [[[5, 6], [7, -1], [-1, -1], [-1, -1]], [[8, 9], [-1, -1], [-1, -1], [-1, -1]]]
    assert logits[0, :2].tolist() == [[0.5, 0.25], [2.0, 0.0]] and ids.dtype == torch.int64
    with pytest.raises(ValueError, match="teacher_logits"):
        pad_teacher({"input_ids": [[1]], "teacher_ids": [[[1]]]}, 1)
    with pytest.raises(ValueError, match="3 tokens|1 teacher_logits"):
        pad_teacher({**batch, "teacher_logits": [[[0.5, 0.25]], [[1.0, -1.0]]]}, 4)
    with pytest.raises(ValueError, match="position 1"):
        pad_teacher({**batch, "teacher_logits": [[[0.5, 0.25], [2.0, 1.0]], [[1.0, -1.0]]]}, 4)
    ids, _ = pad_teacher({"input_ids": [[1]], "teacher_ids": [[]], "teacher_logits": [[]]}, 2)
    assert ids.tolist() == [[[-1], [-1]]]


def test_loss_settings():
    with pytest.raises(NotImplementedError, match="PEFT"):
        forward_loss_factory(B.IndexConfig(loss_fn="kl"))
    with pytest.raises(ValueError, match="label_smoothing"):
        forward_loss_factory(B.IndexConfig(loss_fn="topk_kl", label_smoothing=0.1))
    assert B.IndexConfig().fused_model_ops is False and B.IndexConfig().loss_fn == "ce"


def test_keywords_of_other_attentions_are_refused():
    """What changes an attention's values and is not known here is refused; what does not is let through (the kernels'
    own refusal of CPU tensors comes behind)."""
    q = torch.zeros(2, 4, 5, 16)
    mod = nn.Module()
    for name, value in (("indices", torch.zeros(2, 5, 3)), ("block_indices", torch.zeros(2, 1, 5, 1)),
                        ("position_bias", torch.zeros(1, 4, 5, 5)), ("sliding_window", 4), ("softcap", 30.0),
                        ("s_aux", torch.zeros(4)), ("cu_seq_lens_q", torch.zeros(3)), ("head_mask", torch.ones(4)),
                        ("an_option_of_tomorrow", False), ("output_attentions", True)):
        with pytest.raises(ValueError, match=name):
            fused_model._attention(mod, q, q, q, None, **{name: value})
    with pytest.raises(RuntimeError, match="no CPU path"):
        fused_model._attention(mod, q, q, q, None, position_ids=torch.zeros(2, 5), use_cache=True, sliding_window=None,
                               output_attentions=False, output_router_logits=True, is_causal=None)


def test_causality_the_module_decides():
    """is_causal=None leaves it to the module, like a call without it."""
    q = torch.zeros(2, 4, 5, 16)
    mod = nn.Module()
    mod.is_causal = False
    for kw in ({}, {"is_causal": None}):
        with pytest.raises(ValueError, match="causal"):
            fused_model._attention(mod, q, q, q, None, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fused_model._attention(mod, q, q, q, None, is_causal=True)


def test_keywords_through_a_model_are_refused(monkeypatch):
    """What a model's call, or its layers, hand down to the attention function by keyword (here a choice of keys):
    refused, where it was dropped and every key attended to."""
    import torch.nn.functional as F

    def attention(q, k, v, lengths=None, scale=None):
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        return F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=scale, enable_gqa=True).transpose(1, 2)

    monkeypatch.setattr(fused_model, "causal_attention", attention)
    model = make_llama(torch.float32, "cpu", layers=1, d=32, heads=4, kv_heads=2, mlp=64, vocab=50)
    x = torch.randint(0, 50, (2, 6))
    want = model(x).logits
    with B.fused_model_ops(model):
        assert torch.allclose(model(x, num_items_in_batch=2).logits, want, atol=1e-5)
        with pytest.raises(ValueError, match="indices"):
            model(x, indices=torch.zeros(2, 6, 2, dtype=torch.int64))


class _Part(nn.Module):
    def __init__(self, implementation, takes=True):
        super().__init__()
        self.config = type("Config", (), {"_attn_implementation": implementation})()
        self.takes = takes


class _Whole(_Part):
    """Two parts with configurations of their own under one that, like transformers' composite models, sets them all --
    those that take it."""

    def __init__(self, *parts, takes=True):
        super().__init__("sdpa", takes)
        self.parts = nn.ModuleList(parts)

    def set_attn_implementation(self, name):
        for m in (self, *self.parts):
            if m.takes:
                m.config._attn_implementation = name


def test_every_part_gets_its_own_attention_back():
    model = _Whole(_Part("eager"), _Part("sdpa"))
    of = lambda: [m.config._attn_implementation for m in (model, *model.parts)]
    with B.fused_model_ops(model):
        assert of() == ["bergson_amd"] * 3
    assert of() == ["sdpa", "eager", "sdpa"]
    with pytest.raises(KeyError), B.fused_model_ops(model):
        raise KeyError("inside")
    assert of() == ["sdpa", "eager", "sdpa"]
    unset = _Whole(_Part(None))
    unset.config._attn_implementation = None
    with B.fused_model_ops(unset):
        assert unset.config._attn_implementation == unset.parts[0].config._attn_implementation == "bergson_amd"
    assert unset.config._attn_implementation is None and unset.parts[0].config._attn_implementation is None


def test_an_attention_that_is_not_replaced_is_named():
    """Models outside transformers' registry keep their attention: said by a warning, once, and the rest goes on."""
    with pytest.warns(UserWarning, match="_Whole.*keeps its own attention"), B.fused_model_ops(_Whole(takes=False)):
        pass
    with pytest.warns(UserWarning, match="_Part.*keeps its own attention"), B.fused_model_ops(_Whole(_Part("eager", takes=False))):
        pass
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with B.fused_model_ops(_Whole(_Part("eager"))):
            pass
        with B.fused_model_ops(make_gpt_neox("pythia-14m", torch.float32, "cpu", layers=1)):
            pass
        with B.fused_model_ops(nn.Sequential(nn.LayerNorm(8))):     # nothing there to replace
            pass
