"""Collection runs whose model runs on the fused operators, against the CPU oracle and against plain autograd.

Tolerances are those of the same comparison without the fused operators (test_end_to_end_gpu.py): rel-L2 1e-3 for rows
of an fp32 model whose own passes run on different devices."""
import numpy as np
import pytest
import torch

import bergson_amd as B
from bergson_amd.synthetic import ListDataset, make_gpt_neox, make_llama, random_docs
from helpers import rel_l2
from oracle import loop as oloop

pytestmark = pytest.mark.gpu


def _processor(p):
    return B.GradientProcessor(projection_dim=p, projection_type="normal")


@pytest.mark.parametrize("overlap", [True, False])
def test_store_matches_cpu_loop(device, overlap):
    lengths = [64, 64, 40, 33, 17, 64, 2, 50, 29]
    docs = random_docs(lengths, seed=3)
    batches = B.allocate_batches(lengths, 128)
    cpu = make_gpt_neox("pythia-14m", torch.float32, "cpu", seed=0, layers=3)
    want, want_losses = oloop.collect(cpu, cpu.base_model, docs, batches, p=16)
    model = make_gpt_neox("pythia-14m", torch.float32, device, seed=0, layers=3)
    cfg = B.IndexConfig(run_path="", projection_dim=16, projection_type="normal", fused_model_ops=True)
    col = B.collect_gradients(model, ListDataset(docs), _processor(16), cfg, batches=batches, overlap_backward=overlap)
    assert model.config._attn_implementation != "bergson_amd"
    assert rel_l2(torch.from_numpy(np.array(col.builder.grad_buffer)), want) <= 1e-3
    assert torch.allclose(col.per_doc_losses.cpu(), want_losses, rtol=1e-4, atol=1e-4)


def test_grouped_heads_match_the_library(device):
    """A Llama-shaped model, 4 query heads on 2 key/value heads: the rows of the run without fused operators."""
    lengths = [50, 130, 7, 90]
    docs = random_docs(lengths, vocab=500, seed=1)
    rows = []
    for fused in (False, True):
        model = make_llama(torch.float32, device, layers=2, d=128, heads=4, kv_heads=2, mlp=256, vocab=500, seed=3)
        cfg = B.IndexConfig(run_path="", projection_dim=8, projection_type="normal", fused_model_ops=fused)
        col = B.collect_gradients(model, ListDataset(docs), _processor(8), cfg, batches=[[0, 1], [2, 3]])
        rows.append(torch.from_numpy(np.array(col.builder.grad_buffer)))
    assert rel_l2(rows[1], rows[0]) <= 1e-3


@pytest.mark.parametrize("overlap", [True, False])
def test_checkpointed_model(device, overlap):
    """Activation checkpointing recomputes blocks on the backward pass' threads: the rows of the run without it."""
    lengths = [50, 130, 7, 90]
    docs = random_docs(lengths, vocab=500, seed=1)
    rows = []
    for checkpointed in (False, True):
        model = make_llama(torch.float32, device, layers=2, d=128, heads=4, kv_heads=2, mlp=256, vocab=500, seed=3)
        model.train()
        if checkpointed:
            model.gradient_checkpointing_enable({"use_reentrant": False})
        cfg = B.IndexConfig(run_path="", projection_dim=8, projection_type="normal", fused_model_ops=True)
        col = B.collect_gradients(model, ListDataset(docs), _processor(8), cfg, batches=[[0, 1], [2, 3]],
                                  overlap_backward=overlap)
        rows.append(torch.from_numpy(np.array(col.builder.grad_buffer)))
    assert rel_l2(rows[1], rows[0]) <= 1e-3


def test_sixteen_bit_model(device):
    """bf16: fused and library rows are two roundings of the same fp32 rows -- the fused run is no further from them
    than the library's, up to half as much again."""
    lengths = [200, 77, 140]
    docs = random_docs(lengths, seed=2)
    rows = {}
    for dtype, fused in ((torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True)):
        model = make_gpt_neox("pythia-14m", torch.bfloat16, device, seed=0, layers=2).to(dtype)
        cfg = B.IndexConfig(run_path="", projection_dim=16, projection_type="normal", fused_model_ops=fused)
        col = B.GradientCollector(model=model.base_model, cfg=cfg, data=ListDataset(docs), processor=_processor(16),
                                  store_dtype=torch.float32)
        B.CollectorComputer(model=model, data=ListDataset(docs), collector=col, batches=[[0, 1, 2]], cfg=cfg
                            ).run_with_collector_hooks()
        rows[dtype, fused] = torch.from_numpy(np.array(col.builder.grad_buffer, dtype=np.float32))
    exact = rows[torch.float32, False]
    assert rel_l2(rows[torch.bfloat16, True], exact) <= 1.5 * rel_l2(rows[torch.bfloat16, False], exact)


@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_distillation_rows_match_autograd(device, reduction):
    """loss_fn="topk_kl" with fused operators: unprojected rows against the weight gradients of the definition on the
    CPU; labels that leave tokens out, lists of different lengths, a document weight."""
    lengths, V, tau = [40, 23, 31], 300, 2.0
    docs = random_docs(lengths, vocab=V, seed=5)
    gen = torch.Generator().manual_seed(0)
    ids = [[torch.randperm(V, generator=gen)[:1 + (s % 6)].tolist() for s in range(l)] for l in lengths]
    logits = [[torch.randn(len(t), generator=gen).tolist() for t in doc] for doc in ids]
    labels = [list(d) for d in docs]
    labels[0][:10] = [-100] * 10
    advantage = [1.0, -0.5, 2.0]
    cpu = make_gpt_neox("pythia-14m", torch.float32, "cpu", seed=0, layers=1, vocab=V)
    linears = {n: m for n, m in cpu.base_model.named_modules() if isinstance(m, torch.nn.Linear)}
    for m in linears.values():
        m.weight.requires_grad_(True)
    want, want_losses = [], []
    for n, doc in enumerate(docs):
        z = cpu(torch.tensor([doc])).logits[0]
        loss, count = 0.0, 0
        for s in range(len(doc) - 1):
            if labels[n][s + 1] == -100:
                continue
            log_p = torch.log_softmax(torch.tensor(logits[n][s]) / tau, 0)
            log_q = torch.log_softmax(z[s] / tau, 0)[ids[n][s]]
            loss, count = loss + tau ** 2 * (log_p.exp() * (log_p - log_q)).sum(), count + 1
        loss = loss * advantage[n] / (count if reduction == "mean" else 1)
        want_losses.append(loss.item())
        want.append(torch.cat([g.flatten() for g in torch.autograd.grad(loss, [m.weight for m in linears.values()])]))
    data = ListDataset(docs, labels=labels, advantage=advantage, teacher_ids=ids, teacher_logits=logits)
    model = make_gpt_neox("pythia-14m", torch.float32, device, seed=0, layers=1, vocab=V)
    cfg = B.IndexConfig(run_path="", projection_dim=0, loss_fn="topk_kl", distill_temperature=tau, loss_reduction=reduction,
                        fused_model_ops=True)
    col = B.collect_gradients(model, data, B.GradientProcessor(projection_dim=None), cfg, batches=[[0, 1], [2]])
    got = torch.from_numpy(np.array(col.builder.grad_buffer))
    assert rel_l2(got, torch.stack(want)) <= 1e-3
    assert torch.allclose(col.per_doc_losses.cpu().double(), torch.tensor(want_losses, dtype=torch.float64), rtol=1e-4,
                          atol=1e-4)


def test_training_step_of_a_model(device):
    """Norm weights trained: parameter gradients of a fused model against the library's, fp32."""
    x = torch.randint(0, 400, (3, 70), generator=torch.Generator().manual_seed(1)).to(device)
    grads = []
    for fused in (False, True):
        model = make_gpt_neox("pythia-14m", torch.float32, device, seed=0, layers=2, vocab=400)
        model.requires_grad_(True)
        if fused:
            with B.fused_model_ops(model):
                model(x, labels=x).loss.backward()
        else:
            model(x, labels=x).loss.backward()
        grads.append({n: q.grad for n, q in model.named_parameters() if q.grad is not None})
    assert grads[0].keys() == grads[1].keys() and any("layernorm" in n for n in grads[0])
    for name, want in grads[0].items():
        assert rel_l2(grads[1][name], want) <= 1e-3, name
