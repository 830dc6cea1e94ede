"""Refusals of the model operators (layer norm, causal attention, top-k distillation): every argument that does not
fit is refused before anything is enqueued, by the Python entry points and by the C ABI behind them."""
import ctypes as C

import pytest
import torch

import bergson_amd as B
from bergson_amd import _lib

P = C.c_void_p(256)


def test_layer_norm_refusals():
    x, w = torch.zeros(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        B.layer_norm(x, w, w)
    with pytest.raises(ValueError, match="weight"):
        B.layer_norm(x, torch.ones(7), None)
    with pytest.raises(ValueError, match="bias"):
        B.layer_norm(x, w, torch.ones(1, 8))
    with pytest.raises(ValueError, match="needs a weight"):
        B.layer_norm(x, None, None)
    with pytest.raises(TypeError, match="weight"):
        B.layer_norm(x.bfloat16(), w.half(), None)
    with pytest.raises(TypeError, match="bias"):
        B.layer_norm(x.bfloat16(), w, w.bfloat16())
    with pytest.raises(TypeError, match="unsupported dtype"):
        B.layer_norm(x.double(), w.double(), None)
    with pytest.raises(ValueError, match="1 to 16384"):
        B.layer_norm(torch.zeros(1, 16385), torch.ones(16385), None)
    with pytest.raises(ValueError, match="1 to 16384"):
        B.layer_norm(torch.zeros(3, 0), torch.ones(0), None)
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            B.layer_norm(x, w, None, eps)


def test_causal_attention_refusals():
    q, kv = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)
    cu = torch.tensor([0, 3, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        B.causal_attention(q, kv, kv)
    with pytest.raises(RuntimeError, match="no CPU path"):
        B.causal_attention(q[0], kv[0], kv[0], cu_seqlens=cu)
    with pytest.raises(ValueError, match=r"\[N, S, heads, D\]"):
        B.causal_attention(q[0, 0], kv[0, 0], kv[0, 0])
    with pytest.raises(ValueError, match="do not match"):
        B.causal_attention(q, kv, kv[..., :8])
    with pytest.raises(ValueError, match="do not match"):
        B.causal_attention(q[:, :4], kv, kv)
    with pytest.raises(ValueError, match="4 query heads on 3"):
        B.causal_attention(q, torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 3, 16))
    with pytest.raises(TypeError, match="one dtype"):
        B.causal_attention(q, kv, kv.half())
    with pytest.raises(TypeError, match="unsupported dtype"):
        B.causal_attention(q.double(), kv.double(), kv.double())
    with pytest.raises(ValueError, match="head dimension 136"):
        big = torch.zeros(1, 2, 1, 136)
        B.causal_attention(big, big, big)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            B.causal_attention(q, kv, kv, scale=scale)
    with pytest.raises(ValueError, match="cu_seqlens"):
        B.causal_attention(q, kv, kv, cu_seqlens=cu)
    with pytest.raises(ValueError, match="cu_seqlens"):
        B.causal_attention(q[0], kv[0], kv[0])
    with pytest.raises(ValueError, match="cu_seqlens"):
        B.causal_attention(q[0], kv[0], kv[0], cu_seqlens=cu, lengths=cu)


def test_topk_distillation_refusals():
    z, ids, t = torch.zeros(3, 10), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        B.topk_distillation(z, ids, t)
    with pytest.raises(ValueError, match="do not match|must be"):
        B.topk_distillation(z, ids[:2], t[:2])
    with pytest.raises(ValueError, match="do not match"):
        B.topk_distillation(z, ids, t[:, :1])
    with pytest.raises(ValueError, match="must be"):
        B.topk_distillation(z, ids[:, 0], t[:, 0])
    with pytest.raises(TypeError, match="int64"):
        B.topk_distillation(z, ids.int(), t)
    with pytest.raises(TypeError, match="unsupported dtype"):
        B.topk_distillation(z.double(), ids, t)
    with pytest.raises(ValueError, match="1025 teacher entries"):
        B.topk_distillation(z, torch.zeros(3, 1025, dtype=torch.int64), torch.zeros(3, 1025))
    with pytest.raises(ValueError, match="0 teacher entries"):
        B.topk_distillation(z, ids[:, :0], t[:, :0])
    with pytest.raises(ValueError, match="detach"):
        B.topk_distillation(z, ids, t.clone().requires_grad_())
    for tau in (0.0, -2.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            B.topk_distillation(z, ids, t, temperature=tau)
    with pytest.raises(ValueError, match="valid"):
        B.topk_distillation(z, ids, t, valid=torch.ones(3))
    with pytest.raises(ValueError, match="valid"):
        B.topk_distillation(z, ids, t, valid=torch.ones(2, dtype=torch.bool))


def _plain_calls():
    x, w = torch.zeros(3, 8), torch.ones(8)
    q = torch.zeros(2, 5, 4, 16)
    ids, t = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    return {"layer_norm": (B.layer_norm, (x, w, w.clone())),
            "causal_attention": (B.causal_attention, (q, q.clone(), q.clone())),
            "topk_distillation": (lambda z, t: B.topk_distillation(z, ids, t), (torch.zeros(3, 10), t))}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["layer_norm", "causal_attention", "topk_distillation"])
def test_forward_mode_derivatives_are_refused(which, grad):
    """Every input's tangent: dropped, it would come out as a derivative of zero.  Also while no graph is recorded
    (forward mode does not ask for one), and from torch.func.jvp."""
    import torch.autograd.forward_ad as fwd

    fn, args = _plain_calls()[which]
    for i in range(len(args)):
        with fwd.dual_level(), torch.set_grad_enabled(grad):
            dual = [fwd.make_dual(a, torch.ones_like(a)) if j == i else a for j, a in enumerate(args)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*dual)
        with pytest.raises(NotImplementedError, match="forward-mode"), torch.set_grad_enabled(grad):
            torch.func.jvp(lambda a: fn(*args[:i], a, *args[i + 1:]), (args[i],), (torch.ones_like(args[i]),))
    with fwd.dual_level():
        dual = [fwd.make_dual(a, torch.ones_like(a)) for a in args]
        with pytest.raises(RuntimeError, match="no CPU path"):     # what carries no tangent goes on to the other checks
            fn(*(fwd.unpack_dual(d).primal for d in dual))


def test_struct_layouts_match_the_header():
    # three pointers, int64, five int32, one float
    assert C.sizeof(_lib.AttentionShape) == 3 * 8 + 8 + 5 * 4 + 4
    assert _lib.AttentionShape.rows.offset == 24 and _lib.AttentionShape.scale.offset == 52
    assert C.sizeof(_lib.AttentionRows) == 4 * 8


def test_c_abi_refusals():
    lib = _lib.load()
    norm = lambda x=P, y=P, w=P, wdt=2, rows=4, d=8, dt=2, xs=8, mean=None, rstd=None: lib.bgx_layernorm_forward(
        x, xs, w, None, wdt, rows, d, dt, 1e-5, y, 8, mean, rstd, None)
    assert norm(x=None) == -1 and b"null" in lib.bgx_last_error()
    assert norm(w=None) == -1
    assert norm(rows=-1) == -1
    assert norm(d=16385) == -3 and b"16384" in lib.bgx_last_error()
    assert norm(dt=7) == -2
    assert norm(wdt=1) == -2 and b"weight dtype" in lib.bgx_last_error()
    assert norm(xs=7) == -1 and b"stride" in lib.bgx_last_error()
    assert norm(mean=P) == -1
    assert norm(rows=0, x=None) == 0
    back = lambda ws=P, nbytes=1 << 20, dx=P, dw=P, rows=5000, d=8, mean=P: lib.bgx_layernorm_backward(
        P, 8, P, 8, P, 2, mean, P, rows, d, 2, dx, 8, dw, None, ws, nbytes, None)
    assert back(ws=None, nbytes=0) == -4 and b"workspace" in lib.bgx_last_error()
    assert back(nbytes=8) == -4
    assert back(mean=None) == -1
    assert back(dx=None, dw=None) == 0     # nothing asked for
    assert lib.bgx_layernorm_backward_workspace_bytes(5000, 8) == 512 * 2 * 8 * 4   # a row of partial sums a workgroup
    assert lib.bgx_layernorm_backward_workspace_bytes(20, 7) == 5 * 2 * 7 * 4       # four rows a workgroup
    assert lib.bgx_layernorm_backward_workspace_bytes(1024, 8) == 0                 # few rows: no partial sums
    assert lib.bgx_layernorm_backward_workspace_bytes(0, 8) == 0
    assert lib.bgx_layernorm_backward_workspace_bytes(4, 1 << 20) == 0

    def shape(**kw):
        s = _lib.AttentionShape(None, None, None, 10, 2, 4, 2, 16, 2, 0.25)
        for name, value in kw.items():
            setattr(s, name, value)
        return C.byref(s)

    rows = C.byref(_lib.AttentionRows(256, 16, 16, 16))
    fwd = lambda s, q=rows: lib.bgx_attention_forward(s, q, rows, rows, rows, None, None)
    assert fwd(None) == -1 and b"null" in lib.bgx_last_error()
    assert fwd(shape(), None) == -1
    assert fwd(shape(), C.byref(_lib.AttentionRows(None, 0, 0, 0))) == -1
    assert fwd(shape(kv_heads=3)) == -3 and fwd(shape(heads=0)) == -3
    assert fwd(shape(head_dim=129)) == -3 and b"129" in lib.bgx_last_error()
    assert fwd(shape(head_dim=20)) == -3 and b"16-byte" in lib.bgx_last_error()
    assert fwd(shape(head_dim=6, dtype=0)) == -3
    assert fwd(shape(), C.byref(_lib.AttentionRows(256, 8, (1 << 22) + 1, 8))) == -3 and b"8 MiB" in lib.bgx_last_error()
    assert fwd(shape(), C.byref(_lib.AttentionRows(256, 8, -16, 8))) == -3 and fwd(shape(), C.byref(_lib.AttentionRows(256, 8, 15, 8))) == -3
    assert fwd(shape(dtype=5)) == -2
    assert fwd(shape(scale=0.0)) == -1 and fwd(shape(scale=float("nan"))) == -1
    assert fwd(shape(rows=11)) == -1 and b"one width" in lib.bgx_last_error()
    assert fwd(shape(rows=1 << 31)) == -3
    assert fwd(shape(rows=0, n_seqs=0)) == 0
    assert fwd(shape(cu_seqlens_dev=256, n_seqs=65)) == -1 and b"65 sequences" in lib.bgx_last_error()
    assert fwd(shape(cu_seqlens_dev=256, plan_dev=256)) == -1
    bwd = lambda s, saved=P, ws=P, nbytes=1 << 20: lib.bgx_attention_backward(
        s, rows, rows, rows, rows, saved, rows, rows, rows, rows, ws, nbytes, None)
    assert bwd(shape(), saved=None) == -1 and b"saved" in lib.bgx_last_error()
    assert bwd(shape(), ws=None) == -4 and bwd(shape(), nbytes=16) == -4
    # delta per head and row, and with shared heads and few workgroups fp32 parts of dk and dv per query head
    assert lib.bgx_attention_backward_workspace_bytes(shape()) == 10 * 4 * 4 + 2 * 10 * 4 * 16 * 4
    assert lib.bgx_attention_backward_workspace_bytes(shape(kv_heads=4)) == 10 * 4 * 4
    assert lib.bgx_attention_backward_workspace_bytes(shape(kv_heads=4, dtype=1)) == 2 * 10 * 4 * 4
    assert lib.bgx_attention_backward_workspace_bytes(shape(rows=2 * 128 * 96)) == 2 * 128 * 96 * 4 * 4
    assert bwd(shape(), ws=C.c_void_p(264)) == -5
    # two statistics per head and row; at 16 bits also what the output's rounding cuts off
    assert lib.bgx_attention_saved_bytes(shape()) == 10 * 4 * (2 * 4 + 16 * 2)
    assert lib.bgx_attention_saved_bytes(shape(dtype=0)) == 10 * 4 * 2 * 4
    assert lib.bgx_attention_plan_bytes(1000, 3) == sum(1000 // height + 3 + 2 for height in (128, 64, 32)) * 16
    assert lib.bgx_attention_plan(P, 3, 1000, P, 16, None) == -4
    assert lib.bgx_attention_plan(None, 3, 1000, P, 1 << 20, None) == -1

    dist = lambda z=P, ids=P, V=10, K=2, tau=1.0, dt=2, tdt=0, stride=10, losses=P, rows=4: lib.bgx_distill_forward(
        z, stride, rows, V, dt, ids, P, tdt, K, None, tau, losses, None, None)
    assert dist(z=None) == -1 and dist(ids=None) == -1 and dist(losses=None) == -1
    assert dist(K=1025) == -3 and dist(K=0) == -1 and dist(V=0) == -1
    assert dist(tau=0.0) == -1 and b"temperature" in lib.bgx_last_error()
    assert dist(dt=3) == -2 and dist(tdt=-1) == -2
    assert dist(stride=9) == -1
    assert dist(rows=0, z=None, ids=None, losses=None) == 0
    rc = lib.bgx_distill_backward(P, 10, 4, 10, 2, P, P, 0, 2, 1.0, None, P, P, 10, None)
    assert rc == -1 and b"null" in lib.bgx_last_error()
