"""Layer norm, causal attention and top-k distillation against their definitions in 64 bits, elementwise within the
bounds derived in model_reference.py; plus what must hold exactly: rows outside every sequence, masked tokens,
repeated runs, other layouts of the same values, captured graphs."""
import math
import threading

import pytest
import torch

import bergson_amd as B
from model_reference import assert_within, attention_reference, distill_reference, norm_reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ids_of = lambda v: str(v).removeprefix("torch.").replace(" ", "")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- layer norm ---------------------------------------------------------------------------------------------------

def _norm_case(rows, d, dtype, w_dtype, seed, device):
    g = _gen(seed)
    x = (torch.randn(rows, d, generator=g) * 2 + 0.5).to(dtype).to(device)
    w = (1 + 0.3 * torch.randn(d, generator=g)).to(w_dtype).to(device)
    b = (0.2 * torch.randn(d, generator=g)).to(w_dtype).to(device)
    dy = torch.randn(rows, d, generator=g).to(dtype).to(device)
    return x, w, b, dy


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 768), (3, 7), (5, 64), (37, 129), (66, 511), (9, 512), (4, 513),
                                    (130, 1001), (7, 2047), (6, 2049), (5, 4096), (3, 5001), (2, 8193), (2, 16384),
                                    (2100, 40), (4097, 40), (4500, 1001), (4100, 2050), (4099, 5), (1024, 16), (1025, 16)], ids=str)
def test_layer_norm(device, rows, d, dtype):
    x, w, b, dy = _norm_case(rows, d, dtype, dtype, rows * 31 + d, device)
    for t in (x, w, b):
        t.requires_grad_()
    y = B.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = norm_reference(x, w, b, 1e-5, dy, dtype, dtype)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert got.dtype == dtype
        assert_within(got, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(B.layer_norm(x, w, b), y)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids_of)
@pytest.mark.parametrize("rows,d", [(21, 96), (21, 1500), (21, 5000), (1100, 97)])
def test_layer_norm_fp32_weights(device, dtype, rows, d):
    x, w, b, dy = _norm_case(rows, d, dtype, torch.float32, d, device)
    for t in (x, w, b):
        t.requires_grad_()
    y = B.layer_norm(x, w, b, 1e-3)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ref = norm_reference(x, w, b, 1e-3, dy, dtype, torch.float32)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("rows", [70, 1100])
def test_layer_norm_subsets_of_gradients(device, rows):
    """Frozen weights (a collection run), no bias, frozen input: each gradient equals the one of the full call."""
    x, w, b, dy = _norm_case(rows, 300, torch.bfloat16, torch.bfloat16, 5, device)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(B.layer_norm(*full), full, dy)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False)):
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        asked = [t for t in leaves if t.requires_grad]
        got = iter(torch.autograd.grad(B.layer_norm(*leaves), asked, dy))
        for n, ref in zip(need, want):
            if n:
                assert torch.equal(next(got), ref)
    xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = B.layer_norm(xx, ww)
    ref = norm_reference(x, w, None, 1e-5, dy, torch.bfloat16, torch.bfloat16)
    dx, dw = torch.autograd.grad(y, (xx, ww), dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        assert_within(got, *ref[name], name)


def test_layer_norm_layouts(device):
    """Rows of a wider matrix, an odd storage offset, transposed and broadcast inputs: the values of a plain copy."""
    g = _gen(3)
    base = torch.randn(40, 210, generator=g).to(torch.bfloat16).to(device)
    w, b = torch.rand(101, generator=g).to(torch.bfloat16).to(device), torch.zeros(101, dtype=torch.bfloat16, device=device)
    views = [base[:, 3:104], base[::2, 7:108], base[:, :101].reshape(4, 10, 101).transpose(0, 1),
             base.t()[:101].t(), base[:1, :101].expand(6, 101)]
    for v in views:
        a, c = v.detach().requires_grad_(), v.contiguous().clone().requires_grad_()
        ya, yc = B.layer_norm(a, w, b), B.layer_norm(c, w, b)
        assert torch.equal(ya, yc)
        da, = torch.autograd.grad(ya.sum(), a)    # a broadcast output gradient
        dc, = torch.autograd.grad(yc, c, torch.ones_like(yc))
        assert torch.equal(da, dc)


def test_layer_norm_empty_and_extreme(device):
    w = torch.ones(16, device=device, requires_grad=True)
    x = torch.zeros(0, 16, device=device, requires_grad=True)
    y = B.layer_norm(x, w, w)
    assert y.shape == (0, 16)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 16) and dw.abs().sum() == 0
    # constant rows: xh = 0, dx finite; a NaN or an infinity stays in its row
    x = torch.full((3, 16), 1e4, device=device)
    x[1, 3], x[2, 5] = float("nan"), float("inf")
    y = B.layer_norm(x, w.detach(), None)
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2].isnan().any()
    # a large common offset does not swallow the deviations
    g = _gen(9)
    x = (4096 + torch.randn(8, 600, generator=g)).to(device)
    ref = norm_reference(x, torch.ones(600), None, 1e-5, None, torch.float32, torch.float32)
    assert_within(B.layer_norm(x, torch.ones(600, device=device)), *ref["y"], "offset")


# ---- causal attention ---------------------------------------------------------------------------------------------

def _qkv(lead, heads, kv_heads, dim, dtype, seed, device, gain=1.2):
    g = _gen(seed)
    make = lambda n: (gain * torch.randn(*lead, n, dim, generator=g)).to(dtype).to(device)
    return make(heads), make(kv_heads), make(kv_heads), make(heads)


def _check_sequences(q, k, v, do, out, grads, spans, scale, dtype):
    """Every sequence within its bounds, everything outside the sequences exactly zero."""
    flat = lambda t: t.detach().reshape(-1, *t.shape[-2:])
    q, k, v, do, out = map(flat, (q, k, v, do, out))
    grads = [flat(t) for t in grads]
    covered = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    for a, b in spans:
        covered[a:b] = True
        if a == b:
            continue
        ref = attention_reference(q[a:b], k[a:b], v[a:b], scale, do[a:b], dtype)
        for name, got in zip(("o", "dq", "dk", "dv"), (out, *grads)):
            assert_within(got[a:b], *ref[name], f"{name} of rows {a}:{b}")
    for t in (out, *grads):
        assert (t[~covered] == 0).all()


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 64), (4, 2, 128), (3, 1, 32), (2, 1, 96), (1, 1, 80), (2, 2, 20),
                                                (1, 1, 7)], ids=str)
@pytest.mark.parametrize("lengths", [[1], [2, 33], [64, 1, 31, 65], [129, 127, 300]], ids=str)
def test_attention_packed(device, bgx_env, lengths, heads, kv_heads, dim, dtype, rows):
    bgx_env("BGX_ATTENTION_ROWS", rows)
    T = sum(lengths)
    q, k, v, do = _qkv((T,), heads, kv_heads, dim, dtype, T + dim, device)
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(device)
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=cu)
    grads = torch.autograd.grad(out, (q, k, v), do)
    ends = cu.tolist()
    _check_sequences(q, k, v, do, out, grads, list(zip(ends, ends[1:])), dim ** -0.5, dtype)


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("N,S,lengths", [(1, 1, None), (2, 130, None), (3, 200, [200, 0, 77]), (4, 64, [1, 64, 65, -3])],
                         ids=str)
def test_attention_batch(device, bgx_env, N, S, lengths, dtype, rows):
    """lengths beyond the width or below zero count as the width and zero."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _qkv((N, S), 4, 2, 64, dtype, N * S, device)
    for t in (q, k, v):
        t.requires_grad_()
    dev = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    out = B.causal_attention(q, k, v, lengths=dev, scale=0.21)
    grads = torch.autograd.grad(out, (q, k, v), do)
    spans = [(n * S, n * S + min(max(l, 0), S)) for n, l in enumerate(lengths or [S] * N)]
    _check_sequences(q, k, v, do, out, grads, spans, 0.21, dtype)


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_attention_rows_outside_the_sequences(device, bgx_env, dtype, rows):
    """NaN in rows before, after and between nothing reaches the sequences; those rows come out as zeros."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    T, cu_list = 400, [40, 100, 100, 260]
    q, k, v, do = _qkv((T,), 2, 1, 64, dtype, 8, device)
    outside = torch.ones(T, dtype=torch.bool, device=device)
    outside[40:260] = False
    for t in (q, k, v, do):
        t[outside] = float("nan")
    for t in (q, k, v):
        t.requires_grad_()
    cu = torch.tensor(cu_list, dtype=torch.int32, device=device)
    out = B.causal_attention(q, k, v, cu_seqlens=cu)
    grads = torch.autograd.grad(out, (q, k, v), do)
    _check_sequences(q, k, v, do, out, grads, list(zip(cu_list, cu_list[1:])), 0.125, dtype)
    # the same in the batch layout
    qb, kb, vb, dob = (t.detach()[:400].reshape(2, 200, *t.shape[1:]).clone() for t in (q, k, v, do))
    for t in (qb, kb, vb, dob):
        t.nan_to_num_(nan=0.5)
        t[0, 90:] = float("nan")
        t[1, 7:] = float("inf")
    for t in (qb, kb, vb):
        t.requires_grad_()
    out = B.causal_attention(qb, kb, vb, lengths=torch.tensor([90, 7], dtype=torch.int32, device=device))
    grads = torch.autograd.grad(out, (qb, kb, vb), dob)
    _check_sequences(qb, kb, vb, dob, out, grads, [(0, 90), (200, 207)], 0.125, dtype)


def test_attention_layouts_and_broadcast(device):
    """Views of one projection, heads before positions, shared keys by expand: the bits of plain copies, and the
    gradient of a broadcast input is the sum over its copies."""
    g = _gen(4)
    qkv = torch.randn(2, 150, 3, 3 * 64, generator=g).to(torch.bfloat16).to(device)
    do = torch.randn(2, 150, 3, 64, generator=g).to(torch.bfloat16).to(device)
    views = [qkv.split(64, -1), [t.transpose(1, 2).contiguous().transpose(1, 2) for t in qkv.split(64, -1)]]
    odd = torch.randn(2, 150, 3, 3 * 64 + 1, generator=g).to(torch.bfloat16).to(device)
    odd[..., 1:].copy_(qkv)
    views.append(odd[..., 1:].split(64, -1))
    plain = [t.contiguous().requires_grad_() for t in views[0]]
    want = B.causal_attention(*plain)
    want_grads = torch.autograd.grad(want, plain, do)
    for view in views:
        leaves = [t.detach().requires_grad_() for t in view]
        out = B.causal_attention(*leaves)
        assert torch.equal(out, want)
        for got, ref in zip(torch.autograd.grad(out, leaves, do), want_grads):
            assert torch.equal(got, ref)
    # a transposed output gradient and a broadcast one
    leaves = [t.detach().requires_grad_() for t in views[0]]
    out = B.causal_attention(*leaves)
    a = torch.autograd.grad(out, leaves, do.transpose(1, 2).contiguous().transpose(1, 2), retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(a, want_grads))
    a = torch.autograd.grad(out, leaves, torch.ones((), dtype=do.dtype, device=device).expand_as(out), retain_graph=True)
    b = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = plain[1].detach()[:, :, :1].clone().requires_grad_()
    shared = B.causal_attention(plain[0].detach(), one.expand(2, 150, 3, 64), plain[2].detach())
    copied = plain[1].detach()[:, :, :1].repeat(1, 1, 3, 1).requires_grad_()
    ref = B.causal_attention(plain[0].detach(), copied, plain[2].detach())
    assert torch.equal(shared, ref)
    got, = torch.autograd.grad(shared, one, do)
    full, = torch.autograd.grad(ref, copied, do)
    assert torch.equal(got, full.sum(2, keepdim=True))


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_attention_far_scores(device, bgx_env, dtype, rows):
    """Scores hundreds apart, -inf in a key (its weight is 0 wherever it is seen), keys at the type's lowest values."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _qkv((140,), 1, 1, 32, dtype, 6, device, gain=6.0)
    cu = torch.tensor([0, 140], dtype=torch.int32, device=device)
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=cu, scale=1.0)
    grads = torch.autograd.grad(out, (q, k, v), do)
    _check_sequences(q, k, v, do, out, grads, [(0, 140)], 1.0, dtype)
    # the first 64 keys give scores of -inf: the rows after them see only the rest
    q2, k2 = q.detach().abs() + 0.1, k.detach().clone()
    k2[:64, 0] = float("-inf")
    out = B.causal_attention(q2.to(dtype), k2, v.detach(), cu_seqlens=cu)
    rest = B.causal_attention(q2.to(dtype)[64:], k2[64:], v.detach()[64:],
                              cu_seqlens=torch.tensor([0, 76], dtype=torch.int32, device=device))
    ref = attention_reference(q2.to(dtype)[64:], k2[64:], v.detach()[64:], 32 ** -0.5, None, dtype)
    assert_within(out[64:], *ref["o"], "rows that see finite scores")
    assert_within(rest, *ref["o"], "the same rows alone")
    assert out[:64].isnan().all()     # softmax of nothing but -inf


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_attention_lowest_scores(device, bgx_env, dtype, rows):
    """Scores at the type's lowest value, which the exponents' factor takes past the numbers: the rows that see others
    beside them give those a weight of 0."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, _ = _qkv((140,), 1, 1, 32, dtype, 6, device)
    q[..., 0], k[:64, :, 0] = 1.0, torch.finfo(dtype).min
    out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor([0, 140], dtype=torch.int32, device=device), scale=1.0)
    ref = attention_reference(q[64:], k[64:], v[64:], 1.0, None, dtype)
    assert_within(out[64:], *ref["o"], "rows that see more than the lowest value")


@pytest.mark.parametrize("rows", [128, 64, 32])
def test_attention_small_gradients_in_fp16(device, bgx_env, rows):
    """Output gradients near fp16's smallest normal number: dS itself would vanish among the subnormals."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _qkv((260,), 2, 1, 64, torch.float16, 12, device)
    do = (do.float() * 2.0 ** -12).half()
    do[:100] *= 2.0 ** -2
    cu = torch.tensor([0, 260], dtype=torch.int32, device=device)
    for t in (q, k, v):
        t.requires_grad_()
    grads = torch.autograd.grad(B.causal_attention(q, k, v, cu_seqlens=cu), (q, k, v), do)
    big = torch.autograd.grad(B.causal_attention(q, k, v, cu_seqlens=cu), (q, k, v), (do.float() * 2.0 ** 12).half())
    for small, large in zip(grads, big):
        # scaled by a power of two: the same up to the rounding of the results among the subnormals
        assert (small.double() - large.double() * 2.0 ** -12).abs().max() <= 2.0 ** -25 + 2.0 ** -11 * small.abs().max()
    _check_sequences(q, k, v, do, B.causal_attention(q, k, v, cu_seqlens=cu), grads, [(0, 260)], 0.125, torch.float16)


@pytest.mark.parametrize("rows", [128, 64, 32])
def test_attention_large_values_in_fp16(device, bgx_env, rows):
    """Values near 2^8 and weights far above those of a row's first tile: dS of weights that are not yet divided by
    their sum would leave fp16's range."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _qkv((260,), 2, 1, 64, torch.float16, 13, device, gain=1.0)
    q, k, v = q * 0.1, k * 0.1, v * 64
    q[..., 0], k[:, :, 0] = 1.0, 0.0
    k[130:, :, 0] = 5.0   # 2^7.2 times the weight
    cu = torch.tensor([0, 260], dtype=torch.int32, device=device)
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=cu, scale=1.0)
    grads = torch.autograd.grad(out, (q, k, v), do)
    _check_sequences(q, k, v, do, out, grads, [(0, 260)], 1.0, torch.float16)


# dS in fp16 goes in with the bound of its row (dq) or tile (dk) brought to 2^12 or more: what is rounded as a multiple
# of 2^-24 loses at most 2^-25 2^-12 of that bound, which is no more than the largest |dp - delta|
DS_FLOOR = 2.0 ** -37


@pytest.mark.parametrize("rows", [128, 64, 32])
def test_attention_ds_past_fp16(device, bgx_env, rows):
    """Two positions whose dS is +-625 while the output gradients are small: dq is 156.25 and dk 0, though dS in
    units of the output gradient's size does not fit fp16."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    sign = torch.tensor([1.0, -1.0], device=device).reshape(2, 1, 1)
    ones = torch.ones(2, 1, 64, device=device)
    q, k, v, do = ((t * ones).half() for t in (0.0, sign, 5000.0 * sign, 2.0 ** -8))
    for t in (q, k, v):
        t.requires_grad_()
    cu = torch.tensor([0, 2], dtype=torch.int32, device=device)
    out = B.causal_attention(q, k, v, cu_seqlens=cu)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    assert (dq[0] == 0).all() and (dq[1] == 156.25).all() and (dk == 0).all()
    _check_sequences(q, k, v, do, out, (dq, dk, dv), [(0, 2)], 0.125, torch.float16)


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("size", ["thousands", "growing", "falling", "small"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (1, 1, 128)], ids=str)
def test_attention_ds_of_any_size_in_fp16(device, bgx_env, heads, kv_heads, dim, size, rows):
    """Values in the thousands under small output gradients, values that grow or fall by 2^20 along the sequence, and
    small ones under weights that are spread over the sequence: dS is far from the size of the output gradients."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    L = 300
    q, k, v, do = (t.float() for t in _qkv((L,), heads, kv_heads, dim, torch.float16, dim + rows, device, gain=0.8))
    steps = torch.linspace(-10, 10, L, device=device).reshape(L, 1, 1)
    if size == "thousands":
        v, do = v * 4000, do * 2.0 ** -8
    elif size == "small":
        v, k, do = v * 2.0 ** -13, k * 64, do * 16
    else:
        v, do = v * 2.0 ** (steps if size == "growing" else -steps), do * 2.0 ** -4
    q, k, v, do = (t.half() for t in (q, k, v, do))
    scale = dim ** -0.5 * (2.0 ** -6 if size == "small" else 1.0)
    assert all(t.isfinite().all() for t in (q, k, v, do))
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor([0, L], dtype=torch.int32, device=device), scale=scale)
    grads = torch.autograd.grad(out, (q, k, v), do)
    ref = attention_reference(*(t.detach() for t in (q, k, v)), scale, do, torch.float16, ds_floor=DS_FLOOR)
    for name, got in zip(("o", "dq", "dk", "dv"), (out, *grads)):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("rows", [128, 32])
def test_attention_offsets_past_32_bits(device, bgx_env, rows):
    """Positions 2 MiB apart: the sequence spans more than 4 GiB of each operand, a tile far less."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    T, far = 2600, 1 << 20
    store = [torch.empty(T * far, dtype=torch.bfloat16, device=device) for _ in range(3)]
    views = [torch.as_strided(t, (T, 1, 64), (far, 64, 1)) for t in store]
    plain = _qkv((T,), 1, 1, 64, torch.bfloat16, 3, device)
    for view, t in zip(views, plain):
        view.copy_(t)
        view.requires_grad_()
    cu = torch.tensor([0, T], dtype=torch.int32, device=device)
    out = B.causal_attention(*views, cu_seqlens=cu)
    leaves = [t.clone().requires_grad_() for t in plain[:3]]
    want = B.causal_attention(*leaves, cu_seqlens=cu)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, views, plain[3]), torch.autograd.grad(want, leaves, plain[3])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=ids_of)
@pytest.mark.parametrize("length,dim", [(2, 64), (3, 128), (4, 32), (8, 64)], ids=str)
def test_attention_gradients_of_short_sequences(device, length, dim, dtype):
    """dq and dk of many short sequences are as near as their own rounding: what the kernel's operands lose (dS to 2^-21
    of its value as two of them, the fp32 sums less) is 2^-8 of that rounding, and moves a value across a rounding
    boundary so rarely that a twentieth covers both."""
    n, scale = 80, dim ** -0.5
    q, k, v, do = _qkv((n * length,), 8, 4, dim, dtype, length, device, gain=1.0)
    cu = torch.arange(0, n * length + 1, length, dtype=torch.int32, device=device)
    for t in (q, k, v):
        t.requires_grad_()
    grads = torch.autograd.grad(B.causal_attention(q, k, v, cu_seqlens=cu), (q, k), do)
    refs = [attention_reference(*(t.detach()[a:a + length] for t in (q, k, v)), scale, do[a:a + length], dtype)
            for a in range(0, n * length, length)]
    for got, name in zip(grads, ("dq", "dk")):
        want = torch.cat([r[name][0] for r in refs])
        rounding = (want.to(dtype).double() - want).norm()
        assert (got.cpu().double() - want).norm() <= 1.05 * rounding, name


def _flat_inputs(L, dim, dtype, offset, device):
    """One sequence whose scores are all alike: q and k share no dimension but the first, where q k = offset^2."""
    g = _gen(L + dim)
    q, k, v, do = (torch.zeros(L, dim, dtype=torch.float64) for _ in range(4))
    q[:, 1:32] = torch.randn(L, 31, generator=g)
    k[:, 32:] = torch.randn(L, dim - 32, generator=g)
    q[:, 0] = k[:, 0] = offset
    v[:], do[:] = torch.randn(L, dim, generator=g), torch.randn(L, dim, generator=g)
    return [t.to(dtype).unsqueeze(1).to(device) for t in (q, k, v, do)]


def _flat_results(q, k, v, do, dtype):
    """o, dq, dk, dv of the definition in 64 bits, which has a closed form: the weights of row i are 1 / (i + 1)."""
    q, k, v, do = (t[:, 0].cpu().double() for t in (q, k, v, do))
    L, dim = q.shape
    seen = torch.arange(1, L + 1, dtype=torch.float64).reshape(L, 1)
    o = v.cumsum(0) / seen
    delta = (do * o).sum(1, keepdim=True)
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    back = lambda t: t.flip(0).cumsum(0).flip(0)
    for d in range(32, dim):      # sum over j <= i of (do_i . v_j - delta_i) k_jd / (i + 1)
        dq[:, d] = (((k[:, d:d + 1] * v).cumsum(0) * do).sum(1) - delta[:, 0] * k[:, d].cumsum(0)) / seen[:, 0]
    for d in range(32):           # sum over i >= j of (do_i . v_j - delta_i) q_id / (i + 1)
        w = q[:, d:d + 1] / seen
        dk[:, d] = (back(w * do) * v).sum(1) - back(w * delta)[:, 0]
    # dv with every weight rounded to 2^-8 or 2^-11 of its value, whatever its size
    rounded = (2.0 ** 14 / seen).to(dtype).double() * 2.0 ** -14
    return {"o": o, "dq": dq, "dk": dk, "dv": back(do / seen), "rounded dv": back(rounded * do)}


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=ids_of)
@pytest.mark.parametrize("L,dim", [(32768, 64), (16384, 128)], ids=str)
def test_attention_of_long_flat_sequences(device, bgx_env, L, dim, dtype, rows):
    """Weights of 2^-15: dk and dv are made from operands below fp16's normal numbers.

    What the operands' roundings cost, against the results' own, in the later half (the smallest weights, and values of one
    size: the first rows alone would make the norms of all).  Of dq and dk: a row's or column's dS have random signs, so that the sum
    of their roundings has the size of one rounding of the sum, and the two are independent: 2^(1/2) of it.  Of dv: a row
    has one weight for all its keys, whose rounding error comes back in the whole column sum behind it; a few dozen of such
    errors (of the last rows, in 64 or 128 columns) make the norm, which then varies by a tenth from case to case.  So dv
    is held to what the exact weights' roundings make of these inputs.  In the 32-row workgroups, whose operands keep their
    rests, 1 for all of them.  A twentieth on top for what else is fp32."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _flat_inputs(L, dim, dtype, 0.0, device)
    want = _flat_results(q, k, v, do, dtype)
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor([0, L], dtype=torch.int32, device=device), scale=1.0)
    grads = torch.autograd.grad(out, (q, k, v), do)
    for name, got in zip(("o", "dq", "dk", "dv"), (out, *grads)):
        got, ref = got[L // 2:, 0].detach().cpu().double(), want[name][L // 2:]
        rounding, most = ref.to(dtype).double() - ref, 1.0 if rows == 32 else 2 ** 0.5
        if name == "dv" and rows != 32:
            rounding, most = want["rounded dv"][L // 2:].to(dtype).double() - ref, 1.0
        ratio = float((got - ref).norm() / rounding.norm())
        assert ratio <= 1.05 * most, (name, ratio)


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_large_flat_scores(device, bgx_env, dim, dtype, rows):
    """Scores that are all 2^16 give the bits of scores that are all 0, in every gradient: products, exponents and weights
    are exact in fp32 in both, whatever a shift of that size would lose in one number with the logarithm of the sum."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    cu, results = torch.tensor([0, 600], dtype=torch.int32, device=device), []
    for offset in (0.0, 256.0):
        q, k, v, do = _flat_inputs(600, dim, dtype, offset, device)
        for t in (q, k, v):
            t.requires_grad_()
        out = B.causal_attention(q, k, v, cu_seqlens=cu, scale=1.0)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
        # the dimension of the offset itself apart
        results.append({"o": out, "dq": dq[..., 1:], "dk": dk[..., 1:], "dv": dv})
    for name, first in results[0].items():
        assert torch.equal(first, results[1][name]), name


@pytest.mark.parametrize("rows", [128, 64])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=ids_of)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (2, 2, 96), (4, 2, 64)], ids=str)
def test_attention_of_short_and_long_sequences(device, bgx_env, heads, kv_heads, dim, dtype, rows):
    """Lengths on both sides of 64 in one call, empty ones among them, rows around them: found from the boundaries, from a
    plan, and cut by lengths -- short and long ones may have kernels of their own, and every row is written by one."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    lengths = [3, 300, 64, 0, 65, 1, 700]
    for head, tail, more in ((0, 0, 0), (70, 140, 0), (5, 3, 70)):      # 70 sequences more than go without a plan
        spread = lengths + [200] * 3 * (more > 0) + [1, 90] * (more // 2)
        ends = [head] + [head + int(e) for e in torch.tensor(spread).cumsum(0)]
        q, k, v, do = _qkv((ends[-1] + tail,), heads, kv_heads, dim, dtype, dim + head, device)
        for t in (q, k, v):
            t.requires_grad_()
        out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device=device))
        grads = torch.autograd.grad(out, (q, k, v), do)
        _check_sequences(q, k, v, do, out, grads, list(zip(ends, ends[1:])), dim ** -0.5, dtype)
    q, k, v, do = _qkv((6, 200), heads, kv_heads, dim, dtype, dim, device)
    for t in (q, k, v):
        t.requires_grad_()
    cut = [64, 200, 1, 0, 65, 33]
    out = B.causal_attention(q, k, v, lengths=torch.tensor(cut, dtype=torch.int32, device=device))
    grads = torch.autograd.grad(out, (q, k, v), do)
    _check_sequences(q, k, v, do, out, grads, [(200 * i, 200 * i + l) for i, l in enumerate(cut)], dim ** -0.5, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("length,n", [(3, 90), (48, 40), (64, 80), (65, 80), (300, 30)], ids=str)
def test_attention_output_does_not_depend_on_a_graph(device, dtype, length, n):
    """The same bits while a gradient is recorded and while none is (a checkpointed block runs both)."""
    q, k, v, _ = _qkv((n * length,), 8, 4, 64, dtype, length, device)
    cu = torch.arange(0, n * length + 1, length, dtype=torch.int32, device=device)
    plain = B.causal_attention(q, k, v, cu_seqlens=cu)
    kept = B.causal_attention(q.requires_grad_(), k, v, cu_seqlens=cu)
    assert kept.requires_grad and torch.equal(plain, kept)


def _rounding_ratios(q, k, v, do, grads, spans, scale, dtype):
    """How far dq and dk of the given rows are from the definition, in units of their own rounding."""
    flat = lambda t: t.detach().reshape(-1, *t.shape[-2:])
    q, k, v, do = map(flat, (q, k, v, do))
    refs = [attention_reference(q[a:b], k[a:b], v[a:b], scale, do[a:b], dtype) for a, b in spans]
    for got, name in zip(map(flat, grads), ("dq", "dk")):
        want = torch.cat([r[name][0] for r in refs])
        got = torch.cat([got[a:b] for a, b in spans]).cpu().double()
        yield name, float((got - want).norm() / (want.to(dtype).double() - want).norm())


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=ids_of)
@pytest.mark.parametrize("length,dim", [(2, 64), (5, 128)], ids=str)
def test_attention_gradients_of_short_sequences_beside_long_ones(device, bgx_env, length, dim, dtype, rows):
    """A short document's gradients are as near as in a call of short documents (the bound of
    test_attention_gradients_of_short_sequences), whatever it is packed or padded with."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    n, scale = 80, dim ** -0.5
    T = n * length + 9000
    q, k, v, do = _qkv((T,), 4, 2, dim, dtype, length, device, gain=1.0)
    ends = list(range(0, n * length + 1, length))
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor(ends + [T], dtype=torch.int32, device=device))
    grads = torch.autograd.grad(out, (q, k), do)
    for name, ratio in _rounding_ratios(q, k, v, do, grads, list(zip(ends, ends[1:])), scale, dtype):
        assert ratio <= 1.05, (name, ratio, "packed")
    q, k, v, do = _qkv((n, 130), 4, 2, dim, dtype, length, device, gain=1.0)
    for t in (q, k, v):
        t.requires_grad_()
    out = B.causal_attention(q, k, v, lengths=torch.full((n,), length, dtype=torch.int32, device=device))
    grads = torch.autograd.grad(out, (q, k), do)
    spans = [(i * 130, i * 130 + length) for i in range(n)]
    for name, ratio in _rounding_ratios(q, k, v, do, grads, spans, scale, dtype):
        assert ratio <= 1.05, (name, ratio, "padded")


def test_attention_plan_of_many_sequences(device):
    """More sequences than the planning workgroup has threads, empty ones among them, long ones at the end."""
    g = _gen(2)
    lengths = torch.randint(0, 4, (2600,), generator=g).tolist() + [500, 0, 300]
    T = sum(lengths) + 5
    q, k, v, _ = _qkv((T,), 1, 1, 32, torch.bfloat16, 1, device)
    ends = [0] + torch.tensor(lengths).cumsum(0).tolist()
    cu = torch.tensor(ends, dtype=torch.int32, device=device)
    out = B.causal_attention(q, k, v, cu_seqlens=cu)
    for a, b in zip(ends, ends[1:]):
        if b > a:
            ref = attention_reference(q[a:b], k[a:b], v[a:b], 32 ** -0.5, None, torch.bfloat16)
            assert_within(out[a:b], *ref["o"], f"rows {a}:{b}")
    assert (out[ends[-1]:] == 0).all()


def test_attention_plan_with_folded_levels(device):
    """More tiles than the planning workgroup has threads, so that a level is several tile indices: every tile of every
    sequence once, higher levels first, then the rows outside the sequences."""
    from bergson_amd import _lib

    lengths, head, rows = [70000, 5, 0, 40000, 129, 20000], 17, 140000
    ends = [head]
    for l in lengths:
        ends.append(ends[-1] + l)
    lib, bounds = _lib.load(), torch.tensor(ends, dtype=torch.int32, device=device)
    nbytes = lib.bgx_attention_plan_bytes(rows, len(lengths))
    plan = torch.full((nbytes,), 0x55, dtype=torch.uint8, device=device)
    _lib.check(lib.bgx_attention_plan(bounds.data_ptr(), len(lengths), rows, plan.data_ptr(), nbytes,
                                      torch.cuda.current_stream().cuda_stream), "plan")
    table, at = plan.cpu().view(torch.int32).reshape(-1, 4).tolist(), 0
    for height in (128, 64, 32):
        tiles, n = lambda l: -(-l // height), rows // height + len(lengths) + 2
        entries, at = [tuple(e) for e in table[at:at + n]], at + n
        fold = 0
        while tiles(rows) >> fold >= 1024:
            fold += 1
        assert fold > 0 or height != 128
        want = [(a, l, t, l) for a, l in zip(ends, lengths) for t in range(tiles(l))]
        work = entries[:len(want)]
        assert sorted(work) == sorted(want)
        levels = [t >> fold for _, _, t, _ in work]
        assert levels == sorted(levels, reverse=True)
        clear = ([(0, 0, i, head) for i in range(tiles(head))]
                 + [(ends[-1], 0, i, rows - ends[-1]) for i in range(tiles(rows - ends[-1]))])
        assert entries[len(want):] == clear + [(0, 0, 0, 0)] * (n - len(want) - len(clear))


def test_attention_of_folded_levels(device, bgx_env):
    """Documents packed into more than 1024 tiles of 32 rows: the bits of a call of each document by itself."""
    bgx_env("BGX_ATTENTION_ROWS", 32)
    lengths = [20000, 5, 0, 15000, 7001]
    q, k, v, do = _qkv((sum(lengths),), 4, 4, 32, torch.bfloat16, 40, device)
    ends = [0] + torch.tensor(lengths).cumsum(0).tolist()

    def run(q, k, v, do, ends):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = B.causal_attention(*leaves, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device=device))
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    packed = run(q, k, v, do, ends)
    for a, b in zip(ends, ends[1:]):
        if b > a:
            for whole, alone in zip(packed, run(q[a:b], k[a:b], v[a:b], do[a:b], [0, b - a])):
                assert torch.equal(whole[a:b], alone)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_tiles(device, bgx_env, dim, dtype):
    """2048 rows, scores and output gradients growing along them, so that maxima move on and the powers of two in fp16's dS
    are lowered many times: outputs and gradients against the definition, in every workgroup height."""
    L = 2048
    q, k, v, do = (t.float() for t in _qkv((L,), 2, 1, dim, dtype, dim, device, gain=1.0))
    along = torch.linspace(0, 1, L, device=device).reshape(L, 1, 1)
    q, k, v, do = (t.to(dtype) for t in (q, k * (0.25 + 4 * along), v, do * 2.0 ** (12 * along - 6)))
    for t in (q, k, v):
        t.requires_grad_()
    ref = attention_reference(*(t.detach() for t in (q, k, v)), dim ** -0.5, do, dtype)
    cu = torch.tensor([0, L], dtype=torch.int32, device=device)
    for rows in (128, 64, 32):
        bgx_env("BGX_ATTENTION_ROWS", rows)
        out = B.causal_attention(q, k, v, cu_seqlens=cu)
        for name, got in zip(("o", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, (q, k, v), do))):
            assert_within(got, *ref[name], f"{name} with {rows} rows")


def test_attention_malformed_boundaries_stay_in_bounds(device):
    """Boundaries that are not ascending or lie outside the rows: nothing is promised of the rows, but the call ends,
    and a following call on the same memory is right."""
    q, k, v, _ = _qkv((300,), 2, 2, 64, torch.bfloat16, 3, device)
    for bad in ([0, 500, 200], [-7, 40, 300], [250, 100, 50], [0, 300, 0, 300, 0, 300]):
        out = B.causal_attention(q, k, v, cu_seqlens=torch.tensor(bad, dtype=torch.int32, device=device))
        assert out.shape == q.shape
    cu = torch.tensor([0, 300], dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    assert torch.equal(B.causal_attention(q, k, v, cu_seqlens=cu), B.causal_attention(q[None], k[None], v[None])[0])


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("cu", [[0, 150], [20, 150, 150, 300], [0] * 40 + [300], [300, 300], [0], [0, 7, 14, 200, 299]],
                         ids=lambda c: f"{len(c) - 1}:{c[0]}-{c[-1]}")
def test_attention_plan_or_none(device, bgx_env, cu, rows):
    """The C ABI with a plan and with the boundaries themselves: the same bits, forward and backward, whatever lies
    outside the sequences; and again after 64 sequences, where only the plan is taken."""
    from bergson_amd import _lib

    bgx_env("BGX_ATTENTION_ROWS", rows)
    lib, P = _lib.load(), lambda t: t.data_ptr()
    q, k, v, do = _qkv((300,), 2, 1, 64, torch.bfloat16, 5, device)
    bounds = torch.tensor(cu, dtype=torch.int32, device=device)
    nbytes = lib.bgx_attention_plan_bytes(300, len(cu) - 1)
    plan = torch.empty(nbytes, dtype=torch.uint8, device=device)
    stream = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.bgx_attention_plan(P(bounds), len(cu) - 1, 300, P(plan), nbytes, stream), "plan")
    results = []
    for with_plan in (True, False):
        shape = _lib.AttentionShape(P(plan) if with_plan else None, None if with_plan else P(bounds), None, 300, len(cu) - 1,
                                    2, 1, 64, _lib.BGX_BF16, 0.125)
        rows_of = lambda t: _lib.AttentionRows(P(t), 0, t.stride(0), t.stride(1))
        out = [torch.full_like(t, float("nan")) for t in (q, q, k, v)]
        saved = torch.empty(lib.bgx_attention_saved_bytes(shape), dtype=torch.uint8, device=device)
        ws = torch.empty(lib.bgx_attention_backward_workspace_bytes(shape), dtype=torch.uint8, device=device)
        args = [rows_of(t) for t in (q, k, v)]
        _lib.check(lib.bgx_attention_forward(shape, *args, rows_of(out[0]), P(saved), stream), "forward")
        _lib.check(lib.bgx_attention_backward(shape, *args, rows_of(out[0]), P(saved), rows_of(do),
                                              *(rows_of(t) for t in out[1:]), P(ws), ws.numel(), stream), "backward")
        results.append(out)
    for a, b in zip(*results):
        assert torch.equal(a, b)
    _check_sequences(q, k, v, do, results[0][0], results[0][1:], list(zip(cu, cu[1:])), 0.125, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("N,heads,kv_heads", [(34, 8, 4), (140, 8, 4)], ids=str)
def test_attention_sizes_by_rule(device, N, heads, kv_heads, dtype):
    """Enough sequences and heads that the workgroup sizes follow from the rule: 64 rows in the first case, 128 in the
    second, where a workgroup also sums dk and dv over the heads that share its keys; heads of 128 and 64."""
    g = _gen(N)
    for dim in (128, 64):
        lengths = torch.randint(0, 160, (N,), generator=g).tolist()
        T = sum(lengths)
        q, k, v, do = _qkv((T,), heads, kv_heads, dim, dtype, N + dim, device)
        cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(device)
        for t in (q, k, v):
            t.requires_grad_()
        out = B.causal_attention(q, k, v, cu_seqlens=cu)
        grads = torch.autograd.grad(out, (q, k, v), do)
        ends = cu.tolist()
        _check_sequences(q, k, v, do, out, grads, list(zip(ends, ends[1:])), dim ** -0.5, dtype)


def test_attention_empty_inputs(device):
    for shape, kw in (((0, 2, 32), dict(cu_seqlens=torch.zeros(1, dtype=torch.int32, device=device))),
                      ((0, 5, 2, 32), {}), ((3, 0, 2, 32), {})):
        q = torch.zeros(shape, device=device, requires_grad=True)
        out = B.causal_attention(q, q, q, **kw)
        assert out.shape == shape
        assert torch.autograd.grad(out.sum(), q)[0].shape == shape
    q = torch.randn(5, 2, 32, device=device, requires_grad=True)   # rows, but no sequence
    out = B.causal_attention(q, q, q, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=device))
    assert (out == 0).all() and (torch.autograd.grad(out.sum(), q)[0] == 0).all()


# ---- distillation -------------------------------------------------------------------------------------------------

def _distill_case(rows, V, K, dtype, seed, device, t_dtype=None):
    g = _gen(seed)
    z = 2.5 * torch.randn(rows, V, generator=g)
    top = torch.topk(z + torch.randn(rows, V, generator=g), K, dim=1)
    grad = torch.rand(rows, generator=g) + 0.5
    return z.to(dtype).to(device), top.indices.to(device), top.values.to(t_dtype or dtype).to(device), grad.to(device)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("rows,V,K,tau", [(1, 1, 1, 1.0), (3, 7, 2, 2.0), (5, 1000, 1, 1.0), (4, 2049, 300, 0.5),
                                          (33, 511, 64, 3.0), (2, 50257, 8, 1.0), (2, 5000, 1024, 1.0)], ids=str)
def test_distillation(device, rows, V, K, tau, dtype):
    z, ids, t, grad = _distill_case(rows, V, K, dtype, V + K, device)
    z.requires_grad_()
    loss = B.topk_distillation(z, ids, t, temperature=tau)
    dz, = torch.autograd.grad(loss, z, grad)
    ref = distill_reference(z, ids, t, tau, None, grad, dtype)
    assert loss.dtype == torch.float32 and dz.dtype == dtype
    assert_within(loss, *ref["loss"], "loss")
    assert_within(dz, *ref["dz"], "dz")
    with torch.no_grad():
        assert torch.equal(B.topk_distillation(z, ids, t, temperature=tau), loss)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_distillation_entries(device, dtype):
    """Missing entries, the same id twice, ids past the vocabulary, tokens without entries, excluded tokens with NaN
    logits, a teacher entry of -inf."""
    z, ids, t, grad = _distill_case(7, 300, 6, dtype, 5, device, torch.float32)
    ids[0, 3:] = -1
    ids[1, 4] = ids[1, 0]
    ids[1, 5] = ids[1, 0]
    ids[2, 0], ids[2, 1] = 300, 1 << 40
    ids[3] = -1
    t[4, 2] = float("-inf")
    t[6] = float("-inf")
    valid = torch.tensor([True, True, True, True, True, False, True], device=device)
    z[3] = float("nan")
    z[5] = float("inf")
    z.requires_grad_()
    loss = B.topk_distillation(z, ids, t, temperature=1.5, valid=valid)
    dz, = torch.autograd.grad(loss, z, grad)
    ref = distill_reference(z, ids, t, 1.5, valid, grad, dtype)
    assert_within(loss, *ref["loss"], "loss")
    assert_within(dz, *ref["dz"], "dz")
    assert (loss[[3, 5, 6]] == 0).all() and (dz[[3, 5, 6]] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
@pytest.mark.parametrize("K,distinct", [(600, 1), (600, 40), (600, 500), (9, 2), (1024, 1000)], ids=str)
def test_distillation_repeated_entries(device, dtype, K, distinct):
    """Ids that come a few times, many times, all the same: their probabilities add up, with the same bits every time."""
    z, _, _, grad = _distill_case(3, 2000, 1, dtype, 4, device)
    g = _gen(K + distinct)
    ids = (torch.randint(0, distinct, (3, K), generator=g) * 1024 % 2000).to(device)   # the low bits alike, too
    t = torch.randn(3, K, generator=g).to(device)
    z.requires_grad_()
    loss = B.topk_distillation(z, ids, t)
    dz, = torch.autograd.grad(loss, z, grad)
    ref = distill_reference(z, ids, t, 1.0, None, grad, dtype)
    assert_within(loss, *ref["loss"], "loss")
    assert_within(dz, *ref["dz"], "dz")
    again, = torch.autograd.grad(B.topk_distillation(z, ids, t), z, grad)
    assert torch.equal(dz, again)


def test_distillation_infinite_logits(device):
    """A vocabulary masked with -inf: those entries have no mass and no gradient; a teacher entry among them makes its
    token's loss infinite and leaves the others alone.  NaN stays in its token."""
    z, ids, t, grad = _distill_case(4, 200, 3, torch.float32, 9, device)
    keep = torch.zeros(4, 200, dtype=torch.bool, device=device).scatter_(1, ids, True)
    keep |= torch.rand(4, 200, generator=_gen(1)).to(device) > 0.5
    z[~keep] = float("-inf")
    z[1, ids[1, 0]] = float("-inf")
    z[2, 11] = float("nan")
    z.requires_grad_()
    loss = B.topk_distillation(z, ids, t)
    dz, = torch.autograd.grad(loss, z, grad)
    assert loss[1] == float("inf") and loss[2].isnan() and dz[2].isnan().any()
    assert (dz[[0, 3]][~keep[[0, 3]]] == 0).all()
    rows = [0, 3]
    ref = distill_reference(z[rows].clamp_min(-1e4), ids[rows], t[rows], 1.0, None, grad[rows], torch.float32)
    assert_within(loss[rows], *ref["loss"], "loss")
    assert_within(dz[rows], *ref["dz"], "dz")


@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_distillation_lowest_logits(device, dtype):
    """A vocabulary masked with the type's lowest value, in part and as a whole: what whole threads see of it leaves the
    numbers when it is scaled."""
    z = torch.full((3, 5001), torch.finfo(dtype).min, dtype=dtype, device=device)
    z[0, 17], z[0, 3000], z[1, 17] = 1.0, 2.0, 1.0
    ids, t = torch.tensor([[17, 3000], [17, -1], [17, 3000]], device=device), torch.ones(3, 2, device=device)
    grad = torch.ones(3, device=device)
    z.requires_grad_()
    loss = B.topk_distillation(z, ids, t)
    dz, = torch.autograd.grad(loss, z, grad)
    ref = distill_reference(z, ids, t, 1.0, None, None, dtype)
    assert_within(loss, *ref["loss"], "loss")
    q = torch.zeros(3, 5001, dtype=torch.float64)
    q[0, 17], q[0, 3000], q[1, 17], q[2] = 1 / (1 + math.e), math.e / (1 + math.e), 1.0, 1 / 5001
    p = torch.zeros_like(q)
    p[0, 17] = p[0, 3000] = p[2, 17] = p[2, 3000] = 0.5
    p[1, 17] = 1.0
    # q to (V / 256 + 48) u, the difference to 4 u of both, the rounding to the type
    bound = (68 * 2.0 ** -24) * q + 2.0 ** -22 * (q + p) + torch.finfo(dtype).eps / 2 * (q - p).abs() + torch.finfo(dtype).tiny
    assert_within(dz, q - p, bound, "dz")


def test_distillation_layouts(device):
    """[N, S, V] views, rows of a wider matrix, an odd offset, int ids that are views: the bits of plain copies."""
    z, ids, t, grad = _distill_case(12, 333, 5, torch.bfloat16, 2, device)
    want_leaf = z.clone().requires_grad_()
    want = B.topk_distillation(want_leaf, ids, t)
    want_dz, = torch.autograd.grad(want, want_leaf, grad)
    wide = torch.zeros(12, 400, dtype=z.dtype, device=device)
    wide[:, 5:338] = z
    for view in (wide[:, 5:338], z.t().contiguous().t()):
        leaf = view.detach().requires_grad_()
        loss = B.topk_distillation(leaf, ids.t().contiguous().t(), t)
        assert torch.equal(loss, want)
        assert torch.equal(torch.autograd.grad(loss, leaf, grad)[0], want_dz)
    leaf = z.reshape(3, 4, 333).clone().requires_grad_()
    loss = B.topk_distillation(leaf, ids.reshape(3, 4, 5), t.reshape(3, 4, 5))
    assert loss.shape == (3, 4) and torch.equal(loss.flatten(), want)
    assert torch.equal(torch.autograd.grad(loss.sum(), leaf)[0].reshape(12, 333),
                       torch.autograd.grad(B.topk_distillation(want_leaf, ids, t).sum(), want_leaf)[0])
    empty = torch.zeros(0, 333, device=device, requires_grad=True)
    loss = B.topk_distillation(empty, ids[:0], t[:0])
    assert loss.shape == (0,) and torch.autograd.grad(loss.sum(), empty)[0].shape == (0, 333)


# ---- all of them --------------------------------------------------------------------------------------------------

def _calls(device):
    """(function of leaves, leaves, output gradient) of each operator at a size of a few tiles."""
    x, w, b, dy = _norm_case(300, 768, torch.bfloat16, torch.bfloat16, 1, device)
    q, k, v, do = _qkv((500,), 4, 2, 64, torch.float16, 2, device)
    cu = torch.tensor([0, 130, 131, 420], dtype=torch.int32, device=device)
    z, ids, t, g = _distill_case(40, 3001, 16, torch.bfloat16, 3, device)
    return {"norm": (lambda *a: B.layer_norm(*a), (x, w, b), dy),
            "attention": (lambda *a: B.causal_attention(*a, cu_seqlens=cu), (q, k, v), do),
            "distill": (lambda a: B.topk_distillation(a, ids, t), (z,), g)}


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_same_bits_every_time(device, which):
    fn, leaves, grad = _calls(device)[which]
    leaves = [t.requires_grad_() for t in leaves]
    first = None
    for _ in range(3):
        out = fn(*leaves)
        res = (out, *torch.autograd.grad(out, leaves, grad))
        if first is None:
            first = res
        assert all(torch.equal(a, b) for a, b in zip(first, res))


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_captured_and_replayed(device, which):
    """Forward and backward in one graph, new values in the same leaves, eager work between the replays."""
    fn, leaves, grad = _calls(device)[which]
    static = [t.clone().requires_grad_() for t in leaves]

    def step(args):
        out = fn(*args)
        return (out.detach(), *torch.autograd.grad(out, args, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for i in range(4):
        fresh = [(t.float() * (1 + 0.1 * i)).to(t.dtype) for t in leaves]
        with torch.no_grad():
            for s, f in zip(static, fresh):
                s.copy_(f)
        graph.replay()
        want = step([f.requires_grad_() for f in fresh])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_on_another_stream(device, which):
    fn, leaves, grad = _calls(device)[which]
    leaves = [t.requires_grad_() for t in leaves]
    out = fn(*leaves)
    want = (out, *torch.autograd.grad(out, leaves, grad))
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:      # two calls in flight at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out = fn(*leaves)
            results.append((out, *torch.autograd.grad(out, leaves, grad)))
    torch.cuda.synchronize()
    for res in results:
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_two_graphs_of_the_same_calls(device):
    """Two captured graphs of all three operators, replayed in turn: neither holds anything of the other."""
    calls = _calls(device)
    results = []
    for factor in (1.0, 0.5):
        args = {n: ([(t.float() * factor).to(t.dtype).requires_grad_() for t in leaves], grad)
                for n, (_, leaves, grad) in calls.items()}

        def step():
            out = []
            for n, (leaves, grad) in args.items():
                y = calls[n][0](*leaves)
                out += [y.detach(), *torch.autograd.grad(y, leaves, grad)]
            return out

        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        results.append((graph, captured, want, args))
    for _ in range(3):
        for graph, _, _, _ in results:
            graph.replay()
        torch.cuda.synchronize()
        for _, captured, want, _ in results:
            assert all(torch.equal(a, b) for a, b in zip(captured, want))
            for t in captured:
                t.zero_()


def test_calls_from_several_threads(device):
    """Forward and backward passes of all operators from four threads, each on a stream of its own."""
    calls = _calls(device)
    run = lambda leaves: [r for n, (fn, _, grad) in calls.items()
                          for y in [fn(*leaves[n])] for r in (y.detach(), *torch.autograd.grad(y, leaves[n], grad))]
    fresh = lambda: {n: [t.detach().clone().requires_grad_() for t in leaves] for n, (_, leaves, _) in calls.items()}
    want, got = run(fresh()), {}
    inputs = [fresh() for _ in range(4)]
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(inputs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want))


def test_gradients_against_differences(device):
    """Directional derivatives of a scalar of each operator's fp32 output against central differences of the
    operator's definition in 64 bits: the difference quotient is off by O(step^2), the kernel by its fp32 bounds."""
    g = _gen(21)
    x, w, b, dy = _norm_case(4, 50, torch.float32, torch.float32, 7, device)
    q, k, v, do = _qkv((70,), 2, 1, 16, torch.float32, 7, device)
    z, ids, t, gr = _distill_case(3, 90, 4, torch.float32, 7, device)
    cu = torch.tensor([0, 70], dtype=torch.int32, device=device)
    cases = [
        (lambda *a: B.layer_norm(*a), (x, w, b), dy,
         lambda x, w, b: norm_reference(x, w, b, 1e-5, None, torch.float32, torch.float32)["y"][0]),
        (lambda *a: B.causal_attention(*a, cu_seqlens=cu), (q, k, v), do,
         lambda q, k, v: attention_reference(q, k, v, 0.25, None, torch.float32)["o"][0]),
        (lambda a: B.topk_distillation(a, ids, t), (z,), gr,
         lambda z: distill_reference(z, ids, t, 1.0, None, None, torch.float32)["loss"][0]),
    ]
    for fn, leaves, grad, definition in cases:
        leaves = [l.requires_grad_() for l in leaves]
        grads = torch.autograd.grad(fn(*leaves), leaves, grad)
        point = [l.detach().cpu().double() for l in leaves]
        weight = grad.detach().cpu().double()
        for i, gi in enumerate(grads):
            direction = torch.randn(point[i].shape, generator=g, dtype=torch.float64)
            step = 1e-5
            ends = []
            for sign in (1, -1):
                moved = [p + sign * step * direction if j == i else p for j, p in enumerate(point)]
                ends.append((definition(*moved) * weight).sum())
            slope = (ends[0] - ends[1]) / (2 * step)
            got = (gi.detach().cpu().double() * direction).sum()
            size = (gi.detach().cpu().double() * direction).abs().sum()
            # quotient: third derivatives times step^2 (1e-10) and 64-bit cancellation 1e-16 / 1e-5; kernel: fp32
            # sums of up to a hundred terms, 2^-24 each
            assert (got - slope).abs() <= 1e-5 * size + 1e-7, (i, got, slope)


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_differentiable_once(device, which):
    fn, leaves, grad = _calls(device)[which]
    leaves = [t.requires_grad_() for t in leaves]
    want = torch.autograd.grad(fn(*leaves), leaves, grad)
    got = torch.autograd.grad(fn(*leaves), leaves, grad, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="differentiable once"):
        got[0].float().sum().backward()


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_saved_tensors_may_travel(device, which):
    """What a forward pass saves may be packed away and brought back by saved-tensor hooks."""
    fn, leaves, grad = _calls(device)[which]
    leaves = [t.requires_grad_() for t in leaves]
    want = torch.autograd.grad(fn(*leaves), leaves, grad)
    with torch.autograd.graph.save_on_cpu():
        out = fn(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, grad), want))


@pytest.mark.parametrize("which", ["norm", "attention", "distill"])
def test_transforms_are_refused(device, which):
    """torch.func's vmap and grad hand over tensors without memory of their own: an error, and nothing is launched."""
    fn, leaves, grad = _calls(device)[which]
    with pytest.raises(RuntimeError):
        torch.func.vmap(fn)(*(torch.stack([t, t]) for t in leaves))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda *a: fn(*a).float().sum())(*leaves)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(fn, tuple(leaves), tuple(torch.ones_like(t) for t in leaves))
    torch.cuda.synchronize()


@pytest.mark.parametrize("rows", [128, 64, 32])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids_of)
def test_attention_gradients_that_cancel(device, bgx_env, dtype, rows):
    """Sequences of one token: the softmax is constant, dq and dk are exactly 0 and dv is the sum over the heads,
    times a weight of 1."""
    bgx_env("BGX_ATTENTION_ROWS", rows)
    q, k, v, do = _qkv((40,), 4, 2, 64, dtype, 30, device)
    cu = torch.arange(41, dtype=torch.int32, device=device)
    for t in (q, k, v):
        t.requires_grad_()
    dq, dk, dv = torch.autograd.grad(B.causal_attention(q, k, v, cu_seqlens=cu), (q, k, v), do)
    assert (dq == 0).all() and (dk == 0).all()
    # the weight is 2^(s c - fl(s c)): off from 1 by the rounding of s c (c = scale log2 e) and of the exponential
    wide = [t.detach().double().cpu() for t in (q, k.repeat_interleave(2, 1), do)]
    score = (wide[0] * wide[1]).sum(2, keepdim=True).abs() * 0.125 * 1.4427
    off = ((score + 4) * 2.0 ** -24 * wide[2].abs()).unflatten(1, (2, 2)).sum(2)
    want = wide[2].unflatten(1, (2, 2)).sum(2)
    assert_within(dv, want, off + torch.finfo(dtype).eps / 2 * (want.abs() + off), "dv")
