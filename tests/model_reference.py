"""The model operators' definitions in 64 bits, each with an elementwise bound on what the kernels' arithmetic may be
off by.  The bounds are sums of first-order terms, from

  h   half a step of the outputs' type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), relative to the value, for every
      rounding to that type (inputs are exact),
  u   2^-24: half a step of fp32, for every fp32 operation; a sum of n terms costs at most n u of the sum of their
      magnitudes (the kernels' trees cost less), the hardware's exp2 and log2 at most 2 u.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Absolute error of a rounding among the subnormals."""
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2 if dtype == torch.float16 else f.tiny


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} against {tuple(want.shape)}"
    over = (got - want).abs() - bound
    bad = ~(over <= 0)
    if bad.any():
        i = int(torch.where(bad, torch.nan_to_num(over, nan=float("inf")), -1.0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; worst at {i}: got "
                             f"{got.flatten()[i]} want {want.flatten()[i]} bound {bound.flatten()[i]}")


def norm_reference(x, weight, bias, eps, dy, out_dtype, w_dtype):
    """{name: (value, bound)} of y, dx, dw, db."""
    h, hw = half_step(out_dtype), half_step(w_dtype)
    x, w = x.detach().cpu().double(), weight.detach().cpu().double()
    b = torch.zeros_like(w) if bias is None else bias.detach().cpu().double()
    rows, d = x.shape
    mean = x.mean(1, keepdim=True)
    dev = x - mean
    var = dev.square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = dev * rstd
    # the mean is off by at most n u mean|x| (n terms at the longest lane's sum plus the joins; 16384 / 256 + 16 of
    # them at most, less than 80), a deviation by that and its own rounding; the variance, rstd by the relative errors
    e_mean = 80 * U * x.abs().mean(1, keepdim=True)
    e_dev = e_mean + 2 * U * dev.abs()
    e_rstd = rstd * (2 * (dev.abs() * e_dev).mean(1, keepdim=True) / 2 / (var + eps) + 44 * U)
    e_xh = e_dev * rstd + dev.abs() * e_rstd + 2 * U * xh.abs()
    y = xh * w + b
    e_y = e_xh * w.abs() + 2 * U * (xh * w).abs() + U * y.abs()
    out = {"y": (y, e_y + h * y.abs() + tiny(out_dtype))}
    if dy is None:
        return out
    dy = dy.detach().cpu().double()
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - m1 - xh * m2)
    e_m1 = 82 * U * g.abs().mean(1, keepdim=True)
    e_m2 = 82 * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    inner = g.abs() + m1.abs() + (xh * m2).abs()
    e_dx = e_rstd * inner + rstd * (e_m1 + xh.abs() * e_m2 + e_xh * m2.abs() + 5 * U * inner)
    out["dx"] = (dx, e_dx + h * dx.abs() + tiny(out_dtype))
    # a column is summed over the rows of a wave, the workgroup's waves and the workgroups: at most rows + 40 terms
    n = rows + 40
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = (dy.abs() * e_xh).sum(0) + n * U * (dy * xh).abs().sum(0)
    out["dw"] = (dw, e_dw + hw * dw.abs() + tiny(w_dtype))
    out["db"] = (db, n * U * dy.abs().sum(0) + hw * db.abs() + tiny(w_dtype))
    return out


def attention_reference(q, k, v, scale, do, dtype, ds_floor=None):
    """One sequence, q [L, H, D], k and v [L, Hk, D] -> {name: (value, bound)} of o and, with do, dq, dk, dv.
    ds_floor: what dS in fp16 may lose beside its relative rounding, in units of the largest |dp - delta| of its row
    (dq) or sequence (dk); by default a multiple of the largest |do|."""
    h = half_step(dtype)
    q, k, v = (t.detach().cpu().double().transpose(0, 1) for t in (q, k, v))
    group = q.shape[0] // k.shape[0]
    kq, vq = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    L, D = q.shape[1:]
    past = torch.ones(L, L, dtype=torch.bool).tril()
    s = (q @ kq.transpose(1, 2)) * scale
    p = torch.softmax(s.masked_fill(~past, float("-inf")), dim=2)
    # a score: D products and the factor; the exponent's argument carries the row's statistics too (a maximum, an
    # fp32 logarithm of the sum), of the size of the largest score; the sum over L keys in fp32
    e_s = (D + 4) * U * (q.abs() @ kq.abs().transpose(1, 2)) * scale
    size = torch.where(past, s.abs() + e_s, 0.0).amax(2, keepdim=True)
    e_row = torch.where(past, e_s, 0.0).amax(2, keepdim=True) + 6 * U * (size + 16) + (L + 8) * U
    rel_p = e_s + e_row                      # relative error of a probability before its rounding to the type
    o = p @ vq
    e_o = (p * (rel_p + h + (L + 8) * U)) @ vq.abs() + (e_row + 4 * U) * o.abs() + h * o.abs() + tiny(dtype)
    # probabilities below the smallest normal number: fp16 rounds them to multiples of 2^-24, the others' exponential
    # (no subnormal results) and matrix operands become 0 below 2^-126; each key may lose that much
    e_o = e_o + tiny(dtype) * vq.abs().sum(1, keepdim=True)
    out = {"o": (o.transpose(0, 1), e_o.transpose(0, 1))}
    if do is None:
        return out
    do = do.detach().cpu().double().transpose(0, 1)
    dp, delta = do @ vq.transpose(1, 2), (do * o).sum(2, keepdim=True)
    e_dp = (D + 4) * U * (do.abs() @ vq.abs().transpose(1, 2) + (do * o).abs().sum(2, keepdim=True))
    e_delta = (do.abs() * e_o).sum(2, keepdim=True)
    ds = p * (dp - delta)
    e_ds = (rel_p + h + 4 * U) * ds.abs() + p * (e_dp + e_delta)
    # the same loss of a probability below 2^-126, times dp - delta, and of dS itself
    e_ds = e_ds + torch.where(past, torch.finfo(torch.float32).tiny * ((dp - delta).abs() + 1), 0.0)
    row_floor = floor = 0.0
    if dtype == torch.float16:
        # dS is rounded as a multiple of 2^-24 times the power of two nearest below the tile's largest |do|
        row_floor = floor = tiny(dtype) * 2 * do.abs().amax()
        if ds_floor is not None:
            gap = torch.where(past, (dp - delta).abs(), 0.0)
            row_floor, floor = ds_floor * gap.amax(2, keepdim=True), ds_floor * gap.amax()
    e_ds_q, e_ds_k = (e_ds + torch.where(past, f, 0.0) for f in (row_floor, floor))
    absq, absk = q.abs(), kq.abs()
    dq, e_dq = ds @ kq * scale, (e_ds_q + (L + 8) * U * ds.abs()) @ absk * scale
    dk, e_dk = ds.transpose(1, 2) @ q * scale, (e_ds_k + (group * L + 8) * U * ds.abs()).transpose(1, 2) @ absq * scale
    e_p = p * (rel_p + h + (group * L + 8) * U) + torch.where(past, tiny(dtype), 0.0)
    dv, e_dv = p.transpose(1, 2) @ do, e_p.transpose(1, 2) @ do.abs()
    fold = lambda t: t.unflatten(0, (-1, group)).sum(1)
    dk, e_dk, dv, e_dv = fold(dk), fold(e_dk), fold(dv), fold(e_dv)
    for name, value, e in (("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv)):
        out[name] = (value.transpose(0, 1), (e * (1 + h) + h * value.abs() + tiny(dtype)).transpose(0, 1))
    return out


def distill_reference(z, ids, teacher, tau, valid, grad, dtype):
    """{"loss": ..., "dz": ...}; rows without entries 0."""
    h = half_step(dtype)
    z, t = z.detach().cpu().double(), teacher.detach().cpu().double()
    ids = ids.cpu()
    V, K = z.shape[1], ids.shape[1]
    entry = (ids >= 0) & (ids < V)
    t = t.masked_fill(~entry, float("-inf"))
    used = (t > float("-inf")).any(1)
    if valid is not None:
        used &= valid.cpu()
    z, t = torch.where(used[:, None], z, 0.0), torch.where(used[:, None], t, 0.0)
    safe = ids.clamp(0, V - 1)
    log_q = torch.log_softmax(z / tau, 1)
    log_p = torch.log_softmax(t / tau, 1)
    p = log_p.exp()
    gap = torch.where(p > 0, log_p - log_q.gather(1, safe), 0.0)
    loss = tau ** 2 * (p * gap).sum(1)
    # exponents z - max carry 3 u of their size; the sums over V (K) terms add V / 256 + 40 u (K / 256 + 40 u)
    far = (z.amax(1, keepdim=True) - z) / tau
    e_sum = (V / 256 + 40) * U
    rel_q = 4 * U * far + e_sum
    finite_t = torch.where(p > 0, t, 0.0)
    spread = torch.where(p > 0, (t.amax(1, keepdim=True) - finite_t) / tau, 0.0)
    rel_p = 4 * U * spread + (K / 256 + 48) * U
    far_k = far.gather(1, safe)
    logs = torch.where(p > 0, spread + far_k + torch.log(torch.tensor(float(V))) + 8, 0.0)
    e_loss = tau ** 2 * (p * (rel_p * gap.abs() + 6 * U * logs + e_sum + (K + 8) * U * gap.abs())).sum(1)
    out = {"loss": (torch.where(used, loss, 0.0), torch.where(used, e_loss, 0.0))}
    if grad is None:
        return out
    g = grad.detach().cpu().double()[:, None]
    mass = torch.zeros_like(z).scatter_add_(1, safe, torch.where(entry & used[:, None], p, 0.0))
    e_mass = torch.zeros_like(z).scatter_add_(1, safe, torch.where(entry & used[:, None], p * (rel_p + (K + 4) * U), 0.0))
    dz = g * tau * (log_q.exp() - mass)
    e_dz = g.abs() * tau * (log_q.exp() * (rel_q + 8 * U) + e_mass + 4 * U * (log_q.exp() + mass))
    keep = used[:, None]
    out["dz"] = (torch.where(keep, dz, 0.0), torch.where(keep, e_dz + h * dz.abs() + tiny(dtype), 0.0))
    return out
