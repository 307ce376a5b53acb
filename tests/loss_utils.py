"""Definitions in 64 bits of the soft assignment and of the losses over it, on the CPU, with bounds on what fp32 kernels
may be off by.  u = 2^-24 is the largest relative rounding error of one fp32 operation; a result stored as type t is off by at
most eps(t) / 2 more.

softmax: exp_scaled rounds the difference to the maximum (u |d|), its product (u |d| again, d over the temperature) and the
result (2 u); every term of the row's sum has such an error, and on average over p the differences are at most
log E; a sum of E terms over 64 lanes or more adds at most E / 64 + 16 roundings.  So p is off by a factor of at most
u (2 |d| + 2 log E + E / 64 + 24), beside results below 2^-126, which may be 0."""
import math

import torch

U = 2.0 ** -24
TINY = 2.0 ** -125


def store_error(value, dtype):
    """Rounding of ``value`` to ``dtype``: half a step, subnormal results by half the smallest."""
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def softmax64(x, t=1.0):
    """float64 [n, E] -> p (0 in rows without a finite value), relative error bound of p, distance to the maximum over t,
    log of the sum."""
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    d = (x - m) / t
    e = torch.exp(d)
    total = e.sum(dim=1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    dist = torch.where(p > 0, -d, torch.zeros_like(d))
    size = x.shape[1]
    rel = U * (2 * dist + 2 * math.log(size) + size / 64 + 24)
    return p, rel, d, torch.log(total[:, 0])


def balance64(logits, idx, mask=None, scale=1.0):
    """-> (loss, counts, mean_prob, grad, bounds of loss, mean_prob and grad before it is stored)"""
    n, e = logits.shape
    x = logits.double().cpu()
    idx = idx.cpu().long()
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask.cpu().bool()
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    p, rel, _, _ = softmax64(x) if n else (x, x, x, x)
    p = torch.where(keep[:, None], p, torch.zeros_like(p))
    chosen = idx[keep].reshape(-1)
    chosen = chosen[(chosen >= 0) & (chosen < e)]
    counts = torch.bincount(chosen, minlength=e)
    rows = int(keep.sum())
    f = counts.double() / max(1, len(chosen))
    mean_prob = p.sum(dim=0) / max(1, rows)
    loss = e * (f * mean_prob).sum()
    dot = (p * f).sum(dim=1, keepdim=True)
    factor = scale * e / rows if rows else 0.0
    grad = factor * p * (f - dot)
    # adding up the rows: at most n / 256 + 40 roundings behind one another
    mean_bound = (p * rel).sum(dim=0) / max(1, rows) + mean_prob * U * (n / 256 + 40) + TINY
    loss_bound = e * (f * mean_bound).sum() + loss * 4 * U
    size = U * (e / 64 + 24)
    dot_bound = (p * f * rel).sum(dim=1, keepdim=True) + dot * size
    grad_bound = abs(factor) * (p * rel * (f - dot).abs() + p * (dot_bound + (f + dot) * 4 * U)) + grad.abs() * 4 * U + abs(factor) * TINY
    return loss, counts, mean_prob, grad, loss_bound, mean_bound, grad_bound


def distill64(logits, t_logits, t_idx, mask=None, t=1.0, scale=1.0):
    """-> (loss, row_loss, grad, bounds of loss, row_loss and grad before it is stored)"""
    n, v = logits.shape
    x, tl, idx = logits.double().cpu(), t_logits.double().cpu(), t_idx.cpu().long()
    keep = torch.ones(n, dtype=torch.bool) if mask is None else mask.cpu().bool()
    x = torch.where(keep[:, None], x, torch.zeros_like(x))
    there = (idx >= 0) & (idx < v)
    tl = torch.where(there & keep[:, None], tl, torch.full_like(tl, -math.inf))
    col = torch.where(there, idx, torch.zeros_like(idx))
    if n == 0:
        z = torch.zeros(0, dtype=torch.float64)
        return z.sum(), z, x, z.sum(), z, x
    p, relp, d, logl = softmax64(x, t)
    q, relq, dt, logtl = softmax64(tl, t)
    live = keep & (p.sum(dim=1) > 0) & (q.sum(dim=1) > 0)
    ds = d.gather(1, col)
    terms = torch.where(q > 0, q * (dt - ds), torch.zeros_like(q))
    row = torch.where(live, t * t * (terms.sum(dim=1) + logl - logtl), torch.zeros(n, dtype=torch.float64))
    rows = int(keep.sum())
    loss = row.sum() / max(1, rows)
    big_q = torch.zeros_like(x).scatter_add_(1, col, q)
    relq_sum = torch.zeros_like(x).scatter_add_(1, col, q * relq)
    factor = scale * t / rows if rows else 0.0
    grad = torch.where(live[:, None], factor * (p - big_q), torch.zeros_like(x))
    mag = torch.where(q > 0, q * (dt.abs() + ds.abs()), torch.zeros_like(q))
    k = t_idx.shape[1]
    size_v, size_k = U * (2 * math.log(v) + v / 64 + 24), U * (2 * math.log(k) + k / 64 + 24)
    row_bound = t * t * ((mag * (relq + 6 * U)).sum(dim=1) + mag.sum(dim=1) * size_k + size_v + size_k + 4 * U * (logl.abs() + logtl.abs()))
    row_bound = torch.where(live, row_bound + row.abs() * 4 * U, torch.zeros_like(row))
    loss_bound = row_bound.sum() / max(1, rows) + loss.abs() * 4 * U
    grad_bound = abs(factor) * (p * relp + relq_sum + big_q * size_k + (p + big_q) * 6 * U + TINY)
    grad_bound = torch.where(live[:, None], grad_bound, torch.zeros_like(grad_bound))
    return loss, row, grad, loss_bound, row_bound, grad_bound


def code_logits64(x, code, t, g=None):
    """-> (logits, bound) or, with g, (dx, bound, dcode, bound) before they are stored: a sum of m products is off by at
    most (m + 4) u times the sum of their magnitudes."""
    x, code = x.double().cpu(), code.double().cpu()
    if g is None:
        s = (2 * x @ code.t() - (code * code).sum(dim=1)) / t
        mag = (2 * x.abs() @ code.abs().t() + (code * code).sum(dim=1)) / t
        return s, mag * (x.shape[1] + 4) * U
    g = g.double().cpu()
    dx = 2 / t * (g @ code)
    dx_bound = 2 / t * (g.abs() @ code.abs()) * (code.shape[0] + 4) * U
    dc = 2 / t * (g.t() @ x - g.sum(dim=0)[:, None] * code)
    dc_bound = 2 / t * (g.abs().t() @ x.abs() + g.abs().sum(dim=0)[:, None] * code.abs()) * (x.shape[0] + 8) * U
    return dx, dx_bound, dc, dc_bound


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound everywhere (NaN and infinities have to be the same)."""
    got = got.detach().double().cpu()
    want = want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    err = torch.where(same, torch.zeros_like(want), (got - want).abs())
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound).nan_to_num(nan=math.inf).max()):.3g} of the bound"
