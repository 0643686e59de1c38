"""64-bit definitions of the language-model operators, and bounds on what 32-bit arithmetic may add.

Each `*_bound` gives, per element, how far a computation in 32 bits can be from the exact value: every operation
is off by at most half a step, U = 2^-24 relative to its result, and a sum whose longest chain of additions has k
links by at most k U times the sum of the magnitudes.  `store` adds the one rounding to the output's type.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def store(bound, exact, dtype):
    """The bound after a rounding to dtype: at most half a step, or half the smallest subnormal; 32-bit products and
    exponentials below the smallest normal number may be flushed to zero."""
    f = torch.finfo(dtype)
    half = 0.0 if dtype == torch.float32 else f.eps / 2
    return bound + half * (exact.abs() + bound) + f.smallest_normal * f.eps + 2.0 ** -125


# ---- layer norm ---------------------------------------------------------------------------------------------
def layer_norm(x, weight, bias, eps):
    x = x.double()
    mean = x.mean(-1)
    invstd = 1 / (((x - mean[..., None]) ** 2).mean(-1) + eps).sqrt()
    y = (x - mean[..., None]) * invstd[..., None]
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y, mean, invstd


def layer_norm_bound(x, weight, bias, eps, links=64):
    """(y, mean, invstd).  The mean is off by links U max|x|; the sum of squares around it by as many links and, to
    second order only, by the mean's error; the root and the quotient add 4 U."""
    y, mean, invstd = layer_norm(x, weight, bias, eps)
    x = x.double()
    top = x.abs().amax(-1)
    dmean = (links + 2) * U * top
    drel = (links + 8) * U + (dmean * invstd) ** 2
    w = weight.double().abs() if weight is not None else torch.ones((), dtype=torch.float64, device=x.device)
    xh = ((x - mean[..., None]) * invstd[..., None]).abs()
    b = bias.double().abs() if bias is not None else 0.0
    dy = w * (invstd * dmean)[..., None] + w * xh * (drel[..., None] + 4 * U) + 2 * U * (b + y.abs())
    return dy, dmean, drel * invstd


def layer_norm_backward(x, grad_out, mean, invstd, weight):
    x, dy, r = x.double(), grad_out.double(), invstd.double()[..., None]
    xh = (x - mean.double()[..., None]) * r
    g = dy if weight is None else dy * weight.double()
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    D = x.shape[-1]
    return dx, (dy * xh).reshape(-1, D).sum(0), dy.reshape(-1, D).sum(0)


def layer_norm_backward_bound(x, grad_out, mean, invstd, weight, links=64, row_links=512):
    x, dy, r = x.double(), grad_out.double(), invstd.double()[..., None]
    xh = ((x - mean.double()[..., None]) * r).abs()
    g = (dy if weight is None else dy * weight.double()).abs()
    dx = (links + 12) * U * r * (g + g.mean(-1, keepdim=True) + xh * (g * xh).mean(-1, keepdim=True))
    D = x.shape[-1]
    return dx, (row_links + 4) * U * (dy.abs() * xh).reshape(-1, D).sum(0), row_links * U * dy.abs().reshape(-1, D).sum(0)


# ---- embedding ----------------------------------------------------------------------------------------------
def embedding(table, ids, scale):
    ok = (ids >= 0) & (ids < table.shape[0])
    out = table.double()[ids.long().clamp(0, table.shape[0] - 1)] * scale
    return torch.where(ok[..., None], out, torch.zeros((), dtype=torch.float64, device=out.device))


def embedding_backward(grad_out, ids, rows, scale, padding_id=-1):
    D = grad_out.shape[-1]
    g, i = grad_out.double().reshape(-1, D), ids.long().reshape(-1)
    keep = (i >= 0) & (i < rows) & (i != padding_id)
    out = torch.zeros(rows, D, dtype=torch.float64, device=g.device)
    return out.index_add_(0, i[keep], g[keep]) * scale


def embedding_backward_bound(grad_out, ids, rows, scale, padding_id=-1):
    """A sum of c rows in any order has at most c - 1 links; one more rounding for the scale."""
    mag = embedding_backward(grad_out.abs(), ids, rows, abs(scale), padding_id)
    i = ids.long().reshape(-1)
    keep = (i >= 0) & (i < rows) & (i != padding_id)
    count = torch.bincount(i[keep], minlength=rows)
    return (count[:, None] + 2) * U * mag


# ---- gated recurrence -----------------------------------------------------------------------------------------
def gated_recurrence(gate, x, h0=None):
    """(h [B, T, D], the states before each step [B, T, D], the last state)"""
    g, x = gate.double(), x.double()
    a, z = torch.sigmoid(g), torch.sigmoid(-g)
    h = torch.zeros_like(x[:, 0]) if h0 is None else h0.double()
    out, before = [], []
    for t in range(x.shape[1]):
        before.append(h)
        h = torch.where(a[:, t] == 0, torch.zeros_like(h), a[:, t] * h) + torch.where(z[:, t] == 0, torch.zeros_like(h), z[:, t] * x[:, t])
        out.append(h)
    return torch.stack(out, 1), torch.stack(before, 1), h


def _links(gate):
    """Roundings of one step in units of U: the exponential is off by about (4 + |gate|) U (its argument's rounding
    counts with its size), sum, reciprocal, two products, one addition, and as much again for joining the
    pieces of a scan that was cut: a product of n factors is off by n of these, as n steps are."""
    return 2 * (10 + gate.double().abs().clamp(max=104.0))


def gated_recurrence_bound(gate, x, h0=None):
    """Running error: a step keeps a_t of the earlier one and adds its own roundings."""
    a, z = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    h, before, _ = gated_recurrence(gate, x, h0)
    c = _links(gate) * U
    e = torch.zeros_like(h[:, 0])
    out, prev = [], []
    for t in range(h.shape[1]):
        prev.append(e)
        e = a[:, t] * e + c[:, t] * (a[:, t] * before[:, t].abs() + z[:, t] * x[:, t].double().abs())
        out.append(e)
    return torch.stack(out, 1), torch.stack(prev, 1), e


def gated_recurrence_backward(gate, x, h0, grad_out, grad_last=None):
    g, x, dy = gate.double(), x.double(), grad_out.double()
    a, z = torch.sigmoid(g), torch.sigmoid(-g)
    _, before, _ = gated_recurrence(gate, x, h0)
    e = torch.zeros_like(x[:, 0]) if grad_last is None else grad_last.double()
    dg, dx, sens = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[1] - 1, -1, -1):
        e = e + dy[:, t]
        sens[:, t] = e
        dx[:, t] = e * z[:, t]
        dg[:, t] = e * (before[:, t] - x[:, t]) * a[:, t] * z[:, t]
        e = e * a[:, t]
    return dg, dx, e, sens


def gated_recurrence_backward_bound(gate, x, h0, grad_out, grad_last=None):
    a, z = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    dg, dx, dh0, sens = gated_recurrence_backward(gate, x, h0, grad_out, grad_last)
    _, before, _ = gated_recurrence(gate, x, h0)
    _, dbefore, _ = gated_recurrence_bound(gate, x, h0)
    c, xd, dy = _links(gate) * U, x.double(), grad_out.double().abs()
    f = torch.zeros_like(dh0)                    # error of what arrives from the later step
    later = torch.zeros_like(dh0) if grad_last is None else grad_last.double().abs()
    bg, bx = torch.empty_like(dg), torch.empty_like(dx)
    for t in range(dg.shape[1] - 1, -1, -1):
        f = f + 2 * U * (dy[:, t] + later)
        s = sens[:, t].abs()
        bx[:, t] = z[:, t] * (f + c[:, t] * s)
        diff = (before[:, t] - xd[:, t]).abs()
        bg[:, t] = a[:, t] * z[:, t] * (diff * f + s * (dbefore[:, t] + 2 * U * (before[:, t].abs() + xd[:, t].abs())) + 2 * c[:, t] * s * diff)
        f = a[:, t] * (f + c[:, t] * s)
        later = a[:, t] * s
    return bg, bx, f
