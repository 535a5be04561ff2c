"""64-bit references of the dense and state-space operators, token by token
from their formulas, each with the same sum of absolute terms: the size that a
rounding in a sum is relative to."""

from __future__ import annotations

import math

import torch

# half a step of each output type, relative to the value
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}
U = 2.0**-24


def silu(v):
    return v * torch.sigmoid(v)


def softplus(v):
    return torch.logaddexp(v, torch.zeros_like(v))


def act(v, name):
    if name == "relu2":
        return torch.relu(v).square()
    if name == "silu":
        return silu(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    return v


def linear(W, x, bias, name, resid):
    """(out, size): size bounds the out change per unit of relative error of the terms."""
    W, x = W.double(), x.double()
    v, size = x @ W.t(), x.abs() @ W.abs().t()
    if bias is not None:
        v, size = v + bias.double(), size + bias.double().abs()
    out = act(v, name)
    # |act'| <= 1.2 but for relu2, whose slope is 2 relu(v)
    size = size * (2 * torch.relu(v) + 1e-3 * size if name == "relu2" else 1.2) + out.abs()
    if resid is not None:
        out, size = out + resid.double(), size + resid.double().abs()
    return out, size


def conv(x, w, bias, state, cu, slots, has, use_silu=True):
    """(out, size, state) with out NaN where no sequence is."""
    x, w = x.double(), w.double()
    k = w.shape[1]
    out = torch.full_like(x, math.nan)
    size = torch.zeros_like(x)
    new = None if state is None else state.double().clone()
    for i in range(len(cu) - 1):
        slot = slots[i] if slots is not None else i
        kept = new is not None and 0 <= slot < new.shape[0]
        head = new[slot].clone() if kept and has is not None and has[i] else x.new_zeros(k - 1, x.shape[1])
        line = torch.cat([head, x[cu[i]:cu[i + 1]]])
        m = cu[i + 1] - cu[i]
        v = torch.zeros(m, x.shape[1], dtype=torch.float64)
        s = torch.zeros_like(v)
        if bias is not None:
            v, s = v + bias.double(), s + bias.double().abs()
        for j in range(k):
            v = v + line[j:j + m] * w[:, j]
            s = s + (line[j:j + m] * w[:, j]).abs()
        out[cu[i]:cu[i + 1]] = silu(v) if use_silu else v
        size[cu[i]:cu[i + 1]] = s * 1.2 + v.abs()
        if kept:
            new[slot] = line[line.shape[0] - (k - 1):]
    return out, size, new


def scan(x, dt, A, B, C, D, dt_bias, state, cu, slots, has):
    """x [T, H, P], dt [T, H], B, C [T, G, N] -> (y, y size, state, state size); y NaN where no
    sequence is."""
    x, dt, B, C, A = x.double(), dt.double(), B.double(), C.double(), A.double()
    t_all, h, p = x.shape
    rep = h // B.shape[1]
    n = B.shape[2]
    d = softplus(dt + (dt_bias.double() if dt_bias is not None else 0))
    a = torch.exp(d * A)
    Dv = D.double() if D is not None else x.new_zeros(h)
    y = torch.full_like(x, math.nan)
    ys = torch.zeros_like(x)
    new = None if state is None else state.double().clone()
    new_s = None if state is None else state.double().abs()
    for i in range(len(cu) - 1):
        slot = slots[i] if slots is not None else i
        kept = new is not None and 0 <= slot < new.shape[0]
        s = new[slot].clone() if kept and has is not None and has[i] else x.new_zeros(h, p, n)
        m = s.abs()
        for t in range(cu[i], cu[i + 1]):
            b, c = B[t].repeat_interleave(rep, 0), C[t].repeat_interleave(rep, 0)
            add = (d[t, :, None] * x[t])[:, :, None] * b[:, None]
            s = a[t][:, None, None] * s + add
            m = a[t][:, None, None] * m + add.abs()
            y[t] = (s * c[:, None]).sum(-1) + Dv[:, None] * x[t]
            ys[t] = (m * c.abs()[:, None]).sum(-1) + (Dv[:, None] * x[t]).abs()
        if kept:
            new[slot], new_s[slot] = s, m
    return y, ys, new, new_s


def gated_norm(y, z, w, groups, eps):
    """(out, size)."""
    g = y.double() * (silu(z.double()) if z is not None else 1)
    v = g.reshape(g.shape[0], groups, -1)
    out = (v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)).reshape(g.shape) * w.double()
    return out, out.abs()


def within(got, ref, bound):
    """Every element of got is finite where ref is and off by at most bound."""
    got, ref, bound = got.double().cpu(), ref.cpu(), bound.cpu()
    assert got.shape == ref.shape
    off = (got - ref).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} are off, the first at "
                           f"{[int(v) for v in bad.nonzero()[0]]}: {got[bad][0]} for {ref[bad][0]} "
                           f"within {bound[bad][0]}; worst ratio {float((off / bound)[bad].max()):.3g}")
