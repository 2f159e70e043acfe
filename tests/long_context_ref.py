"""Plain fp64 forms of the long-context operators, with the error each
element may have.

A rounding to bf16 is off by at most half a step, BF = 2^-8 of the value.  The
kernels round P and dS to bf16 before they enter a product, and each bf16
output once; everything else is fp32.  fp32 work is bounded by F = 2^-23 a
step (a tensor core may cut a sum off instead of rounding it), with the
number of steps in front: D + 8 for a dot product over a head, the number of
keys or rows for a sum over them."""
import math

import torch

BF, F = 2.0 ** -8, 2.0 ** -23


def visible(T, K, window, sinks, start, n, device):
    """[T, K] truth: row i (position start + i, padding from n on) sees key j."""
    i = torch.arange(T, device=device)[:, None]
    j = torch.arange(K, device=device)[None]
    t = start + i
    return (j <= t) & ((t - j < window) | (j < sinks)) & (i < n)


def _heads(x, heads, D):
    return x.double().view(x.shape[0], heads, D).transpose(0, 1)  # [heads, rows, D]


def _rows(x):
    return x.transpose(0, 1).reshape(x.shape[1], -1)


def _clean(x, keep):
    """Rows that nothing may read are taken as 0, whatever they hold."""
    return torch.where(keep[:, None], x, torch.zeros_like(x))


def _scores(q, k, see, D):
    s = q @ k.transpose(1, 2) / math.sqrt(D)
    ds = (D + 8) * F * (q.abs() @ k.abs().transpose(1, 2)) / math.sqrt(D)  # fp32 error of a score
    return s.masked_fill(~see, -math.inf), ds.masked_fill(~see, 0.0)


def forward(q, k, v, NH, NKV, D, window, sinks, start, n):
    """One sequence: q [T, NH*D], k, v [K, NKV*D] -> out, l and what they may be off by."""
    T, K, G = q.shape[0], k.shape[0], NH // NKV
    see = visible(T, K, window, sinks, start, n, q.device)
    used = see.any(0)
    q = _clean(q, see.any(1))
    Q = _heads(q, NH, D)
    Kh, Vh = (_heads(_clean(x, used), NKV, D).repeat_interleave(G, 0) for x in (k, v))
    s, ds = _scores(Q, Kh, see, D)
    l = torch.logsumexp(s, -1)
    some = see.any(1)
    p = torch.where(see, torch.exp(s - torch.where(some, l, torch.zeros_like(l))[..., None]), torch.zeros_like(s))
    o = p @ Vh
    steps = K * F
    worst = ds.amax(-1) if K else 0.0
    rel = BF + 2 * steps + 2.0 ** -20
    tol_o = BF * o.abs() + (p * (rel + 2 * worst[..., None])) @ Vh.abs() + 1e-30
    tol_l = worst + steps + 2.0 ** -20 + 4 * F * torch.where(some, l, torch.zeros_like(l)).abs()
    return _rows(o), l.transpose(0, 1), _rows(tol_o), tol_l.transpose(0, 1)


def backward(dO, out, l, q, k, v, NH, NKV, D, window, sinks, n, dq_f32):
    """One sequence, from the out and l given: (dQ, dK, dV) and what each may be off by."""
    T, G = q.shape[0], NH // NKV
    see = visible(T, T, window, sinks, 0, n, q.device)
    some, used = see.any(1), see.any(0)
    dO, out, q = (_clean(x, some) for x in (dO, out, q))
    Q, d, o = (_heads(x, NH, D) for x in (q, dO, out))
    Kh, Vh = (_heads(_clean(x, used), NKV, D).repeat_interleave(G, 0) for x in (k, v))
    L = torch.where(some[:, None], l.double(), torch.zeros_like(l, dtype=torch.float64)).transpose(0, 1)
    s, es = _scores(Q, Kh, see, D)
    p = torch.where(see, torch.exp(s - L[..., None]), torch.zeros_like(s))
    ep = p * (es + 2.0 ** -20 + 4 * F * L.abs()[..., None])  # fp32 error of P
    delta = (d * o).sum(-1)
    dp = d @ Vh.transpose(1, 2)
    edp = (D + 8) * F * (d.abs() @ Vh.abs().transpose(1, 2) + (d * o).abs().sum(-1)[..., None])
    t = dp - delta[..., None]
    ds = p * t / math.sqrt(D)
    eds = BF * ds.abs() + (ep * t.abs() + p * edp) / math.sqrt(D)
    steps = 2 * T * G * F

    def group(x):  # sum over the query heads that share a K/V head
        return x.view(NKV, G, *x.shape[1:]).sum(1)

    dq = ds @ Kh
    tq = eds @ Kh.abs() + steps * (ds.abs() @ Kh.abs()) + (0.0 if dq_f32 else BF) * dq.abs() + 1e-30
    dk = group(ds.transpose(1, 2) @ Q)
    tk = group(eds.transpose(1, 2) @ Q.abs() + steps * (ds.abs().transpose(1, 2) @ Q.abs())) + BF * dk.abs() + 1e-30
    dv = group(p.transpose(1, 2) @ d)
    tv = group((BF * p + ep + steps * p).transpose(1, 2) @ d.abs()) + BF * dv.abs() + 1e-30
    return tuple(_rows(x) for x in (dq, dk, dv)), tuple(_rows(x) for x in (tq, tk, tv))


def rotate(x, heads, D, rot, inter, amp, inv_freq, pos, back=False):
    """x [rows, heads*D] turned by pos [rows]; -> values, and the sums of magnitudes their error scales with."""
    y = x.double().view(x.shape[0], heads, D).clone()
    m = y.abs()
    ang = pos.double()[:, None] * inv_freq
    c, s = torch.cos(ang)[:, None] * amp, torch.sin(ang)[:, None] * amp
    if back:
        s = -s
    ia, ib = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    both = (a.abs() + b.abs()) * abs(amp)
    m[..., ia], m[..., ib] = both, both
    return y.view(x.shape), m.view(x.shape)
