"""Dense attention with capped scores, a bias by distance and segment masks, in float64, and how far a kernel may be
from it: every result comes with the size of what was summed into it, for tolerances that count roundings.

  x = scale q k^T,  s = cap tanh(x / cap) - slope |p_q - p_k|,  P = softmax(s) over visible keys,  out = P v
  dv = P^T g,  dP = g v^T,  delta = sum P dP,  dS = P (dP - delta),  dslope = -sum dS |p_q - p_k|,
  dX = dS (1 - tanh^2),  dq = scale dX k,  dk = scale dX^T q
"""
import math

import torch


def visible(q_segments, k_segments):
    """(N, Lq, Lk) bool: the same segment or the shared one (0); negative numbers are padding."""
    mine, theirs = q_segments[:, :, None], k_segments[:, None]
    return (mine >= 0) & ((mine == theirs) | (theirs == 0))


def attention(q, k, v, grad=None, scale=None, cap=0.0, q_segments=None, k_segments=None, q_points=None, k_points=None, slopes=None,
              unit=2.0 ** -53, tiny=0.0, device="cpu"):
    """Results in float64 and their tolerances for tensors of a type with rounding unit ``unit`` (half a step, relative) and smallest
    rounding ``tiny`` (half the step of its subnormals): dict name -> (value, tolerance).

    What a kernel rounds to the type: each weight of P before its product (unit P, and tiny against the largest of a row), each
    dS before its product, delta through the rounded out, and the result.  All else is fp32: a score from `width` products is off by
    e = (width + 8) 2^-24 times the sum of their sizes (slope times distance and the score itself counted in), a weight by 2 e and
    the sum over the keys, relatively.  A tanh is off relative to itself, no more than the product that goes into it; where results have 16 bits and
    the cap is at most 256 a kernel may form it as the difference of numbers of the cap's size, e then has 2^-20 of the cap as well.
    Exponentials have no subnormals: a weight below 2^-126 may be zero, in the forward against a maximum that is up to 2^8 behind, so 2^-118 of
    the largest, in the backward against the row's sum; dS below that too.  The scale of dS in fp16 keeps it below 2^15 by
    width max|g| max|v|, so that tiny weighs 2^-15 of twice that.  Sizes are floats of all heads, key heads already spread over the heads that share them."""
    to = lambda t: t.detach().to(device).double()
    q, k, v = to(q), to(k), to(v)
    n, lq, m, d = q.shape
    lk, share = k.shape[1], m // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    spread = torch.arange(m, device=device) // share
    qh, kh, vh = q.permute(0, 2, 1, 3), k[:, :, spread].permute(0, 2, 1, 3), v[:, :, spread].permute(0, 2, 1, 3)
    x = scale * (qh @ kh.transpose(-1, -2))
    size = abs(scale) * (qh.abs() @ kh.abs().transpose(-1, -2))
    th = torch.zeros_like(x)
    s = x
    if cap:
        th = torch.tanh(x / cap)
        s = cap * th
    dist = torch.zeros(n, 1, lq, lk, dtype=torch.float64, device=device)
    if slopes is not None:
        pq, pk = to(q_points), to(k_points)
        dist = (pq[:, :, None] - pk[:, None]).pow(2).sum(-1).sqrt()[:, None]
        bias = to(slopes).view(1, m, 1, 1) * dist
        s = s - bias
        size = size + bias.abs()
    see = torch.ones(n, 1, lq, lk, dtype=torch.bool, device=device)
    if k_segments is not None:
        mine = torch.zeros(n, lq, dtype=torch.int32, device=device) if q_segments is None else q_segments.to(device)
        see = visible(mine, k_segments.to(device))[:, None]
    see = see.expand_as(s)
    s = torch.where(see, s, -math.inf)
    top = s.amax(-1, keepdim=True) if lk else torch.zeros(n, m, lq, 1, dtype=torch.float64, device=device)
    p = torch.where(see, torch.exp(s - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)

    def clean(t):          # what is not seen may hold anything
        return torch.where(torch.isfinite(t), t, 0.0)

    kh, vh, qh = clean(kh), clean(vh), clean(qh)
    bent_off = 2.0 ** -20 * cap if unit > 2.0 ** -20 and cap <= 256 else 0.0
    error = torch.where(see, 2.0 ** -24 * (2 * (d + 8) * clean(size) + lk + 64) + 2 * bent_off, 0.0).amax(-1, keepdim=True) if lk else torch.zeros_like(top)
    out = p @ vh
    back = lambda t: t.permute(0, 2, 1, 3)
    gather = lambda t: back(t.reshape(n, k.shape[2], share, lk, -1).sum(2))
    found = {"out": (back(out), back(unit * out.abs() + (2 * unit + error) * (p @ vh.abs()) + (tiny + 2.0 ** -118) * (see.double() @ vh.abs())) + tiny)}
    if grad is None:
        return found
    g = clean(to(grad).permute(0, 2, 1, 3))
    dp = g @ vh.transpose(-1, -2)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    bent = 1 - th * th
    dx = ds * bent
    about = (g.abs() * out.abs()).sum(-1, keepdim=True)
    most = g.abs().max() * vh.abs().max() * d if g.numel() and vh.numel() else 0.0
    # of dS, dX and what they are multiplied by
    off = p * (unit * about + 2 * error * (g.abs() @ vh.abs().transpose(-1, -2) + about))
    off = off + (unit * ds.abs() + see.double() * (tiny * 2.0 ** -15 * most + 2.0 ** -126 * (1 + g.abs() @ vh.abs().transpose(-1, -2) + about)))
    bend = ds.abs() * torch.where(see, error, 0.0) * (2.0 if cap else 0.0)
    dq, dk, dv = scale * (dx @ kh), scale * (dx.transpose(-1, -2) @ qh), p.transpose(-1, -2) @ g
    spot = unit * dx.abs() + off + bend
    found["grad_query"] = (back(dq), back(unit * dq.abs() + abs(scale) * (spot @ kh.abs())) + tiny)
    found["grad_key"] = (gather(dk), gather(2 * unit * dk.abs() + abs(scale) * (spot.transpose(-1, -2) @ qh.abs())) + tiny)
    weight_off = p * (unit + 2 * error) + see.double() * (tiny * 2.0 ** -8 + 2.0 ** -126)
    found["grad_value"] = (gather(dv), gather(2 * unit * dv.abs() + weight_off.transpose(-1, -2) @ g.abs()) + tiny)
    if slopes is not None:
        dist = clean(dist)
        parts = (off + ds.abs() * 2.0 ** -20) * dist
        found["grad_slopes"] = (-(ds * dist).sum((0, 2, 3)), parts.sum((0, 2, 3)) + 1e-30)
    return found
