"""The streaming attention path's operators from their definitions in 64 bits, plain
torch on any device: rotary positions, norms of queries and keys, attention over a
sliding window and the first keys.  Each returns its result and a bound on what a kernel
that computes in fp32 and rounds once may be off by.

A rounding to a type is off by at most half a step, eps / 2 of the value.
"""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def frequencies(rotary_dim, base=10000.0, axes=None, scaling=None, factor=1.0,
                original_length=None, low=1.0, high=32.0):
    """Radians per position and axis of every pair."""
    out, ax = [], []
    for a, n in enumerate([rotary_dim] if axes is None else axes):
        for i in range(n // 2):
            b = base * factor ** (n / (n - 2)) if scaling == "base" and n > 2 else base
            f = 1.0 / b ** (2 * i / n)
            if scaling == "linear":
                f = f / factor
            if scaling == "ramp":
                r = original_length * f / (2 * math.pi)
                g = min(max((r - low) / (high - low), 0.0), 1.0)
                f = (1 - g) * f / factor + g * f
            out.append(f)
            ax.append(a)
    return out, ax


def rope(x, positions, freq, axis, interleaved, scale=1.0, n_axes=1):
    """x [B, L, H, D] turned in 64 bits, and |a| + |b| of every channel's pair."""
    B, L, _, D = x.shape
    x = x.double()
    f = torch.tensor(freq, dtype=torch.float64, device=x.device)
    pos = positions.double()
    if n_axes > 1:
        pos = pos.expand(B, L, n_axes)[..., torch.tensor(axis, device=x.device)]
    else:
        pos = pos.expand(B, L)[..., None]
    t = (pos * f)[:, :, None]
    c, s = torch.cos(t) * scale, torch.sin(t) * scale
    n = len(freq)
    ia = torch.arange(n, device=x.device) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    a, b = x[..., ia], x[..., ib]
    out, size = x.clone(), x.abs()
    out[..., ia], out[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia] = size[..., ib] = (a.abs() + b.abs()) * abs(scale)
    return out, size


def norm(x, weight, eps, across):
    x = x.double()
    mean = x.square().mean((2, 3) if across else 3, keepdim=True)
    y = x / (mean + eps).sqrt()
    return y if weight is None else y * weight.double()


def rope_bound(ref, size, dtype, norm=False):
    """fp32 products and sums of a pair (2^-22 of it with its sines; 2^-19 with a norm's
    sum, root and weight before it), then one rounding."""
    return ref.abs() * HALF_STEP[dtype] + size * (2.0 ** -19 if norm else 2.0 ** -22) + TINY[dtype]


def visible(q_len, k_len, window, sinks, block, causal=True, device="cpu"):
    """bool [q_len, k_len]: the keys each query sees (window 0: none)."""
    p = torch.arange(q_len, device=device) + k_len - q_len
    j = torch.arange(k_len, device=device)[None]
    if not causal:
        return torch.ones(q_len, k_len, dtype=torch.bool, device=device)
    e = (torch.div(p, block, rounding_mode="floor") + 1)[:, None] * block
    near = j >= e - window if window else torch.ones_like(j, dtype=torch.bool)
    return (j < e) & (near | (j < sinks)) & (p[:, None] >= 0)


def attention(q, k, v, seen, sm_scale, dtype, weight_step=None):
    """q [Lq, H, D], k, v [Lk, Hk, D], seen [Lq, Lk].  Returns out [Lq, H, D], lse [H, Lq]
    and their bounds.  Keys and values that a row does not see do not enter.

    The bound of an output: its rounding; the rounding of every weight to the type (half a
    step of sum p |v|, and the type's least step a key, or `weight_step` of the largest
    weight); a logit's fp32 error e_s (D + 2 roundings of its products), twice, in the
    weights; 2^-16 for the exponentials and the sums."""
    Lq, H, D = q.shape
    Lk, Hk, _ = k.shape
    g = H // Hk
    out = torch.zeros(Lq, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    lse = torch.full((H, Lq), -math.inf, dtype=torch.float64, device=q.device)
    lse_tol = torch.zeros_like(lse)
    some = seen.any(1)
    if Lk == 0:
        return out, lse, tol, lse_tol
    for h in range(H):
        kk, vv, qq = k[:, h // g].double(), v[:, h // g].double(), q[:, h].double()
        used = seen.any(0)
        kk = torch.where(used[:, None], kk, torch.zeros_like(kk))
        s = qq @ kk.T.contiguous() * sm_scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        size = qq.abs() @ kk.abs().T.contiguous() * abs(sm_scale)
        size = torch.where(seen, size, torch.zeros_like(size))
        e_s = size.amax(1, keepdim=True) * (D + 2) * 2.0 ** -24
        row = torch.logsumexp(s, 1, keepdim=True)
        p = torch.where(seen, torch.exp(s - row), torch.zeros_like(s))
        clean = torch.where(torch.isfinite(vv), vv, torch.zeros_like(vv))
        o = p @ clean
        mass = p @ clean.abs()
        bad = ~torch.isfinite(vv)
        if bool((bad & used[:, None]).any()):
            for j in torch.nonzero(bad.any(1) & used).flatten().tolist():
                o += torch.where(seen[:, j, None] & bad[j][None], vv[j][None],
                                 torch.zeros_like(o))
        n = seen.sum(1, keepdim=True).double()
        out[:, h] = torch.where(some[:, None], o, torch.zeros_like(o))
        tol[:, h] = (o.abs() * HALF_STEP[dtype] + TINY[dtype]
                     + mass * (HALF_STEP[dtype] + 2 * e_s + 2.0 ** -16)
                     + n * (2 * TINY[dtype] if weight_step is None else weight_step * p.amax(
                         1, keepdim=True)) * clean.abs().amax(0, keepdim=True))
        lse[h] = row[:, 0]
        lse_tol[h] = e_s[:, 0] + 2.0 ** -18 * (1 + row[:, 0].abs())
    return out, lse, tol, lse_tol
