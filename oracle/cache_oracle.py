"""The 8-bit cache from its definition in 64 bits, plain torch on the CPU: quantised appends
and reads, one block of tokens and one head at a time."""
from __future__ import annotations

import math

import torch

LEAST = 2.0 ** -100


def nearest(x, code):
    """x (fp64) rounded to the values of the code, ties to even."""
    if code == torch.int8:
        return torch.round(x).clamp(-127, 127)
    e = torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 1
    step = torch.tensor([2.0 ** (int(n) - 3) for n in e.flatten()],
                        dtype=torch.float64).view(e.shape)
    return (torch.round(x / step) * step).clamp(-448, 448)


def own_scale(most, code):
    if code == torch.int8:
        return float(torch.tensor(most / 127.0, dtype=torch.float64).float())
    if most == 0.0:
        return 0.0
    m, e = math.frexp(most)  # most = m 2^e, m in [1/2, 1); 448 = 0.875 * 2^9
    return 2.0 ** (e - 9 if m <= 0.875 else e - 8)


def append(values, scales, table, block, x, first):
    """Appends x [n, H, D] to one request as keys first, first + 1, ...; values [pages, slots,
    H, D] (fp64, what the codes hold, before their scale) and scales [pages, blocks, H] (fp64)
    change in place, ``code`` being the dtype of the codes."""
    code = values["code"]
    v, slots, n_pages = values["v"], values["v"].shape[1], values["v"].shape[0]
    n, H, _ = x.shape
    cap = len(table) * slots
    lo, hi = max(first, 0), min(first + n, cap)
    for blk in range(lo // block, -(-hi // block) if hi > lo else lo // block):
        t0, t1 = max(blk * block, lo), min((blk + 1) * block, hi)
        page, row = int(table[blk * block // slots]), blk * block % slots
        if not 0 <= page < n_pages:
            continue
        new = x[t0 - first:t1 - first].double()
        kept = t0 - blk * block
        for h in range(H):
            s0 = float(scales[page, row // block, h]) if kept else 0.0
            if not 0.0 < s0 < math.inf:
                s0 = 0.0
            finite = new[:, h][torch.isfinite(new[:, h])]
            most = float(finite.abs().max()) if finite.numel() else 0.0
            s = max(s0, own_scale(most, code), LEAST)
            y = torch.nan_to_num(new[:, h], nan=0.0, posinf=1e300, neginf=-1e300) / s
            v[page, row + kept:row + t1 - blk * block, h] = nearest(y, code)
            if s != s0:
                old = v[page, row:row + kept, h]
                v[page, row:row + kept, h] = nearest(old * s0 / s, code)
            scales[page, row // block, h] = s


def read(v, scales, table, block, lo, hi):
    """Keys lo .. hi - 1 of one request, [hi - lo, H, D] in fp64 (0 where there is no page)."""
    slots, n_pages = v.shape[1], v.shape[0]
    out = torch.zeros(hi - lo, *v.shape[2:], dtype=torch.float64)
    for j in range(lo, hi):
        if j < 0 or j >= len(table) * slots:
            continue
        page, row = int(table[j // slots]), j % slots
        if 0 <= page < n_pages:
            out[j - lo] = v[page, row] * scales[page, row // block, :, None]
    return out


def attention(q, k, v, v_top, seen, sm_scale, dtype):
    """``streaming_oracle.attention`` of the values that codes stand for (k, v in fp64), and the
    bounds of a kernel that rounds a weight times its block's scale to fp16: half a step, 2^-11,
    of it; the type's least half step, 2^-25, where the largest weight is 2^7 at least and a
    scale's unit at most twice the largest scale, so 2^-31 of the largest weight and of
    ``v_top``, the largest scale times the largest code; and the result's own rounding."""
    from oracle import streaming_oracle as so
    top = float(v.abs().max()) if v.numel() else 0.0
    step = 2.0 ** -31 * (v_top / top if top > 0.0 else 0.0)
    out, lse, tol, ltol = so.attention(q, k, v, seen, sm_scale, torch.float16, weight_step=step)
    tol = tol + out.abs() * (so.HALF_STEP[dtype] - so.HALF_STEP[torch.float16])
    if dtype == torch.bfloat16:
        tol = (tol - so.TINY[torch.float16]).clamp(min=0.0)  # (without keys it is not in it)
    return out, lse, tol, ltol
