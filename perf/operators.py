"""Performance cases of the streaming attention path: what a rollout runs on every
chunk of frames, or on every new token, around its windowed key-value cache.

Four operators of ``cast_amd.ops``:

* ``rope``: rotary positions (half or interleaved pairs, part of the head, one to
  three position axes, frequencies scaled for long contexts);
* ``norm_rope``: RMS norms of queries and keys with the rotation in the same pass,
  keys and values written into a paged cache where one is given;
* ``window_attention``: causal attention (per token or per frame) over a sliding
  window and a few first keys that stay visible;
* ``paged_attention``: the same over a paged cache, from one new token per request
  to a whole chunk.

``listed()`` names twelve calls, ``draw(rng)`` makes more of the same ranges,
``prepare`` makes what the program holds before the call, ``run`` is one call
(the framework's where ``own`` is true, else its plain form), ``exact`` the same
outputs in 64 bits.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

FRAME = 880                 # tokens of a frame: a 22 x 40 latent grid
GRID = (22, 40)
AXES = (44, 42, 42)         # channels of a 128-wide head turned by frame, row, column
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# --------------------------------------------------------------------------
# Cases

def listed():
    return [
        # The rotation of one new token of each of a few requests, far into a long
        # context: launch latency.
        {"name": "rope_tokens", "kind": "rope", "dtype": "bf16", "batch": 8, "tokens": 1,
         "heads": 24, "dim": 128, "rotary": 128, "axes": 1, "interleaved": False,
         "scaling": "linear", "factor": 4.0, "first": 900001},
        # Queries (or keys) of a whole world of 44 frames, turned by frame, row and column.
        {"name": "rope_world", "kind": "rope", "dtype": "bf16", "batch": 1,
         "tokens": 44 * FRAME, "heads": 24, "dim": 128, "rotary": 128, "axes": 3,
         "interleaved": True, "scaling": None, "factor": 1.0, "first": 0},
        # Part of an odd-sized head in fp32, an odd number of tokens, a context
        # stretched by blended frequencies.
        {"name": "rope_part_f32", "kind": "rope", "dtype": "f32", "batch": 3, "tokens": 4097,
         "heads": 9, "dim": 80, "rotary": 32, "axes": 1, "interleaved": False,
         "scaling": "ramp", "factor": 8.0, "first": 70000},
        # A serving step: one new token of 64 requests, norms per head, keys and values
        # written to their pages.
        {"name": "prep_tokens", "kind": "prep", "dtype": "bf16", "batch": 64, "tokens": 1,
         "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "axes": 1,
         "interleaved": False, "scaling": None, "factor": 1.0, "across": False,
         "page": 64, "held": 5000},
        # A chunk of four frames: norms over all heads of a token, three position axes,
        # keys and values appended to the rollout's cache.
        {"name": "prep_chunk", "kind": "prep", "dtype": "bf16", "batch": 1,
         "tokens": 4 * FRAME, "heads": 24, "kv_heads": 24, "dim": 128, "rotary": 128,
         "axes": 3, "interleaved": True, "scaling": None, "factor": 1.0, "across": True,
         "page": 128, "held": 10 * FRAME},
        # A long prompt in fp16, norms per head, a larger base, no cache.
        {"name": "prep_long", "kind": "prep", "dtype": "f16", "batch": 2, "tokens": 16391,
         "heads": 16, "kv_heads": 4, "dim": 64, "rotary": 64, "axes": 1,
         "interleaved": False, "scaling": "base", "factor": 4.0, "across": False,
         "page": 0, "held": 0},
        # Every frame of a world against the twelve frames up to it and one anchor frame.
        {"name": "window_frames", "kind": "window", "dtype": "bf16", "batch": 1,
         "queries": 44 * FRAME, "keys": 44 * FRAME, "heads": 24, "kv_heads": 24, "dim": 128,
         "window": 12 * FRAME, "sinks": FRAME, "block": FRAME, "ragged": False},
        # A long prompt with shared key heads, a window of 4096 and four first tokens.
        {"name": "window_long", "kind": "window", "dtype": "bf16", "batch": 1,
         "queries": 32773, "keys": 32773, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 4096, "sinks": 4, "block": 1, "ragged": False},
        # A padded batch of short prompts, all keys up to the token, fp16, 64-wide heads.
        {"name": "window_batch", "kind": "window", "dtype": "f16", "batch": 3,
         "queries": 1111, "keys": 1111, "heads": 6, "kv_heads": 2, "dim": 64,
         "window": 0, "sinks": 0, "block": 1, "ragged": True},
        # One new token of one request over its window: latency.
        {"name": "paged_token", "kind": "paged", "dtype": "bf16", "batch": 1, "queries": 1,
         "keys": 2500, "heads": 24, "kv_heads": 8, "dim": 128, "page": 64, "window": 1024,
         "sinks": 4, "block": 1, "ragged": False},
        # One new token of 48 requests of very different lengths over all their keys.
        {"name": "paged_batch", "kind": "paged", "dtype": "bf16", "batch": 48, "queries": 1,
         "keys": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "window": 0,
         "sinks": 0, "block": 1, "ragged": True},
        # A chunk of four frames against the last twenty frames of the cache and the anchor.
        {"name": "paged_chunk", "kind": "paged", "dtype": "bf16", "batch": 1,
         "queries": 4 * FRAME, "keys": 44 * FRAME, "heads": 24, "kv_heads": 24, "dim": 128,
         "page": 128, "window": 20 * FRAME, "sinks": FRAME, "block": FRAME, "ragged": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _scaling(rng):
    kind = rng.choice([None, None, "linear", "base", "ramp"])
    return {"scaling": kind, "factor": rng.choice([2.0, 4.0, 8.0]) if kind else 1.0}


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 12, 24])
    return {"heads": kv * rng.choice([1, 1, 2, 3, 4, 8] if kv <= 4 else [1, 1, 2, 4] if kv <= 8
                                     else [1]), "kv_heads": kv}


def draw(rng):
    kind = rng.choice(["rope", "rope", "prep", "prep", "window", "window", "paged", "paged"])
    if kind in ("rope", "prep"):
        axes = rng.choice([1, 1, 3])
        dim = 128 if axes == 3 else rng.choice([64, 80, 96, 128, 128, 128, 256])
        rotary = (128 if axes == 3 else
                  rng.choice([dim, dim, dim // 2, dim // 4 // 2 * 2, dim * 3 // 4 // 2 * 2]))
        batch = rng.choice([1, 1, 2, 3, 8, 64])
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "batch": batch, "dim": dim, "rotary": rotary, "axes": axes,
                "interleaved": rng.random() < 0.5}
        case.update({"scaling": None, "factor": 1.0} if axes == 3 else _scaling(rng))
        if kind == "rope":
            heads = rng.choice([1, 3, 8, 9, 24, 32])
            room = 100_000_000 // (batch * heads * dim)
            case.update({"heads": heads, "tokens": _log(rng, 1, min(44 * FRAME, room)),
                         "first": rng.choice([0, 0, _log(rng, 1000, 2_000_000)])
                         if axes == 1 else 0})
        else:
            case.update(_heads(rng))
            room = 60_000_000 // (batch * (case["heads"] + 2 * case["kv_heads"]) * dim)
            page = rng.choice([0, 16, 64, 128, 256])
            case.update({"tokens": _log(rng, 1, max(1, min(20 * FRAME, room))),
                         "across": rng.random() < 0.3, "page": page,
                         "held": _log(rng, 1, 20000) if page else 0})
            if batch * (case["tokens"] + case["held"]) * case["kv_heads"] * dim > 250_000_000:
                case["held"] = 250_000_000 // (batch * case["kv_heads"] * dim)
        return case
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16"]),
            "dim": rng.choice([64, 128, 128])}
    case.update(_heads(rng))
    block = rng.choice([1, 1, 1, FRAME, 130])
    if kind == "window":
        batch = rng.choice([1, 1, 2, 3, 5])
        keys = _log(rng, 1, 32768)
        queries = rng.choice([keys, keys, _log(rng, 1, keys)])
    else:
        batch = rng.choice([1, 1, 4, 16, 48])
        keys = _log(rng, 16, 65536)
        queries = rng.choice([1, 1, 1, min(keys, rng.choice([2, 5, 17])),
                              _log(rng, 1, min(keys, 4 * FRAME))])
        case["page"] = rng.choice([16, 32, 48, 64, 128, 256])
    window = rng.choice([0, _log(rng, 16, 8192), _log(rng, 128, 12 * FRAME)])
    if block > 1 and window:
        window = -(-window // block) * block
    sinks = rng.choice([0, 1, 4, 64, block])
    # no dearer than the largest listed case: the products of all rows and their keys
    while 4.0 * batch * case["heads"] * case["dim"] * queries * min(keys, (window or keys)
                                                                   + sinks) > 4e12:
        queries = max(1, queries // 2)
    while 4 * batch * case["kv_heads"] * case["dim"] * keys > 1_700_000_000:
        keys = max(1, keys // 2)
        queries = min(queries, keys)
    case.update({"batch": batch, "queries": queries, "keys": keys, "window": window,
                 "sinks": sinks, "block": block, "ragged": batch > 1 and rng.random() < 0.6})
    return case


# --------------------------------------------------------------------------
# Inputs

def _device():
    return torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    """Random values of the type, made in pieces of the first dimensions."""
    out = torch.empty(shape, device=_device(), dtype=dtype)
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = torch.randn(n, device=_device(), generator=g).mul_(scale)
    return out


def _shifted(g, shape, dtype):
    """What a projection gives before its norm: a spread of token sizes."""
    x = torch.randn(shape, device=_device(), generator=g)
    x *= torch.exp(0.5 * torch.randn(shape[0], shape[1], 1, 1, device=_device(), generator=g))
    return x.to(dtype)


def _frequencies(case):
    """Radians per position of every pair, 64 bits, and the factor on the rotated part."""
    factor, scaling, rot = case["factor"], case["scaling"], case["rotary"]
    if case["axes"] == 3:
        freq = []
        for n in AXES:
            freq += [10000.0 ** (-2.0 * i / n) for i in range(n // 2)]
        return freq, 1.0
    base = 10000.0
    if scaling == "base" and rot > 2:
        base *= factor ** (rot / (rot - 2.0))
    freq = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    if scaling == "ramp":
        def blend(f):
            turns = case_length(case) * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (32.0 - 1.0)))
            return f * keep + f / factor * (1.0 - keep)
        return [blend(f) for f in freq], 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def case_length(case):
    """The context a stretched model was trained at."""
    return 8192


def _positions(case, g, start):
    """[B, L] token positions, or [L, 3] places on the latent grid."""
    n = case["tokens"]
    if case["axes"] == 3:
        t = torch.arange(n, device=_device())
        return torch.stack([start // FRAME + t // FRAME, t % FRAME // GRID[1], t % GRID[1]], 1)
    first = torch.randint(0, 17, (case["batch"], 1), device=_device(), generator=g) + start
    return first + torch.arange(n, device=_device())[None]


def _pages(g, batch, lengths, page):
    """A block table [B, M] of shuffled pages, -1 past a request's end, and the page count."""
    need = [-(-n // page) for n in lengths]
    total, width = sum(need), max(max(need), 1)
    order = torch.randperm(total + 3, device=_device(), generator=g).to(torch.int32)
    table = torch.full((batch, width), -1, device=_device(), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total + 3


def _lengths(case, seed):
    """Key and query lengths of the requests, as a padded batch has them."""
    rng = torch.Generator().manual_seed(int(seed) + 17)
    nk, nq, b = case["keys"], case["queries"], case["batch"]
    if not case["ragged"]:
        return [nk] * b, [nq] * b
    part = torch.rand(b, generator=rng).tolist()
    keys = [max(1, int(round(math.exp(math.log(max(2, nk // 32)) * (1 - p) + math.log(nk) * p))))
            for p in part]
    keys[int(seed) % b] = nk
    keys = [min(n, nk) for n in keys]
    return keys, [max(1, min(n, nq)) if nq == 1 else max(1, min(nq, int(round(nq * n / nk))))
                  for n in keys]


def prepare(case, seed):
    g = _gen(seed)
    dev, kind, dt = _device(), case["kind"], DTYPES[case["dtype"]]
    st = SimpleNamespace(kind=kind, case=case, cache=None)
    if kind in ("rope", "prep"):
        st.freq, st.factor = _frequencies(case)
        st.axis = ([a for a, n in enumerate(AXES) for _ in range(n // 2)]
                   if case["axes"] == 3 else [0] * len(st.freq))
        st.freq64 = torch.tensor(st.freq, dtype=torch.float64, device=dev)
        st.axis64 = torch.tensor(st.axis, device=dev)
        if own:
            from cast_amd.rotary import rotary_plan
            st.plan = rotary_plan(
                case["rotary"], axes=AXES if case["axes"] == 3 else None,
                interleaved=case["interleaved"], scaling=case["scaling"],
                factor=case["factor"], device=dev,
                original_length=case_length(case) if case["scaling"] == "ramp" else None)
    if kind == "rope":
        b, n, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
        st.x = _randn(g, (b, n, h, d), dt)
        st.pos = _positions(case, g, case["first"])
    elif kind == "prep":
        b, n, d = case["batch"], case["tokens"], case["dim"]
        h, hk, page = case["heads"], case["kv_heads"], case["page"]
        st.q = _shifted(g, (b, n, h, d), dt)
        st.k = _shifted(g, (b, n, hk, d), dt)
        wq, wk = ((h, d), (hk, d)) if case["across"] else ((d,), (d,))
        st.wq = (1.0 + 0.2 * torch.randn(wq, device=dev, generator=g)).to(dt)
        st.wk = (1.0 + 0.2 * torch.randn(wk, device=dev, generator=g)).to(dt)
        st.pos = _positions(case, g, case["held"])
        if page:
            st.v = _shifted(g, (b, n, hk, d), dt)
            st.held = [case["held"] - (i * 37) % max(1, case["held"] // 2) for i in range(b)]
            st.table, n_pages = _pages(g, b, [m + n for m in st.held], page)
            st.kp = _randn(g, (n_pages, page, hk, d), dt)
            st.vp = _randn(g, (n_pages, page, hk, d), dt)
            st.starts = torch.tensor(st.held, device=dev, dtype=torch.int32)
            if own:
                from cast_amd.ops import PagedCache
                st.cache = PagedCache(st.kp, st.vp, st.table)
    else:
        b, nq, nk, d = case["batch"], case["queries"], case["keys"], case["dim"]
        h, hk = case["heads"], case["kv_heads"]
        st.k_len, st.q_len = _lengths(case, seed)
        st.k_lens = torch.tensor(st.k_len, device=dev, dtype=torch.int32)
        st.q_lens = torch.tensor(st.q_len, device=dev, dtype=torch.int32)
        st.q = _randn(g, (b, nq, h, d), dt)
        # rows behind a request's last query stay as the caller left them
        st.out = torch.zeros(b, nq, h, d, device=dev, dtype=dt)
        if kind == "window":
            st.k = _randn(g, (b, nk, hk, d), dt)
            st.v = _randn(g, (b, nk, hk, d), dt)
        else:
            st.table, n_pages = _pages(g, b, st.k_len, case["page"])
            st.kp = _randn(g, (n_pages, case["page"], hk, d), dt)
            st.vp = _randn(g, (n_pages, case["page"], hk, d), dt)
            if own:
                from cast_amd.ops import PagedCache
                st.cache = PagedCache(st.kp, st.vp, st.table)
    return st


# --------------------------------------------------------------------------
# The plain forms

def _angles(st, dtype):
    """cos and sin [B|1, L, 1, R / 2] in ``dtype`` from 64-bit angles."""
    pos = st.pos.to(torch.float64)
    if st.case["axes"] == 3:
        a = (pos.index_select(1, st.axis64) * st.freq64)[None]
    else:
        a = pos[:, :, None] * st.freq64
    a = a[:, :, None, :]
    return (torch.cos(a) * st.factor).to(dtype), (torch.sin(a) * st.factor).to(dtype)


def _turn(x, cos, sin, rot, interleaved):
    """x [B, L, H, D] with its first ``rot`` channels turned."""
    half = rot // 2
    out = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2] = a * cos - b * sin
        out[..., 1:rot:2] = a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:rot]
        out[..., :half] = a * cos - b * sin
        out[..., half:rot] = a * sin + b * cos
    return out


def _normed(x, w, across):
    dims = (2, 3) if across else (3,)
    x = x.float()
    return x * torch.rsqrt(x.square().mean(dims, keepdim=True) + 1e-6) * w.float()


def _page_rows(table, index, page):
    """Rows of the flattened pages that hold keys ``index`` of one request."""
    return table.index_select(0, index // page).long() * page + index % page


def _plain_prep(st):
    c = st.case
    cos, sin = _angles(st, torch.float32)
    q = _turn(_normed(st.q, st.wq, c["across"]), cos, sin, c["rotary"], c["interleaved"])
    k = _turn(_normed(st.k, st.wk, c["across"]), cos, sin, c["rotary"], c["interleaved"])
    q, k = q.to(st.q.dtype), k.to(st.k.dtype)
    if not c["page"]:
        return [q, k]
    at = st.starts[:, None].long() + torch.arange(c["tokens"], device=q.device)
    rows = st.table.gather(1, at // c["page"]).long() * c["page"] + at % c["page"]
    st.kp.view(-1, c["kv_heads"], c["dim"])[rows] = k
    st.vp.view(-1, c["kv_heads"], c["dim"])[rows] = st.v
    return [q, st.kp, st.vp]


def _visible(first, rows, n_keys, window, sinks, block):
    """The keys [lo, hi) of the window of query positions first .. first + rows - 1."""
    def at(p):
        hi = min((p // block + 1) * block, n_keys)
        return (max(0, (p // block + 1) * block - window) if window else 0), hi
    return at(first)[0], at(first + rows - 1)[1]


def _plain_attention(q, k, v, first, window, sinks, block):
    """q [Lq, H, D], k and v [Lk, Hk, D] (fp32 products), rows first, first + 1, ...;
    returns [Lq, H, D] fp32 and the logarithm of each row's sum [H, Lq]."""
    nq, h, d = q.shape
    nk, hk, _ = k.shape
    g = h // hk
    out = torch.empty(nq, h, d, device=q.device)
    lse = torch.empty(h, nq, device=q.device)
    step = max(1, min(nq, 300_000_000 // (h * max(1, min(nk, (window or nk) + sinks + block)))))
    for r0 in range(0, nq, step):
        r1 = min(nq, r0 + step)
        lo, hi = _visible(first + r0, r1 - r0, nk, window, sinks, block)
        first_keys = min(sinks, lo, nk)
        index = torch.cat([torch.arange(first_keys, device=q.device),
                           torch.arange(lo, max(lo, hi), device=q.device)])
        kk = k.index_select(0, index).float().permute(1, 2, 0).contiguous()
        vv = v.index_select(0, index).float().permute(1, 0, 2).contiguous()
        qq = q[r0:r1].float().reshape(r1 - r0, hk, g, d).permute(1, 2, 0, 3)
        s = torch.matmul(qq.reshape(hk, g * (r1 - r0), d), kk).mul_(1.0 / math.sqrt(d))
        end = ((torch.arange(first + r0, first + r1, device=q.device) // block) + 1) * block
        seen = index[None] < end[:, None]
        if window:
            seen &= (index[None] >= end[:, None] - window) | (index[None] < sinks)
        s = s.view(hk, g, r1 - r0, -1).masked_fill_(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        s = s.sub_(top).exp_()
        total = s.sum(-1, keepdim=True)
        o = torch.matmul(s.view(hk, g * (r1 - r0), -1), vv).view(hk, g, r1 - r0, d) / total
        out[r0:r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, h, d)
        lse[:, r0:r1] = (top + total.log()).reshape(h, r1 - r0)
    return out, lse


def _plain_rows(st):
    """(request, q, k, v, first position) of every request's live rows."""
    c = st.case
    for b, (nk, nq) in enumerate(zip(st.k_len, st.q_len)):
        if st.kind == "window":
            k, v = st.k[b, :nk], st.v[b, :nk]
        else:
            rows = _page_rows(st.table[b], torch.arange(nk, device=st.q.device), c["page"])
            k, v = (p.view(-1, c["kv_heads"], c["dim"]).index_select(0, rows)
                    for p in (st.kp, st.vp))
        yield b, st.q[b, :nq], k, v, nk - nq


def run(state):
    st, c = state, state.case
    if own:
        return _run_own(st, c)
    if st.kind == "rope":
        cos, sin = _angles(st, torch.float32)
        return _turn(st.x.float(), cos, sin, c["rotary"], c["interleaved"]).to(st.x.dtype)
    if st.kind == "prep":
        return _plain_prep(st)
    lse = torch.zeros(c["batch"], c["heads"], c["queries"], device=st.q.device)
    for b, q, k, v, first in _plain_rows(st):
        o, s = _plain_attention(q, k, v, first, c["window"], c["sinks"], c["block"])
        st.out[b, :q.shape[0]] = o.to(st.out.dtype)
        lse[b, :, :q.shape[0]] = s
    return [st.out, lse] if st.kind == "paged" and c["queries"] == 1 else st.out


def _run_own(st, c):
    from cast_amd import ops
    if st.kind == "rope":
        return ops.rope(st.x, st.pos, st.plan)
    if st.kind == "prep":
        if not c["page"]:
            return list(ops.norm_rope(st.q, st.k, st.pos, st.plan, q_weight=st.wq,
                                      k_weight=st.wk, across_heads=c["across"]))
        q, _ = ops.norm_rope(st.q, st.k, st.pos, st.plan, q_weight=st.wq, k_weight=st.wk,
                             across_heads=c["across"], v=st.v, cache=st.cache, starts=st.starts)
        return [q, st.kp, st.vp]
    rows = {"window": c["window"] or None, "sinks": c["sinks"], "block": c["block"],
            "out": st.out, "q_lengths": st.q_lens if c["ragged"] else None}
    if st.kind == "window":
        return ops.window_attention(st.q, st.k, st.v,
                                    k_lengths=st.k_lens if c["ragged"] else None, **rows)
    out = ops.paged_attention(st.q, st.cache, st.k_lens, return_lse=c["queries"] == 1, **rows)
    return list(out) if c["queries"] == 1 else out


# --------------------------------------------------------------------------
# 64 bits

def _exact_rotation(x, pos, case):
    """Every pair as a complex number times exp(i angle)."""
    freq, factor = _frequencies(case)
    rot = case["rotary"]
    axis = ([a for a, n in enumerate(AXES) for _ in range(n // 2)] if case["axes"] == 3
            else None)
    pos = pos.to(torch.float64)
    columns = [(pos[None, :, axis[i]] if axis else pos) * f for i, f in enumerate(freq)]
    phase = torch.stack(columns, -1)[:, :, None]
    unit = torch.polar(torch.full_like(phase, factor), phase)
    x = x.double()
    head, rest = x[..., :rot], x[..., rot:]
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:-1], rot // 2, 2).contiguous())
        turned = torch.view_as_real(z * unit).flatten(-2)
    else:
        z = torch.complex(head[..., :rot // 2].contiguous(), head[..., rot // 2:].contiguous())
        z = z * unit
        turned = torch.cat([z.real, z.imag], -1)
    return torch.cat([turned, rest], -1)


def _exact_norm(x, w, across):
    x = x.double()
    flat = x.flatten(2) if across else x
    size = flat.pow(2).sum(-1) / flat.shape[-1] + 1e-6
    size = size[..., None, None] if across else size[..., None]
    return x / size.sqrt() * w.double()


def _exact_attention(q, k, v, first, case):
    """[Lq, H, D] and [H, Lq] in 64 bits, one head and a run of rows at a time."""
    nq, h, d = q.shape
    nk, hk, _ = k.shape
    window, sinks, block = case["window"], case["sinks"], case["block"]
    o = torch.empty(nq, h, d, device=q.device, dtype=torch.float64)
    lse = torch.empty(h, nq, device=q.device, dtype=torch.float64)
    keys = torch.arange(nk, device=q.device)
    rows = max(1, 40_000_000 // max(1, min(nk, (window or nk) + block)))
    for head in range(h):
        kd, vd = k[:, head * hk // h].double(), v[:, head * hk // h].double()
        for r0 in range(0, nq, rows):
            r1 = min(nq, r0 + rows)
            p = torch.arange(first + r0, first + r1, device=q.device)
            end = torch.div(p, block, rounding_mode="floor") * block + block
            start = (first + r0) // block * block + block - window if window else 0
            start = max(0, min(start, nk))
            stop = min(nk, (first + r1 - 1) // block * block + block)
            lead = min(sinks, start)
            use = torch.cat([keys[:lead], keys[start:stop]])
            logit = q[r0:r1, head].double() @ kd[use].T.contiguous() / math.sqrt(d)
            far = end[:, None] - use[None]
            dead = far <= 0
            if window:
                dead |= (far > window) & (use[None] >= sinks)
            logit.masked_fill_(dead, -math.inf)
            row = torch.logsumexp(logit, 1)
            o[r0:r1, head] = torch.exp(logit - row[:, None]) @ vd[use]
            lse[head, r0:r1] = row
    return o, lse


def exact(case, seed):
    st = prepare(case, seed)
    if st.kind == "rope":
        return _exact_rotation(st.x, st.pos, case)
    if st.kind == "prep":
        q = _exact_rotation(_exact_norm(st.q, st.wq, case["across"]), st.pos, case)
        k = _exact_rotation(_exact_norm(st.k, st.wk, case["across"]), st.pos, case)
        if not case["page"]:
            return [q, k]
        kp, vp = st.kp.double(), st.vp.double()
        for b, held in enumerate(st.held):
            at = torch.arange(held, held + case["tokens"], device=q.device)
            page = st.table[b].long()[at // case["page"]]
            kp[page, at % case["page"]] = k[b]
            vp[page, at % case["page"]] = st.v[b].double()
        return [q, kp, vp]
    out = torch.zeros(st.out.shape, device=st.out.device, dtype=torch.float64)
    lse = torch.zeros(case["batch"], case["heads"], case["queries"], device=out.device,
                      dtype=torch.float64)
    for b, (nk, nq) in enumerate(zip(st.k_len, st.q_len)):
        if st.kind == "window":
            k, v = st.k[b, :nk], st.v[b, :nk]
        else:
            at = torch.arange(nk, device=out.device)
            page = st.table[b].long()[at // case["page"]]
            k, v = st.kp[page, at % case["page"]], st.vp[page, at % case["page"]]
        out[b, :nq], lse[b, :, :nq] = _exact_attention(st.q[b, :nq], k, v, nk - nq, case)
    return [out, lse] if st.kind == "paged" and case["queries"] == 1 else out


# --------------------------------------------------------------------------
# Compulsory work

def _row_keys(case, nk, nq):
    """Visible keys summed over a request's rows, and of all of them together."""
    window, sinks, block = case["window"], case["sinks"], case["block"]
    p = torch.arange(nk - nq, nk)
    end = ((p // block) + 1) * block
    hi = end.clamp_max(nk)
    lo = (end - window).clamp_min(0) if window else torch.zeros_like(end)
    count = (hi - lo).clamp_min(0) + torch.minimum(lo, torch.tensor(min(sinks, nk)))
    union = int(hi.max()) - int(lo.min()) + min(sinks, int(lo.min()))
    return int(count.sum()), union


def work(case):
    d, b, size = case["dim"], case["batch"], 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "rope":
        n = b * case["tokens"] * case["heads"] * d
        return {"bytes": 2 * n * size, "flops": 3 * b * case["tokens"] * case["heads"]
                * case["rotary"]}
    if case["kind"] == "prep":
        heads = case["heads"] + case["kv_heads"] * (2 if case["page"] else 1)
        n = b * case["tokens"] * heads * d
        return {"bytes": 2 * n * size, "flops": b * case["tokens"]
                * (case["heads"] + case["kv_heads"]) * (4 * d + 3 * case["rotary"])}
    h, hk = case["heads"], case["kv_heads"]
    total = union = rows = 0
    for nk, nq in zip(*_lengths(case, 0)):
        t, u = _row_keys(case, nk, nq)
        total, union, rows = total + t, union + u, rows + nq
    return {"bytes": 2 * rows * h * d * size + 2 * union * hk * d * size,
            "flops": 4 * total * h * d}
