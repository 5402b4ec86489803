"""Performance cases of serving from a key-value cache held in 8 bits: what a server or a
rollout runs when a prompt comes in, when new tokens join the cache, and when layers read
what the cache holds.

Four operators of ``cast_amd.ops``:

* ``append_cache``: keys and values quantised (int8 or e4m3, one scale for each block of
  tokens and head) as they are written to the pages of a ``QuantizedCache``; padded
  batches or packed sequences;
* ``read_cache``: a range of every request's keys and values read back into dense
  tensors, as the woven layers take them;
* ``paged_attention`` over a ``QuantizedCache``, from one new token to a chunk;
* ``packed_attention``: causal attention over whole prompts of different lengths that
  follow each other without padding.

``listed()`` names twelve calls, ``draw(rng)`` makes more of the same ranges,
``prepare`` makes what the program holds before the call, ``run`` is one call
(the framework's where ``own`` is true, else its plain form), ``exact`` the same
outputs in 64 bits.  An append is run with the read of the blocks that it wrote: the
values that the codes stand for, and their scales, are its outputs.

The format.  A code c of a block and head with scale s (fp32) stands for c * s.  An append
takes a = max |x| of the block's new values; the block's scale becomes

    int8:  max(s0, fp32(a / 127), 2^-100)
    e4m3:  max(s0, the smallest power of two p with a <= 448 p, 2^-100)

with s0 the scale that the block had if tokens before the new ones are in it, else 0.  New
codes are x / s rounded to the nearest (ties to even); where the scale grew, the codes before
the new ones become c * s0 / s, rounded alike.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

FRAME = 880                 # tokens of a frame: a 22 x 40 latent grid
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOOR = 2.0 ** -100         # the smallest scale


# --------------------------------------------------------------------------
# Cases

def listed():
    return [
        # A serving step: one new token of 64 requests joins blocks that are partly full.
        {"name": "append_tokens", "kind": "append", "dtype": "bf16", "code": "int8",
         "batch": 64, "tokens": 1, "packed": False, "kv_heads": 8, "dim": 128, "page": 64,
         "block": 32, "held": 5000},
        # A chunk of four frames joins a rollout's cache.
        {"name": "append_chunk", "kind": "append", "dtype": "bf16", "code": "int8",
         "batch": 1, "tokens": 4 * FRAME, "packed": False, "kv_heads": 24, "dim": 128,
         "page": 128, "block": 128, "held": 10 * FRAME},
        # Prompts of different lengths, packed, fill their first pages.
        {"name": "append_prompts", "kind": "append", "dtype": "f16", "code": "e4m3",
         "batch": 11, "tokens": 8192, "packed": True, "kv_heads": 4, "dim": 64, "page": 16,
         "block": 16, "held": 0},
        # A world of 44 frames read back for a woven layer.
        {"name": "read_world", "kind": "read", "dtype": "bf16", "code": "int8", "batch": 1,
         "tokens": 44 * FRAME, "kv_heads": 24, "dim": 128, "page": 128, "block": 128,
         "held": 0},
        # The last keys of a ragged batch, heads of an odd size.
        {"name": "read_batch", "kind": "read", "dtype": "f16", "code": "e4m3", "batch": 16,
         "tokens": 1003, "kv_heads": 9, "dim": 80, "page": 48, "block": 16, "held": 3001},
        # One new token of one request over its window: latency.
        {"name": "cached_token", "kind": "cached", "dtype": "bf16", "code": "int8",
         "batch": 1, "queries": 1, "keys": 2500, "heads": 24, "kv_heads": 8, "dim": 128,
         "page": 64, "mark": 64, "window": 1024, "sinks": 4, "block": 1, "ragged": False},
        # One new token of 48 requests of very different lengths over all their keys.
        {"name": "cached_batch", "kind": "cached", "dtype": "bf16", "code": "int8",
         "batch": 48, "queries": 1, "keys": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "mark": 16, "window": 0, "sinks": 0, "block": 1, "ragged": True},
        # Five drafted tokens of 24 requests, e4m3, 64-wide heads.
        {"name": "cached_draft", "kind": "cached", "dtype": "f16", "code": "e4m3",
         "batch": 24, "queries": 5, "keys": 8191, "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 16, "mark": 16, "window": 0, "sinks": 0, "block": 1, "ragged": True},
        # A chunk of four frames against the last twenty frames of the cache and the anchor.
        {"name": "cached_chunk", "kind": "cached", "dtype": "bf16", "code": "int8",
         "batch": 1, "queries": 4 * FRAME, "keys": 44 * FRAME, "heads": 24, "kv_heads": 24,
         "dim": 128, "page": 128, "mark": 128, "window": 20 * FRAME, "sinks": FRAME,
         "block": FRAME, "ragged": False},
        # A queue of short prompts, 64-wide heads, fp16: latency.
        {"name": "packed_short", "kind": "packed", "dtype": "f16", "batch": 40,
         "tokens": 301, "context": 0, "heads": 6, "kv_heads": 2, "dim": 64, "window": 0,
         "sinks": 0, "block": 1},
        # Long and short prompts together, shared key heads, some behind keys held before.
        {"name": "packed_prompts", "kind": "packed", "dtype": "bf16", "batch": 9,
         "tokens": 8192, "context": 1500, "heads": 32, "kv_heads": 8, "dim": 128,
         "window": 0, "sinks": 0, "block": 1},
        # Clips of different lengths, causal by frame over twelve frames and the first.
        {"name": "packed_clips", "kind": "packed", "dtype": "bf16", "batch": 4,
         "tokens": 20 * FRAME, "context": 0, "heads": 24, "kv_heads": 24, "dim": 128,
         "window": 12 * FRAME, "sinks": FRAME, "block": FRAME},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 12, 24])
    return {"heads": kv * rng.choice([1, 1, 2, 3, 4, 8] if kv <= 4 else [1, 1, 2, 4] if kv <= 8
                                     else [1]), "kv_heads": kv}


def _paging(rng, mark):
    page = rng.choice([16, 32, 48, 64, 128, 256])
    return {"page": page, mark: rng.choice([n for n in (16, 32, 48, 64, 128, 256)
                                            if page % n == 0])}


def draw(rng):
    kind = rng.choice(["append", "append", "read", "cached", "cached", "cached", "packed",
                       "packed"])
    if kind in ("append", "read"):
        case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "code": rng.choice(["int8", "e4m3"]), "batch": rng.choice([1, 1, 2, 3, 16, 64]),
                "kv_heads": rng.choice([1, 3, 4, 8, 9, 24]),
                "dim": rng.choice([64, 80, 96, 128, 128, 256])}
        room = (24_000_000 if kind == "append" else 110_000_000) // (
            case["batch"] * case["kv_heads"] * case["dim"])
        case["tokens"] = _log(rng, 1, max(1, min(44 * FRAME, room)))
        case["held"] = rng.choice([0, _log(rng, 1, 20000)])
        if case["batch"] * (case["tokens"] + case["held"]) * case["kv_heads"] * case["dim"] \
                > 400_000_000:
            case["held"] = 100_000_000 // (case["batch"] * case["kv_heads"] * case["dim"])
        if kind == "append":
            case["packed"] = rng.random() < 0.4
        case.update(_paging(rng, "block"))
        return case
    case = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16"]),
            "dim": rng.choice([64, 128, 128])}
    case.update(_heads(rng))
    block = rng.choice([1, 1, 1, FRAME, 130])
    window = rng.choice([0, _log(rng, 16, 8192), _log(rng, 128, 12 * FRAME)])
    if block > 1 and window:
        window = -(-window // block) * block
    case.update({"block": block, "window": window,
                 "sinks": rng.choice([0, 1, 4, 64, block]) if window else 0})
    products = 4.0 * case["heads"] * case["dim"]
    if kind == "packed":
        case["batch"] = rng.choice([1, 2, 4, 9, 40])
        case["context"] = rng.choice([0, 0, _log(rng, 1, 4000)])
        tokens = _log(rng, 1, 20 * FRAME)
        # no dearer than the largest listed case: the products of all rows and their keys
        while products * case["batch"] * tokens * min(
                tokens + case["context"], (window or 10 ** 9) + case["sinks"]) > 4e12:
            tokens = max(1, tokens // 2)
        while case["batch"] * (tokens + case["context"]) * case["heads"] * case["dim"] > 2e8:
            tokens, case["context"] = max(1, tokens // 2), case["context"] // 2
        case["tokens"] = tokens
        return case
    case["code"] = rng.choice(["int8", "int8", "e4m3"])
    batch = rng.choice([1, 1, 4, 16, 48])
    keys = _log(rng, 16, 65536)
    queries = rng.choice([1, 1, 1, min(keys, rng.choice([2, 5, 17])),
                          _log(rng, 1, min(keys, 4 * FRAME))])
    while products * batch * queries * min(keys, (window or keys) + case["sinks"]) > 4e12:
        queries = max(1, queries // 2)
    while 2 * batch * case["kv_heads"] * case["dim"] * keys > 1_700_000_000:
        keys = max(1, keys // 2)
        queries = min(queries, keys)
    case.update({"batch": batch, "queries": queries, "keys": keys,
                 "ragged": batch > 1 and rng.random() < 0.6})
    case.update(_paging(rng, "mark"))
    return case


# --------------------------------------------------------------------------
# Inputs

def _device():
    return torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(int(seed))


def _randn(g, shape, dtype, scale=1.0):
    """Random values of the type, made in pieces."""
    out = torch.empty(shape, device=_device(), dtype=dtype)
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        x = torch.randn(n, device=_device(), generator=g).mul_(scale)
        if dtype == torch.int8:
            x = x.round_().clamp_(-127, 127)
        elif dtype == torch.float8_e4m3fn:
            x = x.clamp_(-448, 448)
        flat[i:i + n] = x.to(dtype)
    return out


def _projected(g, shape, dtype):
    """Keys or values as a projection gives them: tokens of different sizes, a few
    channels far larger than the others."""
    x = torch.randn(shape, device=_device(), generator=g)
    x *= torch.exp(0.4 * torch.randn(shape[:-2], device=_device(), generator=g))[..., None, None]
    gain = torch.exp(0.8 * torch.randn(shape[-2:], device=_device(), generator=g))
    return (x * gain).to(dtype)


def _power(e):
    """2^e for whole e of normal fp32 numbers, exactly, in fp32."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pages(g, lengths, page):
    """A block table [B, M] of shuffled pages, -1 past a request's end, and the page count."""
    need = [-(-n // page) for n in lengths]
    total, width = sum(need), max(max(need), 1)
    order = torch.randperm(total + 3, device=_device(), generator=g).to(torch.int32)
    table = torch.full((len(lengths), width), -1, device=_device(), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total + 3


def _cache(st, g, lengths, block):
    """A cache that holds ``lengths`` tokens of each request (room for them, that is)."""
    c = st.case
    page, h, d, code = c["page"], c["kv_heads"], c["dim"], CODES[c["code"]]
    st.table, n = _pages(g, lengths, page)
    wide = 40.0 if code == torch.int8 else 100.0
    st.kc, st.vc = (_randn(g, (n, page, h, d), code, wide) for _ in range(2))
    def scales():
        e = 0.5 * torch.randn((n, page // block, h), device=_device(), generator=g)
        # (the values are of the order of 1)
        return _power(torch.round(e) - 7) if code != torch.int8 else torch.exp(e) / wide
    st.ks, st.vs = scales(), scales()
    if own:
        from cast_amd.ops import QuantizedCache
        st.cache = QuantizedCache(st.kc, st.vc, st.ks, st.vs, st.table)


def _spread(count, longest):
    """``count`` lengths up to ``longest``, spread over their logarithm; one is the longest."""
    rng = torch.Generator().manual_seed(17 * count + longest)
    part = torch.rand(count, generator=rng).tolist()
    low = math.log(max(1, longest // 32))
    n = [max(1, min(longest, int(round(math.exp(low * (1 - p) + math.log(longest) * p)))))
         for p in part]
    n[count // 2] = longest
    return n


def _requests(case):
    """What each request of a case has, as pairs: tokens held before and new tokens
    (append, read), or keys and queries (attention)."""
    kind, b = case["kind"], case["batch"]
    if kind in ("append", "read"):
        n, m = case["tokens"], case["held"]
        count = _spread(b, n) if kind == "read" or case["packed"] else [n] * b
        return [(m - i * 37 % max(1, m // 2) if m else 0, t) for i, t in enumerate(count)]
    if kind == "cached":
        nk, nq = case["keys"], case["queries"]
        keys = _spread(b, nk) if case["ragged"] else [nk] * b
        return [(n, min(n, nq) if nq <= 17 else max(1, nq * n // nk)) for n in keys]
    held = case["context"]
    return [(n + (i * 997 % (held + 1) if i % 2 else 0), n)
            for i, n in enumerate(_spread(b, case["tokens"]))]


def _order(case, seed):
    """The requests in the order in which they came."""
    pairs = _requests(case)
    order = torch.randperm(len(pairs), generator=torch.Generator().manual_seed(int(seed)))
    return [pairs[i] for i in order.tolist()]


def _ints(x):
    return torch.tensor(x, device=_device(), dtype=torch.int32)


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = _gen(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    st = SimpleNamespace(kind=kind, case=case)
    b, d, hk = case["batch"], case["dim"], case["kv_heads"]
    if kind in ("append", "read"):
        n = case["tokens"]
        st.first, st.count = (list(x) for x in zip(*_order(case, seed)))
        st.starts = _ints(st.first)
        st.ends = _ints([s + t for s, t in zip(st.first, st.count)])
        _cache(st, g, [s + t for s, t in zip(st.first, st.count)], case["block"])
        st.lo = list(st.first)
        if kind == "append":
            st.at = _offsets(st.count) if case["packed"] else [i * n for i in range(b + 1)]
            st.offsets = _ints(st.at) if case["packed"] else None
            shape = (st.at[-1], hk, d) if case["packed"] else (b, n, hk, d)
            st.k, st.v = _projected(g, shape, dt), _projected(g, shape, dt)
            # read back from the start of the blocks that the append changes
            st.lo = [s // case["block"] * case["block"] for s in st.first]
        st.los = _ints(st.lo)
        st.size = max(s + t - lo for s, t, lo in zip(st.first, st.count, st.lo))
        # rows behind a request's last key stay as the caller left them
        st.out = [torch.zeros(b, st.size, hk, d, device=_device(), dtype=dt) for _ in range(2)]
        return st
    h = case["heads"]
    if kind == "cached":
        nq = case["queries"]
        st.k_len, st.q_len = (list(x) for x in zip(*_order(case, seed)))
        st.k_lens, st.q_lens = _ints(st.k_len), _ints(st.q_len)
        _cache(st, g, st.k_len, case["mark"])
        st.q = _randn(g, (b, nq, h, d), dt)
        # rows behind a request's last query stay as the caller left them
        st.out = torch.zeros(b, nq, h, d, device=_device(), dtype=dt)
        return st
    st.k_len, st.q_len = (list(x) for x in zip(*_order(case, seed)))
    st.q_at, st.k_at = _offsets(st.q_len), _offsets(st.k_len)
    st.q_offs, st.k_offs = _ints(st.q_at), _ints(st.k_at)
    st.q = _randn(g, (st.q_at[-1], h, d), dt)
    st.k = _randn(g, (st.k_at[-1], hk, d), dt)
    st.v = _randn(g, (st.k_at[-1], hk, d), dt)
    return st


# --------------------------------------------------------------------------
# The plain forms

def _place(st, index):
    """Pages and rows of pages of keys ``index`` [B, R] (any valid place past a table)."""
    page = st.case["page"]
    col = (index // page).clamp(max=st.table.shape[1] - 1)
    return st.table.gather(1, col).long().clamp(min=0), index % page


def _plain_append(st, x, codes, scales):
    """The tokens x of every request into the pages ``codes`` and their ``scales``."""
    c = st.case
    dev, bs, h, d = x.device, c["block"], c["kv_heads"], c["dim"]
    start = torch.tensor(st.first, device=dev)[:, None]
    end = start + torch.tensor(st.count, device=dev)[:, None]
    lo = start // bs * bs
    n_blocks = max(-(-(s + n) // bs) - s // bs for s, n in zip(st.first, st.count))
    j = lo + torch.arange(n_blocks * bs, device=dev)
    new, kept = (j >= start) & (j < end), j < start
    page, row = _place(st, j)
    src = torch.tensor(st.at[:-1], device=dev)[:, None] + (j - start).clamp(min=0)
    flat = x.reshape(-1, h, d)
    # (64 bits: quotients beside the border of two codes)
    y = flat[src.clamp(max=flat.shape[0] - 1)].double() * new[..., None, None]
    split = (j.shape[0], n_blocks, bs, h, d)
    most = y.view(split).abs().amax((2, 4))
    block_page, block_row = page[:, ::bs], row[:, ::bs] // bs
    held = kept.view(j.shape[0], n_blocks, bs)[:, :, 0]
    s0 = scales[block_page, block_row].double() * held[..., None]
    if c["code"] == "int8":
        own_s = (most / 127.0).float().double()
    else:
        own_s = _power(torch.ceil(torch.log2(most.clamp(min=FLOOR) / 448.0))).double()
        own_s = torch.where(own_s * 224.0 >= most, own_s / 2, own_s)
        own_s = torch.where(own_s * 448.0 < most, own_s * 2, own_s)
    s = torch.maximum(s0, own_s).clamp(min=FLOOR)
    each = s[:, :, None, :, None]
    y = y.view(split) / each
    old = codes[page, row].double().view(split) * (s0[:, :, None, :, None] / each)
    y = torch.where(kept.view(split[:3])[..., None, None], old, y).view(*j.shape, h, d)
    y = y.round().clamp(-127, 127) if c["code"] == "int8" else y.float().clamp(-448, 448)
    write = new | kept
    codes[page[write], row[write]] = y[write].to(codes.dtype)
    any_new = new.view(j.shape[0], n_blocks, bs).any(2)
    scales[block_page[any_new], block_row[any_new]] = s[any_new].float()


def _values(st, codes, scales, page, row, block):
    """Codes at the pages and rows as the fp32 values that they stand for."""
    return codes[page, row].float() * scales[page, row // block][..., None]


def _plain_read(st):
    dev = st.table.device
    j = torch.tensor(st.lo, device=dev)[:, None] + torch.arange(st.size, device=dev)
    live = j < st.ends[:, None]
    page, row = _place(st, j)
    for out, codes, scales in zip(st.out, (st.kc, st.vc), (st.ks, st.vs)):
        x = _values(st, codes, scales, page, row, st.case["block"]).to(out.dtype)
        out.copy_(torch.where(live[..., None, None], x, out))
    return list(st.out)


def _plain_attention(q, k, v, first, c):
    """q [Lq, H, D], k and v [Lk, Hk, D] (fp32 products), rows first, first + 1, ...;
    returns [Lq, H, D] fp32 and the logarithm of each row's sum [H, Lq]."""
    nq, h, d = q.shape
    nk, hk, _ = k.shape
    g, window, sinks, block = h // hk, c["window"], c["sinks"], c["block"]
    out = torch.empty(nq, h, d, device=q.device)
    lse = torch.empty(h, nq, device=q.device)
    step = max(1, min(nq, 300_000_000 // (h * max(1, min(nk, (window or nk) + sinks + block)))))
    for r0 in range(0, nq, step):
        r1 = min(nq, r0 + step)
        end = (torch.arange(first + r0, first + r1, device=q.device) // block + 1) * block
        ends = [((first + r) // block + 1) * block for r in (r0, r1 - 1)]
        lo, hi = max(0, ends[0] - window) if window else 0, min(ends[1], nk)
        index = torch.cat([torch.arange(min(sinks, lo, nk), device=q.device),
                           torch.arange(lo, max(lo, hi), device=q.device)])
        kk = k.index_select(0, index).float().permute(1, 2, 0).contiguous()
        vv = v.index_select(0, index).float().permute(1, 0, 2).contiguous()
        qq = q[r0:r1].float().reshape(r1 - r0, hk, g, d).permute(1, 2, 0, 3)
        s = torch.matmul(qq.reshape(hk, g * (r1 - r0), d), kk).mul_(1.0 / math.sqrt(d))
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


def _run_own(st, c):
    from cast_amd import ops
    if st.kind in ("append", "read"):
        if st.kind == "append":
            ops.append_cache(st.k, st.v, st.cache, st.starts, offsets=st.offsets)
        k, v = ops.read_cache(st.cache, st.ends, size=st.size, starts=st.los, out=tuple(st.out))
        return [k, v] + ([st.ks, st.vs] if st.kind == "append" else [])
    rows = {"window": c["window"] or None, "sinks": c["sinks"], "block": c["block"]}
    if st.kind == "packed":
        return ops.packed_attention(st.q, st.k, st.v, st.q_offs, k_offsets=st.k_offs, **rows)
    out = ops.paged_attention(st.q, st.cache, st.k_lens, return_lse=c["queries"] == 1,
                              out=st.out, q_lengths=st.q_lens if c["ragged"] else None, **rows)
    return list(out) if c["queries"] == 1 else out


def run(state):
    st, c = state, state.case
    if own:
        return _run_own(st, c)
    if st.kind == "read":
        return _plain_read(st)
    if st.kind == "append":
        _plain_append(st, st.k, st.kc, st.ks)
        _plain_append(st, st.v, st.vc, st.vs)
        return _plain_read(st) + [st.ks, st.vs]
    if st.kind == "packed":
        out = torch.empty_like(st.q)
        for q0, q1, k0, k1 in zip(st.q_at, st.q_at[1:], st.k_at, st.k_at[1:]):
            out[q0:q1] = _plain_attention(st.q[q0:q1], st.k[k0:k1], st.v[k0:k1],
                                          (k1 - k0) - (q1 - q0), c)[0].to(out.dtype)
        return out
    lse = torch.zeros(c["batch"], c["heads"], c["queries"], device=st.q.device)
    for b, (nk, nq) in enumerate(zip(st.k_len, st.q_len)):
        j = torch.arange(nk, device=st.q.device)
        page, row = st.table[b].long()[j // c["page"]], j % c["page"]
        k, v = (_values(st, x, s, page, row, c["mark"])
                for x, s in ((st.kc, st.ks), (st.vc, st.vs)))
        o, m = _plain_attention(st.q[b, :nq], k, v, nk - nq, c)
        st.out[b, :nq] = o.to(st.out.dtype)
        lse[b, :, :nq] = m
    return [st.out, lse] if c["queries"] == 1 else st.out


# --------------------------------------------------------------------------
# 64 bits

def _nearest(x, code):
    """x rounded to the values of the code, ties to even."""
    if code == "int8":
        return torch.round(x)
    # 1 + 3 bits, the smallest normal number 2^-6
    power = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = _power(power - 3).double()
    return torch.round(x / step) * step


def _exact_append(st, x, codes, scales):
    """(codes in 64 bits, scales in 64 bits) after the append, one block at a time."""
    c = st.case
    bs, page, code = c["block"], c["page"], c["code"]
    y, s = codes.double(), scales.double()
    rows = x.reshape(-1, c["kv_heads"], c["dim"])
    for b, (first, count) in enumerate(zip(st.first, st.count)):
        table = st.table[b].tolist()
        for block in range(first // bs, -(-(first + count) // bs)):
            t0, t1 = max(block * bs, first), min((block + 1) * bs, first + count)
            new = rows[st.at[b] + t0 - first:st.at[b] + t1 - first].double()
            pg, at = table[block * bs // page], block * bs % page
            old = s[pg, at // bs].clone() if t0 > block * bs else torch.zeros_like(s[pg, 0])
            top = new.abs().amax((0, 2))
            if code == "int8":
                mine = (top / 127).float().double()    # (a scale is held in fp32)
            else:
                m, e = torch.frexp(top)                # top = m 2^e, m in [1/2, 1)
                mine = _power(torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)).double()
            now = torch.stack([old, mine, torch.full_like(old, FLOOR)]).amax(0)
            kept = y[pg, at:at + t0 - block * bs]
            y[pg, at:at + t0 - block * bs] = _nearest(kept * (old / now)[:, None], code)
            y[pg, at + t0 - block * bs:at + t1 - block * bs] = _nearest(new / now[:, None], code)
            s[pg, at // bs] = now
    return y, s


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
            use = torch.cat([keys[:min(sinks, start)], keys[start:stop]])
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
    dev, page = _device(), case.get("page")
    if st.kind == "packed":
        out = torch.empty(st.q.shape, device=dev, dtype=torch.float64)
        for b, nq in enumerate(st.q_len):
            q0, k0, nk = st.q_at[b], st.k_at[b], st.k_len[b]
            out[q0:q0 + nq] = _exact_attention(st.q[q0:q0 + nq], st.k[k0:k0 + nk],
                                               st.v[k0:k0 + nk], nk - nq, case)[0]
        return out
    block = case["mark"] if st.kind == "cached" else case["block"]
    held = [(st.kc, st.ks), (st.vc, st.vs)]
    if st.kind == "append":
        held = [_exact_append(st, x, *h) for x, h in zip((st.k, st.v), held)]

    def keys_of(b, lo, hi):
        j = torch.arange(lo, hi, device=dev)
        pg = st.table[b].long()[j // page]
        return [y[pg, j % page].double() * s[pg, j % page // block].double()[..., None]
                for y, s in held]

    if st.kind in ("append", "read"):
        out = [torch.zeros(x.shape, device=dev, dtype=torch.float64) for x in st.out]
        for b, (lo, first, n) in enumerate(zip(st.lo, st.first, st.count)):
            for x, y in zip(out, keys_of(b, lo, first + n)):
                x[b, :first + n - lo] = y
        return out + ([s for _, s in held] if st.kind == "append" else [])
    out = torch.zeros(st.out.shape, device=dev, dtype=torch.float64)
    lse = torch.zeros(case["batch"], case["heads"], case["queries"], device=dev,
                      dtype=torch.float64)
    for b, (nk, nq) in enumerate(zip(st.k_len, st.q_len)):
        k, v = keys_of(b, 0, nk)
        out[b, :nq], lse[b, :, :nq] = _exact_attention(st.q[b, :nq], k, v, nk - nq, case)
    return [out, lse] if case["queries"] == 1 else out


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
    d, hk = case["dim"], case["kv_heads"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] in ("append", "read"):
        n = sum(t for _, t in _requests(case))
        # read: a code in, a value out; append: a value in, a code out, and that read
        each = (1 + size) * (2 if case["kind"] == "append" else 1)
        scales = 4.0 / case["block"] * (2 if case["kind"] == "append" else 1)
        return {"bytes": 2 * n * hk * (d * each + scales), "flops": 4 * n * hk * d}
    h = case["heads"]
    each = d + 4.0 / case["mark"] if case["kind"] == "cached" else 2.0 * d
    total = union = rows = 0
    for nk, nq in _requests(case):
        t, u = _row_keys(case, nk, nq)
        total, union, rows = total + t, union + u, rows + nq
    return {"bytes": 2 * rows * h * d * size + 2 * union * hk * each,
            "flops": 4 * total * h * d}
