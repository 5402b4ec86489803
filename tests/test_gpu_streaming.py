"""The streaming operators together, as a decoder runs them: norms and rotations into a paged
cache, attention over it in chunks and then by tokens, captured steps, a rolling cache; and
what a long cache brings: offsets past 32 bits, storage full of values that are no numbers.

Tolerances: each operator's bound of the 64-bit oracle, on what the one before it wrote."""
import math

import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _same(got, ref, tol, what):
    """Within the bound; NaN and infinities where the oracle has them."""
    got = got.double()
    off = (got - ref).abs()
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    worst = torch.where(same, torch.zeros_like(off), off - tol).max().item()
    assert worst <= 0.0, f"{what}: {worst} past the bound"


def _int(dev, *v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Decoder:
    """One layer's attention over a paged cache: its inputs of every position, what the
    operators wrote, and the checks of both."""

    def __init__(self, dev, B, L, Hq, Hk, D, page, window, sinks, block, dtype, table, pages):
        from cast_amd import ops
        from cast_amd.rotary import rotary_plan
        g = torch.Generator().manual_seed(L + D)
        self.q, self.k, self.v = (torch.randn(B, L, h, D, generator=g).to(dtype).to(dev)
                                  for h in (Hq, Hk, Hk))
        self.w = (1 + 0.1 * torch.randn(2, D, generator=g)).to(dtype).to(dev)
        self.plan, self.freq = rotary_plan(D, device=dev), so.frequencies(D)
        self.cache = ops.PagedCache(
            torch.full((pages, page, Hk, D), float("nan"), dtype=dtype, device=dev),
            torch.full((pages, page, Hk, D), float("nan"), dtype=dtype, device=dev),
            table.to(dev))
        self.rule, self.L, self.dev = (window, sinks, block), L, dev
        self.out = torch.zeros_like(self.q)
        self.kw = dict(window=window or None, sinks=sinks, block=block)
        # what the cache has held, by position
        self.keys = torch.zeros(B, L, Hk, D, dtype=dtype, device=dev)
        self.turned = torch.zeros_like(self.q)

    def step(self, q, k, v, positions, starts, fed, ends, **kw):
        from cast_amd import ops
        qr, _ = ops.norm_rope(q, k, positions, self.plan, q_weight=self.w[0], k_weight=self.w[1],
                              v=v, cache=self.cache, starts=starts, lengths=fed)
        return qr, ops.paged_attention(qr, self.cache, ends, **self.kw, **kw)

    def feed(self, start, n):
        """Positions start[b] .. start[b] + n[b] of every request."""
        T = max(n)
        at = torch.tensor(start)[:, None] + torch.arange(T)
        rows = at.clamp_max(self.L - 1).to(self.dev)
        b = torch.arange(len(n), device=self.dev)[:, None]
        starts, fed = _int(self.dev, *start), _int(self.dev, *n)
        qr, out = self.step(self.q[b, rows], self.k[b, rows], self.v[b, rows], rows, starts, fed,
                            starts + fed, q_lengths=fed)
        page = self.cache.k.shape[1]
        for i, (s, m) in enumerate(zip(start, n)):
            self.out[i, s:s + m], self.turned[i, s:s + m] = out[i, :m], qr[i, :m]
            j = torch.arange(s, s + m, device=self.dev)
            self.keys[i, s:s + m] = self.cache.k[self.cache.table[i, j // page].long(), j % page]

    def check(self, ends):
        window, sinks, block = self.rule
        for i, end in enumerate(ends):
            pos = torch.arange(end, device=self.dev)
            for got, x, w in ((self.turned, self.q, self.w[0]), (self.keys, self.k, self.w[1])):
                ref, size = so.rope(so.norm(x[i:i + 1, :end], w, 1e-6, False), pos, *self.freq,
                                    False)
                _same(got[i:i + 1, :end], ref, so.rope_bound(ref, size, got.dtype, norm=True),
                      f"norm and rotation of request {i}")
            seen = so.visible(end, end, window, sinks, block, device=self.dev)
            ref, _, tol, _ = so.attention(self.turned[i, :end], self.keys[i, :end],
                                          self.v[i, :end], seen, self.q.shape[-1] ** -0.5,
                                          self.q.dtype)
            _same(self.out[i, :end], ref, tol, f"attention of request {i}")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hk,D,page,window,sinks", [
    (8, 2, 128, 16, 0, 0), (6, 3, 64, 48, 100, 7), (4, 4, 128, 64, 250, 64)])
def test_chunks_then_tokens(dev, dtype, Hq, Hk, D, page, window, sinks):
    """A ragged batch: chunks of own lengths, then single tokens, one request idle at
    times; every position against the oracle."""
    B, L, M = 3, 700, -(-700 // page)
    table = torch.randperm(B * M, generator=torch.Generator().manual_seed(page)).int().view(B, M)
    d = Decoder(dev, B, L, Hq, Hk, D, page, window, sinks, 1, dtype, table, B * M)
    at = [0, 0, 0]
    for n in ([300, 17, 129], [211, 90, 1], [1, 1, 33], [0, 1, 1], [1, 0, 1], [1, 1, 1]):
        d.feed(at, n)
        at = [a + b for a, b in zip(at, n)]
    d.check(at)


def test_rolling_pages(dev):
    """Frames through a cache that holds the first keys' page and a ring of pages for the
    window: the table is written once, old pages are overwritten."""
    B, frame, frames, page, Hq, Hk, D = 2, 48, 14, 16, 4, 4, 128
    window, sinks = 4 * frame, 16
    M, ring = frame * frames // page, (window + frame) // page
    table = torch.empty(B, M, dtype=torch.int32)
    for b in range(B):
        for i in range(M):
            table[b, i] = b * (ring + 1) + (0 if i == 0 else 1 + i % ring)
    d = Decoder(dev, B, frame * frames, Hq, Hk, D, page, window, sinks, frame, BF, table,
                B * (ring + 1))
    for f in range(frames):
        d.feed([f * frame] * B, [frame] * B)
    d.check([frame * frames] * B)


def test_captured_steps(dev):
    """One captured step of a token, replayed token by token over device-held positions and
    lengths, with eager steps of another layer between: bit for bit the eager steps."""
    B, L, Hq, Hk, D, page, M = 2, 200, 8, 2, 128, 16, 13
    table = torch.arange(B * M, dtype=torch.int32).view(B, M)
    made = [Decoder(dev, B, L, Hq, Hk, D, page, 90, 4, 1, BF, table, B * M) for _ in range(2)]
    for d in made:
        d.feed([0, 0], [120, 77])
    eager, d = made
    q, k, v = (t[:, :1].clone() for t in (d.q, d.k, d.v))
    starts, one = _int(dev, 120, 77), _int(dev, 1, 1)
    positions, ends = starts[:, None].clone(), starts + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d.step(q, k, v, positions, starts, one, ends, max_length=L)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, out = d.step(q, k, v, positions, starts, one, ends, max_length=L)
    at = [120, 77]
    for i in range(20):
        rows = torch.tensor(at, device=dev)
        b = torch.arange(B, device=dev)
        for t, x in ((q, d.q), (k, d.k), (v, d.v)):
            t.copy_(x[b, rows][:, None])
        starts.copy_(rows)
        positions.copy_(rows[:, None])
        ends.copy_(rows + 1)
        graph.replay()
        want_q, want = eager.step(q, k, v, positions, starts, one, ends, max_length=L)
        torch.cuda.synchronize()
        assert torch.equal(qr, want_q) and torch.equal(out, want), i
        at = [n + 1 for n in at]
    live = ~torch.isnan(d.cache.k)
    assert torch.equal(live, ~torch.isnan(eager.cache.k))
    assert torch.equal(d.cache.k[live], eager.cache.k[live])


@pytest.mark.parametrize("Lq,n_split", [(700, None), (700, 3), (4, None), (4, 2)])
@pytest.mark.parametrize("paged", [False, True])
def test_storage_full_of_no_numbers(dev, Lq, n_split, paged):
    """Every third key's value holds a NaN or an infinity in a channel of its own, the first
    key's among them: what a row sees it carries, and only there."""
    from cast_amd import ops
    Lk, Hq, Hk, D, page = 700, 4, 2, 128, 64
    g = torch.Generator().manual_seed(Lq)
    q, k, v = (torch.randn(1, n, h, D, generator=g).to(BF) for n, h in
               ((Lq, Hq), (Lk, Hk), (Lk, Hk)))
    for j in range(0, Lk, 3):
        v[0, j, j % Hk, j * 5 % D] = (float("nan"), float("inf"), -float("inf"))[j % 9 // 3]
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    for window, sinks in ((0, 0), (40, 2)):
        kw = dict(window=window or None, sinks=sinks, return_lse=True, n_split=n_split)
        if paged:
            pad = torch.full((1, 704 - Lk, Hk, D), float("nan"), dtype=BF, device=dev)
            cache = ops.PagedCache(*(torch.cat([t, pad], 1).view(11, page, Hk, D) for t in (k, v)),
                                   torch.arange(11, dtype=torch.int32, device=dev)[None])
            out, lse = ops.paged_attention(q, cache, _int(dev, Lk), **kw)
        else:
            out, lse = ops.window_attention(q, k, v, **kw)
        seen = so.visible(Lq, Lk, window, sinks, 1, device=dev)
        ref, rlse, tol, ltol = so.attention(q[0], k[0], v[0], seen, D ** -0.5, BF)
        _same(out[0], ref, tol, (window, "rows"))
        _same(lse[0], rlse, ltol, (window, "sums"))


def _far(dev, n, gap, D):
    """Rows of D values, gap elements apart, in one block of storage."""
    free = torch.cuda.mem_get_info()[0]
    if free < 2 * n * gap + (8 << 30):
        pytest.skip("not enough memory")
    return torch.empty((n - 1) * gap + 4 * D, dtype=BF, device=dev)


@pytest.mark.parametrize("Lq", [1, 150])
def test_offsets_past_32_bits(dev, Lq):
    """Keys and queries whose rows lie further apart than 32 bits count, in elements and in
    bytes."""
    from cast_amd import ops
    D, Lk, gap = 128, 300, 1 << 24
    store = _far(dev, Lk, gap, D)
    g = torch.Generator().manual_seed(Lq)
    q, k, v = (torch.randn(1, n, 1, D, generator=g).to(BF).to(dev) for n in (Lq, Lk, Lk))
    fq, fk, fv, fo = (store[i * D:].as_strided((1, n, 1, D), (gap * n, gap, D, 1),
                                               i * D) for i, n in enumerate((Lq, Lk, Lk, Lq)))
    fq.copy_(q), fk.copy_(k), fv.copy_(v)
    for window, sinks in ((None, 0), (70, 5)):
        want = ops.window_attention(q, k, v, window=window, sinks=sinks)
        got = ops.window_attention(fq, fk, fv, window=window, sinks=sinks, out=fo)
        assert got.data_ptr() == fo.data_ptr() and torch.equal(got, want)
    del fq, fk, fv, fo, store
    torch.cuda.empty_cache()


def test_pages_past_32_bits(dev):
    """Pages further apart than 32 bits count: rows go to them and are read from them."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    D, Hq, Hk, page, pages, L = 128, 4, 2, 16, 9, 120
    gap = 1 << 30
    store = _far(dev, pages, gap, page * Hk * D)
    fk, fv = (store.as_strided((pages, page, Hk, D), (gap, Hk * D, D, 1), i * page * Hk * D)
              for i in range(2))
    near = [torch.empty(pages, page, Hk, D, dtype=BF, device=dev) for _ in range(2)]
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int()[None].to(dev)
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, L, h, D, generator=g).to(BF).to(dev) for h in (Hq, Hk, Hk))
    plan, pos = rotary_plan(D, device=dev), torch.arange(L, device=dev)
    far, near = ops.PagedCache(fk, fv, table), ops.PagedCache(*near, table)
    res = []
    for cache in (far, near):
        qr, _ = ops.norm_rope(q, k, pos, plan, v=v, cache=cache)
        lens = _int(dev, L)
        res.append([qr, ops.paged_attention(qr, cache, lens),
                    ops.paged_attention(qr[:, -1:], cache, lens, window=50, sinks=4)])
    assert all(torch.equal(a, b) for a, b in zip(*res))
    j = torch.arange(L, device=dev)
    at = table[0, j // page].long(), j % page
    assert torch.equal(fk[at], near.k[at]) and torch.equal(fv[at], v[0])
    del fk, fv, far, cache, store
    torch.cuda.empty_cache()


@pytest.mark.parametrize("window,sinks", [(1, 1), (33, 33), (64, 31), (100, 0), (0, 0)])
def test_units_of_every_length(dev, window, sinks):
    """Few rows in units of one wavefront: requests of 0 to 255 keys, so that windows and
    first keys begin and end anywhere in a tile."""
    from cast_amd import _lib
    B, T, Hq, Hk, D, page = 256, 2, 4, 2, 64, 16
    g = torch.Generator().manual_seed(window)
    q = torch.randn(B, T, Hq, D, generator=g).to(BF).to(dev)
    k, v = (torch.randn(1, B, Hk, D, generator=g).to(BF).to(dev) for _ in range(2))
    table = torch.arange(B // page, dtype=torch.int32, device=dev).expand(B, -1).contiguous()
    lens = torch.arange(B, dtype=torch.int32, device=dev)
    out, lse = _lib.torch_ops().window_attention(
        q, k.view(-1, page, Hk, D), v.view(-1, page, Hk, D), table, None, lens, window, sinks, 1,
        None, True, None, 0, -1)
    for n in range(B):
        seen = so.visible(T, n, window, sinks, 1, device=dev)
        ref, rlse, tol, ltol = so.attention(q[n], k[0, :n], v[0, :n], seen, D ** -0.5, BF)
        _same(out[n], ref, tol, (n, "rows"))
        _same(lse[n], rlse, ltol, (n, "sums"))


def test_calls_with_nothing_to_do(dev):
    """No requests, no positions, no heads of channels: empty results or a refusal, and
    nothing else written."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    plan = rotary_plan(64, device=dev)
    x = torch.randn(2, 3, 4, 64, device=dev).to(BF)
    pos = torch.arange(3, device=dev)
    pages = torch.zeros(4, 16, 4, 64, device=dev, dtype=BF)
    table = torch.zeros(2, 2, device=dev, dtype=torch.int32)
    cache = ops.PagedCache(pages, pages.clone(), table)
    q, k = ops.norm_rope(x[:0], x[:0], pos, plan)
    assert q.shape == k.shape == (0, 3, 4, 64)
    q, k = ops.norm_rope(x[:, :0], x[:, :0], pos[:0], plan, v=x[:, :0], cache=cache)
    assert q.shape == (2, 0, 4, 64) and k is None and (pages == 0).all()
    out, lse = ops.window_attention(x[:0], x[:0], x[:0], return_lse=True)
    assert out.shape == (0, 3, 4, 64) and lse.shape == (0, 4, 3)
    out = ops.paged_attention(x[:, :0], cache, _int(dev, 5, 5))
    assert out.shape == (2, 0, 4, 64)
    with pytest.raises(RuntimeError, match="no channels"):
        ops.window_attention(x[..., :0], x[..., :0], x[..., :0])
    with pytest.raises(ValueError):
        ops.window_attention(x, x[:, :, :0], x[:, :, :0])
    with pytest.raises(RuntimeError, match="no heads"):
        ops.norm_rope(x, x[:, :, :0], pos, plan)


def test_refusals_beside_a_cache(dev):
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    plan = rotary_plan(64, device=dev)
    x = torch.randn(2, 3, 4, 64, device=dev).to(BF)
    pos = torch.arange(3, device=dev)
    pages = torch.zeros(4, 16, 4, 64, device=dev, dtype=BF)
    table = torch.zeros(2, 2, device=dev, dtype=torch.int32)
    cache = ops.PagedCache(pages, pages.clone(), table)
    starts = _int(dev, 0, 0)
    for kw, err in ((dict(v=x), ValueError), (dict(cache=cache), ValueError),
                    (dict(starts=starts), ValueError),
                    (dict(v=x, cache=cache, k_out=x.clone()), ValueError),
                    (dict(v=x.float(), cache=cache), TypeError),
                    (dict(v=x[:, :2], cache=cache), RuntimeError),
                    (dict(v=x, cache=cache, starts=starts.long()), RuntimeError),
                    (dict(v=x, cache=cache, starts=starts[:1]), RuntimeError),
                    (dict(v=x, cache=cache._replace(table=table[:1])), RuntimeError),
                    (dict(v=x, cache=cache._replace(k=pages[:, :, :2])), RuntimeError),
                    (dict(v=x, cache=cache._replace(v=pages.half())), RuntimeError),
                    (dict(lengths=starts.cpu()), RuntimeError)):
        with pytest.raises(err):
            ops.norm_rope(x, x, pos, plan, **kw)
    assert (pages == 0).all()


@pytest.mark.parametrize("Lq", [1, 40])
def test_limits_of_the_rule(dev, Lq):
    """Windows, first keys and blocks past every position, up to 64 bits: all keys in order,
    or a block's."""
    from cast_amd import ops
    g = torch.Generator().manual_seed(Lq)
    q, k, v = (torch.randn(1, n, 2, 64, generator=g).to(BF).to(dev) for n in (Lq, 90, 90))
    want = ops.window_attention(q, k, v)
    for most in (90, 1 << 30, (1 << 63) - 1):
        assert torch.equal(ops.window_attention(q, k, v, window=most), want)
        assert torch.equal(ops.window_attention(q, k, v, window=most, sinks=most), want)
        assert torch.equal(ops.window_attention(q, k, v, window=5, sinks=most), want)
        assert torch.equal(ops.window_attention(q, k, v, block=most),
                           ops.window_attention(q, k, v, causal=False))
