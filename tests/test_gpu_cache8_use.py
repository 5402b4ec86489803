"""The 8-bit cache and packed attention as a server uses them together: prompts of different
lengths, packed, then tokens one by one and in chunks, dense reads beside them; captured steps;
calls on two streams; and what the wrappers refuse.

The cache has to hold exactly what the oracle's appends give for the tokens that were appended;
attention is held to the oracle's bounds (``cache_oracle.attention``,
``streaming_oracle.attention``)."""
import pytest
import torch

from oracle import cache_oracle as co
from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
I8, F8 = torch.int8, torch.float8_e4m3fn


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _cache(dev, code, B, pages, page, block, H, D, width, seed=0):
    """An empty cache (its memory holds whatever was there) and a table of own pages."""
    from cast_amd.ops import QuantizedCache
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(-100, 100, (pages, page, H, D), generator=g, dtype=torch.int8).to(dev)
             for _ in range(2)]
    scales = [torch.rand(pages, page // block, H, generator=g).to(dev) for _ in range(2)]
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int().to(dev)
    return QuantizedCache(codes[0].view(code), codes[1].view(code), *scales, table)


class Held:
    """What a cache holds, in 64 bits: appended to beside it."""

    def __init__(self, cache):
        self.block, self.code = cache.k.shape[1] // cache.k_scale.shape[1], cache.k.dtype
        self.table = cache.table.cpu()
        self.v = [{"v": torch.nan_to_num(t.cpu().float()).double(), "code": self.code}
                  for t in (cache.k, cache.v)]
        self.s = [t.cpu().double() for t in (cache.k_scale, cache.v_scale)]

    def append(self, b, k, v, first):
        for kv, x in enumerate((k, v)):
            co.append(self.v[kv], self.s[kv], self.table[b].tolist(), self.block, x.cpu(), first)

    def keys(self, kv, b, n):
        j = torch.arange(n)
        slots = self.v[kv]["v"].shape[1]
        page = self.table[b, j // slots].long()
        return (self.v[kv]["v"][page, j % slots]
                * self.s[kv][page, j % slots // self.block][..., None])

    def check(self, cache, lens):
        """Codes and scales of every request's keys are the oracle's."""
        for kv, (c, s) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
            c, s, slots = c.cpu().float().double(), s.cpu().double(), c.shape[1]
            for b, n in enumerate(lens):
                j = torch.arange(n)
                page = self.table[b, j // slots].long()
                assert torch.equal(c[page, j % slots], self.v[kv]["v"][page, j % slots]), (kv, b)
                blk = j % slots // self.block
                assert torch.equal(s[page, blk], self.s[kv][page, blk]), (kv, b)


def _check(out, q, held, b, n, window, sinks, dev):
    """Rows of one request over its n keys, the queries its last positions."""
    seen = so.visible(q.shape[0], n, window, sinks, 1)
    top = (127.0 if held.code == I8 else 448.0) * float(held.s[1].max())
    ref, _, tol, _ = (t.cpu() for t in co.attention(
        q.to(dev), held.keys(0, b, n).to(dev), held.keys(1, b, n).to(dev), top, seen.to(dev),
        q.shape[-1] ** -0.5, q.dtype))
    worst = ((out.cpu().double() - ref).abs() - tol).max().item()
    assert worst <= 0.0, (b, n, worst)


@pytest.mark.parametrize("code,dtype,window,sinks", [(I8, BF, 0, 0), (F8, HF, 150, 4)])
def test_a_served_batch(dev, code, dtype, window, sinks):
    """Packed prompts are rotated, attended and appended; then steps of one token and a chunk of
    five append and attend over the cache; a dense read gives the held keys to a dense call."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    Hq, Hk, D, page, block, width = 4, 2, 128, 64, 32, 6
    count = [130, 1, 0, 67, 260]
    B, T = len(count), sum(count)
    at = [0]
    for n in count:
        at.append(at[-1] + n)
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)
    plan = rotary_plan(D, device=dev)
    cache = _cache(dev, code, B, 40, page, block, Hk, D, width)
    held = Held(cache)
    rows = dict(window=window or None, sinks=sinks)

    q, k, v = rand(1, T, Hq, D), rand(1, T, Hk, D), rand(1, T, Hk, D)
    pos = torch.cat([torch.arange(n) for n in count]).to(dev)[None]
    q, k = ops.norm_rope(q, k, pos, plan)
    offs = _i32(at, dev)
    out = ops.packed_attention(q[0], k[0], v[0], offs, **rows)
    assert ops.append_cache(k[0], v[0], cache, offsets=offs) is cache
    for b, n in enumerate(count):
        s = slice(at[b], at[b + 1])
        held.append(b, k[0, s], v[0, s], 0)
        if n == 0:
            continue
        seen = so.visible(n, n, window, sinks, 1)
        ref, _, tol, _ = (t.cpu() for t in so.attention(
            q[0, s], k[0, s], v[0, s], seen.to(dev), D ** -0.5, dtype))
        worst = ((out[s].cpu().double() - ref).abs() - tol).max().item()
        assert worst <= 0.0, (b, worst)
    lens = list(count)
    held.check(cache, lens)

    for new in (1, 1, 5, 1):
        q, k, v = rand(B, new, Hq, D), rand(B, new, Hk, D), rand(B, new, Hk, D)
        starts = _i32(lens, dev)
        q, k = ops.norm_rope(q, k, starts[:, None] + torch.arange(new, device=dev), plan)
        ops.append_cache(k, v, cache, starts)
        out = ops.paged_attention(q, cache, starts + new, **rows)
        for b in range(B):
            held.append(b, k[b], v[b], lens[b])
            lens[b] += new
            _check(out[b], q[b].cpu(), held, b, lens[b], window, sinks, dev)
        held.check(cache, lens)

    # the keys as a dense call reads them: rounded once, as the oracle's values are
    size = max(lens)
    dense = tuple(torch.zeros(B, size, Hk, D, dtype=dtype, device=dev) for _ in range(2))
    ops.read_cache(cache, _i32(lens, dev), size=size, out=dense)
    for b, n in enumerate(lens):
        for kv in range(2):
            assert torch.equal(dense[kv][b, :n].cpu(), held.keys(kv, b, n).to(dtype)), (kv, b)
            assert (dense[kv][b, n:] == 0).all()
    q = rand(B, 3, Hq, D)
    out = ops.window_attention(q, *dense, k_lengths=_i32(lens, dev), **rows)
    for b, n in enumerate(lens):
        seen = so.visible(3, n, window, sinks, 1)
        ref, _, tol, _ = (t.cpu() for t in so.attention(
            q[b], dense[0][b, :n], dense[1][b, :n], seen.to(dev), D ** -0.5, dtype))
        assert ((out[b].cpu().double() - ref).abs() - tol).max().item() <= 0.0, b


def test_chunks_and_tokens_hold_the_same_scales(dev):
    """A prompt appended whole, in chunks and by token: the scales are the largest of what each
    block got, so they agree; codes differ by the roundings that growing scales cost alone."""
    from cast_amd import ops
    B, H, D, n = 2, 2, 64, 90
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(B, n, H, D, generator=g).to(BF).to(dev) for _ in range(2))
    scales = []
    for step in (n, 17, 1):
        cache = _cache(dev, I8, B, 16, 32, 16, H, D, 4)
        held = Held(cache)
        for t in range(0, n, step):
            m = min(step, n - t)
            ops.append_cache(k[:, t:t + m], v[:, t:t + m], cache, _i32([t] * B, dev))
            for b in range(B):
                held.append(b, k[b, t:t + m], v[b, t:t + m], t)
        held.check(cache, [n] * B)
        blocks = [(b, r) for b in range(B) for r in range(n // 16)]
        scales.append(torch.stack([cache.k_scale[cache.table[b, r // 2].item(), r % 2]
                                   for b, r in blocks]))
    assert torch.equal(scales[0], scales[1]) and torch.equal(scales[0], scales[2])


def test_a_captured_step(dev):
    """A step's rotation, append and attention in one graph: every replay is the eager step's."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    B, Hq, Hk, D, new = 3, 8, 2, 64, 2
    plan = rotary_plan(D, device=dev)
    caches = [_cache(dev, I8, B, 60, 32, 32, Hk, D, 20, seed=3) for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    x = [torch.zeros(B, new, h, D, dtype=BF, device=dev) for h in (Hq, Hk, Hk)]
    starts = _i32([0] * B, dev)
    outs = [torch.zeros(B, new, Hq, D, dtype=BF, device=dev) for _ in range(2)]

    def step(i):
        q, k = ops.norm_rope(x[0], x[1], starts[:, None] + torch.arange(new, device=dev), plan)
        ops.append_cache(k, x[2], caches[i], starts)
        ops.paged_attention(q, caches[i], starts + new, out=outs[i])

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(0)
    stream.synchronize()
    step(1)  # (the other cache gets the same tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    for at in ([0, 500, 31], [2, 502, 33], [4, 504, 35], [6, 506, 37]):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        starts.copy_(_i32(at, dev))
        graph.replay()
        step(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]), at
    for a, b in zip(caches[0], caches[1]):
        if a.dtype == I8:  # (rows behind a request's keys were alike from the start)
            assert torch.equal(a, b)


def test_calls_on_two_streams(dev):
    """Calls beside each other use memory of their own."""
    from cast_amd import ops
    B, Hq, Hk, D = 2, 8, 2, 128
    cache = _cache(dev, I8, B, 400, 32, 32, Hk, D, 190)
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(B, 6000, Hk, D, generator=g).to(BF).to(dev) for _ in range(2))
    ops.append_cache(k, v, cache)
    q = [torch.randn(B, 1, Hq, D, generator=g).to(BF).to(dev) for _ in range(2)]
    p = [torch.randn(900, Hq, D, generator=g).to(BF).to(dev) for _ in range(2)]
    pk, pv = k[0, :900], v[0, :900]
    offs, lens = _i32([0, 200, 900], dev), _i32([6000, 5000], dev)
    call = lambda i: (ops.paged_attention(q[i], cache, lens),
                      ops.packed_attention(p[i], pk, pv, offs, n_split=3))
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i])), i


def test_refusals(dev):
    from torch.autograd import forward_ad
    from cast_amd import ops
    B, Hk, D = 2, 2, 64
    cache = _cache(dev, I8, B, 8, 32, 16, Hk, D, 3)
    was = [t.clone() for t in cache]
    x = torch.randn(B, 4, Hk, D, device=dev).to(BF)
    lens = _i32([3, 4], dev)
    grad = torch.zeros(B, 4, Hk, D, device=dev, requires_grad=True)
    wide = torch.zeros(8, 32, 1, D, device=dev, dtype=I8).expand(8, 32, Hk, D)
    c = cache._replace
    for err, call in (
            (TypeError, lambda: ops.append_cache(x.int(), x.int(), cache)),
            (TypeError, lambda: ops.append_cache(x, x.float(), cache)),
            (TypeError, lambda: ops.append_cache(x, x, c(k=x.new_zeros(8, 32, Hk, D)))),
            (TypeError, lambda: ops.append_cache(x, x, c(v=cache.v.view(F8)))),
            (TypeError, lambda: ops.append_cache(x, x, c(k_scale=cache.k_scale.double()))),
            (ValueError, lambda: ops.append_cache(x, x[:, :3], cache)),
            (ValueError, lambda: ops.append_cache(x[:, :, :1], x[:, :, :1], cache)),
            (ValueError, lambda: ops.append_cache(x[..., :32], x[..., :32], cache)),
            (ValueError, lambda: ops.append_cache(x.transpose(2, 3), x.transpose(2, 3), cache)),
            (ValueError, lambda: ops.append_cache(x[0], x[0], cache)),
            (ValueError, lambda: ops.append_cache(x, x, cache, offsets=_i32([0, 2, 4], dev))),
            (ValueError, lambda: ops.append_cache(x[0], x[0], cache, lengths=lens,
                                                  offsets=_i32([0, 2, 4], dev))),
            (ValueError, lambda: ops.append_cache(x, x, c(k_scale=cache.k_scale[:, :1].clone()))),
            (ValueError, lambda: ops.append_cache(x, x, c(
                k_scale=torch.zeros(8, 4, Hk, device=dev),
                v_scale=torch.zeros(8, 4, Hk, device=dev)))),  # blocks of 8 slots
            (RuntimeError, lambda: ops.append_cache(x, x, c(table=cache.table[:1]))),
            (RuntimeError, lambda: ops.append_cache(x, x, c(table=cache.table.long()))),
            (RuntimeError, lambda: ops.append_cache(x, x, cache, lens[:1])),
            (RuntimeError, lambda: ops.append_cache(x, x, cache, lens.long())),
            (RuntimeError, lambda: ops.append_cache(x, x, cache, lengths=lens.cpu())),
            (RuntimeError, lambda: ops.append_cache(x[0], x[0], cache, offsets=lens.long())),
            (RuntimeError, lambda: ops.append_cache(grad, grad, cache)),
            (RuntimeError, lambda: ops.append_cache(x, x, c(k=wide))),  # expanded codes
            (ValueError, lambda: ops.append_cache(x, x, c(v=cache.k))),
            (ValueError, lambda: ops.append_cache(x, x, c(v_scale=cache.k_scale))),
            (ValueError, lambda: ops.append_cache(
                cache.k.view(-1)[:x.numel() * 2].view(BF).view(x.shape), x, cache)),
            (ValueError, lambda: ops.read_cache(cache, lens, size=-1)),
            (TypeError, lambda: ops.read_cache(cache, lens, size=4, dtype=torch.float64)),
            (RuntimeError, lambda: ops.read_cache(cache, lens.long(), size=4)),
            (RuntimeError, lambda: ops.read_cache(cache, lens[None], size=4)),
            (RuntimeError, lambda: ops.read_cache(cache, lens, size=4, starts=lens[:1])),
            (RuntimeError, lambda: ops.read_cache(cache, lens, size=4, out=(x, x[:, :3]))),
            (RuntimeError, lambda: ops.read_cache(cache, lens, size=4, out=(x, x.float()))),
            (ValueError, lambda: ops.read_cache(cache, lens, size=4, out=(x, x))),
            (ValueError, lambda: ops.read_cache(cache, lens, size=4, out=(x, None))),
            (RuntimeError, lambda: ops.read_cache(
                cache, lens, size=4, out=(x, x[:, :1].clone().expand(B, 4, Hk, D)))),
            (RuntimeError, lambda: ops.read_cache(cache, lens, size=4, out=(grad, grad.clone()))),
            (TypeError, lambda: ops.paged_attention(x.float(), cache, lens)),
            (TypeError, lambda: ops.paged_attention(x, c(v=cache.v.view(F8)), lens)),
            (ValueError, lambda: ops.paged_attention(x, c(k_scale=cache.k_scale[:4]), lens)),
            (TypeError, lambda: ops.paged_attention(x, c(v_scale=cache.v_scale.half()), lens)),
            (ValueError, lambda: ops.paged_attention(x[..., :32], cache, lens)),
            (ValueError, lambda: ops.paged_attention(x[:, :, :1].expand(B, 4, 3, D), cache, lens)),
            (RuntimeError, lambda: ops.paged_attention(x, cache, lens[:1])),
            (RuntimeError, lambda: ops.paged_attention(x, cache, lens, n_split=65)),
            (RuntimeError, lambda: ops.paged_attention(x, c(table=cache.table[:1]), lens)),
            (RuntimeError, lambda: ops.paged_attention(x.clone().requires_grad_(), cache, lens)),
            (ValueError, lambda: ops.paged_attention(
                x, cache, lens, out=cache.v.view(-1)[:x.numel() * 2].view(BF).view(x.shape)))):
        with pytest.raises(err):
            call()
    with pytest.raises(RuntimeError, match="status"):  # codes off a 16-byte boundary
        odd = torch.zeros(8 * 32 * Hk * D + 8, device=dev, dtype=I8)[8:].view(8, 32, Hk, D)
        ops.paged_attention(x, c(k=odd), lens)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.append_cache(d, x, cache), lambda: ops.append_cache(x, d, cache),
                     lambda: ops.paged_attention(d, cache, lens),
                     lambda: ops.read_cache(cache, lens, size=4, out=(x, d))):
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
    assert all(torch.equal(a, b) for a, b in zip(cache, was))


def test_packed_refusals(dev):
    from torch.autograd import forward_ad
    from cast_amd import ops
    q, k, v = (torch.randn(10, h, 64, device=dev).to(BF) for h in (4, 2, 2))
    offs = _i32([0, 4, 10], dev)
    store = torch.randn(11 * 4 * 64, device=dev).to(BF)
    a, b = store[:2560].view(10, 4, 64), store[64:2624].view(10, 4, 64)
    was = store.clone()
    for err, call in (
            (TypeError, lambda: ops.packed_attention(q.float(), k.float(), v.float(), offs)),
            (TypeError, lambda: ops.packed_attention(q, k, v.half(), offs)),
            (ValueError, lambda: ops.packed_attention(q[None], k, v, offs)),
            (ValueError, lambda: ops.packed_attention(q[:, :3], k, v, offs)),
            (ValueError, lambda: ops.packed_attention(q, k, v[:9], offs)),
            (ValueError, lambda: ops.packed_attention(q, k[:9], v[:9], offs)),  # no k_offsets
            (ValueError, lambda: ops.packed_attention(q, k[..., :32], v[..., :32], offs)),
            (ValueError, lambda: ops.packed_attention(q.transpose(1, 2), k, v, offs)),
            (RuntimeError, lambda: ops.packed_attention(q[..., :32], k[..., :32], v[..., :32],
                                                        offs)),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs.long())),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs[None])),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs[:0])),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs[::2])),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs, k_offsets=offs[:2])),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs.cpu())),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs, n_split=65)),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs, out=q[:9].clone())),
            (RuntimeError, lambda: ops.packed_attention(q, k, v, offs, out=q.float())),
            (RuntimeError, lambda: ops.packed_attention(
                q, k, v, offs, out=q[:, :1].clone().expand(10, 4, 64))),
            (RuntimeError, lambda: ops.packed_attention(q.clone().requires_grad_(), k, v, offs)),
            (ValueError, lambda: ops.packed_attention(a, k, v, offs, out=a)),
            (ValueError, lambda: ops.packed_attention(a, k, v, offs, out=b)),
            (ValueError, lambda: ops.packed_attention(q, a, a, offs, out=b))):
        with pytest.raises(err):
            call()
    with forward_ad.dual_level():
        d = forward_ad.make_dual(q, torch.ones_like(q))
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            ops.packed_attention(d, k, v, offs)
    assert torch.equal(store, was)
    with pytest.raises(RuntimeError, match="status"):  # keys off a 16-byte boundary
        odd = torch.zeros(10 * 2 * 64 + 8, device=dev, dtype=BF)[1:1281].view(10, 2, 64)
        ops.packed_attention(q, odd, v, offs)
    # nothing to do
    assert ops.packed_attention(q[:0], k[:0], v[:0], offs).shape == (0, 4, 64)
    out = torch.full_like(q, 3.0)
    ops.packed_attention(q, k, v, offs[:1], out=out)  # no requests: rows of nobody
    assert (out == 3.0).all()


@pytest.mark.parametrize("n_split", [None, 17, 64])
def test_many_shares(dev, n_split):
    """A chunk over a long cache: more shares than some rows have tiles."""
    from cast_amd import ops
    B, Lq, Hq, Hk, D = 2, 70, 4, 2, 128
    lens = [4000, 75]
    cache = _cache(dev, I8, B, 130, 64, 64, Hk, D, 63, seed=9)
    held = Held(cache)
    q = torch.randn(B, Lq, Hq, D, generator=torch.Generator().manual_seed(4)).to(BF)
    out = ops.paged_attention(q.to(dev), cache, _i32(lens, dev), n_split=n_split)
    for b, n in enumerate(lens):
        _check(out[b], q[b], held, b, n, 0, 0, dev)


@pytest.mark.parametrize("beside", ["pages", "slots"])
def test_keys_and_values_in_one_allocation(dev, beside):
    """Keys and values of a page (or a slot) side by side: views of one tensor."""
    from cast_amd import ops
    B, H, D, page, block, n = 2, 2, 64, 32, 16, 75
    shape = (10, 2, page, H, D) if beside == "pages" else (10, page, 2, H, D)
    store = torch.zeros(shape, dtype=I8, device=dev)
    scales = torch.zeros(10, page // block, 2, H, device=dev)
    kc, vc = store.unbind(1 if beside == "pages" else 2)
    ks, vs = scales.unbind(2)
    table = torch.arange(10, device=dev, dtype=torch.int32).view(B, 5)
    cache = ops.QuantizedCache(kc, vc, ks, vs, table)
    held = Held(cache)
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(B, n, H, D, generator=g).to(BF).to(dev) for _ in range(2))
    ops.append_cache(k, v, cache)
    for b in range(B):
        held.append(b, k[b], v[b], 0)
    held.check(cache, [n] * B)
    got = ops.read_cache(cache, _i32([n] * B, dev), size=n)
    for rows in (1, 80):
        q = torch.randn(B, rows, 4, D, generator=g).to(BF)
        out = ops.paged_attention(q.to(dev), cache, _i32([n] * B, dev))
        for b in range(B):
            _check(out[b], q[b], held, b, n, 0, 0, dev)
            for kv in range(2):
                assert torch.equal(got[kv][b].cpu(), held.keys(kv, b, n).to(BF))


def test_packed_many_heads_over_many_keys(dev):
    """65535 heads over so many keys that rows times keys pass 2^38: every row is taken.  The
    values are 1, so the outputs are, to the roundings of the weights (2^-8 each, which their
    sum has too) and of the result."""
    from cast_amd import ops
    G, Tk, D = 65535, 4_195_000, 64
    k = torch.zeros(Tk, 1, D, dtype=BF, device=dev)
    q = torch.zeros(1, G, D, dtype=BF, device=dev)
    out = torch.full((1, G, D), 9.0, dtype=BF, device=dev)
    ops.packed_attention(q, k, torch.ones_like(k), _i32([0, 1], dev), k_offsets=_i32([0, Tk], dev),
                         out=out)
    assert ((out.float() - 1.0).abs() <= 2 * 2.0 ** -8).all()
