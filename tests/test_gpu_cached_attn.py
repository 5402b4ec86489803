"""``ops.paged_attention`` over a ``QuantizedCache`` against the 64-bit oracle: few rows in every
form, blocks of 128 rows, windows, first keys, shared key heads, padded batches, pages and
blocks of any size, what unseen codes and scales hold, strides, far pages, graphs.

Tolerances: the oracle's bound (see ``cache_oracle.attention``)."""
import math

import pytest
import torch

from oracle import cache_oracle as co
from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
I8, F8 = torch.int8, torch.float8_e4m3fn


def _codes(g, shape, code):
    x = torch.randn(shape, generator=g)
    if code == I8:
        return (x * 40).round().clamp(-127, 127).to(I8)
    return (x * 100).clamp(-448, 448).to(F8)


class Cache:
    """Shuffled pages of random codes; every request holds k_len keys."""

    def __init__(self, dev, seed, code, k_len, page, block, H, D, spread=0.3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.code, self.block, self.page, self.dev = code, block, page, dev
        need = [-(-n // page) for n in k_len]
        n = sum(need) + 2
        order = torch.randperm(n, generator=g).int()
        self.table = torch.full((len(k_len), width or max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        wide = 1 / 40 if code == I8 else 1 / 100
        self.c = [_codes(g, (n, page, H, D), code) for _ in range(2)]
        self.s = [wide * torch.exp(spread * torch.randn(n, page // block, H, generator=g))
                  for _ in range(2)]
        self.v_shift = 0.0

    def cache(self, heads_first=False):
        from cast_amd.ops import QuantizedCache
        c, s = [t.to(self.dev) for t in self.c], [t.to(self.dev) for t in self.s]
        if heads_first:
            c = [t.view(torch.uint8).transpose(1, 2).contiguous().view(self.code).transpose(1, 2)
                 for t in c]
            s = [t.permute(2, 0, 1).contiguous().permute(1, 2, 0) for t in s]
        return QuantizedCache(c[0], c[1], s[0], s[1], self.table.to(self.dev))

    def values(self, kv, b, n):
        """[n, H, D] fp64 and which of the keys are there."""
        j = torch.arange(n)
        page = self.table[b, j // self.page].long()
        there = (page >= 0) & (page < self.c[0].shape[0])
        page = page.clamp(0, self.c[0].shape[0] - 1)
        s = self.s[kv][page, j % self.page // self.block].double()
        s = torch.where((s > 0) & (s < 2.0 ** 126), s, torch.zeros_like(s))
        return self.c[kv].float()[page, j % self.page].double() * s[..., None], there


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _check(out, lse, q, c, q_len, k_len, window, sinks, block, causal, sm_scale, fill=None):
    out, lse = out.cpu(), None if lse is None else lse.cpu()
    dev = c.dev
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        if nq == 0:
            continue
        seen = so.visible(nq, nk, window, sinks, block, causal)
        k, there = c.values(0, b, nk)
        v, _ = c.values(1, b, nk)
        seen &= there[None]
        used = seen.any(0)[:, None, None]
        v = torch.where(used & ~torch.isnan(v), v, torch.zeros_like(v))
        top = 127.0 if c.code == I8 else 448.0
        s = c.s[1][torch.isfinite(c.s[1])]
        ref, rlse, tol, ltol = (t.cpu() for t in co.attention(
            q[b, :nq].to(dev), k.to(dev), v.to(dev), float(s.max()) * top, seen.to(dev), sm_scale,
            q.dtype))
        off = (out[b, :nq].double() - ref).abs()
        same = torch.isnan(out[b, :nq]) & torch.isnan(ref)
        worst = torch.where(same, torch.zeros_like(off), off - tol)
        assert not torch.isnan(worst).any(), b
        assert worst.max().item() <= 0.0, (b, worst.max().item(), off.max().item())
        if lse is not None:
            got = lse[b, :, :nq].double()
            none = torch.isinf(rlse)
            assert torch.equal(got[none], rlse[none]), b
            worst = ((got - rlse).abs() - ltol)[~none & ~torch.isnan(rlse)]
            assert worst.numel() == 0 or worst.max().item() <= 0.0, (b, worst.max().item())
    if fill is not None:
        for b, nq in enumerate(q_len):
            assert (out[b, nq:] == fill).all(), b


def _queries(seed, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


CASES = [  # B, Lq, Lk, Hq, Hk, D, page, mark, window, sinks, block
    (1, 1, 1, 1, 1, 128, 16, 16, 0, 0, 1), (1, 1, 33, 4, 4, 64, 16, 16, 0, 0, 1),
    (2, 7, 70, 3, 1, 128, 48, 16, 3, 1, 1), (1, 1, 5000, 24, 8, 128, 64, 64, 1024, 4, 1),
    (2, 1, 3000, 32, 8, 128, 32, 16, 0, 0, 1), (1, 5, 700, 40, 8, 64, 16, 16, 0, 0, 1),
    (1, 32, 600, 2, 2, 128, 128, 32, 0, 0, 1 << 30), (3, 4, 1000, 6, 2, 64, 256, 256, 130, 70, 1),
    (1, 128, 128, 2, 2, 128, 32, 32, 0, 0, 1), (1, 129, 300, 2, 1, 64, 16, 16, 64, 4, 1),
    (1, 500, 500, 4, 2, 128, 48, 48, 100, 33, 1), (2, 95, 1000, 6, 2, 128, 64, 16, 0, 0, 1),
    (1, 331, 331, 1, 1, 64, 128, 128, 1, 0, 1), (1, 400, 400, 2, 2, 128, 16, 16, 32, 32, 32),
    (1, 440, 880, 2, 1, 128, 64, 32, 220, 110, 110), (3, 40, 20, 2, 2, 128, 16, 16, 0, 0, 1),
    (1, 64, 4096, 8, 1, 128, 256, 128, 1024, 5, 1), (1, 200, 200, 5, 5, 64, 32, 32, 1000, 7, 1),
    (1, 70, 300, 2, 2, 128, 96, 32, 0, 300, 1)]


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hk,D,page,mark,window,sinks,block", CASES)
def test_shapes(dev, dtype, code, B, Lq, Lk, Hq, Hk, D, page, mark, window, sinks, block):
    from cast_amd import ops
    print("cached", dtype, code, B, Lq, Lk, Hq, Hk, D, page, mark, window, flush=True)
    c = Cache(dev, Lq * 7 + Lk, code, [Lk] * B, page, mark, Hk, D)
    q = _queries(Lk, (B, Lq, Hq, D), dtype)
    out, lse = ops.paged_attention(q.to(dev), c.cache(), _i32([Lk] * B, dev), window=window or None,
                                   sinks=sinks, block=block, return_lse=True)
    _check(out, lse, q, c, [Lq] * B, [Lk] * B, window, sinks, block, True, D ** -0.5)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("n_split", [-1, 0, 1, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_forms(dev, D, n_split, code):
    """Every form of a launch of few rows, over the torch op: a workgroup a key head, units,
    blocks whole and in shares; ragged, windows and first keys."""
    from cast_amd import _lib
    ops_ = _lib.torch_ops()
    B, T, Hq, Hk, page = 5, 4, 16, 2, 48
    k_len, q_len = [800, 333, 4, 0, 70], [4, 2, 4, 3, 0]
    c = Cache(dev, D + n_split, code, k_len, page, 16, Hk, D)
    q = _queries(D, (B, T, Hq, D), BF)
    cache = c.cache()
    for window, sinks in ((0, 0), (65, 40)):
        print("forms", D, n_split, code, window, flush=True)
        out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
        res = ops_.window_attention(
            q.to(dev), cache.k, cache.v, cache.table, _i32(q_len, dev), _i32(k_len, dev), window,
            sinks, 1, D ** -0.5, True, out, n_split, -1, cache.k_scale, cache.v_scale)
        _check(*res, q, c, q_len, k_len, window, sinks, 1, True, D ** -0.5, fill=9.0)


@pytest.mark.parametrize("Lq", [1, 9, 150])
@pytest.mark.parametrize("n_split", [None, 1, 5])
def test_padded_batch(dev, Lq, n_split):
    from cast_amd import ops
    B, Lk, Hq, Hk, D = 5, 310, 6, 2, 128
    q_len, k_len = [Lq, max(Lq // 2, 1), 0, Lq, Lq], [Lk, 77, 50, 0, 3]
    c = Cache(dev, Lq, I8, k_len, 32, 32, Hk, D)
    q = _queries(Lq, (B, Lq, Hq, D), BF)
    for window, sinks in ((0, 0), (40, 8)):
        print("padded", Lq, n_split, window, flush=True)
        out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
        got, lse = ops.paged_attention(q.to(dev), c.cache(), _i32(k_len, dev),
                                       q_lengths=_i32(q_len, dev), window=window or None,
                                       sinks=sinks, out=out, return_lse=True, n_split=n_split)
        assert got.data_ptr() == out.data_ptr()
        _check(out, lse, q, c, q_len, k_len, window, sinks, 1, True, D ** -0.5, fill=9.0)


@pytest.mark.parametrize("B", [70, 600])
def test_many_requests(dev, B):
    from cast_amd import ops
    k_len = [(37 * b) % 98 for b in range(B)]
    q_len = [int(b % 11 != 3) for b in range(B)]
    c = Cache(dev, B, F8, k_len, 16, 16, 2, 64)
    q = _queries(B, (B, 1, 4, 64), BF)
    out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
    got, lse = ops.paged_attention(q.to(dev), c.cache(), _i32(k_len, dev), out=out,
                                   q_lengths=_i32(q_len, dev), return_lse=True)
    _check(out, lse, q, c, q_len, k_len, 0, 0, 1, True, 1 / 8, fill=9.0)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("Lq", [1, 3, 140])
def test_unseen_codes_and_scales(dev, code, Lq):
    """Scales that are no numbers, codes that hold none, hidden pages: rows that do not see them
    are as without them."""
    from cast_amd import ops
    Hq, Hk, D, page, Lk, window = 4, 2, 128, 32, 500, 150
    c = Cache(dev, Lq, code, [Lk, Lk], page, 16, Hk, D)
    q = _queries(3, (2, Lq, Hq, D), BF)
    first = Lk - Lq - window + 1  # the first key that a row sees
    bad = c.c[0].view(torch.uint8), c.c[1].view(torch.uint8)
    for b in range(2):
        for j in list(range(0, first)) + list(range(Lk, -(-Lk // page) * page)):
            pg, row = int(c.table[b, j // page]), j % page
            if code == F8:
                bad[0][pg, row] = 0x7f
                bad[1][pg, row] = 0xff
            blk = j // 16 * 16
            if blk + 16 <= first or blk >= Lk:
                c.s[0][pg, row // 16], c.s[1][pg, row // 16] = float("nan"), float("inf")
    c.table[1, (first + 70) // page] = -1       # hidden keys inside the window
    c.table[1, 2] = 10 ** 9                     # far outside it
    for n_split in (None, 1, 4):
        print("unseen", code, Lq, n_split, flush=True)
        out, lse = ops.paged_attention(q.to(dev), c.cache(), _i32([Lk, Lk], dev), window=window,
                                       return_lse=True, n_split=n_split)
        _check(out, lse, q, c, [Lq] * 2, [Lk] * 2, window, 0, 1, True, D ** -0.5)


@pytest.mark.parametrize("Lq", [2, 40])
def test_codes_without_a_number(dev, Lq):
    """An e4m3 value code that holds no number counts as 0, a key's makes the rows that see it
    NaN and no others."""
    from cast_amd import ops
    Hk, D, Lk = 2, 64, 90
    c = Cache(dev, 1, F8, [Lk], 16, 16, Hk, D)
    at = lambda j: (int(c.table[0, j // 16]), j % 16)  # noqa: E731
    c.c[1].view(torch.uint8)[(*at(30), 1, 5)] = 0x7f
    c.c[0].view(torch.uint8)[(*at(Lk - 1), 0, 7)] = 0xff
    q = _queries(2, (1, Lq, 4, D), HF)
    out, lse = ops.paged_attention(q.to(dev), c.cache(), _i32([Lk], dev), return_lse=True)
    assert torch.isnan(out[0, -1, :2]).all() and not torch.isnan(out[0, -1, 2:]).any()
    _check(out[:, :, 2:], lse[:, 2:], q[:, :, 2:], _head(c, 1), [Lq], [Lk], 0, 0, 1, True, 1 / 8)
    _check(out[:, :-1], lse[:, :, :-1], q[:, :-1], c, [Lq - 1], [Lk - 1], 0, 0, 1, True, 1 / 8)


def _head(c, h):
    import copy
    d = copy.copy(c)
    d.c, d.s = [t[:, :, h:h + 1] for t in c.c], [t[:, :, h:h + 1] for t in c.s]
    return d


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("Lq", [1, 130])
def test_scales_far_apart(dev, code, Lq):
    """Blocks whose scales differ by up to 2^20, zero scales, queries of any size."""
    from cast_amd import ops
    Hk, D, Lk = 2, 128, 700
    c = Cache(dev, 4, code, [Lk], 32, 32, Hk, D, spread=3.0)
    c.s[1][::5] = 0.0
    c.s[0][::7] = 2.0 ** -100
    c.s[0] = c.s[0].clamp(max=0.1)
    q = _queries(5, (1, Lq, 4, D), BF)
    q[:, :, 1] *= 2.0 ** -100
    q[:, :, 2] = 0.0
    q[:, 0, 3, 7] = 60.0
    for n_split in (None, 1, 3):
        out, lse = ops.paged_attention(q.to(dev), c.cache(), _i32([Lk], dev), return_lse=True,
                                       n_split=n_split)
        _check(out, lse, q, c, [Lq], [Lk], 0, 0, 1, True, D ** -0.5)
    # the largest queries, the smallest scale of the logits
    big = _queries(6, (1, Lq, 4, D), BF, 2.0 ** 120)
    out, lse = ops.paged_attention(big.to(dev), c.cache(), _i32([Lk], dev), return_lse=True,
                                   sm_scale=2.0 ** -122)
    _check(out, lse, big, c, [Lq], [Lk], 0, 0, 1, True, 2.0 ** -122)


@pytest.mark.parametrize("Lq", [1, 150])
def test_all_keys_scale_and_peaks(dev, Lq):
    """Rows without order, a given scale, logits that move the running maximum often."""
    from cast_amd import ops
    c = Cache(dev, 8, I8, [333, 333], 16, 16, 2, 128)
    q = _queries(3, (2, Lq, 4, 128), BF, 3.0)
    out, lse = ops.paged_attention(q.to(dev), c.cache(), _i32([333] * 2, dev), causal=False,
                                   sm_scale=0.3, return_lse=True)
    _check(out, lse, q, c, [Lq] * 2, [333] * 2, 0, 0, 1, False, 0.3)


@pytest.mark.parametrize("Lq", [1, 140])
def test_strides(dev, Lq):
    """Pages and scales with the heads first, a transposed output."""
    from cast_amd import ops
    c = Cache(dev, 8, F8, [200, 90], 32, 16, 3, 64)
    q = _queries(3, (2, 6, Lq, 64), BF).transpose(1, 2)
    out = torch.zeros(2, 6, Lq, 64, dtype=BF, device=dev).transpose(1, 2)
    ops.paged_attention(q.to(dev), c.cache(True), _i32([200, 90], dev), out=out)
    _check(out, None, q, c, [Lq] * 2, [200, 90], 0, 0, 1, True, 1 / 8)


@pytest.mark.parametrize("Lq", [1, 40])
def test_far_pages(dev, Lq):
    """Pages past 4 GiB from the first, of codes and of their table's row."""
    from cast_amd.ops import QuantizedCache
    from cast_amd import ops
    H, D, page, Lk = 8, 128, 128, 300
    c = Cache(dev, 8, I8, [Lk], page, 32, H, D)
    n = (1 << 32) // (page * H * D) + 50
    far = torch.tensor([n - 3, 5, n - 1], dtype=torch.int32)
    cache = QuantizedCache(*(torch.empty(n, page, H, D, dtype=I8, device=dev) for _ in range(2)),
                           *(torch.empty(n, page // 32, H, device=dev) for _ in range(2)),
                           far[None].to(dev))
    for i in range(3):
        src = int(c.table[0, i])
        for kv in range(2):
            cache[kv][int(far[i])] = c.c[kv][src].to(dev)
            cache[2 + kv][int(far[i])] = c.s[kv][src].to(dev)
    q = _queries(3, (1, Lq, 16, D), BF)
    out, lse = ops.paged_attention(q.to(dev), cache, _i32([Lk], dev), return_lse=True)
    _check(out, lse, q, c, [Lq], [Lk], 0, 0, 1, True, D ** -0.5)
    x = torch.randn(1, 40, H, D, generator=torch.Generator().manual_seed(1)).to(BF).to(dev)
    ops.append_cache(x, x, cache, _i32([270], dev))
    k, v = ops.read_cache(cache, _i32([310], dev), starts=_i32([270], dev), size=40)
    step = cache.k_scale[far[2].item(), :2].max().item()
    assert (k.float() - x.float()).abs().max().item() <= step / 2 + x.float().abs().max() * 2.0 ** -8


def test_graph(dev):
    """A captured call follows the lengths, the table, the codes and their scales."""
    from cast_amd import ops
    B, Hk, D = 3, 2, 128
    c = Cache(dev, 8, I8, [400, 300, 200], 32, 32, Hk, D)
    cache = c.cache()
    q = _queries(1, (B, 1, 8, D), BF).to(dev)
    lens = _i32([400, 300, 200], dev)
    out = torch.zeros(B, 1, 8, D, dtype=BF, device=dev)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.paged_attention(q, cache, lens, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, cache, lens, out=out)
    for step, n in enumerate(([400, 1, 200], [3, 300, 0], [77, 299, 33])):
        c.s[1] = c.s[1] * (1.5 + step)
        cache.v_scale.copy_(c.s[1])
        lens.copy_(_i32(n, dev))
        q.copy_(_queries(9 + step, q.shape, BF))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, None, q.cpu(), c, [1] * B, n, 0, 0, 1, True, D ** -0.5)
