"""``ops.window_attention`` and ``ops.paged_attention`` against the 64-bit oracle: windows,
first keys, blocks of positions, shared key heads, padded batches, empty rows, pages, what
unseen keys hold, strides, shares, streams and graphs.

Tolerances: the oracle's bound (see ``streaming_oracle.attention``)."""
import math

import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _inputs(seed, B, Lq, Lk, Hq, Hk, D, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(B, Lq, Hq, D, generator=g) * scale).to(dtype)
    k = (torch.randn(B, Lk, Hk, D, generator=g)).to(dtype)
    v = (torch.randn(B, Lk, Hk, D, generator=g) + 0.5).to(dtype)
    return q, k, v


def _check(out, lse, q, k, v, q_len, k_len, window, sinks, block, causal, sm_scale, hidden=None,
           fill=None):
    """Every request's live rows against the oracle, its other rows against ``fill``."""
    out, lse = out.cpu(), None if lse is None else lse.cpu()
    dev = "cuda:0"  # (the oracle's fp64 products)
    for b, (nq, nk) in enumerate(zip(q_len, k_len)):
        if nq == 0:
            continue
        seen = so.visible(nq, nk, window, sinks, block, causal)
        if hidden is not None:
            seen &= ~hidden[b][None, :nk]
        ref, rlse, tol, ltol = (t.cpu() for t in so.attention(
            q[b, :nq].to(dev), k[b, :nk].to(dev), v[b, :nk].to(dev), seen.to(dev), sm_scale,
            q.dtype))
        off = (out[b, :nq].double() - ref).abs()
        same = (out[b, :nq].double() == ref) | (torch.isnan(out[b, :nq]) & torch.isnan(ref))
        worst = torch.where(same, torch.zeros_like(off), off - tol).max().item()
        assert worst <= 0.0, (b, worst, off.max().item())
        if lse is not None:
            got = lse[b, :, :nq].double()
            none = torch.isinf(rlse)
            assert torch.equal(got[none], rlse[none]), b
            worst = ((got - rlse).abs() - ltol)[~none]
            assert worst.numel() == 0 or worst.max().item() <= 0.0, (b, worst.max().item())
    if fill is not None:
        for b, nq in enumerate(q_len):
            assert (out[b, nq:] == fill).all(), b


CASES = [  # B, Lq, Lk, Hq, Hk, D, window, sinks, block
    (1, 1, 1, 1, 1, 128, 0, 0, 1), (1, 1, 33, 4, 4, 64, 0, 0, 1), (2, 7, 7, 3, 1, 128, 3, 1, 1),
    (1, 128, 128, 2, 2, 128, 0, 0, 1), (1, 129, 300, 2, 1, 64, 64, 4, 1),
    (1, 500, 500, 4, 2, 128, 100, 33, 1), (2, 95, 1000, 6, 2, 128, 0, 0, 1),
    (1, 331, 331, 1, 1, 64, 1, 0, 1), (1, 400, 400, 2, 2, 128, 32, 32, 32),
    (1, 440, 880, 2, 1, 128, 220, 110, 110), (1, 130, 777, 2, 2, 64, 130, 0, 130),
    (3, 40, 20, 2, 2, 128, 0, 0, 1), (1, 64, 4096, 8, 1, 128, 1024, 5, 1),
    (1, 1, 5000, 24, 8, 128, 1024, 4, 1), (2, 1, 3000, 32, 8, 128, 0, 0, 1),
    (1, 5, 700, 40, 8, 64, 0, 0, 1), (1, 200, 200, 5, 5, 64, 1000, 7, 1),
    (1, 33, 600, 2, 2, 128, 0, 0, 1 << 30), (1, 70, 300, 2, 2, 128, 0, 300, 1)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hk,D,window,sinks,block", CASES)
def test_window_shapes(dev, dtype, B, Lq, Lk, Hq, Hk, D, window, sinks, block):
    from cast_amd import ops
    print("window", dtype, B, Lq, Lk, Hq, Hk, D, window, sinks, block, flush=True)
    q, k, v = _inputs(Lq * 7 + Lk, B, Lq, Lk, Hq, Hk, D, dtype)
    out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), window=window or None,
                                    sinks=sinks, block=block, return_lse=True)
    _check(out, lse, q, k, v, [Lq] * B, [Lk] * B, window, sinks, block, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("n_split", [-1, 0, 1, 3])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_forms(dev, D, n_split):
    """Every form of a launch of few rows, over the torch op: a workgroup a key head, units,
    blocks; padded, paged, with first keys, NaN in unseen values of rows that see less."""
    from cast_amd import _lib, ops
    ops_ = _lib.torch_ops()
    B, T, Hq, Hk, Lk, page = 5, 4, 16, 2, 800, 48
    q, k, v = _inputs(D + n_split, B, T, Lk, Hq, Hk, D, BF)
    k_len, q_len = [800, 333, 4, 0, 70], [4, 2, 4, 3, 0]
    v[0, 798, 1, 5] = float("nan")  # queries 2 and 3 of request 0 see it
    v[4, 69] = float("inf")
    kp, vp, table = (t.to(dev) for t in _pages(D, k, v, k_len, page))
    ql, kl = (torch.tensor(n, dtype=torch.int32, device=dev) for n in (q_len, k_len))
    for window, sinks in ((0, 0), (65, 40)):
        for paged in (False, True):
            print("few rows", D, n_split, window, paged, flush=True)
            out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
            res = ops_.window_attention(
                q.to(dev), kp if paged else k.to(dev), vp if paged else v.to(dev),
                table if paged else None, ql, kl, window, sinks, 1, D ** -0.5, True, out, n_split,
                -1)
            _check(*res, q, k, v, q_len, k_len, window, sinks, 1, True, D ** -0.5, fill=9.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n_split", [2, 3, 7, 64])
def test_window_shares(dev, dtype, n_split):
    """Any number of shares, some of them empty."""
    from cast_amd import ops
    for B, Lq, Lk, Hq, Hk, D, window, sinks, block in (
            (1, 130, 700, 4, 2, 128, 300, 40, 1), (2, 3, 90, 2, 1, 64, 0, 0, 1),
            (1, 1, 4000, 8, 2, 128, 0, 0, 1), (1, 50, 20, 2, 2, 128, 0, 0, 1)):
        print("shares", n_split, Lq, Lk, flush=True)
        q, k, v = _inputs(n_split, B, Lq, Lk, Hq, Hk, D, dtype)
        out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), window=window or None,
                                        sinks=sinks, block=block, return_lse=True,
                                        n_split=n_split)
        _check(out, lse, q, k, v, [Lq] * B, [Lk] * B, window, sinks, block, True,
               1 / math.sqrt(D))


@pytest.mark.parametrize("D", [64, 128])
def test_all_keys_and_scale(dev, D):
    """Rows without order, a given scale, logits that move the running maximum often."""
    from cast_amd import ops
    q, k, v = _inputs(3, 2, 150, 333, 4, 2, D, BF, scale=3.0)
    out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), causal=False, sm_scale=0.3,
                                    return_lse=True)
    _check(out, lse, q, k, v, [150] * 2, [333] * 2, 0, 0, 1, False, 0.3)


@pytest.mark.parametrize("n_split", [None, 1, 5])
@pytest.mark.parametrize("Lq", [1, 9, 300])
def test_padded_batch(dev, Lq, n_split):
    """Own lengths of every request, from none to all: rows behind the last query stay as
    they were, storage past the keys holds NaN."""
    from cast_amd import ops
    B, Lk, Hq, Hk, D = 5, 310, 6, 2, 128
    q, k, v = _inputs(Lq, B, Lq, Lk, Hq, Hk, D, BF)
    q_len = [Lq, max(Lq // 2, 1), 0, Lq, Lq]
    k_len = [Lk, 77, 50, 0, 3]
    for b, n in enumerate(k_len):
        k[b, n:] = float("nan")
        v[b, n:] = float("nan")
    out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
    ql = torch.tensor(q_len, dtype=torch.int32, device=dev)
    kl = torch.tensor(k_len, dtype=torch.int32, device=dev)
    for window, sinks in ((0, 0), (40, 8)):
        print("padded", Lq, n_split, window, flush=True)
        out.fill_(9.0)
        got, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), window=window or None,
                                        sinks=sinks, q_lengths=ql, k_lengths=kl, out=out,
                                        return_lse=True, n_split=n_split)
        assert got.data_ptr() == out.data_ptr()
        _check(out, lse, q, k, v, q_len, k_len, window, sinks, 1, True, 1 / math.sqrt(D), fill=9.0)


def test_lengths_past_the_storage_and_negative(dev):
    """Lengths are clamped to the storage."""
    from cast_amd import ops
    q, k, v = _inputs(1, 3, 4, 50, 2, 2, 64, BF)
    out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
    ops.window_attention(q.to(dev), k.to(dev), v.to(dev), out=out,
                         q_lengths=torch.tensor([4, 99, -3], dtype=torch.int32, device=dev),
                         k_lengths=torch.tensor([1000, 20, 50], dtype=torch.int32, device=dev))
    _check(out, None, q, k, v, [4, 4, 0], [50, 20, 50], 0, 0, 1, True, 1 / 8, fill=9.0)


def test_many_requests(dev):
    """More requests than a wavefront has lanes, and more than it plans for: every length,
    none too, one new token."""
    from cast_amd import ops
    for B in (70, 600):
        q, k, v = _inputs(B, B, 1, 97, 4, 2, 64, BF)
        k_len = [(37 * b) % 98 for b in range(B)]
        q_len = [int(b % 11 != 3) for b in range(B)]
        out = torch.full(q.shape, 9.0, dtype=BF, device=dev)
        got, lse = ops.window_attention(
            q.to(dev), k.to(dev), v.to(dev), out=out, return_lse=True,
            q_lengths=torch.tensor(q_len, dtype=torch.int32, device=dev),
            k_lengths=torch.tensor(k_len, dtype=torch.int32, device=dev))
        _check(out, lse, q, k, v, q_len, k_len, 0, 0, 1, True, 1 / 8, fill=9.0)


def test_no_keys(dev):
    from cast_amd import ops
    q, k, v = (t.to(dev) for t in _inputs(1, 2, 5, 0, 2, 2, 64, BF))
    out, lse = ops.window_attention(q, k, v, return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all() and (lse < 0).all()
    assert ops.window_attention(q[:, :0], q, q).shape == (2, 0, 2, 64)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("n_split", [1, 3])
def test_unseen_keys_do_not_reach_a_row(dev, dtype, n_split):
    """NaN and infinities in keys and values: rows that see them carry them, the others
    are those of finite storage."""
    from cast_amd import ops
    B, L, Hq, Hk, D, window, sinks = 1, 300, 4, 2, 128, 60, 5
    q, k, v = _inputs(11, B, L, L, Hq, Hk, D, dtype)
    v[0, 130, 0, 7] = float("nan")
    v[0, 131, 1, 3] = float("inf")
    v[0, 200, 1, 90] = float("-inf")
    k[0, 250, 0] = float("nan")
    out, lse = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), window=window, sinks=sinks,
                                    return_lse=True, n_split=n_split)
    # rows that see the NaN key are NaN throughout; the oracle takes the others
    seen = so.visible(L, L, window, sinks, 1)
    hit = seen[:, 250]
    assert torch.isnan(out[0, hit][:, :2].float()).all()
    out, lse = out.cpu(), lse.cpu()
    ref, rlse, tol, ltol = so.attention(q[0, ~hit], k[0].nan_to_num(0.0), v[0], seen[~hit],
                                        1 / math.sqrt(D), dtype)
    got = out[0, ~hit].double()
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    assert ((got - ref).abs()[~same] <= tol[~same]).all()
    assert torch.isnan(got[130 - 0, :2, 7]).all() and torch.isinf(got[131, 2:, 3]).all()
    assert ((lse[0, :, ~hit].double() - rlse).abs() <= ltol).all()


def test_strides(dev):
    """Head-major storage, a fused projection, an output of other strides, shared keys."""
    from cast_amd import ops
    q, k, v = _inputs(6, 2, 70, 90, 4, 4, 64, BF)
    w = dict(window=50, sinks=3)
    want = ops.window_attention(q.to(dev), k.to(dev), v.to(dev), **w)
    hm = [t.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for t in (q, k, v)]
    out = torch.empty(2, 4, 70, 64, dtype=BF, device=dev).transpose(1, 2)
    assert torch.equal(ops.window_attention(*hm, out=out, **w), want)
    fused = torch.stack([k, v], 2).to(dev)
    assert torch.equal(ops.window_attention(hm[0], fused[:, :, 0], fused[:, :, 1], **w), want)
    one_k, one_v = (t[:1, :, :1].to(dev).expand(2, 90, 4, 64) for t in (k, v))
    got = ops.window_attention(q.to(dev), one_k, one_v, **w)
    _check(got, None, q, k[:1, :, :1].expand(2, 90, 4, 64), v[:1, :, :1].expand(2, 90, 4, 64),
           [70] * 2, [90] * 2, 50, 3, 1, True, 1 / 8)


def _pages(seed, k, v, k_len, page, spare=3):
    """Shuffled pages of dense k, v; unused rows hold NaN, unused entries nonsense."""
    B, Lk, Hk, D = k.shape
    M = max(1, -(-Lk // page))
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(B * M + spare, generator=g)
    table = torch.full((B, M), -7, dtype=torch.int32)
    kp = torch.full((B * M + spare, page, Hk, D), float("nan"), dtype=k.dtype)
    vp = kp.clone()
    for b in range(B):
        for i in range(-(-k_len[b] // page)):
            p = int(order[b * M + i])
            table[b, i] = p
            n = min(page, k_len[b] - i * page)
            kp[p, :n], vp[p, :n] = k[b, i * page:i * page + n], v[b, i * page:i * page + n]
    return kp, vp, table


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [16, 48, 128, 256])
@pytest.mark.parametrize("T,Hq,Hk,D,window,sinks,block,n_split", [
    (1, 8, 2, 128, 0, 0, 1, None), (1, 24, 24, 64, 100, 4, 1, None), (3, 8, 1, 128, 333, 20, 1, 4),
    (200, 4, 2, 128, 300, 30, 1, 1), (130, 2, 2, 64, 260, 130, 130, 2), (17, 6, 3, 128, 0, 0, 1, 1),
    (1, 64, 1, 128, 0, 0, 1, 5), (1, 1, 1, 64, 64, 0, 1, 1)])
def test_paged(dev, dtype, page, T, Hq, Hk, D, window, sinks, block, n_split):
    from cast_amd import ops
    print("paged", dtype, page, T, Hq, Hk, D, window, sinks, block, n_split, flush=True)
    B, Lk = 4, 1300
    q, k, v = _inputs(T + page, B, T, Lk, Hq, Hk, D, dtype)
    k_len = [Lk, 517, T, 0]
    kp, vp, table = _pages(page, k, v, k_len, page)
    cache = ops.PagedCache(kp.to(dev), vp.to(dev), table.to(dev))
    out, lse = ops.paged_attention(q.to(dev), cache,
                                   torch.tensor(k_len, dtype=torch.int32, device=dev),
                                   window=window or None, sinks=sinks, block=block,
                                   return_lse=True, n_split=n_split)
    _check(out, lse, q, k, v, [T] * B, k_len, window, sinks, block, True, 1 / math.sqrt(D))


@pytest.mark.parametrize("T", [1, 40])
def test_pages_that_are_not_there(dev, T):
    """Entries outside the pages hide their keys, whether negative or too large; entries
    between the first keys and the window are not read."""
    from cast_amd import ops
    B, Lk, Hq, Hk, D, page = 2, 500, 4, 2, 128, 32
    q, k, v = _inputs(T, B, T, Lk, Hq, Hk, D, BF)
    kp, vp, table = _pages(4, k, v, [Lk, Lk], page)
    hidden = torch.zeros(B, Lk, dtype=torch.bool)
    for b, i, bad in ((0, 3, -1), (0, 15, 1 << 20), (1, 0, 2 ** 31 - 1), (1, 14, -2 ** 31)):
        table[b, i] = bad
        hidden[b, i * page:(i + 1) * page] = True
    cache = ops.PagedCache(kp.to(dev), vp.to(dev), table.to(dev))
    lens = torch.tensor([Lk, Lk], dtype=torch.int32, device=dev)
    for window, sinks in ((0, 0), (100, 20)):
        out, lse = ops.paged_attention(q.to(dev), cache, lens, window=window or None, sinks=sinks,
                                       return_lse=True)
        _check(out, lse, q, k, v, [T] * B, [Lk] * B, window, sinks, 1, True, 1 / math.sqrt(D),
               hidden=hidden)
    table[:, :] = -1
    cache.table.copy_(table)
    out, lse = ops.paged_attention(q.to(dev), cache, lens, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_paged_max_length_is_only_a_plan(dev):
    from cast_amd import ops
    q, k, v = _inputs(2, 2, 1, 900, 4, 4, 64, BF)
    kp, vp, table = _pages(1, k, v, [900, 31], 64)
    cache = ops.PagedCache(kp.to(dev), vp.to(dev), table.to(dev))
    lens = torch.tensor([900, 31], dtype=torch.int32, device=dev)
    for most in (None, 900, 10, 0):
        out = ops.paged_attention(q.to(dev), cache, lens, max_length=most)
        _check(out, None, q, k, v, [1, 1], [900, 31], 0, 0, 1, True, 1 / 8)


def test_streams_and_graphs(dev):
    """Two calls at once on two streams; a captured pair of calls with shares (each with a
    workspace of its own), replayed over new inputs and lengths beside eager calls, bit for
    bit the eager result."""
    from cast_amd import ops
    q, k, v = (t.to(dev) for t in _inputs(5, 2, 3, 2000, 8, 2, 128, BF))
    kp, vp, table = (t.to(dev) for t in _pages(1, k.cpu(), v.cpu(), [2000, 2000], 64))
    cache = ops.PagedCache(kp.nan_to_num(0.0), vp.nan_to_num(0.0), table)
    lens = torch.tensor([1999, 700], dtype=torch.int32, device=dev)

    def both():
        return [*ops.paged_attention(q, cache, lens, n_split=6, return_lse=True),
                *ops.window_attention(q, k, v, window=300, sinks=4, n_split=4, return_lse=True)]

    want = both()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(both())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for res in got:
        assert all(torch.equal(a, b) for a, b in zip(res, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = both()
    for i in range(4):
        q.copy_(torch.randn(q.shape, device=dev))
        lens -= 100
        want = both()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), i


def test_refusals(dev):
    from cast_amd import ops
    q, k, v = (t.to(dev) for t in _inputs(5, 2, 4, 20, 4, 2, 64, BF))
    for kw, err in ((dict(window=0), ValueError), (dict(window=-5), ValueError),
                    (dict(sinks=-1), ValueError), (dict(block=0), ValueError),
                    (dict(causal=False, window=5), ValueError),
                    (dict(causal=False, sinks=5), ValueError), (dict(sm_scale=0.0), ValueError),
                    (dict(sm_scale=-0.1), ValueError), (dict(n_split=0), ValueError),
                    (dict(n_split=65), RuntimeError),
                    (dict(k_lengths=torch.tensor([1, 2], device=dev)), RuntimeError),
                    (dict(k_lengths=torch.tensor([1], device=dev).int()), RuntimeError),
                    (dict(q_lengths=torch.tensor([1, 2]).int()), RuntimeError),
                    (dict(out=torch.empty(2, 4, 4, 64, device=dev)), RuntimeError),
                    (dict(out=torch.empty(2, 4, 1, 64, device=dev, dtype=BF).expand(2, 4, 4, 64)),
                     RuntimeError)):
        with pytest.raises(err):
            ops.window_attention(q, k, v, **kw)
    with pytest.raises(TypeError):
        ops.window_attention(q.float(), k.float(), v.float())
    with pytest.raises(TypeError):
        ops.window_attention(q, k, v.half())
    with pytest.raises(ValueError):
        ops.window_attention(q[:, :, :3], k, v)
    with pytest.raises(ValueError):
        ops.window_attention(q, k, v[:, :10])
    with pytest.raises(RuntimeError):
        ops.window_attention(q[..., :32], k[..., :32], v[..., :32])
    with pytest.raises(RuntimeError, match="gradient"):
        ops.window_attention(q.clone().requires_grad_(), k, v)
    with pytest.raises(RuntimeError, match="status"):  # keys off a 16-byte boundary
        off = torch.zeros(2 * 20 * 2 * 64 + 8, device=dev, dtype=BF)[1:1 + 2 * 20 * 2 * 64]
        ops.window_attention(q, off.view(2, 20, 2, 64), v)
    pages = torch.zeros(8, 24, 2, 64, device=dev, dtype=BF)
    table = torch.zeros(2, 2, device=dev, dtype=torch.int32)
    lens = torch.ones(2, device=dev, dtype=torch.int32)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.paged_attention(q, ops.PagedCache(pages, pages, table), lens)
    pages = pages[:, :16]
    with pytest.raises(RuntimeError, match="table"):
        ops.paged_attention(q, ops.PagedCache(pages, pages, table[:1]), lens)
    with pytest.raises(RuntimeError, match="lengths"):
        ops.paged_attention(q, ops.PagedCache(pages, pages, table), lens[:1])
