"""``ops.packed_attention`` against the 64-bit oracle: prompts of any lengths behind each other,
keys held before them, windows, first keys, shared key heads, shares, rows of nobody, what
unseen keys hold, strides, graphs.

Tolerances: the oracle's bound (see ``streaming_oracle.attention``)."""
import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _offsets(count, first=0):
    out = [first]
    for n in count:
        out.append(out[-1] + n)
    return out


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _inputs(seed, T, Tk, Hq, Hk, D, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(T, Hq, D, generator=g) * scale).to(dtype),
            torch.randn(Tk, Hk, D, generator=g).to(dtype),
            (torch.randn(Tk, Hk, D, generator=g) + 0.5).to(dtype))


def _check(out, lse, q, k, v, q_at, k_at, window, sinks, block, causal, sm_scale, fill=None):
    out, lse = out.cpu(), None if lse is None else lse.cpu()
    dev = "cuda:0"  # (the oracle's fp64 products)
    mine = torch.zeros(out.shape[0], dtype=torch.bool)
    for b, (q0, q1, k0, k1) in enumerate(zip(q_at, q_at[1:], k_at, k_at[1:])):
        mine[q0:q1] = True
        if q0 == q1:
            continue
        seen = so.visible(q1 - q0, k1 - k0, window, sinks, block, causal)
        ref, rlse, tol, ltol = (t.cpu() for t in so.attention(
            q[q0:q1].to(dev), k[k0:k1].to(dev), v[k0:k1].to(dev), seen.to(dev), sm_scale, q.dtype))
        got = out[q0:q1].double()
        same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
        worst = torch.where(same, torch.zeros_like(ref), (got - ref).abs() - tol)
        assert worst.max().item() <= 0.0, (b, worst.max().item())
        if lse is not None:
            got = lse[:, q0:q1].double()
            none = torch.isinf(rlse)
            assert torch.equal(got[none], rlse[none]), b
            worst = ((got - rlse).abs() - ltol)[~none]
            assert worst.numel() == 0 or worst.max().item() <= 0.0, (b, worst.max().item())
    if fill is not None:
        assert (out[~mine] == fill).all()


CASES = [  # lengths, keys before them, Hq, Hk, D, window, sinks, block
    ([1], [0], 1, 1, 128, 0, 0, 1), ([5, 1, 130], [0, 0, 0], 4, 2, 64, 0, 0, 1),
    ([128, 128, 1, 127], [0, 3, 700, 1], 8, 2, 128, 0, 0, 1), ([300, 0, 17, 64], [0] * 4, 3, 1, 64, 0, 0, 1),
    ([500, 33, 260], [10, 600, 0], 4, 4, 128, 100, 33, 1), ([129], [1000], 16, 2, 64, 64, 4, 1),
    ([220, 110, 330], [0, 0, 0], 2, 2, 128, 220, 110, 110), ([40, 9], [-20, -9], 2, 2, 128, 0, 0, 1),
    ([64, 65], [300, 0], 2, 1, 64, 0, 0, 130), ([700, 1, 1, 1, 350], [0] * 5, 12, 2, 128, 0, 0, 1)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("count,before,Hq,Hk,D,window,sinks,block", CASES)
def test_shapes(dev, dtype, count, before, Hq, Hk, D, window, sinks, block):
    """Rows ahead of the first request and behind the last are nobody's."""
    from cast_amd import ops
    q_at = _offsets(count, 2)
    k_at = _offsets([n + m for n, m in zip(count, before)], 1)
    q, k, v = _inputs(q_at[-1], q_at[-1] + 3, k_at[-1] + 5, Hq, Hk, D, dtype)
    for n_split in (None, 1, 3):
        print("packed", dtype, count, Hq, Hk, D, window, n_split, flush=True)
        out = torch.full(q.shape, 9.0, dtype=dtype, device=dev)
        got, lse = ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), _i32(q_at, dev),
                                        k_offsets=_i32(k_at, dev), window=window or None,
                                        sinks=sinks, block=block, return_lse=True, out=out,
                                        n_split=n_split)
        assert got.data_ptr() == out.data_ptr()
        _check(got, lse, q, k, v, q_at, k_at, window, sinks, block, True, D ** -0.5, fill=9.0)


@pytest.mark.parametrize("B", [63, 64, 65, 130, 512, 513, 4097])
@pytest.mark.parametrize("window", [0, 20])
def test_many_requests(dev, B, window):
    """Both orders of the row blocks, requests past a search's 64 and past those that are
    ranked; some have no rows."""
    from cast_amd import ops
    count = [(29 * b) % 37 if b % 5 else 0 for b in range(B)]
    count[B // 3] = 300
    before = [(7 * b) % 50 if b % 3 == 0 else 0 for b in range(B)]
    q_at, k_at = _offsets(count), _offsets([n + m for n, m in zip(count, before)])
    q, k, v = _inputs(B, q_at[-1], k_at[-1], 2, 1, 64, BF)
    out, lse = ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), _i32(q_at, dev),
                                    k_offsets=_i32(k_at, dev), window=window or None,
                                    return_lse=True)
    pick = sorted(set(range(0, B, max(1, B // 60))) | {B // 3, B - 1})
    for b in pick:
        sl, kl = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        n, m = count[b], count[b] + before[b]
        _check(out[sl], lse[:, sl], q[sl], k[kl], v[kl], [0, n], [0, m], window, 0, 1, True, 1 / 8)
    # every row was written: the padded form of the same batch gives the same values
    live = torch.zeros(q_at[-1], dtype=torch.bool)
    live[:] = True
    assert torch.isfinite(out[live.to(dev)].float()).all()


def test_equals_the_dense_form(dev):
    """One request: the same sums in the same order as window_attention's whole blocks."""
    from cast_amd import ops
    q, k, v = (t.to(dev) for t in _inputs(5, 777, 777, 4, 2, 128, BF))
    for window, sinks in ((None, 0), (100, 5)):
        want = ops.window_attention(q[None], k[None], v[None], window=window, sinks=sinks, n_split=1)
        got = ops.packed_attention(q, k, v, _i32([0, 777], dev), window=window, sinks=sinks, n_split=1)
        assert torch.equal(got, want[0])


@pytest.mark.parametrize("n_split", [None, 2])
def test_all_keys_and_unseen_values(dev, n_split):
    """Rows without order; a neighbour's NaN and infinities beside a request's last keys."""
    from cast_amd import ops
    q_at, k_at = _offsets([50, 70, 3]), _offsets([45, 130, 10])
    q, k, v = _inputs(3, 123, 185, 4, 2, 64, BF)
    k[45:60], v[45:60] = float("nan"), float("inf")
    v[44, 1, 3] = float("-inf")
    for causal in (False, True):
        out, lse = ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), _i32(q_at, dev),
                                        k_offsets=_i32(k_at, dev), causal=causal, sm_scale=0.3,
                                        return_lse=True, n_split=n_split)
        for b in (0, 2):
            sl = slice(q_at[b], q_at[b + 1])
            kl = slice(k_at[b], k_at[b + 1])
            _check(out[sl], lse[:, sl], q[sl], k[kl], v[kl], [0, q_at[b + 1] - q_at[b]],
                   [0, k_at[b + 1] - k_at[b]], 0, 0, 1, causal, 0.3)


def test_offsets_past_the_rows(dev):
    """Offsets are held within the rows; where they decrease, which is not allowed, rows that
    one request has are still its own (those that two have may be either's)."""
    from cast_amd import ops
    q, k, v = _inputs(4, 100, 100, 2, 2, 64, HF)
    out = torch.full(q.shape, 9.0, dtype=HF, device=dev)
    ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), _i32([-5, 40, 90, 70, 900], dev), out=out)
    for lo, hi, own in ((0, 40, 40), (40, 90, 70), (70, 100, 100)):
        got = torch.full(q.shape, 9.0, dtype=HF, device=dev)
        ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), _i32([lo, hi], dev), out=got)
        _check(got[lo:hi], None, q[lo:hi], k[lo:hi], v[lo:hi], [0, hi - lo], [0, hi - lo], 0, 0, 1,
               True, 1 / 8)
        first = max(lo, 90) if lo == 70 else lo
        assert torch.equal(out[first:own], got[first:own])


def test_strides_and_no_keys(dev):
    """Parts of a fused projection; no keys; no rows; no requests."""
    from cast_amd import ops
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(150, 6, 128, generator=g).to(BF).to(dev)
    q, k, v = qkv[:, :4], qkv[:, 4:5], qkv[:, 5:]
    at = [0, 100, 150]
    out, lse = ops.packed_attention(q, k, v, _i32(at, dev), return_lse=True)
    _check(out, lse, *(t.cpu() for t in (q, k, v)), at, at, 0, 0, 1, True, 128 ** -0.5)
    none = torch.empty(0, 1, 128, dtype=BF, device=dev)
    out, lse = ops.packed_attention(q, none, none, _i32(at, dev), k_offsets=_i32([0, 0, 0], dev),
                                    return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all() and (lse < 0).all()
    assert ops.packed_attention(q[:0], none, none, _i32([0, 0], dev)).shape == (0, 4, 128)
    assert ops.packed_attention(q, k, v, _i32([0], dev)).shape == q.shape


def test_graph_and_stream(dev):
    """A captured call follows the offsets; two captured calls beside each other; another
    stream."""
    from cast_amd import ops
    q, k, v = _inputs(4, 400, 400, 4, 2, 128, BF)
    dq, dk, dv = (t.to(dev) for t in (q, k, v))
    at = _i32([0, 100, 400], dev)
    outs = [torch.full(q.shape, 9.0, dtype=BF, device=dev) for _ in range(2)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.packed_attention(dq, dk, dv, at, out=outs[0], n_split=3)
    stream.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in outs]
    for g, out, n in zip(graphs, outs, (3, 2)):
        with torch.cuda.graph(g):
            ops.packed_attention(dq, dk, dv, at, out=out, n_split=n)
    for offs in ([0, 200, 400], [10, 10, 390], [0, 1, 2], [0, 399, 400]):
        at.copy_(_i32(offs, dev))
        for out in outs:
            out.fill_(9.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            _check(out, None, q, k, v, offs, offs, 0, 0, 1, True, 128 ** -0.5, fill=9.0)


def test_far_rows(dev):
    """Keys, values, queries and outputs whose offsets pass 32 bits."""
    from cast_amd import ops
    T, Tk, Hq, D, wide = 310, 10000, 2, 128, 1 << 18
    q, k, v = _inputs(6, T, Tk, Hq, 1, D, BF)
    store = torch.empty(Tk, wide, dtype=BF, device=dev)  # 5.2 GB
    far_k, far_v = store[:, :D].unsqueeze(1), store[:, D:2 * D].unsqueeze(1)
    far_k.copy_(k)
    far_v.copy_(v)
    far_q = store[-T:, 2 * D:4 * D].unflatten(1, (Hq, D))
    far_o = store[-T:, 4 * D:6 * D].unflatten(1, (Hq, D))
    far_q.copy_(q)
    offs, k_offs = _i32([0, 300, 310], dev), _i32([0, 9000, 10000], dev)
    for kw in (dict(), dict(window=400), dict(n_split=3)):
        want = ops.packed_attention(q.to(dev), k.to(dev), v.to(dev), offs, k_offsets=k_offs, **kw)
        ops.packed_attention(far_q, far_k, far_v, offs, k_offsets=k_offs, out=far_o, **kw)
        assert torch.equal(far_o, want), kw
