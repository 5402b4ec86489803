"""Outputs of the cache's and the attention's calls that overlap the lengths, starts, offsets or
tables that the kernels read beside them: refused before a launch."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _ints(t, *shape):
    """int32 values in the first bytes of t's memory."""
    n = 1
    for m in shape:
        n *= m
    return t.reshape(-1).view(torch.int32)[:n].view(shape)


@pytest.fixture()
def world(dev):
    from cast_amd import ops
    B, H, D, page, block = 2, 2, 64, 32, 16
    codes = [torch.zeros(8, page, H, D, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.ones(8, page // block, H, device=dev) for _ in range(2)]
    table = torch.arange(8, dtype=torch.int32, device=dev).view(B, 4)
    cache = ops.QuantizedCache(*codes, *scales, table)
    x = torch.ones(B, 3, H, D, dtype=BF, device=dev)
    return ops, cache, x, torch.full((B,), 3, dtype=torch.int32, device=dev)


def test_appends(world):
    ops, cache, x, n = world
    was = [t.clone() for t in cache]
    for own in (cache.k, cache.v, cache.k_scale, cache.v_scale):
        at = _ints(own, 2)
        for call in (lambda: ops.append_cache(x, x, cache, at),
                     lambda: ops.append_cache(x, x, cache, lengths=at),
                     lambda: ops.append_cache(x[0], x[0], cache._replace(table=cache.table[:1]),
                                              offsets=at)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    assert all(torch.equal(a, b) for a, b in zip(cache, was))
    ops.append_cache(x, x, cache, n, lengths=n)  # (apart: taken)


def test_reads(world):
    ops, cache, x, n = world
    out = (torch.zeros_like(x), torch.zeros_like(x))
    for own in out:
        with pytest.raises(ValueError, match="overlap"):
            ops.read_cache(cache, _ints(own, 2), size=3, out=out)
        with pytest.raises(ValueError, match="overlap"):
            ops.read_cache(cache, n, size=3, starts=_ints(own, 2), out=out)
    assert all((t == 0).all() for t in out)
    ops.read_cache(cache, n, size=3, starts=n, out=out)


def test_attention(world):
    ops, cache, x, n = world
    pages = ops.PagedCache(*(t.to(BF) for t in cache[:2]), cache.table)
    out = torch.zeros_like(x)
    at = _ints(out, 2)
    offs = torch.tensor([0, 1, 3], dtype=torch.int32, device=x.device)
    for call in [lambda c=c: ops.paged_attention(x, c, at, out=out) for c in (cache, pages)] + [
            lambda c=c: ops.paged_attention(x, c, n, q_lengths=at, out=out)
            for c in (cache, pages)] + [
            lambda c=c: ops.paged_attention(x, c._replace(table=_ints(out, 2, 4)), n, out=out)
            for c in (cache, pages)] + [
            lambda: ops.window_attention(x, x, x, k_lengths=at, out=out),
            lambda: ops.packed_attention(x[0], x[0], x[0], _ints(out[0], 3), out=out[0]),
            lambda: ops.packed_attention(x[0], x[0], x[0], offs, k_offsets=_ints(out[0], 3),
                                         out=out[0])]:
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert (out == 0).all()
    for c in (cache, pages):
        ops.paged_attention(x, c, n, q_lengths=n, out=out)
    ops.packed_attention(x[0], x[0], x[0], offs, k_offsets=offs, out=out[0])
