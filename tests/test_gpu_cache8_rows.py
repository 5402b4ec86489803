"""``ops.append_cache`` and ``ops.read_cache`` with fp32 rows that are 16-byte aligned and no
more: strides of a multiple of 4 elements; a long packed request among short ones.  Codes, scales and values are those of contiguous
tensors, which the definition's tests hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(dev, code, B, pages, page, block, H, D):
    from cast_amd.ops import QuantizedCache
    codes = [torch.zeros(pages, page, H, D, dtype=torch.int8, device=dev).view(code)
             for _ in range(2)]
    scales = [torch.zeros(pages, page // block, H, device=dev) for _ in range(2)]
    return QuantizedCache(*codes, *scales,
                          torch.arange(pages, dtype=torch.int32, device=dev).view(B, -1))


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("packed", [False, True])
def test_rows_of_16_bytes(dev, code, packed):
    from cast_amd import ops
    B, L, H, D, page, block = 2, 37, 3, 64, 32, 16
    g = torch.Generator().manual_seed(3)
    # head strides of 68, token strides of 3 * 68 + 4, a first row 16 bytes into the memory
    wide = torch.randn(2, B, L, H * (D + 4) + 4, generator=g).to(dev)
    rows = wide[..., 4:].unflatten(3, (H, D + 4))[..., :D]
    k, v = rows[0], rows[1]
    assert k.stride(2) % 8 == 4 and k.data_ptr() % 32 == 16
    caches = [_cache(dev, code, B, 4, page, block, H, D) for _ in range(2)]
    offsets = torch.tensor([0, L, 2 * L], dtype=torch.int32, device=dev) if packed else None
    for c, (a, b) in zip(caches, ((k, v), (k.contiguous(), v.contiguous()))):
        if packed:
            a, b = a.flatten(0, 1), b.flatten(0, 1)
        ops.append_cache(a, b, c, offsets=offsets)
    for a, b in zip(caches[0][:2], caches[1][:2]):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))
    for a, b in zip(caches[0][2:], caches[1][2:]):
        assert torch.equal(a, b)
    n = torch.full((B,), L, dtype=torch.int32, device=dev)
    out = wide.clone()[..., 4:].unflatten(3, (H, D + 4))
    was = out.clone()
    ops.read_cache(caches[0], n, size=L, out=(out[0, ..., :D], out[1, ..., :D]))
    want = ops.read_cache(caches[0], n, size=L, dtype=torch.float32)
    for i in range(2):
        assert torch.equal(out[i, ..., :D], want[i])
    assert torch.equal(out[..., D:], was[..., D:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
def test_a_long_packed_request_among_short_ones(dev, code, dtype):
    """Blocks far larger than what the requests get on average: the long one's codes and scales
    are those of an append of its own."""
    from cast_amd import ops
    H, D, page, block = 2, 256, 256, 256
    count = [3] * 10 + [700] + [2, 0, 5] * 5
    B, start = len(count), 100
    at = [0]
    for n in count:
        at.append(at[-1] + n)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(at[-1], H, D, generator=g).to(dtype).to(dev) for _ in range(2))
    k[at[10] + 200, 1, 7], v[at[10] + 600, 0, 3] = float("inf"), float("nan")
    starts = torch.full((B,), start, dtype=torch.int32, device=dev)
    packed, alone = (_cache(dev, code, B, 4 * B, page, block, H, D) for _ in range(2))
    ops.append_cache(k, v, packed, starts,
                     offsets=torch.tensor(at, dtype=torch.int32, device=dev))
    for b, n in enumerate(count):
        rows = slice(at[b], at[b + 1])
        ops.append_cache(k[None, rows], v[None, rows], alone._replace(table=alone.table[b:b + 1]),
                         starts[:1])
    for a, b in zip(packed[:2], alone[:2]):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))
    for a, b in zip(packed[2:4], alone[2:4]):
        assert torch.equal(a, b)
