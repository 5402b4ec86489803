"""``ops.append_cache`` and ``ops.read_cache`` against the definition in 64 bits: codes and
scales are equal; a value read back is off by the rounding of c * s to fp32 and that to the
type, half a step each."""
import pytest
import torch

from oracle import cache_oracle as co

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
I8, F8 = torch.int8, torch.float8_e4m3fn
HALF_STEP = {BF: 2.0 ** -8, HF: 2.0 ** -11, F32: 0.0}


class Cache:
    """A cache of random codes on the device and what it holds in 64 bits on the CPU."""

    def __init__(self, dev, seed, code, pages, slots, block, H, D, width, heads_first=False):
        g = torch.Generator().manual_seed(seed)
        shape = (pages, slots, H, D)
        self.code, self.block = code, block
        self.v, self.s, self.t = [], [], []
        for _ in range(2):
            x = torch.randn(shape, generator=g) * (40.0 if code == I8 else 90.0)
            x = x.round().clamp(-127, 127).to(I8) if code == I8 else x.clamp(-448, 448).to(F8)
            e = torch.randint(-9, -4, (pages, slots // block, H), generator=g)
            s = (torch.rand(e.shape, generator=g) + 1) * 0.01 if code == I8 else \
                torch.tensor([2.0 ** int(n) for n in e.flatten()]).view(e.shape)
            self.v.append({"v": x.double(), "code": code})
            self.s.append(s.double())
            if heads_first:  # pages [pages, H, slots, D], scales [blocks, pages, H]
                x = x.view(torch.uint8).transpose(1, 2).contiguous().to(dev).view(code)
                x = x.transpose(1, 2)
                s = s.transpose(0, 1).contiguous().to(dev).transpose(0, 1)
            self.t += [x.to(dev), s.to(dev)]
        self.table = torch.randperm(pages, generator=g)[:width[0] * width[1]].view(width).int()
        self.dev = dev

    def cache(self):
        from cast_amd.ops import QuantizedCache
        return QuantizedCache(self.t[0], self.t[2], self.t[1], self.t[3], self.table.to(self.dev))

    def append(self, kv, b, x, first):
        co.append(self.v[kv], self.s[kv], self.table[b].tolist(), self.block, x, first)

    def check(self):
        """Every code and scale, those that no append reaches too."""
        for kv in range(2):
            got = self.t[2 * kv].cpu().float().double()
            assert torch.equal(got, self.v[kv]["v"]), (kv, (got != self.v[kv]["v"]).sum().item())
            scale = self.t[2 * kv + 1].cpu().double()
            same = (scale == self.s[kv]) | (torch.isnan(scale) & torch.isnan(self.s[kv]))
            assert same.all(), kv


def _tokens(seed, shape, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x = x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=g))
    return x.to(dtype)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


SHAPES = [  # H, D, slots, block
    (1, 64, 16, 16), (3, 128, 64, 32), (2, 80, 48, 16), (4, 256, 32, 32), (2, 96, 256, 256),
    (5, 8, 16, 16), (2, 128, 128, 128), (1, 256, 512, 512)]


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("H,D,slots,block", SHAPES)
def test_append(dev, dtype, code, H, D, slots, block):
    """Appends behind each other from any start: blocks that begin, grow and are passed over,
    scales that grow and stay, zeros, infinities and NaN."""
    from cast_amd import ops
    print("append", dtype, code, H, D, slots, block, flush=True)
    B, width = 3, 4
    c = Cache(dev, D + slots, code, B * width + 2, slots, block, H, D, (B, width))
    c.table[1, 2] = -1
    c.table[2, 3] = B * width + 2
    at = [0, block - 1, 2 * slots - 3]
    for step, L in enumerate((1, block + 5, 2, 1, slots)):
        k, v = (_tokens(7 * step + i, (B, L, H, D), dtype) for i in range(2))
        k[0, 0, 0] = 0.0
        v[1, L // 2, H - 1, D - 1] = float("inf")
        v[1, L // 2, H - 1, 0] = float("-inf")
        k[2, 0, 0, 3] = float("nan")
        n = [L, max(1, L // 2), L - 1]
        ops.append_cache(k.to(dev), v.to(dev), c.cache(), _i32(at, dev), lengths=_i32(n, dev))
        for b in range(B):
            c.append(0, b, k[b, :n[b]], at[b])
            c.append(1, b, v[b, :n[b]], at[b])
            at[b] += n[b]
        c.check()


@pytest.mark.parametrize("code", [I8, F8])
def test_append_places(dev, code):
    """Starts before the first key and past the table, lengths past the tokens, no tokens."""
    from cast_amd import ops
    H, D, slots = 2, 64, 32
    c = Cache(dev, 3, code, 30, slots, 16, H, D, (6, 3))
    starts = [-5, 90, 96, 2 ** 31 - 1, -2 ** 31, 7]
    lengths = [20, 99, 20, 20, 20, -4]
    k, v = (_tokens(i, (6, 20, H, D), BF) for i in range(2))
    ops.append_cache(k.to(dev), v.to(dev), c.cache(), _i32(starts, dev),
                     lengths=_i32(lengths, dev))
    for b in range(6):
        n = max(0, min(20, lengths[b]))
        c.append(0, b, k[b, :n], starts[b])
        c.append(1, b, v[b, :n], starts[b])
    c.check()
    # no starts: from key 0, and the blocks' old scales count for nothing
    ops.append_cache(k.to(dev), v.to(dev), c.cache())
    for b in range(6):
        c.append(0, b, k[b], 0)
        c.append(1, b, v[b], 0)
    c.check()


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_values(dev, dtype, code):
    """Values halfway between two codes, the smallest and the largest of a type, old scales that
    hold nothing; a block of zeros."""
    from cast_amd import ops
    H, D, B = 1, 64, 8
    c = Cache(dev, 5, code, 20, 16, 16, H, D, (B, 2))
    k = torch.zeros(B, 9, H, D)
    ramp = torch.arange(D, dtype=torch.float32)
    k[0, :, 0] = ramp * 2 / 127 * 63.5          # x / s = 127 x / max, many of them n + 1/2
    k[1, :, 0] = (ramp - 31.5) / 31.5 * 448     # e4m3: between its steps
    k[2, :, 0] = ramp * 2.0 ** -126             # under the least scale
    k[3, :, 0] = (ramp - 30) * 5e36             # the largest
    k[4, 3, 0, 7] = 2.0 ** -133                 # a subnormal alone
    k[5, :, 0] = 448 * 2.0 ** -3 * (1 + ramp[:9, None] * 2.0 ** -7)  # around a power's border
    k[6, :, 0] = ramp * 2.0 ** -101             # around the least scale
    k = k.to(dtype)
    starts = [0, 0, 0, 0, 0, 3, 5, 9]
    c.s[0][:, :, :] = torch.where(torch.arange(20)[:, None, None] % 2 == 0, c.s[0], c.s[0] * 2.0 ** 4)
    for b, bad in ((5, float("nan")), (6, -1.0), (7, float("inf"))):
        c.s[0][c.table[b, 0]] = bad
    c.t[1].copy_(c.s[0].float())
    c.s[0] = c.t[1].cpu().double()
    ops.append_cache(k.to(dev), k.to(dev), c.cache(), _i32(starts, dev))
    for b in range(B):
        c.append(0, b, k[b], starts[b])
        c.append(1, b, k[b], starts[b])
    c.check()


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("B", [1, 5, 64, 65, 200])
def test_append_packed(dev, code, B):
    """Packed requests of any number and length, none too; rows before the first and behind the
    last belong to nobody."""
    from cast_amd import ops
    H, D, slots = 2, 64, 32
    c = Cache(dev, B, code, B * 3, slots, 16, H, D, (B, 3))
    count = [(29 * b) % 41 if b % 7 else 0 for b in range(B)]
    starts = [(11 * b) % 23 for b in range(B)]
    offsets = [3]
    for n in count:
        offsets.append(offsets[-1] + n)
    k, v = (_tokens(i, (offsets[-1] + 5, H, D), HF) for i in range(2))
    print("packed append", B, flush=True)
    ops.append_cache(k.to(dev), v.to(dev), c.cache(), _i32(starts, dev),
                     offsets=_i32(offsets, dev))
    for b in range(B):
        for kv, x in enumerate((k, v)):
            c.append(kv, b, x[offsets[b]:offsets[b + 1]], starts[b])
    c.check()


def test_append_packed_offsets_past_the_rows(dev):
    """Offsets are held within the rows."""
    from cast_amd import ops
    H, D = 1, 64
    c = Cache(dev, 9, I8, 12, 32, 16, H, D, (3, 4))
    k, v = (_tokens(i, (50, H, D), BF) for i in range(2))
    ops.append_cache(k.to(dev), v.to(dev), c.cache(), offsets=_i32([-7, 20, 45, 900], dev))
    for b, (lo, hi) in enumerate(((0, 20), (20, 45), (45, 50))):
        c.append(0, b, k[lo:hi], 0)
        c.append(1, b, v[lo:hi], 0)
    c.check()


@pytest.mark.parametrize("code", [I8, F8])
def test_strides(dev, code):
    """Pages with the heads ahead of the slots, tokens of a fused projection."""
    from cast_amd import ops
    B, L, H, D = 2, 37, 3, 128
    c = Cache(dev, 21, code, 9, 64, 32, H, D, (B, 2), heads_first=True)
    qkv = _tokens(1, (B, L, 3, H, D), BF).to(dev)
    k, v = qkv[:, :, 1], qkv[:, :, 2]
    ops.append_cache(k, v, c.cache(), _i32([0, 40], dev))
    for b in range(B):
        c.append(0, b, k[b].cpu(), 40 * b)
        c.append(1, b, v[b].cpu(), 40 * b)
    c.check()
    out = torch.full((B, H, 80, D), 9.0, dtype=BF, device=dev)
    ko, vo = out.transpose(1, 2), out.clone().transpose(1, 2)
    ops.read_cache(c.cache(), _i32([37, 77], dev), size=80, out=(ko, vo))
    for kv, x in enumerate((ko, vo)):
        _check_read(x, c, kv, [0, 0], [37, 77], BF, fill=9.0)


def _check_read(out, c, kv, starts, lengths, dtype, fill=None):
    out = out.cpu().double()
    size, cap = out.shape[1], c.table.shape[1] * c.v[0]["v"].shape[1]
    for b, (lo, n) in enumerate(zip(starts, lengths)):
        ref = co.read(c.v[kv]["v"], c.s[kv], c.table[b].tolist(), c.block, lo, lo + size)
        j = lo + torch.arange(size)
        live = (j >= 0) & (j < min(n, cap))
        off = (out[b] - ref).abs() - ref.abs() * (2.0 ** -24 * (1 + 2.0 ** -8) + HALF_STEP[dtype]) \
            - (2.0 ** -25 if dtype == HF else 0.0)
        assert (off[live] <= 0).all(), (b, off[live].max().item())
        if fill is not None:
            assert (out[b][~live] == fill).all(), b


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("H,D,slots,block", SHAPES)
def test_read(dev, dtype, code, H, D, slots, block):
    """Any range of keys: within a page, over pages that are not there, past the end."""
    from cast_amd import ops
    print("read", dtype, code, H, D, slots, block, flush=True)
    B, width = 5, 3
    c = Cache(dev, D * slots, code, B * width, slots, block, H, D, (B, width))
    c.table[1, 1] = -1
    c.table[2, 0] = 10 ** 6
    cap = width * slots
    starts, lengths = [0, 5, -3, cap - 2, 7], [cap, cap - 1, 11, 2 ** 31 - 1, 0]
    size = 2 * slots + 7
    out = tuple(torch.full((B, size, H, D), 9.0, dtype=dtype, device=dev) for _ in range(2))
    got = ops.read_cache(c.cache(), _i32(lengths, dev), size=size, starts=_i32(starts, dev),
                         out=out)
    for kv in range(2):
        assert got[kv].data_ptr() == out[kv].data_ptr()
        _check_read(out[kv], c, kv, starts, lengths, dtype, fill=9.0)
    k, v = ops.read_cache(c.cache(), _i32([size] * B, dev), size=size, dtype=dtype)
    assert k.dtype == dtype and k.shape == (B, size, H, D)
    _check_read(v, c, 1, [0] * B, [size] * B, dtype)


def test_read_where_values_overflow(dev):
    """c * s past fp16: infinities, as a conversion gives them; bf16 and fp32 hold it."""
    from cast_amd import ops
    c = Cache(dev, 2, I8, 2, 16, 16, 1, 64, (1, 2))
    c.t[1].fill_(1e4)
    c.s[0].fill_(float(torch.tensor(1e4)))
    n = _i32([32], dev)
    for dtype in (BF, F32):
        _check_read(ops.read_cache(c.cache(), n, size=32, dtype=dtype)[0], c, 0, [0], [32], dtype)
    ref = co.read(c.v[0]["v"], c.s[0], c.table[0].tolist(), 16, 0, 32).to(HF)
    assert torch.equal(ops.read_cache(c.cache(), n, size=32, dtype=HF)[0][0].cpu(), ref)
    assert torch.isinf(ref).any()


def test_empty_calls(dev):
    from cast_amd import ops
    c = Cache(dev, 2, I8, 4, 16, 16, 2, 64, (2, 2))
    none = torch.empty(2, 0, 2, 64, dtype=BF, device=dev)
    ops.append_cache(none, none, c.cache(), _i32([3, 4], dev))
    none = torch.empty(0, 2, 64, dtype=BF, device=dev)
    ops.append_cache(none, none, c.cache(), offsets=_i32([0, 0, 0], dev))
    c.check()
    assert ops.read_cache(c.cache(), _i32([3, 4], dev), size=0)[0].shape == (2, 0, 2, 64)


def test_append_graph_and_stream(dev):
    """A captured append follows starts, tokens and table; another stream than the default."""
    from cast_amd import ops
    B, H, D = 3, 2, 128
    c = Cache(dev, 4, I8, 12, 32, 16, H, D, (B, 4))
    cache = c.cache()
    k, v = (torch.zeros(B, 1, H, D, dtype=BF, device=dev) for _ in range(2))
    starts, ends = _i32([0] * B, dev), _i32([1] * B, dev)
    out = tuple(torch.zeros(B, 40, H, D, dtype=BF, device=dev) for _ in range(2))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ops.append_cache(k, v, cache, starts)
        ops.read_cache(cache, ends, size=40, out=out)
    stream.synchronize()
    for b in range(B):
        c.append(0, b, k[b].cpu(), 0)
        c.append(1, b, v[b].cpu(), 0)
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.append_cache(k, v, cache, starts)
        ops.read_cache(cache, ends, size=40, out=out)
    for step in range(5):
        k.copy_(_tokens(step, k.shape, BF))
        v.copy_(_tokens(50 + step, v.shape, BF))
        at = [step, 15 + step, 31 + step]
        starts.copy_(_i32(at, dev))
        ends.copy_(_i32([n + 1 for n in at], dev))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            c.append(0, b, k[b].cpu(), at[b])
            c.append(1, b, v[b].cpu(), at[b])
        c.check()
        _check_read(out[1], c, 1, [0] * B, [n + 1 for n in at], BF)


@pytest.mark.parametrize("code", [I8, F8])
def test_far_pages(dev, code):
    """Codes, tokens and dense rows whose offsets pass 32 bits."""
    from cast_amd import ops
    B, L, H, D, pages, page, block = 2, 70, 2, 64, 12, 32, 16
    c = Cache(dev, 21, code, pages, page, block, H, D, (B, 3))
    near = c.cache()
    store = torch.empty(pages, 1 << 29, dtype=torch.int8, device=dev)  # 6.4 GB
    size = page * H * D
    far = [store[:, i * size:(i + 1) * size].view(code).unflatten(1, (page, H, D))
           for i in range(2)]
    far[0].view(torch.uint8).copy_(near.k.view(torch.uint8))
    far[1].view(torch.uint8).copy_(near.v.view(torch.uint8))
    far = ops.QuantizedCache(*far, near.k_scale.clone(), near.v_scale.clone(), near.table)
    rows = torch.empty(B * L, 1 << 23, dtype=BF, device=dev)[:, :4 * H * D]  # 2.3 GB
    k, v, ko, vo = rows.unflatten(1, (4, H, D)).unflatten(0, (B, L)).unbind(2)
    for seed, t in enumerate((k, v)):
        t.copy_(_tokens(seed, t.shape, BF))
    starts, ends = _i32([0, 9], dev), _i32([L, 9 + L], dev)
    ops.append_cache(k.contiguous(), v.contiguous(), near, starts)
    ops.append_cache(k, v, far, starts)
    for a, b in ((near.k, far.k), (near.v, far.v)):
        assert torch.equal(a.view(torch.uint8), b.contiguous().view(torch.uint8))
    assert torch.equal(near.k_scale, far.k_scale) and torch.equal(near.v_scale, far.v_scale)
    want = ops.read_cache(near, ends, size=L, starts=starts)
    ops.read_cache(far, ends, size=L, starts=starts, out=(ko, vo))
    assert torch.equal(ko, want[0]) and torch.equal(vo, want[1])
