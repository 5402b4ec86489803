"""``ops.paged_attention`` over a ``QuantizedCache`` beside blocks that no row sees: behind a
request's keys, ahead of its window, on stale pages of its table.  Whatever their scales hold,
the rows are those that scales of 0 there give, to the bit, and within the oracle's bound of the
definition, with the largest scale that is *seen* in it (see ``cache_oracle.attention``)."""
import pytest
import torch

from oracle import cache_oracle as co
from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
I8, F8 = torch.int8, torch.float8_e4m3fn
TOP = {I8: 127.0, F8: 448.0}


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _queries(seed, shape, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Pages:
    """Requests of `width` pages each, all of them there, and which of their blocks are seen."""

    def __init__(self, dev, seed, code, k_len, page, mark, H, D, width):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.code, self.page, self.mark = dev, code, page, mark
        n = len(k_len) * width
        x = [torch.randn(n, page, H, D, generator=g) for _ in range(2)]
        self.c = [(t * 40).round().clamp(-127, 127).to(I8) if code == I8 else
                  (t * 100).clamp(-448, 448).to(F8) for t in x]
        wide = 1 / 40 if code == I8 else 1 / 100
        self.s = [wide * (1 + torch.rand(n, page // mark, H, generator=g)) for _ in range(2)]
        self.table = torch.randperm(n, generator=g).view(len(k_len), width).int()

    def block_of(self, b, j):
        """Page and block of keys j of request b."""
        return self.table[b, j // self.page].long(), j % self.page // self.mark

    def unseen(self, seen):
        """bool [pages, blocks]: no key of the block is among seen[b] (bool [rows, keys])."""
        free = torch.ones(self.s[0].shape[:2], dtype=torch.bool)
        for b, rows in enumerate(seen):
            free[self.block_of(b, rows.any(0).nonzero()[:, 0])] = False
        return free

    def cache(self, kv, free, far):
        """The cache with scales `far` (of keys: kv 0, of values: 1) where `free`."""
        from cast_amd.ops import QuantizedCache
        s = [t.clone() for t in self.s]
        s[kv][free] = far
        c, s = [t.to(self.dev) for t in self.c], [t.to(self.dev) for t in s]
        return QuantizedCache(c[0], c[1], s[0], s[1], self.table.to(self.dev))

    def check(self, out, lse, q, seen, sm_scale):
        dev = self.dev
        for b, rows in enumerate(seen):
            j = torch.arange(rows.shape[1])
            page, blk = self.block_of(b, j)
            k, v = (c.float()[page, j % self.page].double() * s[page, blk].double()[..., None]
                    for c, s in zip(self.c, self.s))
            used = rows.any(0)
            v = torch.where(used[:, None, None], v, torch.zeros_like(v))
            top = float(self.s[1][page, blk][used].max()) * TOP[self.code]
            ref, rlse, tol, ltol = (t.cpu() for t in co.attention(
                q[b].to(dev), k.to(dev), v.to(dev), top, rows.to(dev), sm_scale, q.dtype))
            worst = ((out[b].cpu().double() - ref).abs() - tol).max().item()
            assert worst <= 0.0, (b, worst)
            worst = ((lse[b].cpu().double() - rlse).abs() - ltol).max().item()
            assert worst <= 0.0, (b, worst)


CASES = [  # Lq, Hq, D, page, mark, window, sinks
    (1, 4, 128, 32, 16, 0, 0), (1, 2, 64, 48, 16, 0, 0), (1, 8, 128, 16, 16, 40, 0),
    (3, 6, 64, 64, 16, 50, 3), (5, 4, 128, 48, 48, 0, 0), (2, 2, 128, 128, 128, 0, 0),
    (40, 4, 128, 32, 16, 0, 0), (40, 2, 64, 48, 16, 70, 5), (130, 2, 128, 16, 16, 0, 0),
    (70, 4, 64, 64, 16, 20, 0), (40, 4, 128, 64, 64, 100, 0)]


def _seen_of(Lq, k_len, window, sinks):
    return [so.visible(Lq, n, window, sinks, 1) for n in k_len]


def _forms(Lq, Hq, Hk):
    """Shares of the launch: planned, and each form that takes the rows."""
    return (-2, -1, 0, 1, 3) if Lq * Hq // Hk <= 32 else (-2, 1, 3)


def _call(cache, q, k_len, window, sinks, n_split, dev):
    from cast_amd import _lib
    return _lib.torch_ops().window_attention(
        q.to(dev), cache.k, cache.v, cache.table, None, _i32(k_len, dev), window, sinks, 1, None,
        True, None, n_split, -1, cache.k_scale, cache.v_scale)


@pytest.mark.parametrize("code,dtype", [(I8, BF), (F8, HF)])
@pytest.mark.parametrize("Lq,Hq,D,page,mark,window,sinks", CASES)
def test_value_scales_of_unseen_blocks(dev, code, dtype, Lq, Hq, D, page, mark, window, sinks):
    Hk, k_len = 2, [Lq + 9, 170 + Lq % 2, 332]  # (the last tiles end in their first half)
    p = Pages(dev, Lq + page, code, k_len, page, mark, Hk, D, -(-400 // page))
    q = _queries(Lq, (3, Lq, Hq, D), dtype)
    seen = _seen_of(Lq, k_len, window, sinks)
    free = p.unseen(seen)
    for n_split in _forms(Lq, Hq, Hk):
        print("unseen", code, Lq, page, mark, window, n_split, flush=True)
        want = _call(p.cache(1, free, 0.0), q, k_len, window, sinks, n_split, dev)
        p.check(*want, q, seen, D ** -0.5)
        for far in (1e4, 1e6, 1e20, 2.0 ** 125):
            got = _call(p.cache(1, free, far), q, k_len, window, sinks, n_split, dev)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (n_split, far)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("page,mark", [(32, 16), (48, 16), (64, 32), (48, 48)])
@pytest.mark.parametrize("window", [0, 64])
def test_value_scales_that_other_rows_see(dev, code, page, mark, window):
    """Blocks of 128 rows, whose wavefronts take 32 each: large scales of the keys that only the
    last 32 rows see (under a window also those that only the first 32 see) leave the others'
    results as they are."""
    Lq, Lk, Hk, D = 128, 192, 1, 128  # (row i is position i + 64)
    p = Pages(dev, page + mark, code, [Lk], page, mark, Hk, D, Lk // page)
    q = _queries(9, (1, Lq, 1, D), BF)
    seen = so.visible(Lq, Lk, window, 0, 1)
    for own, free in ((slice(0, 96), p.unseen([seen[:96]])), (slice(32, 128), p.unseen([seen[32:]]))):
        if not free.any():
            continue
        print("others", code, page, mark, window, own, flush=True)
        want = _call(p.cache(1, free, 1e-3), q, [Lk], window, 0, 1, dev)
        for far in (1e4, 1e20):
            got = _call(p.cache(1, free, far), q, [Lk], window, 0, 1, dev)
            assert torch.equal(got[0][:, own], want[0][:, own]), (own, far)
            assert torch.equal(got[1][:, :, own], want[1][:, :, own]), (own, far)


@pytest.mark.parametrize("code,dtype", [(I8, BF), (F8, HF)])
@pytest.mark.parametrize("Lq,Hq,D,page,mark,window,sinks", CASES)
def test_key_scales_of_unseen_blocks(dev, code, dtype, Lq, Hq, D, page, mark, window, sinks):
    """Queries of either sign's sum: what a code's offset takes off a logit has it too."""
    Hk, k_len = 2, [Lq + 9, 170 + Lq % 2, 332]
    p = Pages(dev, Lq + page, code, k_len, page, mark, Hk, D, -(-400 // page))
    q = _queries(Lq, (3, Lq, Hq, D), dtype) - 0.2
    q[:, :, 0] = -q[:, :, 0]
    seen = _seen_of(Lq, k_len, window, sinks)
    free = p.unseen(seen)
    for n_split in _forms(Lq, Hq, Hk):
        print("unseen keys", code, Lq, page, mark, window, n_split, flush=True)
        want = _call(p.cache(0, free, 0.0), q, k_len, window, sinks, n_split, dev)
        p.check(*want, q, seen, D ** -0.5)
        for far in (1e6, 1e20, 2.0 ** 125):
            got = _call(p.cache(0, free, far), q, k_len, window, sinks, n_split, dev)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (n_split, far)


@pytest.mark.parametrize("page,mark", [(32, 16), (48, 16), (64, 32), (48, 48)])
@pytest.mark.parametrize("window", [0, 64])
def test_key_scales_that_other_rows_see(dev, page, mark, window):
    """As for the values: scales so large that a logit's offset overflows."""
    Lq, Lk, Hk, D = 128, 192, 1, 128
    p = Pages(dev, page + mark, I8, [Lk], page, mark, Hk, D, Lk // page)
    seen = so.visible(Lq, Lk, window, 0, 1)
    for sign in (-1.0, 1.0):
        q = sign * (_queries(9, (1, Lq, 1, D), BF) + 0.3)
        for own, free in ((slice(0, 96), p.unseen([seen[:96]])),
                          (slice(32, 128), p.unseen([seen[32:]]))):
            if not free.any():
                continue
            print("other rows' keys", page, mark, window, own, sign, flush=True)
            want = _call(p.cache(0, free, 1e-3), q, [Lk], window, 0, 1, dev)
            for far in (1e20, 2.0 ** 125):
                got = _call(p.cache(0, free, far), q, [Lk], window, 0, 1, dev)
                assert torch.equal(got[0][:, own], want[0][:, own]), (own, far)
                assert torch.equal(got[1][:, :, own], want[1][:, :, own]), (own, far)


@pytest.mark.parametrize("kv", [0, 1])
@pytest.mark.parametrize("code,dtype", [(I8, BF), (F8, HF)])
@pytest.mark.parametrize("page,mark", [(32, 16), (48, 16), (64, 32), (48, 48)])
@pytest.mark.parametrize("Lq,window", [(30, 0), (30, 40), (100, 0), (100, 50)])
def test_scales_that_later_rows_see(dev, kv, code, dtype, page, mark, Lq, window):
    """Rows beside each other (few, or blocks of them): any scale of a block that starts behind
    a row's position, or ends ahead of its window, leaves the row within the bound of the scales
    that it sees."""
    Lk, Hk, D = 300, 1, 128
    p = Pages(dev, page + mark, code, [Lk], page, mark, Hk, D, -(-Lk // page))
    q = _queries(9, (1, Lq, 1, D), dtype) - 0.2
    seen = so.visible(Lq, Lk, window, 0, 1)
    cut = 288 - (Lk - Lq)  # the rows ahead of key 288, a block's first whatever the mark
    for rows in (slice(0, cut), slice(Lq - 8, Lq)):
        free = p.unseen([seen[rows]])
        if not free.any():
            continue
        for n_split in _forms(Lq, 1, Hk):
            for far in (1e6, 1e20, 2.0 ** 125):
                print("later rows", kv, code, page, mark, Lq, window, rows, n_split, far, flush=True)
                out, lse = _call(p.cache(kv, free, far), q, [Lk], window, 0, n_split, dev)
                p.check(out[:, rows], lse[:, :, rows], q[:, rows], [seen[rows]], D ** -0.5)
