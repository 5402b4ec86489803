"""``ops.window_attention`` and ``ops.paged_attention`` where rows, weights and shares come to
their edges: rows that see no key beside values that are no numbers, shares whose weight underflows,
weights far below the largest.

Tolerances: the oracle's bound (see ``streaming_oracle.attention``)."""
import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
NAN, INF = float("nan"), float("inf")


def _inputs(seed, B, Lq, Lk, Hq, Hk, D, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Lq, Hq, D, generator=g)
    k = torch.randn(B, Lk, Hk, D, generator=g)
    v = torch.randn(B, Lk, Hk, D, generator=g) + 0.5
    return tuple(t.to(dtype).to(dev) for t in (q, k, v))


def _within(got, ref, tol, what):
    """Within the bound; NaN and infinities where the oracle has them."""
    got = got.double()
    off = (got - ref).abs()
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    worst = torch.where(same, torch.zeros_like(off), off - tol)
    worst = torch.nan_to_num(worst, nan=INF).max().item()
    assert worst <= 0.0, f"{what}: {worst} past the bound"


def _call(q, k, v, page, table, n_split, window, sinks, block, sm_scale):
    """One request of q [1, Lq, Hq, D] over dense keys, or (page > 0) over pages of them whose
    last page is filled up with NaN; n_split 0 and -1 are the forms of few rows."""
    from cast_amd import _lib
    n, Lk = k.shape[1], k.shape[1]
    lens = None
    if page:
        M = max(1, -(-n // page))
        pad = torch.full((1, M * page - n, *k.shape[2:]), NAN, dtype=k.dtype, device=k.device)
        k, v = (torch.cat([t, pad], 1).view(M, page, *t.shape[2:]) for t in (k, v))
        lens = torch.tensor([Lk], dtype=torch.int32, device=q.device)
        if table is None:
            table = torch.arange(M, dtype=torch.int32, device=q.device)[None]
    return _lib.torch_ops().window_attention(
        q, k, v, table if page else None, None, lens, window, sinks, block, sm_scale, True, None,
        -2 if n_split is None else n_split, -1)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("Lq,Lk,window,sinks,block,n_split", [
    (128, 10, 0, 0, 1, 1), (128, 64, 0, 0, 1, 1), (128, 64, 0, 0, 1, None), (300, 70, 0, 0, 1, 3),
    (150, 70, 100, 0, 880, 1), (150, 70, 100, 0, 880, 2), (4, 70, 100, 0, 880, 0),
    (4, 70, 100, 0, 880, -1), (10, 5, 0, 0, 1, 0), (10, 5, 0, 0, 1, -1), (1, 70, 32, 0, 128, 0)])
def test_rows_without_keys_beside_no_numbers(dev, dtype, page, Lq, Lk, window, sinks, block,
                                             n_split):
    """Rows before the first key, or whose window lies behind the last one, give 0 and -inf,
    whatever the values that their neighbours see, or the last tile holds."""
    print("rows without keys", dtype, page, Lq, Lk, window, block, n_split, flush=True)
    q, k, v = _inputs(Lq + Lk, 1, Lq, Lk, 2, 1, 64, dtype, dev)
    v[0, Lk // 2, 0, 3], v[0, Lk - 1, 0, 9], v[0, 1, 0, 60] = INF, NAN, -INF
    out, lse = _call(q, k, v, page, None, n_split, window, sinks, block, 0.125)
    seen = so.visible(Lq, Lk, window, sinks, block, device=dev)
    assert not seen.any(1).all()
    ref, rlse, tol, ltol = so.attention(q[0], k[0], v[0], seen, 0.125, dtype)
    _within(out[0], ref, tol, "rows")
    _within(lse[0], rlse, ltol, "sums")


@pytest.mark.parametrize("n_split", [None, 1, 2])
def test_rows_of_hidden_pages_beside_no_numbers(dev, n_split):
    """32 rows whose pages are all hidden, in a block whose last rows see an infinity."""
    Lq, page, window = 128, 16, 16
    q, k, v = _inputs(7, 1, Lq, Lq, 1, 1, 128, BF, dev)
    v[0, 100, 0, 5], v[0, 3, 0, 6] = INF, NAN
    table = torch.arange(Lq // page, dtype=torch.int32, device=dev)[None].contiguous()
    table[0, 1:4] = -1
    out, lse = _call(q, k, v, page, table, n_split, window, 0, 1, 0.1)
    seen = so.visible(Lq, Lq, window, 0, 1, device=dev)
    seen[:, page:4 * page] = False
    assert not seen[32:64].any()
    ref, rlse, tol, ltol = so.attention(q[0], k[0], v[0], seen, 0.1, BF)
    _within(out[0], ref, tol, "rows")
    _within(lse[0], rlse, ltol, "sums")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [0, 48])
@pytest.mark.parametrize("Lq,n_split", [
    (40, 1), (40, 2), (40, 5), (4, 1), (4, 3), (4, 0), (4, -1), (4, None)])
def test_infinities_in_a_share_of_no_weight(dev, dtype, page, Lq, n_split):
    """The first half of the keys stands e^-256 below the second: its finite values vanish,
    its infinities and NaN reach every row, however the keys are shared."""
    Lk, D = 700, 64
    q, k, v = _inputs(Lq, 1, Lq, Lk, 2, 1, D, dtype, dev)
    q[..., 0], k[:, :350, :, 0], k[:, 350:, :, 0] = 8.0, -16.0, 16.0
    v[0, 3, 0, 7], v[0, 40, 0, 9], v[0, 340, 0, 11], v[0, 5, 0, 20] = INF, NAN, -INF, 60000.0
    out, lse = _call(q, k, v, page, None, n_split, 0, 0, 1, 1.0)
    seen = so.visible(Lq, Lk, 0, 0, 1, device=dev)
    ref, rlse, tol, ltol = so.attention(q[0], k[0], v[0], seen, 1.0, dtype)
    assert torch.isinf(ref[..., 7]).all() and torch.isnan(ref[..., 9]).all()
    _within(out[0], ref, tol, "rows")
    _within(lse[0], rlse, ltol, "sums")


@pytest.mark.parametrize("tail", [22.5, 25.2])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("page,Lq,n_split", [
    (0, 40, 1), (0, 40, 8), (64, 40, 2), (0, 1, 0), (64, 1, 0), (0, 1, -1), (64, 1, None)])
def test_many_small_weights(dev, page, Lq, n_split, odd, tail):
    """fp16: one key and 2^16 others at 2^-22.5 or 2^-25.2 of its weight, which together are a
    part of the result: their weights keep the bits down to 2^-32 of the largest.  ``odd``:
    beside an infinity, whose rows are taken again.

    The bound: a weight's least step, half of fp16's 2^-24 at a factor of 2^7, 2^-32 of the
    largest; the sums of up to 2048 tiles in fp32, a rounding a tile of the row's sum and two of
    its products, 3 * 2048 * 2^-24 of the result."""
    Lk, D = 1 + (1 << 16), 64
    g = torch.Generator().manual_seed(Lq)
    q, k = (torch.zeros(1, n, 1, D, device=dev, dtype=HF) for n in (Lq, Lk))
    v = (1.0 + 0.1 * torch.randn(1, Lk, 1, D, generator=g)).to(HF).to(dev)
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 1.0, tail * 0.6931471805599453, 0.0
    if odd:
        v[0, 4000, 0, 17] = INF
    out, lse = _call(q, k, v, page, None, n_split, 0, 0, 1, 1.0)
    seen = so.visible(Lq, Lk, 0, 0, 1, device=dev)
    ref, rlse, tol, ltol = so.attention(q[0], k[0], v[0], seen, 1.0, HF, weight_step=2.0 ** -32)
    steps = 2049 * 2.0 ** -24
    _within(out[0], ref, tol + 3 * steps * ref.abs(), "rows")
    _within(lse[0], rlse, ltol + steps, "sums")


def test_plan_of_2_31_tiles(dev):
    """64 requests of 2^30 - 16 keys each, over a table whose entries repeat eight pages: the
    plan counts 2^31 tiles, and every unit finds its place.

    The bound: units of 2^31 / (4 * 3072) tiles, a rounding a tile of the row's sum and two of
    its products in fp32; a weight's half step; logits as in the oracle."""
    from cast_amd import _lib
    B, page, N, D = 64, 16, 8, 64
    M = (1 << 26) - 1
    g = torch.Generator().manual_seed(3)
    q = torch.randn(B, 1, 1, D, generator=g).to(BF).to(dev)
    k, v = (torch.randn(N, page, 1, D, generator=g).to(BF).to(dev) for _ in range(2))
    table = (torch.arange(M, dtype=torch.int32, device=dev) % N)[None].expand(B, M)
    lens = torch.full((B,), M * page, dtype=torch.int32, device=dev)
    out, lse = _lib.torch_ops().window_attention(q, k, v, table, None, lens, 0, 0, 1, 0.125, True,
                                                 None, 0, -1)
    times = torch.tensor([M // N + (i < M % N) for i in range(N)], device=dev).double()
    s = q[:, 0, 0].double() @ k.view(-1, D).double().T.contiguous() * 0.125
    s = s + times.log().repeat_interleave(page)
    row = torch.logsumexp(s, 1, keepdim=True)
    p, vv = torch.exp(s - row), v.view(-1, D).double()
    steps = 2.0 ** 31 / (4 * 3072) * 2.0 ** -24
    tol = (p @ vv.abs()) * (2.0 ** -7 + 3 * steps) + 1e-4
    _within(out[:, 0, 0], p @ vv, tol, "rows")
    _within(lse[:, 0, 0], row[:, 0], torch.full_like(row[:, 0], steps + 1e-3), "sums")


@pytest.mark.parametrize("Lk,window,sinks", [
    (1, 0, 0), (64, 0, 0), (65, 0, 0), (4000, 0, 0), (4000, 100, 40), (4000, 1, 0),
    (200000, 0, 0)])
def test_units_stay_in_their_workspace(dev, Lk, window, sinks):
    """A call over the C ABI with a workspace of just its size: what lies behind it stays, the
    result is that of the torch call."""
    import ctypes
    from cast_amd import _lib
    lib = _lib.load()
    B, Lq, Hq, Hk, D = 2, 3, 8, 2, 128
    q, k, v = _inputs(Lk, B, Lq, Lk, Hq, Hk, D, BF, dev)
    dims = (ctypes.c_int64 * 6)(B, Lq, Lk, Hq, Hk, D)
    need = lib.rcsa_window_attn_workspace_bytes_for(dims, 0, Lk, window, sinks)
    assert need > 0
    ws = torch.full((need + (1 << 20),), 0x5a, dtype=torch.uint8, device=dev)
    out = torch.empty_like(q)
    strides = (ctypes.c_int64 * 12)(*(s for t in (q, k, v, out) for s in t.stride()[:3]))
    assert lib.rcsa_window_attn(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), None, 0, dims, strides, None,
        None, None, 0, 0, 0, 0, window, sinks, 1, 0.1, 0, ws.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream) == 0
    want = _lib.torch_ops().window_attention(q, k, v, None, None, None, window, sinks, 1, 0.1,
                                             False, None, 0, -1)[0]
    assert torch.equal(out, want)
    assert (ws[need:] == 0x5a).all()
