"""``ops.rope`` and ``ops.norm_rope`` against the 64-bit oracle: types, pair layouts, parts
of the head, position axes, far positions, odd sizes, strides, caches and lengths.

Tolerances: the oracle's bound (one rounding to the type, fp32 before it)."""
import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _close(got, ref, tol, what):
    got = got.double().cpu()
    off = (got - ref.cpu()).abs()
    worst = (off - tol.cpu()).max().item()
    assert worst <= 0.0, f"{what}: {worst} past the bound (error {off.max().item()})"


def _plan(dev, R, interleaved=False, **kw):
    from cast_amd.rotary import rotary_plan
    return rotary_plan(R, interleaved=interleaved, device=dev, **kw), *so.frequencies(R, **kw)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,L,H,D,R", [
    (1, 1, 1, 128, 128), (2, 5, 3, 64, 64), (1, 1025, 24, 128, 128), (3, 37, 9, 80, 32),
    (2, 19, 5, 96, 24), (1, 33, 2, 256, 256), (4, 3, 7, 128, 20), (2, 7, 3, 66, 66),
    (1, 9, 1, 6, 2), (1, 300, 33, 16, 16), (2, 4, 2, 512, 510), (1, 6, 4, 128, 0),
    (64, 1, 8, 48, 48), (1, 17, 300, 32, 16)])
def test_rope_shapes(dev, dtype, inter, B, L, H, D, R):
    from cast_amd import ops
    print("rope", dtype, inter, B, L, H, D, R, flush=True)
    plan, freq, axis = _plan(dev, R, inter)
    g = torch.Generator().manual_seed(B * 1000 + L + D)
    x = torch.randn(B, L, H, D, generator=g).to(dtype)
    pos = torch.randint(-50, 5000, (B, L), generator=g, dtype=torch.int32)
    out = ops.rope(x.to(dev), pos.to(dev), plan)
    ref, size = so.rope(x, pos, freq, axis, inter)
    _close(out, ref, so.rope_bound(ref, size, dtype), "rope")


@pytest.mark.parametrize("pos_dtype", [torch.int32, torch.int64])
def test_rope_far_positions(dev, pos_dtype):
    """Angles at positions near 2^31 (int64: 2^40) keep fp32's precision."""
    from cast_amd import ops
    plan, freq, axis = _plan(dev, 64)
    far = 2 ** 31 - 70 if pos_dtype == torch.int32 else 2 ** 40
    pos = (torch.arange(64, dtype=torch.int64) + far).to(pos_dtype)
    x = torch.randn(1, 64, 2, 64, generator=torch.Generator().manual_seed(5))
    out = ops.rope(x.to(dev), pos.to(dev), plan)
    # the product in 64 bits is off by 2^-53 of the position a pair: radians
    ref, size = so.rope(x, pos, freq, axis, False)
    _close(out, ref, so.rope_bound(ref, size, F32) + size * far * 2.0 ** -51, "far")


@pytest.mark.parametrize("scaling,kw", [
    ("linear", dict(factor=4.0)), ("base", dict(factor=8.0)),
    ("ramp", dict(factor=8.0, original_length=4096))])
def test_rope_scaled(dev, scaling, kw):
    from cast_amd import ops
    plan, freq, axis = _plan(dev, 128, scaling=scaling, **kw)
    pos = torch.randint(0, 131072, (2, 40), generator=torch.Generator().manual_seed(3))
    x = torch.randn(2, 40, 4, 128, generator=torch.Generator().manual_seed(4)).to(BF)
    out = ops.rope(x.to(dev), pos.to(dev), plan)
    ref, size = so.rope(x, pos, freq, axis, False, plan.scale)
    _close(out, ref, so.rope_bound(ref, size, BF), scaling)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("per_batch", [False, True])
def test_rope_axes(dev, inter, per_batch):
    from cast_amd import ops
    axes = (44, 42, 42)
    plan, freq, axis = _plan(dev, 128, inter, axes=axes)
    t = torch.arange(2 * 22 * 40)
    pos = torch.stack([t // 880, t % 880 // 40, t % 40], 1)[300:1100]
    if per_batch:
        pos = torch.stack([pos, pos + 3])
    x = torch.randn(2, 800, 3, 128, generator=torch.Generator().manual_seed(8)).to(BF)
    out = ops.rope(x.to(dev), pos.to(dev), plan)
    ref, size = so.rope(x, pos, freq, axis, inter, n_axes=3)
    _close(out, ref, so.rope_bound(ref, size, BF), "axes")


@pytest.mark.parametrize("R", [64, 20])
def test_rope_strides_in_place_and_back(dev, R):
    """Head-major and fused sources, an output of other strides, in place, an odd offset,
    and the rotation undone by negated positions."""
    from cast_amd import ops
    plan, freq, axis = _plan(dev, R)
    g = torch.Generator().manual_seed(9)
    pos = torch.arange(50, dtype=torch.int32)
    x = torch.randn(2, 50, 3, 64, generator=g).to(BF)
    ref, size = so.rope(x, pos, freq, axis, False)
    tol = so.rope_bound(ref, size, BF)
    d = pos.to(dev)
    heads = x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    _close(ops.rope(heads, d, plan), ref, tol, "head-major")
    out = torch.full((2, 3, 50, 64), 7.0, device=dev, dtype=BF).transpose(1, 2)
    assert ops.rope(x.to(dev), d, plan, out=out) is not None
    _close(out, ref, tol, "out strides")
    fused = torch.randn(2, 50, 3, 3, 64, generator=g).to(BF).to(dev)
    keep = fused.clone()
    fused[:, :, 1] = x.to(dev)
    ops.rope(fused[:, :, 1], d, plan, out=fused[:, :, 1])
    _close(fused[:, :, 1], ref, tol, "in place")
    assert torch.equal(fused[:, :, 0], keep[:, :, 0]) and torch.equal(fused[:, :, 2], keep[:, :, 2])
    odd = torch.zeros(2 * 50 * 3 * 64 + 1, device=dev, dtype=BF)
    view = odd[1:].view(2, 50, 3, 64)
    view.copy_(x)
    _close(ops.rope(view, d, plan), ref, tol, "odd offset")
    wide = torch.zeros(2, 50, 3, 67, device=dev, dtype=BF)
    wide[..., :64] = x.to(dev)
    _close(ops.rope(wide[..., :64], d, plan), ref, tol, "odd strides")
    y = torch.randn(2, 50, 3, 64, generator=g)
    back = ops.rope(ops.rope(y.to(dev), d, plan), -d, plan)
    _close(back, y.double(), y.abs().double() * 2.0 ** -20 + 2.0 ** -20, "undone")


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk,D,R,inter", [
    (1, 1, 1, 1, 128, 128, False), (2, 33, 32, 8, 128, 128, False), (1, 700, 24, 24, 128, 128, True),
    (3, 5, 6, 2, 80, 32, False), (2, 9, 3, 1, 96, 24, True), (2, 11, 4, 2, 256, 128, False),
    (1, 7, 5, 5, 66, 20, False), (2, 40, 16, 4, 64, 64, True), (1, 3, 130, 2, 128, 64, False)])
def test_norm_rope(dev, dtype, across, B, L, Hq, Hk, D, R, inter):
    from cast_amd import ops
    print("norm_rope", dtype, across, B, L, Hq, Hk, D, R, inter, flush=True)
    plan, freq, axis = _plan(dev, R, inter)
    g = torch.Generator().manual_seed(L + D)
    q = (torch.randn(B, L, Hq, D, generator=g) * 3).to(dtype)
    k = (torch.randn(B, L, Hk, D, generator=g) * 0.2).to(dtype)
    wq = (1 + 0.2 * torch.randn(*((Hq, D) if across else (D,)), generator=g)).to(dtype)
    wk = (1 + 0.2 * torch.randn(*((Hk, D) if across else (D,)), generator=g)).to(dtype)
    pos = torch.randint(0, 9000, (B, L), generator=g)
    qo, ko = ops.norm_rope(q.to(dev), k.to(dev), pos.to(dev), plan, q_weight=wq.to(dev),
                           k_weight=wk.to(dev), across_heads=across)
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        ref, size = so.rope(so.norm(x, w, 1e-6, across), pos, freq, axis, inter)
        _close(got, ref, so.rope_bound(ref, size, dtype, norm=True), "norm_rope")


def test_norm_rope_weights_and_zero_rows(dev):
    """No weight, one per head without the joint norm, fp32 weights beside bf16 rows; a
    row of zeros stays zero and a row of NaN stays its own."""
    from cast_amd import ops
    plan, freq, axis = _plan(dev, 128)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(2, 6, 4, 128, generator=g).to(BF)
    k = torch.randn(2, 6, 2, 128, generator=g).to(BF)
    q[0, 2] = 0
    q[1, 3, 1] = float("nan")
    w = torch.randn(4, 128, generator=g)
    pos = torch.arange(6)
    qo, ko = ops.norm_rope(q.to(dev), k.to(dev), pos.to(dev), plan, q_weight=w.to(dev), eps=1e-5)
    ref, size = so.rope(so.norm(q, w, 1e-5, False), pos, freq, axis, False)
    assert torch.isnan(qo[1, 3, 1]).all() and torch.isnan(ref[1, 3, 1]).all()
    qo, ref, size = qo.cpu().nan_to_num(0.0), ref.nan_to_num(0.0), size.nan_to_num(0.0)
    _close(qo, ref, so.rope_bound(ref, size, BF, norm=True), "head weights")
    assert (qo[0, 2] == 0).all()
    ref, size = so.rope(so.norm(k, None, 1e-5, False), pos, freq, axis, False)
    _close(ko, ref, so.rope_bound(ref, size, BF, norm=True), "no weight")


@pytest.mark.parametrize("D,R,page", [(128, 128, 16), (64, 20, 48), (80, 32, 7)])
def test_norm_rope_into_pages(dev, D, R, page):
    """Keys and values reach their pages, tokens past a request's length, pages that are
    not there and rows past the table are dropped, every other row stays as it was."""
    from cast_amd import ops
    B, L, Hq, Hk, M, N = 3, 40, 4, 2, 6, 25
    plan, freq, axis = _plan(dev, R)
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(B, L, h, D, generator=g).to(BF) for h in (Hq, Hk, Hk))
    table = torch.randperm(N, generator=g)[:B * M].view(B, M).int()
    table[1, 1], table[1, 2] = -1, N + 5
    starts = torch.tensor([0, 3, M * page - 17], dtype=torch.int32)
    lengths = torch.tensor([L, L - 5, 0 if page == 48 else L], dtype=torch.int32)
    kp, vp = (torch.randn(N, page, Hk, D, generator=g).to(BF) for _ in range(2))
    pos = starts[:, None] + torch.arange(L, dtype=torch.int32)
    kd, vd = kp.to(dev), vp.to(dev)
    cache = ops.PagedCache(kd, vd, table.to(dev))
    q_out = torch.full((B, L, Hq, D), 5.0, device=dev, dtype=BF)
    qo, ko = ops.norm_rope(q.to(dev), k.to(dev), pos.to(dev), plan, v=v.to(dev), cache=cache,
                           starts=starts.to(dev), lengths=lengths.to(dev), q_out=q_out)
    assert ko is None and qo.data_ptr() == q_out.data_ptr()
    kr, ks = so.rope(so.norm(k, None, 1e-6, False), pos, freq, axis, False)
    qr, qs = so.rope(so.norm(q, None, 1e-6, False), pos, freq, axis, False)
    kref, vref, ktol = kp.double(), vp.clone(), torch.zeros(N, page, Hk, D, dtype=torch.float64)
    bound = so.rope_bound(kr, ks, BF, norm=True)
    for b in range(B):
        for t in range(int(lengths[b])):
            at = int(starts[b]) + t
            if at < M * page and 0 <= table[b, at // page] < N:
                row = int(table[b, at // page]), at % page
                kref[row], vref[row], ktol[row] = kr[b, t], v[b, t], bound[b, t]
    _close(kd, kref, ktol, "keys")
    assert torch.equal(vd.cpu(), vref)
    live = torch.arange(L)[None] < lengths[:, None]
    _close(qo.cpu()[live], qr[live], so.rope_bound(qr, qs, BF, norm=True)[live], "queries")
    assert (qo.cpu()[~live] == 5.0).all()


def test_rope_other_stream_and_graph(dev):
    """A call on a side stream, and replays of a captured call over new inputs, give the
    eager result bit for bit."""
    from cast_amd import ops
    plan, _, _ = _plan(dev, 64)
    x = torch.randn(2, 100, 4, 64, device=dev).to(BF)
    k = torch.randn(2, 100, 2, 64, device=dev).to(BF)
    pos = torch.arange(100, device=dev)
    want = ops.rope(x, pos, plan), *ops.norm_rope(x, k, pos, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rope(x, pos, plan), *ops.norm_rope(x, k, pos, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rope(x, pos, plan), *ops.norm_rope(x, k, pos, plan)
    for i in range(3):
        x.copy_(torch.randn(x.shape, device=dev))
        pos += 7
        want = ops.rope(x, pos, plan), *ops.norm_rope(x, k, pos, plan)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_empty_and_refused(dev):
    from cast_amd import ops
    plan, _, _ = _plan(dev, 64)
    assert ops.rope(torch.empty(2, 0, 4, 64, device=dev), torch.empty(0, device=dev).int(),
                    plan).shape == (2, 0, 4, 64)
    x = torch.randn(2, 5, 4, 64, device=dev)
    pos = torch.arange(5, device=dev)
    with pytest.raises(RuntimeError, match="positions"):
        ops.rope(x, torch.arange(6, device=dev), plan)
    with pytest.raises(RuntimeError, match="positions"):
        ops.rope(x, pos.float(), plan)
    with pytest.raises(ValueError, match="turns 64 channels"):
        ops.rope(x[..., :32], pos, plan)
    with pytest.raises(TypeError):
        ops.rope(x.double(), pos, plan)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.rope(x.clone().requires_grad_(), pos, plan)
    with pytest.raises(RuntimeError, match="expanded"):
        ops.rope(x, pos, plan, out=torch.empty(1, 5, 4, 64, device=dev).expand(2, 5, 4, 64))
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.rope(x, pos.cpu(), plan)
    with pytest.raises(ValueError, match="together"):
        ops.norm_rope(x, x, pos, plan, v=x)
    with pytest.raises(RuntimeError, match="weight"):
        ops.norm_rope(x, x, pos, plan, q_weight=torch.ones(32, device=dev))
    with pytest.raises(RuntimeError, match="q and k differ"):
        ops.norm_rope(x, x[:, :4], pos, plan)
