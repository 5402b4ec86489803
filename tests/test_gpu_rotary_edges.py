"""``ops.rope`` and ``ops.norm_rope`` at the edges of what they take."""
import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _close(got, ref, tol, what):
    worst = ((got.double() - ref).abs() - tol).max().item()
    assert worst <= 0.0, f"{what}: {worst} past the bound"


@pytest.mark.parametrize("shape", [(0,), (4, 0)])
def test_weights_of_no_channels(dev, shape):
    """Heads of 0 channels give empty results, with weights as without."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    plan = rotary_plan(0, device=dev)
    x = torch.empty(2, 3, 4, 0, device=dev, dtype=BF)
    w = torch.empty(shape, device=dev, dtype=BF)
    pos = torch.arange(3, device=dev)
    q, k = ops.norm_rope(x, x, pos, plan, q_weight=w, k_weight=w)
    assert q.shape == k.shape == x.shape
    with pytest.raises(RuntimeError, match="weight"):
        ops.norm_rope(x, x, pos, plan, q_weight=torch.ones(3, device=dev, dtype=BF))


@pytest.mark.parametrize("D,H,L", [
    (3, 1, (1 << 26) + 77),   # element by element, a workgroup a token, past 2^32 threads
    (128, 80, 65537 + 9),     # 16-byte runs, a workgroup a token, past one row of the grid
    (6, 3, 65537 * 16 + 5)])  # runs of two
def test_grids_of_many_tokens(dev, D, H, L):
    """Every token is turned, wherever its workgroup lies in the grid."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    print("many tokens", D, H, L, flush=True)
    R = D // 2 * 2
    plan, (freq, axis) = rotary_plan(R, device=dev), so.frequencies(R)
    x = torch.empty(1, L, H, D, device=dev, dtype=BF)
    for i in range(0, L, 1 << 22):  # (pieces: the random numbers are fp32)
        x[:, i:i + (1 << 22)] = torch.randn(x[:, i:i + (1 << 22)].shape, device=dev)
    pos = torch.arange(L, device=dev, dtype=torch.int32)
    out = torch.full_like(x, float("nan"))
    assert ops.rope(x, pos, plan, out=out).data_ptr() == out.data_ptr()
    assert not torch.isnan(out).any()
    for i in sorted({0, 65500 % L, (1 << 16) % L, L // 2, max(0, (1 << 26) - 50) % L, L - 100}):
        s = slice(i, i + 100)
        ref, size = so.rope(x[:, s], pos[s], freq, axis, False)
        _close(out[:, s], ref, so.rope_bound(ref, size, BF), i)


@pytest.mark.parametrize("D,Hq,Hk", [(128, 12, 6), (5, 2, 1)])
def test_norms_of_many_tokens(dev, D, Hq, Hk):
    """Norms, keys and values of more tokens than a row of the grid holds: pages filled to
    the last token."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    L, page = 65537 + 20, 64
    R, M = D // 2 * 2, -(-(65537 + 20) // 64)
    plan, (freq, axis) = rotary_plan(R, device=dev), so.frequencies(R)
    q, k, v = (torch.randn(1, L, h, D, device=dev).to(BF) for h in (Hq, Hk, Hk))
    kp, vp = (torch.full((M, page, Hk, D), float("nan"), device=dev, dtype=BF) for _ in range(2))
    table = torch.arange(M, dtype=torch.int32, device=dev)[None].contiguous()
    pos = torch.arange(L, device=dev)
    qo, _ = ops.norm_rope(q, k, pos, plan, v=v, cache=ops.PagedCache(kp, vp, table))
    assert torch.equal(vp.view(-1, Hk, D)[:L], v[0])
    for got, x in ((qo, q), (kp.view(1, -1, Hk, D)[:, :L], k)):
        ref, size = so.rope(so.norm(x, None, 1e-6, False), pos, freq, axis, False)
        _close(got, ref, so.rope_bound(ref, size, BF, norm=True), (D, x.shape[2]))


def test_forward_mode_gradients_are_refused(dev):
    """A dual tensor's tangent is not dropped silently, with or without no_grad."""
    from torch.autograd import forward_ad
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    plan = rotary_plan(64, device=dev)
    x = torch.randn(2, 16, 4, 64, device=dev).to(BF)
    pos = torch.arange(16, device=dev)
    pages = torch.zeros(4, 16, 4, 64, device=dev, dtype=BF)
    table = torch.zeros(2, 1, device=dev, dtype=torch.int32)
    lens = torch.ones(2, device=dev, dtype=torch.int32)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.rope(d, pos, plan), lambda: ops.rope(x, pos, plan, out=d),
                     lambda: ops.norm_rope(d, x, pos, plan), lambda: ops.norm_rope(x, d, pos, plan),
                     lambda: ops.norm_rope(x, x, pos, plan, q_weight=d[0, 0]),
                     lambda: ops.window_attention(d, x, x), lambda: ops.window_attention(x, x, d),
                     lambda: ops.paged_attention(d, ops.PagedCache(pages, pages, table), lens)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        y = forward_ad.unpack_dual(d).primal
        assert torch.equal(ops.rope(y, pos, plan), ops.rope(x, pos, plan))


def test_outputs_that_overlap_are_refused(dev):
    """An output may be its own input, or a part of a fused projection beside it; shifted,
    turned or another operand's memory is refused before anything is written."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    plan = rotary_plan(64, device=dev)
    pos = torch.arange(16, device=dev)
    store = torch.randn(2 * 17 * 4 * 64, device=dev).to(BF)
    x, shifted = store[:8192].view(2, 16, 4, 64), store[64:8256].view(2, 16, 4, 64)
    k, v = torch.randn(2, 2, 16, 4, 64, device=dev).to(BF)
    pages = torch.randn(2, 16, 4, 64, device=dev).to(BF)
    table = torch.arange(2, device=dev, dtype=torch.int32)[:, None].contiguous()
    lens = torch.full((2,), 16, device=dev, dtype=torch.int32)
    cache = ops.PagedCache(pages, pages.clone(), table)
    was = store.clone(), k.clone(), v.clone(), pages.clone()
    for call in (lambda: ops.rope(x, pos, plan, out=shifted),
                 lambda: ops.rope(x[:, :4], pos[:4], plan, out=x[:, :4].transpose(1, 2)),
                 lambda: ops.norm_rope(x, k, pos, plan, q_out=shifted),
                 lambda: ops.norm_rope(x, k, pos, plan, q_out=k),
                 lambda: ops.norm_rope(x, k, pos, plan, k_out=x),
                 lambda: ops.norm_rope(x, k, pos, plan, q_out=v, k_out=v),
                 lambda: ops.norm_rope(x, k, pos, plan, v=v, cache=cache, q_out=v),
                 lambda: ops.norm_rope(x, k, pos, plan, v=v, cache=cache, q_out=pages),
                 lambda: ops.norm_rope(x, k, pos, plan, v=v, cache=cache._replace(v=pages)),
                 lambda: ops.norm_rope(pages, k, pos, plan, v=v, cache=cache),
                 lambda: ops.window_attention(x, k, v, out=x),
                 lambda: ops.window_attention(x, k, v, out=shifted),
                 lambda: ops.window_attention(x, k, v, out=k),
                 lambda: ops.window_attention(x, k, v, out=v),
                 lambda: ops.window_attention(x[:, 3:5], k, v, out=k[:, 3:5]),
                 lambda: ops.paged_attention(x, cache, lens, out=pages)):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert all(torch.equal(a, b) for a, b in zip((store, k, v, pages), was))
    fused = torch.randn(2, 16, 4, 4, 64, device=dev).to(BF)
    q, k, v, o = fused.unbind(2)
    want = ops.window_attention(*(t.contiguous() for t in (q, k, v)))
    assert torch.equal(ops.window_attention(q, k, v, out=o), want)
    want = ops.norm_rope(q.contiguous(), k.contiguous(), pos, plan)
    assert ops.norm_rope(q, k, pos, plan, q_out=q, k_out=k)[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_weight_shapes(dev):
    """[D], [H, D] and the flat [H * D] of a projection's norm; a turned or split shape of as
    many elements is refused."""
    from cast_amd import ops
    from cast_amd.rotary import rotary_plan
    H, D = 4, 64
    plan = rotary_plan(D, device=dev)
    pos = torch.arange(5, device=dev)
    x = torch.randn(2, 5, H, D, device=dev).to(BF)
    w = torch.randn(H, D, device=dev).to(BF)
    for across in (False, True):
        kw = dict(across_heads=across)
        want = ops.norm_rope(x, x, pos, plan, q_weight=w, k_weight=w, **kw)
        for shape in ((H * D,), (1, 1, H, D), (2, H // 2, D)):
            got = ops.norm_rope(x, x, pos, plan, q_weight=w.view(shape), k_weight=w.view(shape),
                                **kw)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), shape
        one = ops.norm_rope(x, x, pos, plan, q_weight=w[0], **kw)[0]
        assert torch.equal(ops.norm_rope(x, x, pos, plan, q_weight=w[:1], **kw)[0], one)
        for shape in ((D, H), (H, D, 1), (2 * H, D // 2), (8, 8), (D, 1)):
            n = shape[0] * shape[1] * (shape[2] if len(shape) > 2 else 1)
            with pytest.raises(RuntimeError, match="weight"):
                ops.norm_rope(x, x, pos, plan, q_weight=w.view(-1)[:n].view(shape), **kw)
