"""``ops.packed_attention`` of many requests: every row of every request against the 64-bit
oracle, in outputs that hold NaN before the call, so that a row which no workgroup takes
fails.

Tolerances: the oracle's bound (see ``streaming_oracle.attention``)."""
import pytest
import torch

from oracle import streaming_oracle as so

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("B", [64, 65, 512, 513, 2100])
@pytest.mark.parametrize("window", [0, 20])
def test_every_row(dev, B, window):
    """Both orders of the row blocks, requests past a search's 64 and past those that are
    ranked; two fill several blocks, some have no rows."""
    from cast_amd import ops
    Hq, Hk, D = 4, 2, 64
    count = [(29 * b) % 37 if b % 5 else 0 for b in range(B)]
    count[B // 3], count[B - 2] = 300, 129
    before = [(7 * b) % 50 if b % 3 == 0 else 0 for b in range(B)]
    q_at, k_at = [0], [0]
    for n, m in zip(count, before):
        q_at.append(q_at[-1] + n)
        k_at.append(k_at[-1] + n + m)
    g = torch.Generator().manual_seed(B)
    q, k, v = (torch.randn(n, h, D, generator=g).to(BF).to(dev)
               for n, h in ((q_at[-1], Hq), (k_at[-1], Hk), (k_at[-1], Hk)))
    offs = [torch.tensor(t, dtype=torch.int32, device=dev) for t in (q_at, k_at)]
    out = torch.full_like(q, float("nan"))
    got, lse = ops.packed_attention(q, k, v, offs[0], k_offsets=offs[1], window=window or None,
                                    return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert not torch.isnan(out).any(), torch.isnan(out).any(2).any(1).nonzero()[:8, 0].tolist()
    worst = []
    for b in range(B):
        rows, keys = slice(q_at[b], q_at[b + 1]), slice(k_at[b], k_at[b + 1])
        if count[b] == 0:
            continue
        seen = so.visible(count[b], count[b] + before[b], window, 0, 1, device=dev)
        ref, rlse, tol, ltol = so.attention(q[rows], k[keys], v[keys], seen, D ** -0.5, BF)
        worst.append(torch.stack([((out[rows].double() - ref).abs() - tol).max(),
                                  ((lse[:, rows].double() - rlse).abs() - ltol).max()]))
    worst = torch.stack(worst).max(0).values.tolist()
    assert max(worst) <= 0.0, worst
