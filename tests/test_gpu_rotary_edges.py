"""``ops.rope`` and ``ops.norm_rope`` at the edges of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


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
