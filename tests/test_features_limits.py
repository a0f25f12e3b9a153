"""Sizes beyond what the group-norm entry points take, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("shape", [(1, (1 << 32) + 8), (1, 1, (1 << 32) + 32), (1, 1 << 32), (1 << 28, 8), (1 << 31, 1, 1)], ids=str)
def test_group_norm_refuses_too_many_channels(bsx_lib, shape):
    """Channel counts are 32-bit in the C interface: a larger one is refused, not cut to its low half."""
    import brush_b200 as bsx
    from brush_b200.norm import _call

    x = torch.zeros(()).expand(shape)
    with pytest.raises((ValueError, bsx.BsxError)):
        _call(x, None, None, bsx.GroupNormConfig(groups=8 if shape[-1] % 8 == 0 else 1))


@pytest.mark.parametrize("groups", [(1 << 32) + 1, 1 << 32])
def test_group_norm_refuses_groups_beyond_32_bits(bsx_lib, groups):
    import brush_b200 as bsx
    from brush_b200.norm import _call

    with pytest.raises((ValueError, bsx.BsxError)):
        _call(torch.zeros(()).expand(1, groups), None, None, bsx.GroupNormConfig(groups=groups))
