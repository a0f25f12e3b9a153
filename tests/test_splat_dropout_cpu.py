"""Splat dropout without a GPU: what is refused, whatever the exchange."""
import math

import pytest
import torch


@pytest.mark.parametrize("p", [1.0, 1.5, -0.1, math.nan, math.inf])
@pytest.mark.parametrize("exchange", ["auto", "peer", "nvls", "nccl"])
def test_every_exchange_refuses_the_same_probabilities(bsx_lib, exchange, p):
    import brush_b200 as bsx

    with pytest.raises(bsx.BsxError, match="splat dropout"):
        bsx.SplatTrainer(bsx.TrainConfig(splat_dropout=p), None, exchange=exchange)


def test_step_opacities(bsx_lib):
    import brush_b200 as bsx
    from brush_b200.train import step_opacities

    logits = torch.randn(5)
    assert step_opacities(logits, bsx.TrainConfig(), 3) is logits  # off by default
    for p in (1.0, -0.1, math.nan):
        with pytest.raises(bsx.BsxError):
            step_opacities(logits, bsx.TrainConfig(splat_dropout=p), 1)
