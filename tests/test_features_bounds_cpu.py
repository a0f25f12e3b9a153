"""What the bounds of features_bounds.py admit, without a GPU."""
import numpy as np
import pytest
import torch

import features_bounds as bounds
import features_ref as ref


@pytest.mark.parametrize("shape", [(1, (600, 500), 12, 3), (2, (300, 100), 64, 8)])
def test_bounds_refuse_statistics_without_a_pivot(shape):
    """Sums of the values and of their squares, even where they are added in pairs, lose the spread beside a mean of 2000."""
    n, sp, c, g = shape
    x = 2000.0 + bounds.normal((n, *sp, c), 40)
    r = bounds.GroupNorm(x, None, None, g, pivot=True)
    _, (mean, t_mean), (rstd, t_rstd) = r.forward()
    xg = x.reshape(n, -1, g, c // g).transpose(1, 2).reshape(n, g, -1).numpy()
    m = np.stack([[np.sum(q, dtype=np.float32) / np.float32(q.size) for q in s] for s in xg])
    sq = np.stack([[np.sum(q * q, dtype=np.float32) / np.float32(q.size) for q in s] for s in xg])
    naive = 1 / np.sqrt(np.maximum(sq - m * m, 0).astype(np.float64) + 1e-5)
    # (squares near 4e6 come in steps of 1/4, so that a group's variance may still land on 1)
    assert (np.abs(naive - rstd.numpy()) > t_rstd.numpy()).any()
    # a mean that is off by a thousandth of the spread is refused too, and so is a spread
    assert (t_mean < 2e-3).all() and (t_rstd < 5e-3 * rstd).all()


def test_bounds_refuse_gates_that_stop():
    """A gate held at 2^-60 leaves z 2^-60 of a channel that is off."""
    b = torch.tensor([-1e6, -1e9, float(torch.finfo(torch.float32).min), 0.0])
    x = bounds.normal((2, 30, 4), 3)
    for act in ("silu", "gelu_tanh"):
        r = bounds.GroupNorm(x, None, b, 4, act=act)
        (y, t), _, _ = r.forward()
        (v_x, tv), _, (v_b, tb) = r.backward(torch.ones_like(x))
        for k in range(3):
            assert (y[..., k] == 0).all() and (t[..., k] < abs(float(b[k])) * 2.0**-62).all()
            assert v_b[k] == 0 and tb[k] < 1e-30 and (tv[..., k] < 1e-30).all()


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
def test_bounds_share_the_definition(act):
    """The values are those of features_ref.py, which differences check."""
    x, v = bounds.normal((2, 9, 12), 1), bounds.normal((2, 9, 12), 2)
    w, b = bounds.normal((12,), 3), bounds.normal((12,), 4)
    drop = (ref.mask(x.numel(), 0.3, 3, 1), 0.3)
    one, two = (k.GroupNorm(x, w, b, 3, act=act, drop=drop) for k in (ref, bounds))
    for (y, _), (z, _) in zip(one.forward() + one.backward(v), two.forward() + two.backward(v)):
        assert (y - z).abs().max() <= 1e-13
