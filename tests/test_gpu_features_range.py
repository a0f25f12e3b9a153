"""Group norm's activations far from zero, on the GPU against the 64-bit restatement."""
import pytest
import torch

import features_bounds as bounds
import features_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
LOWEST = float(torch.finfo(torch.float32).min)
# channels switched off by their biases, far on, and at the ends of the exponential's range, beside ordinary ones
BIASES = [0.0, -1e6, -45.0, LOWEST, 0.5, -1e9, -88.0, 1e6, -62.0, 1e13, -1e13, 30.0, -7.3, 1e30, -104.0, -12.0, -65504.0]


def _normal(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _far_inputs(n, sp, c, dtype, ptype):
    x, v = _normal((n, *sp, c), 1, dtype), _normal((n, *sp, c), 2, dtype)
    limits = torch.finfo(ptype)
    b = torch.tensor([BIASES[k % len(BIASES)] for k in range(c)], dtype=torch.float64)
    b = b.clamp(float(limits.min), float(limits.max) if dtype != torch.float16 else 3e4).to(ptype)  # f16 results stay finite
    return x, (1 + 0.2 * _normal(c, 3)).to(ptype), b, v


# vectors and single elements in registers, vectors, pairs and odd samples in rings; a channel a group and several
@pytest.mark.parametrize("n,sp,c,g", [(2, (9, 7), 64, 16), (2, (13, 7), 51, 51), (1, (300, 200), 64, 64),
                                      (1, (60_001,), 34, 17), (2, (40_001,), 37, 37)],
                         ids=["small", "single", "large", "pairs", "odd"])
@pytest.mark.parametrize("dtype,same", [(torch.float32, True), (torch.bfloat16, False), (torch.bfloat16, True),
                                        (torch.float16, False), (torch.float16, True)], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_group_norm_far_activations(cuda, n, sp, c, g, dtype, same, act):
    """Biases down to the type's lowest value: the activation and its slope go to 0 (above, to z and 1) with
    the digits that 32 bits have, and nothing of a channel that is off reaches its group."""
    import brush_b200 as bsx

    x, w, b, v = _far_inputs(n, sp, c, dtype, dtype if same else torch.float32)
    r = bounds.GroupNorm(x, w, b, g, act=act)
    cfg = bsx.GroupNormConfig(groups=g, activation=act)
    d = [t.cuda() for t in (x, w, b, v)]
    out, mean, rstd = bsx.group_norm_forward(*d[:3], cfg)
    ref.close(out, r.forward()[0])
    grads = bsx.group_norm_backward(d[3], *d[:3], r.mean.float().cuda(), r.rstd.float().cuda(), cfg)
    for got, want in zip(grads, r.backward(v)):
        ref.close(got, want)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_channel_off_leaves_the_others(cuda, act, dtype):
    """A group's channels beside one that is off have the gradients that they have where its gradient is 0."""
    import brush_b200 as bsx

    x, v = _normal((2, 20, 21, 16), 5, dtype).cuda(), _normal((2, 20, 21, 16), 6, dtype).cuda()
    w = torch.ones(16, device="cuda")
    cfg = bsx.GroupNormConfig(groups=2, activation=act)
    zero = v.clone()
    zero[..., 3] = 0
    for off in (-1e6, -1e9, LOWEST):
        b = torch.zeros(16, device="cuda")
        b[3] = off
        out, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
        assert (out[..., 3] == 0).all()
        got = bsx.group_norm_backward(v, x, w, b, mean, rstd, cfg)
        want = bsx.group_norm_backward(zero, x, w, b, mean, rstd, cfg)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
@pytest.mark.parametrize("n,sp,c,g", [(2, (9, 7), 64, 16), (1, (200, 150), 64, 16), (2, (40_001,), 37, 37), (3, (13, 7), 21, 7)],
                         ids=["small", "large", "odd", "single"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_group_norm_nan_parameters_stay_in_their_channels(cuda, act, n, sp, c, g, dtype):
    """Lanes share reciprocals: a NaN among the weights or biases reaches its own channel, and the gradients of its group."""
    import brush_b200 as bsx

    x, v = _normal((n, *sp, c), 7, dtype).cuda(), _normal((n, *sp, c), 8, dtype).cuda()
    per, cfg = c // g, bsx.GroupNormConfig(groups=g, activation=act)
    for which in (0, 1):
        params = [torch.ones(c), torch.zeros(c)]
        params[which][5] = float("nan")
        w, b = (t.cuda() for t in params)
        out, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
        v_x, v_w, v_b = bsx.group_norm_backward(v, x, w, b, mean, rstd, cfg)
        channel = torch.arange(c, device="cuda") == 5
        group = torch.arange(c, device="cuda") // per == 5 // per
        assert mean.isfinite().all() and rstd.isfinite().all()
        assert torch.equal(out.isnan(), channel.expand_as(out)) and out[..., ~channel].isfinite().all()
        if act == "none" and which == 1:  # the bias has no part in the gradients
            assert all(t.isfinite().all() for t in (v_x, v_w, v_b))
            continue
        assert torch.equal(v_x.isnan(), group.expand_as(v_x)) and v_x[..., ~group].isfinite().all()
        if act == "none":  # nor has the weight in its own
            assert v_w.isfinite().all() and v_b.isfinite().all()
        else:
            assert torch.equal(v_w.isnan(), channel) and torch.equal(v_b.isnan(), channel)
