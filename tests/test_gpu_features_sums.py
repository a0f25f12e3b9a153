"""Long sums of the group-norm kernels, against bounds that follow the kernels' own chains."""
import pytest
import torch

import features_bounds as bounds
import features_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
LARGE = [(1, (600, 500), 12, 3), (2, (512, 300), 64, 8), (2, (100_001,), 37, 1), (1, (700,), 8192, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", LARGE, ids=lambda s: f"{s[0]}x{'x'.join(map(str, s[1]))}x{s[2]}g{s[3]}")
@pytest.mark.parametrize("offset", [0.0, 200.0, 2000.0])
def test_statistics_of_large_samples(cuda, shape, dtype, offset):
    """Means and spreads of values around a mean far above their spread: within some hundred half steps of the spread."""
    import brush_b200 as bsx

    n, sp, c, g = shape
    x = (offset + bounds.normal((n, *sp, c), 40)).to(dtype)
    w, b = 1 + 0.2 * bounds.normal((c,), 41), 0.3 * bounds.normal((c,), 42)
    r = bounds.GroupNorm(x, w, b, g, act="silu", pivot=True)
    out, mean, rstd = bsx.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), bsx.GroupNormConfig(groups=g, activation="silu"))
    for got, want in zip((out, mean, rstd), r.forward()):
        ref.close(got, want)


@pytest.mark.parametrize("shape", LARGE, ids=lambda s: f"{s[0]}x{'x'.join(map(str, s[1]))}x{s[2]}g{s[3]}")
@pytest.mark.parametrize("dtype,act,p", [(torch.float32, "none", 0.0), (torch.bfloat16, "silu", 0.2),
                                         (torch.float16, "gelu_tanh", 0.0)], ids=str)
def test_gradients_of_large_samples(cuda, shape, dtype, act, p):
    """Gradients about a value above their spread."""
    import brush_b200 as bsx

    n, sp, c, g = shape
    x, v = bounds.normal((n, *sp, c), 50, dtype), (0.9 + 0.1 * bounds.normal((n, *sp, c), 51)).to(dtype)
    w, b = 1 + 0.2 * bounds.normal((c,), 52), 0.3 * bounds.normal((c,), 53)
    drop = bsx.DropoutConfig(p=p, seed=31, step=2) if p else None
    r = bounds.GroupNorm(x, w, b, g, act=act, drop=(ref.mask(x.numel(), p, 31, 2), p) if p else None, pivot=True)
    got = bsx.group_norm_backward(v.cuda(), x.cuda(), w.cuda(), b.cuda(), r.mean.float().cuda(), r.rstd.float().cuda(),
                                  bsx.GroupNormConfig(groups=g, activation=act, dropout=drop))
    for a, want in zip(got, r.backward(v)):
        ref.close(a, want)


# Where every gradient is the same number, each addition of a running sum rounds the same way until the sum doubles: a
# chain of k additions is off by k / 6 half steps (k = 7085 of 0.9: by 1100). Sums of sums of at most 64 rows are off
# by at most 64 + rows / 64 half steps, and what joins them by 64 (a block's copies of a channel: 8 + 4 additions with 8
# threads a channel, blocks: 5 of a lane and 5 shuffles).


def _same_gradient(n, pixels, c, groups):
    import brush_b200 as bsx

    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn((n, pixels, c), generator=gen, device="cuda")
    v = torch.full_like(x, 0.9)
    mean = torch.zeros(n, groups, device="cuda")
    ones = torch.ones(c, device="cuda")
    v_x, v_w, v_b = bsx.group_norm_backward(v, x, ones, ones, mean, mean + 1, bsx.GroupNormConfig(groups=groups))
    del v
    one = float(torch.tensor(0.9))
    want = one * n * pixels
    return x, v_x, v_w, v_b, one, want


def test_gradient_sums_of_a_long_sample(cuda):
    """7085 rows a block: bias gradients are a count times the gradient, and v_x is what the definition leaves of it."""
    px, c, g, rows = 32 * 148 * 7085, 64, 16, 7085
    x, v_x, v_w, v_b, one, want = _same_gradient(1, px, c, g)
    chain = (64 + rows / 64 + 64) * ref.U
    assert ((v_b.double() - want).abs() <= chain * want).all()
    per_channel = torch.stack([x[0, :, k].double().sum() for k in range(c)])
    size = torch.stack([x[0, :, k].double().abs().sum() for k in range(c)])
    assert ((v_w.double() - one * per_channel).abs() <= (chain + 3 * ref.U) * one * size).all()
    # mean 0 and rstd 1 are given: v_x = 0.9 - s1 - x s2 with s1 = 0.9 up to its sum's bound, s2 = 0.9 mean(x)
    s2 = one * per_channel.reshape(g, -1).mean(1).repeat_interleave(c // g) / px
    t2 = (chain + 8 * ref.U) * one * size.reshape(g, -1).mean(1).repeat_interleave(c // g) / px
    part = x[0, :: px // 1000]
    off = (v_x[0, :: px // 1000].double() + part.double() * s2).abs()
    assert (off <= (chain + 8 * ref.U) * one + part.double().abs() * (t2 + 2 * ref.U * s2.abs())).all()
    del x, v_x
    torch.cuda.empty_cache()


def test_gradient_sums_of_many_samples(cuda):
    """Samples of one pixel, some ten thousand a block."""
    n, c = 1 << 22, 64
    x, v_x, v_w, v_b, one, want = _same_gradient(n, 1, c, 8)
    rows = n / 148  # a block an SM at least
    chain = (64 + rows / 64 + 64) * ref.U
    assert ((v_b.double() - want).abs() <= chain * want).all()
    per_channel, size = x.double().sum((0, 1)), x.double().abs().sum((0, 1))
    assert ((v_w.double() - one * per_channel).abs() <= (chain + 3 * ref.U) * one * size).all()
    del x, v_x
    torch.cuda.empty_cache()
