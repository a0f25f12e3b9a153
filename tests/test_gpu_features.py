"""Dropout and group norm on the GPU against the 64-bit restatements (features_ref.py)."""
import threading

import pytest
import torch

import features_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _normal(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- dropout ----


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count,share", [(1, 1), (7, 1), (8, 1), (9, 1), (255, 1), (4096, 1), (100_003, 1),
                                         (100_003, 2), (99_999, 3), (40_001, 7), (4096, 8), (4104, 24), (48_000, 48),
                                         (4800, 100), (1000, 1000), (37 * 211, 37), (5, 1 << 40), (66_000, 6600)])
def test_dropout_equals_restatement(cuda, dtype, count, share):
    """Equal bit for bit: the kernel's product, sum and rounding are single IEEE operations."""
    import brush_b200 as bsx

    x, r = _normal(count, 1, dtype), _normal(count, 2, dtype)
    for p, seed, step in [(0.1, 42, 1), (0.4999, (1 << 64) - 5, (1 << 32) - 1)]:
        cfg = bsx.DropoutConfig(p=p, seed=seed, step=step, share=share)
        s = min(share, count)  # the restatement repeats each draw `share` times
        want = ref.dropout(x, p, seed, step, s)
        assert torch.equal(bsx.dropout_forward(x.cuda(), cfg).cpu(), want)
        assert torch.equal(bsx.dropout_backward(x.cuda(), cfg).cpu(), want)
        got = bsx.dropout_forward(x.cuda(), cfg, residual=r.cuda()).cpu()
        assert torch.equal(got, ref.dropout(x, p, seed, step, s, residual=r))


def test_dropout_ties_take_the_low_halfword(cuda):
    """Draws whose high halfword equals the threshold's (one in 65536) are decided by the low one."""
    import brush_b200 as bsx

    n, p = 1 << 21, 0.3 + 2.0**-18
    d = ref.draws(0, n, 5, 6)
    t = round(p * 2**32)
    tied = (d >> 16) == (t >> 16)
    assert 8 < tied.sum() < 100 and 0 < (d[tied] >= t).sum() < tied.sum()
    y = bsx.dropout_forward(torch.ones(n, device="cuda"), bsx.DropoutConfig(p=p, seed=5, step=6)).cpu()
    assert torch.equal(y != 0, torch.from_numpy(d >= t))


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_all_and_nothing(cuda, dtype):
    import brush_b200 as bsx

    x = _normal(10_001, 3, dtype)
    x[5], x[6], x[7] = float("inf"), float("nan"), -float("inf")
    g = x.cuda()
    assert torch.equal(bsx.dropout_forward(g, bsx.DropoutConfig(p=0.0)).cpu().nan_to_num(7), x.nan_to_num(7))
    assert torch.equal(bsx.dropout_forward(g, bsx.DropoutConfig(p=1.0)).cpu(), torch.zeros_like(x))
    r = _normal(10_001, 4, dtype)
    assert torch.equal(bsx.dropout_forward(g, bsx.DropoutConfig(p=1.0), residual=r.cuda()).cpu(), r)
    # infinities and NaN leave nothing where they are dropped
    bad = torch.full((4096,), float("nan"), dtype=dtype)
    keep = ref.mask(4096, 0.5, 42, 9)
    y = bsx.dropout_backward(bad.cuda(), bsx.DropoutConfig(p=0.5, step=9)).cpu()
    assert (y[~keep] == 0).all() and y[keep].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("share", [1, 5, 16])
def test_dropout_unaligned_and_strided(cuda, dtype, offset, share):
    import brush_b200 as bsx

    base, res = _normal(5000, 5, dtype).cuda(), _normal(5000, 6, dtype).cuda()
    cfg = bsx.DropoutConfig(p=0.25, seed=8, step=2, share=share)
    n = 4000 + offset
    x, r = base[offset:offset + n], res[2 * offset:2 * offset + n]  # the residual's alignment differs
    want = ref.dropout(x.cpu(), 0.25, 8, 2, share, residual=r.cpu())
    assert torch.equal(bsx.dropout_forward(x, cfg, residual=r).cpu(), want)
    t = base[:4992].reshape(96, 52).t()  # strides: the draw goes by the logical order
    assert torch.equal(bsx.dropout_forward(t, cfg).cpu(), ref.dropout(t.cpu().contiguous(), 0.25, 8, 2, share))


def test_dropout_far_elements(cuda):
    """Element and draw numbers beyond 2^31."""
    import brush_b200 as bsx

    n = (1 << 31) + 1003
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    for share in (1, 3):
        y = bsx.dropout_forward(x, bsx.DropoutConfig(p=0.5, seed=3, step=4, share=share))
        for first, count in ((0, 1000), ((1 << 31) - 500, 1000), (n - 1000, 1000)):
            assert torch.equal(y[first:first + count].cpu() != 0, ref.mask(count, 0.5, 3, 4, share, first))
        del y
    del x
    torch.cuda.empty_cache()


def test_dropout_empty(cuda):
    import brush_b200 as bsx

    assert bsx.dropout_forward(torch.empty(0, 4, device="cuda"), bsx.DropoutConfig()).shape == (0, 4)
    assert bsx.dropout_backward(torch.empty(0, device="cuda"), bsx.DropoutConfig()).shape == (0,)


def test_dropout_step_tensor_in_a_graph(cuda):
    """A captured call reads its step when it runs."""
    import brush_b200 as bsx

    x = _normal(4099, 7)
    g, step = x.cuda(), torch.tensor([1], dtype=torch.int32, device="cuda")
    cfg = bsx.DropoutConfig(p=0.2, seed=11, step=step)
    assert torch.equal(bsx.dropout_forward(g, cfg).cpu(), ref.dropout(x, 0.2, 11, 1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = bsx.dropout_forward(g, cfg)
        v = bsx.dropout_backward(y, cfg)
        step.add_(1)
    step.fill_(1)
    for k in (1, 2, 3):
        graph.replay()
        want = ref.dropout(x, 0.2, 11, k)
        assert torch.equal(y.cpu(), want)
        assert torch.equal(v.cpu(), ref.dropout(want, 0.2, 11, k))


def test_dropout_refusals(cuda):
    import brush_b200 as bsx

    x, cfg = torch.zeros(4, 8, device="cuda"), bsx.DropoutConfig()
    for args in [(x.cpu(), cfg), (x.double(), cfg), (x, bsx.DropoutConfig(p=2.0)), (x, cfg, x[:2]), (x, cfg, x.half()),
                 (x, cfg, x.cpu()), (x, bsx.DropoutConfig(step=torch.zeros(1, dtype=torch.int32)))]:
        with pytest.raises(ValueError):
            bsx.dropout_forward(*args)


def test_dropout_entry_point_errors(cuda, bsx_lib):
    import ctypes as C

    from brush_b200._context import context

    ctx, L = context(0), bsx_lib.lib()
    x = torch.zeros(64, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    call = lambda c, n=64, t=0, p=x.data_ptr(): L.bsx_dropout_fwd(ctx.handle, p, None, n, t, C.byref(c), p, s)  # noqa: E731
    assert call(bsx_lib.DropoutCfg(0.5, 1, 1, None, 0)) == 0
    for c, kw in [(bsx_lib.DropoutCfg(1.5, 1, 1, None, 0), {}), (bsx_lib.DropoutCfg(float("nan"), 1, 1, None, 0), {}),
                  (bsx_lib.DropoutCfg(0.5, 1, 0, None, 0), {}), (bsx_lib.DropoutCfg(0.5, 1, 1, None, 0), dict(t=3)),
                  (bsx_lib.DropoutCfg(0.5, 1, 1, None, 0), dict(p=None)),
                  (bsx_lib.DropoutCfg(0.5, 1, 1, None, 0), dict(n=3, p=x.data_ptr() + 2))]:
        assert call(c, **kw) == 1
        assert L.bsx_last_error(ctx.handle)
    assert call(bsx_lib.DropoutCfg(0.5, 1, 1, None, 0), n=(1 << 64) - 1) == 3
    ctx.sync()


# ---- group norm ----

SHAPES = [  # (n, spatial, channels, groups)
    (1, (1,), 1, 1), (1, (1,), 8, 8), (2, (), 6, 2), (1, (3,), 5, 1), (3, (4, 5), 12, 4), (2, (7, 9), 37, 1),
    (2, (7, 9), 37, 37), (1, (16, 16), 32, 8), (4, (33, 17), 64, 16), (2, (64, 64), 256, 32), (2, (31, 29), 90, 6),
    (300, (1,), 512, 32), (70, (2, 3), 40, 5), (1, (128, 129), 24, 3), (1, (5,), 2560, 32), (2, (3, 3), 4100, 2),
    (1, (211, 307), 16, 16), (3, (50, 50), 30, 10), (1, (9,), 10007, 1), (5, (1000,), 2, 2), (1, (40_000,), 3, 3),
    (2, (512, 300), 64, 8), (9, (24, 24), 192, 24),
    # tiles of columns: whole groups in a block's registers, wide rows, one group across tiles
    (3, (40,), 8192, 64), (1, (700,), 8192, 2), (1, (70,), 5000, 1), (2, (3,), 70_000, 7),
    # more samples than share the blocks evenly, so that a block's rows cross samples; odd sizes among them
    (50, (26, 20), 64, 8), (50, (27, 19), 65, 5), (33, (130, 41), 16, 8), (40, (90, 77), 6, 3),
]


def _inputs(shape, dtype, ptype, seed):
    n, sp, c, _ = shape
    x = _normal((n, *sp, c), seed) * (0.5 + torch.rand(c, generator=torch.Generator().manual_seed(seed + 1)))
    x = (x + 0.7 * _normal((n,) + (1,) * len(sp) + (c,), seed + 2)).to(dtype)
    pt = torch.float32 if ptype == "f32" else dtype
    return x, (1 + 0.2 * _normal(c, seed + 3)).to(pt), (0.3 * _normal(c, seed + 4)).to(pt), _normal(x.shape, seed + 5, dtype)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{'x'.join(map(str, s[1]))}x{s[2]}g{s[3]}")
@pytest.mark.parametrize("dtype,ptype,act,p", [
    (torch.float32, "f32", "none", 0.0), (torch.float32, "f32", "gelu_tanh", 0.3), (torch.bfloat16, "f32", "silu", 0.0),
    (torch.bfloat16, "same", "silu", 0.1), (torch.float16, "same", "gelu_tanh", 0.0), (torch.float16, "f32", "none", 0.5),
], ids=lambda v: str(v).replace("torch.", ""))
def test_group_norm_matches_restatement(cuda, shape, dtype, ptype, act, p):
    import brush_b200 as bsx

    x, w, b, v = _inputs(shape, dtype, ptype, 20)
    g = shape[3]
    drop = bsx.DropoutConfig(p=p, seed=99, step=5) if p else None
    cfg = bsx.GroupNormConfig(groups=g, activation=act, dropout=drop)
    r = ref.GroupNorm(x, w, b, g, act=act, drop=(ref.mask(x.numel(), p, 99, 5), p) if p else None)
    d = [t.cuda() for t in (x, w, b, v)]
    out, mean, rstd = bsx.group_norm_forward(*d[:3], cfg)
    for got, want in zip((out, mean, rstd), r.forward()):
        ref.close(got, want)
    stats = [t.float().cuda() for t in (r.mean, r.rstd)]
    grads = bsx.group_norm_backward(d[3], *d[:3], *stats, cfg)
    for got, want in zip(grads, r.backward(v)):
        ref.close(got, want)
    assert out.dtype == grads[0].dtype == dtype and grads[1].dtype == grads[2].dtype == w.dtype


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape", [(2, (9, 11), 24, 4), (1, (5, 5), 9, 3), (3, (300, 20), 64, 8)],
                         ids=["vector", "odd", "long"])
def test_group_norm_without_parameters(cuda, has_w, has_b, shape):
    import brush_b200 as bsx

    x, w, b, v = _inputs(shape, torch.float32, "f32", 30)
    w, b = (w if has_w else None), (b if has_b else None)
    r = ref.GroupNorm(x, w, b, shape[3], act="silu")
    cfg = bsx.GroupNormConfig(groups=shape[3], activation="silu")
    dw, db = (None if t is None else t.cuda() for t in (w, b))
    out, mean, rstd = bsx.group_norm_forward(x.cuda(), dw, db, cfg)
    ref.close(out, r.forward()[0])
    grads = bsx.group_norm_backward(v.cuda(), x.cuda(), dw, db, r.mean.float().cuda(), r.rstd.float().cuda(), cfg)
    want = r.backward(v)
    ref.close(grads[0], want[0])
    for has, got, wnt in ((has_w, grads[1], want[1]), (has_b, grads[2], want[2])):
        assert (got is None) == (not has)
        if has:
            ref.close(got, wnt)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, (20, 20), 32, 8), (1, (600, 500), 12, 3), (2, (33, 5), 21, 7)])
def test_group_norm_hard_values(cuda, dtype, shape):
    """Constant groups, means far above the spread, one value far from the rest."""
    import brush_b200 as bsx

    n, sp, c, g = shape
    for kind in ("constant", "offset", "spike_first", "spike_late"):
        x, w, b, v = _inputs(shape, dtype, "f32", 40)
        if kind == "constant":
            x = torch.full_like(x, 3.0)
        elif kind == "offset":
            x = (200.0 + x.float()).to(dtype)
        elif kind == "spike_first":
            x.reshape(n, -1, c)[:, 0, 0] = 3000.0
        else:
            x.reshape(n, -1, c)[:, -1, c - 1] = -3000.0
        r = ref.GroupNorm(x, w, b, g, act="silu")
        out, mean, rstd = bsx.group_norm_forward(x.cuda(), w.cuda(), b.cuda(),
                                                 bsx.GroupNormConfig(groups=g, activation="silu"))
        for got, want in zip((out, mean, rstd), r.forward()):
            ref.close(got, want)


@pytest.mark.parametrize("shape", [(3, (9, 9), 24, 4), (3, (9, 9), 21, 7), (3, (200, 300), 32, 8), (40, (2,), 16, 4)])
@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_nan_stays_in_its_group(cuda, shape, dtype):
    import brush_b200 as bsx

    n, sp, c, g = shape
    x, w, b, v = _inputs(shape, dtype, "f32", 50)
    clean = bsx.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), bsx.GroupNormConfig(groups=g))
    cfg = bsx.GroupNormConfig(groups=g)
    back = bsx.group_norm_backward(v.cuda(), x.cuda(), w.cuda(), b.cuda(), *clean[1:], cfg)[0]
    per = c // g
    y = x.clone().reshape(n, -1, c)
    y[1, -1, per] = float("nan")  # sample 1, group 1
    y[2, 0, 0] = float("inf")     # sample 2, group 0
    y = y.reshape(x.shape)
    out, mean, rstd = bsx.group_norm_forward(y.cuda(), w.cuda(), b.cuda(), cfg)
    v_x = bsx.group_norm_backward(v.cuda(), y.cuda(), w.cuda(), b.cuda(), mean, rstd, cfg)[0]
    hit = torch.zeros(n, g, dtype=torch.bool)
    hit[1, 1] = hit[2, 0] = True
    assert torch.equal(rstd.cpu().isnan(), hit)
    m = hit.repeat_interleave(per, 1)[:, None, :].expand(n, x.numel() // n // c, c).reshape(x.shape)
    for got, want in ((out, clean[0]), (v_x, back)):
        got, want = got.cpu(), want.cpu()
        assert torch.equal(got[~m], want[~m])
        assert got[m].isnan().all()


def test_group_norm_drops_like_dropout(cuda):
    """The fused form draws the mask that dropout_forward draws for its output, and nothing of a dropped NaN stays."""
    import brush_b200 as bsx

    x, w, b, v = _inputs((2, (40, 41), 48, 8), torch.float32, "f32", 60)
    d = [t.cuda() for t in (x, w, b, v)]
    drop = bsx.DropoutConfig(p=0.37, seed=4, step=8)
    plain, mean, rstd = bsx.group_norm_forward(*d[:3], bsx.GroupNormConfig(groups=8, activation="silu"))
    fused = bsx.group_norm_forward(*d[:3], bsx.GroupNormConfig(groups=8, activation="silu", dropout=drop))[0]
    assert torch.equal(bsx.dropout_forward(plain, drop), fused)
    # backward: dropout's gradient through the plain norm's
    cfg = bsx.GroupNormConfig(groups=8, activation="silu")
    two = bsx.group_norm_backward(bsx.dropout_backward(d[3], drop), *d[:3], mean, rstd, cfg)
    one = bsx.group_norm_backward(d[3], *d[:3], mean, rstd,
                                  bsx.GroupNormConfig(groups=8, activation="silu", dropout=drop))
    r = ref.GroupNorm(x, w, b, 8, act="silu", drop=(ref.mask(x.numel(), 0.37, 4, 8), 0.37))
    for a, c, want in zip(one, two, r.backward(v)):
        ref.close(a, want)
        ref.close(c, want)
    keep = ref.mask(x.numel(), 0.37, 4, 8).reshape(x.shape)
    bad = v.clone()
    bad[~keep] = float("nan")
    again = bsx.group_norm_backward(bad.cuda(), *d[:3], mean, rstd,
                                    bsx.GroupNormConfig(groups=8, activation="silu", dropout=drop))
    assert all(torch.equal(a, c) for a, c in zip(one, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, (13, 7), 32, 8), (2, (13, 7), 33, 3), (1, (400, 333), 8, 2)])
def test_group_norm_unaligned_and_strided(cuda, dtype, shape):
    import brush_b200 as bsx

    n, sp, c, g = shape
    x, w, b, v = _inputs(shape, dtype, "same", 70)
    cfg = bsx.GroupNormConfig(groups=g, activation="silu")
    r = ref.GroupNorm(x, w, b, g, act="silu")

    def shifted(t):
        base = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
        base[1:] = t.reshape(-1).cuda()
        return base[1:].reshape(t.shape)

    nchw = torch.empty((n, c, *sp), dtype=dtype, device="cuda").copy_(x.movedim(-1, 1).cuda())
    for make in (shifted, lambda t: nchw.movedim(1, -1) if t is x else t.cuda()):
        d = [make(t) for t in (x, w, b, v)]
        for got, want in zip(bsx.group_norm_forward(*d[:3], cfg), r.forward()):
            ref.close(got, want)
        grads = bsx.group_norm_backward(d[3], *d[:3], r.mean.float().cuda(), r.rstd.float().cuda(), cfg)
        for got, want in zip(grads, r.backward(v)):
            ref.close(got, want)


def test_group_norm_gradient_against_differences(cuda):
    """Directional derivatives of the 64-bit forward equal the kernel's gradients along the direction."""
    import brush_b200 as bsx

    shape = (2, (11, 10), 24, 6)
    x, w, b, v = _inputs(shape, torch.float32, "f32", 80)
    drop = bsx.DropoutConfig(p=0.2, seed=1, step=2)
    cfg = bsx.GroupNormConfig(groups=6, activation="gelu_tanh", dropout=drop)
    keep = ref.mask(x.numel(), 0.2, 1, 2)
    out, mean, rstd = bsx.group_norm_forward(x.cuda(), w.cuda(), b.cuda(), cfg)
    grads = bsx.group_norm_backward(v.cuda(), x.cuda(), w.cuda(), b.cuda(), mean, rstd, cfg)
    dirs = [_normal(t.shape, 90 + k).double() for k, t in enumerate((x, w, b))]
    ref.HALF_STEP.setdefault(torch.float64, 0.0)
    ref.TINY.setdefault(torch.float64, 0.0)

    def loss(h):
        a = [t.double() + h * d for t, d in zip((x, w, b), dirs)]
        return float((ref.GroupNorm(*a, 6, act="gelu_tanh", drop=(keep, 0.2)).forward()[0][0] * v.double()).sum())

    h = 1e-5
    num = (loss(h) - loss(-h)) / (2 * h)
    got = sum(float((q.double().cpu() * d).sum()) for q, d in zip(grads, dirs))
    # each gradient is within its bound; the difference quotient adds h^2 and cancellation, both below 1e-6 of the terms
    r = ref.GroupNorm(x, w, b, 6, act="gelu_tanh", drop=(keep, 0.2)).backward(v)
    bound = sum(float((t * d.abs()).sum()) for (_, t), d in zip(r, dirs))
    scale = sum(float((q.abs() * d.abs()).sum()) for (q, _), d in zip(r, dirs))
    assert abs(got - num) <= bound + 1e-6 * scale


# Samples of an odd number of elements: large ones, read across vectors in 16 bits (one and many of them, a block's rows
# crossing them, a channel a group and one group, last vectors of every odd length), and smaller and even ones.
SHIFTED = [(1, (80_001,), 37, 37), (2, (100_001,), 37, 1), (3, (7777,), 185, 5), (3, (2001,), 511, 7), (1, (1_000_001,), 3, 3),
           (200, (501,), 37, 1), (61, (4801,), 9, 3), (9, (60_007,), 5, 1), (7, (18_003,), 21, 7), (4, (20_001,), 3, 3),
           (3, (1235, 21), 12, 4), (2, (9001,), 14, 7)]


@pytest.mark.parametrize("shape", SHIFTED, ids=lambda s: f"{s[0]}x{'x'.join(map(str, s[1]))}x{s[2]}g{s[3]}")
@pytest.mark.parametrize("dtype,act,p", [(torch.float32, "silu", 0.2), (torch.bfloat16, "gelu_tanh", 0.0),
                                         (torch.bfloat16, "silu", 0.3), (torch.float16, "none", 0.5)],
                         ids=lambda v: str(v).replace("torch.", ""))
def test_group_norm_samples_off_a_vector(cuda, shape, dtype, act, p):
    import brush_b200 as bsx

    x, w, b, v = _inputs(shape, dtype, "f32", 70)
    g = shape[3]
    drop = bsx.DropoutConfig(p=p, seed=31, step=2) if p else None
    cfg = bsx.GroupNormConfig(groups=g, activation=act, dropout=drop)
    r = ref.GroupNorm(x, w, b, g, act=act, drop=(ref.mask(x.numel(), p, 31, 2), p) if p else None)
    d = [t.cuda() for t in (x, w, b, v)]
    stats = [t.float().cuda() for t in (r.mean, r.rstd)]
    once = [bsx.group_norm_forward(*d[:3], cfg), bsx.group_norm_backward(d[3], *d[:3], *stats, cfg)]
    for got, want in zip(once[0], r.forward()):
        ref.close(got, want)
    for got, want in zip(once[1], r.backward(v)):
        ref.close(got, want)
    again = [bsx.group_norm_forward(*d[:3], cfg), bsx.group_norm_backward(d[3], *d[:3], *stats, cfg)]
    for a, c in zip(once, again):
        assert all(torch.equal(s, t) for s, t in zip(a, c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [0, 1, 2])
def test_group_norm_neighbours_of_a_bad_sample(cuda, dtype, bad):
    # A vector across two samples holds values of both: a sample of NaN leaves the others as they are, bit for bit.
    import brush_b200 as bsx

    x, w, b, v = (t.cuda() for t in _inputs((3, (25_001,), 37, 37), dtype, "f32", 75))
    cfg = bsx.GroupNormConfig(groups=37, activation="silu", dropout=bsx.DropoutConfig(p=0.25, seed=4, step=1))
    out, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
    vx = bsx.group_norm_backward(v, x, w, b, mean, rstd, cfg)[0]
    x2, v2 = x.clone(), v.clone()
    x2[bad] = float("nan")
    v2[bad] = float("nan")
    out2, mean2, rstd2 = bsx.group_norm_forward(x2, w, b, cfg)
    vx2 = bsx.group_norm_backward(v2, x2, w, b, mean2, rstd2, cfg)[0]
    for k in range(3):
        if k == bad:
            assert mean2[k].isnan().all() and rstd2[k].isnan().all()
            kept = ref.mask(x.numel(), 0.25, 4, 1).view(3, 25_001, 37)[k]
            assert torch.equal(out2[k].isnan().cpu(), kept) and (out2[k].cpu()[~kept] == 0).all()
        else:
            for one, two in ((out, out2), (mean, mean2), (rstd, rstd2), (vx, vx2)):
                assert torch.equal(one[k], two[k])


@pytest.mark.parametrize("shape", [(3, (20, 20), 64, 8), (2, (300, 200), 48, 8), (2, (31, 17), 37, 37)])
def test_group_norm_repeats_bit_for_bit(cuda, shape):
    import brush_b200 as bsx

    x, w, b, v = (t.cuda() for t in _inputs(shape, torch.float32, "f32", 100))
    cfg = bsx.GroupNormConfig(groups=shape[3], activation="silu")
    first = None
    for _ in range(4):
        f = bsx.group_norm_forward(x, w, b, cfg)
        got = f + bsx.group_norm_backward(v, x, w, b, f[1], f[2], cfg)
        first = first or got
        assert all(torch.equal(a, c) for a, c in zip(first, got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, (13, 7), 32, 8), (1, (400, 90), 64, 16), (3, (201, 7), 21, 7)])
def test_group_norm_drops_everything(cuda, dtype, shape):
    """p = 1 leaves nothing, whatever the gradient holds, and the statistics as they are."""
    import brush_b200 as bsx

    x, w, b, v = (t.cuda() for t in _inputs(shape, dtype, "f32", 65))
    cfg = bsx.GroupNormConfig(groups=shape[3], activation="silu", dropout=bsx.DropoutConfig(p=1.0))
    out, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
    plain = bsx.group_norm_forward(x, w, b, bsx.GroupNormConfig(groups=shape[3], activation="silu"))
    assert (out == 0).all() and torch.equal(mean, plain[1]) and torch.equal(rstd, plain[2])
    v[0] = float("nan")
    for g in bsx.group_norm_backward(v, x, w, b, mean, rstd, cfg):
        assert (g == 0).all()


def test_two_graphs_at_once(cuda):
    """Graphs of large norms, whose blocks wait for one another, replayed on two streams at the same time."""
    import brush_b200 as bsx

    shape = (2, (120, 130), 64, 8)
    data = [[t.cuda() for t in _inputs(shape, torch.float32, "f32", 300 + 10 * k)] for k in range(2)]
    want = [_block(bsx, *d, 1) for d in data]
    graphs = []
    for d in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _block(bsx, *d, 1)
        graphs.append((graph, got, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, s in graphs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, got, _), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))


def test_group_norm_empty_batch(cuda):
    import brush_b200 as bsx

    x, cfg = torch.empty(0, 4, 4, 8, device="cuda"), bsx.GroupNormConfig(groups=2)
    w = torch.ones(8, device="cuda")
    out, mean, rstd = bsx.group_norm_forward(x, w, w, cfg)
    assert out.shape == x.shape and mean.shape == rstd.shape == (0, 2)
    v_x, v_w, v_b = bsx.group_norm_backward(x, x, w, w, mean, rstd, cfg)
    assert v_x.shape == x.shape and (v_w == 0).all() and (v_b == 0).all()


def test_group_norm_far_elements(cuda):
    """Offsets beyond 2^31 elements: the last sample equals the same sample alone."""
    import brush_b200 as bsx

    def step_apart(a, b):
        # the two split their sums differently, so their 32-bit values differ by far less than a bf16 step (2^-7 of
        # the value at most) and round to the same number or to neighbours
        a, b = a.float(), b.float()
        return bool(((a - b).abs() <= 2.0**-7 * torch.maximum(a.abs(), b.abs()) + 1e-4).all())

    torch.manual_seed(0)
    n, px, c = 33, 1 << 20, 64  # 2.2e9 elements
    one = torch.randn(1, px, c, device="cuda").bfloat16()
    x = one.expand(n, px, c).contiguous()
    v = torch.randn(1, px, c, device="cuda").bfloat16().expand(n, px, c).contiguous()
    w, b = torch.randn(c, device="cuda"), torch.randn(c, device="cuda")
    cfg = bsx.GroupNormConfig(groups=16, activation="silu")
    out, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
    want = bsx.group_norm_forward(one, w, b, cfg)
    x64 = one.double().reshape(px, 16, 4)
    m64 = x64.mean((0, 2))
    assert (mean.double() - m64).abs().max() <= 1e-5 and (mean[-1] - want[1][0]).abs().max() <= 1e-6
    assert (rstd[-1] / want[2][0] - 1).abs().max() <= 1e-5
    assert step_apart(out[-1], want[0][0])
    del out
    v_x, v_w, v_b = bsx.group_norm_backward(v, x, w, b, mean, rstd, cfg)
    g = bsx.group_norm_backward(v[:1], one, w, b, mean[:1].contiguous(), rstd[:1].contiguous(), cfg)
    assert step_apart(v_x[-1], g[0][0])
    assert (v_w / n - g[1]).abs().max() <= 1e-3 * g[1].abs().max()
    del x, v, v_x
    torch.cuda.empty_cache()


def test_group_norm_refusals(cuda):
    import brush_b200 as bsx

    x, cfg = torch.zeros(2, 4, 8, device="cuda"), bsx.GroupNormConfig(groups=2)
    w = torch.ones(8, device="cuda")
    for args in [(x.cpu(), None, None, cfg), (x.double(), None, None, cfg), (x, w.cpu(), None, cfg),
                 (x[0, 0], None, None, cfg), (x[:, :0], None, None, cfg)]:
        with pytest.raises(ValueError):
            bsx.group_norm_forward(*args)
    st = torch.zeros(2, 2, device="cuda")
    for args in [(x[:1], x, w, w, st, st, cfg), (x.half(), x, w, w, st, st, cfg), (x, x, w, w, st[:1], st, cfg),
                 (x, x, w, w, st, st.half(), cfg), (x, x, w, w, st, st.cpu(), cfg)]:
        with pytest.raises(ValueError):
            bsx.group_norm_backward(*args)


def test_group_norm_entry_point_errors(cuda, bsx_lib):
    import ctypes as C

    from brush_b200._context import context

    ctx, L = context(0), bsx_lib.lib()
    x = torch.zeros(2 * 9000 * 8, device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    st = torch.zeros(64, device="cuda")
    s = torch.cuda.current_stream().cuda_stream

    def call(g=2, eps=1e-5, act=0, pt=0, t=0, n=2, px=16, c=8, xp=x.data_ptr(), wsp=ws.data_ptr(), wsn=ws.numel()):
        cfg = bsx_lib.GroupNormCfg(g, eps, act, pt, None)
        f = L.bsx_group_norm_fwd(ctx.handle, xp, None, None, n, px, c, t, C.byref(cfg), xp, st.data_ptr(),
                                 st.data_ptr(), wsp, wsn, s)
        b = L.bsx_group_norm_bwd(ctx.handle, xp, xp, None, None, st.data_ptr(), st.data_ptr(), n, px, c, t, C.byref(cfg),
                                 xp, None, None, wsp, wsn, s)
        assert f == b
        return f

    for kw, want in [(dict(g=3), 2), (dict(g=0), 2), (dict(c=0), 2), (dict(px=0), 2), (dict(n=1 << 31), 2),
                     (dict(px=1 << 62), 2), (dict(eps=-1.0), 1), (dict(act=3), 1), (dict(pt=1), 1), (dict(t=3), 1),
                     (dict(t=-1), 1), (dict(xp=None), 1), (dict(xp=x.data_ptr() + 2), 1),
                     (dict(wsp=ws.data_ptr() + 4), 1),
                     # samples that a block holds need no workspace in the forward; these do
                     (dict(wsn=0, px=9000), 3), (dict(wsp=None, px=9000), 3)]:
        assert call(**kw) == want, kw
        assert L.bsx_last_error(ctx.handle)
    ctx.sync()


# ---- together ----


def _block(bsx, x, w, b, v, step):
    """One residual-block prologue, forward and backward: out = x + drop(silu(norm(x))), and its gradients."""
    cfg = bsx.GroupNormConfig(groups=8, activation="silu")
    drop = bsx.DropoutConfig(p=0.25, seed=17, step=step)
    h, mean, rstd = bsx.group_norm_forward(x, w, b, cfg)
    out = bsx.dropout_forward(h, drop, residual=x)
    v_x, v_w, v_b = bsx.group_norm_backward(bsx.dropout_backward(v, drop), x, w, b, mean, rstd, cfg)
    return out, v + v_x, v_w, v_b


def _block_want(x, w, b, v, step):
    keep = ref.mask(x.numel(), 0.25, 17, step)
    r = ref.GroupNorm(x, w, b, 8, act="silu", drop=(keep, 0.25))
    (y, t), _, _ = r.forward()
    gx, gw, gb = r.backward(v)
    u = ref.U
    return ((y + x.double(), t + 2 * u * (y.abs() + x.abs().double())),
            (gx[0] + v.double(), gx[1] + 2 * u * (gx[0].abs() + v.abs().double())), gw, gb)


def test_block_runs_together_in_a_graph(cuda):
    """Forward and backward captured once, replayed with new inputs and steps; an eager run lives beside it."""
    import brush_b200 as bsx

    shape = (2, (30, 31), 32, 8)
    w, b = _inputs(shape, torch.float32, "f32", 110)[1:3]
    sx, sv = (torch.zeros(2, 30, 31, 32, device="cuda") for _ in range(2))
    step = torch.zeros(1, dtype=torch.int32, device="cuda")
    dw, db = w.cuda(), b.cuda()
    _block(bsx, sx, dw, db, sv, step)
    graphs = []
    for _ in range(2):  # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _block(bsx, sx, dw, db, sv, step)
        graphs.append((graph, got))
    for k in range(3):
        x, _, _, v = _inputs(shape, torch.float32, "f32", 120 + 10 * k)
        eager = _block(bsx, x.cuda(), dw, db, v.cuda(), k)
        sx.copy_(x), sv.copy_(v), step.fill_(k)
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = _block_want(x, w, b, v, k)
        for graph, got in graphs:
            for e, a, wnt in zip(eager, got, want):
                assert torch.equal(e, a)
                ref.close(a, wnt)


def test_streams_and_threads(cuda):
    """Calls on two streams from two threads at once, with work that takes a while in front of them."""
    import brush_b200 as bsx

    shape = (2, (64, 64), 64, 8)
    data = [_inputs(shape, torch.float32, "f32", 200 + 10 * k) for k in range(2)]
    want = [_block(bsx, *(t.cuda() for t in d), 3) for d in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                d = [t.cuda() for t in data[k]]
                for _ in range(20):
                    got[k] = _block(bsx, *d, 3)
            s.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, c in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_operators_leave_the_context_stream_alone(cuda):
    """A render state made on one stream is still usable after a feature operator ran on another."""
    import brush_b200 as bsx
    from brush_b200.splats import config1_scene

    splats, cam, size, gt = config1_scene("cpu", seed=1, n=512)
    g = splats.to("cuda:0")
    out = bsx.render(cam, size, g.transforms, g.sh_coeffs, g.raw_opacities)
    loss, v = bsx.image_loss_fused(out.out_img, gt.cuda(), bsx.ImageLossConfig())
    vc = bsx.rasterize_bwd(v, True)
    before = bsx.project_bwd(vc, g.num_splats, g.sh_coeffs_per_splat).v_coeffs.clone()
    out = bsx.render(cam, size, g.transforms, g.sh_coeffs, g.raw_opacities)
    img = out.out_img[None].contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        feats, mean, rstd = bsx.group_norm_forward(img, None, None, bsx.GroupNormConfig(groups=2, activation="silu"))
    torch.cuda.current_stream().wait_stream(side)
    ref.close(feats, ref.GroupNorm(img.cpu(), None, None, 2, act="silu").forward()[0])
    loss, v = bsx.image_loss_fused(out.out_img, gt.cuda(), bsx.ImageLossConfig())
    vc = bsx.rasterize_bwd(v, True)
    after = bsx.project_bwd(vc, g.num_splats, g.sh_coeffs_per_splat).v_coeffs
    assert (after - before).abs().max() <= 1e-5 * before.abs().max()


def test_launches_are_counted_and_profiled(cuda):
    import brush_b200 as bsx
    from brush_b200._context import context

    x = torch.randn(2, 8, 8, 16, device="cuda")
    ctx = context(0)
    n = ctx.launches()
    ctx.profile(True)
    ctx.profile_reset()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        bsx.dropout_forward(x, bsx.DropoutConfig())
        bsx.group_norm_forward(x, None, None, bsx.GroupNormConfig(groups=4))
    prof = ctx.profile_read()
    ctx.profile(False)
    assert ctx.launches() >= n + 2
    assert any("dropout" in k for k in prof) and any("norm" in k for k in prof)
    assert all(ms > 0 for ms, _ in prof.values())


# ---- splat dropout in the training step ----


@pytest.mark.parametrize("p", [0.3, 0.7])
def test_splat_dropout_trains_the_kept_splats(cuda, bsx_lib, p):
    """A step with splat dropout renders, and moves, exactly the splats its mask keeps: its loss and update equal
    those of a trainer that holds only these splats; the others stay as they are."""
    import brush_b200 as bsx
    from brush_b200.splats import Splats, clustered_scene, orbit_camera, random_gt

    full = clustered_scene(6001, 1, "cpu", seed=3)
    w, h = 160, 96
    cam, gt = orbit_camera(0, 3, 8.0, w, h), random_gt(h, w, 8, "cpu").cuda()
    n = full.num_splats
    keep = ref.mask(n, p, 77, 1)
    g = full.to("cuda")
    cfg = bsx.TrainConfig(mean_noise=False, splat_dropout=p, dropout_seed=77)
    before = g.clone()
    tr = bsx.SplatTrainer(cfg, g)
    st = tr.step(cam, (w, h), gt, g)
    k = keep.cuda()
    part = Splats(before.transforms[k].contiguous(), before.sh_coeffs[k].contiguous(), before.raw_opacities[k].contiguous(),
                  before.render_mode)
    tr2 = bsx.SplatTrainer(bsx.TrainConfig(mean_noise=False), part)
    # the rate of the means follows the bounds of all splats
    tr2.median_scale = tr.median_scale
    tr2.native.ctx.check(bsx_lib.lib().bsx_trainer_set_median_scale(tr2.native.handle, tr.median_scale))
    st2 = tr2.step(cam, (w, h), gt, part)
    assert st.num_visible == st2.num_visible and st.num_intersections == st2.num_intersections
    assert torch.equal(st.loss, st2.loss)  # the same splats in the same order
    assert torch.equal(tr.record.vis_weight.cpu() > 0, (tr.record.vis_weight.cpu() > 0) & keep)
    for name in ("transforms", "sh_coeffs", "raw_opacities"):
        a, b, o = getattr(g, name), getattr(part, name), getattr(before, name)
        assert torch.equal(a[~k], o[~k])
        # the first AdamScaled step moves a parameter by its rate times the gradient's sign: sums of gradients in
        # another order can turn the sign only where they cancel
        same = (a[k] - b).abs() <= 1e-6 * (1 + b.abs())
        assert same.float().mean() >= 0.999
        assert not torch.equal(a[k], o[k])
    # another step leaves others out
    st3 = tr.step(cam, (w, h), gt, g)
    assert st3.num_visible > 0
    tr.close(), tr2.close()


def test_splat_dropout_refusals_and_default(cuda, bsx_lib):
    import brush_b200 as bsx
    from brush_b200.splats import clustered_scene

    g = clustered_scene(1000, 1, "cpu", seed=3).to("cuda")
    for p in (1.0, -0.1, float("nan")):
        with pytest.raises(bsx.BsxError):
            bsx.SplatTrainer(bsx.TrainConfig(splat_dropout=p), g)
    tr = bsx.SplatTrainer(bsx.TrainConfig(), g)
    ctx = tr.native.ctx
    ctx.profile(True)
    ctx.profile_reset()
    from brush_b200.splats import orbit_camera, random_gt
    tr.step(orbit_camera(0, 3, 8.0, 64, 64), (64, 64), random_gt(64, 64, 1, "cpu").cuda(), g)
    names = set(ctx.profile_read())
    ctx.profile(False)
    assert "splat_dropout_kernel" not in names  # off by default: the step launches what it did
    tr.close()
