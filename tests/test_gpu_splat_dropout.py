"""Splat dropout over several steps, with live moments, and in each form of the training step."""
import ctypes as C

import pytest
import torch

import features_ref as ref

pytestmark = pytest.mark.gpu

P, SEED = 0.4, 77
SIZE = (160, 96)


def _scene():
    from brush_b200.splats import clustered_scene, orbit_camera, random_gt

    w, h = SIZE
    return clustered_scene(6001, 1, "cpu", seed=3).to("cuda"), orbit_camera(0, 3, 8.0, w, h), random_gt(h, w, 8, "cpu").cuda()


def _config(**kw):
    import brush_b200 as bsx

    return bsx.TrainConfig(mean_noise=False, uniform_lr=1e-3, **{"splat_dropout": P, "dropout_seed": SEED, **kw})


def _visible(g, cam, keep):
    """What a render of the kept splats alone sees, by global id."""
    import brush_b200 as bsx

    opac = torch.where(keep.cuda(), g.raw_opacities, torch.full_like(g.raw_opacities, -float("inf")))
    out = bsx.render(cam, SIZE, g.transforms, g.sh_coeffs, opac, g.render_mode)
    return out.aux.num_visible, out.aux.visible.clone() > 0


def _equal(a, b):
    return all(torch.equal(getattr(a, k), getattr(b, k)) for k in ("transforms", "sh_coeffs", "raw_opacities"))


def test_each_step_draws_its_own_mask(cuda):
    """Steps 1 to 3 see what renders of their masks' splats see; a splat that is left out has gradients of 0, and
    AdamScaled moves it by its moments alone, like one out of view."""
    import brush_b200 as bsx

    g, cam, gt = _scene()
    n = g.num_splats
    tr = bsx.SplatTrainer(_config(), g, keep_gradients=True)
    seen, masks = torch.zeros(n, device="cuda"), []
    for step in (1, 2, 3):
        keep = ref.mask(n, P, SEED, step)
        masks.append(keep)
        count, visible = _visible(g, cam, keep)
        before = g.clone()
        state = tr.native.optimizer_state()
        old = None if state is None else [[t.clone() for t in s] for s in state]
        st = tr.step(cam, SIZE, gt, g)
        assert st.num_visible == count
        seen += visible
        assert torch.equal(tr.record.vis_weight > 0, seen > 0)
        out = ~keep.cuda()
        for grad in (tr.grads.v_transforms, tr.grads.v_coeffs, tr.grads.v_raw_opac):
            assert (grad[out] == 0).all() and (grad[~out] != 0).any()
        if old is None:
            assert all(torch.equal(getattr(g, k)[out], getattr(before, k)[out]) for k in ("transforms", "raw_opacities"))
            continue
        m, v = tr.native.optimizer_state()
        for k in range(3):  # 0.9 m and 0.999 v: one rounding each, of the product and of the constant
            for new, was, beta in ((m[k], old[0][k], 0.9), (v[k], old[1][k], 0.999)):
                want = beta * was[out].double()
                assert ((new[out].double() - want).abs() <= 4 * ref.U * want.abs() + 1e-44).all()
        moved, still = old[0][2].abs() > 1e-9, old[0][2] == 0  # a step of 1e-3 m / sqrt(v) that a logit of order 1 shows
        assert (out & moved).any() and (g.raw_opacities != before.raw_opacities)[out & moved].all()
        assert torch.equal(g.raw_opacities[out & still], before.raw_opacities[out & still])
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])
    tr.close()


def _without_ranks(monkeypatch, tr, g):
    """The several-rank step around torch's collectives, on one rank's gradients: the collective left out."""
    from brush_b200 import train

    monkeypatch.setattr(train, "reduce_gradients", lambda grad, refine, group: 1.0)
    tr.world, tr.exchange, tr.shard_optimizer = 2, "nccl", False
    tr._alloc(g)
    return tr


@pytest.mark.parametrize("seed", [SEED, -3, (1 << 64) - 3])
def test_collective_step_draws_the_native_mask(cuda, monkeypatch, seed):
    import brush_b200 as bsx

    g, cam, gt = _scene()
    h = g.clone()
    one = bsx.SplatTrainer(_config(dropout_seed=seed), g)
    two = _without_ranks(monkeypatch, bsx.SplatTrainer(_config(dropout_seed=seed), h), h)
    assert two.native is None
    for step in (1, 2, 3):
        a, b = one.step(cam, SIZE, gt, g), two.step(cam, SIZE, gt, h)
        assert (a.num_visible, a.num_intersections) == (b.num_visible, b.num_intersections)
        assert torch.equal(one.record.vis_weight > 0, two.record.vis_weight > 0)
        if step == 1:
            assert torch.equal(a.loss, b.loss)
            keep = ref.mask(g.num_splats, P, seed % 2**64, 1)
            assert _visible(h, cam, keep)[0] <= keep.sum() and torch.equal(two.record.vis_weight > 0,
                                                                          (two.record.vis_weight > 0) & keep.cuda())
        for name in ("transforms", "sh_coeffs", "raw_opacities"):
            setattr(h, name, getattr(g, name).clone())  # sums of gradients differ in their order: the same start again
    one.close(), two.close()


def test_collective_step_refuses_what_the_native_one_refuses(cuda, monkeypatch):
    import brush_b200 as bsx

    g, cam, gt = _scene()
    tr = _without_ranks(monkeypatch, bsx.SplatTrainer(_config(), g), g)
    for p in (1.0, -0.1, float("nan")):
        tr.config.splat_dropout = p
        with pytest.raises(bsx.BsxError):
            tr.step(cam, SIZE, gt, g)
