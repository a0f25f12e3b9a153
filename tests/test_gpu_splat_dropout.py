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


def _exchange(g):
    """The structures of bsx_train_step_dp for one rank, over the splats' own tensors."""
    from brush_b200 import _lib

    n, c = g.num_splats, g.sh_coeffs_per_splat
    z = lambda *shape, **kw: torch.zeros(shape, device="cuda", **kw)  # noqa: E731
    bufs = dict(flags=z(_lib.BSX_DP_FLAG_WORDS, dtype=torch.int32), refine=z(n), gate=z(n), vt=z(n, 10), vs=z(n, c, 3), vo=z(n))
    ex, sp = _lib.DpExchange(), _lib.DpSplats()
    ex.rank, ex.world, ex.refine_rows, ex.timeout_ns = 0, 1, n, int(1e9)
    for field, t in ((ex.d_flags, bufs["flags"]), (ex.d_refine, bufs["refine"]), (ex.d_gate, bufs["gate"]),
                     (sp.d_transforms, g.transforms), (sp.d_sh_coeffs, g.sh_coeffs), (sp.d_raw_opac, g.raw_opacities),
                     (sp.d_v_transforms, bufs["vt"]), (sp.d_v_sh_coeffs, bufs["vs"]), (sp.d_v_raw_opac, bufs["vo"])):
        field[0] = t.data_ptr()
    return ex, sp, bufs


def test_data_parallel_step_counts_its_mask_from_the_moments(cuda, bsx_lib):
    """bsx_train_step_dp draws the mask of the step that it reports, also where the moments start anew."""
    import brush_b200 as bsx

    g, cam, gt = _scene()
    n, L = g.num_splats, bsx_lib.lib()
    tr = bsx.SplatTrainer(_config(), g)
    ex, sp, bufs = _exchange(g)

    def step():
        st, cc = bsx_lib.TrainStats(), cam.to_c()
        masks = [_visible(g, cam, ref.mask(n, P, SEED, k)) for k in (1, 2, 3, 4)]
        assert len({c for c, _ in masks}) == 4  # each mask sees another number of splats
        tr.native.ctx.check(L.bsx_train_step_dp(tr.native.handle, C.byref(cc), *SIZE, gt.data_ptr(), C.byref(ex), C.byref(sp),
                                                1, tr.loss.data_ptr(), C.byref(st)))
        torch.cuda.synchronize()
        return st.step, [c for c, _ in masks].index(st.num_visible) + 1

    assert step() == (1, 1)
    assert step() == (2, 2)
    # another shard's moments: the next step of all splats starts from zero, as the single-GPU step's does
    half = [t[:n // 2].clone() for s in tr.native.optimizer_state() for t in s]
    tr.native.load_optimizer_state(half[:3], half[3:], n // 2, 2, 0)
    assert step() == (1, 1)
    assert step() == (2, 2)
    tr.native.load_optimizer_state(half[:3], half[3:], n // 2, 2, 0)
    st = tr.step(cam, SIZE, gt, g)
    assert tr.step_count == 1
    tr.close()
