"""What the feature operators share with other threads and with stream capture: error texts,
launch counts and launch times."""
import ctypes as C
import threading

import pytest
import torch

import features_ref as ref

pytestmark = pytest.mark.gpu


def _refused(bsx_lib, handle, x, share, dtype):
    """A dropout call that is refused: for its share (0), or for its element type."""
    cfg = bsx_lib.DropoutCfg(0.5, 1, share, None, 0)
    return bsx_lib.lib().bsx_dropout_fwd(handle, x.data_ptr(), None, 8, dtype, C.byref(cfg), x.data_ptr(), None)


def _in_thread(f):
    out = []
    t = threading.Thread(target=lambda: out.append(f()))
    t.start()
    t.join()
    return out[0]


def test_error_texts_belong_to_their_threads(cuda, bsx_lib):
    from brush_b200._context import context

    h, L, x = context(0).handle, bsx_lib.lib(), torch.zeros(8, device="cuda")
    text = lambda: L.bsx_last_error(h)  # noqa: E731
    assert _refused(bsx_lib, h, x, 0, 0) == 1
    mine = text()
    assert b"share" in mine
    # another thread's failure changes this thread's text no more, and that thread reads its own
    assert b"type" in _in_thread(lambda: (_refused(bsx_lib, h, x, 1, 9), text())[1])
    assert text() == mine
    # a thread without a failure of its own reads the context's last one
    assert b"type" in _in_thread(text)
    assert _refused(bsx_lib, h, x, 1, 9) == 1 and b"type" in text()


def test_errors_from_two_threads_at_once(cuda, bsx_lib):
    """Each failing call raises its own text."""
    from brush_b200._context import context

    ctx, x, wrong = context(0), torch.zeros(8, device="cuda"), []

    def work(share, dtype, word):
        for _ in range(3000):
            try:
                ctx.check(_refused(bsx_lib, ctx.handle, x, share, dtype))
                wrong.append("no error")
            except bsx_lib.BsxError as e:
                if word not in str(e):
                    wrong.append(str(e))

    threads = [threading.Thread(target=work, args=a) for a in [(0, 0, "share"), (1, 9, "type")]]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_profiling_leaves_captures_alone(cuda):
    """A call captured while launches are timed has no time of its own, and no error comes of it later."""
    import brush_b200 as bsx
    from brush_b200._context import context

    x = torch.randn(2, 9, 9, 16, device="cuda")
    ctx, drop = context(0), bsx.DropoutConfig(p=0.3, seed=2, step=1)
    norm = bsx.GroupNormConfig(groups=4)
    bsx.group_norm_forward(bsx.dropout_forward(x, drop), None, None, norm)
    torch.cuda.synchronize()
    ctx.profile(True)
    try:
        ctx.profile_reset()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = bsx.dropout_forward(x, drop)
            y = bsx.group_norm_forward(h, None, None, norm)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert ctx.profile_read() == {}
        assert torch.equal(h.cpu(), ref.dropout(x.cpu(), 0.3, 2, 1))  # the next launch reports no error of the times
        assert torch.equal(bsx.group_norm_forward(bsx.dropout_forward(x, drop), None, None, norm)[0], y)
        prof = ctx.profile_read()
        assert sorted(prof) == ["dropout_fwd_kernel", "norm_fwd_kernel"]
        assert all(n == 1 and ms > 0 for ms, n in prof.values())
    finally:
        ctx.profile(False)
        ctx.profile_reset()


def test_launches_of_threads_beside_a_render(cuda):
    """Renders on one thread and feature operators on two others, timed: each launch is counted and timed once."""
    import brush_b200 as bsx
    from brush_b200._context import context
    from brush_b200.splats import config1_scene

    splats, cam, size, _ = config1_scene("cpu", seed=1, n=512)
    g = splats.to("cuda:0")
    x = torch.randn(2, 30, 30, 32, device="cuda")
    ctx, drop, norm = context(0), bsx.DropoutConfig(p=0.3), bsx.GroupNormConfig(groups=4)
    want = bsx.group_norm_forward(x, None, None, norm)[0]
    image = bsx.render(cam, size, g.transforms, g.sh_coeffs, g.raw_opacities).out_img.clone()
    torch.cuda.synchronize()
    ctx.profile(True)
    ctx.profile_reset()
    bsx.render(cam, size, g.transforms, g.sh_coeffs, g.raw_opacities)
    each = sum(n for _, n in ctx.profile_read().values())
    ctx.profile_reset()
    before, rounds, errors = ctx.launches(), 60, []

    def features():
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(rounds):
                    bsx.dropout_forward(x, drop)
                    got = bsx.group_norm_forward(x, None, None, norm)[0]
            s.synchronize()
            assert torch.equal(got, want)
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=features) for _ in range(2)]
    for t in threads:
        t.start()
    for _ in range(rounds):
        out = bsx.render(cam, size, g.transforms, g.sh_coeffs, g.raw_opacities).out_img
    for t in threads:
        t.join()
    prof = ctx.profile_read()
    ctx.profile(False)
    ctx.profile_reset()
    assert not errors and torch.equal(out, image)
    assert ctx.launches() - before == rounds * (each + 4)
    assert prof["dropout_fwd_kernel"][1] == prof["norm_fwd_kernel"][1] == 2 * rounds
    assert sum(n for _, n in prof.values()) == rounds * (each + 4)
