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
