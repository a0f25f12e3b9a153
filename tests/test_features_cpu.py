"""Dropout and group norm without a GPU: the generator's known answers, the 64-bit formulas
against differences, argument checks, struct layouts."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

import features_ref as ref

ROOT = Path(__file__).resolve().parent.parent


def test_generator_known_answers():
    """The published vectors of Philox-4x32 (Salmon et al. 2011) for 7 and 10 rounds."""
    f = 0xFFFFFFFF
    pi = ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0))
    for args, rounds, want in [
        (((0, 0, 0, 0), (0, 0)), 7, (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
        (((f, f, f, f), (f, f)), 7, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
        (((0, 0, 0, 0), (0, 0)), 10, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
        (((f, f, f, f), (f, f)), 10, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
        (pi, 10, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
    ]:
        assert tuple(int(w) for w in ref.philox(*args, rounds=rounds)) == want


def test_mask_statistics():
    n = 1 << 20
    for p in (0.1, 0.5):
        k = ref.mask(n, p, 7, 3).double()
        assert abs(k.mean() - (1 - p)) <= 5 * (p * (1 - p) / n) ** 0.5
        # neighbours, and the same place in the next step, are independent
        other = ref.mask(n, p, 7, 4).double()
        for a, b in ((k[1:], k[:-1]), (k, other)):
            cov = ((a - (1 - p)) * (b - (1 - p))).mean()
            assert abs(cov) <= 5 * p * (1 - p) / n**0.5
    assert ref.mask(1000, 0.0, 1, 1).all() and not ref.mask(1000, 1.0, 1, 1).any()
    assert torch.equal(ref.mask(1000, 0.3, 9, 2)[123:456], ref.mask(333, 0.3, 9, 2, first=123))
    assert torch.equal(ref.mask(1000, 0.3, 9, 2, share=7), ref.mask(143, 0.3, 9, 2).repeat_interleave(7)[:1000])


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_formulas_match_differences(act, p):
    """The backward formulas against central differences of the forward, all in 64 bits."""
    gen = torch.Generator().manual_seed(5)
    n, s, c, g = 2, 5, 6, 3
    x = torch.randn(n, s, c, generator=gen, dtype=torch.float64)
    w, b = torch.randn(c, generator=gen, dtype=torch.float64), torch.randn(c, generator=gen, dtype=torch.float64)
    v = torch.randn(n, s, c, generator=gen, dtype=torch.float64)
    drop = (ref.mask(x.numel(), p, 3, 1), p) if p else None
    ref.HALF_STEP.setdefault(torch.float64, 0.0)
    ref.TINY.setdefault(torch.float64, 0.0)

    def loss(x_, w_, b_):
        return float((ref.GroupNorm(x_, w_, b_, g, act=act, drop=drop).forward()[0][0] * v).sum())

    grads = [q[0] for q in ref.GroupNorm(x, w, b, g, act=act, drop=drop).backward(v)]
    h = 1e-5
    for k, t in enumerate((x, w, b)):
        for i in range(t.numel()):
            d = torch.zeros_like(t).reshape(-1)
            d[i] = h
            args = lambda sign: [q + sign * d.reshape(t.shape) if j == k else q for j, q in enumerate((x, w, b))]  # noqa: E731
            num = (loss(*args(1)) - loss(*args(-1))) / (2 * h)
            # truncation h^2 |f'''| / 6 with third derivatives of order 10, cancellation 2^-53 |f| / h
            assert abs(num - float(grads[k].reshape(-1)[i])) <= 1e-7


def test_configuration_refusals(bsx_lib):
    import brush_b200 as bsx
    from brush_b200.dropout import feature_tensor, like_tensor
    from brush_b200.norm import _call

    dev = torch.device("cpu")
    for kw in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(seed=-1), dict(seed=1 << 64), dict(step=-1),
               dict(step=1 << 32), dict(share=0), dict(step=torch.zeros(2, dtype=torch.int32)),
               dict(step=torch.zeros(1)), dict(step=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError):
            bsx.DropoutConfig(**kw).to_c(dev)
    c = bsx.DropoutConfig(p=np.float32(0.25), seed=np.int64(7), step=np.int32(3), share=np.int64(2)).to_c(dev)
    assert (c.p, c.seed, c.step, c.share) == (0.25, 7, 3, 2)
    c = bsx.DropoutConfig(p=0.25, seed=(1 << 64) - 1, step=(1 << 32) - 1, share=3).to_c(dev)
    assert (c.p, c.seed, c.step, c.share, c.d_step) == (0.25, (1 << 64) - 1, (1 << 32) - 1, 3, None)

    for t in (torch.zeros(3, dtype=torch.float64), torch.zeros(3, dtype=torch.int32), [1.0], torch.zeros(3)):
        with pytest.raises(ValueError):
            feature_tensor(t, "x")
    x = torch.zeros(2, 3, 8)
    for t in (torch.zeros(2, 3, 4), torch.zeros(2, 3, 8, dtype=torch.float16), None):
        with pytest.raises(ValueError):
            like_tensor(t, x, "v_output")

    ok = bsx.GroupNormConfig(groups=4)
    assert _call(x, None, None, ok)[0][:3] == (2, 3, 8)
    half = torch.zeros(8, dtype=torch.float16)
    for bad_x, w, b, cfg in [
        (torch.zeros(8), None, None, ok),                                   # no batch
        (x, None, None, bsx.GroupNormConfig(groups=3)),                     # 8 % 3
        (x, None, None, bsx.GroupNormConfig(groups=0)),
        (torch.zeros(2, 0, 8), None, None, ok),                             # no pixel
        (torch.zeros(2, 3, 0), None, None, ok),
        (x, torch.zeros(4), None, ok),                                      # weight per group
        (x, None, torch.zeros(8, 1), ok),
        (x, half, None, ok),                                                # neither float32 nor x's type
        (x.half(), half, torch.zeros(8), ok),                               # two types
        (x, None, None, bsx.GroupNormConfig(groups=4, eps=-1.0)),
        (x, None, None, bsx.GroupNormConfig(groups=4, eps=float("nan"))),
        (x, None, None, bsx.GroupNormConfig(groups=4, activation="relu")),
        (x, None, None, bsx.GroupNormConfig(groups=4, dropout=bsx.DropoutConfig(share=8))),
        (x, None, None, bsx.GroupNormConfig(groups=4, dropout=bsx.DropoutConfig(p=2.0))),
    ]:
        with pytest.raises(ValueError):
            _call(bad_x, w, b, cfg)


def test_entry_points_refuse_without_a_context(bsx_lib):
    lib = bsx_lib.lib()
    d, g = bsx_lib.DropoutCfg(), bsx_lib.GroupNormCfg()
    assert lib.bsx_dropout_fwd(None, None, None, 0, 0, C.byref(d), None, None) == 1
    assert lib.bsx_dropout_bwd(None, None, 0, 0, C.byref(d), None, None) == 1
    assert lib.bsx_group_norm_fwd(None, None, None, None, 0, 0, 0, 0, C.byref(g), None, None, None, None, 0, None) == 1
    assert lib.bsx_group_norm_bwd(None, None, None, None, None, None, None, 0, 0, 0, 0, C.byref(g), None, None, None,
                                  None, 0, None) == 1


def test_workspace_sizes(bsx_lib):
    lib = bsx_lib.lib()
    need = C.c_uint64()
    for n, s, c, g in [(0, 5, 8, 2), (1, 1, 1, 1), (3, 1 << 40, 64, 16), (100000, 7, 21, 3)]:
        for bwd in (0, 1):
            assert lib.bsx_group_norm_workspace(n, s, c, g, bwd, C.byref(need)) == 0
            assert need.value < 1 << 34
    for n, s, c, g in [(1, 1, 8, 3), (1, 1, 0, 1), (1, 1, 8, 0), (1 << 31, 1, 8, 8), (4, 1 << 62, 64, 16)]:
        assert lib.bsx_group_norm_workspace(n, s, c, g, 0, C.byref(need)) == 2
    assert lib.bsx_group_norm_workspace(1, 1, 8, 8, 0, None) == 1


def test_struct_layouts_match_header(bsx_lib, tmp_path):
    structs = {"DropoutCfg": "bsx_dropout_cfg", "GroupNormCfg": "bsx_group_norm_cfg"}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "bsx.h"}"', "int main(void) {"]
    want = []
    for py, cname in structs.items():
        t = getattr(bsx_lib, py)
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(C.sizeof(t))
        for field, _ in t._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {field}));')
            want.append(getattr(t, field).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    assert [int(v) for v in out.split()] == want
