"""64-bit restatements of dropout and group norm for the tests, with error bounds.

The bounds are worst cases counted from the operations, u = 2^-24 being half a step of a
32-bit float: a sum whose longest chain has k additions is off by at most k u times the sum of
its terms' sizes; an exponential of w is off by (4 + 2 |w|) u relative (rounding w log2(e), the
exponential and its result); a result rounded to type T is off by eps(T) / 2 relative. Terms
of second order in u are covered by counting a few roundings more than there are.
"""
import numpy as np
import torch

U = 2.0**-24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}  # absolute, below normal numbers


def philox(c, k, rounds=7):
    """Philox-4x32 on uint64 arrays holding 32-bit words."""
    c0, c1, c2, c3 = (np.asarray(x, np.uint64) for x in c)
    k0, k1 = k
    m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> s) ^ c1 ^ np.uint64(k0), b & m, (a >> s) ^ c3 ^ np.uint64(k1), a & m
        k0, k1 = (k0 + 0x9E3779B9) % 2**32, (k1 + 0xBB67AE85) % 2**32
    return c0, c1, c2, c3


def draws(first, count, seed, step):
    """The 32-bit draws [first, first + count)."""
    m = np.arange(first, first + count, dtype=np.uint64)
    q0 = first // 8
    q = np.arange(q0, (first + count + 7) // 8 + 1, dtype=np.uint64)
    u = np.zeros(q.size * 8, np.uint64)
    for half in (0, 1):
        w = philox((q & np.uint64(0xFFFFFFFF), q >> np.uint64(32), np.full_like(q, step), np.full_like(q, half)),
                   (seed % 2**32, seed >> 32))
        h = np.stack([x for v in w for x in (v & np.uint64(0xFFFF), v >> np.uint64(16))], 1).reshape(-1)
        u = (u << np.uint64(16)) | h
    return u[(m - np.uint64(q0 * 8)).astype(np.int64)]


def mask(count, p, seed, step, share=1, first=0):
    """Which of the elements [first, first + count) are kept."""
    d0, d1 = first // share, (first + count - 1) // share
    keep = draws(d0, d1 - d0 + 1, seed, step) >= np.uint64(round(p * 2**32))
    return torch.from_numpy(np.repeat(keep, share)[first - d0 * share:][:count])


def dropout(x, p, seed, step, share=1, residual=None):
    """The kernel's own arithmetic in 32 bits: product, sum, one rounding (so results are equal, not near)."""
    keep = mask(x.numel(), p, seed, step, share).reshape(x.shape)
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    y = torch.where(keep, x.float() * float(scale), torch.zeros(()))
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _gate(z, act):
    if act == "none":
        return torch.ones_like(z), torch.zeros_like(z), torch.zeros_like(z)
    a = 2.0 * (2.0 / np.pi) ** 0.5
    w, dw = (z, torch.ones_like(z)) if act == "silu" else (a * (z + 0.044715 * z**3), a * (1 + 0.134145 * z * z))
    return torch.sigmoid(w), dw, w


class GroupNorm:
    """Forward and backward in 64 bits for inputs of any type, and the kernels' error bounds."""

    def __init__(self, x, weight, bias, groups, eps=1e-5, act="none", drop=None):
        self.x, self.act, self.g = x.double().cpu(), act, groups
        self.type, self.shape = x.dtype, x.shape
        n, c = x.shape[0], x.shape[-1]
        self.ptype = weight.dtype if weight is not None else bias.dtype if bias is not None else torch.float32
        self.x = self.x.reshape(n, -1, c)
        self.w = torch.ones(c).double() if weight is None else weight.double().cpu()
        self.b = torch.zeros(c).double() if bias is None else bias.double().cpu()
        self.n, self.c, self.per = n, c, c // groups
        self.m = self.x.shape[1] * self.per
        xg = self.x.reshape(n, -1, groups, self.per)
        self.mean = xg.mean((1, 3))
        self.var = (xg - self.mean[:, None, :, None]).square().mean((1, 3))
        self.rstd = 1.0 / (self.var + eps).sqrt()
        # no sum of the kernels chains more additions than this
        self.chain = 64 + self.m / 128
        size = xg.abs().mean((1, 3))
        spread = (xg - self.mean[:, None, :, None]).abs().mean((1, 3))
        # the mean is a sum of deviations from a value of the group, or of the values themselves
        self.t_mean = self.chain * U * torch.maximum(size, spread) + 2 * U * self.mean.abs()
        # squares of deviations: each is off by two roundings and by the pivot's, the sum by its chain; a mean that
        # is off by t_mean adds its square. Half of that is rstd's, and three roundings of its own
        rel = (2 * self.chain + 16) * U + self.t_mean**2 * self.rstd**2 + 4 * U * size * self.rstd
        self.t_rstd = self.rstd * (rel / 2 + 4 * U)
        # dropped: None, or (keep mask, p)
        self.keep = None if drop is None else drop[0].reshape(self.x.shape)
        self.scale = 1.0 if drop is None else (1.0 / (1.0 - drop[1]) if drop[1] < 1 else 0.0)

    def _of(self, q):
        return q.repeat_interleave(self.per, 1)[:, None, :]

    def _drop(self, v):
        return v if self.keep is None else torch.where(self.keep, v * self.scale, torch.zeros_like(v))

    def _z(self, t_mean, t_rstd):
        xh = (self.x - self._of(self.mean)) * self._of(self.rstd)
        # the kernels may fold the statistics into the scale and shift: x a + b with a = gamma rstd, b = beta - mean a
        t_xh = (self._of(self.rstd * t_mean) + 6 * U * (self.x.abs() + self._of(self.mean.abs())) * self._of(self.rstd)
                + xh.abs() * self._of(t_rstd / self.rstd))
        z = xh * self.w + self.b
        t_z = self.w.abs() * t_xh + 4 * U * (self.b.abs() + z.abs())
        return xh, t_xh, z, t_z

    def _round(self, y, t, dtype):
        return t + HALF_STEP[dtype] * (y.abs() + t) * 1.01 + TINY[dtype]

    def forward(self):
        """(out, bound), (mean, bound), (rstd, bound)"""
        _, _, z, t_z = self._z(self.t_mean, self.t_rstd)
        g, _, w = _gate(z, self.act)
        y = z * g
        # the slope of z gate(z) stays below 1.13
        t = 1.13 * t_z + y.abs() * (12 + 4 * w.abs()) * U + z.abs() * 2.0**-60 * (w < -41)  # gates stop at 2^-60
        y, t = self._drop(y), t * self.scale * (1 + 2 * U)
        if self.keep is not None:
            t = torch.where(self.keep, t, torch.zeros_like(t))
        t = self._round(y, t, self.type)
        r = lambda q: q.reshape(self.shape)  # noqa: E731
        return (r(y), r(t)), (self.mean, self.t_mean), (self.rstd, self.t_rstd)

    def backward(self, v):
        """(v_x, bound), (v_weight, bound), (v_bias, bound), with the exact statistics rounded to 32 bits as inputs."""
        xh, t_xh, z, t_z = self._z(U * self.mean.abs(), U * self.rstd)
        g, dw, w = _gate(z, self.act)
        v = self._drop(v.double().cpu().reshape(self.x.shape))
        slope = g + z * g * (1 - g) * dw
        # second derivative below 1.2; the slope's own roundings, with the exponential's
        t_slope = 1.2 * t_z + (16 + 8 * w.abs()) * U * (1 + (z * dw).abs() * (1 - g) * g * 4)
        t_slope = t_slope + (1 + (z * dw).abs()) * 2.0**-60 * (w < -41)  # gates stop at 2^-60
        dz = v * slope
        t_dz = v.abs() * t_slope + 4 * U * dz.abs()
        chain = (64 + self.x.shape[1] / 128) * U
        a, b = dz.sum(1), (dz * xh).sum(1)
        t_a = t_dz.sum(1) + chain * dz.abs().sum(1)
        t_bb = t_dz * xh.abs() + dz.abs() * t_xh
        t_b = t_bb.sum(1) + chain * (dz * xh).abs().sum(1)
        group = lambda q: q.reshape(self.n, self.g, -1).sum(2) / self.m  # noqa: E731
        gc = (self.per + 16) * U
        s1, s2 = group(a * self.w), group(b * self.w)
        t1 = group(t_a * self.w.abs()) + gc * group((a * self.w).abs()) + 2 * U * s1.abs()
        t2 = group(t_b * self.w.abs()) + gc * group((b * self.w).abs()) + 2 * U * s2.abs()
        of, rstd = self._of, self._of(self.rstd)
        v_x = rstd * (dz * self.w - of(s1) - xh * of(s2))
        t = rstd * (t_dz * self.w.abs() + of(t1) + xh.abs() * of(t2) + t_xh * of(s2.abs())
                    + 6 * U * ((dz * self.w).abs() + of(s1.abs()) + (xh * of(s2)).abs()))
        nc = (self.n + 64) * U
        v_w, t_w = b.sum(0), t_b.sum(0) + nc * b.abs().sum(0)
        v_b, t_b2 = a.sum(0), t_a.sum(0) + nc * a.abs().sum(0)
        return ((v_x.reshape(self.shape), self._round(v_x, t, self.type).reshape(self.shape)),
                (v_w, self._round(v_w, t_w, self.ptype)), (v_b, self._round(v_b, t_b2, self.ptype)))


def close(got, want):
    """Every value of `got` within its bound of the 64-bit result."""
    y, t = want
    got = got.double().cpu()
    assert got.shape == y.shape
    off = (got - y).abs()
    bad = ~(off <= t)
    if bad.any():
        i = int((off / t).nan_to_num(float("inf")).reshape(-1).argmax())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} out of bounds; worst at {i}: got "
                             f"{got.reshape(-1)[i]}, want {y.reshape(-1)[i]} +- {t.reshape(-1)[i]}")
