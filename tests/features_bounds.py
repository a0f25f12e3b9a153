"""Error bounds for the feature operators that follow the kernels' own sums and the activations'
tails, for tests at sizes and values where those of features_ref.py say little.

Counted like those, u = 2^-24. A large sample's sums are deviations from a pivot, a value between
the group's smallest and largest, and no addition chain of the kernels is longer than CHAIN plus
one for each 64 rows that a thread walks: at most 64 rows of 4 lanes go into a partial sum, then
come the partial sums, the walk over a block's items (2 a thread and 5 shuffles for groups of few
channels), 148 blocks and the last halvings.
"""
import torch

import features_ref as ref

U = ref.U
CHAIN = 640


def normal(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _parts(z, act):
    """w, w', w'' of the gate s(w(z))."""
    if act == "silu":
        return z, torch.ones_like(z), torch.zeros_like(z)
    a, b = 2.0 * (2.0 / torch.pi) ** 0.5, 0.044715
    return a * (z + b * z**3), a * (1 + 3 * b * z * z), a * 6 * b * z


def _most(z, t, act):
    """The largest |act'| and |act''| between z - t and z + t, from act' = s (1 + (1 - s) z w') and
    act'' = s (1 - s) (2 w' + z w'' + (1 - 2 s) z w'^2), s and |z w'| being monotonic on each side of 0."""
    lo, hi = z - t, z + t
    near, far = torch.where(z < 0, hi, lo), torch.where(z < 0, lo, hi)
    w, _, _ = _parts(near, act)
    _, dw, ddw = _parts(far, act)
    tail = torch.sigmoid(-w.abs())  # s below 0, 1 - s above
    same = (lo > 0) | (hi < 0)
    slope = torch.where(hi < 0, (tail * (1 + (far * dw).abs())).clamp(max=1.13), torch.full_like(z, 1.13))
    bend = (tail * (2 * dw.abs() + (far * ddw).abs() + far.abs() * dw * dw)).clamp(max=1.2)
    return slope, torch.where(same, bend, torch.full_like(z, 1.2))


class GroupNorm(ref.GroupNorm):
    """`pivot`: the sample is large, so that its statistics are sums of deviations from a pivot."""

    def __init__(self, x, weight, bias, groups, eps=1e-5, act="none", drop=None, pivot=False):
        super().__init__(x, weight, bias, groups, eps, act, drop)
        if not pivot:
            return
        self.chain = CHAIN + self.x.shape[1] / (64 * 148)  # rows are dealt to the blocks
        off = (self.x.reshape(self.n, -1, groups, self.per) - self.mean[:, None, :, None]).abs()
        # the pivot is the mean of some values, rounded to their type
        p = off.amax((1, 3)) + ref.HALF_STEP[self.type] * self.mean.abs()
        # sums of deviations, and a few roundings at the mean's size: of the pivot's sum, the blocks' means, the result
        self.t_mean = self.chain * U * (off.mean((1, 3)) + p) + 6 * U * self.mean.abs()
        # squares of deviations from the pivot, less the square of their mean; the blocks' means are rounded
        sd = self.var.sqrt()
        rel = (3 * (self.chain + 6) * U * (sd + p) ** 2 + 4 * U * self.mean.abs() * sd) * self.rstd**2
        self.t_rstd = self.rstd * (rel / 2 + 4 * U)

    def forward(self):
        """(out, bound), (mean, bound), (rstd, bound)"""
        _, _, z, t_z = self._z(self.t_mean, self.t_rstd)
        if self.act == "none":
            y, t = z, t_z
        else:
            w, _, _ = _parts(z, self.act)
            y = z * torch.sigmoid(w)
            # the exponent has at most eight roundings relative to w (gelu's constants among them); gates are off by
            # 2^-62 besides, and 0 where they are less
            t = _most(z, t_z, self.act)[0] * t_z + y.abs() * (12 + 8 * w.abs()) * U
            t = t + torch.where(w > -45, z.abs() * 2.0**-62 * (w < 45), y.abs())
        y, t = self._drop(y), t * self.scale * (1 + 2 * U)
        if self.keep is not None:
            t = torch.where(self.keep, t, torch.zeros_like(t))
        t = self._round(y, t, self.type)
        return (y.reshape(self.shape), t.reshape(self.shape)), (self.mean, self.t_mean), (self.rstd, self.t_rstd)

    def backward(self, v):
        """As the base class: the exact statistics rounded to 32 bits are inputs."""
        xh, t_xh, z, t_z = self._z(U * self.mean.abs(), U * self.rstd)
        v = self._drop(v.double().cpu().reshape(self.x.shape))
        if self.act == "none":
            slope, t_slope = torch.ones_like(z), torch.zeros_like(z)
        else:
            w, dw, _ = _parts(z, self.act)
            s, q = torch.sigmoid(w), (z * dw).abs()
            c = torch.sigmoid(-w)
            slope = s * (1 + c * z * dw)
            t_slope = _most(z, t_z, self.act)[1] * t_z + (16 + 16 * w.abs()) * U * s * (1 + 2 * c * q)
            t_slope = t_slope + torch.where(w > -45, (1 + q) * 2.0**-61 * (w < 45), slope.abs())
        dz = v * slope
        t_dz = v.abs() * t_slope + 4 * U * dz.abs()
        chain = (CHAIN + self.x.shape[1] / (64 * 148)) * U
        a, b = dz.sum(1), (dz * xh).sum(1)
        t_a = t_dz.sum(1) + chain * dz.abs().sum(1)
        t_b = (t_dz * xh.abs() + dz.abs() * t_xh).sum(1) + chain * (dz * xh).abs().sum(1)
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
