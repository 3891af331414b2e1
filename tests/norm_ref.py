"""64-bit formulas of the group norm and of the 8-bit product, for the tests."""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
E32 = 2.0 ** -24


def act(z, name, slope=0.1):
    if name == 'leaky':
        return torch.where(z > 0, z, z * slope)
    return z * torch.sigmoid(z) if name == 'silu' else z


def act_grad(z, name, slope=0.1):
    if name == 'leaky':
        return torch.where(z > 0, 1.0, slope).to(z.dtype)
    if name == 'silu':
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


class GroupNormRef:
    """Everything in float64 on the CPU, channels first: y, z, xhat, rstd, and with dy the gradients; err_* are what fp32
    arithmetic may be off by (64 roundings of the largest term of each sum)."""

    def __init__(self, x, groups, weight, bias, eps, name, slope=0.1, dy=None):
        b, c = x.shape[:2]
        v = x.detach().cpu().double().reshape(b, groups, -1)
        shape = (1, c) + (1,) * (x.dim() - 2)
        g = torch.ones(c).double() if weight is None else weight.detach().cpu().double()
        h = torch.zeros(c).double() if bias is None else bias.detach().cpu().double()
        self.mean = v.mean(2)
        self.rstd = 1 / torch.sqrt(((v - self.mean[..., None]) ** 2).mean(2) + eps)
        self.xhat = ((v - self.mean[..., None]) * self.rstd[..., None]).reshape(x.shape)
        g, h = g.reshape(shape), h.reshape(shape)
        self.z = self.xhat * g + h
        self.y = act(self.z, name, slope)
        spread = (v.abs().amax(2) * self.rstd)[..., None].expand(v.shape).reshape(x.shape)  # max |x| in deviations
        self.err_y = 64 * E32 * (spread * g.abs() + h.abs() + self.z.abs())
        if dy is None:
            return
        dims = [0] + list(range(2, x.dim()))
        dz = dy.detach().cpu().double() * act_grad(self.z, name, slope)
        self.dgamma, self.dbeta = (dz * self.xhat).sum(dims), dz.sum(dims)
        t = (dz * g).reshape(v.shape)
        u = self.xhat.reshape(v.shape)
        r = self.rstd[..., None]
        self.dx = (r * (t - t.mean(2, keepdim=True) - u * (t * u).mean(2, keepdim=True))).reshape(x.shape)
        # dz is off by act'' (below 1) times what z is off, and xhat by what x - mean is
        ddz = dy.detach().cpu().double().abs() * (64 * E32) * (1 + spread * g.abs() + h.abs())
        self.err_dbeta = ddz.sum(dims) + 64 * E32 * dz.abs().sum(dims)
        self.err_dgamma = (ddz * self.xhat.abs() + dz.abs() * 64 * E32 * (1 + spread + self.xhat.abs())).sum(dims)
        top = (ddz * g.abs() + 64 * E32 * (dz * g).abs()).reshape(v.shape).amax(2, keepdim=True)
        big = t.abs().amax(2, keepdim=True)
        off = 64 * E32 * (1 + spread.reshape(v.shape))
        self.err_dx = (r * (top * (2 + u.abs() * u.abs().amax(2, keepdim=True)) + big * off * (1 + 2 * u.abs().amax(2, keepdim=True)))).reshape(x.shape)


def close(got, want, err, what):
    """|got - want| <= err + half a step of got's type."""
    u = U[got.dtype]
    g = got.detach().cpu().double()
    tiny = 2.0 ** -25 if got.dtype is torch.float16 else 0.0  # half a step of fp16's subnormals
    far = (g - want).abs() - (err + u * want.abs() * (1 + 2 * u) + tiny)
    assert g.shape == want.shape and bool(torch.isfinite(g).all()), '%s: shape %s, finite %s' % (what, tuple(g.shape), bool(torch.isfinite(g).all()))
    assert float(far.max()) <= 0, '%s: off by %g more than allowed (max difference %g)' % (what, float(far.max()), float((g - want).abs().max()))
