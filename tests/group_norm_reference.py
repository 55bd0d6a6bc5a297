"""Group norm with an activation function in 64 bits, and bounds on what fp32 leaves of it.  Tensors are [N, P, C]; the CPU, without the package."""
import torch

import q8_reference as ref

U = 2.0 ** -24


def act(z, kind):
    """Value and slope."""
    return (z, torch.ones_like(z)) if kind is None else ref.act(z, kind)


def held(x):
    """What the checkpoint of rows x stands for."""
    return ref.held(x.reshape(-1, x.shape[-1])).reshape(x.shape)


def split(t, groups):
    return t.unflatten(-1, (groups, -1))


def outputs(x, kept, dy, w, b, groups, eps, kind):
    """y, mean, rstd, dx, dw, db: statistics of x, the backward pass from kept."""
    g = split(x, groups)
    mu = g.mean(dim=(1, 3), keepdim=True)
    r = 1.0 / torch.sqrt(((g - mu) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    w, b = w.view(groups, -1), b.view(groups, -1)
    y = act((g - mu) * r * w + b, kind)[0]
    h = (split(kept, groups) - mu) * r
    dz = split(dy, groups) * act(h * w + b, kind)[1]
    u = dz * w
    dx = r * (u - u.mean(dim=(1, 3), keepdim=True) - h * (u * h).mean(dim=(1, 3), keepdim=True))
    return (y.flatten(2), mu[:, 0, :, 0], r[:, 0, :, 0], dx.flatten(2), (dz * h).sum(dim=(0, 1)).view(-1), dz.sum(dim=(0, 1)).view(-1))


def errors(x, kept, dy, w, b, groups, eps, kind, dtype):
    """Bounds on the fp32 error of the outputs.

    A sum over a group goes through at most 64 + P / 8 roundings a term: a thread's rows (8, or P over the threads of a row and the tiles), the threads'
    and wavefronts' joins, the group's channels by eight lanes, the tiles by eight lanes.  A thread sums differences from its
    first value, at most twice the group's largest deviation, and their squares.  The slope of the activation functions changes by at
    most as much as its argument (the second derivatives are at most 0.8), the value by 1.13 times it."""
    p = x.shape[1]
    k = 64 + p // 8
    g = split(x, groups)
    mean = dict(dim=(1, 3), keepdim=True)
    mu = g.mean(**mean)
    d = (g - mu).abs()
    far = d.amax(dim=(1, 3), keepdim=True)
    var = (d ** 2).mean(**mean)
    r = 1.0 / torch.sqrt(var + eps)
    e_mu = k * U * (g.abs().mean(**mean) + 2 * far)
    e_var = 2 * far * (e_mu + U * far) + e_mu ** 2 + k * U * 4 * far ** 2
    rho = 0.5 * e_var * r * r + 4 * U
    w, b = w.view(groups, -1), b.view(groups, -1)

    def z_of(v):
        h = (v - mu) * r
        e_h = h.abs() * (rho + 3 * U) + r * e_mu
        return h, e_h, h * w + b, w.abs() * e_h + 3 * U * ((h * w).abs() + (h * w + b).abs())

    def of_act(z, e_z, which):
        if kind is None:
            return e_z if which == 0 else torch.zeros_like(z)
        value, slope = ref.act_error(z, kind, dtype)
        return value + 1.13 * e_z if which == 0 else slope + e_z

    h, e_h, z, e_z = z_of(g)
    e_y = of_act(z, e_z, 0)
    h, e_h, z, e_z = z_of(split(kept, groups))
    slope, dy = act(z, kind)[1], split(dy, groups)
    dz, e_dz = dy * slope, dy.abs() * (of_act(z, e_z, 1) + 2 * U * slope.abs())
    u, e_u = dz * w, w.abs() * (e_dz + 2 * U * dz.abs())
    s1, s2 = u.mean(**mean), (u * h).mean(**mean)
    e1 = e_u.mean(**mean) + (k + 2) * U * u.abs().mean(**mean)
    e_uh = u.abs() * e_h + e_u * (h.abs() + e_h)
    e2 = e_uh.mean(**mean) + (k + 4) * U * (u * h).abs().mean(**mean)
    inner = u - s1 - h * s2
    e_dx = r * (6 * U * (u.abs() + s1.abs() + (h * s2).abs()) + e_u + e1 + h.abs() * e2 + e_h * (s2.abs() + e2)
                + (u.abs() + s1.abs() + (h * s2).abs()) * rho) + inner.abs() * r * (rho + 2 * U)
    n = k + x.shape[0] + 80
    e_dw = (dz.abs() * e_h + e_dz * (h.abs() + e_h)).sum(dim=(0, 1)) + n * U * (dz * h).abs().sum(dim=(0, 1))
    e_db = e_dz.sum(dim=(0, 1)) + n * U * dz.abs().sum(dim=(0, 1))
    return e_y.flatten(2), e_mu[:, 0, :, 0], (r * rho)[:, 0, :, 0], e_dx.flatten(2), e_dw.view(-1), e_db.view(-1)
