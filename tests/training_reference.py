"""The training operators in 64 bits, with the error each output may have.

Every bound is first-order arithmetic on the 64-bit values: with u the largest
relative rounding of the 16-bit type (``eps / 2``) and gamma(K) = (K + 8) 2^-23 for
a sum of K products in FP32 (each addition of the tensor cores off by at most
2^-23 of the running sum of magnitudes, rounding or truncating),

* a rounded value v is off by u |v| (and half a step of the smallest subnormal);
* a product P Q of operands off by dP, dQ is off by dP |Q| + |P| dQ + gamma |P| |Q|.

``SLACK`` covers the second-order terms and the FP32 elementwise steps (each a few
2^-23, against u >= 2^-11)."""

from __future__ import annotations

import torch

SLACK = 1.05


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def floor_of(dtype) -> float:
    """Half a step between subnormal numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def gamma(k: int) -> float:
    return (k + 8) * 2.0 ** -23


def rounded(v, err, dtype):
    """The error of a value off by err after rounding to dtype."""
    return err + unit(dtype) * (v.abs() + err) + floor_of(dtype)


def product(p, dp, q, dq):
    """p @ q in FP32 and its error; dp or dq None: exact operands."""
    err = gamma(p.shape[1]) * (p.abs() @ q.abs())
    if dp is not None:
        err = err + dp @ q.abs()
    if dq is not None:
        err = err + p.abs() @ dq
    return p @ q, err


def ffn(x, gate, up, down, dy=None):
    """[(value, error)] of y, and with dy of dx, dgate, dup, ddown."""
    dtype = x.dtype
    x, gate, up, down = (t.detach().double() for t in (x, gate, up, down))
    g, eg = product(x, None, gate.T, None)
    u, eu = product(x, None, up.T, None)
    s = torch.sigmoid(g)
    silu, slope = g * s, s * (1 + g * (1 - s))
    bend = s * (1 - s) * (2 + g * (1 - 2 * s))
    # exp and the reciprocal in FP32: 2^-20 with the argument's rounding, up to |g| of 8.
    fast = 2.0 ** -23 * (8 + g.abs())
    h = silu * u
    eh = rounded(h, slope.abs() * eg * u.abs() + silu.abs() * eu + fast * h.abs(), dtype)
    y, ey = product(h, eh, down.T, None)
    out = [(y, SLACK * rounded(y, ey, dtype))]
    if dy is None:
        return out
    dy = dy.double()
    # The backward pass multiplies by silu(g) and u silu'(g) as kept, rounded.
    es = rounded(silu, slope.abs() * eg + fast * silu.abs(), dtype)
    ed = rounded(u * slope, eu * slope.abs() + u.abs() * (bend.abs() * eg + fast), dtype)
    dh, edh = product(dy, None, down, None)
    du, dg = dh * silu, dh * u * slope
    edu = rounded(du, edh * silu.abs() + dh.abs() * es, dtype)
    edg = rounded(dg, edh * (u * slope).abs() + dh.abs() * ed, dtype)
    a, ea = product(dg, edg, gate, None)
    b, eb = product(du, edu, up, None)
    dx, edx = a + b, ea + eb + gamma(1) * (a.abs() + b.abs())
    pairs = [(dx, edx), product(dg.T, edg.T, x, None), product(du.T, edu.T, x, None), product(dy.T, None, h, eh)]
    return out + [(v, SLACK * rounded(v, e, dtype)) for v, e in pairs]


def loss(x, weight, target, reduction, ignore, dloss=None):
    """[(value, error)] of the loss, and with dloss of dx and dweight."""
    dtype = x.dtype
    x, weight = x.detach().double(), weight.detach().double()
    keep = target != ignore
    at = torch.where(keep, target, torch.zeros_like(target))[:, None]
    z, ez = product(x, None, weight.T, None)
    lse = torch.logsumexp(z, 1, keepdim=True)
    # exp2 of (z - max) log2(e): 2^-22, and the argument's two roundings; a sum of V.
    spread = (z.max(1, keepdim=True).values - z).abs().clamp(max=100.0)
    eexp = 2.0 ** -23 * (4 + 3 * spread)
    p = torch.exp(z - lse)
    # The sum runs per 32 columns, then over these, then over tiles: 32 + V / 32 terms deep at most.
    deep = (40 + z.shape[1] / 32) * 2.0 ** -24
    else_ = (p * (ez + eexp)).sum(1, keepdim=True) + deep + 2.0 ** -22 * (1 + lse.abs())
    tz, et = z.gather(1, at), ez.gather(1, at)
    each = (lse - tz).squeeze(1) * keep
    eeach = (else_ + et + 2.0 ** -22 * (1 + (lse - tz).abs() + (z.max(1, keepdim=True).values - tz).abs())).squeeze(1) * keep
    count = int(keep.sum())
    if reduction == "none":
        out = [(each, SLACK * eeach)]
    else:
        n = count if reduction == "mean" else 1
        v = each.sum() / n
        out = [(v, SLACK * (eeach.sum() / n + 2.0 ** -23 * v.abs()))]
    if dloss is None:
        return out
    scale = dloss.double().expand(len(target)) * keep
    if reduction == "mean":
        scale = scale / max(count, 1)
    top = scale.abs().max()
    d = p.clone()
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    ed = p * (ez + else_ + eexp + 2.0 ** -23 * (4 + lse.abs())) + 2.0 ** -22 * d.abs()
    # dz is stored as 2^14 (p - onehot) row / max row, in 16 bits.
    dz = d * scale[:, None]
    edz = ed * scale[:, None].abs() + unit(dtype) * dz.abs() + floor_of(dtype) * 2.0 ** -14 * top
    edz = edz * keep[:, None]
    more = 2.0 ** -20   # the pieces' FP32 additions and the last factor
    pairs = [product(dz, edz, weight, None), product(dz.T, edz.T, x, None)]
    return out + [(v, SLACK * rounded(v, e + more * v.abs() + 64 * 2.0 ** -24 * e, dtype)) for v, e in pairs]


def step_values(s, coefficients, steps):
    """The singular values after each step."""
    a, b, c = coefficients
    seen = [s]
    for _ in range(steps):
        s = s * (a + s ** 2 * (b + c * s ** 2))
        seen.append(s)
    return seen


def orthogonalize(g, steps, coefficients, eps):
    """(value, bound on the Frobenius norm of the error), for one matrix.

    The steps are one odd function f of the singular values, U f(S) V^T. An error E
    brought in after step k comes out as at most amp_k |E|, with amp_k the largest
    divided difference of the remaining steps' function over all pairs of (signed)
    singular values (and f(s) / s towards the longer side's other directions):
    that is the derivative of such a function. A step brings in what its three
    products and roundings are off by (u and gamma as above, in FP16 inside)."""
    dtype = g.dtype
    x = g.double()
    x = x / (torch.linalg.vector_norm(x) + eps)
    u, s, vt = torch.linalg.svd(x, full_matrices=False)
    seen = step_values(s, coefficients, steps)
    value = u @ torch.diag(seen[-1]) @ vt
    a, b, c = (abs(v) for v in coefficients)
    half = unit(torch.float16)
    long = max(g.shape)
    n = len(s)

    def amp(k):
        now, end = seen[k], seen[-1]
        signed = torch.cat([now, -now])
        image = torch.cat([end, -end])
        near = signed[:, None] - signed[None, :]
        rise = (image[:, None] - image[None, :]).abs() / near.abs().clamp(min=1e-9)
        rise = torch.where(near.abs() < 1e-6, torch.zeros_like(rise), rise)
        # Where two values are closer than that, the derivative itself.
        slope = torch.ones_like(now)
        for q in range(k, steps):
            v = seen[q]
            slope = slope * (coefficients[0] + 3 * coefficients[1] * v ** 2 + 5 * coefficients[2] * v ** 4)
        side = (end / now.clamp(min=1e-12)).abs().max()
        return float(torch.stack([rise.max(), slope.abs().max(), side]).max())

    fro = [float(torch.linalg.vector_norm(v)) for v in seen]
    # Half a subnormal step of FP16 at the scale of 2^8 for X, 1 for the products.
    dust_x = floor_of(torch.float16) * 2.0 ** -8 * (g.numel() ** 0.5)
    dust_p = floor_of(torch.float16) * n
    total = amp(0) * (half * fro[0] + dust_x + 2.0 ** -22 * fro[0])
    for k in range(steps):
        v = seen[k]
        top = float(v.max())
        gram = float(torch.linalg.vector_norm(v ** 2))
        # |X| |X|^T elementwise is at most |X|_F^2 in norm, and so on for the sums.
        egram = half * gram + gamma(long) * fro[k] ** 2 + dust_p
        epoly = half * (b * gram + c * float(torch.linalg.vector_norm(v ** 4))) + \
            egram * (b + 2 * c * top ** 2) + gamma(n) * c * gram ** 2 + dust_p
        poly = b * gram + c * float(torch.linalg.vector_norm(v ** 4))
        enext = epoly * top + gamma(n) * poly * fro[k] + 2.0 ** -22 * (a + b + c) * fro[k]
        if k + 1 < steps:
            enext += half * fro[k + 1] + dust_x
        total += amp(k + 1) * enext
    total += unit(dtype) * fro[-1] + floor_of(dtype) * g.numel() ** 0.5
    return value, SLACK * total
