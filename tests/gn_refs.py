"""Group normalisation with an activation and 8-bit blocks in 64 bits, with the bounds that their tests use.

The bounds count: half a step of the result's type, and K = 64 units of 2^-24 of the magnitudes that the fp32
arithmetic adds up. The longest fp32 chain is a thread's own sum (some hundred terms, whose errors grow like the square
root for the random terms used here); the hardware's exponential and reciprocal behind 16-bit results are good to 2^-21 =
8 units. A slope with a step at 0 (relu, leaky_relu) may fall on either side where z is within its own error of 0.
"""
import torch
import torch.nn.functional as F

K = 64 * 2.0 ** -24
CL = torch.channels_last_3d


def act64(z, act, slope):
    return {"none": lambda: z, "relu": lambda: torch.relu(z), "leaky_relu": lambda: F.leaky_relu(z, slope),
            "silu": lambda: F.silu(z), "gelu": lambda: F.gelu(z)}[act]()


def half_step(v, dtype):
    """The most by which rounding v to dtype moves it."""
    info = torch.finfo(dtype)
    return v.abs() * (info.eps / 2) + info.smallest_normal * info.eps / 2


def ref(x, groups, w, b, eps, act, slope, dy=None, kept=None):
    """dict of (value, bound) in 64 bits for y and, with dy, dx, dw, db; ``kept``: what 8 bits hold of x."""
    n, c = x.shape[:2]
    each = (1, c) + (1,) * (x.dim() - 2)
    xd = x.detach().double()
    wd = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    bd = torch.zeros_like(wd) if b is None else b.detach().double()
    wd, bd = wd.reshape(each), bd.reshape(each)

    def over(t, f):
        """f over a sample's group, as wide as t."""
        v = f(t.reshape(n, groups, -1), -1, True)
        return v.expand(n, groups, t.numel() // max(1, n * groups)).reshape(t.shape)

    mean = over(xd, torch.mean)
    rstd = (over((xd - mean) ** 2, torch.mean) + eps) ** -0.5

    def z_of(t):
        xh = (t - mean) * rstd
        # fp32 mean (half a unit of |mean|) and rstd, the product and sum
        return xh, xh * wd + bd, K * ((xh * wd).abs() + bd.abs()) + 2.0 ** -22 * (mean * rstd * wd).abs()

    xh, z, dz_err = z_of(xd)
    y = act64(z, act, slope)
    out = {"y": (y, half_step(y, x.dtype) + 1.2 * dz_err + K * y.abs())}
    if dy is None:
        return out
    if kept is not None:
        xh, z, dz_err = z_of(kept.detach().double())
    xh_err = K * xh.abs() + 2.0 ** -22 * (mean * rstd).abs()
    zz = z.clone().requires_grad_(True)
    slope_of, = torch.autograd.grad(act64(zz, act, slope).sum(), zz)
    gy = dy.detach().double()
    dz = gy * slope_of
    # |act''| <= 1 for silu and gelu; a step where z may be on the other side of 0
    step = {"relu": 1.0, "leaky_relu": abs(1.0 - slope)}.get(act, 0.0)
    dz_e = gy.abs() * (dz_err + K * (1.0 + z.abs()) + torch.where(z.abs() <= dz_err, step, 0.0))
    dims = (0, *range(2, x.dim()))
    g, ge = dz * wd, dz_e * wd.abs()
    a, bb = over(g, torch.mean), over(g * xh, torch.mean)
    a_e = over(ge + K * g.abs(), torch.mean)
    b_e = over(ge * xh.abs() + g.abs() * xh_err + K * (g * xh).abs(), torch.mean)
    dx = rstd * (g - a - xh * bb)
    dx_e = rstd * (ge + a_e + xh.abs() * b_e + xh_err * bb.abs() + K * (g.abs() + a.abs() + (xh * bb).abs()))
    out["dx"] = (dx, half_step(dx, x.dtype) + dx_e)
    for name, t, p in (("dw", dz * xh, w), ("db", dz, b)):
        if p is not None:
            e = dz_e * (xh.abs() if name == "dw" else 1.0) + K * t.abs() + (dz.abs() * xh_err if name == "dw" else 0.0)
            v = t.sum(dims)
            out[name] = (v, half_step(v, p.dtype) + e.sum(dims))
    return out


def check(got, want, names=None):
    for k, (v, bound) in want.items():
        if names is not None and k not in names:
            continue
        t = got[k].detach().double()
        d = (t - v).abs()
        # beyond its type's range a value rounds to infinity (a group of one element has rstd = eps^-1/2 = 316, and with
        # x in 8 bits xh = 316 (x8 - x): dx = -rstd g xh^2 passes 65504)
        d = torch.where(t.isinf() & (t.sign() == v.sign()) & (v.abs() + bound >= torch.finfo(got[k].dtype).max), 0.0, d)
        worst = (d - bound).max().item() if d.numel() else 0.0
        assert d.numel() == 0 or bool((d <= bound).all()), f"{k}: {worst:.3e} beyond its bound"


def blocks64(flat, fmt):
    """What 8 bits hold of a flat tensor, in 64 bits and before it is rounded to its type; NaN where not finite."""
    v = flat.detach().double()
    count = v.numel()
    v = torch.cat([v, v.new_zeros(-count % 32)]).reshape(-1, 32)
    most = 127.0 if fmt == "int8" else 448.0
    finite = v.isfinite()
    u = torch.where(finite, v, 0.0)
    big = u.abs().amax(1, keepdim=True)
    e = torch.full_like(big, -127.0)
    for _ in range(260):                                 # the least exponent, by its definition
        e = torch.where(big > most * torch.exp2(e), e + 1, e)
    q = u / torch.exp2(e)
    if fmt == "int8":
        q = torch.round(q)
    else:
        _, k = torch.frexp(q.abs().clamp(min=2.0 ** -6))
        ulp = torch.exp2(k.double() - 4)                 # three bits behind the leading one
        q = torch.round(q / ulp) * ulp
    return torch.where(finite, q * torch.exp2(e), float("nan")).reshape(-1)[:count]


def held(x, fmt):
    """What 8 bits hold of a channels-last x, in x's type."""
    last = x.detach().movedim(1, -1).contiguous()
    limit = torch.finfo(x.dtype).max
    v = blocks64(last.reshape(-1), fmt).clamp(-limit, limit).to(x.dtype)
    return v.reshape(last.shape).movedim(-1, 1)
