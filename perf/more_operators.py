"""Workloads of the group normalisation and 8-bit activation operators, for timing and comparing.

``listed()`` names them, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run``
makes one pass: in elementary fp32 torch operations, or, where the module's
``own`` is true, through ``rdna4_conv3d``. ``exact`` is the definition in
64 bits, ``work`` the bytes and operations that a pass cannot do without.

Two operators:

* ``group_norm`` -- act(group_norm(x) * weight + bias) of a channels-last
  activation; with ``train`` also the gradients of x, weight and bias for a
  given gradient of the output. With ``keep`` the backward pass has x in 8
  bits only: it is taken at the values that those hold, with the statistics
  of x itself.
* ``eight_bit`` -- an activation written in 8 bits for the backward pass and
  read back. Every 32 elements, in memory order, share the power of two 2^e
  with the smallest e >= -127 that brings their largest finite magnitude to
  at most 127 (``int8``: whole numbers) or 448 (``e4m3``: 8-bit floating
  point); x / 2^e is rounded to the nearest, ties to even. What is read back
  is the code times 2^e in x's type, at most its largest finite number.
"""
import os
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-conv3d-wmma_b200")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5
_SLOPE = 0.01
_BLOCK = 32


def _gn(n, c, d, h, w, groups, dtype, act, train=False, keep=""):
    return dict(op="group_norm", n=n, c=c, d=d, h=h, w=w, groups=groups, dtype=dtype, act=act, train=train, keep=keep)


def _q8(n, c, d, h, w, dtype, keep):
    return dict(op="eight_bit", n=n, c=c, d=d, h=h, w=w, groups=1, dtype=dtype, act="none", train=False, keep=keep)


def listed():
    return [
        # the deepest level of one small patch, answered by a server: latency counts
        dict(_gn(1, 192, 4, 8, 8, 8, "bf16", "silu"), name="gn patch"),
        # the first level of the segmentation network on its benchmark volume, predicting
        dict(_gn(4, 24, 64, 128, 128, 8, "bf16", "relu"), name="gn volume"),
        # a scan of odd extents, channels that are no multiple of a vector
        dict(_gn(2, 30, 37, 41, 53, 6, "fp16", "gelu"), name="gn odd"),
        # training: the network's four levels, deepest to first
        dict(_gn(4, 192, 8, 16, 16, 8, "bf16", "silu", train=True), name="gn train level 3"),
        dict(_gn(4, 48, 32, 64, 64, 8, "fp16", "relu", train=True), name="gn train level 1"),
        dict(_gn(4, 24, 64, 128, 128, 8, "bf16", "silu", train=True), name="gn train level 0"),
        # many small patches, each channel a group of its own
        dict(_gn(64, 96, 6, 6, 6, 96, "bf16", "leaky_relu", train=True), name="gn train patches"),
        # full precision, odd extents
        dict(_gn(2, 32, 33, 47, 50, 4, "fp32", "gelu", train=True), name="gn train fp32"),
        # the first level with its input kept in 8 bits
        dict(_gn(4, 24, 64, 128, 128, 8, "bf16", "silu", train=True, keep="int8"), name="gn train level 0 kept"),
        # a ragged volume, kept in 8-bit floating point
        dict(_gn(3, 40, 21, 35, 45, 10, "fp16", "relu", train=True, keep="e4m3"), name="gn train ragged kept"),
        # the decoder's concatenation, input of the widest layer, kept until its weight gradient
        dict(_q8(4, 48, 64, 128, 128, "bf16", "int8"), name="8 bit concatenation"),
        # a small odd activation in full precision: latency counts
        dict(_q8(1, 33, 9, 23, 29, "fp32", "e4m3"), name="8 bit small"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    # channels: the network's own, multiples of 8, or any number
    c = rng.choice((rng.choice((24, 48, 96, 192)), 8 * log_int(1, 48), log_int(1, 200)))
    most = 1 << 25                                       # elements of a drawn case: a third of the first level's
    n = rng.choice((1, 2, 4, log_int(1, 64)))
    vox = log_int(8, max(8, min(1 << 20, most // (n * c))))
    w = min(vox, log_int(2, 130))
    h = max(1, min(vox // w, log_int(2, 130)))
    d = max(1, vox // (w * h))
    if rng.random() < 0.25:
        return _q8(n, c, d, h, w, dtype, rng.choice(("int8", "e4m3")))
    groups = rng.choice([g for g in range(1, c + 1) if c % g == 0])
    train = rng.random() < 0.7
    keep = rng.choice(("", "int8", "e4m3")) if train else ""
    act = rng.choice(("none", "relu", "leaky_relu", "silu", "gelu"))
    return _gn(n, c, d, h, w, groups, dtype, act, train, keep)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    kw = dict(device=dev, generator=g)
    n, c, d, h, w = (case[k] for k in ("n", "c", "d", "h", "w"))
    dt = _DTYPES[case["dtype"]]
    # a convolution's outputs: channels of different spread and centre
    spread = torch.exp(torch.randn(c, **kw) * 0.5)
    centre = torch.randn(c, **kw)
    x = torch.randn((n, d, h, w, c), dtype=dt, **kw)
    x.mul_(spread.to(dt)).add_(centre.to(dt))
    if case["op"] == "eight_bit":                        # an activation's outputs: none below 0
        x.relu_()
    x = x.permute(0, 4, 1, 2, 3)
    state = dict(case=dict(case), x=x)
    if case["op"] == "group_norm":
        state["weight"] = 1.0 + 0.2 * torch.randn(c, **kw)
        state["bias"] = 0.2 * torch.randn(c, **kw)
    if case["train"]:
        # fp16 trains with a loss scale, so do the gradients come in
        dy = torch.randn((n, d, h, w, c), dtype=dt, **kw).mul_(0.25 if dt == torch.float16 else 2.0 ** -10)
        state["dy"] = dy.permute(0, 4, 1, 2, 3)
        for k in ("x", "weight", "bias"):
            state[k].requires_grad_(True)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "eight_bit":
        return _run_eight_bit(state, case) if own else _from_blocks(state["x"], case["keep"])
    return _run_group_norm(state, case) if own else _plain_group_norm(state, case)


def _run_eight_bit(s, case):
    from rdna4_conv3d.checkpoint8 import pack8, unpack8
    return unpack8(pack8(s["x"], case["keep"]))


def _run_group_norm(s, case):
    from rdna4_conv3d.group_norm import group_norm_act
    y = group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], _EPS, activation=case["act"],
                       negative_slope=_SLOPE, checkpoint=case["keep"] or None)
    if not case["train"]:
        return y
    dx, dw, db = torch.autograd.grad((y,), (s["x"], s["weight"], s["bias"]), (s["dy"],))
    return dict(y=y, dx=dx, dweight=dw, dbias=db)


def _by_group(t, groups):
    """(N, C, D, H, W) channels last -> (N, voxels, groups, channels of a group)."""
    n, c = t.shape[:2]
    return t.detach().permute(0, 2, 3, 4, 1).reshape(n, -1, groups, c // groups)


def _back(t, like):
    """The reverse of _by_group, in the activation's own type."""
    n, c, d, h, w = like.shape
    return t.to(like.dtype).reshape(n, d, h, w, c).permute(0, 4, 1, 2, 3)


def _power_of_two(exponent):
    """2^exponent as fp32, exactly, for exponents from -127 to 127."""
    bits = torch.where(exponent == -127, 1 << 22, (exponent + 127) << 23)
    return bits.to(torch.int32).view(torch.float32)


def _from_blocks(x, keep):
    """x as its 8 bits hold it, in x's type."""
    most, top, least = (127.0, 7, 127.0 / 128) if keep == "int8" else (448.0, 9, 0.875)
    xl = x.detach().permute(0, 2, 3, 4, 1)
    flat = xl.reshape(-1).float()
    count = flat.numel()
    b = torch.nn.functional.pad(flat, (0, -count % _BLOCK)).reshape(-1, _BLOCK)
    finite = b.abs() < float("inf")
    m, e = torch.frexp(torch.where(finite, b.abs(), 0.0).amax(1, keepdim=True))
    e = torch.where(m == 0, -127, e - top + (m > least)).clamp(min=-127).to(torch.int32)
    q = b * _power_of_two(-e)
    if keep == "int8":
        q = torch.round(q).clamp(-most, most)
    else:
        q = q.to(torch.float8_e4m3fn).float()
    v = torch.where(finite, q * _power_of_two(e), float("nan"))
    limit = torch.finfo(x.dtype).max
    v = v.clamp(-limit, limit).reshape(-1)[:count].to(x.dtype)
    return v.reshape(xl.shape).permute(0, 4, 1, 2, 3)


def _act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "leaky_relu":
        return torch.where(z > 0, z, z * _SLOPE)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.7071067811865476))
    return z


def _act_slope(z, name):
    if name == "relu":
        return torch.where(z > 0, 1.0, 0.0)
    if name == "leaky_relu":
        return torch.where(z > 0, 1.0, _SLOPE)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    return torch.ones_like(z)


def _plain_group_norm(s, case):
    x, groups, act = s["x"], case["groups"], case["act"]
    w = s["weight"].detach().reshape(groups, -1)
    b = s["bias"].detach().reshape(groups, -1)
    xr = _by_group(x, groups).float()
    m = xr.shape[1] * xr.shape[3]
    # long sums in 64 bits
    mean = (xr.sum((1, 3), keepdim=True, dtype=torch.float64) / m).float()
    diff = xr - mean
    var = (diff * diff).sum((1, 3), keepdim=True, dtype=torch.float64) / m
    rstd = (1.0 / torch.sqrt(var + _EPS)).float()
    y = _back(_act(diff * rstd * w + b, act), x)
    if not case["train"]:
        return y
    if case["keep"]:
        diff = _by_group(_from_blocks(x, case["keep"]), groups).float() - mean
    xh = diff * rstd
    dz = _by_group(s["dy"], groups).float() * _act_slope(xh * w + b, act)
    dweight = (dz * xh).sum((0, 1), dtype=torch.float64)
    dbias = dz.sum((0, 1), dtype=torch.float64)
    gz = dz * w
    mean_g = (gz.sum((1, 3), keepdim=True, dtype=torch.float64) / m).float()
    mean_gx = ((gz * xh).sum((1, 3), keepdim=True, dtype=torch.float64) / m).float()
    dx = (gz - mean_g - xh * mean_gx) * rstd
    return dict(y=y, dx=_back(dx, x), dweight=dweight.float().reshape(-1), dbias=dbias.float().reshape(-1))


def _exact_eight_bit(x, keep):
    """Codes from logarithms and divisions in 64 bits; (N, D, H, W, C)."""
    xl = x.detach().permute(0, 2, 3, 4, 1).contiguous()
    flat = xl.reshape(-1)
    out = torch.empty(flat.numel(), dtype=torch.float64, device=x.device)
    most = 127.0 if keep == "int8" else 448.0
    step = 1 << 25                                       # a multiple of a block
    for a in range(0, flat.numel(), step):
        v = flat[a:a + step].double()
        count = v.numel()
        v = torch.cat([v, v.new_zeros(-count % _BLOCK)]).reshape(-1, _BLOCK)
        big = v.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(big.clamp(min=2.0 ** -140) / most)) - 1
        for _ in range(3):                               # the logarithm may be off by its rounding
            e = torch.where(big > most * torch.exp2(e), e + 1, e)
        e = e.clamp(min=-127.0)
        unit = torch.exp2(e)
        u = v / unit
        if keep == "e4m3":                               # 3 bits behind the leading one, spacing 2^-9 below 2^-6
            low = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))
            low = torch.where(torch.exp2(low) > u.abs().clamp(min=2.0 ** -6), low - 1, low)
            unit8 = torch.exp2(low - 3)
            u = torch.round(u / unit8) * unit8
        else:
            u = torch.round(u)
        limit = torch.finfo(x.dtype).max
        out[a:a + count] = (u * unit).clamp(-limit, limit).reshape(-1)[:count]
    return out.reshape(xl.shape)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].detach()
    n, c, d, h, w_ = x.shape
    kept = _exact_eight_bit(x, case["keep"]) if case["keep"] else None
    if case["op"] == "eight_bit":
        return kept.permute(0, 4, 1, 2, 3)
    acts = dict(none=lambda t: t, relu=torch.relu, silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu,
                leaky_relu=lambda t: torch.nn.functional.leaky_relu(t, _SLOPE))
    act, groups = acts[case["act"]], case["groups"]
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    y = torch.empty((n, d, h, w_, c), dtype=torch.float64, device=x.device)
    dx, dw, db = torch.empty_like(y), torch.zeros_like(w), torch.zeros_like(w)
    for i in range(n):
        xi = x[i].movedim(0, -1).double().reshape(-1, c)
        m = xi.shape[0] * (c // groups)

        def mean_of(t):
            """(voxels, C) -> the mean over each channel's group, (C,)."""
            return (t.sum(0).reshape(groups, -1).sum(1) / m).repeat_interleave(c // groups)

        mu = mean_of(xi)
        r = (mean_of((xi - mu) ** 2) + _EPS) ** -0.5
        y[i] = act((xi - mu) * r * w + b).reshape(d, h, w_, c)
        if case["train"]:
            xi = kept[i].reshape(-1, c) if kept is not None else xi
            xh = (xi - mu) * r
            z = (xh * w + b).requires_grad_(True)
            dz, = torch.autograd.grad(act(z), z, s["dy"][i].movedim(0, -1).reshape(-1, c).double())
            dw += (dz * xh).sum(0)
            db += dz.sum(0)
            dx[i] = (r * (dz * w - mean_of(dz * w) - xh * mean_of(dz * w * xh))).reshape(d, h, w_, c)
    y = y.permute(0, 4, 1, 2, 3)
    if not case["train"]:
        return y
    return dict(y=y, dx=dx.permute(0, 4, 1, 2, 3), dweight=dw, dbias=db)


def work(case):
    elems = case["n"] * case["c"] * case["d"] * case["h"] * case["w"]
    size = _BYTES[case["dtype"]]
    coded = elems + -(-elems // _BLOCK)                  # codes and one exponent for every 32
    if case["op"] == "eight_bit":
        # read, written in 8 bits; those read, written back; a maximum, a scaling and a rounding each way
        return {"bytes": 2 * elems * size + 2 * coded, "flops": 5 * elems}
    b = 2 * elems * size + 8 * case["c"]
    f = 10 * elems                                       # sum, square, normalisation, activation
    if case["train"]:
        # backward: dy and x (or its 8 bits) read, dx written
        b += 2 * elems * size + 16 * case["c"] + (2 * coded if case["keep"] else elems * size)
        f += 20 * elems
    return {"bytes": b, "flops": f}
