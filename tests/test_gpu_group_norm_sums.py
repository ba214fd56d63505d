"""Group norm where sums cancel: activations far from zero, groups without a spread, gradients that nearly vanish.

u = 2^-24 is half a step of fp32. What the kernels may be off by: the mean (one rounding: u |mean|), rstd (u), a
product or sum each (u), and fp32 sums of one thread, at most 64 terms at these sizes, each addition off by at most u of
the sum of magnitudes. Beyond a thread sums are taken in 64 bits, which loses nothing that would show here.
"""
import pytest
import torch

import gn_refs as R
from rdna4_conv3d import _native
from rdna4_conv3d.checkpoint8 import Packed8, unpack8
from rdna4_conv3d.group_norm import group_norm_act

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
CHAIN = 64 * U


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _last(t):
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def _over(t, groups):
    n = t.shape[0]
    m = t.reshape(n, groups, -1).mean(-1, keepdim=True)
    return m.expand(n, groups, t.numel() // (n * groups)).reshape(t.shape)


def _affine_check(x, groups, w, b, dy, fmt=None, eps=1e-5):
    """y, dx, dw, db of act 'none' against 64 bits, with bounds of arithmetic on x - mean."""
    x, w, b = (t.detach().requires_grad_(True) for t in (x, w, b))
    y = group_norm_act(x, groups, w, b, eps, checkpoint=fmt)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)), y=y)
    each = (1, x.shape[1]) + (1,) * (x.dim() - 2)
    dims = (0, *range(2, x.dim()))
    xd, g = x.detach().double(), dy.double()
    wd, bd = w.detach().double().reshape(each), b.detach().double().reshape(each)
    mean = _over(xd, groups)
    rstd = (_over((xd - mean) ** 2, groups) + eps) ** -0.5
    shift = U * (mean * rstd).abs()                      # of every xh: the mean's rounding
    xh = (xd - mean) * rstd
    want = {"y": (xh * wd + bd, R.half_step(xh * wd + bd, x.dtype) + (shift + 4 * U * xh.abs()) * wd.abs() + 2 * U * bd.abs())}
    kept = xd if fmt is None else R.held(x, fmt).double()
    xh = (kept - mean) * rstd
    xh_e = shift + 4 * U * xh.abs()
    gw = g * wd
    a, c = _over(gw, groups), _over(gw * xh, groups)
    # sums of a thread and of a channel's parts times w (one rounding each)
    a_e = _over(gw.abs(), groups) * (CHAIN + 4 * U)
    c_e = _over(gw.abs() * xh_e + (CHAIN + 4 * U) * (gw * xh).abs(), groups)
    dx = rstd * (gw - a - xh * c)
    dx_e = rstd * (a_e + xh.abs() * c_e + xh_e * c.abs() + 8 * U * (gw.abs() + a.abs() + (xh * c).abs()))
    want["dx"] = dx, R.half_step(dx, x.dtype) + dx_e
    dw = (g * xh).sum(dims)
    want["dw"] = dw, ((CHAIN + 4 * U) * (g * xh).abs() + g.abs() * xh_e).sum(dims) + R.half_step(dw, w.dtype)
    db = g.sum(dims)
    want["db"] = db, CHAIN * g.abs().sum(dims) + R.half_step(db, b.dtype)
    R.check(got, want)


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (1, 24, 24, 60, 40), (2, 25, 9, 20, 21), (2, 24, 64, 128, 128)])
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype,centre,spread", [(HF, 1000.0, 2.0), (BF, 500.0, 4.0), (HF, -300.0, 0.25), (FP, 1000.0, 0.25)])
def test_far_from_zero_gradients(cuda_ready, shape, fmt, dtype, centre, spread):
    """|mean| hundreds of spreads, gradients of one sign: sum dz x and mean sum dz nearly cancel."""
    c, kw = shape[1], dict(device="cuda", generator=_gen(11))
    x = _last((centre + spread * torch.randn(shape, **kw)).to(dtype))
    dy = _last((0.3 + 0.05 * torch.randn(shape, **kw)).to(dtype))
    w, b = 1 + 0.2 * torch.randn(c, **kw), 0.2 * torch.randn(c, **kw)
    _affine_check(x, c if c == 25 else 8, w, b, dy, fmt)


@pytest.mark.parametrize("shape,groups", [((1, 2048, 7001), 2048), ((1, 2040, 6000), 255), ((1, 4104, 3000), 8)])
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_widest_rows(cuda_ready, shape, groups, fmt):
    """As many channels as a block has threads for, in two passes: the largest tables in shared memory."""
    c, kw = shape[1], dict(device="cuda", generator=_gen(15))
    x, dy = (_last(torch.randn(shape, **kw).to(BF)) for _ in range(2))
    _affine_check(x, groups, 1 + 0.2 * torch.randn(c, **kw), 0.2 * torch.randn(c, **kw), dy, fmt)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("places", [(0, 1, 3), (0, 2, 3), (1, 2, 3), (0, 1, 2)])
@pytest.mark.parametrize("voxels", [4, 20000])
def test_sums_of_threads_in_64_bits(cuda_ready, dtype, places, voxels):
    """db = 2^30 + 1 - 2^30, dw likewise, from voxels of different threads (the rest 0, and xh = 1 in them)."""
    c = 8
    x = torch.zeros(1, voxels, c, device="cuda")
    x[:, ::2], x[:, 1::2] = 1.0, -1.0                    # mean 0, rstd 1 (eps 0)
    x[:, :4] = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda").reshape(4, 1)
    at = [p * voxels // 4 for p in places]
    dy = torch.zeros(1, voxels, c, device="cuda")
    sign = x[0, :, 0].clone()
    for i, v in zip(at, (2.0 ** 30, 1.0, -2.0 ** 30)):
        dy[0, i] = v
    x, dy = (t.to(dtype).movedim(-1, 1) for t in (x, dy))
    w = torch.ones(c, device="cuda", requires_grad=True)
    b = torch.zeros(c, device="cuda", requires_grad=True)
    y = group_norm_act(x, 1, w, b, 0.0)
    _, db = torch.autograd.grad(y, (w, b), dy, retain_graph=True)
    assert bool((db == 1.0).all())
    dw, _ = torch.autograd.grad(y, (w, b), dy * sign.to(dtype))
    assert bool((dw == 1.0).all())


@pytest.mark.parametrize("shape,groups", [((2, 24, 5, 6, 7), 8), ((1, 24, 24, 60, 40), 8), ((2, 25, 9, 20, 21), 5)])
@pytest.mark.parametrize("dtype,value", [(BF, 100.0), (HF, 30000.0), (HF, 1000.0), (FP, 30000.0), (FP, 1e6), (FP, 0.1)])
def test_constant_far_from_zero(cuda_ready, shape, groups, dtype, value):
    """A background of one value: the variance is 0 however large the value, y is the bias, dx = (dz w - A) / sqrt(eps)."""
    c, kw = shape[1], dict(device="cuda", generator=_gen(12))
    x = _last(torch.full(shape, value, device="cuda").to(dtype))
    dy = _last((torch.randn(shape, **kw) / 64).to(dtype))
    w, b = 1 + 0.2 * torch.randn(c, **kw), 0.2 * torch.randn(c, **kw)
    _affine_check(x, groups, w, b, dy)
    y = group_norm_act(x, groups, w, b)
    assert torch.equal(y, b.to(dtype).reshape(1, c, 1, 1, 1).expand(shape))


@pytest.mark.parametrize("shape,groups", [((2, 24, 16, 32, 32), 8), ((2, 24, 64, 64, 64), 8)])
@pytest.mark.parametrize("dtype,value,step", [(FP, 30000.0, 0.03125), (BF, 100.0, 0.5), (HF, 1000.0, 0.5)])
def test_one_voxel_apart(cuda_ready, shape, groups, dtype, value, step):
    """A group that is one value but for one voxel, and one whose first element is that voxel."""
    c, kw = shape[1], dict(device="cuda", generator=_gen(13))
    x = torch.full(shape, value, device="cuda")
    x[0, ::3, 3, 4, 5] += step
    x[1, ::3, 0, 0, 0] += step
    dy = _last((torch.randn(shape, **kw) / 64).to(dtype))
    w, b = 1 + 0.2 * torch.randn(c, **kw), 0.2 * torch.randn(c, **kw)
    _affine_check(_last(x.to(dtype)), groups, w, b, dy)


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (2, 24, 40, 64, 64)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_bad_first_element_stays_in_its_group(cuda_ready, shape, bad):
    """What a group's sums are taken about."""
    kw = dict(device="cuda", generator=_gen(16))
    x, dy = (_last(torch.randn(shape, **kw).to(BF)) for _ in range(2))

    def run(x):
        x = x.detach().requires_grad_(True)
        y = group_norm_act(x, 8, activation="silu")
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    clean = run(x)
    x[1, 6, 0, 0, 0] = bad
    for got, want in zip(run(x), clean):
        got, want = got.unflatten(1, (8, 3)), want.unflatten(1, (8, 3))
        assert bool(got[1, 2].isnan().all())
        got[1, 2] = want[1, 2]
        assert torch.equal(got, want)


@pytest.mark.parametrize("shape", [(1, 16, 40), (1, 8, 3, 4, 5), (1, 16, 8, 64, 64), (1, 25, 9, 10)])
def test_codes_are_read_in_the_activations_type(cuda_ready, shape):
    """fp16 values below 2^-14 that have a fraction of its smallest step: the backward takes them rounded, as unpack8 does."""
    c, count = shape[1], torch.Size(shape).numel()
    kw = dict(device="cuda", generator=_gen(14))
    plan = _native.gn_plan(torch.Size(shape), 1, HF, FP, 1e-5, 0, 0.0)
    codes = torch.randint(0, 256, (count,), dtype=torch.uint8, **kw)
    codes[(codes & 0x7f) == 0x7f] = 0x11                 # (no NaN)
    exps = torch.randint(96, 120, (-(-count // 32),), dtype=torch.uint8, **kw)
    q8 = torch.zeros(plan.q8_bytes, dtype=torch.uint8, device="cuda")
    q8[:count] = codes
    q8[plan.q8_at:plan.q8_at + exps.numel()] = exps
    last = torch.Size((shape[0], *shape[2:], c))
    x = unpack8(Packed8(codes, exps, last, torch.empty(last).stride(), HF, "e4m3")).movedim(-1, 1)
    assert bool(x.isfinite().all())
    dy = _last(torch.randn(shape, **kw).to(HF))
    stats = torch.zeros(plan.kept, device="cuda")
    stats[:2] = torch.tensor([0.0, 2.0 ** 16], device="cuda")
    w, b = torch.ones(c, device="cuda"), torch.zeros(c, device="cuda")
    want = _native.gn_backward(dy, plan, x, None, stats, w, b, True, True)
    got = _native.gn_backward(dy, plan, q8, 1, stats, w, b, True, True)
    for g, v in zip(got, want):
        assert torch.equal(g, v)
