"""group_norm_act on the native kernels against 64 bits (bounds: gn_refs.py), and what may go wrong around a call."""
import pytest
import torch
import torch.nn as nn
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

import gn_refs as R
from rdna4_conv3d import _native
from rdna4_conv3d.checkpoint8 import checkpoint_activations, pack8, unpack8
from rdna4_conv3d.group_norm import ACTIVATIONS, GroupNormAct3d, fuse_group_norm, group_norm_act

pytestmark = pytest.mark.gpu

CL = torch.channels_last_3d
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
SLOPE = 0.2


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _last(t):
    return t.movedim(1, -1).contiguous().movedim(-1, 1)


def _inputs(shape, dtype, seed=1, pdtype=FP, centre=2.0):
    g, c = _gen(seed), shape[1]
    kw = dict(device="cuda", generator=g)
    x = _last((torch.randn(shape, **kw) * 1.5 + centre * torch.randn(c, **kw).reshape(1, c, *(1,) * (len(shape) - 2))).to(dtype))
    w = (1 + 0.2 * torch.randn(c, **kw)).to(pdtype)
    b = (0.2 * torch.randn(c, **kw)).to(pdtype)
    dy = _last(torch.randn(shape, **kw).to(dtype))
    return tuple(t.requires_grad_(True) for t in (x, w, b)) + (dy,)


def _run(x, groups, w, b, dy, act="relu", fmt=None, eps=1e-5):
    n0 = _native.launch_count()
    y = group_norm_act(x, groups, w, b, eps, activation=act, negative_slope=SLOPE, checkpoint=fmt)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert _native.launch_count() - n0 >= 2
    return dict(y=y, dx=dx, dw=dw, db=db)


def _verify(x, groups, w, b, dy, act="relu", fmt=None, eps=1e-5):
    got = _run(x, groups, w, b, dy, act, fmt, eps)
    assert got["y"].dtype == x.dtype and got["dx"].dtype == x.dtype and got["dw"].dtype == w.dtype
    assert got["y"].movedim(1, -1).is_contiguous()
    kept = None if fmt is None else R.held(x, fmt)
    R.check(got, R.ref(x, groups, w, b, eps, act, SLOPE, dy, kept))
    return got


# channels and groups: multiples of a vector, odd ones, one group, one channel a group, wider than a block
SHAPES = [((2, 24, 5, 6, 7), 8), ((1, 1, 9, 1, 1), 1), ((3, 30, 3, 5, 7), 6), ((2, 25, 3, 3, 5), 25), ((2, 20, 4, 3, 2), 1),
          ((1, 7, 1, 2, 3), 7), ((4, 192, 4, 8, 8), 8), ((2, 48, 16, 16, 16), 3), ((5, 33), 11), ((2, 2056, 3), 8),
          ((1, 4104, 2, 2), 4104), ((2, 1025, 3), 5), ((70, 96, 6, 6, 6), 96), ((1, 16, 1, 1, 40001), 2), ((3, 8, 1, 1, 1), 1),
          ((2, 2, 33, 31, 3), 1)]


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else f"g{v}")
def test_shapes(cuda_ready, shape, groups, dtype, fmt):
    _verify(*_args(shape, groups, dtype), act="silu", fmt=fmt)


def _args(shape, groups, dtype, **kw):
    x, w, b, dy = _inputs(shape, dtype, **kw)
    return x, groups, w, b, dy


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("shape", [(2, 24, 9, 10, 11), (2, 24, 40, 64, 64)])
def test_activations(cuda_ready, act, dtype, fmt, shape):
    _verify(*_args(shape, 8, dtype), act=act, fmt=fmt)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_training_volume(cuda_ready, dtype, fmt):
    """The first level of the segmentation network; every part of the data takes part."""
    _verify(*_args((2, 24, 64, 128, 128), 8, dtype), act="silu", fmt=fmt)


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (3, 24, 64, 64, 64)])
def test_far_from_zero(cuda_ready, shape):
    """|mean| thousands of times the spread, in full precision: nothing may cancel in the sums."""
    x, w, b, dy = _inputs(shape, FP)
    x = (x.detach() / 8 + 1000.0).requires_grad_(True)
    _verify(x, 8, w, b, dy, act="silu")


@pytest.mark.parametrize("shape", [(1, 8, 3, 4, 5), (2, 24, 32, 64, 64)])
def test_first_elements_far_out(cuda_ready, shape):
    """The elements that sums are taken around are a hundred spreads away from the rest."""
    x, w, b, dy = _inputs(shape, FP, centre=0.0)
    x = x.detach()
    flat = x.movedim(1, -1).reshape(shape[0], -1, shape[1])
    flat[:, ::997] += 150.0
    _verify(x.requires_grad_(True), 8, w, b, dy, act="none")


@pytest.mark.parametrize("pdtype", [BF, HF, torch.float64])
def test_parameter_types(cuda_ready, pdtype):
    _verify(*_args((2, 24, 5, 6, 7), 4, BF, pdtype=pdtype), act="gelu")
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), HF)
    _verify(x, 4, w.detach().bfloat16().requires_grad_(True), b, dy)
    for ww, bb in ((None, None), (w, None), (None, b)):
        y = group_norm_act(x, 4, ww, bb, activation="silu")
        want = R.ref(x, 4, ww, bb, 1e-5, "silu", SLOPE, dy)
        wrt = [t for t in (x, ww, bb) if t is not None]
        got = dict(zip([k for k, t in zip(("dx", "dw", "db"), (x, ww, bb)) if t is not None],
                       torch.autograd.grad(y, wrt, dy)), y=y)
        assert set(got) == set(want)
        R.check(got, want)


def test_wanted_gradients_alone(cuda_ready):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    want = R.ref(x, 8, w, b, 1e-5, "relu", SLOPE, dy)
    for names in (("dx",), ("dw",), ("db",), ("dw", "db"), ("dx", "db")):
        ins = [t if k in names else t.detach() for k, t in (("dx", x), ("dw", w), ("db", b))]
        y = group_norm_act(ins[0], 8, ins[1], ins[2], activation="relu")
        wrt = [t for t in ins if t.requires_grad]
        R.check(dict(zip(names, torch.autograd.grad(y, wrt, dy))), want, names)


def _layouts(x):
    yield x.contiguous()                                             # channels first
    yield torch.cat([x, x], 1).contiguous(memory_format=CL)[:, :x.shape[1]]   # a channel slice
    yield x.permute(0, 1, 4, 3, 2).contiguous().permute(0, 1, 4, 3, 2)
    wide = torch.zeros(x.numel() + 1, dtype=x.dtype, device=x.device)
    off = wide[1:].reshape(x.movedim(1, -1).shape)
    off.copy_(x.movedim(1, -1))
    yield off.movedim(-1, 1)                                         # off its 16 bytes


@pytest.mark.parametrize("fmt", [None, "int8"])
def test_layouts(cuda_ready, fmt):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    want = _run(x, 8, w, b, dy, "silu", fmt)
    for i, other in enumerate(_layouts(x.detach())):
        for gy in (dy, dy.contiguous()) + ((list(_layouts(dy))[3],) if i == 0 else ()):
            got = _run(other.detach().requires_grad_(True), 8, w, b, gy, "silu", fmt)
            for k in want:
                assert torch.equal(got[k], want[k]), (i, k)
    one = torch.full((), 0.5, device="cuda", dtype=BF).expand(dy.shape)      # a gradient that overlaps itself
    for k, v in _run(x, 8, w, b, one, "silu", fmt).items():
        assert torch.equal(v, _run(x, 8, w, b, one.contiguous(memory_format=CL), "silu", fmt)[k])


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (2, 24, 32, 64, 64)])
@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
def test_bad_values_stay_in_their_group(cuda_ready, shape, fmt):
    x, w, b, dy = _inputs(shape, BF)
    clean = _run(x, 8, w, b, dy, "silu", fmt)
    with torch.no_grad():
        x[0, 4, 1, 2, 3] = float("nan")
        x[1, 23, 2, 0, 1] = float("inf")
    got = _run(x, 8, w, b, dy, "silu", fmt)
    for k in ("y", "dx"):
        v, c = (t[k].unflatten(1, (8, 3)) for t in (got, clean))
        bad = torch.zeros(v.shape[:2], dtype=torch.bool, device="cuda")
        bad[0, 1] = bad[1, 7] = True
        assert bool(v[bad].isnan().all())
        # (a block of 32 elements that loses its largest value may take a finer step)
        if k == "y" or fmt is None:
            assert torch.equal(v[~bad], c[~bad])
        else:
            assert bool(v[~bad].isfinite().all())
    assert bool(got["dw"][3:6].isnan().all()) and bool(got["dw"][:3].isfinite().all())


def test_constant_groups(cuda_ready):
    """No spread at all: xh is 0, the gradient finite."""
    x = torch.full((2, 8, 4, 4, 4), 3.25, device="cuda", dtype=BF).contiguous(memory_format=CL).requires_grad_(True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    b = torch.linspace(-1, 1, 8, device="cuda", requires_grad=True)
    dy = torch.randn(x.shape, device="cuda", generator=_gen(3)).to(BF).contiguous(memory_format=CL)
    for fmt in (None, "int8"):
        _verify(x, 2, w, b, dy, "none", fmt)


def test_empty(cuda_ready):
    for shape in ((0, 24, 2, 2, 2), (2, 24, 0, 3, 4), (0, 24)):
        for fmt in (None, "int8"):
            x = torch.zeros(shape, device="cuda", dtype=BF, requires_grad=True)
            w = torch.ones(24, device="cuda", requires_grad=True)
            b = torch.ones(24, device="cuda", requires_grad=True)
            y = group_norm_act(x, 8, w, b, activation="silu", checkpoint=fmt)
            assert y.shape == shape and group_norm_act(x.detach(), 8, w.detach()).shape == shape
            y.sum().backward()
            assert x.grad.shape == shape and bool((w.grad == 0).all()) and bool((b.grad == 0).all())


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (4, 24, 32, 64, 64), (1, 48, 64, 64, 64)])
@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_same_bits_every_time(cuda_ready, shape, fmt):
    args = _args(shape, 8, BF)
    first = _run(*args, "silu", fmt)
    for _ in range(5):
        for k, v in _run(*args, "silu", fmt).items():
            assert torch.equal(v, first[k]), k


def test_gradient_against_differences(cuda_ready):
    x, w, b, dy = _inputs((2, 16, 6, 5, 4), FP, centre=0.5)
    got = _run(x, 4, w, b, dy, "silu")
    h = 2.0 ** -6

    def f(x, w, b):
        return (group_norm_act(x.detach(), 4, w.detach(), b.detach(), activation="silu").double() * dy.double()).sum()

    for k, i in (("dx", 0), ("dw", 1), ("db", 2)):
        v = torch.randn((x, w, b)[i].shape, device="cuda", generator=_gen(9))
        args = [[x, w, b], [x, w, b]]
        args[0][i], args[1][i] = args[0][i] + h * v, args[1][i] - h * v
        slope = (f(*args[0]) - f(*args[1])) / (2 * h)
        want = (got[k].double() * v.double()).sum()
        # third derivatives: h^2 / 6 of something near the sum's own spread; rounding: 2^-24 sqrt(elements) / h
        scale = (got[k].double().abs() * v.double().abs()).sum()
        assert abs(slope - want) <= scale * h * h + 2.0 ** -20 * dy.abs().sum() / h / dy.numel() ** 0.5, k


def _reversed(t):
    back = tuple(reversed(range(t.dim())))
    return t.clone().permute(back).contiguous().permute(back)


def _padded(t):
    if t.dim() == 0:
        return t.clone()
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


HOOKS = {"cpu": save_on_cpu, "reversed": lambda: saved_tensors_hooks(_reversed, lambda t: t),
         "padded": lambda: saved_tensors_hooks(_padded, lambda t: t)}


@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_hooks_on_saved_tensors(cuda_ready, fmt, hook):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    want = _run(x, 8, w, b, dy, "silu", fmt)
    with HOOKS[hook]():
        y = group_norm_act(x, 8, w, b, activation="silu", checkpoint=fmt)
    for g, k in zip(torch.autograd.grad(y, (x, w, b), dy), ("dx", "dw", "db")):
        assert torch.equal(g, want[k]), k
    with saved_tensors_hooks(lambda t: t[:1].clone(), lambda t: t):
        y = group_norm_act(x, 8, w, b, activation="silu", checkpoint=fmt)
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(y, (x, w, b), dy)


def test_changed_in_place_is_an_error(cuda_ready):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    x2 = x * 1
    y = group_norm_act(x2, 8, w, b)
    x2.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)
    x2 = x * 1
    y = group_norm_act(x2, 8, w, b, checkpoint="int8")           # x itself is not kept
    x2.mul_(2)
    y.backward(dy)


def test_refusals_on_the_device(cuda_ready):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    with pytest.raises(TypeError):
        group_norm_act(x.double(), 8)
    with pytest.raises(ValueError):
        group_norm_act(x, 8, w.cpu())
    y = group_norm_act(x, 8, w, b)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y, x, dy, create_graph=True)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        for args in ((fwAD.make_dual(x.detach(), dy), 8, w, b), (x.detach(), 8, fwAD.make_dual(w.detach(), b.detach()), b)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                group_norm_act(*args)
    with pytest.raises(Exception):
        torch.func.grad(lambda t: group_norm_act(t, 8, w, b).float().sum())(x.detach())
    with pytest.raises(RuntimeError, match="make_fx"):
        torch.fx.experimental.proxy_tensor.make_fx(lambda t: group_norm_act(t, 8))(x.detach())


def test_side_streams_side_by_side(cuda_ready):
    """Two calls at once on two streams: workspaces are each call's own."""
    sets = [_args((2, 24, 16, 32, 32), 8, BF, seed=s) for s in (1, 2)]
    want = [_run(*a, "silu", "int8") for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        got = []
        for s, a in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(_run(*a, "silu", "int8"))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for k in w:
                assert torch.equal(g[k], w[k])


@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (2, 24, 32, 64, 64)])
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_captured_and_replayed(cuda_ready, shape, fmt):
    sets = [_args(shape, 8, BF, seed=s) for s in (1, 2, 3)]
    want = [_run(*a, "silu", fmt) for a in sets]
    x, groups, w, b, dy = [t.detach().clone() if torch.is_tensor(t) else t for t in sets[0]]
    for t in (x, w, b):
        t.requires_grad_(True)
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(x, groups, w, b, dy, "silu", fmt)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):                                   # two graphs of the same call, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _run(x, groups, w, b, dy, "silu", fmt)
        graphs.append((g, out))
    for i in (1, 2, 0, 1):
        with torch.no_grad():
            for t, v in zip((x, w, b, dy), (sets[i][0], sets[i][2], sets[i][3], sets[i][4])):
                t.copy_(v)
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for k in out:
                assert torch.equal(out[k], want[i][k]), k


def test_past_32_bits(cuda_ready):
    """More than 2^32 bytes and 2^31 elements; the last sample against itself alone."""
    n = 9
    shape = (n, 24, 80, 320, 400)                        # 2.2 G elements of 2 bytes
    x = torch.empty((n, 80, 320, 400, 24), device="cuda", dtype=BF).normal_(generator=_gen(1)).movedim(-1, 1)
    assert x.numel() > 2 ** 31 and x.shape == shape
    w = torch.linspace(0.5, 1.5, 24, device="cuda", requires_grad=True)
    x.requires_grad_(True)
    y = group_norm_act(x, 8, w, None, activation="silu", checkpoint="int8")
    dy = torch.zeros_like(y)
    dy[n - 1] = y.detach()[n - 1]
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    last = x.detach()[n - 1:].requires_grad_(True)
    y1 = group_norm_act(last, 8, w, None, activation="silu", checkpoint="int8")
    dx1, dw1 = torch.autograd.grad(y1, (last, w), dy[n - 1:])
    # (other numbers of blocks share out the sums: the last bits of mean and rstd may differ, a rounding of y with them)
    assert (y[n - 1:].detach() - y1.detach()).abs().max() <= 2.0 ** -7 * 8
    assert ((y[n - 1:] != y1).sum() <= 1e-3 * y1.numel()) and ((dx[n - 1:] != dx1).sum() <= 1e-2 * dx1.numel())
    torch.testing.assert_close(dw, dw1, rtol=1e-4, atol=1e-2)
    assert not bool(dx[:n - 1].any())


def test_many_samples(cuda_ready):
    """More samples than a grid's other dimensions take."""
    x, w, b, dy = _inputs((70001, 16), BF)
    _verify(x, 2, w, b, dy, "relu")
    x, w, b, dy = _inputs((66000, 3, 2), HF)
    _verify(x, 3, w, b, dy, "gelu", "int8")


# --- modules and models ----------------------------------------------------------
def test_module_and_fuse(cuda_ready):
    torch.manual_seed(0)
    seq = nn.Sequential(nn.GroupNorm(4, 16), nn.SiLU(), nn.GroupNorm(2, 16), nn.LeakyReLU(0.1)).cuda()
    x = torch.randn(2, 16, 6, 7, 8, device="cuda").to(BF).contiguous(memory_format=CL)
    with torch.no_grad():
        want = seq(x.float())
        n0 = _native.launch_count()
        assert fuse_group_norm(seq) == 2
        got = seq(x)
    assert _native.launch_count() > n0 and got.dtype == BF
    assert (got.float() - want).abs().max() <= 2.0 ** -6 * want.abs().max()
    with torch.autocast("cuda", dtype=BF):
        assert seq(x).dtype == BF


def test_stock_backend(cuda_ready, monkeypatch):
    import sys
    cw = sys.modules["rdna4_conv3d.conv3d_wmma"]
    m = GroupNormAct3d(4, 16, activation="gelu", checkpoint="int8").cuda()
    x = torch.randn(2, 16, 6, 7, 8, device="cuda").to(BF).contiguous(memory_format=CL).requires_grad_(True)
    dy = torch.randn(x.shape, device="cuda").to(BF)
    want = torch.autograd.grad(m(x), (x, m.weight), dy)
    monkeypatch.setattr(cw, "_wmma_hw", lambda: False)
    n0 = _native.launch_count()
    got = torch.autograd.grad(m(x), (x, m.weight), dy)
    assert _native.launch_count() == n0
    for a, e in zip(got, want):
        torch.testing.assert_close(a, e, rtol=2e-2, atol=2e-2)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("shape,cout,k", [((2, 24, 6, 8, 10), 24, 3), ((1, 5, 6, 7, 9), 7, 3), ((2, 48, 4, 8, 8), 4, 1), ((2, 1, 8, 8, 16), 24, 3)])
def test_conv_kept_in_8_bits(cuda_ready, shape, cout, k, fmt, dtype):
    """y, dX and db as without, dW as that of the values that the 8 bits hold."""
    from rdna4_conv3d import conv3d_wmma
    for fmt_in in (CL, torch.contiguous_format):
        x = torch.randn(shape, device="cuda", generator=_gen(1)).to(dtype).contiguous(memory_format=fmt_in).requires_grad_(True)
        w = (torch.randn(cout, shape[1], k, k, k, device="cuda", generator=_gen(2)) * 0.1).requires_grad_(True)
        b = torch.randn(cout, device="cuda", generator=_gen(3)).requires_grad_(True)
        plain = conv3d_wmma(x, w, b, 1, k // 2)
        dy = torch.randn(plain.shape, device="cuda", generator=_gen(4)).to(dtype).contiguous(memory_format=fmt_in)
        dx0, dw0, db0 = torch.autograd.grad(plain, (x, w, b), dy)
        y = conv3d_wmma(x, w, b, 1, k // 2, checkpoint=fmt)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert torch.equal(y, plain) and torch.equal(dx, dx0) and torch.equal(db, db0) and dx.stride() == dx0.stride()
        xk = unpack8(pack8(x, fmt)).requires_grad_(True)
        want, = torch.autograd.grad(conv3d_wmma(xk, w, b, 1, k // 2), w, dy)
        assert torch.equal(dw, want) and not torch.equal(dw, dw0)
        # without a weight gradient there is nothing to keep
        y = conv3d_wmma(x, w.detach(), None, 1, k // 2, checkpoint=fmt)
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx0)


def _saved_bytes(net, x):
    seen = {}

    def pack(t):
        seen[(t.data_ptr(), t.numel())] = t.numel() * t.element_size()
        return t

    with saved_tensors_hooks(pack, lambda t: t), torch.autocast("cuda", dtype=BF):
        y = net(x)
    return y, sum(seen.values())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_unet_training_step(cuda_ready, fmt):
    """The network on group norms, whole and in 8 bits: the same output, gradients near, less kept."""
    from rdna4_conv3d.losses import cross_entropy
    from rdna4_conv3d.unet3d import unet3d
    torch.manual_seed(1)
    net = unet3d(24, levels=3, norm="group", groups=8, activation="silu", device="cuda")
    x = torch.randn(1, 1, 16, 32, 32, device="cuda").contiguous(memory_format=CL)
    t = torch.randint(0, 4, (1, 16, 32, 32), device="cuda")
    res = {}
    for f in (None, fmt):
        assert checkpoint_activations(net, f) > 0
        net.zero_grad(set_to_none=True)
        y, kept = _saved_bytes(net, x)
        cross_entropy(y, t).backward()
        res[f] = y.detach(), kept, [p.grad.clone() for p in net.parameters()]
    y0, k0, g0 = res[None]
    y1, k1, g1 = res[fmt]
    assert torch.equal(y0, y1) and k1 < 0.75 * k0
    # a gradient at values that are off by at most 2^-4 of themselves (e4m3; int8: 1/254 of the block's largest)
    num = sum(((a - b).double() ** 2).sum() for a, b in zip(g0, g1)) ** 0.5
    den = sum((a.double() ** 2).sum() for a in g0) ** 0.5
    assert 0 < num <= 2.0 ** -3 * den


def test_captured_training_step(cuda_ready):
    from rdna4_conv3d.losses import cross_entropy
    from rdna4_conv3d.unet3d import unet3d
    torch.manual_seed(1)
    net = unet3d(8, levels=2, norm="group", groups=4, device="cuda", checkpoint="int8")
    x = torch.randn(1, 1, 8, 16, 16, device="cuda").contiguous(memory_format=CL)
    t = torch.randint(0, 4, (1, 8, 16, 16), device="cuda")

    def step():
        with torch.autocast("cuda", dtype=BF):
            loss = cross_entropy(net(x), t)
        return torch.autograd.grad(loss, list(net.parameters()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want = [g.clone() for g in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_compiled_between_graphs(cuda_ready):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    fn = torch.compile(lambda x, w, b: group_norm_act(x * 2, 8, w, b, activation="silu") + 1, backend="eager")
    y = fn(x, w, b)
    assert torch.equal(y, group_norm_act(x * 2, 8, w, b, activation="silu") + 1)
    torch.autograd.grad(y, (x, w, b), dy)




# samples that begin and end inside a vector or a row of several voxels: nothing but edges, one whole row, many
EDGES = [((3, 1, 1, 1, 3), 1), ((3, 3, 1, 1, 1), 3), ((7, 5, 1, 1, 7), 5), ((5, 12, 1, 3, 3), 4), ((3, 20, 3, 3, 3), 5),
         ((3, 30, 7, 11, 13), 6), ((2, 30, 37, 41, 53), 6), ((3, 199, 3, 5, 7), 199), ((2, 255, 3, 3, 3), 17),
         ((3, 257, 3, 3, 3), 257), ((2, 300, 5, 5, 5), 3), ((3, 1028, 3, 3, 1), 4), ((9, 36, 1, 1, 5), 1), ((5, 13, 21, 23, 25), 1)]


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("shape,groups", EDGES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else f"g{v}")
def test_edges_of_samples(cuda_ready, shape, groups, dtype, fmt):
    _verify(*_args(shape, groups, dtype), act="gelu" if dtype is FP else "silu", fmt=fmt)
    x, _, w, b, dy = _args(shape, groups, dtype, seed=5)
    y = group_norm_act(x.detach(), groups, w.detach(), b.detach(), activation="relu")
    R.check(dict(y=y), R.ref(x, groups, w, b, 1e-5, "relu", SLOPE))


def test_one_sample_past_32_bits(cuda_ready):
    """A single sample of 2.2 G elements: offsets inside it pass 32 bits."""
    x = torch.empty((1, 720, 320, 400, 24), device="cuda", dtype=BF).normal_(generator=_gen(1)).movedim(-1, 1)
    assert x.numel() > 2 ** 31
    w = torch.linspace(0.5, 1.5, 24, device="cuda")
    s1 = torch.zeros(8, dtype=torch.float64, device="cuda")
    s2 = torch.zeros_like(s1)
    for part in x[0].split(40, 1):
        v = part.movedim(0, -1).reshape(-1, 8, 3).float()
        s1 += v.sum((0, 2), dtype=torch.float64)
        s2 += (v * v).sum((0, 2), dtype=torch.float64)
        del v
    m = x.numel() / 8
    mean = (s1 / m).repeat_interleave(3).reshape(24, 1, 1)
    rstd = ((s2 / m - (s1 / m) ** 2 + 1e-5) ** -0.5).repeat_interleave(3).reshape(24, 1, 1)
    y = group_norm_act(x, 8, w)
    for d in (0, 359, 719):
        want = (x[0, :, d].double() - mean) * rstd * w.double().reshape(24, 1, 1)
        # half a step, and the sums of squares taken here in fp32 products (2^-24 each, unbiased) far below it
        assert bool(((y[0, :, d].double() - want).abs() <= R.half_step(want, BF) + R.K * (1 + want.abs())).all())
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = group_norm_act(x, 8, w, checkpoint="e4m3")
    dy = torch.zeros_like(y)
    dy[0, :, 719] = 1.0                                   # dz = w there: dw = the sum of xh over the last plane
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xh = (R.held(x.detach()[:, :, 719:], "e4m3")[0, :, 0].double() - mean) * rstd
    # (blocks of 32 elements are the same: a plane is a whole number of them)
    torch.testing.assert_close(dw.double(), xh.sum((1, 2)), rtol=1e-4, atol=128000 * R.K)
    assert bool(dx[0, :, 719].abs().amax() > 0.1) and bool(dx[0, :, 0].abs().amax() < 1e-2)


def test_refuses_a_second_differentiation_of_kept_convs(cuda_ready):
    from rdna4_conv3d import conv3d_wmma
    x = torch.randn(1, 8, 4, 8, 8, device="cuda", dtype=BF).contiguous(memory_format=CL).requires_grad_(True)
    w = torch.randn(8, 8, 3, 3, 3, device="cuda", requires_grad=True)
    y = conv3d_wmma(x, w, None, 1, 1, checkpoint="int8")
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.float().sum(), w, create_graph=True)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_hooks_on_kept_convs(cuda_ready, fmt):
    from rdna4_conv3d import conv3d_wmma
    x = torch.randn(2, 24, 6, 8, 10, device="cuda", dtype=BF, generator=_gen(1)).contiguous(memory_format=CL).requires_grad_(True)
    w = torch.randn(24, 24, 3, 3, 3, device="cuda", generator=_gen(2), requires_grad=True)
    want = torch.autograd.grad(conv3d_wmma(x, w, None, 1, 1, checkpoint=fmt).float().sum(), (x, w))
    for hook in HOOKS.values():
        with hook():
            y = conv3d_wmma(x, w, None, 1, 1, checkpoint=fmt)
        for a, b in zip(torch.autograd.grad(y.float().sum(), (x, w)), want):
            assert torch.equal(a, b)
    with saved_tensors_hooks(lambda t: t[:3].clone(), lambda t: t):
        y = conv3d_wmma(x, w, None, 1, 1, checkpoint=fmt)
    with pytest.raises((RuntimeError, ValueError)):
        torch.autograd.grad(y.float().sum(), w)


def test_inference_and_frozen_parts(cuda_ready):
    x, w, b, dy = _inputs((2, 24, 5, 6, 7), BF)
    want = R.ref(x, 8, w, b, 1e-5, "gelu", SLOPE)
    with torch.inference_mode():
        R.check(dict(y=group_norm_act(x, 8, w, b, activation="gelu", checkpoint="int8")), want)
    m = GroupNormAct3d(8, 24, activation="gelu", checkpoint="int8").cuda().requires_grad_(False)
    y = m(x.detach())
    assert not y.requires_grad
    y = m(x)
    assert torch.equal(y, m(x.detach()))
    y.backward(dy)
    assert x.grad is not None and m.weight.grad is None


@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("shape", [(2, 24, 5, 6, 7), (2, 24, 32, 64, 64)])
def test_traces_run_the_operator_again(cuda_ready, shape, fmt, wants_grad):
    """A trace computes from the inputs that it is given, or there is none."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, b, _ = _inputs(shape, BF)
    more = _inputs(shape, BF, seed=8)[0]
    x, more = (t.detach().requires_grad_(wants_grad) for t in (x, more))
    w, b = (t.detach().requires_grad_(wants_grad) for t in (w, b))
    # (parameters as inputs: torch.jit.trace takes no constants that require gradients)
    f = lambda t, w, b: group_norm_act(t, 8, w, b, activation="silu", checkpoint=fmt) * 2  # noqa: E731
    want = f(more, w, b)
    assert torch.equal(torch.jit.trace(f, (x, w, b), check_trace=False)(more, w, b), want)
    torch._dynamo.reset()
    assert torch.equal(torch.compile(f, backend="eager")(more, w, b), want)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(x, w, b)


def test_packing_is_not_traced(cuda_ready):
    x = torch.randn(1000, device="cuda")
    p = pack8(x)
    for f in (lambda t: pack8(t).codes, lambda t: unpack8(p._replace(codes=t.to(torch.uint8)[:1000])) * 1):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
    torch._dynamo.reset()
    f = lambda t: unpack8(pack8(t * 2, "e4m3")) + 1  # noqa: E731
    assert torch.equal(torch.compile(f, backend="eager")(x), f(x))


def test_kept_convs_in_traces(cuda_ready):
    from rdna4_conv3d import conv3d_wmma
    x, more = (torch.randn(1, 8, 4, 8, 8, device="cuda", dtype=BF, generator=_gen(s)).contiguous(memory_format=CL) for s in (1, 2))
    w = torch.randn(8, 8, 3, 3, 3, device="cuda", generator=_gen(3), requires_grad=True)
    f = lambda t, w: conv3d_wmma(t, w, None, 1, 1, checkpoint="int8") * 2  # noqa: E731
    want = f(more, w)
    assert torch.equal(torch.jit.trace(f, (x, w), check_trace=False)(more, w), want)


@pytest.mark.parametrize("fmt", [None, "int8"])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_steep(cuda_ready, act, dtype, fmt):
    """Weights of some hundred, either sign: the activations' flat ends, exponentials out of range."""
    for shape in ((2, 24, 9, 10, 11), (2, 24, 32, 48, 48)):
        x, w, b, dy = _inputs(shape, dtype)
        with torch.no_grad():
            w.mul_(torch.linspace(-400, 400, 24, device="cuda"))
            b.mul_(200)
        got = _verify(x, 8, w, b, dy, act, fmt)
        assert all(bool(v.isfinite().all()) for v in got.values())


@pytest.mark.parametrize("fmt", [None, "e4m3"])
@pytest.mark.parametrize("shape", [(3, 24), (2, 24, 50), (2, 24, 9, 11), (2, 24, 3, 4, 5, 6), (2, 1, 7, 8, 9)])
def test_dimensions(cuda_ready, shape, fmt):
    """Tokens, sequences, images, volumes and more, channels last or first."""
    groups = 4 if shape[1] > 1 else 1
    args = _args(shape, groups, HF)
    want = _verify(*args, act="gelu", fmt=fmt)
    x, _, w, b, dy = args
    first = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
    for k, v in _run(first, groups, w, b, dy.contiguous(), "gelu", fmt).items():
        assert torch.equal(v, want[k]), k
