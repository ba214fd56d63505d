"""group_norm_act, GroupNormAct3d and pack8 / unpack8 on the CPU: values, gradients, refusals, model switches."""
import ctypes

import pytest
import torch
import torch.nn as nn

import gn_refs as R
from rdna4_conv3d import _native
from rdna4_conv3d.checkpoint8 import Packed8, checkpoint_activations, pack8, unpack8
from rdna4_conv3d.group_norm import ACTIVATIONS, GroupNormAct3d, fuse_group_norm, group_norm_act


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _inputs(shape, dtype=torch.float32, seed=1):
    g = _gen(seed)
    c = shape[1]
    x = (torch.randn(shape, generator=g) * 1.5 + 2.0).to(dtype)
    w = 1 + 0.2 * torch.randn(c, generator=g)
    b = 0.2 * torch.randn(c, generator=g)
    dy = torch.randn(shape, generator=g).to(dtype)
    return x, w, b, dy


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("shape,groups", [((2, 12, 3, 4, 5), 4), ((3, 6), 2), ((1, 5, 7), 5), ((2, 4, 3, 3), 1)])
def test_values_and_gradients(shape, groups, act, fmt):
    x, w, b, dy = _inputs(shape)
    for t in (x, w, b):
        t.requires_grad_(True)
    y = group_norm_act(x, groups, w, b, 1e-5, activation=act, negative_slope=0.2, checkpoint=fmt)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert y.movedim(1, -1).is_contiguous()
    kept = None if fmt is None else R.held(x, fmt)
    R.check(dict(y=y, dx=dx, dw=dw, db=db), R.ref(x, groups, w, b, 1e-5, act, 0.2, dy, kept))


@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_gradient_against_differences(act):
    x, w, b, _ = _inputs((2, 6, 2, 3, 2))
    x, w, b = (t.double().requires_grad_(True) for t in (x, w, b))
    fn = lambda x, w, b: group_norm_act(x, 3, w, b, 1e-5, activation=act)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (x, w, b))
    assert torch.autograd.gradgradcheck(fn, (x, w, b))


def test_stock_modules_agree():
    x, _, _, _ = _inputs((2, 8, 4, 4, 4))
    seq = nn.Sequential(nn.Conv3d(8, 8, 1), nn.GroupNorm(4, 8), nn.SiLU(), nn.Sequential(nn.GroupNorm(2, 8), nn.GELU()),
                        nn.GroupNorm(8, 8), nn.LeakyReLU(0.3), nn.GroupNorm(8, 8), nn.GELU("tanh"), nn.GroupNorm(1, 8))
    for m in seq.modules():
        if isinstance(m, nn.GroupNorm):
            nn.init.normal_(m.weight)
            nn.init.normal_(m.bias)
    # in 64 bits: each norm divides by a spread that random weights can make small, so that an fp32 rounding of the first
    # layer may grow a thousandfold in each that follows (1e-16 by 1e3 each in four layers of which one is plain: 1e-7)
    seq, x = seq.double(), x.double()
    want = seq(x)
    keys = list(seq.state_dict())
    seq.eval()
    assert fuse_group_norm(seq) == 3
    assert list(seq.state_dict()) == keys and not seq[1].training
    assert isinstance(seq[1], GroupNormAct3d) and seq[5].extra_repr() == "" and seq[4].negative_slope == 0.3
    assert type(seq[6]) is nn.GroupNorm and type(seq[8]) is nn.GroupNorm
    torch.testing.assert_close(seq(x), want, rtol=1e-7, atol=1e-7)


def test_refusals():
    x, w, b, _ = _inputs((2, 12, 3, 4, 5))
    bad = [
        (ValueError, dict(x=x[0, :, 0, 0, 0])), (ValueError, dict(num_groups=5)), (ValueError, dict(num_groups=0)),
        (TypeError, dict(x=x.long())), (TypeError, dict(x=x.double(), checkpoint="int8")),
        (ValueError, dict(weight=w[:11])), (ValueError, dict(bias=b[None])), (TypeError, dict(weight=w.long())),
        (ValueError, dict(weight=w.to("meta"))), (ValueError, dict(eps=-1.0)), (ValueError, dict(eps=float("nan"))),
        (ValueError, dict(activation="tanh")), (ValueError, dict(negative_slope=float("inf"))),
        (ValueError, dict(checkpoint="int4")), (ValueError, dict(checkpoint="")),
    ]
    for error, change in bad:
        args = dict(x=x, num_groups=4, weight=w, bias=b)
        args.update(change)
        with pytest.raises(error):
            group_norm_act(**args)
    with pytest.raises(ValueError):
        GroupNormAct3d(4, 8, activation="swish")
    with pytest.raises(ValueError):
        GroupNormAct3d(4, 8, checkpoint="fp8")
    y = group_norm_act(x.requires_grad_(True), 4, w, b, checkpoint="int8")
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_empty_and_degenerate():
    for shape in ((0, 6, 2, 2, 2), (2, 6, 0, 2, 2), (0, 6)):
        x = torch.zeros(shape, requires_grad=True)
        w = torch.ones(6, requires_grad=True)
        y = group_norm_act(x, 3, w, None, activation="relu", checkpoint="int8")
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and bool((w.grad == 0).all())
    # a group of one element has no spread: the bias is what is left
    x, w, b, _ = _inputs((2, 5))
    torch.testing.assert_close(group_norm_act(x, 5, w, b), b.expand(2, 5))


def test_empty_bias():
    x, b = torch.zeros(2, 6, 0), torch.ones(6, requires_grad=True)
    group_norm_act(x, 3, None, b).sum().backward()
    assert bool((b.grad == 0).all())


# --- 8 bits ------------------------------------------------------------------
def special(dtype, seed=2):
    """Blocks that a format can go wrong at: nothing, one value, border values, subnormals, huge and non-finite ones."""
    info = torch.finfo(dtype)
    g = _gen(seed)
    rows = [torch.zeros(32), torch.randn(32, generator=g), torch.randn(32, generator=g) * 1e-3,
            torch.cat([torch.tensor([127.0, 127.5, -127.0, 0.5, 1.5, 2.5, -0.5, -1.5]), torch.arange(24.0)]),
            torch.cat([torch.tensor([448.0, 449.0, -448.0, 2.0 ** -6, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -0.0]),
                       torch.arange(24.0) + 0.5]),
            torch.full((32,), info.max), torch.full((32,), -info.max) * torch.rand(32, generator=g),
            torch.full((32,), info.tiny), torch.randn(32, generator=g) * info.tiny,
            torch.full((32,), info.tiny * info.eps),
            torch.cat([torch.tensor([float("nan"), float("inf"), -float("inf")]), torch.randn(29, generator=g)]),
            torch.full((32,), float("nan")), torch.full((32,), -float("inf"))]
    scales = torch.exp2(torch.arange(-20.0, 15.0))
    rows += [torch.randn(32, generator=g) * s for s in scales]
    return torch.cat(rows + [torch.randn(7, generator=g)]).to(dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_pack8_values(dtype, fmt):
    x = special(dtype)
    p = pack8(x, fmt)
    assert p.codes.shape == x.shape and p.exponents.numel() == -(-x.numel() // 32)
    v = unpack8(p)
    assert v.dtype == dtype
    limit = torch.finfo(dtype).max
    want = R.blocks64(x, fmt).clamp(-limit, limit).to(dtype)
    torch.testing.assert_close(v, want, rtol=0, atol=0, equal_nan=True)
    assert bool((v.isnan() == ~x.isfinite()).all())
    # the error that the documentation promises
    fin = x.isfinite()
    unit = torch.exp2(p.exponents.double() - 127).repeat_interleave(32)[:x.numel()]
    err = (v.double() - x.double()).abs()[fin]
    u, mag = unit[fin], x.double().abs()[fin]
    bound = u / 2 if fmt == "int8" else torch.maximum(mag / 16, u / 1024)
    assert bool((err <= bound).all())


def test_pack8_layouts():
    x = torch.randn(2, 5, 3, 4, 7, generator=_gen(4))
    for t in (x, x.contiguous(memory_format=torch.channels_last_3d), x.permute(4, 2, 0, 1, 3), x[:, 1:3], x[..., ::2],
              x[0, 0, 0, 0, :1].expand(3, 6), torch.tensor(2.5), x[:0], x[:, :, 0]):
        p = pack8(t, "int8")
        v = unpack8(p)
        assert v.shape == t.shape and v.stride() == p.stride
        bound = torch.exp2(p.exponents.double() - 127).max() / 2 if t.numel() else 0.0
        assert t.numel() == 0 or (v - t).abs().max().item() <= bound
    cl = x.contiguous(memory_format=torch.channels_last_3d)
    assert unpack8(pack8(cl)).stride() == cl.stride()


def test_pack8_refusals():
    x = torch.randn(40)
    p = pack8(x)
    for error, fn in ((ValueError, lambda: pack8(x, "int4")), (TypeError, lambda: pack8(x.double())),
                      (TypeError, lambda: pack8(x.to(torch.uint8))),
                      (ValueError, lambda: unpack8(p._replace(codes=p.codes[:39]))),
                      (ValueError, lambda: unpack8(p._replace(exponents=p.exponents[:1]))),
                      (ValueError, lambda: unpack8(p._replace(format="fp8"))),
                      (ValueError, lambda: unpack8(p._replace(codes=p.codes.to(torch.int8)))),
                      (ValueError, lambda: unpack8(p._replace(stride=(0,)))),
                      (TypeError, lambda: unpack8(p._replace(dtype=torch.float64)))):
        with pytest.raises(error):
            fn()
    assert isinstance(p, Packed8)


def test_switches():
    from rdna4_conv3d.unet3d import unet3d
    net = unet3d(8, levels=2, norm="group", groups=4, activation="silu", checkpoint="int8")
    norms = [m for m in net.modules() if isinstance(m, GroupNormAct3d)]
    assert len(norms) == 6 and all(m.checkpoint == "int8" and m.activation == "silu" for m in norms)
    assert checkpoint_activations(net, None) == 6 + 7 and all(m.checkpoint is None for m in norms)
    assert checkpoint_activations(net, "e4m3") == 13 and net.head.checkpoint == "e4m3"
    with pytest.raises(ValueError):
        checkpoint_activations(net, "int4")
    with pytest.raises(ValueError):
        unet3d(8, levels=2, wmma=False, checkpoint="int8")
    with pytest.raises(ValueError):
        unet3d(8, levels=2, norm="layer")
    with pytest.raises(ValueError):
        unet3d(8, levels=2, norm="group", activation="tanh")
    from rdna4_conv3d import conv3d_wmma
    with pytest.raises(ValueError):
        conv3d_wmma(torch.randn(1, 2, 3, 3, 3), torch.randn(2, 2, 1, 1, 1), checkpoint="int4")
    # same keys and, on the CPU, same values as the stock layers
    torch.manual_seed(0)
    stock = unet3d(8, levels=2, norm="group", groups=4, wmma=False)
    own = unet3d(8, levels=2, norm="group", groups=4)
    own.load_state_dict(stock.state_dict())
    x = torch.randn(1, 1, 8, 8, 8, generator=_gen(5))
    torch.testing.assert_close(own(x), stock(x), rtol=1e-4, atol=1e-4)


# --- C entries, on the host ----------------------------------------------------
def _d(**kw):
    d = dict(samples=2, inner=64, channels=24, groups=8, dtype=0, param_dtype=2, activation=1, eps=1e-5, slope=0.0)
    d.update(kw)
    return _native.GnDesc(**d)


def test_entries_refuse():
    lib = _native.lib()
    buf = (ctypes.c_char * 4096)()
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    p = ctypes.c_void_p(at)
    odd = ctypes.c_void_p(at + 2)

    def fwd(d, x=p, y=p, mr=p, fmt=0, codes=None, exps=None, ws=p, nb=1 << 40):
        return lib.r4c_gn_fwd(d, x, None, None, y, mr, fmt, codes, exps, ws, nb, None)

    def bwd(d, dy=p, x=p, fmt=0, exps=None, mr=p, dx=p, ws=p, nb=1 << 40):
        return lib.r4c_gn_bwd(d, dy, x, fmt, exps, mr, None, None, dx, None, None, ws, nb, None)

    for change in (dict(samples=-1), dict(inner=-1), dict(channels=0), dict(groups=0), dict(groups=7), dict(dtype=5),
                   dict(param_dtype=-1), dict(activation=5), dict(activation=-1), dict(eps=-1.0),
                   dict(eps=float("nan"))):
        assert fwd(_d(**change)) == -1 and bwd(_d(**change)) == -1, change
        assert lib.r4c_gn_workspace_size(_d(**change), 0) == 0
    huge = _d(samples=1 << 40, inner=1 << 40)
    assert fwd(huge) == -7 and bwd(huge) == -7 and lib.r4c_gn_workspace_size(huge, 1) == 0
    assert fwd(_d(), x=None) == -1 and fwd(_d(), y=None) == -1 and fwd(_d(), mr=None) == -1
    assert fwd(_d(), codes=p) == -1 and fwd(_d(), codes=p, exps=p, fmt=2) == -1
    assert fwd(_d(), x=odd) == -5 and fwd(_d(), y=odd) == -5
    assert bwd(_d(), dy=None) == -1 and bwd(_d(), x=None) == -1 and bwd(_d(), exps=p, fmt=-1) == -1
    assert bwd(_d(), dy=odd) == -5 and bwd(_d(), dx=odd) == -5
    for back in (0, 1):
        need = lib.r4c_gn_workspace_size(_d(), back)
        if need:
            assert (bwd if back else fwd)(_d(), nb=need - 1) == -3
    assert fwd(_d(samples=0)) == 0 and fwd(_d(inner=0)) == 0
    for back in (0, 1):                                  # sizes of nothing, and of one voxel
        for change in (dict(samples=0), dict(inner=0), dict(inner=1), dict(inner=1, channels=1, groups=1)):
            assert lib.r4c_gn_workspace_size(_d(**change), back) >= 0
    for fn in (lib.r4c_pack8, ):
        assert fn(p, 8, 5, 0, p, p, None) == -1 and fn(p, 8, 0, 2, p, p, None) == -1 and fn(p, -1, 0, 0, p, p, None) == -1
        assert fn(None, 8, 0, 0, p, p, None) == -1 and fn(p, 8, 0, 0, odd, p, None) == -1
        assert fn(None, 0, 0, 0, None, None, None) == 0
    assert lib.r4c_unpack8(p, p, 8, 7, 0, p, None) == -1 and lib.r4c_unpack8(p, None, 8, 0, 0, p, None) == -1
