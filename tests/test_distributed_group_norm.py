"""Group norms of a depth-sharded model on CPU (gloo, two ranks), and what sharding a model keeps of it."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.nn as nn

from test_distributed_gloo import _init, _run, _slab


def _unfused_unet(**kw):
    from rdna4_conv3d.unet3d import unet3d
    torch.manual_seed(3)
    net = unet3d(4, levels=2, n_classes=2, norm="group", groups=2, wmma=False, **kw).double()
    for p in net.parameters():
        nn.init.normal_(p, std=0.3)
    return net


def _data():
    g = torch.Generator().manual_seed(9)
    kw = dict(generator=g, dtype=torch.float64)
    return torch.randn(2, 1, 16, 8, 8, **kw), torch.randn(2, 2, 16, 8, 8, **kw)


def _worker_unfused(rank, port, outdir):
    from rdna4_conv3d.distributed import DepthShardedGroupNormAct3d, GradSync, depth_shard_model
    _init(rank, port)
    try:
        net = _unfused_unet()
        partial = depth_shard_model(net)
        assert sum(isinstance(m, DepthShardedGroupNormAct3d) for m in net.modules()) == 6
        GradSync(partial, average=False)
        x, gy = _data()
        y = net(_slab(x, rank))
        (y * _slab(gy, rank)).sum().backward()
        torch.save({"y": y.detach(), "grads": {n: p.grad.clone() for n, p in net.named_parameters()}},
                   os.path.join(outdir, f"r{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_plain_group_norms_take_the_whole_volume():
    """nn.GroupNorm that no fusing replaced: fp64, against the unsharded model."""
    res = _run(_worker_unfused)
    net = _unfused_unet()
    assert sum(type(m) is nn.GroupNorm for m in net.modules()) == 6
    x, gy = _data()
    y = net(x)
    (y * gy).sum().backward()
    torch.testing.assert_close(torch.cat([r["y"] for r in res], dim=2), y.detach(), rtol=1e-9, atol=1e-9)
    for r in res:
        for n, p in net.named_parameters():
            torch.testing.assert_close(r["grads"][n], p.grad, rtol=1e-8, atol=1e-9, msg=n)


class _OwnNorm(nn.GroupNorm):
    def forward(self, x):
        return super().forward(x) + 1


def test_norms_of_another_class_are_refused():
    """Their forward is not known, so neither is what it would need of the other slabs; nothing is converted."""
    from rdna4_conv3d.distributed import depth_shard_model
    from rdna4_conv3d.group_norm import GroupNormAct3d

    class OwnAct(GroupNormAct3d):
        pass

    for norm in (_OwnNorm(2, 8), OwnAct(2, 8)):
        net = nn.Sequential(nn.Conv3d(8, 8, 3, padding=1), norm)
        with pytest.raises(TypeError, match="cannot be sharded"):
            depth_shard_model(net)
        assert type(net[0]) is nn.Conv3d and net[1] is norm


def _every_kind():
    from rdna4_conv3d.bn_relu import BatchNormReLU3d
    from rdna4_conv3d.group_norm import GroupNormAct3d
    return nn.Sequential(nn.Conv3d(8, 8, 3, padding=1), nn.BatchNorm3d(8), BatchNormReLU3d(8), nn.GroupNorm(2, 8),
                         GroupNormAct3d(4, 8, activation="silu"), nn.Conv3d(8, 8, 1))


def test_sharding_keeps_parameters_statistics_mode_and_hooks():
    """Frozen ones stay frozen, an optimizer's stay its own, eval stays eval; not-frozen convs alone are returned."""
    from rdna4_conv3d.distributed import depth_shard_model
    net = _every_kind().eval()
    net[3].requires_grad_(False)
    net[1].train()
    was = dict(net.named_parameters()), dict(net.named_buffers())
    seen = []
    for i, m in enumerate(net):
        m.register_forward_hook(lambda m, a, y, i=i: seen.append(i))
    partial = depth_shard_model(net)
    now = dict(net.named_parameters()), dict(net.named_buffers())
    for a, b in zip(was, now):
        assert list(a) == list(b) and all(a[k] is b[k] for k in a)
    assert [type(m).__name__[:12] for m in net] == ["DepthSharded"] * 5 + ["Conv3d"]
    assert [m.training for m in net] == [False, True, False, False, False, False]
    assert len(partial) == 2 and partial[0] is net[5].weight and partial[1] is net[5].bias
    # (without a process group the modules take their own slab as the volume; the conv asks for one)
    net[1:](torch.randn(1, 8, 2, 3, 4))
    assert seen == [1, 2, 3, 4, 5]


def test_a_module_used_twice_is_sharded_twice():
    from rdna4_conv3d.distributed import DepthShardedGroupNormAct3d, depth_shard_model
    norm, conv = nn.GroupNorm(2, 8), nn.Conv3d(8, 8, 1)
    net = nn.Sequential(norm, conv, norm, nn.Sequential(norm, conv))
    partial = depth_shard_model(net)
    assert all(isinstance(m, DepthShardedGroupNormAct3d) for m in (net[0], net[2], net[3][0]))
    assert net[0] is net[2] and net[0] is net[3][0]
    assert len(partial) == 2


@pytest.mark.parametrize("root", [0, 1, 2, 3, 4])
def test_a_single_layer_is_refused(root):
    """It cannot be replaced inside itself, and would run unsharded without a word."""
    from rdna4_conv3d.distributed import depth_shard_model
    with pytest.raises(TypeError, match="inside"):
        depth_shard_model(_every_kind()[root])


@pytest.fixture
def alone():
    """A process group of this process alone."""
    import datetime

    from test_distributed_gloo import _free_port
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{_free_port()}", rank=0, world_size=1,
                            timeout=datetime.timedelta(seconds=60))
    yield
    dist.destroy_process_group()


def test_a_second_differentiation_is_refused(alone):
    """It would pass by the sums over the ranks."""
    from rdna4_conv3d.distributed import DepthShardedGroupNormAct3d
    x = torch.randn(1, 8, 2, 3, 4, requires_grad=True)
    y = DepthShardedGroupNormAct3d(2, 8, activation="silu")(x)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def _far(value, dtype):
    x = torch.full((1, 8, 4, 3, 5), value, dtype=dtype)
    x[0, 0, 1, 2, 3] += 0.25                             # one group with a spread
    return x, torch.randn(x.shape, generator=torch.Generator().manual_seed(4)).to(dtype)


def _check_far(value, dtype, y, dx, ulps):
    """(ulps: of the norm's own type; the mean's rounding moves x - mean by half a one of it)"""
    x, dy = _far(value, dtype)
    u = torch.finfo(torch.promote_types(dtype, torch.float32)).eps / 2
    xd, g = (t.double().reshape(1, 4, -1) for t in (x, dy))
    mean = xd.mean(-1, keepdim=True)
    rstd = (((xd - mean) ** 2).mean(-1, keepdim=True) + 1e-5) ** -0.5
    xh = (xd - mean) * rstd
    c = (g * xh).mean(-1, keepdim=True)
    want = rstd * (g - g.mean(-1, keepdim=True) - xh * c)
    e = u * (abs(value) * rstd + ulps * xh.abs())
    assert bool(((y.double().reshape(xh.shape) - xh).abs() <= e).all())
    bound = rstd * (e * c.abs() + xh.abs() * (e * g.abs()).mean(-1, keepdim=True)
                    + ulps * u * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)))
    assert bool(((dx.double().reshape(want.shape) - want).abs() <= bound).all())


def _worker_far(rank, port, outdir):
    from rdna4_conv3d.distributed import DepthShardedGroupNormAct3d
    _init(rank, port)
    try:
        out = []
        for value, dtype in ((30000.0, torch.float32), (1e6, torch.float32), (-1e9, torch.float64)):
            x, dy = (_slab(t, rank) for t in _far(value, dtype))
            x.requires_grad_(True)
            y = DepthShardedGroupNormAct3d(4, 8, affine=False)(x)
            out.append((y.detach(), torch.autograd.grad(y, x, dy)[0]))
        torch.save(out, os.path.join(outdir, f"r{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_statistics_far_from_zero():
    """A slab of one large value: nothing may cancel in the variance over the ranks."""
    res = _run(_worker_far)
    for i, (value, dtype) in enumerate(((30000.0, torch.float32), (1e6, torch.float32), (-1e9, torch.float64))):
        y, dx = (torch.cat([r[i][k] for r in res], dim=2) for k in (0, 1))
        # 16: a few products, and torch's blocked sums of 15 to 30 elements
        _check_far(value, dtype, y, dx, 16)


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("last", [True, False])
def test_an_in_place_activation_may_follow(alone, affine, last):
    """As behind a stock norm; the result lies as the input does."""
    from rdna4_conv3d.distributed import depth_shard_model
    net = nn.Sequential(nn.GroupNorm(2, 8, affine=affine), nn.ReLU(inplace=True)).double()
    x = torch.randn(2, 8, 2, 3, 4, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    if last:
        x = x.contiguous(memory_format=torch.channels_last_3d)
    x.requires_grad_(True)
    want = net(x)
    gx, = torch.autograd.grad((want ** 2).sum(), x)
    depth_shard_model(net)
    y = net(x)
    assert y.stride() == x.stride()
    torch.testing.assert_close(y, want, rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(torch.autograd.grad((y ** 2).sum(), x)[0], gx, rtol=1e-10, atol=1e-10)


def _worker_uneven(rank, port, outdir):
    from rdna4_conv3d.distributed import DepthShardedGroupNormAct3d
    _init(rank, port)
    try:
        out = []
        for cut in (0, 1, 4):                            # planes of the first rank: none, one, all
            x, dy = (t[:, :, :cut] if rank == 0 else t[:, :, cut:] for t in _far(3.0, torch.float64))
            x = x.contiguous().requires_grad_(True)
            norm = DepthShardedGroupNormAct3d(4, 8, activation="silu").double()
            y = norm(x)
            y.backward(dy)
            out.append((y.detach(), x.grad, norm.weight.grad, norm.bias.grad))
        torch.save(out, os.path.join(outdir, f"r{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_slabs_of_any_depth():
    """A rank without a plane of its own takes part all the same."""
    from rdna4_conv3d.group_norm import GroupNormAct3d
    res = _run(_worker_uneven)
    x, dy = _far(3.0, torch.float64)
    norm = GroupNormAct3d(4, 8, activation="silu").double()
    x.requires_grad_(True)
    y = norm(x)
    y.backward(dy)
    kw = dict(rtol=1e-9, atol=1e-9)
    for i in range(3):
        torch.testing.assert_close(torch.cat([r[i][0] for r in res], dim=2), y.detach(), **kw)
        torch.testing.assert_close(torch.cat([r[i][1] for r in res], dim=2), x.grad, **kw)
        for r in res:
            torch.testing.assert_close(r[i][2], norm.weight.grad, **kw)
            torch.testing.assert_close(r[i][3], norm.bias.grad, **kw)
