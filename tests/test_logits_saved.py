"""What autograd may ask of log_probs and distill_topk beyond a plain backward.

Forward-mode derivatives, which the kernels do not have, are refused. Hooks on saved tensors (``torch.autograd.graph``: offloading, packing) give
the same values back, but with any strides. The kernels read through addresses
and a descriptor, so here, on the CPU and in place of the launch, the
descriptor is walked over the tensors that the launch would get: every place
must lie inside them and hold the row's own value.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.graph import saved_tensors_hooks

from rdna4_conv3d import _native
from rdna4_conv3d.logprobs import LogProbsFn, log_probs
from rdna4_conv3d.losses import DistillTopKFn, distill_topk


def _walk(t, desc, outer, inner, cls):
    """Element offsets of (rows, C) from t's first element, checked against t's storage."""
    r = torch.arange(desc.rows)[:, None]
    at = (r // desc.inner) * outer + (r % desc.inner) * inner + torch.arange(desc.classes) * cls
    room = t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()
    assert int(at.min()) >= 0 and int(at.max()) < room, f"reaches {int(at.max())} of {room}"
    return t.as_strided((room,), (1,))[at]


def _rows(t):
    return t.movedim(1, -1).reshape(-1, t.shape[1])


@pytest.fixture
def launches(monkeypatch):
    """Backward launches are noted as (z, desc, dz, per-row tensors); nothing runs."""
    seen = []

    def note(z, desc, dense):
        dz = _native.rows_grad(z, desc)
        for t in dense:
            assert t is None or t.is_contiguous() and (t.dtype != torch.uint8 or t.data_ptr() % 16 == 0)
        seen.append((z, desc, dz, dense))
        return dz

    monkeypatch.setattr(_native, "_launch", lambda *a: None)
    monkeypatch.setattr(_native, "logp_backward", lambda z, d, target, ign, entropy, stats, *g: note(
        z, d, [target, entropy, stats]))
    monkeypatch.setattr(_native, "distill_backward", lambda z, d, v, i, rest, w, mean, state, g: note(
        z, d, [v, i, w, state]))
    return seen


def _same(t):
    return t


def _dense(t):
    return t.clone(memory_format=torch.contiguous_format)


def _reversed(t):
    """The same values in the opposite memory order."""
    return t.clone().permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))


def _padded(t):
    """The same values inside something wider."""
    if t.dim() == 0:
        return t.clone()
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype)
    wide[..., 1:-2] = t
    return wide[..., 1:-2]


def _views(c):
    g = torch.Generator().manual_seed(c)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"rows": r(5, c), "slice": r(5, c + 14)[:, 1:c + 1], "transposed": r(c, 5).t(), "expanded": r(1, c).expand(5, c),
            "last": r(2, c, 3, 2, 4).contiguous(memory_format=torch.channels_last_3d), "first": r(2, c, 3, 2, 4),
            "cut": r(2, c, 4, 3, 5)[:, :, 1:, :, 1:],
            "wide": r(2, c + 3, 3, 2, 4).contiguous(memory_format=torch.channels_last_3d)[:, 1:c + 1]}


PACKS = pytest.mark.parametrize("pack", [_same, _dense, _reversed, _padded], ids=lambda f: f.__name__[1:])
VIEWS = pytest.mark.parametrize("view", sorted(_views(4)))
CLASSES = pytest.mark.parametrize("c", [1, 4, 40, 1030])


def _checked(launches, logits, dz):
    (z, d, grad, _), = launches
    assert d.rows == _rows(logits).shape[0] and d.classes == logits.shape[1]
    assert torch.equal(_walk(z, d, d.outer_stride, d.inner_stride, d.class_stride), _rows(logits))
    assert d.class_stride == 1 or d.classes <= _native._TILE_CLASSES
    assert dz.shape == logits.shape
    grad.copy_(torch.arange(grad.numel(), dtype=torch.float32).view(grad.shape))
    assert torch.equal(_walk(grad, d, d.grad_outer_stride, d.grad_inner_stride, d.grad_class_stride), _rows(grad))


@CLASSES
@VIEWS
@PACKS
def test_log_probs_reads_the_logits_that_come_back(launches, c, view, pack):
    z = _views(c)[view].requires_grad_(True)
    target = torch.zeros(z.shape[:1] + z.shape[2:], dtype=torch.int64)
    with saved_tensors_hooks(pack, _same):
        out = LogProbsFn.apply(z, target, 1, 2.0, -100)
    dz, = torch.autograd.grad(out[1].sum(), z)
    _checked(launches, z.detach(), dz)


@CLASSES
@VIEWS
@PACKS
def test_distill_reads_the_logits_that_come_back(launches, c, view, pack):
    z = _views(c)[view].requires_grad_(True)
    rows = z.shape[:1] + z.shape[2:]
    v, i, w = torch.zeros(*rows, 3), torch.zeros(*rows, 3, dtype=torch.int32), torch.ones(rows)
    with saved_tensors_hooks(pack, _same):
        loss = DistillTopKFn.apply(z, v, i, 2.0, True, w, True)
    dz, = torch.autograd.grad(loss, z)
    _checked(launches, z.detach(), dz)


@pytest.mark.parametrize("spoil", [lambda t: t.double() if t.is_floating_point() else t.short(), lambda t: t.to("meta"),
                                   lambda t: t.reshape(-1)[:-1]], ids=["type", "device", "shape"])
@pytest.mark.parametrize("which", range(5))
def test_tensors_that_are_not_the_saved_ones_are_refused(launches, which, spoil):
    """A hook that breaks its contract: other types, devices or shapes never reach a kernel."""
    z = torch.randn(6, 1030, requires_grad=True)
    target = torch.zeros(6, dtype=torch.int64)
    v, i, w = torch.zeros(6, 3), torch.zeros(6, 3, dtype=torch.int32), torch.ones(6)
    for f, n in ((lambda: LogProbsFn.apply(z, target, 1, 2.0, -100)[1].sum(), 4),
                 (lambda: DistillTopKFn.apply(z, v, i, 2.0, True, w, True), 5)):
        if which >= n:
            continue
        count = iter(range(100))
        with saved_tensors_hooks(lambda t: spoil(t) if next(count) == which else t, _same):
            y = f()
        with pytest.raises(RuntimeError, match="saved"):
            torch.autograd.grad(y, z)
    assert not launches


class _OnDevice(torch.Tensor):
    """A CPU tensor that calls itself one of a CUDA device: the native path up to its launches."""
    is_cuda = True


@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("c", [5, 1030])
def test_forward_mode_is_refused(launches, c, wants_grad):
    """The kernels carry no tangent; outputs without one would read as a derivative of zero."""
    z = torch.randn(3, c).as_subclass(_OnDevice)
    v, i = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    calls = (lambda x: log_probs(x).entropy, lambda x: distill_topk(x, v, i))
    with fwAD.dual_level():
        x = fwAD.make_dual(z.requires_grad_(wants_grad), torch.ones(3, c))
        assert x.is_cuda and x.requires_grad == wants_grad
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(x)
            call(z.detach())                             # within a level, without a tangent
    for call in calls:
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, (z.detach(),), (torch.ones(3, c),))


def test_forward_mode_on_the_cpu():
    """The torch path has tangents: they agree with the gradient."""
    z, u = torch.randn(3, 7, dtype=torch.float64), torch.randn(3, 7, dtype=torch.float64)
    v, i = torch.log(torch.full((3, 2), 0.3)), torch.tensor([[0, 1]] * 3)
    for call in (lambda x: log_probs(x).entropy.sum(), lambda x: distill_topk(x, v, i, rest=True)):
        tangent = torch.func.jvp(call, (z,), (u,))[1]
        x = z.clone().requires_grad_(True)
        dz, = torch.autograd.grad(call(x), x)
        assert abs(float(tangent) - float((dz * u).sum())) < 1e-12
