"""log_probs and distill_topk on a B200 where rows, layouts or callers are unusual.

Each test compares with the 64-bit definitions, or with another call of the
same operator that the definitions say is the same.
"""
from contextlib import nullcontext

import pytest
import torch

from logit_edge_refs import no_rest_ref, stored, student
from logit_refs import NEG, assert_grad, assert_values, log_probs_ref, rows_of
from test_gpu_logits import BF, DTYPES, FP, HF, _check_distill, _gen, _logits, _teacher

pytestmark = pytest.mark.gpu


def _transposed_copy(t):
    """The same values in the opposite memory order."""
    back = tuple(reversed(range(t.dim())))
    return t.clone().permute(back).contiguous().permute(back)


@pytest.mark.parametrize("hooks", ["cpu", "pinned", "transposed"])
@pytest.mark.parametrize("c", [4, 105, 1030])
@pytest.mark.parametrize("view", ["slice", "last", "first", "wide"])
def test_gradients_under_saved_tensor_hooks(cuda_ready, view, c, hooks):
    """Saved tensors that come back with other strides: each row's gradient is that of the same call without hooks.
    Other places of a row's classes in the kernels' lanes add its sums in another order, hence the derived bounds."""
    from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    if view == "slice":
        z = _logits((5, c + 14), BF)[:, 3:c + 3]
    elif view == "last":
        z = _logits((2, c, 3, 4, 5), BF).contiguous(memory_format=torch.channels_last_3d)
    elif view == "first":
        z = _logits((2, c, 3, 4, 5), BF)
    else:
        z = _logits((2, c + 3, 3, 4, 5), BF).contiguous(memory_format=torch.channels_last_3d)[:, 1:c + 1]
    z.requires_grad_(True)
    rows = z.shape[:1] + z.shape[2:]
    t = torch.randint(0, c, rows, device="cuda", generator=_gen(2))
    v, idx = _teacher(rows.numel(), c, 3)
    v, idx = v.view(*rows, 3), idx.view(*rows, 3)
    wt = torch.rand(rows, device="cuda", generator=_gen(3))

    def grads(hook):
        with hook():
            o = log_probs(z, t, temperature=2.0)
            loss = distill_topk(z, v, idx, temperature=2.0, rest=c > 4, weight=wt, reduction="none")
        a, = torch.autograd.grad(o.logp.sum() - o.entropy.sum(), z)
        b, = torch.autograd.grad(loss.sum(), z)
        return rows_of(a), rows_of(b)

    hook = {"cpu": save_on_cpu, "pinned": lambda: save_on_cpu(pin_memory=True),
            "transposed": lambda: saved_tensors_hooks(_transposed_copy, lambda x: x)}[hooks]
    for got, want in zip(grads(hook), grads(nullcontext)):
        assert_grad(got, want, BF)


@DTYPES
@pytest.mark.parametrize("c", [4, 7, 105, 1000, 3000])
def test_a_bad_row_without_upstream_gradient_has_none(cuda_ready, c, dtype):
    """0 times NaN is not a gradient: rows that hold a NaN or +inf and are ignored (or whose upstream values are all
    zero) leave the weights alone; with an upstream gradient they are NaN; so it is in the 64-bit definition."""
    from rdna4_conv3d.logprobs import log_probs
    z = _logits((8, c), dtype)
    z[1, c // 2] = float("nan")
    z[2, c - 1] = float("inf")
    z[3] = float("nan")
    z[4, 0] = float("nan")
    z[5] = NEG
    z.requires_grad_(True)
    t = torch.arange(8, device="cuda") % c
    t[1:4] = -100
    ones, zeros = torch.ones(8).double(), torch.zeros(8).double()
    out = log_probs(z, t)
    dz, = torch.autograd.grad(out.logp.sum(), z)
    ref = log_probs_ref(rows_of(z), t.cpu(), 0, 1.0, -100, ones)
    assert not ref["dz"][1:4].any() and bool(ref["dz"][4].isnan().all())
    assert_grad(rows_of(dz), ref["dz"], dtype)
    out = log_probs(z, t)
    gh = ones.clone()
    gh[[1, 3, 4]] = 0.0
    dz, = torch.autograd.grad((out.logp, out.entropy), z, (zeros.float().cuda(), gh.float().cuda()))
    assert_grad(rows_of(dz), log_probs_ref(rows_of(z), t.cpu(), 0, 1.0, -100, zeros, gh)["dz"], dtype)


@pytest.mark.parametrize("shape", [(0, 4), (2, 4, 0, 3, 3), (2, 4, 3, 0, 3), (2, 4, 3, 3, 0), (2, 40, 3, 0, 0), (2, 1030, 2, 0)],
                         ids=str)
def test_empty_maps(cuda_ready, shape):
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    z = torch.zeros(shape, dtype=BF, device="cuda", requires_grad=True)
    rows = z.shape[:1] + z.shape[2:]
    out = log_probs(z, torch.zeros(rows, dtype=torch.long, device="cuda"), top_k=2)
    assert out.logp.shape == rows and out.top_index.shape == (*rows, 2)
    assert torch.autograd.grad(out.entropy.sum(), z)[0].shape == z.shape
    v, idx = torch.zeros((*rows, 3), device="cuda"), torch.zeros((*rows, 3), dtype=torch.int32, device="cuda")
    for rest in (False, True):
        none = distill_topk(z, v, idx, rest=rest, reduction="none")
        assert none.shape == rows and torch.autograd.grad(none.sum(), z)[0].shape == z.shape
        mean = distill_topk(z, v, idx, rest=rest)
        assert torch.isnan(mean) and torch.autograd.grad(mean, z)[0].shape == z.shape


TEACHERS = pytest.mark.parametrize("stored_as", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])


@TEACHERS
@pytest.mark.parametrize("wide", [False, True], ids=["int32", "int64"])
@pytest.mark.parametrize("c,k", [(2, 2), (4, 4), (5, 5), (20, 20), (128, 128), (40, 7), (300, 128), (1030, 20), (9001, 128)])
def test_a_stored_teacher_that_lists_all_there_is(cuda_ready, c, k, wide, stored_as):
    """As on the CPU: no class is left, so the stored values' rounding is no mass of a rest."""
    from rdna4_conv3d.losses import distill_topk
    v, idx = stored(c, k, 40, stored_as)
    z = student(c, k, idx).cuda().requires_grad_(True)
    loss = distill_topk(z, v.cuda(), (idx if wide else idx.int()).cuda(), temperature=2.0, rest=True, reduction="none")
    want, dwant = no_rest_ref(z.detach().cpu().double(), v.double(), idx, 2.0)
    assert_values(loss, want, "loss", 1.2e-4, 5e-6)
    dz, = torch.autograd.grad(loss.sum(), z)
    assert_grad(dz, dwant, FP)


@TEACHERS
@pytest.mark.parametrize("wide", [False, True], ids=["int32", "int64"])
@pytest.mark.parametrize("c", [12, 200, 3000])
def test_a_stored_teacher_that_does_not(cuda_ready, c, wide, stored_as):
    from rdna4_conv3d.losses import distill_topk
    v, idx = stored(c, 6, 50, stored_as)
    v = (v.double() + torch.log(torch.tensor(0.8).double())).to(stored_as)
    ti = (idx if wide else idx.int()).cuda()
    _check_distill(_logits((50, c), FP), v.float().cuda(), ti, 1.0, True, None, "none")
    z = _logits((50, c), FP).requires_grad_(True)
    loss = distill_topk(z, v.cuda(), ti, rest=True, reduction="none")
    same = distill_topk(z, v.float().cuda(), ti, rest=True, reduction="none")
    assert_values(loss, same.detach().cpu().double(), "loss", 3e-5, 5e-6)
    out = distill_topk(student(c, 6, idx).cuda(), v.cuda(), ti, rest=True, reduction="none")
    assert bool(torch.isinf(out).all())


@pytest.mark.parametrize("c", [5, 2000])
def test_forward_mode_is_refused(cuda_ready, c):
    import torch.autograd.forward_ad as fwAD
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    z = _logits((3, c), FP)
    v, idx = _teacher(3, c, 2)
    for call in (lambda x: log_probs(x).entropy, lambda x: distill_topk(x, v, idx)):
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(fwAD.make_dual(z, torch.ones_like(z)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(call, (z,), (torch.ones_like(z),))
        # nor does any other transform see through the kernels: none goes by in silence
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(z[None])
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x: call(x).sum())(z)


@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("c", [6, 2000])
def test_traces_run_the_operators_again(cuda_ready, c, wants_grad):
    """A trace computes from the inputs that it is given, or there is none."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    z, more = _logits((4, c), BF).requires_grad_(wants_grad), _logits((4, c), BF, seed=8).requires_grad_(wants_grad)
    v, idx = _teacher(4, c, 2)
    for f in (lambda x: log_probs(x, top_k=2).entropy * 2, lambda x: log_probs(x, top_k=2).top_logp * 2,
              lambda x: distill_topk(x, v, idx) * 2):
        want = f(more)
        assert torch.equal(torch.jit.trace(f, (z,), check_trace=False)(more), want)
        torch._dynamo.reset()
        assert torch.equal(torch.compile(f, backend="eager")(more), want)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(z)
