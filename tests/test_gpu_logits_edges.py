"""log_probs and distill_topk on a B200 where rows, layouts or callers are unusual.

Each test compares with the 64-bit definitions, or with another call of the
same operator that the definitions say is the same.
"""
from contextlib import nullcontext

import pytest
import torch

from logit_edge_refs import assert_gradients, no_rest_ref, stored, student
from logit_refs import NEG, assert_grad, assert_values, distill_ref, log_probs_ref, rows_of
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


# ---- the pairs that log_probs returns: int32 classes with fp32 log-probabilities -----------------------------
def _check_pairs(z, v, idx, temperature, rest, weight=None):
    """Row losses and gradients with int32 classes; the gradient's bound counts the terms that cancel in it."""
    from rdna4_conv3d import _native
    from rdna4_conv3d.losses import distill_topk
    z = z.detach().requires_grad_(True)
    rows, k = z.shape[:1] + z.shape[2:], v.shape[-1]
    ti = idx.int().view(*rows, k)
    wt = None if weight is None else weight.view(rows)
    loss = distill_topk(z, v.view(*rows, k), ti, temperature=temperature, rest=rest, weight=wt, reduction="none")
    up = torch.randn(rows, device="cuda", generator=_gen(9))
    dz, = torch.autograd.grad(loss, z, up)
    w = torch.ones(rows.numel()).double() if weight is None else weight.cpu().double()
    want, _, dwant = distill_ref(rows_of(z), v.cpu().double(), idx.cpu(), temperature, rest, w)
    u = up.cpu().double().reshape(-1, 1)
    assert_values(loss.reshape(-1), want, "loss", 3e-5 * max(1.0, temperature ** 2) * max(1.0, float(w.max())), 5e-6)
    assert_gradients(rows_of(dz), dwant * u, z.dtype, temperature * w[:, None] * u.abs())
    assert _native.device_error() == 0
    same = distill_topk(z, v.view(*rows, k), ti.long(), temperature=temperature, rest=rest, weight=wt, reduction="none")
    assert torch.equal(torch.isnan(loss), torch.isnan(same))
    assert_values(loss.reshape(-1), same.detach().cpu().double().reshape(-1), "int64", 6e-5 * max(1.0, temperature ** 2), 1e-5)


RESTS = pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])


@RESTS
@DTYPES
@pytest.mark.parametrize("k", [1, 2, 3, 4, 6, 8])
@pytest.mark.parametrize("c", [8, 9, 24, 31, 40, 105, 600, 5000])
def test_int32_pairs_void_and_double(cuda_ready, c, k, dtype, rest):
    v, idx = _teacher(11, c, k)
    idx[0, 1:] = -1
    idx[1] = -1                                          # nothing left
    v[2, k // 2] = NEG
    v[3] = NEG                                           # nothing left
    idx[4, k - 1] = idx[4, 0]                            # listed twice, in the lanes' first and last places
    idx[5, :] = idx[5, 0].clone()
    v[5] = -2.5
    if k > 2:
        idx[7, 1] = idx[7, 0]                            # neighbours
        idx[8, 2] = idx[8, 0]
        idx[8, 1] = -1
    idx[9, 0] = -7
    wt = torch.ones(11, device="cuda")
    wt[6] = 0.0
    _check_pairs(_logits((11, c), dtype), v, idx, 1.5, rest, wt)


@RESTS
@DTYPES
@pytest.mark.parametrize("k", [2, 3, 4])
@pytest.mark.parametrize("c", [8, 9, 40, 105, 600, 5000, 40000])
def test_int32_pairs_special_rows(cuda_ready, c, k, dtype, rest):
    z = _logits((9, c), dtype)
    low = torch.finfo(dtype).min
    v, idx = _teacher(9, c, k)
    z[0] = NEG                                           # no student
    z[1, idx[1, 0]] = NEG                                # a listed class ruled out
    z[2] = NEG
    z[2, idx[2]] = 1.0                                   # the unlisted ones ruled out
    z[3] = low
    z[4, c // 2:] = NEG
    z[4, idx[4]] = 0.5
    z[5, idx[5]] = 60.0 + torch.arange(k, device="cuda").to(dtype)
    z[6] = low
    z[6, idx[6, 0]] = 3.0
    _check_pairs(z, v, idx, 1.0, rest)


@RESTS
@pytest.mark.parametrize("c,k", [(32, 31), (33, 32), (64, 40), (128, 128), (200, 64), (300, 128), (1000, 100), (2000, 128),
                                 (50021, 127)])
def test_int32_pairs_many(cuda_ready, c, k, rest):
    v, idx = _teacher(5, c, k)
    idx[1, k - 1] = idx[1, 0]
    idx[2, k // 2:] = -1
    idx[3, ::2] = idx[3, :1]
    v[3] -= 1.0                                          # (their sum stays below 1)
    for dtype in (BF, FP):
        _check_pairs(_logits((5, c), dtype), v, idx, 1.0, rest and k < c)


@RESTS
@pytest.mark.parametrize("k", [1, 2, 3, 4])
@pytest.mark.parametrize("layout", ["last", "first", "slice", "cut", "odd"])
@pytest.mark.parametrize("shape", [(2, 4, 3, 5, 7), (3, 16, 2, 3, 4), (1, 24, 5, 1, 3), (2, 37, 2, 3, 3), (2, 5, 4, 3, 9)], ids=str)
def test_int32_pairs_volumes(cuda_ready, shape, layout, k, rest):
    n, c, d, h, w = shape
    if layout == "first":
        z = _logits(shape, BF)
    elif layout == "last":
        z = _logits(shape, BF).contiguous(memory_format=torch.channels_last_3d)
    elif layout == "slice":
        z = _logits((n, c + 3, d, h, w), BF).contiguous(memory_format=torch.channels_last_3d)[:, 1:c + 1]
    elif layout == "cut":
        z = _logits((n, c, d + 1, h + 1, w + 2), BF)[:, :, 1:, :h, 1:w + 1]
    else:                                                # dense rows that begin two bytes off
        z = _logits((n * d * h * w * c + 1,), BF)[1:].view(n, d, h, w, c).permute(0, 4, 1, 2, 3)
    v, idx = _teacher(n * d * h * w, c, k)
    wt = torch.rand(n * d * h * w, device="cuda", generator=_gen(6))
    wt[::5] = 0.0
    _check_pairs(z, v, idx, 2.0, rest and k < c, wt)


# ---- two alternatives -----------------------------------------------------------------------------------------
@DTYPES
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("c", [2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 105, 1000])
def test_two_alternatives(cuda_ready, c, offset, dtype):
    """The two largest of a short row come from one pass: ties, masks, signs of zero, rows with nothing and bad rows,
    among rows that begin in the middle of a word (an odd number of 16-bit classes, or an odd start)."""
    from rdna4_conv3d.logprobs import log_probs
    n, low, inf = 400, torch.finfo(dtype).min, float("inf")
    z = _logits((n * c + offset,), dtype)[offset:].view(n, c)
    a, b = 0, c - 1
    z[0] = 0.0
    z[1] = NEG
    z[2] = NEG
    z[2, b] = 1.0                                        # the second is the first masked class
    z[3] = NEG
    z[3, a] = -1.0
    z[4] = low
    z[5] = z[5, 0]                                       # all equal
    z[6, b] = z[6].max()                                 # the largest twice, or once at the end
    z[7, a] = z[7].max()
    z[8] = 0.0
    z[8, ::2] = -0.0                                     # equal, whatever their sign
    z[9, c // 2] = float("nan")
    z[10, a] = float("nan")
    z[11, b] = inf
    z[12] = NEG
    z[12, b] = float("nan")
    z[13] = torch.arange(c, device="cuda").to(dtype)
    z[14] = -torch.arange(c, device="cuda").to(dtype)
    z[15] = low
    z[15, a] = NEG
    z[16:200] = z[16:200].round()
    z[200:300, : c // 2] = NEG
    out = log_probs(z, top_k=2, temperature=2.0)
    ref = log_probs_ref(rows_of(z), None, 2, 2.0)
    assert torch.equal(out.top_index.cpu().long(), ref["top_index"])
    for name in ("entropy", "lse", "top_logp"):
        assert_values(getattr(out, name), ref[name], name)
    three = log_probs(z, top_k=min(3, c), temperature=2.0)
    assert torch.equal(three.top_index[:, :2], out.top_index)
    # places for the pairs that are not 8-byte aligned take the general way
    if offset:
        from rdna4_conv3d import _native
        rows = _native.Rows(z, 2.0)
        tl, ti = torch.zeros(n * 2 + 1, device="cuda"), torch.zeros(n * 2 + 1, dtype=torch.int32, device="cuda")
        e, s = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        L = _native.lib()
        assert L.r4c_logp_fwd(rows.desc, rows.z.data_ptr(), None, -100, 2, None, e.data_ptr(), s.data_ptr(),
                              tl[1:].data_ptr(), ti[1:].data_ptr(), None, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(ti[1:].view(n, 2), out.top_index)
        assert_values(tl[1:].view(n, 2), ref["top_logp"], "unaligned")
