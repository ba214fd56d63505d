"""log_probs and distill_topk on the CPU: values, gradients, refusals, strides.

The CPU path computes the same formulas in torch operations; here it is held
to the 64-bit definitions, its gradients to finite differences, and the
argument checks (shared with the CUDA path) to their errors. The descriptor
that the kernels get is checked element by element against the strides.
"""
import itertools

import pytest
import torch

from logit_refs import NEG, assert_grad, assert_values, distill_ref, log_probs_ref, rows_of, unrows
from rdna4_conv3d import _native
from rdna4_conv3d.losses import distill_topk
from rdna4_conv3d.logprobs import log_probs


def _logits(shape, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (3 * torch.randn(shape, generator=g, dtype=torch.float64)).to(dtype)


def _special(c):
    """Rows where a mask leaves everything, something or nothing."""
    z = _logits((9, c), seed=7)
    z[1] = NEG
    z[2, : c // 2] = NEG
    z[3] = NEG
    z[3, c - 1] = 1.5
    z[4] = torch.finfo(torch.float32).min
    z[5] = 0.0
    z[6, 0] = float("nan")
    z[7, c - 1] = float("inf")
    z[8, 0] = 3.0e38
    return z


@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (4, 7), (2, 4, 3, 2, 5), (1, 5, 0, 2, 2), (2, 3, 4)])
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_log_probs_values(shape, temperature):
    z = _logits(shape).requires_grad_(True)
    c = shape[1]
    rows = shape[:1] + shape[2:]
    g = torch.Generator().manual_seed(1)
    t = torch.randint(0, c, rows, generator=g)
    t.view(-1)[::3] = -100
    k = min(c, 3)
    out = log_probs(z, t, top_k=k, temperature=temperature)
    gl, gh, gs = (torch.randn(rows, generator=g, dtype=torch.float64) for _ in range(3))
    dz, = torch.autograd.grad((out.logp, out.entropy, out.lse), z, (gl, gh, gs))
    ref = log_probs_ref(rows_of(z), t.reshape(-1), k, temperature, -100, gl.reshape(-1), gh.reshape(-1), gs.reshape(-1))
    for name in ("logp", "entropy", "lse"):
        assert_values(getattr(out, name).reshape(-1), ref[name], name, 1e-12, 1e-12)
    assert_values(out.top_logp.reshape(-1, k), ref["top_logp"], "top_logp", 1e-12, 1e-12)
    assert torch.equal(out.top_index.reshape(-1, k).long(), ref["top_index"])
    assert out.top_index.dtype == torch.int32 and out.top_logp.shape == (*rows, k)
    assert not out.top_logp.requires_grad
    assert torch.allclose(rows_of(dz), ref["dz"], atol=1e-12)


def test_log_probs_special_rows():
    z = _special(6).requires_grad_(True)
    t = torch.zeros(9, dtype=torch.long)
    out = log_probs(z, t, top_k=6)
    ref = log_probs_ref(z.detach(), t, 6, 1.0, -100, torch.ones(9), torch.ones(9), torch.ones(9))
    for name in ("logp", "entropy", "lse"):
        assert_values(getattr(out, name), ref[name], name, 1e-12, 1e-12)
    assert_values(out.top_logp, ref["top_logp"], "top_logp", 1e-12, 1e-12)
    assert torch.equal(out.top_index.long(), ref["top_index"])
    dz, = torch.autograd.grad((out.logp, out.entropy, out.lse), z, (torch.ones(9, dtype=torch.float64),) * 3)
    fine = [0, 1, 2, 3, 4, 5, 8]                         # a masked label (row 2) still gets its own term
    assert torch.allclose(dz[fine], ref["dz"][fine], atol=1e-12)
    assert out.top_index[6].tolist() == [-1] * 6 and out.top_index[1].tolist() == [0, 1, 2, 3, 4, 5]


def test_log_probs_differences():
    z = _logits((3, 4, 2)).requires_grad_(True)
    t = torch.tensor([[0, 3], [1, -100], [2, 2]])
    assert torch.autograd.gradcheck(lambda x: log_probs(x, t, temperature=1.5)[:3], (z,))
    masked = z.detach().clone()
    masked[0, 1] = NEG
    masked[1, :, 0] = NEG
    masked.requires_grad_(True)
    out = log_probs(masked, t)
    dz, = torch.autograd.grad(out.entropy.sum() + out.logp[2].sum(), masked)
    assert torch.isfinite(dz).all() and float(dz[1, :, 0].abs().max()) == 0.0


def _teacher(rows, c, k, seed=3):
    g = torch.Generator().manual_seed(seed)
    idx = torch.argsort(torch.rand((rows, c), generator=g), 1)[:, :k]
    v = torch.randn((rows, k + 1), generator=g, dtype=torch.float64)
    v = (v - torch.logsumexp(v, 1, keepdim=True))[:, :k]
    return v, idx


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("shape,k", [((1, 1), 1), ((3, 4), 2), ((4, 7), 7), ((2, 5, 3, 1, 2), 3)])
def test_distill_values(shape, k, rest):
    z = _logits(shape).requires_grad_(True)
    rows = shape[:1] + shape[2:]
    n, c = rows_of(z).shape
    v, idx = _teacher(n, c, k)
    idx[0, 0] = -1
    w = torch.rand(n, dtype=torch.float64)
    w[-1] = 0.0 if n > 1 else 1.0
    tv, ti, tw = v.reshape(*rows, k), idx.reshape(*rows, k), w.reshape(rows)
    for weight in (None, tw):
        loss, wsum, dref = distill_ref(rows_of(z), v, idx, 2.0, rest, None if weight is None else w)
        got = distill_topk(z, tv, ti, temperature=2.0, rest=rest, weight=weight, reduction="none")
        assert torch.allclose(got.reshape(-1), loss, atol=1e-12)
        mean = distill_topk(z, tv, ti, temperature=2.0, rest=rest, weight=weight)
        if float(wsum.sum()) == 0.0:
            assert torch.isnan(mean)
            continue
        assert torch.allclose(mean, loss.sum() / wsum.sum(), atol=1e-12)
        dz, = torch.autograd.grad(mean, z)
        assert torch.allclose(rows_of(dz), dref / wsum.sum(), atol=1e-12)


@pytest.mark.parametrize("rest", [False, True])
def test_distill_differences(rest):
    z = _logits((5, 6)).requires_grad_(True)
    v, idx = _teacher(5, 6, 3)
    idx[1, 2] = idx[1, 0]                                # listed twice
    idx[2, 1] = -1
    idx[3] = -1                                          # no pairs at all
    w = torch.tensor([1.0, 0.5, 2.0, 1.0, 0.0], dtype=torch.float64)
    for red in ("mean", "none"):
        assert torch.autograd.gradcheck(
            lambda x: distill_topk(x, v, idx, temperature=1.5, rest=rest, weight=w, reduction=red), (z,))


def test_distill_special_rows():
    z = _logits((4, 5)).requires_grad_(True)
    with torch.no_grad():
        z[0] = NEG                                       # no student: takes no part
        z[1, 2] = NEG                                    # the student rules out a class the teacher lists
        z[2, 1:] = NEG                                   # ... or all the classes it does not list
    v = torch.log(torch.full((4, 2), 0.3, dtype=torch.float64))
    idx = torch.tensor([[0, 1], [2, 3], [0, 0], [1, 4]])
    out = distill_topk(z, v, idx, rest=True, reduction="none")
    assert float(out[0].detach()) == 0.0 and float(out[1].detach()) == float("inf") and float(out[2].detach()) == float("inf")
    assert torch.isfinite(out[3])
    dz, = torch.autograd.grad(out, z, torch.ones(4, dtype=torch.float64))
    assert torch.isfinite(dz).all() and float(dz[0].abs().max()) == 0.0
    _, _, ref = distill_ref(z.detach(), v, idx, 1.0, True)
    assert torch.allclose(dz, ref, atol=1e-12)
    # a teacher that stores its classes with -inf for unused places
    v2 = torch.tensor([[0.0, NEG]], dtype=torch.float64)
    one = distill_topk(_logits((1, 3)), v2, torch.tensor([[1, 0]]))
    assert torch.allclose(one, -torch.log_softmax(_logits((1, 3)), 1)[0, 1])


def test_refusals():
    z = torch.zeros(2, 4, 3)
    t = torch.zeros(2, 3, dtype=torch.long)
    bad = [
        (ValueError, lambda: log_probs(torch.zeros(4))),
        (ValueError, lambda: log_probs(torch.zeros(2, 0))),
        (TypeError, lambda: log_probs(torch.zeros(2, 3, dtype=torch.long))),
        (ValueError, lambda: log_probs(z, t, temperature=0.0)),
        (ValueError, lambda: log_probs(z, t, temperature=float("nan"))),
        (ValueError, lambda: log_probs(z, t, top_k=5)),
        (ValueError, lambda: log_probs(z, t, top_k=-1)),
        (ValueError, lambda: log_probs(torch.zeros(1, 300), top_k=129)),
        (ValueError, lambda: log_probs(z, t[:1])),
        (TypeError, lambda: log_probs(z, t.float())),
        (IndexError, lambda: log_probs(z, t + 4)),
    ]
    v, i = torch.zeros(2, 3, 2), torch.zeros(2, 3, 2, dtype=torch.long)
    bad += [
        (ValueError, lambda: distill_topk(z, v, i, reduction="sum")),
        (ValueError, lambda: distill_topk(z, v[:, :2], i[:, :2])),
        (ValueError, lambda: distill_topk(z, v, i[..., :1])),
        (ValueError, lambda: distill_topk(z, v[..., :0], i[..., :0])),
        (ValueError, lambda: distill_topk(torch.zeros(1, 300), torch.zeros(1, 129), torch.zeros(1, 129, dtype=torch.long))),
        (TypeError, lambda: distill_topk(z, v.long(), i)),
        (TypeError, lambda: distill_topk(z, v, i.to(torch.int16))),
        (ValueError, lambda: distill_topk(z, v, i, weight=torch.ones(2))),
        (ValueError, lambda: distill_topk(z, v, i, temperature=-1.0)),
        (IndexError, lambda: distill_topk(z, v, i + 4)),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()


def _places(desc, rows, c):
    """The element offsets that the kernels compute, (rows, C)."""
    r = torch.arange(rows)[:, None]
    return (r // desc.inner) * desc.outer_stride + (r % desc.inner) * desc.inner_stride + torch.arange(c) * desc.class_stride


@pytest.mark.parametrize("c", [1, 4, 40])
def test_row_descriptors_walk_the_logits(c):
    base = torch.arange(2 * 2 * (c + 3) * 3 * 4 * 5, dtype=torch.float32)
    full = base[: 2 * c * 3 * 4 * 5].view(2, c, 3, 4, 5)
    cl = base[: 2 * c * 3 * 4 * 5].view(2, 3, 4, 5, c).permute(0, 4, 1, 2, 3)
    wide = base[: 2 * (c + 3) * 60].view(2, 3, 4, 5, c + 3).permute(0, 4, 1, 2, 3)
    views = [full, cl, wide[:, 1:c + 1], full[:, :, 1:], cl[:, :, :, 1:2], cl[:, :, ::2], full[1:], cl[..., 0],
             full.transpose(2, 4), base[: 7 * c].view(7, c), base[: 7 * c].view(c, 7).t(),
             base[: 7 * (c + 3)].view(7, c + 3)[:, 2:c + 2], base[:c].view(1, c).expand(6, c), full[:, :, :0]]
    for z in views:
        rows = _native.Rows(z, 1.0)
        n = rows.desc.rows
        assert n == z.shape[0] * torch.Size(z.shape[2:]).numel() and rows.desc.classes == z.shape[1]
        if n == 0:
            continue
        flat = rows.z.as_strided((rows.z.untyped_storage().nbytes() // 4,), (1,), 0)
        got = flat[_places(rows.desc, n, c) + rows.z.storage_offset()]
        assert torch.equal(got, z.movedim(1, -1).reshape(-1, c)), z.stride()
        d = rows.desc
        dz = _native.rows_grad(rows.z, d)
        assert dz.shape == z.shape
        seen = (torch.arange(n)[:, None] // d.inner) * d.grad_outer_stride + \
            (torch.arange(n)[:, None] % d.inner) * d.grad_inner_stride + torch.arange(c) * d.grad_class_stride
        assert sorted(seen.reshape(-1).tolist()) == list(range(n * c))
        want = dz.as_strided((n * c,), (1,)).copy_(torch.arange(n * c, dtype=torch.float32))
        assert want.numel() == n * c and torch.equal(dz.movedim(1, -1).reshape(-1, c), seen.to(torch.float32))
        if c > _native._TILE_CLASSES:
            assert d.class_stride == 1                   # wide rows are read along the classes


def test_shared_gradients_have_increment_zero():
    g, inc = _native._grad_inc(torch.tensor(2.0).expand(3, 4))
    assert inc == 0 and g.numel() == 1
    g, inc = _native._grad_inc(torch.ones(3, 4).t())
    assert inc == 1 and g.is_contiguous()
    assert _native._grad_inc(None) == (None, 0)


def test_c_entries_check_their_arguments():
    L = _native.lib()
    d = _native.RowsDesc(4, 4, 0, 8, 1, 0, 8, 1, 8, _native.R4C_BF16, 1.0)
    null = [None] * 6
    assert L.r4c_logp_fwd(None, *[None] * 2, -100, 0, *null, None) == -1
    assert L.r4c_logp_fwd(d, *[None] * 2, -100, 0, *null, None) == -1
    assert L.r4c_logp_fwd(d, 1 << 20, None, -100, 9, *null, None) == -1          # more than the classes
    assert L.r4c_logp_bwd(d, None, None, -100, None, None, None, 1, None, 1, None, 1, None, None) == -1
    assert L.r4c_distill_fwd(d, None, 0, None, 0, None, 32, 0, *[None] * 4, 0, None) == -1
    for field, value in (("temperature", 0.0), ("temperature", float("inf")), ("classes", 0), ("rows", -1), ("inner", 0)):
        e = _native.RowsDesc(4, 4, 0, 8, 1, 0, 8, 1, 8, _native.R4C_BF16, 1.0)
        setattr(e, field, value)
        assert L.r4c_logp_stats_size(e) == 0 and L.r4c_distill_state_size(e) == 0
        assert L.r4c_logp_fwd(e, *[None] * 2, -100, 0, *null, None) == -1
    e = _native.RowsDesc(0, 1, 0, 8, 1, 0, 8, 1, 8, _native.R4C_BF16, 1.0)
    assert L.r4c_logp_fwd(e, *[None] * 2, -100, 0, *null, None) == 0              # no rows: nothing to do
