"""log_probs and distill_topk on the CPU where rows, types or callers are unusual."""
import pytest
import torch

from logit_edge_refs import no_rest_ref, stored, student
from logit_refs import NEG, assert_grad, assert_values, distill_ref, log_probs_ref, rows_of
from rdna4_conv3d import _native
from rdna4_conv3d.losses import distill_topk
from rdna4_conv3d.logprobs import log_probs

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _teacher(rows, c, k, seed=3):
    idx = torch.argsort(torch.rand((rows, c), generator=_gen(seed)), 1)[:, :k]
    v = torch.randn((rows, k + 1), generator=_gen(seed + 1))
    return (v - torch.logsumexp(v, 1, keepdim=True))[:, :k], idx


@DTYPES
@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
def test_distill_of_large_logits(dtype, rest, temperature):
    """Rows far from zero, where a log-sum-exp of the logits themselves swallows ln S; fp32 arithmetic, so the
    bounds of the kernels: 3e-5 T^2 absolute and 5e-6 relative for a loss."""
    top, low = torch.finfo(dtype).max, torch.finfo(dtype).min
    c = 8
    z = 3 * torch.randn((9, c), generator=_gen(0))
    z[0] = min(1e9, top)
    z[1] = low
    z[2] += 3e4
    z[3] -= 3e4
    z[4] = top
    z = z.to(dtype)
    v, idx = _teacher(9, c, 3)
    z[5] = low                                           # the unlisted classes far below the listed ones
    z[5, idx[5]] = torch.tensor([0.0, 1.0, 2.0]).to(dtype)
    z[6] = 1.0
    z[6, idx[6]] = low / 2                               # ... and far above them
    z[7] = NEG
    z[7, :4] = low
    z[8, idx[8]] = NEG
    z.requires_grad_(True)
    loss = distill_topk(z, v, idx, temperature=temperature, rest=rest, reduction="none")
    dz, = torch.autograd.grad(loss, z, torch.ones(9))
    want, _, dwant = distill_ref(rows_of(z), v.double(), idx, temperature, rest)
    want = torch.where(want > torch.finfo(torch.float32).max, torch.full_like(want, float("inf")), want)
    assert_values(loss, want, "loss", 3e-5 * temperature ** 2, 5e-6)
    assert_grad(rows_of(dz), dwant, dtype)


EMPTY = [(0, 4), (0, 4, 2, 2, 2), (2, 4, 0, 3, 3), (2, 4, 3, 0, 3), (2, 4, 3, 3, 0), (2, 4, 0), (2, 40, 3, 0, 0), (2, 1030, 2, 0),
         (1, 1, 0)]


@pytest.mark.parametrize("layout", ["first", "last", "cut"])
@pytest.mark.parametrize("shape", EMPTY, ids=str)
def test_empty_maps_have_a_descriptor(shape, layout):
    z = torch.zeros(shape)
    if layout == "last":
        z = z.movedim(1, -1).contiguous().movedim(-1, 1)
    elif layout == "cut":
        z = torch.zeros([s + 1 for s in shape])[tuple(slice(0, s) for s in shape)]
    rows = _native.Rows(z, 1.0)
    assert rows.desc.rows == 0 and rows.desc.classes == shape[1] and rows.desc.inner > 0
    assert rows.shape == z.shape[:1] + z.shape[2:] and rows.z.shape == z.shape
    assert shape[1] <= 1024 or rows.desc.class_stride == 1
    assert _native.rows_grad(rows.z, rows.desc).shape == z.shape
    assert shape[1] <= 1024 or rows.desc.grad_class_stride == 1


def test_the_c_entry_of_distill_takes_no_rows():
    """An empty tensor has a null address: the rows' losses of no rows are nothing to write."""
    L = _native.lib()
    d = _native.RowsDesc(0, 1, 0, 8, 1, 0, 8, 1, 8, _native.R4C_BF16, 1.0)
    nothing = [None] * 2
    assert L.r4c_distill_fwd(d, None, 2, None, _native.R4C_F32, None, 32, 0, None, *nothing, None, 0, None) == 0
    assert L.r4c_distill_fwd(d, None, 0, None, _native.R4C_F32, None, 32, 0, None, *nothing, None, 0, None) == -1
    d.rows, d.inner = 4, 4                               # rows, and no place for their losses
    one = torch.zeros(16)
    at = one.data_ptr()
    assert L.r4c_distill_fwd(d, at, 2, at, _native.R4C_F32, at, 32, 0, None, *nothing, None, 0, None) == -1


@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("gap", [0.1, 1e-3, 1e-6])
def test_distill_gradient_where_the_student_agrees(gap, rest):
    """p - q of fp32 logits close to the teacher's own: rounded once, not left to the roundings of p and q."""
    want_p = torch.log_softmax(3 * torch.randn((300, 2), generator=_gen(0), dtype=torch.float64), 1).float()
    z = (want_p + gap * torch.randn((300, 2), generator=_gen(1))).requires_grad_(True)
    idx = torch.tensor([1, 0]).expand(300, 2)
    v = want_p[:, [1, 0]]
    loss = distill_topk(z, v, idx, rest=rest, reduction="none")
    dz, = torch.autograd.grad(loss.sum(), z)
    _, _, want = distill_ref(rows_of(z), v.double(), idx, 1.0, rest)
    assert_grad(dz, want, torch.float32)


TEACHERS = pytest.mark.parametrize("stored_as", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])


@TEACHERS
@pytest.mark.parametrize("c,k", [(2, 2), (5, 5), (20, 20), (128, 128), (40, 7)])
def test_a_stored_teacher_that_lists_all_there_is(c, k, stored_as):
    """What its rounding leaves of 1 is not mass on classes that the student does not have; fp32 arithmetic,
    the kernels' bounds."""
    v, idx = stored(c, k, 400, stored_as)
    z = student(c, k, idx).requires_grad_(True)
    loss = distill_topk(z, v, idx, temperature=2.0, rest=True, reduction="none")
    want, dwant = no_rest_ref(z.detach().double(), v.double(), idx, 2.0)
    assert_values(loss, want, "loss", 1.2e-4, 5e-6)
    dz, = torch.autograd.grad(loss.sum(), z)
    assert_grad(dz, dwant, torch.float32)


@TEACHERS
def test_a_stored_teacher_that_does_not(stored_as):
    """Missing mass beyond the rounding still counts: against live classes as it is, against none as infinite."""
    v, idx = stored(12, 6, 50, stored_as)
    v = (v.double() + torch.log(torch.tensor(0.8).double())).to(stored_as)
    z = 3 * torch.randn((50, 12), generator=_gen(2))
    loss = distill_topk(z, v, idx, rest=True, reduction="none")
    assert_values(loss, distill_ref(z.double(), v.double(), idx, 1.0, True)[0], "loss", 3e-5, 5e-6)
    assert torch.isinf(distill_topk(student(12, 6, idx), v, idx, rest=True, reduction="none")).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64], ids=["fp32", "fp64"])
def test_gradients_of_bad_rows(dtype):
    """NaN for a row of NaN or +inf logits that has an upstream gradient, as on a CUDA device; 0 for one that has none."""
    z = 3 * torch.randn((9, 6), generator=_gen(4), dtype=torch.float64)
    z[1, 2] = z[4, 0] = z[6, 5] = float("nan")
    z[2, 5] = z[7, 1] = float("inf")
    z[3] = float("nan")
    z[5] = NEG
    z = z.to(dtype).requires_grad_(True)
    t = torch.arange(9) % 6
    t[1:4] = -100
    ones = torch.ones(9, dtype=torch.float64)
    some = ones.clone()
    some[[4, 7]] = 0.0
    for gl, gh, gs in ((ones, None, None), (None, some, None), (None, None, some), (some, some, None), (ones, ones, ones),
                       (some, 0 * ones, some)):
        out = log_probs(z, t)
        ups = [(o, g) for o, g in zip(out[:3], (gl, gh, gs)) if g is not None]
        dz, = torch.autograd.grad([o for o, _ in ups], z, [g.to(o.dtype) for o, g in ups])
        assert_grad(dz, log_probs_ref(rows_of(z), t, 0, 1.0, -100, gl, gh, gs)["dz"], torch.float32)


def test_log_probs_in_transforms():
    """On the CPU the operator stays a composition that torch can transform."""
    z, u = torch.randn(2, 3, 7, dtype=torch.float64), torch.randn(2, 3, 7, dtype=torch.float64)
    f = lambda x: (lambda o: o.entropy.sum() + o.lse.sum())(log_probs(x))  # noqa: E731
    each = torch.stack([f(x) for x in z])
    assert torch.allclose(torch.func.vmap(f)(z), each)
    dz = torch.func.vmap(torch.func.grad(f))(z)
    assert torch.allclose(torch.func.jvp(torch.func.vmap(f), (z,), (u,))[1], (dz * u).sum((1, 2)))
    assert torch.autograd.gradgradcheck(f, (z[0].clone().requires_grad_(True),))


def test_a_rest_over_too_many_classes_is_refused():
    """The marks of the listed classes of one row fill the shared memory of a cluster at about four million classes."""
    L = _native.lib()
    one = torch.zeros(16)
    at, state = one.data_ptr(), torch.zeros(1 << 17, dtype=torch.uint8)
    sp = (state.data_ptr() + 15) // 16 * 16

    def call(c, rest):
        d = _native.RowsDesc(0, 1, 0, c, 1, 0, c, 1, c, _native.R4C_BF16, 1.0)
        return L.r4c_distill_fwd(d, at, 2, at, _native.R4C_F32, at, 32, rest, None, at, None, sp, 1 << 16, None)

    too_large = -7
    assert [call(c, 1) for c in (1 << 20, 4000000, 5000000)] == [0, 0, too_large] and call(5000000, 0) == 0
    assert "four million" in distill_topk.__doc__
