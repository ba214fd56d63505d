"""log_probs and distill_topk on a B200 against their 64-bit definitions.

Sizes around every boundary of the kernels (one class, one row, widths that do
not divide into vectors, warps, blocks or clusters), the three types, dense
and strided layouts, masks that leave a row nothing, and gradients.
"""
import pytest
import torch

from logit_refs import NEG, assert_grad, assert_values, distill_ref, log_probs_ref, rows_of

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
DTYPES = pytest.mark.parametrize("dtype", [BF, HF, FP], ids=["bf16", "fp16", "fp32"])
SHAPES = [(1, 1), (1, 2), (5, 3), (700, 4), (33, 5), (300, 7), (257, 8), (9, 12), (65, 16), (70, 17), (31, 31), (64, 32),
          (40, 33), (66, 64), (50, 65), (37, 105), (20, 128), (19, 129), (17, 256), (9, 500), (5, 512), (7, 1000),
          (3, 1024), (3, 1025), (2, 2047), (3, 2048), (2, 4099), (1, 9000), (2, 50021), (1, 131072), (200, 1500), (2, 262147)]
VOLUMES = [(2, 4, 3, 5, 7), (1, 1, 2, 2, 2), (3, 16, 2, 3, 4), (1, 24, 5, 1, 3), (2, 37, 2, 3, 3), (1, 105, 3, 4, 5)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(shape, dtype, seed=0):
    return (3 * torch.randn(shape, device="cuda", generator=_gen(seed))).to(dtype)


def _check_log_probs(z, dtype, k, temperature, seed=1, with_target=True):
    from rdna4_conv3d import _native
    from rdna4_conv3d.logprobs import log_probs
    z = z.detach().requires_grad_(True)
    rows, c = z.shape[:1] + z.shape[2:], z.shape[1]
    g = _gen(seed)
    t = None
    if with_target:
        t = torch.randint(0, c, rows, device="cuda", generator=g)
        t.view(-1)[3::4] = -100
    n0 = _native.launch_count()
    out = log_probs(z, t, top_k=k, temperature=temperature)
    assert _native.launch_count() > n0, "not on the native kernels"
    ups = [torch.randn(rows, device="cuda", generator=g) for _ in range(3)]
    outs = [out.logp, out.entropy, out.lse]
    if not with_target:
        assert out.logp is None
        ups, outs = ups[1:], outs[1:]
    dz, = torch.autograd.grad(outs, z, ups)
    u = [x.cpu().double().reshape(-1) for x in ups]
    if not with_target:
        u = [None] + u
    ref = log_probs_ref(rows_of(z), None if t is None else t.cpu().reshape(-1), k, temperature, -100, *u)
    if with_target:
        assert_values(out.logp.reshape(-1), ref["logp"], "logp")
    assert_values(out.entropy.reshape(-1), ref["entropy"], "entropy")
    assert_values(out.lse.reshape(-1), ref["lse"], "lse")
    if k:
        assert out.top_index.dtype == torch.int32 and tuple(out.top_index.shape) == (*rows, k)
        assert torch.equal(out.top_index.cpu().reshape(-1, k).long(), ref["top_index"])
        assert_values(out.top_logp.reshape(-1, k), ref["top_logp"], "top_logp")
    assert dz.dtype == dtype and dz.shape == z.shape
    assert_grad(rows_of(dz), ref["dz"], dtype)
    assert _native.device_error() == 0
    return out, dz


@DTYPES
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_log_probs_rows(cuda_ready, shape, dtype):
    _check_log_probs(_logits(shape, dtype), dtype, min(shape[1], 5), 1.0)


@DTYPES
@pytest.mark.parametrize("shape", VOLUMES, ids=str)
@pytest.mark.parametrize("layout", ["last", "first", "slice", "cut"])
def test_log_probs_volumes(cuda_ready, shape, dtype, layout):
    n, c, d, h, w = shape
    if layout == "first":
        z = _logits(shape, dtype)
    elif layout == "last":
        z = _logits(shape, dtype).contiguous(memory_format=torch.channels_last_3d)
    elif layout == "slice":                              # classes inside wider voxels
        z = _logits((n, c + 3, d, h, w), dtype).contiguous(memory_format=torch.channels_last_3d)[:, 1:c + 1]
    else:                                                # a crop: voxels that no single stride walks
        z = _logits((n, c, d + 1, h + 1, w + 2), dtype)[:, :, 1:, :h, 1:w + 1]
    _check_log_probs(z, dtype, min(c, 3), 2.0)


@pytest.mark.parametrize("c", [4, 105, 1030, 70001])
@pytest.mark.parametrize("view", ["pitch", "offset", "transposed", "expanded", "batch"])
def test_log_probs_strides(cuda_ready, c, view):
    if view == "pitch":
        z = _logits((5, c + 5), BF)[:, 2:c + 2]
    elif view == "offset":
        z = _logits((5 * c + 1,), BF)[1:].view(5, c)
    elif view == "transposed":
        z = _logits((c, 5), BF).t()
    elif view == "expanded":
        z = _logits((1, c), BF).expand(5, c)
    else:                                                # (B, T, C) tokens with the classes moved to dim 1
        z = _logits((2, 3, c), BF).transpose(1, 2)
    _check_log_probs(z, BF, 4, 1.0)


@DTYPES
@pytest.mark.parametrize("c", [3, 16, 40, 300, 1024, 3000, 40000])
def test_log_probs_special_rows(cuda_ready, c, dtype):
    z = _logits((12, c), dtype)
    low = torch.finfo(dtype).min
    z[1] = NEG
    z[2, : c // 2] = NEG
    z[3] = NEG
    z[3, c - 1] = 1.5
    z[4] = low
    z[5] = 0.0
    z[6, c // 2] = float("nan")
    z[7, c - 1] = float("inf")
    z[8, 0] = torch.finfo(dtype).max
    z[9] = low
    z[9, c // 3] = 2.0
    z[10] = torch.arange(c, device="cuda").to(dtype)     # sorted, with ties where the type runs out of steps
    z[11] = -z[10]
    _check_log_probs(z, dtype, min(c, 20), 1.0)


@pytest.mark.parametrize("c", [20, 128, 1000, 5000, 131072])
def test_log_probs_many_alternatives(cuda_ready, c):
    k = min(c, 128)
    _check_log_probs(_logits((3, c), FP), FP, k, 1.0)
    # the k largest far apart, in one thread's reach, and all over a coarse grid of values
    z = _logits((4, c), FP)
    z[0, :: max(1, c // 31)] += 20.0
    z[1, : min(c, 300)] += 20.0
    z[2] = (z[2] * 0.5).round()
    z[3] = z[3].sign()
    _check_log_probs(z, FP, k, 1.0)


def test_log_probs_concentrated_alternatives(cuda_ready):
    # every stride that a block's threads may walk with: all large values in the same threads
    for step in (4096, 2048, 1024, 512, 8192):
        z = torch.zeros((1, 131072), device="cuda")
        z[0, ::step] = torch.arange(131072 // step, device="cuda") + 1.0
        for j in range(1, 8):
            z[0, j::step] = 0.5
        _check_log_probs(z, FP, 100, 1.0)


def test_log_probs_without_target_and_scales(cuda_ready):
    for c in (6, 200, 3000):
        _check_log_probs(_logits((4, c), BF), BF, 2, 0.5, with_target=False)
        _check_log_probs(_logits((4, c), FP) * 50, FP, 2, 3.0)
        _check_log_probs(_logits((4, c), FP) + 1000, FP, 2, 1.0)


def test_log_probs_partial_gradients(cuda_ready):
    from rdna4_conv3d.logprobs import log_probs
    for c in (5, 100, 5000):
        z = _logits((6, c), FP).requires_grad_(True)
        t = torch.arange(6, device="cuda") % c
        for pick in ("logp", "entropy", "lse"):
            out = log_probs(z, t)
            dz, = torch.autograd.grad(getattr(out, pick).mean(), z, retain_graph=True)   # one shared upstream value
            again, = torch.autograd.grad(getattr(out, pick).mean(), z)
            assert torch.equal(dz, again)
            one = torch.full((6,), 1 / 6).double()
            ups = {"logp": (one, None, None), "entropy": (None, one, None), "lse": (None, None, one)}[pick]
            ref = log_probs_ref(rows_of(z), t.cpu(), 0, 1.0, -100, *ups)
            assert_grad(rows_of(dz), ref["dz"], FP, pick)


@pytest.mark.parametrize("c", [4, 60, 2500])
def test_log_probs_differences(cuda_ready, c):
    """The gradient against central differences of the operator's own values.
    fp32 values carry 2e-6; a step of 2^-6 along a random direction of norm 1
    leaves 2 * 2e-6 * sqrt(rows) / 2^-5 plus the third derivative's 2^-12 / 6."""
    from rdna4_conv3d.logprobs import log_probs
    z = _logits((4, c), FP).requires_grad_(True)
    t = torch.arange(4, device="cuda") % c
    u = torch.randn(z.shape, device="cuda", generator=_gen(5))
    u = u / u.norm()
    f = lambda x: (lambda o: o.logp.double().sum() + 0.5 * o.entropy.double().sum() - 0.25 * o.lse.double().sum())(log_probs(x, t))  # noqa: E731
    dz, = torch.autograd.grad(f(z), z)
    h = 2.0 ** -6
    with torch.no_grad():
        diff = (f(z + h * u) - f(z - h * u)) / (2 * h)
    assert abs(float(diff) - float((dz.double() * u.double()).sum())) <= 1.5e-3


def test_sizes_in_any_order(cuda_ready):
    """One kernel with growing and shrinking tiles: what a launch allows it must not be taken back by another."""
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    for lo, hi in ((33, 63), (66, 127), (129, 255), (260, 511), (520, 1023), (1100, 50021)):
        for n in (1, 40, 900 if hi < 2000 else 20):
            for c in (hi, lo, hi, lo + 1, hi - 2, lo, hi):
                z = torch.zeros(n, c, device="cuda", requires_grad=True)
                v, idx = torch.zeros(n, 3, device="cuda"), torch.arange(3, device="cuda").expand(n, 3)
                o = log_probs(z, top_k=2)
                loss = distill_topk(z, v, idx) + o.entropy.sum()
                dz, = torch.autograd.grad(loss, z)
                assert o.top_index[-1].tolist() == [0, 1]
                assert abs(float(o.lse.detach()[0]) - float(torch.tensor(float(c)).log())) < 1e-4


def test_second_derivatives_are_refused(cuda_ready):
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    z = _logits((3, 5), FP).requires_grad_(True)
    v, idx = _teacher(3, 5, 2)
    for y in (log_probs(z).entropy.sum(), distill_topk(z, v, idx)):
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(y, z, create_graph=True)


def test_log_probs_out_of_range_sets_the_flag(cuda_ready):
    from rdna4_conv3d import _native
    from rdna4_conv3d.logprobs import log_probs
    for c in (4, 100, 5000):
        z = _logits((3, c), BF)
        t = torch.tensor([0, c, -3], device="cuda")
        out = log_probs(z, t)
        assert _native.device_error() == 6
        assert out.logp[1:].tolist() == [0.0, 0.0] and float(out.logp[0]) < 0
        assert _native.device_error() == 0


def test_log_probs_types_and_empty(cuda_ready):
    from rdna4_conv3d.logprobs import log_probs
    z = _logits((0, 4, 2, 2, 2), BF).requires_grad_(True)
    out = log_probs(z, torch.zeros(0, 2, 2, 2, dtype=torch.long, device="cuda"), top_k=2)
    assert out.top_index.shape == (0, 2, 2, 2, 2)
    assert torch.autograd.grad(out.logp.sum(), z)[0].shape == z.shape
    z = _logits((3, 7), HF)
    a = log_probs(z, torch.tensor([1, 2, 3], device="cuda", dtype=torch.int32))
    b = log_probs(z, torch.tensor([1, 2, 3], device="cuda"))
    assert torch.equal(a.logp, b.logp)
    with pytest.raises(TypeError):
        log_probs(z.double())
    with pytest.raises(ValueError):
        log_probs(z, torch.zeros(3, dtype=torch.long))


# ---------------------------------------------------------------------------
def _teacher(rows, c, k, seed=3):
    g = _gen(seed)
    if c <= 4096:
        idx = torch.argsort(torch.rand((rows, c), device="cuda", generator=g), 1)[:, :k]
    else:
        part = c // k
        idx = torch.arange(k, device="cuda") * part + torch.randint(0, part, (rows, k), device="cuda", generator=g)
    v = 2 * torch.randn((rows, k + 1), device="cuda", generator=g)
    v = (v - torch.logsumexp(v, 1, keepdim=True))[:, :k]
    return v.contiguous(), idx.contiguous()


def _check_distill(z, v, idx, temperature, rest, weight=None, reduction="mean", scale=1.0):
    """Loss: each row's terms carry the values' error (2e-5 absolute on a log-probability, weights summing to one)
    times T^2; the mean is no worse than its rows."""
    from rdna4_conv3d import _native
    from rdna4_conv3d.losses import distill_topk
    dtype = z.dtype
    z = z.detach().requires_grad_(True)
    rows = z.shape[:1] + z.shape[2:]
    k = v.shape[-1]
    tv, ti = v.reshape(*rows, k), idx.reshape(*rows, k)
    tw = None if weight is None else weight.reshape(rows)
    n0 = _native.launch_count()
    loss = distill_topk(z, tv, ti, temperature=temperature, rest=rest, weight=tw, reduction=reduction)
    assert _native.launch_count() > n0, "not on the native kernels"
    up = torch.tensor(scale, device="cuda")
    if reduction == "none":
        up = scale * torch.randn(rows, device="cuda", generator=_gen(9))
    dz, = torch.autograd.grad(loss, z, up)
    lref, wref, dref = distill_ref(rows_of(z), v.cpu().double(), idx.cpu(), temperature, rest,
                                   None if weight is None else weight.cpu().double())
    tol = 3e-5 * max(1.0, temperature ** 2) * (1.0 if weight is None else max(1.0, float(weight.max())))
    assert loss.dtype == torch.float32 and dz.dtype == dtype and dz.shape == z.shape
    if reduction == "none":
        assert_values(loss.reshape(-1), lref, "loss", tol, 5e-6)
        assert_grad(rows_of(dz), dref * up.cpu().double().reshape(-1, 1), dtype)
    elif float(wref.sum()) == 0.0:
        assert torch.isnan(loss) and float(dz.abs().max()) == 0.0
    else:
        assert_values(loss.reshape(1), (lref.sum() / wref.sum()).reshape(1), "loss", tol, 5e-6)
        assert_grad(rows_of(dz), dref * scale / wref.sum(), dtype)
    assert _native.device_error() == 0
    return loss, dz


@DTYPES
@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_distill_rows(cuda_ready, shape, rest, dtype):
    n, c = shape
    z = _logits(shape, dtype)
    v, idx = _teacher(n, c, max(1, min(c - 1, 6)))
    scale = 65536.0 if dtype == HF else 1.0
    _check_distill(z, v, idx, 2.0, rest, scale=scale)
    _check_distill(z, v, idx.int(), 1.0, rest, torch.rand(n, device="cuda", generator=_gen(4)) + 0.1, "none")


@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("shape", VOLUMES, ids=str)
@pytest.mark.parametrize("layout", ["last", "first", "slice"])
def test_distill_volumes(cuda_ready, shape, layout, rest):
    n, c, d, h, w = shape
    z = _logits(shape, BF)
    if layout == "last":
        z = z.contiguous(memory_format=torch.channels_last_3d)
    elif layout == "slice":
        z = _logits((n, c + 3, d, h, w), BF).contiguous(memory_format=torch.channels_last_3d)[:, 1:c + 1]
    v, idx = _teacher(n * d * h * w, c, min(c, 3))
    wt = torch.rand(n * d * h * w, device="cuda", generator=_gen(6))
    wt[::5] = 0.0
    _check_distill(z, v, idx, 2.0, rest and c > 3, wt)


@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("c,k", [(32, 31), (128, 128), (300, 128), (1000, 100), (2000, 128), (50021, 128), (131072, 1)])
def test_distill_many_pairs(cuda_ready, c, k, rest):
    v, idx = _teacher(3, c, k)
    _check_distill(_logits((3, c), BF), v, idx, 1.0, rest and k < c)
    for tdt in (BF, HF):                                 # stored in 16 bits; renormalised, so that rounding cannot pass 1
        vv = v.to(tdt).float()
        a = _check_distill(_logits((3, c), FP), vv, idx, 1.0, False)
        from rdna4_conv3d.losses import distill_topk
        b = distill_topk(_logits((3, c), FP), vv.to(tdt), idx)
        assert torch.equal(a[0], b)


@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("c", [8, 40, 600, 5000])
def test_distill_void_and_double_pairs(cuda_ready, c, rest):
    v, idx = _teacher(9, c, 4)
    idx[0, 1:] = -1
    idx[1] = -1                                          # nothing left
    v[2, 2] = NEG
    v[3] = NEG                                           # nothing left
    idx[4, 3] = idx[4, 0]                                # listed twice
    idx[5, :] = idx[5, 0]
    v[5] = torch.log(torch.tensor(0.2, device="cuda"))
    wt = torch.ones(9, device="cuda")
    wt[6] = 0.0
    for red in ("mean", "none"):
        _check_distill(_logits((9, c), FP), v, idx, 1.5, rest, wt, red)
    none = torch.full_like(idx, -1)
    _check_distill(_logits((9, c), BF), v, none, 1.0, rest)      # no row takes part


@DTYPES
@pytest.mark.parametrize("c", [8, 40, 600, 5000, 40000])
def test_distill_special_rows(cuda_ready, c, dtype):
    z = _logits((9, c), dtype)
    low = torch.finfo(dtype).min
    v, idx = _teacher(9, c, 3)
    z[0] = NEG                                           # no student
    z[1, idx[1, 0]] = NEG                                # a listed class ruled out: infinite, gradient finite
    z[2] = NEG
    z[2, idx[2]] = 1.0                                   # the unlisted ones ruled out
    z[3] = low
    z[4, c // 2:] = NEG
    z[4, idx[4]] = 0.5
    z[5, idx[5]] = torch.tensor([60.0, 61.0, 62.0], device="cuda").to(dtype)   # a rest mass far below fp32's step
    z[6] = low
    z[6, idx[6, 0]] = 3.0
    for rest in (False, True):
        _check_distill(z, v, idx, 1.0, rest, None, "none")
    # a poisoned row stays a row: NaN loss and gradient, the others untouched
    z = _logits((3, c), dtype)
    v, idx = _teacher(3, c, 3)
    z[1, c - 1] = float("nan")
    from rdna4_conv3d.losses import distill_topk
    zz = z.clone().requires_grad_(True)
    out = distill_topk(zz, v, idx, rest=True, reduction="none")
    dz, = torch.autograd.grad(out, zz, torch.ones(3, device="cuda"))
    assert torch.isnan(out).tolist() == [False, True, False]
    assert bool(torch.isnan(dz[1]).any()) and bool(torch.isfinite(dz[[0, 2]]).all())


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("c", [4, 60, 2500])
def test_distill_differences(cuda_ready, c, rest):
    """As for log_probs; the loss's terms are its log-probabilities weighted by q <= 1."""
    from rdna4_conv3d.losses import distill_topk
    z = _logits((4, c), FP).requires_grad_(True)
    v, idx = _teacher(4, c, 3)
    u = torch.randn(z.shape, device="cuda", generator=_gen(5))
    u = u / u.norm()
    f = lambda x: distill_topk(x, v, idx, rest=rest, reduction="none").double().sum()  # noqa: E731
    dz, = torch.autograd.grad(f(z), z)
    h = 2.0 ** -6
    with torch.no_grad():
        diff = (f(z + h * u) - f(z - h * u)) / (2 * h)
    assert abs(float(diff) - float((dz.double() * u.double()).sum())) <= 1.5e-3


def test_distill_strided_inputs_and_flag(cuda_ready):
    from rdna4_conv3d import _native
    from rdna4_conv3d.losses import distill_topk
    for c in (6, 200, 3000):
        z = _logits((5, c + 3), BF)[:, 1:c + 1]
        v, idx = _teacher(5, c, 4)
        _check_distill(z, v, idx, 1.0, True)
        wide = torch.zeros(5, 8, device="cuda")
        wide[:, ::2] = v
        wt = torch.rand(1, device="cuda").expand(5) + 0.0
        a = distill_topk(z, wide[:, ::2], idx, weight=wt)
        assert torch.equal(a, distill_topk(z, v, idx, weight=wt.contiguous()))
        over = idx.clone()
        over[2, 1] = c
        gone = idx.clone()
        gone[2, 1] = -1
        b = distill_topk(z, v, over)
        assert _native.device_error() == 6
        assert torch.equal(b, distill_topk(z, v, gone)) and _native.device_error() == 0
    e = distill_topk(_logits((0, 4), BF), v[:0], idx[:0])
    assert torch.isnan(e)


@pytest.mark.parametrize("c", [4, 105, 3000, 131072])
def test_same_results_every_time_and_on_any_stream(cuda_ready, c):
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    n = 3000 if c < 1000 else 40
    z = _logits((n, c), BF).requires_grad_(True)
    t = torch.randint(0, c, (n,), device="cuda")

    def once():
        o = log_probs(z, t, top_k=3)
        loss = distill_topk(z, o.top_logp.detach(), o.top_index, rest=True, temperature=2.0)
        return [*o, loss, *torch.autograd.grad((loss, o.entropy), z, (torch.ones((), device="cuda"), torch.ones(n, device="cuda")))]

    a = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = once()
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_steps_in_a_graph(cuda_ready):
    """Forward and backward captured once, replayed on new values."""
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    for c in (4, 105, 5000):
        z = _logits((64, c), BF).requires_grad_(True)
        v, idx = _teacher(64, c, 3)
        t = torch.arange(64, device="cuda") % c

        def step():
            o = log_probs(z, t, top_k=2)
            loss = distill_topk(z, v, idx, rest=True) + o.entropy.mean()
            return loss.detach(), o.top_index, torch.autograd.grad(loss, z)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        with torch.no_grad():
            z.copy_(_logits((64, c), BF, seed=8))
        graph.replay()
        got = [x.clone() for x in out]
        for x, y in zip(got, step()):
            assert torch.equal(x, y)


@pytest.mark.parametrize("c", [2, 70000])
def test_many_rows_past_32_bits(cuda_ready, c):
    """Rows whose element offsets pass 2^31: the last rows against those rows
    alone (a few long rows are split over blocks, which sums in another order,
    so values agree to the derived bounds and classes exactly)."""
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import distill_topk
    n = (2 ** 31 + 2 ** 20) // c
    z = torch.empty((n, c), dtype=BF, device="cuda").normal_(generator=_gen(1)).requires_grad_(True)
    t = torch.zeros(n, dtype=torch.long, device="cuda")
    o = log_probs(z, t, top_k=1)
    v = torch.zeros(n, 1, device="cuda")
    w = torch.zeros(n, device="cuda")
    w[-3:] = 1.0
    loss = distill_topk(z, v, o.top_index, weight=w)
    dz, = torch.autograd.grad(loss, z)
    tail = z.detach()[-3:].clone().requires_grad_(True)
    p = log_probs(tail, t[-3:], top_k=1)
    for name in ("logp", "entropy", "lse", "top_logp"):
        assert_values(getattr(o, name)[-3:], getattr(p, name).detach().cpu().double(), name)
    assert torch.equal(o.top_index[-3:], p.top_index)
    small = distill_topk(tail, v[-3:], p.top_index)
    assert_values(loss.reshape(1), small.detach().cpu().double().reshape(1), "loss", 3e-5, 5e-6)
    ref, = torch.autograd.grad(small, tail)
    assert_grad(rows_of(dz[-3:]), rows_of(ref), BF)
    assert float(dz[:-3].abs().max()) == 0.0
