"""log_probs and distill_topk on a B200 with several rows, or tiles of rows, for each resident block.

The kernels' blocks walk over their rows, reading ahead and clearing what the
last row left in shared memory. Here every row is compared with a 64-bit
definition, with void rows, rows of weight 0 and rows with doubled pairs
between the others, so that each kind follows each.
"""
import pytest
import torch

from logit_edge_refs import assert_gradients, distill_rows, log_probs_rows
from logit_refs import NEG, assert_values
from test_gpu_logits import BF, FP, HF, _gen

pytestmark = pytest.mark.gpu


def _compare(got, want, name, atol=2e-5, rtol=2e-6):
    assert_values(got, want.cpu(), name, atol, rtol)


def _chunks(n, c):
    step = max(1, (1 << 24) // c)
    return [slice(a, min(n, a + step)) for a in range(0, n, step)]


@pytest.mark.parametrize("rest", [False, True], ids=["renorm", "rest"])
@pytest.mark.parametrize("n,c,k,dtype", [
    (12000, 1500, 4, BF),          # a warp a row, every block some rows
    (9000, 1031, 3, FP),
    (3000, 9001, 33, BF),          # 256 threads a row, rows that begin anywhere
    (2500, 9001, 128, HF),
    (1300, 20011, 8, FP),
    (150, 1100003, 5, BF),         # marks too large for one block: clusters of two, two rounds of them
    (150, 530005, 4, FP),
    (300000, 105, 8, BF),          # tiles
    (70000, 105, 20, HF),
    (60000, 300, 40, FP),
    (2500000, 4, 2, BF),
    (2000000, 5, 3, HF),
    (900000, 24, 4, FP),
], ids=str)
def test_distill_many_rows(cuda_ready, n, c, k, dtype, rest):
    from rdna4_conv3d.losses import distill_topk
    g = _gen(n + c)
    z = torch.empty((n, c), dtype=dtype, device="cuda").normal_(0, 2.5, generator=g).requires_grad_(True)
    part = c // k
    idx = torch.arange(k, device="cuda") * part + torch.randint(0, part, (n, k), device="cuda", generator=g)
    kind = torch.randint(0, 8, (n,), device="cuda", generator=g)
    if k > 1:
        idx[:, 1] = torch.where(kind == 1, idx[:, 0], idx[:, 1])                  # listed twice
        idx[:, 0] = torch.where(kind == 2, -1, idx[:, 0])                         # one place unused
    idx = torch.where((kind == 3)[:, None], -1, idx)                              # none used
    idx = idx.to(torch.int32)
    v = torch.empty((n, k + 1), device="cuda").normal_(0, 2, generator=g)
    v = (v - torch.logsumexp(v, 1, keepdim=True))[:, :k].contiguous()
    v = torch.where((kind == 5)[:, None] & (torch.arange(k, device="cuda") == k - 1), NEG, v)
    w = torch.rand(n, device="cuda", generator=g) + 0.1
    w[kind == 4] = 0.0
    w[0], idx[0] = 1.0, torch.arange(k, device="cuda", dtype=torch.int32)
    loss = distill_topk(z, v, idx, temperature=1.5, rest=rest, weight=w, reduction="none")
    up = torch.empty(n, device="cuda").normal_(generator=g)
    dz, = torch.autograd.grad(loss, z, up)
    mean = distill_topk(z, v, idx, temperature=1.5, rest=rest, weight=w)
    dm, = torch.autograd.grad(mean, z)
    total, weight = 0.0, 0.0
    refs = []
    for r in _chunks(n, c):
        lr, wr, gr, terms = distill_rows(z.detach()[r], v[r], idx[r], 1.5, rest, w[r])
        _compare(loss[r], lr, "loss", 3e-5 * 1.5 ** 2 * 1.1, 5e-6)
        assert_gradients(dz[r], gr * up[r].double()[:, None], dtype, terms * up[r].double().abs()[:, None])
        total, weight = total + lr.sum(), weight + wr.sum()
        refs.append((r, gr, terms) if n * c < 1 << 27 else None)
    _compare(mean.reshape(1), (total / weight).reshape(1), "mean", 3e-5 * 1.5 ** 2 * 1.1, 5e-6)
    for ref in refs:
        if ref:
            r, gr, terms = ref
            assert_gradients(dm[r], gr / weight, dtype, terms / weight)


@pytest.mark.parametrize("k", [0, 1, 2, 20])
@pytest.mark.parametrize("n,c,dtype", [
    (12000, 1500, BF), (9000, 1031, FP), (3000, 9001, BF), (2500, 9001, HF), (1300, 20011, FP), (700, 40001, BF),
    (300000, 105, BF), (70000, 105, HF), (60000, 300, FP), (2500000, 4, BF), (2000000, 5, HF), (900000, 24, FP),
    (400000, 31, BF), (30000, 1000, BF),
], ids=str)
def test_log_probs_many_rows(cuda_ready, n, c, dtype, k):
    from rdna4_conv3d.logprobs import log_probs
    if k > c:
        k = c
    g = _gen(n + c + k)
    z = torch.empty((n, c), dtype=dtype, device="cuda").normal_(0, 2.5, generator=g)
    kind = torch.randint(0, 8, (n,), device="cuda", generator=g)
    z = torch.where((kind == 1)[:, None], z.round(), z)                           # ties
    z = torch.where((kind == 2)[:, None], torch.zeros_like(z), z)                 # nothing but ties
    z = torch.where((kind == 3)[:, None] & (torch.arange(c, device="cuda") % 3 != 0), torch.full_like(z, NEG), z)
    z.requires_grad_(True)
    t = torch.randint(0, c, (n,), device="cuda", generator=g)
    t = torch.where(kind == 3, t - t % 3, t)                                      # a class that is not masked
    t = torch.where(kind == 4, -100, t)
    ups = [torch.empty(n, device="cuda").normal_(generator=g) for _ in range(3)]
    out = log_probs(z, t, top_k=k, temperature=1.5)
    dz, = torch.autograd.grad(out[:3], z, ups)
    for r in _chunks(n, c):
        ref = log_probs_rows(z.detach()[r], t[r], k, 1.5, *(u[r] for u in ups))
        for name in ("logp", "entropy", "lse"):
            _compare(getattr(out, name)[r], ref[name], name)
        if k:
            assert torch.equal(out.top_index[r].long(), ref["top_index"])
            _compare(out.top_logp[r], ref["top_logp"], "top_logp")
        assert_gradients(dz[r], ref["dz"], dtype, ref["terms"])
