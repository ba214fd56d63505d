"""The distillation example: the log-probability and distillation operators together in a training run."""
import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

from conftest import ROOT


def _example():
    spec = importlib.util.spec_from_file_location("distill_unet3d", os.path.join(ROOT, "examples", "distill_unet3d.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_example_on_cpu():
    losses = _example().main(["--device", "cpu", "--steps", "2", "--batch", "1", "--size", "16", "16", "16"])
    assert len(losses) == 2 and all(map(lambda v: v == v and v > 0, losses))


@pytest.mark.gpu
def test_example_learns_on_the_kernels(cuda_ready):
    from rdna4_conv3d import _native
    n0 = _native.launch_count()
    losses = _example().main(["--steps", "12", "--batch", "2", "--size", "16", "32", "32"])
    assert _native.launch_count() > n0 and _native.device_error() == 0
    assert losses[-1] < losses[0]


@pytest.mark.gpu
def test_step_gradient_matches_plain_torch(cuda_ready):
    """The example's loss on given logits against the same loss in plain fp32 torch."""
    from rdna4_conv3d.logprobs import log_probs
    from rdna4_conv3d.losses import cross_entropy, distill_topk
    g = torch.Generator(device="cuda").manual_seed(0)
    shape = (2, 4, 8, 16, 16)
    z = (2 * torch.randn(shape, device="cuda", generator=g)).to(torch.bfloat16)
    z = z.contiguous(memory_format=torch.channels_last_3d).requires_grad_(True)
    t = (2 * torch.randn(shape, device="cuda", generator=g)).to(torch.bfloat16)
    labels = torch.randint(0, 4, (2, 8, 16, 16), device="cuda", generator=g)
    out = log_probs(t.contiguous(memory_format=torch.channels_last_3d), top_k=2, temperature=2.0)
    loss = 0.7 * distill_topk(z, out.top_logp, out.top_index, temperature=2.0, rest=True) + 0.3 * cross_entropy(z, labels)
    loss.backward()
    zr = z.detach().float().requires_grad_(True)
    q = torch.log_softmax(t.float() / 2, 1).exp().movedim(1, -1)
    lp = torch.log_softmax(zr / 2, 1).movedim(1, -1)
    top = q.topk(2, -1)
    rest_q = 1 - top.values.sum(-1)
    keep = torch.ones_like(q).scatter(-1, top.indices, 0.0)
    rest_p = torch.logsumexp(lp.masked_fill(keep == 0, float("-inf")), -1)
    kl = (top.values * (top.values.log() - lp.gather(-1, top.indices))).sum(-1) + rest_q * (rest_q.log() - rest_p)
    ref = 0.7 * 4 * kl.mean() + 0.3 * F.cross_entropy(zr, labels)
    ref.backward()
    # two bf16 gradients, each rounded once, then their sum once more
    assert abs(float(loss.detach()) - float(ref.detach())) <= 2e-5 * abs(float(ref.detach())) + 2e-5
    err = (z.grad.float() - zr.grad).abs().max()
    assert float(err) <= 3 * 2.0 ** -8 * float(zr.grad.abs().max())
