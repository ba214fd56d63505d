"""Train a small UNet3D on a larger one's two likeliest labels per voxel.

The larger network (base 32) labels volumes once: ``log_probs(..., top_k=2)``
gives, per voxel, its two most probable classes with their log-probabilities
and the entropy that says how sure it is -- 16 bytes a voxel, stored instead of
full logits. The smaller one (base 24) then trains on that store:
``distill_topk`` with one bucket for the other classes, plus the ordinary
cross-entropy on the labels, under bf16 autocast. Confidence weights (voxels
the teacher is unsure of count less) come from the entropy.

    python examples/distill_unet3d.py [--steps 40] [--size 64 128 128]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-conv3d-wmma_b200"))

from rdna4_conv3d.logprobs import log_probs  # noqa: E402
from rdna4_conv3d.losses import cross_entropy, distill_topk  # noqa: E402
from rdna4_conv3d.unet3d import unet3d  # noqa: E402


def export(teacher, x, k=2, temperature=2.0):
    """(log-probabilities, classes, weights) of a teacher's k best classes per voxel."""
    with torch.no_grad(), torch.autocast(x.device.type, dtype=torch.bfloat16):
        logits = teacher(x)
    out = log_probs(logits, top_k=k, temperature=temperature)
    weight = 1.0 - 0.5 * out.entropy / math.log(logits.shape[1])
    return out.top_logp, out.top_index, weight


def step(student, opt, x, labels, store, temperature=2.0, alpha=0.7):
    """One training step; returns the loss."""
    top_logp, top_index, weight = store
    opt.zero_grad(set_to_none=True)
    with torch.autocast(x.device.type, dtype=torch.bfloat16):
        logits = student(x)
        loss = alpha * distill_topk(logits, top_logp, top_index, temperature=temperature, rest=True, weight=weight)
        loss = loss + (1.0 - alpha) * cross_entropy(logits, labels)
    loss.backward()
    opt.step()
    return loss.detach()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--size", type=int, nargs=3, default=(64, 128, 128))
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--device", default="cuda")
    a = ap.parse_args(argv)
    dev = torch.device(a.device)
    torch.manual_seed(0)
    on_gpu = dev.type == "cuda"
    teacher, student = unet3d(32, wmma=on_gpu, device=dev), unet3d(24, wmma=on_gpu, device=dev)
    teacher.train(False)
    x = torch.randn(a.batch, 1, *a.size, device=dev).contiguous(memory_format=torch.channels_last_3d)
    labels = torch.randint(0, 4, (a.batch, *a.size), device=dev)
    store = export(teacher, x)
    opt = torch.optim.Adam(student.parameters(), lr=1e-3)
    losses = [step(student, opt, x, labels, store) for _ in range(a.steps)]
    student.train(False)
    with torch.no_grad(), torch.autocast(dev.type, dtype=torch.bfloat16):
        seen = log_probs(student(x), labels, top_k=1)
    agree = (seen.top_index[..., 0] == store[1][..., 0]).float().mean()
    print(f"loss {float(losses[0]):.4f} -> {float(losses[-1]):.4f}; agrees with the teacher on "
          f"{100 * float(agree):.1f} % of voxels; mean entropy {float(seen.entropy.mean()):.3f}")
    return [float(v) for v in losses]


if __name__ == "__main__":
    main()
