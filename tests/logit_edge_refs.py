"""More definitions in 64 bits for the tests of the operators on rows of logits."""
import torch

from logit_refs import NEG


def no_rest_ref(z, v, idx, temperature):
    """Distillation with the teacher's pairs as they are and no class beside them that counts:
    L = T^2 sum q (ln q - ln p), dL/dz = T (Q p - q). z (rows, C), v and idx (rows, k), all pairs valid -> (L, dL/dz)."""
    d = (z - z.amax(1, keepdim=True)) / temperature
    ln_p = d - torch.logsumexp(d, 1, keepdim=True)
    q = torch.exp(v)
    loss = temperature ** 2 * (q * (v - ln_p.gather(1, idx))).sum(1)
    g = q.sum(1, keepdim=True) * torch.exp(ln_p)
    return loss, temperature * g.scatter_add(1, idx, -q)


def stored(c, k, rows, dtype, seed=0):
    """A teacher that gives all its mass to k of c classes, as it is stored in ``dtype``: (v, idx)."""
    g = torch.Generator().manual_seed(seed)
    s = 3 * torch.randn((rows, k), generator=g, dtype=torch.float64)
    s[0] = 0.0                                           # uniform: every rounding has the same sign
    s[1, 0] += 30.0                                      # sure of one class
    idx = torch.argsort(torch.rand((rows, c), generator=g), 1)[:, :k]
    return torch.log_softmax(s, 1).to(dtype), idx


def student(c, k, idx, seed=1):
    """Logits (fp32) whose classes beyond the listed ones are ruled out."""
    z = 3 * torch.randn((idx.shape[0], c), generator=torch.Generator().manual_seed(seed))
    return z if k == c else torch.full_like(z, NEG).scatter(1, idx, z.gather(1, idx))
