"""More definitions in 64 bits for the tests of the operators on rows of logits."""
import math

import torch

from logit_refs import NEG, TINY, ULP


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


def log_probs_rows(z, t, k, temperature, g_logp, g_entropy, g_lse, ignore=-100):
    """The definition in 64 bits over many rows at once, on z's device: z (rows, C) with a finite logit in each row.
    -> dict of logp, entropy, lse, top_logp, top_index, dz, and the size of the terms that a gradient sums."""
    z = z.double()
    d = (z - z.amax(1, keepdim=True)) / temperature
    ln_s = torch.logsumexp(d, 1, keepdim=True)
    ln_p = d - ln_s
    p = ln_p.exp()
    pl = p * ln_p.masked_fill(ln_p == NEG, 0.0)
    h = -pl.sum(1, keepdim=True)
    at = t.clamp(min=0)[:, None]
    counted = (t != ignore)[:, None]
    gl = torch.where(counted, g_logp.double()[:, None], 0.0)
    gh, gs = g_entropy.double()[:, None], g_lse.double()[:, None]
    dz = p * (gs - gl - gh * h) - gh * pl
    dz = dz.scatter_add(1, at, gl) / temperature
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    terms = (gl.abs() + gs.abs() + gh.abs() * (1.0 + math.log(z.shape[1]))) / temperature
    return dict(logp=torch.where(counted, ln_p.gather(1, at), 0.0)[:, 0], entropy=h[:, 0],
                lse=(ln_s[:, 0] + z.amax(1) / temperature), top_logp=ln_p.gather(1, order), top_index=order, dz=dz, terms=terms)


def distill_rows(z, v, idx, temperature, rest, weight):
    """As ``logit_refs.distill_ref`` over many rows at once, on z's device; every row has a finite logit.
    -> w L per row, the weight of the rows that take part, w dL/dz, and the size of the terms that it sums."""
    z, v, idx, w = z.double(), v.double(), idx.long(), weight.double()
    valid = (idx >= 0) & (v > NEG)
    w = torch.where(valid.any(1), w, 0.0)
    idx = idx.clamp(min=0)
    d = (z - z.amax(1, keepdim=True)) / temperature
    ln_p = d - torch.logsumexp(d, 1, keepdim=True)
    lv = v.masked_fill(~valid, NEG)
    if not rest:
        lv = (lv - torch.logsumexp(lv, 1, keepdim=True)).masked_fill(~valid, NEG)
    q = lv.exp()
    loss = torch.where(q > 0, q * (lv.masked_fill(lv == NEG, 0.0) - ln_p.gather(1, idx)), 0.0).sum(1)
    mass = q.sum(1, keepdim=True)
    g = torch.zeros_like(z)
    if rest:
        qr = 1.0 - mass
        qr = torch.where(qr >= 1e-6, qr, 0.0)
        seen = torch.zeros_like(z).scatter_add(1, idx, valid.double()) > 0
        ln_r = ln_p.masked_fill(seen, NEG)
        lse_r = torch.logsumexp(ln_r, 1, keepdim=True)
        loss = loss + torch.where(qr > 0, qr * (qr.clamp(min=1e-300).log() - lse_r), 0.0)[:, 0]
        mass = mass + qr
        g = -qr * (ln_r - lse_r).exp().masked_fill(seen, 0.0)
    g = (g + mass * ln_p.exp()).scatter_add(1, idx, -q)
    on = w != 0
    loss = torch.where(on, w * temperature ** 2 * loss, 0.0)
    g = torch.where(on[:, None], (w * temperature)[:, None] * g, 0.0)
    return loss, w, g, (w * temperature)[:, None]


def assert_gradients(got, want, dtype, terms, name="dz"):
    """got, want (rows, C) on one device, terms (rows, 1): the size of the terms whose difference a gradient is.
    Each term has the relative error of an exponential (2^-22), of its argument (p |t| 2^-23 < 2^-23) and of a
    sum in chains of some hundred (2^-24 times their root, about 2^-20 at most); then one rounding to ``dtype``."""
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    err = torch.nan_to_num(got - want).abs() - ULP[dtype] * torch.nan_to_num(want).abs() - 2.0 ** -19 * terms - TINY[dtype]
    assert err.numel() == 0 or float(err.max()) <= 0, (name, float(err.max()))
