"""Definitions in 64 bits of the operators on rows of logits, for the tests.

Written from the formulas row by row over a (rows, C) matrix, with no use of
the package. ``tol_*`` are the bounds derived from the arithmetic:

* values (fp32): a scaled difference s_c - m is rounded at 2^-24 of its own
  size (at most about 100 here), the hardware exponential at 2^-22, a sum of n
  terms at about sqrt(n) 2^-24 in each of its partial chains (n <= 4096), so
  2e-5 absolute and 2e-6 relative leave a margin of about four;
* gradients: the same relative error on each term, 1e-5 of the row's largest
  entry, and one rounding to the logits' type (2^-9, 2^-12 relative for bf16
  and fp16, doubled for terms that nearly cancel before it), plus fp16's and
  bf16's smallest step.
"""
import torch

NEG = float("-inf")
ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -23}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}


def rows_of(t):
    """(N, C, ...) -> (rows, C) in 64 bits on the CPU."""
    t = t.detach().cpu().double()
    return t.movedim(1, -1).reshape(-1, t.shape[1])


def unrows(t, shape):
    """(rows, C) -> (N, C, ...)."""
    return t.reshape(shape[0], *shape[2:], shape[1]).movedim(-1, 1)


def log_probs_ref(z, target, k, temperature, ignore=-100, g_logp=None, g_entropy=None, g_lse=None):
    """z (rows, C) double, target (rows) or None -> dict of logp, entropy, lse, top_logp, top_index, dz."""
    n, c = z.shape
    out = dict(logp=torch.zeros(n).double(), entropy=torch.zeros(n).double(), lse=torch.full((n,), NEG).double(),
               top_logp=torch.full((n, k), NEG).double(), top_index=torch.zeros(n, k).long(), dz=torch.zeros(n, c).double())
    for r in range(n):
        row = z[r]
        t = -1 if target is None or int(target[r]) == ignore else int(target[r])
        gl = float(g_logp[r]) if g_logp is not None and t >= 0 else 0.0
        gh = float(g_entropy[r]) if g_entropy is not None else 0.0
        gs = float(g_lse[r]) if g_lse is not None else 0.0
        if bool(row.isnan().any()) or bool((row == float("inf")).any()):
            for name in ("entropy", "lse", "top_logp"):
                out[name][r] = float("nan")
            out["logp"][r] = float("nan") if t >= 0 else 0.0
            out["top_index"][r] = -1
            out["dz"][r] = float("nan") if (gl or gh or gs) else 0.0
            continue
        order = sorted(range(c), key=lambda i: (-float(row[i]), i))[:k] if c <= 4096 else \
            torch.sort(row, descending=True, stable=True).indices[:k].tolist()
        if k:
            out["top_index"][r] = torch.tensor(order)
        if bool((row == NEG).all()):
            out["logp"][r] = NEG if t >= 0 else 0.0
            continue
        s = row / temperature
        m = s.max()
        e = torch.exp(s - m)
        lse = m + torch.log(e.sum())
        ln_p = (s - m) - torch.log(e.sum())
        p = torch.exp(ln_p)
        pl = torch.where(p > 0, p * ln_p.clamp(min=-1e300), torch.zeros_like(p))
        h = -pl.sum()
        out["lse"][r], out["entropy"][r] = lse, h
        if t >= 0:
            out["logp"][r] = ln_p[t]
        if k:
            out["top_logp"][r] = ln_p[order]
        g = p * (gs - gl - gh * h) - gh * pl
        if t >= 0:
            g[t] += gl
        out["dz"][r] = g / temperature
    return out


def distill_ref(z, v, idx, temperature, rest, weight=None):
    """z (rows, C), v and idx (rows, k) -> (w L per row, weight of the rows that take part, w dL/dz), double."""
    n, c = z.shape
    loss, wsum, dz = torch.zeros(n).double(), torch.zeros(n).double(), torch.zeros(n, c).double()
    for r in range(n):
        w = 1.0 if weight is None else float(weight[r])
        pairs = [(float(a), int(b)) for a, b in zip(v[r], idx[r]) if int(b) >= 0 and float(a) != NEG]
        if not pairs or w == 0.0 or bool((z[r] == NEG).all()):
            continue
        s = z[r] / temperature
        m = s.max()
        d = s - m                                            # lse would swallow ln S beside the type's lowest values
        ln_s = torch.logsumexp(d, 0)
        ln_p = d - ln_s
        lv = torch.tensor([a for a, _ in pairs], dtype=torch.float64)
        if not rest:
            lv = lv - torch.logsumexp(lv, 0)
        q = torch.zeros(c).double()
        total = 0.0
        for a, (_, b) in zip(lv, pairs):
            qa = torch.exp(a)
            q[b] += qa
            if qa > 0:
                total = total + qa * (a - ln_p[b])
        mass = torch.exp(lv).sum()
        g = -q
        if rest:
            qr = 1.0 - mass
            qr = qr if qr >= 1e-6 else torch.zeros(()).double()
            mass = mass + qr
            un = torch.ones(c, dtype=torch.bool)
            un[[b for _, b in pairs]] = False
            alive = un & (s > NEG)
            ln_r = torch.logsumexp(d[alive], 0) if bool(alive.any()) else torch.tensor(NEG).double()
            if qr > 0:
                total = total + qr * (torch.log(qr) - (ln_r - ln_s))
            if bool(alive.any()):
                g = g - qr * torch.softmax(d.masked_fill(~alive, NEG), 0)     # its own maximum, as above
        g = g + mass * torch.exp(ln_p)
        loss[r] = w * temperature ** 2 * total
        wsum[r] = w
        dz[r] = w * temperature * g
    return loss, wsum, dz


def assert_values(got, want, name, atol=2e-5, rtol=2e-6):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    same = ~fin & ~torch.isnan(want)
    assert torch.equal(got[same], want[same]), name
    err = (got - want)[fin].abs() - (atol + rtol * want[fin].abs())
    assert err.numel() == 0 or float(err.max()) <= 0, (name, float(err.max()))


def assert_grad(got, want, dtype, name="dz"):
    """got, want (rows, C)."""
    got, want = got.detach().cpu().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    over = want.abs() > torch.finfo(dtype).max * (1 + ULP[dtype] / 4)    # what the type rounds to infinity
    assert torch.equal(got[over], torch.sign(want[over]) * float("inf")), name
    want0 = torch.nan_to_num(want.masked_fill(over, 0.0))
    got0 = torch.nan_to_num(got.masked_fill(over, 0.0))
    bound = ULP[dtype] * want0.abs() + 1e-5 * want0.abs().amax(1, keepdim=True) + TINY[dtype]
    worst = float(((got0 - want0).abs() - bound).max()) if want.numel() else 0.0
    assert worst <= 0, (name, worst)
