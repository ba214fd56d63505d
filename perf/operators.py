"""Workloads of the log-probability and distillation operators, for timing and comparing.

``listed()`` names them, ``draw(rng)`` gives more of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run``
makes one pass: in elementary fp32 torch operations, or, where the module's
``own`` is true, through ``rdna4_conv3d``. ``exact`` is the definition in
64 bits, ``work`` the bytes and operations that a pass cannot do without.

Two operators:

* ``log_probs`` -- per row of logits (a voxel of an (N, C, D, H, W) map, or a
  token of an (R, C) matrix): log-probability of the given label, entropy,
  log-sum-exp and the ``k`` most probable classes; with ``grad`` also the
  logits' gradient for given gradients of log-probability and entropy.
* ``distill_topk`` -- the weighted mean over rows of T^2 KL(teacher || student)
  where the teacher is given by ``k`` log-probabilities and classes per row,
  renormalised or with one bucket for all other classes (``rest``), and the
  logits' gradient.
"""
import os
import sys

import torch

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rdna4-conv3d-wmma_b200")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_IGNORE = -100
_NOISE = 1e-6      # a rest mass below this is the rounding of the teacher's sum


def _case(op, n, classes, dtype, k, d=0, h=0, w=0, layout="last", temperature=1.0, grad=False, rest=False,
          weighted=False, pad=0, ragged=False):
    return dict(op=op, n=n, classes=classes, d=d, h=h, w=w, dtype=dtype, k=k, layout=layout, temperature=temperature,
                grad=grad, rest=rest, weighted=weighted, pad=pad, ragged=ragged)


def listed():
    lp, ds = "log_probs", "distill_topk"
    return [
        # a server answers one new token with its alternatives: latency counts
        dict(_case(lp, 1, 131072, "bf16", 20), name="lp one token"),
        # one decoding step of an uneven batch, fp32 logits, the padded end of the classes masked
        dict(_case(lp, 37, 50021, "fp32", 5, pad=21), name="lp decode batch"),
        # scoring whole prompts with a few alternatives
        dict(_case(lp, 2048, 131072, "bf16", 4), name="lp prompts"),
        # a policy's update: log-probability and entropy of the chosen classes and the gradient; odd rows and classes
        dict(_case(lp, 4095, 32771, "bf16", 0, grad=True), name="lp policy update"),
        # the segmentation network's own output: per-voxel confidence and the two likeliest labels (a teacher's export)
        dict(_case(lp, 4, 4, "bf16", 2, 64, 128, 128, temperature=2.0), name="lp voxels"),
        # a labelling of many structures, fp16, trained on log-probabilities
        dict(_case(lp, 1, 105, "fp16", 0, 48, 96, 80, grad=True), name="lp many labels"),
        # the stock dense layout (classes outermost), fp32
        dict(_case(lp, 2, 16, "fp32", 3, 32, 64, 64, layout="first"), name="lp classes first"),
        # a small classifier's batch: latency counts
        dict(_case(ds, 8, 1000, "fp32", 10, temperature=2.0), name="ds small batch"),
        # training on stored teacher distributions over a large vocabulary; the largest
        dict(_case(ds, 4096, 131072, "bf16", 64, rest=True), name="ds vocabulary"),
        # packed sequences: masked rows, rows with fewer stored classes or none, odd sizes
        dict(_case(ds, 511, 50021, "fp16", 32, temperature=2.0, weighted=True, ragged=True), name="ds ragged"),
        # the segmentation network distilled from a larger one
        dict(_case(ds, 4, 4, "bf16", 2, 64, 128, 128, temperature=2.0, rest=True), name="ds voxels"),
        # many structures, voxels weighted (borders, unlabelled regions)
        dict(_case(ds, 1, 105, "bf16", 8, 48, 96, 80, temperature=4.0, weighted=True), name="ds many labels"),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(("log_probs", "distill_topk"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    temperature = rng.choice((1.0, 1.0, 1.5, 2.0, 4.0))
    most = 1 << 28                                       # logits of a drawn case: half of the largest listed one's
    if rng.random() < 0.4:                               # volumes: a few to some hundred labels
        c = log_int(2, 300)
        vox = min(most // 4 // c, log_int(4000, 4 << 20))
        n = rng.choice((1, 2, 4))
        w = log_int(7, 160)
        h = log_int(7, 160)
        d = max(1, vox // (n * w * h))
        shape = dict(n=n, d=d, h=h, w=w, layout=rng.choice(("last", "last", "first")) if c <= 32 else "last")
    else:                                                # rows of classes
        c = log_int(500, 200000)
        shape = dict(n=max(1, min(most // c, log_int(1, 8192))))
    k = min(c, log_int(1, 64)) if op == "distill_topk" else min(c, rng.choice((0, 1, 2, 5, 10, 20)))
    more = dict(grad=rng.random() < 0.4, pad=rng.choice((0, 0, min(c // 4, 17))) if c > 64 else 0)
    if op == "distill_topk":
        more = dict(rest=k < c and rng.random() < 0.5, weighted=rng.random() < 0.5, ragged=rng.random() < 0.3)
    return _case(op, classes=c, dtype=dtype, k=k, temperature=temperature, **shape, **more)


def _shape(case):
    n, c = case["n"], case["classes"]
    return (n, c, case["d"], case["h"], case["w"]) if case["d"] else (n, c)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    shape, c, k = _shape(case), case["classes"], case["k"]
    out_shape = shape[:1] + shape[2:]
    rows = 1
    for v in out_shape:
        rows *= v
    dt = _DTYPES[case["dtype"]]
    kw = dict(device=dev, generator=g)
    z = torch.randn((rows, c), dtype=dt, **kw).mul_(2.5)
    idx = None
    if case["op"] == "distill_topk":                     # distinct classes: one out of each of k equal parts, rotated
        part = c // k
        idx = torch.arange(k, device=dev) * part + torch.randint(0, part, (rows, k), **kw)
        idx = (idx + torch.randint(0, c, (rows, 1), **kw)) % c
        z.scatter_add_(1, idx, torch.full((1, 1), 3.0, dtype=dt, device=dev).expand(rows, k))
    else:                                                # trained rows are peaked
        for _ in range(3):                               # one after the other: two of them may be the same class
            few = torch.randint(0, c, (rows, 1), **kw)
            z.scatter_add_(1, few, torch.rand((rows, 1), **kw).mul_(9.0).to(dt))
    if case["pad"]:
        z[:, c - case["pad"]:] = float("-inf")
    if len(shape) == 5:
        z = z.reshape(shape[0], *shape[2:], c).permute(0, 4, 1, 2, 3)
        if case["layout"] == "first":
            z = z.contiguous()
    state = dict(case=dict(case), logits=z, temperature=case["temperature"])
    if case["op"] == "log_probs":
        t = torch.randint(0, c - case["pad"], (rows,), **kw)
        t[torch.rand(rows, **kw) < 0.05] = _IGNORE
        state["target"] = t.reshape(out_shape)
        if case["grad"]:
            # an update's gradients: advantages over the rows, a small entropy bonus, the loss scale of fp16 training
            scale = (65536.0 if dt == torch.float16 else 1.0) / rows
            state["g_logp"] = (torch.randn(rows, **kw) * scale).reshape(out_shape)
            state["g_entropy"] = torch.full((rows,), -0.01 * scale, device=dev).reshape(out_shape)
            state["logits"].requires_grad_(True)
    else:
        v = torch.randn((rows, k + 1), **kw).mul_(2.0)
        v = (v - torch.logsumexp(v, 1, keepdim=True))[:, :k].sort(1, descending=True).values
        idx = idx.to(torch.int32)
        if case["ragged"]:                               # rows with fewer classes stored, some with none
            have = torch.randint(0, k + 1, (rows, 1), **kw)
            have[0] = k
            gone = torch.arange(k, device=dev) >= have
            idx = idx.masked_fill(gone, -1)
            v = v.masked_fill(gone, float("-inf"))
        state["teacher_logp"] = v.reshape(*out_shape, k).contiguous()
        state["teacher_index"] = idx.reshape(*out_shape, k).contiguous()
        state["weight"] = None
        if case["weighted"]:
            wt = torch.rand(rows, **kw)
            wt[wt < 0.2] = 0.0
            wt[0] = 1.0
            state["weight"] = wt.reshape(out_shape)
        state["scale"] = torch.tensor(65536.0 if dt == torch.float16 else 1.0, device=dev)
        state["logits"].requires_grad_(True)
    return state


def run(state):
    case = state["case"]
    if case["op"] == "log_probs":
        return _run_log_probs(state, case) if own else _plain_log_probs(state, case)
    return _run_distill(state, case) if own else _plain_distill(state, case)


def _run_log_probs(s, case):
    from rdna4_conv3d.logprobs import log_probs
    out = log_probs(s["logits"], s["target"], top_k=case["k"], temperature=s["temperature"], ignore_index=_IGNORE)
    res = dict(logp=out.logp, entropy=out.entropy, lse=out.lse)
    if case["k"]:
        res.update(top_logp=out.top_logp, top_index=out.top_index)
    if case["grad"]:
        res["dlogits"], = torch.autograd.grad((out.logp, out.entropy), (s["logits"],), (s["g_logp"], s["g_entropy"]))
    return res


def _run_distill(s, case):
    from rdna4_conv3d.losses import distill_topk
    loss = distill_topk(s["logits"], s["teacher_logp"], s["teacher_index"], temperature=s["temperature"],
                        rest=case["rest"], weight=s["weight"])
    dlogits, = torch.autograd.grad((loss,), (s["logits"],), (s["scale"],))
    return dict(loss=loss, dlogits=dlogits)


def _rows(t):
    """(N, C, ...) -> (rows, C), classes last."""
    return t.detach().movedim(1, -1).reshape(-1, t.shape[1])


def _unrows(t, like):
    """(rows, C) -> the logits' own shape, layout and type."""
    t = t.to(like.dtype)
    if like.dim() == 2:
        return t
    t = t.reshape(like.shape[0], *like.shape[2:], like.shape[1]).movedim(-1, 1)
    return t.contiguous() if like.is_contiguous() else t


def _plain_log_probs(s, case):
    z0 = s["logits"]
    z = _rows(z0).float()
    zt = z / s["temperature"]
    t = s["target"].reshape(-1)
    shape = s["target"].shape
    m = zt.amax(1, keepdim=True)
    e = torch.exp(zt - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    p = e / total
    ln_p = zt - lse
    pln = torch.where(p > 0, p * ln_p, 0.0)
    h = -pln.sum(1)
    counted = t != _IGNORE
    at = t.clamp(min=0)[:, None]
    logp = torch.where(counted, ln_p.gather(1, at)[:, 0], 0.0)
    res = dict(logp=logp.reshape(shape), entropy=h.reshape(shape), lse=lse.reshape(shape))
    k = case["k"]
    if k:
        # unique 64-bit keys: the value's order above, the class below, so that ties go to the lowest class
        bits = (z + 0.0).view(torch.int32)
        order = torch.where(bits < 0, ~bits ^ (-2 ** 31), bits).long()
        key = order * 2 ** 32 + (2 ** 31 - torch.arange(z.shape[1], device=z.device))
        key = torch.topk(key, k, dim=1).values
        top = 2 ** 31 - key % 2 ** 32
        res["top_logp"] = ln_p.gather(1, top).reshape(*shape, k)
        res["top_index"] = top.to(torch.int32).reshape(*shape, k)
    if case["grad"]:
        gl = torch.where(counted, s["g_logp"].reshape(-1), 0.0)[:, None]
        gh = s["g_entropy"].reshape(-1)[:, None]
        dz = -gl * p - gh * (pln + p * h[:, None])
        dz = dz.scatter_add(1, at, gl) / s["temperature"]
        res["dlogits"] = _unrows(dz, z0)
    return res


def _plain_distill(s, case):
    z0, tau = s["logits"], s["temperature"]
    z = _rows(z0).float() / tau
    k = case["k"]
    v = s["teacher_logp"].reshape(-1, k)
    idx = s["teacher_index"].reshape(-1, k).long()
    valid = (idx >= 0) & (v > float("-inf"))
    idx = idx.clamp(min=0)
    w = torch.ones_like(z[:, 0]) if s["weight"] is None else s["weight"].reshape(-1)
    w = torch.where(valid.any(1), w, 0.0)
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = m + torch.log(total)
    if case["rest"]:
        q = torch.where(valid, torch.exp(v), 0.0)
    else:
        top = torch.where(valid, v, -1e30)
        q = torch.where(valid, torch.exp(top - top.amax(1, keepdim=True)), 0.0)
        q = q / q.sum(1, keepdim=True).clamp(min=1e-30)
    ln_q = torch.log(torch.where(q > 0, q, 1.0))
    ln_p = z.gather(1, idx) - lse
    row = torch.where(q > 0, q * (ln_q - ln_p), 0.0).sum(1)
    mass = q.sum(1, keepdim=True)
    dz = None
    if case["rest"]:
        qr = 1.0 - mass
        qr = torch.where(qr >= _NOISE, qr, 0.0)
        listed_ = torch.zeros_like(z).scatter_add(1, idx, valid.float()) > 0
        zr = torch.where(listed_, float("-inf"), z)
        mr = zr.amax(1, keepdim=True)
        er = torch.exp(zr - mr)
        tr = er.sum(1, keepdim=True)
        lse_r = mr + torch.log(tr)
        row = row + torch.where(qr > 0, qr * (torch.log(torch.where(qr > 0, qr, 1.0)) - (lse_r - lse)), 0.0)[:, 0]
        mass = mass + qr
        dz = mass * e / total - qr * er / tr
    else:
        dz = mass * e / total
    dz = dz.scatter_add(1, idx, -q)
    # losses and weights summed in 64 bits: the rows are many
    loss = (tau * tau * (row * w).double().sum() / w.double().sum()).float()
    dz = dz * (tau * s["scale"] * w / w.double().sum().float())[:, None]
    return dict(loss=loss, dlogits=_unrows(dz, z0))


def exact(case, seed):
    s = prepare(case, seed)
    z0 = s["logits"].detach()
    zall = z0.movedim(1, -1).reshape(-1, z0.shape[1])
    rows, c = zall.shape
    shape = z0.shape[:1] + z0.shape[2:]
    tau, k = s["temperature"], case["k"]
    step = max(1, (1 << 26) // c)
    parts, sums, weights = [], 0.0, 0.0
    if case["op"] == "distill_topk":
        full_w = torch.ones(rows, dtype=torch.float64, device=z0.device)
        if s["weight"] is not None:
            full_w = s["weight"].reshape(-1).double()
        ti = s["teacher_index"].reshape(-1, k).long()
        tv = s["teacher_logp"].reshape(-1, k).double()
        full_w = full_w * ((ti >= 0) & (tv > float("-inf"))).any(1)
        weights = full_w.sum()
    for a in range(0, rows, step):
        r = slice(a, min(rows, a + step))
        z = zall[r].double().requires_grad_(True)
        ls = torch.log_softmax(z / tau, 1)
        if case["op"] == "log_probs":
            t = s["target"].reshape(-1)[r]
            logp = torch.where(t == _IGNORE, 0.0, ls.gather(1, t.clamp(min=0)[:, None])[:, 0])
            ent = -(ls.exp() * ls.masked_fill(ls == float("-inf"), 0.0)).sum(1)
            got = [logp.detach(), ent.detach(), torch.logsumexp(z.detach() / tau, 1)]
            if k:
                got.append(ls.detach().topk(k, 1).values)
            if case["grad"]:
                up = (s["g_logp"].reshape(-1)[r].double(), s["g_entropy"].reshape(-1)[r].double())
                got.append(torch.autograd.grad((logp, ent), z, up)[0])
        else:
            i, v, w = ti[r], tv[r], full_w[r]
            ok = (i >= 0) & (v > float("-inf"))
            v = v.masked_fill(~ok, float("-inf"))
            if not case["rest"]:
                v = (v - torch.logsumexp(v, 1, keepdim=True)).masked_fill(~ok, float("-inf"))
            i = i.clamp(min=0)
            q = v.exp()
            row = torch.where(ok, q * (v.masked_fill(~ok, 0.0) - ls.gather(1, i)), 0.0).sum(1)
            if case["rest"]:
                qr = 1.0 - q.sum(1)
                qr = torch.where(qr >= _NOISE, qr, 0.0)
                seen = torch.zeros(z.shape, device=z.device).scatter_add(1, i, ok.float()) > 0
                lr = torch.logsumexp(ls.masked_fill(seen, float("-inf")), 1)
                row = row + torch.where(qr > 0, qr * (qr.clamp(min=1e-300).log() - lr), 0.0)
            part = tau * tau * (row * w).sum() / weights
            sums = sums + part.detach()
            got = [torch.autograd.grad(part, z, s["scale"].double())[0]]
        parts.append(got)
    cat = [torch.cat([p[j] for p in parts]) for j in range(len(parts[0]))]
    back = lambda t: t if len(z0.shape) == 2 else t.reshape(*shape, c).movedim(-1, 1)  # noqa: E731
    if case["op"] == "distill_topk":
        return dict(loss=sums, dlogits=back(cat[0]))
    res = dict(logp=cat[0].reshape(shape), entropy=cat[1].reshape(shape), lse=cat[2].reshape(shape))
    if k:
        res.update(top_logp=cat[3].reshape(*shape, k), top_index=None)
    if case["grad"]:
        res["dlogits"] = back(cat[-1])
    return res


def work(case):
    c, k = case["classes"], case["k"]
    rows = 1
    for v in (case["n"], case["d"], case["h"], case["w"]):
        rows *= v or 1
    z = rows * c * _BYTES[case["dtype"]]
    # a subtraction, a scaling, an exponential and a sum for each logit; the entropy's product and sum
    if case["op"] == "log_probs":
        b = z + rows * (8 + 12 + 8 * k)
        f = rows * c * 6
        if case["grad"]:
            b += z + rows * 8
            f += rows * c * 7
    else:
        b = 2 * z + rows * (8 * k + (4 if case["weighted"] else 0)) + 4
        f = rows * c * 9
    return {"bytes": b, "flops": f}
