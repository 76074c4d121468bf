"""Cases of the operators on a network's answers: label scores (log probability of given labels, entropy, top alternatives),
the distillation loss against a teacher's top answers, and the gradients of both.

``run`` computes them in plain torch operations (``own`` false) or through ``dosma_amd.models`` (``own`` true)."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CAP_LOGITS = 160 * 1000 * 1000  # of a drawn case: below the largest listed one


# A case: op = scores | scores_grad | distill | distill_grad; layout "rows" = (rows, classes), "planes" = (batch, classes, pixels), the
# layout torch networks answer in; background: the implicit category 0 with logit 0; entries = the teacher's top answers per row.
def _case(name, op, layout, dtype, batch, pixels, classes, **kw):
    c = dict(op=op, layout=layout, dtype=dtype, batch=batch, pixels=pixels, classes=classes, background=False,
             temperature=1.0, top=0, entries=0, tail=False, entropy_grad=False)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one answer over a large set of labels with its alternatives: the call whose latency counts
        _case("scores one row", "scores", "rows", "bf16", 1, 1, 131071, top=20),
        # a batch of answers over a large set of labels
        _case("scores batch", "scores", "rows", "bf16", 1, 1024, 100003, top=8, temperature=0.7),
        # the knee volume: confidence, entropy, label map and runner-up of a 4-tissue network on 512 x 512 x 160 voxels
        _case("scores knee volume", "scores", "rows", "f32", 1, 512 * 512 * 160, 4, background=True, top=2),
        # an atlas of 117 structures, 8 slices of 384 x 384, as a torch network answers
        _case("scores atlas planes", "scores", "planes", "f16", 8, 384 * 384, 117, top=3),
        # training on labels with an entropy term: a 4-tissue network, 16 slices of 384 x 384 as torch holds them
        _case("grad slices planes", "scores_grad", "planes", "f32", 16, 384 * 384, 4, background=True, entropy_grad=True),
        # training on labels of a large set
        _case("grad batch", "scores_grad", "rows", "bf16", 1, 1024, 100003),
        # a few rows against stored top answers: latency
        _case("distill few rows", "distill", "rows", "f32", 1, 7, 50021, entries=16, temperature=2.0),
        # the fast precision against the parity mode's stored two best labels, one 384 x 384 x 160 volume
        _case("distill knee volume", "distill", "rows", "f32", 1, 384 * 384 * 160, 4, background=True, entries=2, tail=True),
        # a batch against a teacher's 64 best
        _case("distill batch", "distill", "rows", "bf16", 1, 2048, 65537, entries=64, tail=True),
        # its gradient for a student network in training, 16 slices
        _case("distill grad slices planes", "distill_grad", "planes", "f16", 16, 384 * 384, 5, entries=3, temperature=2.0),
        _case("distill grad knee volume", "distill_grad", "rows", "f32", 1, 384 * 384 * 160, 4, background=True, entries=2, tail=True),
        _case("distill grad batch", "distill_grad", "rows", "bf16", 1, 2048, 65537, entries=64, temperature=2.0),
    ]


def _logspread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scores", "scores_grad", "distill", "distill_grad"])
    layout = rng.choice(["rows", "rows", "planes"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    cap = CAP_LOGITS if dtype != "f32" else CAP_LOGITS // 2
    if op in ("scores_grad", "distill_grad"):
        cap //= 2
    classes = _logspread(rng, 2, 131071 if layout == "rows" else 200)
    n = _logspread(rng, 1, max(1, min(cap // (classes + 8), 512 * 512 * 160)))
    batch = rng.choice([1, 2, 5, 16]) if layout == "planes" else 1
    kw = dict(temperature=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]), background=classes <= 200 and rng.random() < 0.5)
    cats = classes + (1 if kw["background"] else 0)
    if op == "scores":
        kw["top"] = rng.choice([0, 1, 2, min(5, cats), min(20, cats)])
        if classes > 200 and n * classes > 4 * 10 ** 7:
            kw["top"] = min(kw["top"], 8)
    elif op == "scores_grad":
        kw["entropy_grad"] = rng.random() < 0.5
    else:
        kw["entries"] = min(_logspread(rng, 1, 64), cats)
        kw["tail"] = rng.random() < 0.5
        if kw["tail"]:
            kw["entries"] = min(kw["entries"], max(1, cats - 1))
    return _case(None, op, layout, dtype, batch, max(1, n // batch), classes, **kw)


def _shape(case):
    if case["layout"] == "planes":
        return (case["batch"], case["classes"], case["pixels"])
    return (case["pixels"], case["classes"])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    cls = 1 if case["layout"] == "planes" else -1
    C, bg, T = case["classes"], case["background"], case["temperature"]
    small = C <= 200
    z = torch.randn(_shape(case), generator=g, device=DEV)
    rows_shape = z.select(cls, 0).shape
    if small:
        # a segmentation network: most categories well below zero, one raised by a varying amount
        z.mul_(2.0).sub_(4.0)
        pick = torch.randint(0, C, rows_shape, generator=g, device=DEV)
        lift = torch.rand(rows_shape, generator=g, device=DEV) * 10.0
        z.scatter_add_(cls, pick.unsqueeze(cls), lift.unsqueeze(cls))
    else:
        # a large set of labels: a bulk of small scores with a heavy tail, some labels not offered (masked)
        z.mul_(1.5 + 1.0 * torch.rand(rows_shape, generator=g, device=DEV).unsqueeze(cls))
        z.add_(z.clamp(min=2.0).sub_(2.0).mul_(1.5))
        z.masked_fill_(torch.rand(C, generator=g, device=DEV) < 0.001, float("-inf"))
    logits = z.to(DTYPES[case["dtype"]], copy=True)  # (the teacher below goes on from z)
    st = {"case": case, "logits": logits, "dim": cls}
    cats = C + (1 if bg else 0)
    if case["op"] in ("scores", "scores_grad"):
        # labels: the answer itself for most rows, another label for some, no label (255 / -1) for a few
        lab = torch.randint(0, cats, rows_shape, generator=g, device=DEV)
        if small:
            best, at = logits.max(cls)
            at = at + 1 if bg else at
            if bg:
                at = torch.where(best.float() > 0, at, torch.zeros_like(at))
            lab = torch.where(torch.rand(rows_shape, generator=g, device=DEV) < 0.9, at, lab)
        drop = torch.rand(rows_shape, generator=g, device=DEV) < 0.02
        if small and cats < 255:
            st["labels"], st["ignore"] = lab.masked_fill_(drop, 255).to(torch.uint8), 255
        else:
            st["labels"], st["ignore"] = lab.masked_fill_(drop, -1), -1
    else:
        K = case["entries"]
        # the teacher: the student's scores, sharper and perturbed; its best K answers, some slots empty
        zt = z.mul_(1.2)
        zt.add_(torch.randn(zt.shape, generator=g, device=DEV))
        if bg:
            zt = torch.cat([torch.zeros_like(zt.narrow(cls, 0, 1)), zt], cls)
        zt = zt.movedim(cls, -1)
        v, i = torch.topk(zt, K, dim=-1)
        if case["tail"]:
            lse = torch.empty(rows_shape, dtype=torch.float64, device=DEV)
            flat, out = zt.reshape(-1, cats), lse.view(-1)
            step = max(1, 50000000 // cats)
            for r in range(0, flat.shape[0], step):
                out[r:r + step] = torch.logsumexp(flat[r:r + step].double() / T, -1)
            v = (v.double() / T - lse.unsqueeze(-1)).float()
            st["values"] = v.contiguous()
        else:
            st["values"] = v.to(DTYPES[case["dtype"]]).contiguous()
        if K > 1:
            cut = torch.rand(rows_shape, generator=g, device=DEV) < 0.02
            i[..., K - 1].masked_fill_(cut, -1)
        st["index"] = i.to(torch.int32).contiguous()
    del z
    if case["op"] == "scores_grad":
        st["g_log_prob"] = -(0.5 + torch.rand(rows_shape, generator=g, device=DEV))
        st["g_entropy"] = 0.1 * torch.randn(rows_shape, generator=g, device=DEV) if case["entropy_grad"] else None
        st.update(_saved_scores(st))
    if case["op"] == "distill_grad":
        st["g_loss"] = 0.5 + torch.rand(rows_shape, generator=g, device=DEV)
        st.update(_saved_distill(st))
    return st


# ---- what the forward pass leaves for the gradient: the row maximum, ln sum exp((z - max) / T), the entropy, ln p(tail) ----
def _chunks(st):
    """Slices of the rows, so that the 64-bit work below keeps to a few hundred MB."""
    x = st["logits"]
    if st["dim"] == 1:
        return [slice(b, b + 1) for b in range(x.shape[0])]
    step = max(1, 60000000 // x.shape[1])
    return [slice(r, min(r + step, x.shape[0])) for r in range(0, x.shape[0], step)]


def _wide(st, sl, dtype):
    """The categories' values of a slice, last axis, with the implicit background, in ``dtype``."""
    z = st["logits"][sl].movedim(st["dim"], -1).to(dtype)
    if st["case"]["background"]:
        z = torch.cat([torch.zeros_like(z[..., :1]), z], -1)
    return z


def _saved_scores(st):
    T = st["case"]["temperature"]
    norm, ent = [], []
    for sl in _chunks(st):
        z = _wide(st, sl, torch.float64)
        m = z.amax(-1)
        ls = torch.logsumexp((z - m.unsqueeze(-1)) / T, -1)
        lp = (z - m.unsqueeze(-1)) / T - ls.unsqueeze(-1)
        ent.append(-(lp.exp() * lp.clamp(min=-1e30)).sum(-1))
        norm.append(torch.stack([m, ls], -1))
    return {"norm": torch.cat(norm).float().contiguous(), "entropy": torch.cat(ent).float().contiguous()}


def _saved_distill(st):
    T = st["case"]["temperature"]
    norm, tail = [], []
    for sl in _chunks(st):
        z = _wide(st, sl, torch.float64)
        m = z.amax(-1)
        ls = torch.logsumexp((z - m.unsqueeze(-1)) / T, -1)
        norm.append(torch.stack([m, ls], -1))
        if st["case"]["tail"]:
            idx = st["index"][sl].long()
            lp = (z - m.unsqueeze(-1)) / T - ls.unsqueeze(-1)
            lp = torch.cat([lp, torch.zeros_like(lp[..., :1])], -1)  # a place for the empty slots
            lp.scatter_(-1, torch.where(idx < 0, lp.shape[-1] - 1, idx), float("-inf"))
            lp[..., -1] = float("-inf")
            tail.append(torch.logsumexp(lp, -1))
    return {"norm": torch.cat(norm).float().contiguous(), "log_tail": torch.cat(tail).float().contiguous() if tail else None}


# ---- the framework's operators ------------------------------------------------------------------------------------------
def _run_own(st):
    from dosma_amd import models as M

    c = st["case"]
    kw = dict(dim=st["dim"], temperature=c["temperature"], background=c["background"])
    if c["op"] == "scores":
        r = M.label_scores(st["logits"], st["labels"], top=c["top"], ignore_label=st["ignore"], **kw)
        out = {"log_prob": r.log_prob, "entropy": r.entropy}
        if c["top"]:
            out.update(top_log_prob=r.top_log_prob, top_label=r.top_label)
        return out
    if c["op"] == "scores_grad":
        return M.label_scores_grad(st["logits"], st["labels"], st["norm"], grad_log_prob=st["g_log_prob"],
                                   entropy=st["entropy"] if c["entropy_grad"] else None, grad_entropy=st["g_entropy"],
                                   ignore_label=st["ignore"], **kw)
    if c["op"] == "distill":
        return M.distill_loss(st["logits"], st["index"], st["values"], tail=c["tail"], **kw).loss
    return M.distill_loss_grad(st["logits"], st["index"], st["values"], st["norm"], log_tail=st["log_tail"],
                               grad_loss=st["g_loss"], tail=c["tail"], **kw)


# ---- the plain forms, 32 bits ---------------------------------------------------------------------------------------------
def _plain_rows(z, T):
    m = z.amax(-1, keepdim=True)
    base = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    d = (z - base) / T
    e = torch.exp(d)
    return d, e, e.sum(-1)


def _narrow(g, st):
    """Gradient of the categories -> of the logits: without the implicit one, rounded, in the logits' layout."""
    if st["case"]["background"]:
        g = g[..., 1:]
    return g.to(st["logits"].dtype).movedim(-1, st["dim"]).contiguous()


def _plain_scores(st):
    c = st["case"]
    z = _wide(st, slice(None), torch.float32)
    cats = z.shape[-1]
    d, e, s = _plain_rows(z, c["temperature"])
    ls = torch.log(s)
    lab = st["labels"].long()
    skip = lab == st["ignore"]
    lp = d.gather(-1, lab.masked_fill(skip, 0).unsqueeze(-1)).squeeze(-1) - ls
    out = {"log_prob": lp.masked_fill_(skip, 0.0),
           "entropy": ls - (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(-1) / s}
    if c["top"]:
        # the largest logit (before the subtraction, which rounds), then the lowest label that holds it; struck out for the next turn
        n = torch.arange(cats, device=z.device, dtype=torch.int32)
        top = z.amax(-1, keepdim=True)
        base = torch.where(top == float("-inf"), torch.zeros_like(top), top)
        z = z.clone() if z.data_ptr() == st["logits"].data_ptr() else z
        vals, labs = [], []
        for _ in range(c["top"]):
            v = z.amax(-1, keepdim=True)
            at = torch.where(z == v, n, cats).amin(-1, keepdim=True)
            z.scatter_(-1, at.long(), float("-inf"))
            vals.append((v - base) / c["temperature"] - ls.unsqueeze(-1))
            labs.append(at.masked_fill(v == float("-inf"), -1))
        out["top_log_prob"] = torch.cat(vals, -1)
        out["top_label"] = torch.cat(labs, -1)
    return out


def _plain_log_p(st, z):
    norm = st["norm"]
    return (z - norm[..., :1]) / st["case"]["temperature"] - norm[..., 1:]


def _plain_scores_grad(st):
    c = st["case"]
    lp = _plain_log_p(st, _wide(st, slice(None), torch.float32))
    p = torch.exp(lp)
    lab = st["labels"].long()
    skip = lab == st["ignore"]
    a = st["g_log_prob"].masked_fill(skip, 0.0).unsqueeze(-1)
    g = -a * p
    g.scatter_add_(-1, lab.masked_fill(skip, 0).unsqueeze(-1), a)
    if c["entropy_grad"]:
        g -= st["g_entropy"].unsqueeze(-1) * p * (torch.where(p > 0, lp, torch.zeros_like(lp)) + st["entropy"].unsqueeze(-1))
    return _narrow(g / c["temperature"], st)


def _plain_teacher(st):
    """Teacher's weights q, log q (0 / -inf in empty slots), the mass outside the entries."""
    c = st["case"]
    ok = st["index"] >= 0
    v = st["values"].float().masked_fill(~ok, float("-inf"))
    if c["tail"]:
        q = torch.exp(v)
        rest = (1.0 - torch.exp(v.double()).sum(-1)).float()
        rest = torch.where(rest > c["entries"] * 2.0 ** -24, rest, torch.zeros_like(rest)) * ok.any(-1)
        return ok, q, v, rest
    v = v / c["temperature"]
    m = v.amax(-1, keepdim=True)
    e = torch.exp(v - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    s = e.sum(-1, keepdim=True)
    q = torch.where(s > 0, e / s, torch.zeros_like(e))
    return ok, q, v - m - torch.log(s), None


def _member(st, ok, cats):
    idx = torch.where(ok, st["index"], cats).long()
    return torch.zeros(ok.shape[:-1] + (cats + 1,), dtype=torch.bool, device=ok.device).scatter_(-1, idx, True)[..., :cats], idx


def _plain_distill(st):
    c = st["case"]
    z = _wide(st, slice(None), torch.float32)
    d, e, s = _plain_rows(z, c["temperature"])
    ls = torch.log(s)
    ok, q, lq, rest = _plain_teacher(st)
    lp = d.gather(-1, torch.where(ok, st["index"], 0).long()) - ls.unsqueeze(-1)
    loss = torch.where(q > 0, q * (lq - lp), torch.zeros_like(q)).sum(-1)
    if c["tail"]:
        member, _ = _member(st, ok, z.shape[-1])
        lt = torch.log(e.masked_fill_(member, 0.0).sum(-1)) - ls
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - lt), torch.zeros_like(rest))
    return loss


def _plain_distill_grad(st):
    c = st["case"]
    p = torch.exp(_plain_log_p(st, _wide(st, slice(None), torch.float32)))
    ok, q, _, rest = _plain_teacher(st)
    cats = p.shape[-1]
    total = q.sum(-1)
    if c["tail"]:
        total = total + rest
        member, idx = _member(st, ok, cats)
        share = torch.where(rest > 0, rest * torch.exp(-st["log_tail"]), torch.zeros_like(rest))
        g = p * (total.unsqueeze(-1) - torch.where(member, torch.zeros_like(share.unsqueeze(-1)), share.unsqueeze(-1)))
    else:
        idx = torch.where(ok, st["index"], cats).long()
        g = p * total.unsqueeze(-1)
    g = torch.cat([g, torch.zeros_like(g[..., :1])], -1).scatter_add_(-1, idx, -q)[..., :cats]
    return _narrow(g * (st["g_loss"] / c["temperature"]).unsqueeze(-1), st)


PLAIN = {"scores": _plain_scores, "scores_grad": _plain_scores_grad, "distill": _plain_distill, "distill_grad": _plain_distill_grad}


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- the definitions, 64 bits, a slice of rows at a time ------------------------------------------------------------------
def _exact_slice(st, sl):
    c = st["case"]
    T = c["temperature"]
    z = _wide(st, sl, torch.float64)
    cats = z.shape[-1]
    logp = torch.log_softmax(z / T, dim=-1)
    if c["op"] == "scores":
        lab = st["labels"][sl].long()
        hit = torch.arange(cats, device=z.device) if cats <= 8 else None
        if hit is not None:
            lp = torch.where(hit == lab.unsqueeze(-1), logp, torch.zeros_like(logp)).sum(-1)
        else:
            lp = torch.where(lab == st["ignore"], 0.0, torch.take_along_dim(logp, lab.clamp(0, cats - 1).unsqueeze(-1), -1).squeeze(-1))
        out = {"log_prob": torch.where(lab == st["ignore"], torch.zeros_like(lp), lp), "entropy": torch.special.entr(logp.exp()).sum(-1)}
        if c["top"]:
            v, i = torch.sort(z, dim=-1, descending=True, stable=True)
            v, i = v[..., :c["top"]], i[..., :c["top"]]
            out["top_log_prob"] = torch.take_along_dim(logp, i, -1)
            out["top_label"] = torch.where(v == float("-inf"), -1, i).to(torch.int32)
        return out
    if c["op"] == "scores_grad":
        # d log p_l / dz_j = (delta - p_j) / T ; dH / dz_j = -p_j (log p_j + H) / T
        p = logp.exp()
        lab = st["labels"][sl].long()
        g = torch.zeros_like(p)
        a = torch.where(lab == st["ignore"], 0.0, st["g_log_prob"][sl].double())
        g.scatter_(-1, lab.clamp(0, cats - 1).unsqueeze(-1), a.unsqueeze(-1))
        g -= p * a.unsqueeze(-1)
        if c["entropy_grad"]:
            ent = torch.special.entr(p)
            g -= st["g_entropy"][sl].double().unsqueeze(-1) * (p * ent.sum(-1, keepdim=True) - ent)
        g /= T
    else:
        idx = st["index"][sl].long()
        ok = (idx >= 0) & (idx < cats)
        v = torch.where(ok, st["values"][sl].double(), float("-inf"))
        if c["tail"]:
            lq = v
            rest = 1.0 - lq.exp().sum(-1)
            rest = torch.where((rest > c["entries"] * 2.0 ** -24) & ok.any(-1), rest, torch.zeros_like(rest))
        else:
            lq = torch.log_softmax(v / T, -1)
            lq = torch.where(ok.any(-1, keepdim=True), lq, float("-inf"))
            rest = torch.zeros_like(lq[..., 0])
        q = lq.exp()
        outside = torch.ones(idx.shape[:-1] + (cats + 1,), dtype=torch.bool, device=z.device)
        outside.scatter_(-1, torch.where(ok, idx, cats), False)
        lt = torch.logsumexp(torch.where(outside[..., :cats], logp, float("-inf")), -1)
        if c["op"] == "distill":
            lp = torch.take_along_dim(logp, idx.clamp(0, cats - 1), -1)
            return torch.where(q > 0, q * (lq - lp), 0.0).sum(-1) + torch.where(rest > 0, rest * (rest.log() - lt), 0.0)
        p = logp.exp()
        g = p * (q.sum(-1) + rest).unsqueeze(-1)
        g -= torch.where(outside[..., :cats] & (rest > 0).unsqueeze(-1), rest.unsqueeze(-1) * (logp - lt.unsqueeze(-1)).exp(), 0.0)
        pad = torch.zeros(idx.shape[:-1] + (cats + 1,), dtype=torch.float64, device=z.device)
        pad.scatter_add_(-1, torch.where(ok, idx, cats), q)
        g = (g - pad[..., :cats]) * (st["g_loss"][sl].double() / T).unsqueeze(-1)
    if c["background"]:
        g = g[..., 1:]
    return g.movedim(-1, st["dim"])


def exact(case, seed):
    st = prepare(case, seed)
    parts = [_exact_slice(st, sl) for sl in _chunks(st)]
    if isinstance(parts[0], dict):
        return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    return torch.cat(parts)


def work(case):
    n = case["pixels"] * (case["batch"] if case["layout"] == "planes" else 1)
    C = case["classes"]
    e = SIZE[case["dtype"]]
    logits = n * C * e
    small = C <= 200 and C + (1 if case["background"] else 0) < 255
    label = n * (1 if small else 8)
    answers = n * case["entries"] * (4 + (4 if case["tail"] else e))
    if case["op"] == "scores":
        return {"bytes": logits + label + n * (8 + 8 * case["top"]), "flops": 8 * n * C}
    if case["op"] == "scores_grad":
        return {"bytes": 2 * logits + label + n * (12 + (8 if case["entropy_grad"] else 0)), "flops": 8 * n * C}
    if case["op"] == "distill":
        return {"bytes": logits + answers + 4 * n, "flops": 6 * n * C + 8 * n * case["entries"]}
    return {"bytes": 2 * logits + answers + n * (12 + (4 if case["tail"] else 0)), "flops": 6 * n * C + 8 * n * case["entries"]}
