"""The operators at a model's output whose speed is measured, with their plain
forms: what a program that trains, evaluates or distils a classifier over many
classes has this package do after its last block.

Kinds of case:
  layernorm  LayerNorm of rows of any width (fused_block_ops.fused_layernorm),
             forward alone or with the gradients of rows, weight and bias
  logprobs   log probability of each row's label, entropy and the top classes
             (class_logprobs.class_logprobs), alone or with the gradient of
             the logits
  distill    the loss against a teacher's top classes
             (distill.distill_topk_loss), alone or with the gradient of the
             logits

Every input comes from the seed. `run` computes the plain forms in float32 (the
per-row logarithms and the teacher's list, where differences of near values
count, in float64) and rounds once; with `own` set it makes the package's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100


def listed():
    return [
        # One token's row through a final norm while answering: latency.
        dict(name="ln_token_4096_bf16", op="layernorm", rows=1, width=4096, dtype="bf16", weight="bf16", train=False),
        # Output norm of the four-layer production model: five concatenated
        # 256-wide states of the 24,492-node graph.
        dict(name="ln_states_1280_f32", op="layernorm", rows=24492, width=1280, dtype="f32", weight="f32", train=True),
        # Odd rows of odd width, bf16 rows under float32 weights.
        dict(name="ln_odd_1001_bf16", op="layernorm", rows=10007, width=1001, dtype="bf16", weight="f32", train=True),
        # A long training batch of wide rows.
        dict(name="ln_wide_8192_bf16", op="layernorm", rows=16384, width=8192, dtype="bf16", weight="bf16",
             train=True),
        # One sampled token's answer over a large vocabulary, with the
        # alternatives a user is shown: latency, one row over the whole card.
        dict(name="lp_answer_131072_bf16", op="logprobs", rows=1, classes=131072, dtype="bf16", top_k=20, masked=0.0,
             ignored=0.0, temperature=1.0, train=False),
        # Cross-entropy of a node classifier: five classes, half of the nodes
        # outside the training mask.
        dict(name="lp_nodes_5_f32", op="logprobs", rows=24492, classes=5, dtype="f32", top_k=0, masked=0.0,
             ignored=0.5, temperature=1.0, train=True),
        # Evaluation over an odd vocabulary of which a quarter is masked.
        dict(name="lp_eval_50001_f32", op="logprobs", rows=777, classes=50001, dtype="f32", top_k=5, masked=0.25,
             ignored=0.1, temperature=0.7, train=False),
        # Training step of token log probabilities with an entropy bonus.
        dict(name="lp_train_32000_bf16", op="logprobs", rows=8192, classes=32000, dtype="bf16", top_k=0, masked=0.0,
             ignored=0.1, temperature=1.0, train=True),
        # A small node classifier taught by a larger one's five best classes.
        dict(name="ds_nodes_18_f32", op="distill", rows=24492, classes=18, top_k=5, dtype="f32", temperature=1.0,
             tail=True, padded=0.2, train=True),
        # Token distillation on short lists over an odd vocabulary, with the
        # rest of the teacher's mass as one more class.
        dict(name="ds_odd_50001_f32", op="distill", rows=301, classes=50001, top_k=17, dtype="f32", temperature=1.0,
             tail=True, padded=0.2, train=True),
        # Token distillation on renormalised lists at a raised temperature.
        dict(name="ds_train_32000_bf16", op="distill", rows=4096, classes=32000, top_k=64, dtype="bf16",
             temperature=2.0, tail=False, padded=0.0, train=True),
        # The same over a large vocabulary with long lists and the tail.
        dict(name="ds_large_131072_bf16", op="distill", rows=2048, classes=131072, top_k=128, dtype="bf16",
             temperature=1.0, tail=True, padded=0.0, train=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm, odd half of the time."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return min(hi, max(lo, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    op = rng.choice(["layernorm", "logprobs", "distill"])
    dtype = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.7
    if op == "layernorm":
        width = _log_int(rng, 16, 16384)
        rows = _log_int(rng, 1, min(200000, (1 << 26) // width))
        return dict(op=op, rows=rows, width=width, dtype=dtype, weight=rng.choice(["f32", dtype]), train=train)
    classes = _log_int(rng, 2, 200000)
    rows = _log_int(rng, 1, min(60000, (1 << 27) // classes))
    if op == "logprobs":
        masked = rng.choice([0.0, 0.0, 0.3])
        room = max(1, int(classes * (1.0 - masked)) // 2)
        top_k = rng.choice([0, 1, _log_int(rng, 1, min(64, room))])
        return dict(op=op, rows=rows, classes=classes, dtype=dtype, top_k=top_k, masked=masked,
                    ignored=rng.choice([0.0, 0.1, 0.5]), temperature=rng.choice([1.0, 0.7, 1.5]), train=train)
    return dict(op=op, rows=rows, classes=classes, top_k=_log_int(rng, 1, min(128, classes)), dtype=dtype,
                temperature=rng.choice([1.0, 2.0, 4.0]), tail=rng.random() < 0.5, padded=rng.choice([0.0, 0.2]),
                train=train)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _logits(gen, rows, classes, dtype):
    """Logits as a model leaves them: a spread of a few units, an offset of
    the row, and classes the model is sure of (a fixed pseudo-random tenth of
    a percent stands out)."""
    x = torch.randn(rows, classes, generator=gen, device=DEV)
    x.mul_(2.0).add_(torch.randn(rows, 1, generator=gen, device=DEV))
    stands_out = torch.randint(0, classes, (rows, max(1, classes // 1000)), generator=gen, device=DEV)
    x.scatter_add_(1, stands_out, torch.full(stands_out.shape, 5.0, device=DEV))
    return x.to(dtype)


def _first_occurrences(index):
    """True where an index of a row is the first of its value in the list."""
    order = index.sort(dim=1, stable=True)
    first = torch.ones_like(index, dtype=torch.bool)
    first[:, 1:] = order.values[:, 1:] != order.values[:, :-1]
    return torch.zeros_like(first).scatter_(1, order.indices, first)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    rows, dtype = case["rows"], DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    rand = lambda *s: torch.rand(*s, generator=gen, device=DEV)
    st = dict(case=case)
    if case["op"] == "layernorm":
        width, wt = case["width"], DTYPES[case["weight"]]
        st["x"] = (randn(rows, width) * 1.5 + 0.3 * randn(rows, 1)).to(dtype)
        st["weight"] = (1.0 + 0.2 * randn(width)).to(wt)
        st["bias"] = (0.2 * randn(width)).to(wt)
        st["eps"] = 1e-5
        st["grad"] = randn(rows, width).to(dtype) if case["train"] else None
        inputs = ("x", "weight", "bias")
    elif case["op"] == "logprobs":
        classes = case["classes"]
        x = _logits(gen, rows, classes, dtype)
        labels = torch.randint(0, classes, (rows,), generator=gen, device=DEV)
        if case["masked"]:
            # the masked classes are the same for every row; no label among them
            off = rand(classes) < case["masked"]
            off[0] = False
            labels = torch.where(off[labels], torch.zeros_like(labels), labels)
            x.masked_fill_(off, -math.inf)
        labels = torch.where(rand(rows) < case["ignored"], torch.full_like(labels, IGNORE), labels)
        st.update(logits=x, labels=labels)
        st["grad"] = [randn(rows), 0.1 * randn(rows)] if case["train"] else None
        inputs = ("logits",)
    else:
        classes, k = case["classes"], case["top_k"]
        x = _logits(gen, rows, classes, dtype)
        # A teacher that agrees in part: k distinct classes, some of the
        # student's best among them, in the teacher's falling order.
        drawn = torch.randint(0, classes, (rows, 2 * k), generator=gen, device=DEV)
        if classes <= 8 * k:
            index = rand(rows, classes).argsort(dim=1)[:, :k].contiguous()
            keep = torch.ones_like(index, dtype=torch.bool)
        else:
            # twice as many draws as places; a place whose draw came before stays empty
            keep = _first_occurrences(drawn)
            order = (~keep).to(torch.uint8).argsort(dim=1, stable=True)[:, :k]
            index, keep = drawn.gather(1, order), keep.gather(1, order)
        t = 0.7 * x.gather(1, index).float() + 2.0 * randn(rows, k)
        t = t / case["temperature"]
        mass = 0.5 + 0.49 * rand(rows, 1)  # what the list holds of the teacher's probability
        t = torch.log_softmax(t.double(), dim=1) + torch.log(mass.double())
        t, order = t.sort(dim=1, descending=True)
        index, keep = index.gather(1, order), keep.gather(1, order)
        index = torch.where(keep & (rand(rows, k) >= case["padded"]), index, torch.full_like(index, -1))
        st.update(logits=x, teacher_logprobs=t.float(), teacher_index=index)
        st["grad"] = rand(rows) + 0.5 if case["train"] else None
        inputs = ("logits",)
    st["inputs"] = [st[n] for n in inputs]
    if case["train"]:
        for t in st["inputs"]:
            t.requires_grad_()
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    case = st["case"]
    if case["op"] == "layernorm":
        from cign_amd.fused_block_ops import fused_layernorm

        y = fused_layernorm(st["x"], st["weight"], st["bias"], st["eps"])
        out = dict(y=y)
        if case["train"]:
            out["grad_x"], out["grad_weight"], out["grad_bias"] = torch.autograd.grad(y, st["inputs"], st["grad"])
    elif case["op"] == "logprobs":
        from cign_amd.class_logprobs import class_logprobs

        r = class_logprobs(st["logits"], st["labels"], top_k=case["top_k"], temperature=case["temperature"],
                           ignore_index=IGNORE)
        out = dict(logprob=r.logprob, entropy=r.entropy)
        if case["top_k"]:
            out.update(top_logprobs=r.top_logprobs, top_index=r.top_index)
        if case["train"]:
            out["grad_logits"], = torch.autograd.grad([r.logprob, r.entropy], st["inputs"], st["grad"])
    else:
        from cign_amd.distill import distill_topk_loss

        loss = distill_topk_loss(st["logits"], st["teacher_logprobs"], st["teacher_index"],
                                 temperature=case["temperature"], tail=case["tail"])
        out = dict(loss=loss)
        if case["train"]:
            out["grad_logits"], = torch.autograd.grad(loss, st["inputs"], st["grad"])
    return {k: v.detach() for k, v in out.items()}


@torch.no_grad()
def _run_plain(st):
    case = st["case"]
    if case["op"] == "layernorm":
        return _plain_layernorm(st["x"], st["weight"], st["bias"], st["eps"], st["grad"])
    if case["op"] == "logprobs":
        return _plain_logprobs(st["logits"], st["labels"], case["top_k"], case["temperature"], st["grad"])
    return _plain_distill(st["logits"], st["teacher_logprobs"], st["teacher_index"], case["temperature"],
                          case["tail"], st["grad"])


def _plain_layernorm(x, weight, bias, eps, grad):
    xf = x.float()
    centred = xf - xf.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + eps)
    xhat = centred * rstd
    out = dict(y=(xhat * weight.float() + bias.float()).to(x.dtype))
    if grad is not None:
        g = grad.float()
        gw = g * weight.float()
        gx = rstd * (gw - gw.mean(dim=1, keepdim=True) - xhat * (gw * xhat).mean(dim=1, keepdim=True))
        out.update(grad_x=gx.to(x.dtype), grad_weight=(g * xhat).sum(dim=0).to(weight.dtype),
                   grad_bias=g.sum(dim=0).to(bias.dtype))
    return out


def _softmax_parts(l):
    """(shift [N,1], sum of exp(l - shift) [N,1]); the shift is the row's
    largest value, 0 where every class is masked."""
    m = l.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    return m, torch.exp(l - m).sum(dim=1, keepdim=True)


def _top(x, k):
    """Indices of the k largest values of each row, ties to the lowest index:
    k rounds of argmax over the values' order-preserving integers (a class
    already taken falls below every value, a masked one does not)."""
    v = x.float() + 0.0  # -0 becomes +0
    bits = torch.where(v.isnan(), torch.full_like(v, -math.inf), v).view(torch.int32)
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF)
    picked = []
    for _ in range(k):
        i = key.argmax(dim=1, keepdim=True)
        picked.append(i)
        key.scatter_(1, i, torch.iinfo(torch.int32).min)
    return torch.cat(picked, dim=1)


def _plain_logprobs(logits, labels, top_k, temperature, grad):
    l = logits.float() / temperature
    m, s = _softmax_parts(l)
    logs = s.double().log()
    p = torch.exp(l - m) / s.clamp_min(torch.finfo(torch.float32).tiny)
    lp = torch.where(p > 0, l - m, torch.zeros_like(l))  # 0 * -inf counts nothing
    entropy = (logs[:, 0] - (p * lp).sum(dim=1).double()).float()
    entropy = torch.where(s[:, 0] > 0, entropy, torch.zeros_like(entropy))
    given = labels != IGNORE
    at = torch.where(given, labels, torch.zeros_like(labels))[:, None]
    value = l.gather(1, at).double() - m.double()
    logprob = torch.where(value == -math.inf, value, value - logs)[:, 0].float()
    logprob = torch.where(given, logprob, torch.zeros_like(logprob))
    out = dict(logprob=logprob, entropy=entropy)
    if top_k:
        index = _top(logits, top_k)
        value = l.gather(1, index).double() - m.double()
        out.update(top_logprobs=torch.where(value == -math.inf, value, value - logs).float(), top_index=index)
    if grad is not None:
        g = torch.where(given, grad[0], torch.zeros_like(grad[0]))[:, None]
        gx = -p * (g + grad[1][:, None] * (lp - logs.float() + entropy[:, None]))
        gx.scatter_add_(1, at, g)
        out["grad_logits"] = (gx / temperature).to(logits.dtype)
    return out


def _plain_distill(logits, teacher_logprobs, teacher_index, temperature, tail, grad):
    l = logits.float() / temperature
    present = teacher_index >= 0
    at = teacher_index.clamp_min(0)
    t = torch.where(present, teacher_logprobs.double(), torch.full_like(teacher_logprobs.double(), -math.inf))
    if not tail:
        top = t.amax(dim=1, keepdim=True)
        t = t - torch.where(top == -math.inf, torch.zeros_like(top), top)
        total = torch.exp(t).sum(dim=1, keepdim=True)
        t = torch.where(total > 0, t - total.log(), t)
    p = torch.exp(t)
    m, s = _softmax_parts(l)
    logs = s.double().log()
    value = l.gather(1, at).double() - m.double() - logs
    terms = torch.where(p > 0, p * (t - value), torch.zeros_like(p))
    loss = terms.sum(dim=1)
    mass = p.sum(dim=1, keepdim=True)
    rest_p = rest_grad = None
    if tail:
        # the classes outside the list, as one class
        spare = torch.where(present, teacher_index, torch.full_like(teacher_index, l.shape[1]))
        listed_here = torch.zeros(l.shape[0], l.shape[1] + 1, dtype=torch.bool, device=l.device)
        listed_here = listed_here.scatter_(1, spare, True)[:, :-1]
        members = listed_here.sum(dim=1, keepdim=True)
        active = (members < l.shape[1]) & present.any(dim=1, keepdim=True)
        rest_p = torch.where(active, (1.0 - mass).clamp_min(0.0), torch.zeros_like(mass))
        rest = l.masked_fill(listed_here, -math.inf)
        rm, rs = _softmax_parts(rest)
        rest_log = rm.double() - m.double() + rs.double().log() - logs
        loss = loss + torch.where(rest_p > 0, rest_p * (rest_p.log() - rest_log), torch.zeros_like(rest_p))[:, 0]
        mass = mass + rest_p
        rest_grad = torch.exp(rest - rm) * (rest_p / rs.double().clamp_min(1e-300)).float()
    out = dict(loss=(loss * temperature**2).float())
    if grad is not None:
        gx = torch.exp(l - m) * (mass / s.double().clamp_min(1e-300)).float()
        if tail:
            gx -= rest_grad
        gx.scatter_add_(1, at, torch.where(present, -p, torch.zeros_like(p)).float())
        out["grad_logits"] = (gx * (grad[:, None] * temperature)).to(logits.dtype)
    return out


# ---------------------------------------------------------------------------
# Work and exact values
# ---------------------------------------------------------------------------


def work(case):
    rows, es = case["rows"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "layernorm":
        width, ws = case["width"], 2 if case["weight"] == "bf16" else 4
        cells = rows * width
        if case["train"]:  # rows and their gradient in, result and gradient out; weight, bias and their gradients
            return dict(bytes=4 * cells * es + 4 * width * ws, flops=18 * cells)
        return dict(bytes=2 * cells * es + 2 * width * ws, flops=7 * cells)
    cells = rows * case["classes"]
    if case["op"] == "logprobs":
        per_row = 8 + 4 + 4 + 12 * case["top_k"] + (8 if case["train"] else 0)
    else:
        per_row = 12 * case["top_k"] + 4 + (4 if case["train"] else 0)
    return dict(bytes=cells * es * (2 if case["train"] else 1) + rows * per_row,
                flops=cells * (9 if case["train"] else 5))


def exact(case, seed):
    """The outputs by their definitions, in float64, a block of rows at a time."""
    st = prepare(case, seed)
    rows = case["rows"]
    wide = case["width"] if case["op"] == "layernorm" else case["classes"]
    step = max(1, (1 << 26) // wide)
    f = {"layernorm": _exact_layernorm, "logprobs": _exact_logprobs, "distill": _exact_distill}[case["op"]]
    with torch.no_grad():
        blocks = [f(st, slice(a, min(rows, a + step))) for a in range(0, rows, step)]
    out = {}
    for k in blocks[0]:
        v = [b[k] for b in blocks]
        out[k] = torch.stack(v).sum(dim=0) if k in ("grad_weight", "grad_bias") else torch.cat(v)
    return out


def _exact_layernorm(st, r):
    x = st["x"].detach()[r].double()
    w, b = st["weight"].detach().double(), st["bias"].detach().double()
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    sigma = torch.sqrt(var + st["eps"])
    z = (x - mean) / sigma
    out = dict(y=z * w + b)
    if st["grad"] is not None:
        g = st["grad"][r].double()
        dz = g * w
        n = x.shape[1]
        dvar = (dz * (x - mean)).sum(dim=1, keepdim=True) * -0.5 / sigma**3
        dmean = -dz.sum(dim=1, keepdim=True) / sigma
        out.update(grad_x=dz / sigma + dvar * 2.0 * (x - mean) / n + dmean / n, grad_weight=(g * z).sum(dim=0),
                   grad_bias=g.sum(dim=0))
    return out


def _exact_logprobs(st, r):
    case = st["case"]
    x = st["logits"].detach()[r]
    lp = torch.log_softmax(x.double() / case["temperature"], dim=1)
    lp = torch.where((x == -math.inf).all(dim=1, keepdim=True), torch.full_like(lp, -math.inf), lp)
    p = lp.exp()
    plogp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    labels = st["labels"][r]
    given = labels != IGNORE
    safe = labels.clamp_min(0)
    row = torch.arange(lp.shape[0], device=lp.device)
    out = dict(logprob=torch.where(given, lp[row, safe], torch.zeros_like(lp[:, 0])), entropy=-plogp.sum(dim=1))
    if case["top_k"]:
        order = (x.double() + 0.0).sort(dim=1, descending=True, stable=True).indices[:, : case["top_k"]]
        out.update(top_logprobs=lp.gather(1, order), top_index=order)
    if st["grad"] is not None:
        g, h = (t[r].double()[:, None] for t in st["grad"])
        g = torch.where(given[:, None], g, torch.zeros_like(g))
        chosen = torch.zeros_like(p)
        chosen[row, safe] = given.double()
        gx = g * (chosen - p) - h * (plogp + p * out["entropy"][:, None])
        out["grad_logits"] = gx / case["temperature"]
    return out


def _exact_distill(st, r):
    case = st["case"]
    T = case["temperature"]
    lq = torch.log_softmax(st["logits"].detach()[r].double() / T, dim=1)
    index, t = st["teacher_index"][r], st["teacher_logprobs"][r].double()
    n, classes = lq.shape
    here = index >= 0
    some = here.any(dim=1)
    if not case["tail"]:
        t = torch.where(here, t, torch.full_like(t, -math.inf))
        t = torch.where(some[:, None], t, torch.zeros_like(t)).log_softmax(dim=1)
    # the teacher over all classes and one more for the rest; a spare column takes the empty places
    spare = torch.where(here, index, torch.full_like(index, classes))
    tp = torch.zeros(n, classes + 1, dtype=torch.float64, device=lq.device)
    tp.scatter_(1, spare, torch.where(here, t.exp(), torch.zeros_like(t)))
    member = torch.zeros(n, classes + 1, dtype=torch.bool, device=lq.device).scatter_(1, spare, True)[:, :classes]
    tp = tp[:, :classes]
    kl = torch.where(tp > 0, tp * (tp.log() - lq), torch.zeros_like(tp)).sum(dim=1)
    q = lq.exp()
    gx = tp.sum(dim=1, keepdim=True) * q - tp
    if case["tail"]:
        left = (1.0 - tp.sum(dim=1)).clamp_min(0.0)
        left = torch.where(member.all(dim=1) | ~some, torch.zeros_like(left), left)
        lrest = lq.masked_fill(member, -math.inf)
        total = lrest.logsumexp(dim=1)
        kl = kl + torch.where(left > 0, left * (left.log() - total), torch.zeros_like(left))
        share = torch.where(member, torch.zeros_like(q), (lrest - total[:, None]).exp())
        gx = gx + left[:, None] * (q - share)
    kl = torch.where(some, kl, torch.zeros_like(kl))
    gx = torch.where(some[:, None], gx, torch.zeros_like(gx))
    out = dict(loss=kl * T * T)
    if st["grad"] is not None:
        out["grad_logits"] = gx * st["grad"][r].double()[:, None] * T
    return out
