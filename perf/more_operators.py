"""The operators of a training step around a model's blocks whose speed is
measured, with their plain forms: what a program that trains or scores a deep
model over many classes has this package do between two blocks, at its
classifier and before its optimizer.

Kinds of case:
  boundary   the end of one block and the start of the next: the norm of the
             branch, its gate and residual scale, the residual and the next
             block's norm (fused_block_ops.fused_gated_residual_norm), forward
             alone or with every gradient
  loss       cross entropy of a linear classifier over a large vocabulary, by
             pieces of the vocabulary, the logits never kept
             (linear_cross_entropy.linear_cross_entropy), alone or with the
             gradients of rows, weight and bias
  clip       the global norm of many gradients (grad_norm.global_grad_norm),
             and the gradients clipped to it (grad_norm.clip_grad_norm)

Every input comes from the seed. `run` computes the plain forms in float32 (the
logarithms of the rows' sums in float64) and rounds once; with `own` set it
makes the package's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
IGNORE = -100


def listed():
    return [
        # One token's row between two blocks while answering: latency.
        dict(name="bd_token_4096_bf16", op="boundary", rows=1, width=4096, dtype="bf16", norm="rms", gate="none",
             train=False),
        # The production model's blocks: 24,492 nodes of width 256, one gate a node.
        dict(name="bd_nodes_256_f32", op="boundary", rows=24492, width=256, dtype="f32", norm="layer", gate="row",
             train=True),
        # Odd rows of odd width, a gate a value.
        dict(name="bd_odd_1001_bf16", op="boundary", rows=10007, width=1001, dtype="bf16", norm="layer", gate="value",
             train=True),
        # A long training batch of wide rows.
        dict(name="bd_train_4096_bf16", op="boundary", rows=16384, width=4096, dtype="bf16", norm="rms", gate="value",
             train=True),
        # How likely one token is over a large vocabulary: the weight is read once.
        dict(name="ce_token_131072_bf16", op="loss", rows=1, width=4096, classes=131072, dtype="bf16", bias=False,
             ignored=0.0, train=False),
        # Scoring rows of odd width over an odd vocabulary, a tenth of them not counted.
        dict(name="ce_score_50001_f32", op="loss", rows=777, width=1001, classes=50001, dtype="f32", bias=True,
             ignored=0.1, train=False),
        # The production model's five concatenated states over many classes, half
        # of the nodes outside the training mask.
        dict(name="ce_nodes_2000_f32", op="loss", rows=24492, width=1280, classes=2000, dtype="f32", bias=True,
             ignored=0.5, train=True),
        # A training step of token prediction.
        dict(name="ce_train_32000_bf16", op="loss", rows=8192, width=4096, classes=32000, dtype="bf16", bias=False,
             ignored=0.1, train=True),
        # The same on narrower rows over a large vocabulary.
        dict(name="ce_train_131072_bf16", op="loss", rows=4096, width=2048, classes=131072, dtype="bf16", bias=False,
             ignored=0.0, train=True),
        # The norm and the clipped gradients of the four-layer production model: latency.
        dict(name="gn_model_f32", op="clip", tensors=62, values=2600000, dtype="f32", clip=True),
        # The norm alone, of many tensors of odd sizes and both types.
        dict(name="gn_norm_mixed", op="clip", tensors=333, values=40000003, dtype="mixed", clip=False),
        # The clipped gradients of a large model's shard.
        dict(name="gn_large_bf16", op="clip", tensors=200, values=500000000, dtype="bf16", clip=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm, odd half of the time."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return min(hi, max(lo, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    op = rng.choice(["boundary", "loss", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.7
    if op == "boundary":
        width = _log_int(rng, 16, 8192)
        cells = 1 << 26 if dtype == "bf16" else 1 << 25
        return dict(op=op, rows=_log_int(rng, 1, min(200000, cells // width)), width=width, dtype=dtype,
                    norm=rng.choice(["layer", "rms"]), gate=rng.choice(["none", "row", "value"]), train=train)
    if op == "loss":
        width, classes = _log_int(rng, 64, 4096), _log_int(rng, 1000, 131072)
        products = 10**12 if dtype == "bf16" else 10**11
        most = min(30000, products // (width * classes))
        rows = _log_int(rng, min(64, most), most) if train else _log_int(rng, 1, most)
        return dict(op=op, rows=rows, width=width, classes=classes, dtype=dtype, bias=rng.random() < 0.5,
                    ignored=rng.choice([0.0, 0.1, 0.5]), train=train)
    return dict(op=op, tensors=_log_int(rng, 1, 400), values=_log_int(rng, 2000, 10**8),
                dtype=rng.choice(["f32", "bf16", "mixed"]), clip=rng.random() < 0.7)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _sizes(case):
    """Sizes of a model's tensors: a few large matrices, many vectors."""
    rng = random.Random(case["tensors"] * 1000003 + case["values"])
    share = [math.exp(rng.uniform(-8.0, 0.0)) for _ in range(case["tensors"])]
    scale = case["values"] / sum(share)
    return [max(1, int(s * scale)) for s in share]


def _types(case):
    n = case["tensors"]
    return [torch.float32 if case["dtype"] == "f32" or (case["dtype"] == "mixed" and i % 2) else torch.bfloat16
            for i in range(n)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    rand = lambda *s: torch.rand(*s, generator=gen, device=DEV)
    st = dict(case=case)
    if case["op"] == "clip":
        grads, out = [], []
        flat = {}
        sizes, types = _sizes(case), _types(case)
        for t in dict.fromkeys(types):
            # the clipped gradients go into one flat buffer, as an optimizer or an all-reduce takes them
            flat[t] = torch.empty(sum(s for s, u in zip(sizes, types) if u == t), dtype=t, device=DEV)
        at = dict.fromkeys(flat, 0)
        for size, t in zip(sizes, types):
            # gradients of different layers differ by orders of magnitude
            grads.append((randn(size) * (0.01 * 10 ** rand(1))).to(t))
            out.append(flat[t][at[t]: at[t] + size])
            at[t] += size
        st.update(grads=grads, out=out, flat=[flat[t] for t in flat], max_norm=1.0)
        return st
    rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
    if case["op"] == "boundary":
        st["branch"] = (randn(rows, width) * 0.7 + 0.2 * randn(rows, 1)).to(dtype)
        st["residual"] = (randn(rows, width) * 1.5).to(dtype)
        vector = lambda mean, spread: (mean + spread * randn(width)).to(dtype)
        st["post_weight"], st["scale"], st["next_weight"] = vector(1.0, 0.2), vector(0.5, 0.1), vector(1.0, 0.2)
        if case["norm"] == "layer":
            st["post_bias"], st["next_bias"] = vector(0.0, 0.2), vector(0.0, 0.2)
        if case["gate"] != "none":
            st["gate"] = randn(rows, 1 if case["gate"] == "row" else width).to(dtype)
        st["eps"] = 1e-5
        st["grads"] = [randn(rows, width).to(dtype), randn(rows, width).to(dtype)] if case["train"] else None
        names = ("branch", "residual", "post_weight", "post_bias", "scale", "gate", "next_weight", "next_bias")
    else:
        classes = case["classes"]
        # logits of a spread of 1.5, the label's a few units above: a model that has learned something
        weight = randn(classes, width).mul_(1.5 / math.sqrt(width))
        labels = torch.randint(0, classes, (rows,), generator=gen, device=DEV)
        st["x"] = (randn(rows, width) + 2.0 * weight[labels]).to(dtype)
        st["weight"] = weight.to(dtype)
        if case["bias"]:
            st["bias"] = randn(classes).to(dtype)
        st["labels"] = torch.where(rand(rows) < case["ignored"], torch.full_like(labels, IGNORE), labels)
        st["grad"] = (rand(rows) + 0.5) / rows if case["train"] else None
        names = ("x", "weight", "bias")
    st["names"] = [n for n in names if n in st]
    st["inputs"] = [st[n] for n in st["names"]]
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
    if case["op"] == "clip":
        from cign_amd.grad_norm import clip_grad_norm, global_grad_norm

        if not case["clip"]:
            return dict(norm=global_grad_norm(st["grads"]))
        norm = clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
        return dict(norm=norm, clipped=st["flat"])
    if case["op"] == "boundary":
        from cign_amd.fused_block_ops import fused_gated_residual_norm

        hidden, normed = fused_gated_residual_norm(
            st["branch"], st["residual"], post_weight=st["post_weight"], post_bias=st.get("post_bias"),
            scale=st["scale"], gate=st.get("gate"), next_weight=st["next_weight"], next_bias=st.get("next_bias"),
            eps=st["eps"], norm=case["norm"])
        out, results, grads = dict(hidden=hidden, normed=normed), [hidden, normed], st["grads"]
    else:
        from cign_amd.linear_cross_entropy import linear_cross_entropy

        r = linear_cross_entropy(st["x"], st["weight"], st["labels"], bias=st.get("bias"), ignore_index=IGNORE)
        out, results, grads = dict(loss=r.loss, logsumexp=r.logsumexp), [r.loss], [st["grad"]]
    if case["train"]:
        given = torch.autograd.grad(results, st["inputs"], grads)
        out.update({"grad_" + n: g for n, g in zip(st["names"], given)})
    return {k: v.detach() for k, v in out.items()}


@torch.no_grad()
def _run_plain(st):
    return {"boundary": _plain_boundary, "loss": _plain_loss, "clip": _plain_clip}[st["case"]["op"]](st)


def _plain_norm(x, weight, bias, eps, layer):
    """(normalised rows, 1 / sigma, weighted and shifted) of float32 rows."""
    c = x - x.mean(dim=1, keepdim=True) if layer else x
    r = torch.rsqrt((c * c).mean(dim=1, keepdim=True) + eps)
    n = c * r
    y = n * weight
    return n, r, y if bias is None else y + bias


def _plain_norm_grad(d, n, r, layer):
    """Gradient of the rows from d, that of the normalised rows."""
    g = d - n * (d * n).mean(dim=1, keepdim=True)
    return r * (g - d.mean(dim=1, keepdim=True) if layer else g)


def _plain_boundary(st):
    case = st["case"]
    layer = case["norm"] == "layer"
    f = {k: st[k].float() for k in st["names"]}
    dtype = st["branch"].dtype
    n1, r1, v = _plain_norm(f["branch"], f["post_weight"], f.get("post_bias"), st["eps"], layer)
    s = torch.sigmoid(f["gate"]) if "gate" in f else torch.ones_like(f["scale"])
    hidden = f["residual"] + f["scale"] * s * v
    n2, r2, y = _plain_norm(hidden, f["next_weight"], f.get("next_bias"), st["eps"], layer)
    out = dict(hidden=hidden.to(dtype), normed=y.to(dtype))
    if st["grads"] is None:
        return out
    gh, gy = (t.float() for t in st["grads"])
    gh = gh + _plain_norm_grad(gy * f["next_weight"], n2, r2, layer)
    gv = gh * f["scale"] * s
    g = dict(branch=_plain_norm_grad(gv * f["post_weight"], n1, r1, layer), residual=gh,
             post_weight=(gv * n1).sum(dim=0), scale=(gh * s * v).sum(dim=0), next_weight=(gy * n2).sum(dim=0))
    if layer:
        g.update(post_bias=gv.sum(dim=0), next_bias=gy.sum(dim=0))
    if "gate" in f:
        g["gate"] = gh * f["scale"] * v * s * (1.0 - s)
        if case["gate"] == "row":
            g["gate"] = g["gate"].sum(dim=1, keepdim=True)
    out.update({"grad_" + k: g[k].to(st[k].dtype) for k in st["names"]})
    return out


def _plain_loss(st):
    x, w, labels = st["x"].float(), st["weight"].float(), st["labels"]
    z = x @ w.t()
    if "bias" in st:
        z += st["bias"].float()
    m = z.amax(dim=1, keepdim=True)
    given = labels != IGNORE
    at = torch.where(given, labels, torch.zeros_like(labels))[:, None]
    chosen = z.gather(1, at)[:, 0].double()
    z -= m
    p = z.exp_()
    s = p.sum(dim=1, keepdim=True)
    lse = m[:, 0].double() + s[:, 0].double().log()
    loss = torch.where(given, lse - chosen, torch.zeros_like(lse))
    out = dict(loss=loss.float(), logsumexp=lse.float())
    if st["grad"] is not None:
        g = torch.where(given, st["grad"], torch.zeros_like(st["grad"]))[:, None]
        p *= g / s
        p.scatter_add_(1, at, -g)
        out["grad_x"] = (p @ w).to(st["x"].dtype)
        out["grad_weight"] = (p.t() @ x).to(st["weight"].dtype)
        if "bias" in st:
            out["grad_bias"] = p.sum(dim=0).to(st["bias"].dtype)
    return out


def _plain_clip(st):
    squares = [g.float().square().sum() for g in st["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    if not st["case"]["clip"]:
        return dict(norm=norm)
    scale = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    torch._foreach_copy_(st["out"], [g.float() * scale for g in st["grads"]])
    return dict(norm=norm, clipped=st["flat"])


# ---------------------------------------------------------------------------
# Work and exact values
# ---------------------------------------------------------------------------


def work(case):
    if case["op"] == "clip":
        sizes, types = _sizes(case), _types(case)
        read = sum(s * (4 if t == torch.float32 else 2) for s, t in zip(sizes, types))
        return dict(bytes=read * (2 if case["clip"] else 1) + 4, flops=sum(sizes) * (3 if case["clip"] else 2))
    es = 2 if case["dtype"] == "bf16" else 4
    rows, width = case["rows"], case["width"]
    cells = rows * width
    if case["op"] == "boundary":
        gate = {"none": 0, "row": rows, "value": cells}[case["gate"]]
        params = width * (5 if case["norm"] == "layer" else 3)
        if case["train"]:
            # branch, residual, gate, both gradients in; both results and the gradients out
            return dict(bytes=es * (8 * cells + 2 * gate + 2 * params), flops=50 * cells)
        return dict(bytes=es * (4 * cells + gate + params), flops=18 * cells)
    classes = case["classes"]
    params = classes * (width + (1 if case["bias"] else 0))
    if case["train"]:
        return dict(bytes=2 * es * (cells + params) + rows * 20, flops=6 * cells * classes)
    return dict(bytes=es * (cells + params) + rows * 16, flops=2 * cells * classes)


def exact(case, seed):
    """The outputs by their definitions, in float64."""
    with torch.no_grad():
        st = prepare(case, seed)
        return {"boundary": _exact_boundary, "loss": _exact_loss, "clip": _exact_clip}[case["op"]](st)


def _exact_clip(st):
    parts = [torch.linalg.vector_norm(g.double()) for g in st["grads"]]
    norm = torch.linalg.vector_norm(torch.stack(parts))
    if not st["case"]["clip"]:
        return dict(norm=norm)
    factor = min(1.0, st["max_norm"] / (float(norm) + 1e-6))
    types = dict.fromkeys(g.dtype for g in st["grads"])
    return dict(norm=norm, clipped=[torch.cat([g for g in st["grads"] if g.dtype == t]).double() * factor for t in types])


def _exact_boundary(st):
    """A block of rows at a time; the parameters' gradients are added over the blocks."""
    case = st["case"]
    step = max(1, (1 << 24) // case["width"])
    blocks = [_exact_boundary_rows(st, slice(a, a + step)) for a in range(0, case["rows"], step)]
    vectors = {"grad_" + k for k in st["names"] if st[k].dim() == 1}
    return {k: sum(b[k] for b in blocks) if k in vectors else torch.cat([b[k] for b in blocks]) for k in blocks[0]}


def _exact_boundary_rows(st, r):
    case, eps = st["case"], st["eps"]
    n = case["width"]
    d = {k: (st[k] if st[k].dim() == 1 else st[k][r]).double() for k in st["names"]}
    zero, one = torch.zeros(n, dtype=torch.float64, device=DEV), torch.ones(1, dtype=torch.float64, device=DEV)

    def moments(t):
        mu = t.sum(dim=1, keepdim=True) / n if case["norm"] == "layer" else torch.zeros_like(t[:, :1])
        return mu, torch.sqrt(((t - mu) ** 2).sum(dim=1, keepdim=True) / n + eps)

    def back(g, t, mu, sigma):
        """through (t - mu) / sigma"""
        along = (g * (t - mu)).sum(dim=1, keepdim=True) / (n * sigma**2)
        out = (g - along * (t - mu)) / sigma
        return out - out.mean(dim=1, keepdim=True) if case["norm"] == "layer" else out

    u = d["branch"]
    mu1, sd1 = moments(u)
    v = (u - mu1) / sd1 * d["post_weight"] + d.get("post_bias", zero)
    open_ = 1.0 / (1.0 + torch.exp(-d["gate"])) if "gate" in d else one
    h = d["residual"] + open_ * v * d["scale"]
    mu2, sd2 = moments(h)
    out = dict(hidden=h, normed=(h - mu2) / sd2 * d["next_weight"] + d.get("next_bias", zero))
    if st["grads"] is None:
        return out
    g_hidden, g_normed = (t[r].double() for t in st["grads"])
    total = g_hidden + back(g_normed * d["next_weight"], h, mu2, sd2)
    into = total * open_ * d["scale"]
    grads = dict(residual=total, branch=back(into * d["post_weight"], u, mu1, sd1),
                 next_weight=(g_normed * (h - mu2) / sd2).sum(dim=0), next_bias=g_normed.sum(dim=0),
                 post_weight=(into * (u - mu1) / sd1).sum(dim=0), post_bias=into.sum(dim=0),
                 scale=(total * open_ * v).sum(dim=0))
    if "gate" in d:
        slope = torch.exp(-d["gate"]) * open_**2
        grads["gate"] = total * d["scale"] * v * slope
        if d["gate"].shape[1] < n:
            grads["gate"] = grads["gate"].sum(dim=1, keepdim=True)
    out.update({"grad_" + k: grads[k] for k in st["names"]})
    return out


def _exact_loss(st):
    """A block of rows at a time; the gradients of weight and bias are added over the blocks."""
    case = st["case"]
    rows, classes = case["rows"], case["classes"]
    w = st["weight"].detach().double()
    b = st["bias"].detach().double() if "bias" in st else 0.0
    step = max(1, (1 << 27) // classes)
    loss, lse, gx = [], [], []
    gw, gb = 0.0, 0.0
    for a in range(0, rows, step):
        x = st["x"].detach()[a: a + step].double()
        labels = st["labels"][a: a + step]
        logp = x @ w.t() + b
        total = torch.logsumexp(logp, dim=1)
        logp -= total[:, None]
        row = torch.arange(labels.numel(), device=DEV)
        counts = (labels != IGNORE).double()
        index = labels.clamp_min(0)
        loss.append(-logp[row, index] * counts)
        lse.append(total)
        if st["grad"] is not None:
            weight = st["grad"][a: a + step].double() * counts
            dz = logp.exp_()
            dz *= weight[:, None]
            dz[row, index] -= weight
            gx.append(dz @ w)
            gw = gw + dz.t() @ x
            gb = gb + dz.sum(dim=0)
    out = dict(loss=torch.cat(loss), logsumexp=torch.cat(lse))
    if st["grad"] is not None:
        out.update(grad_x=torch.cat(gx), grad_weight=gw)
        if "bias" in st:
            out["grad_bias"] = gb
    return out
