"""GPU: fused_gated_residual_norm against the formula in float64.

Tolerances, u = 2^-24. A row's sums run over at most 16 values a thread, then 6 to
10 pairwise steps: a mean is off by at most 32 u of the mean of absolute values, the
variance (of centred values) by 64 u of itself and what the centring lost, so a
normalised value N by at most K u (1 + max|t| rstd) with K = 128, products and sums of
three or four such factors in proportion. Each result is held to K u times the
largest of its terms in the row (a sum's error reaches every value of the row),
once more 2^-8 (bf16) of itself for the rounding of what is stored. The vectors'
gradients are sums over rows: K u (and the row count's share, 1 u a row a thread
adds up) times the sum of absolute terms, then their type's rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
NAMES = ("branch", "residual", "post_weight", "post_bias", "scale", "gate", "next_weight", "next_bias")


def _inputs(n, D, dtype, wdtype, norm="layer", gate="value", seed=0, scale=1.0, offset=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    a = dict(branch=(rn(n, D) * scale + offset).to(dtype), residual=(rn(n, D) * 1.5).to(dtype),
             post_weight=(1 + 0.3 * rn(D)).to(wdtype), post_bias=(0.3 * rn(D)).to(wdtype),
             scale=(0.5 + 0.2 * rn(D)).to(wdtype), next_weight=(1 + 0.3 * rn(D)).to(wdtype),
             next_bias=(0.3 * rn(D)).to(wdtype))
    if gate != "none":
        a["gate"] = (2 * rn(n, 1 if gate == "row" else D)).to(dtype)
    return a, (rn(n, D).to(dtype), rn(n, D).to(dtype))


def _oracle(a, g, norm, eps):
    """Results, gradients, and the scale of each one's terms (the docstring's)."""
    d = {k: v.detach().double().requires_grad_() for k, v in a.items()}
    layer = norm == "layer"

    def N(t):
        c = t - t.mean(1, keepdim=True) if layer else t
        r = (c.square().mean(1, keepdim=True) + eps).rsqrt()
        return c * r, r, (1 + t.abs().amax(1, keepdim=True) * r)

    D = d["branch"].shape[1]
    one = lambda k: d[k] if k in d else torch.ones(D, dtype=torch.float64, device="cuda")
    zero = lambda k: d[k] if k in d else torch.zeros(D, dtype=torch.float64, device="cuda")
    m, r1, k1 = N(d["branch"])
    v = m * one("post_weight") + zero("post_bias")
    s = torch.sigmoid(d["gate"]) if "gate" in d else torch.ones(1, dtype=torch.float64, device="cuda")
    hidden = d["residual"] + one("scale") * s * v
    n2, r2, k2 = N(hidden)
    y = n2 * one("next_weight") + zero("next_bias")
    grads = dict(zip(d, torch.autograd.grad([hidden, y], list(d.values()), [t.double() for t in g], allow_unused=True)))
    with torch.no_grad():
        row = lambda t: t.abs().amax(1, keepdim=True)
        vs = (row(m * one("post_weight")) * k1 + zero("post_bias").abs().max())
        hs = row(d["residual"]) + one("scale").abs().max() * vs
        ns = row(n2) * k2 + hs * r2            # a normalised value's error over u
        ys = ns * one("next_weight").abs().max() + zero("next_bias").abs().max()
        g1, g2 = (t.double() for t in g)
        d2 = g2 * one("next_weight")
        ghs = row(g1) + r2 * row(d2) * (2 + ns * (1 + row(n2)))
        gvs = ghs * one("scale").abs().max()
        d1s = gvs * one("post_weight").abs().max()
        scales = dict(hidden=hs, normed=ys, residual=ghs, branch=r1 * d1s * (2 + (row(m) * k1) * (1 + row(m))),
                      gate=ghs * one("scale").abs().max() * vs * (D if "gate" in d and d["gate"].shape[1] < D else 1),
                      post_weight=(gvs * row(m) * k1).sum(0), post_bias=gvs.sum(0), scale=(ghs * vs).sum(0),
                      next_weight=(row(g2) * ns).sum(0), next_bias=row(g2).sum(0))
    return hidden.detach(), y.detach(), grads, scales


def _check(a, g, norm="layer", eps=1e-5, K=128.0):
    from cign_amd.fused_block_ops import fused_gated_residual_norm

    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
    hidden, normed = fused_gated_residual_norm(**leaves, eps=eps, norm=norm)
    got = dict(zip(leaves, torch.autograd.grad([hidden, normed], list(leaves.values()), g)))
    want_h, want_y, want, scales = _oracle(a, g, norm, eps)
    n = a["branch"].shape[0]
    for name, x, ref in [("hidden", hidden, want_h), ("normed", normed, want_y)] + [(k, got[k], want[k]) for k in got]:
        assert x.dtype == (a[name] if name in a else a["branch"]).dtype and x.shape == ref.shape, name
        k = K + (n / 256 if x.dim() == 1 else 0)
        tol = k * U * scales[name] + HALF[x.dtype] * ref.abs() + 1e-37
        err = (x.double() - ref).abs()
        assert bool((err <= tol).all()), (name, float((err / tol).max()))
    with torch.no_grad():
        h2, y2 = fused_gated_residual_norm(**a, eps=eps, norm=norm)
    assert torch.equal(h2, hidden) and torch.equal(y2, normed)


WIDTHS = [1, 2, 3, 4, 7, 8, 15, 16, 31, 64, 65, 255, 256, 257, 511, 512, 513, 1001, 1024, 1025, 2048, 2050, 4096, 4097,
          5000, 8190, 8191, 8192]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_widths(D, dtype, wdtype):
    k = WIDTHS.index(D)
    norm, gate = ("layer", "rms")[k % 2], ("value", "row", "none")[k % 3]
    if D == 1 and gate == "row":
        gate = "value"
    _check(*_inputs(37, D, dtype, wdtype, norm, gate, seed=k), norm=norm)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("gate", ["none", "row", "value"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [5, 96, 256, 1001, 8192])
def test_forms(D, dtype, gate, norm):
    _check(*_inputs(53, D, dtype, torch.float32, norm, gate, seed=7), norm=norm)


@pytest.mark.parametrize("n", [1, 2, 255, 1029, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_row_counts(n, dtype):
    _check(*_inputs(n, 100, dtype, dtype, seed=n))


def test_rows_far_from_zero_and_tiny():
    _check(*_inputs(40, 300, torch.float32, torch.float32, offset=100.0))
    _check(*_inputs(40, 300, torch.float32, torch.float32, scale=1e-6))


def test_without_vectors_and_partial_gradients():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    a, g = _inputs(50, 260, torch.float32, torch.float32)
    bare = {k: a[k] for k in ("branch", "residual")}
    _check(bare, g)
    _check({k: a[k] for k in ("branch", "residual", "gate", "scale")}, g, norm="rms")
    _check({k: a[k] for k in ("branch", "residual", "post_bias", "next_bias")}, g)
    full = {k: v.detach().requires_grad_() for k, v in a.items()}
    h, y = op(**full)
    every = dict(zip(full, torch.autograd.grad([h, y], list(full.values()), g)))
    for k in full:  # each gradient alone has the bits of all together
        one = {j: v.detach().requires_grad_(j == k) for j, v in a.items()}
        h, y = op(**one)
        got, = torch.autograd.grad([h, y], [one[k]], g)
        assert torch.equal(got, every[k]), k
    for i in range(2):  # one result's gradient alone is that of zeros for the other
        h, y = op(**full)
        got = torch.autograd.grad((h, y)[i], list(full.values()), g[i], allow_unused=True)
        h, y = op(**full)
        both = torch.autograd.grad([h, y], list(full.values()), [g[0] if i == 0 else torch.zeros_like(g[0]),
                                                                 g[1] if i == 1 else torch.zeros_like(g[1])])
        for k, p, q in zip(full, got, both):
            assert torch.equal(p, q), (i, k)


def test_strides_and_shapes():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    gen = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(2, 5, 4, 70, generator=gen, device="cuda")
    branch, residual, gate = base[:, :, 0, 1:66], base[:, :, 1, 2:67], base[:, :, 2, 3:68]
    want = op(branch.contiguous(), residual.contiguous(), gate=gate.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(op(branch, residual, gate=gate), want))
    t = base[0, 0].t()[:60]  # last axis strided: [60, 4]
    assert all(torch.equal(p, q) for p, q in zip(op(t, t), op(t.contiguous(), t.contiguous())))
    row = gate[..., :1]
    got = op(branch, residual, gate=row, scale=base[0, 0, 0, ::1][:65])
    full = op(branch, residual, gate=row.expand(2, 5, 65).contiguous(), scale=base[0, 0, 0, :65].clone())
    assert all((p - q).abs().max() <= 1e-6 for p, q in zip(got, full))
    wide = torch.randn(1, 65, generator=gen, device="cuda").expand(7, 65).requires_grad_()  # one row for all
    h, y = op(wide, wide)
    g, = torch.autograd.grad(y.sum() + h.square().sum(), wide)
    assert g.shape == (7, 65) and torch.equal(g[0], g[6])


def test_empty_rows_and_shared_inputs():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    a, _ = _inputs(4, 32, torch.float32, torch.float32)
    e = {k: (v[:0] if v.dim() == 2 else v).detach().requires_grad_() for k, v in a.items()}
    h, y = op(**e)
    assert h.shape == y.shape == (0, 32)
    got = torch.autograd.grad([h.sum() + y.sum()], list(e.values()))
    for k, g in zip(e, got):
        assert g.shape == e[k].shape and not g.any()
    x = a["branch"].requires_grad_()
    h, y = op(x, x)  # the same tensor twice
    g, = torch.autograd.grad([h, y], x, [torch.ones_like(h), a["gate"]])
    p, q = x.detach().requires_grad_(), x.detach().requires_grad_()
    h, y = op(p, q)
    gp, gq = torch.autograd.grad([h, y], [p, q], [torch.ones_like(h), a["gate"]])
    assert torch.equal(g, gp + gq)


def test_nonfinite_rows_stay_in_their_rows():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    a, _ = _inputs(9, 130, torch.float32, torch.float32)
    clean = op(**a)
    a["branch"][3, 5], a["residual"][5, 1], a["gate"][7, 2] = float("inf"), float("nan"), float("-inf")
    got = op(**a)
    for c, g in zip(clean, got):
        keep = [0, 1, 2, 4, 6, 8]
        assert torch.equal(c[keep], g[keep])
        assert g[5].isnan().any()
    assert got[0][7].isfinite().all() and got[0][7, 2] == a["residual"][7, 2]  # a closed gate
    a["gate"][7, 2] = 200.0
    h = op(**a)[0][7, 2]
    assert h.isfinite()


def test_gradient_against_differences():
    """Central differences of the float64 formula along random directions, 1e-6
    steps: a relative error of 1e-9 from the third derivative and 1e-10 from
    rounding, so the float32 gradient's own 1e-4 is what counts."""
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    a, g = _inputs(6, 24, torch.float32, torch.float32, seed=5)
    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
    h, y = op(**leaves)
    grads = dict(zip(leaves, torch.autograd.grad([h, y], list(leaves.values()), g)))

    def value(b):
        N = lambda t: (t - t.mean(1, keepdim=True)) / (t.var(1, keepdim=True, correction=0) + 1e-5).sqrt()
        hid = b["residual"] + b["scale"] * torch.sigmoid(b["gate"]) * (N(b["branch"]) * b["post_weight"] + b["post_bias"])
        return (hid * g[0].double()).sum() + ((N(hid) * b["next_weight"] + b["next_bias"]) * g[1].double()).sum()

    gen = torch.Generator(device="cuda").manual_seed(1)
    for k in a:
        d = torch.randn(a[k].shape, generator=gen, device="cuda").double()
        at = lambda t: value({j: v.double() + (t * d if j == k else 0) for j, v in a.items()})
        slope = (at(1e-6) - at(-1e-6)) / 2e-6
        mine = (grads[k].double() * d).sum()
        assert abs(slope - mine) <= 1e-4 * (grads[k].double() * d).abs().sum(), k


def test_deterministic_row_local_and_on_streams():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    a, g = _inputs(3001, 1001, torch.bfloat16, torch.bfloat16, gate="row")
    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}

    def step():
        h, y = op(**leaves)
        grads = torch.autograd.grad([h, y], list(leaves.values()), g)
        return [t.detach() for t in (h, y, *grads)]

    want = step()
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in side:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for r in got for p, q in zip(want, r))
    few = {k: v[100:103] if v.dim() == 2 else v for k, v in a.items()}
    assert all(torch.equal(p, q[100:103]) for p, q in zip(op(**few), want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            leaves["branch"].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, want)), i


def test_refusals():
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    x = torch.zeros(4, 32, device="cuda")
    v = torch.ones(32, device="cuda")
    for kw, err in ((dict(branch=x[:, :0], residual=x[:, :0]), ValueError), (dict(residual=x[:3]), ValueError),
                    (dict(residual=x.bfloat16()), TypeError), (dict(residual=x.cpu()), ValueError),
                    (dict(gate=x[:, :2]), ValueError), (dict(gate=x.bfloat16()), TypeError),
                    (dict(scale=v[:31]), ValueError), (dict(scale=v.bfloat16()), TypeError),
                    (dict(scale=v.cpu()), ValueError), (dict(post_weight=v.double()), TypeError),
                    (dict(norm="batch"), ValueError), (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError),
                    (dict(branch=x.half()), TypeError),
                    (dict(branch=torch.zeros(2, 8193, device="cuda"), residual=torch.zeros(2, 8193, device="cuda")),
                     ValueError)):
        with pytest.raises(err):
            op(**(dict(branch=x, residual=x) | kw))
    b = x.bfloat16()
    with pytest.raises(TypeError, match="all be float32"):
        op(b, b, scale=v, next_weight=v.bfloat16())
    r = x.clone().requires_grad_()
    h, y = op(r, x)
    g, = torch.autograd.grad(y.sum() + h.square().sum(), r, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
