"""GPU parity of fused_layernorm (any width) with the formula in float64, its
gradients, strides, streams, graphs and the model's output norm.

Bounds, with u = 2^-24 and D values a row. xh is what (x - mean) * rstd gives
for float32 sums: the mean is off by at most e_m = (L + 2) u max|x|, where L =
log2 of the row's threads plus the values a thread adds is the longest chain of
additions (at most 6 + 4 + 20), and each centred value by e_m plus u |x - mean|; the
variance's relative error is at most 2 (L + 3) u + 2 e_m / sigma'; so |xh error|
<= 1.5 e_m rstd + (L + 6) u |xh| plus the variance's cross term. The tests take L + 6 =
36 and double the sum, |y error| <= 72 u (|xh| + max|x| rstd) |w| + 2 u (|y| +
|b|), and, for bf16 rows, 2^-8 |y| for the store."""
import math

import numpy as np
import pytest
import torch

from tests.conftest import assert_within

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _n(t):
    return t.detach().double().cpu().numpy()


def _oracle(x, w, b, eps, g):
    """float64 forward and backward of [n, D] arrays, and the magnitudes the
    bounds need."""
    mean = x.mean(axis=1, keepdims=True)
    rstd = 1.0 / np.sqrt(((x - mean) ** 2).mean(axis=1, keepdims=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    d = g * w
    gx = rstd * (d - d.mean(axis=1, keepdims=True) - xh * (d * xh).mean(axis=1, keepdims=True))
    return dict(y=y, xh=xh, rstd=rstd, gx=gx, gw=(g * xh).sum(axis=0), gb=g.sum(axis=0), d=d)


def _bounds(x, w, b, g, o, dtype, wdtype):
    D = x.shape[1]
    half = HALF[dtype]
    big = np.abs(x).max(axis=1, keepdims=True) * o["rstd"]
    exh = 72 * U * (np.abs(o["xh"]) + big)  # of each normalised value
    ey = exh * np.abs(w) + 2 * U * (np.abs(o["y"]) + np.abs(b))
    # grad_x = rstd (d - c1 - xh c2): its terms' magnitudes, each with the error of xh or of a sum
    d = np.abs(o["d"])
    c1 = d.mean(axis=1, keepdims=True)
    c2 = (d * np.abs(o["xh"])).mean(axis=1, keepdims=True)
    ec2 = (d * exh).mean(axis=1, keepdims=True) + 72 * U * c2
    terms = d + c1 + np.abs(o["xh"]) * c2
    eg = o["rstd"] * (72 * U * terms + exh * c2 + np.abs(o["xh"]) * ec2)
    n = max(1, x.shape[0])
    chain = (2.0 * np.sqrt(n) + 64) * U  # a workgroup's rows, its slots, then the partial rows
    egw = chain * np.abs(g * o["xh"]).sum(axis=0) + (np.abs(g) * exh).sum(axis=0)
    egb = chain * np.abs(g).sum(axis=0)
    wh = HALF[wdtype]
    return dict(y=ey + half * (np.abs(o["y"]) + ey), gx=eg + half * (np.abs(o["gx"]) + eg),
                gw=egw + wh * (np.abs(o["gw"]) + egw), gb=egb + wh * (np.abs(o["gb"]) + egb))


def _inputs(n, D, dtype, wdtype, seed, scale=1.0, offset=0.0):
    rng = np.random.default_rng(seed)
    t = lambda a, ty: torch.from_numpy(np.asarray(a, np.float32)).cuda().to(ty)
    return (t(rng.standard_normal((n, D)) * scale + offset, dtype), t(1 + 0.3 * rng.standard_normal(D), wdtype),
            t(0.3 * rng.standard_normal(D), wdtype), t(rng.standard_normal((n, D)), dtype))


def _check(n, D, dtype, wdtype, seed=0, eps=1e-5, scale=1.0, offset=0.0):
    from cign_amd.fused_block_ops import fused_layernorm

    x, w, b, g = _inputs(n, D, dtype, wdtype, seed, scale, offset)
    for t in (x, w, b):
        t.requires_grad_()
    y = fused_layernorm(x, w, b, eps)
    assert y.dtype == dtype and y.shape == x.shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    with torch.no_grad():
        assert torch.equal(fused_layernorm(x, w, b, eps), y)  # without the statistics: the same values
    a = [_n(t) for t in (x, w, b, g)]
    o = _oracle(a[0], a[1], a[2], eps, a[3])
    bound = _bounds(*a, o, dtype, wdtype)
    for name, got in (("y", y), ("gx", gx), ("gw", gw), ("gb", gb)):
        assert_within(_n(got), o[name], bound[name], f"{name} n={n} D={D}")


F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16)]
# every width at which the kernel's shape changes, and odd ones around them
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 17, 31, 64, 100, 255, 256, 257, 511, 513, 768, 1001, 1024, 1025, 1280, 1283, 2047,
          2049, 4096, 4099, 8192, 8193, 16384]


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_layernorm_matches_the_formula(D, dtype, wdtype):
    print(f"layernorm D={D} {dtype} {wdtype}", flush=True)
    # narrow rows: eps of the variance's order keeps the formula's own condition bounded
    _check(37, D, dtype, wdtype, seed=D, eps=1e-2 if D < 16 else 1e-5)


@pytest.mark.parametrize("D", [1281, 1536, 1537, 2048, 9001, 12288, 12290])
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_layernorm_at_the_edges_of_the_workgroups_shapes(D, dtype, wdtype):
    """With more rows than workgroups, so that each takes several."""
    print(f"layernorm D={D} {dtype} {wdtype}", flush=True)
    _check(1100 if D < 4096 else 530, D, dtype, wdtype, seed=D)


@pytest.mark.parametrize("n", [1, 2, 255, 1029, 20011])
@pytest.mark.parametrize("dtype,wdtype", TYPES)
def test_layernorm_row_counts(n, dtype, wdtype):
    print(f"layernorm n={n} {dtype} {wdtype}", flush=True)
    _check(n, 129, dtype, wdtype, seed=n)


def test_layernorm_offset_rows():
    """A large common offset: the variance is that of the centred values."""
    _check(50, 1280, F32, F32, offset=100.0)
    _check(50, 4096, F32, F32, offset=-1000.0, scale=3.0)


def test_layernorm_without_parameters_and_partial_gradients():
    from cign_amd.fused_block_ops import fused_layernorm

    for dtype in (F32, BF16):
        x, w, b, g = _inputs(19, 300, dtype, F32, 5)
        ones, zeros = torch.ones_like(w), torch.zeros_like(b)
        with torch.no_grad():
            assert torch.equal(fused_layernorm(x), fused_layernorm(x, ones, zeros))
            assert torch.equal(fused_layernorm(x, w), fused_layernorm(x, w, zeros))
            assert torch.equal(fused_layernorm(x, None, b), fused_layernorm(x, ones, b))
        full = [t.clone().requires_grad_() for t in (x, w, b)]
        want = torch.autograd.grad(fused_layernorm(*full), full, g)
        for keep in range(3):  # one gradient at a time
            part = [t.clone().requires_grad_(i == keep) for i, t in enumerate((x, w, b))]
            got, = torch.autograd.grad(fused_layernorm(*part), part[keep], g)
            assert torch.equal(got, want[keep])
        xa = x.clone().requires_grad_()
        xb = x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(fused_layernorm(xa), xa, g)[0],
                           torch.autograd.grad(fused_layernorm(xb, ones, zeros), xb, g)[0])
        bias = b.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(fused_layernorm(x, None, bias), bias, g)[0], want[2])


def test_layernorm_strides_and_shapes():
    from cign_amd.fused_block_ops import fused_layernorm

    gen = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(40, 3, 1001, generator=gen, device="cuda")
    w, b = torch.randn(2, 333, generator=gen, device="cuda")
    views = [big[:, 1, 5:338], big[:, :, 600:933], big[::3, 2, 1:334], big[0, :, ::3][:, :333], big[:33, 0, :333].t()[:, :33]]
    for v in views:
        D = v.shape[-1]
        a = v.detach().clone().contiguous().requires_grad_()
        s = v.detach().requires_grad_()  # the view itself
        ya, ys = (fused_layernorm(t, w[:D], b[:D]) for t in (a, s))
        assert torch.equal(ya, ys) and ys.is_contiguous()
        g = torch.randn(*ya.shape, 2, generator=gen, device="cuda")[..., 0]  # a strided gradient
        assert torch.equal(torch.autograd.grad(ya, a, g.contiguous())[0], torch.autograd.grad(ys, s, g)[0])
        one = torch.ones((), device="cuda").expand(ya.shape)  # what .sum() hands back
        a2, s2 = a.detach().requires_grad_(), s.detach().requires_grad_()
        assert torch.equal(torch.autograd.grad(fused_layernorm(a2, w[:D], b[:D]), a2, one)[0],
                           torch.autograd.grad(fused_layernorm(s2, w[:D], b[:D]).sum(), s2)[0])
    row = torch.randn(333, generator=gen, device="cuda")
    assert torch.equal(fused_layernorm(row, w, b), fused_layernorm(row[None], w, b)[0])
    same = row.expand(6, 333).requires_grad_()  # one row read six times
    assert torch.equal(fused_layernorm(same, w, b)[5], fused_layernorm(row, w, b))


def test_layernorm_empty_and_constant_rows():
    from cign_amd.fused_block_ops import fused_layernorm

    w = torch.randn(64, device="cuda").requires_grad_()
    b = torch.randn(64, device="cuda").requires_grad_()
    x = torch.empty(0, 5, 64, device="cuda").requires_grad_()
    y = fused_layernorm(x, w, b)
    assert y.shape == x.shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == x.shape and not gw.any() and not gb.any()
    c = torch.full((3, 64), 7.25, device="cuda")
    assert torch.equal(fused_layernorm(c, w, b), b.detach().expand(3, 64))


def test_layernorm_nonfinite_rows_stay_in_their_rows():
    from cign_amd.fused_block_ops import fused_layernorm

    x = torch.randn(9, 1283, device="cuda")
    clean = fused_layernorm(x)
    bad = x.clone()
    bad[4, 1282] = math.nan
    bad[6, 0] = math.inf
    y = fused_layernorm(bad)
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(y[keep], clean[keep]) and y[4].isnan().all() and y[6].isnan().all()


def test_layernorm_gradient_against_differences():
    """Central differences of the float64 formula at the kernel's inputs."""
    from cign_amd.fused_block_ops import fused_layernorm

    x, w, b, g = _inputs(3, 23, F32, F32, 11)
    for t in (x, w, b):
        t.requires_grad_()
    grads = torch.autograd.grad(fused_layernorm(x, w, b, 1e-3), (x, w, b), g)
    arrays = [_n(t) for t in (x, w, b)]
    gn = _n(g)
    f = lambda: (_oracle(*arrays, 1e-3, gn)["y"] * gn).sum()
    h = 1e-5
    for a, got in zip(arrays, grads):
        num = np.empty_like(a)
        for i in np.ndindex(a.shape):
            v = a[i]
            a[i] = v + h
            up = f()
            a[i] = v - h
            num[i] = (up - f()) / (2 * h)
            a[i] = v
        # the differences' own error (h^2 times third derivatives, 1e-16 / h) is below 1e-7 here
        assert_within(_n(got), num, 1e-5 + 1e-5 * np.abs(num), "gradient")


def test_layernorm_is_deterministic_and_row_local():
    """Runs agree bit for bit, and a row's values do not depend on the others
    in the call."""
    from cign_amd.fused_block_ops import fused_layernorm

    for D, dtype in ((1280, F32), (4096, BF16), (1001, BF16)):
        x, w, b, g = _inputs(700, D, dtype, F32, D)
        for t in (x, w, b):
            t.requires_grad_()
        first = torch.autograd.grad(fused_layernorm(x, w, b), (x, w, b), g)
        again = torch.autograd.grad(fused_layernorm(x, w, b), (x, w, b), g)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
        with torch.no_grad():
            assert torch.equal(fused_layernorm(x[13:14], w, b), fused_layernorm(x, w, b)[13:14])


def test_layernorm_on_a_side_stream_and_in_a_graph():
    from cign_amd.fused_block_ops import fused_layernorm

    x, w, b, g = _inputs(513, 1281, BF16, F32, 2)
    for t in (x, w, b):
        t.requires_grad_()

    def step():
        y = fused_layernorm(x, w, b)
        # detached: no eager graph of the leaves lives on while a step is captured
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    eager = [t.clone() for t in step()]
    assert all(torch.equal(p, q) for p, q in zip(on_side, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        with torch.no_grad():
            x.add_(0.25 * k)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), k


def test_layernorm_refusals():
    from cign_amd.fused_block_ops import fused_layernorm

    x = torch.randn(4, 32, device="cuda")
    w, b = torch.ones(32, device="cuda"), torch.zeros(32, device="cuda")
    for bad in (x.double(), x.half(), x.cpu(), [1.0]):
        with pytest.raises(TypeError, match="x must be CUDA"):
            fused_layernorm(bad, w, b)
    with pytest.raises(ValueError, match="D<=16384"):
        fused_layernorm(torch.zeros(1, 16385, device="cuda"))
    with pytest.raises(ValueError, match="1<=D"):
        fused_layernorm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(ValueError, match=r"\[..., D\]"):
        fused_layernorm(torch.zeros((), device="cuda"))
    with pytest.raises(ValueError, match="weight must have shape"):
        fused_layernorm(x, w[:31], b)
    with pytest.raises(ValueError, match="bias must have shape"):
        fused_layernorm(x, w, b[None])
    with pytest.raises(ValueError, match="must be on"):
        fused_layernorm(x, w.cpu(), b)
    for ww, bb in ((w.bfloat16(), b.bfloat16()), (w.half(), None)):
        with pytest.raises(TypeError, match="weight/bias"):
            fused_layernorm(x, ww, bb)
    with pytest.raises(TypeError, match="weight/bias"):
        fused_layernorm(x.bfloat16(), w, b.bfloat16())
    for eps in (-1e-5, math.nan, math.inf):
        with pytest.raises(ValueError, match="eps"):
            fused_layernorm(x, w, b, eps)
    xr = x.clone().requires_grad_()
    gx, = torch.autograd.grad(fused_layernorm(xr, w, b).pow(2).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        gx.sum().backward()
