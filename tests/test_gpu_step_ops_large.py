"""The operators of a training step on tensors of more than 2^31 and 2^32 values, where
an offset of 32 bits would wrap: rows and classes at the far end against the same ones
alone, or against float64."""
import torch
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B = torch.bfloat16


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_boundary_rows_beyond_32_bits():
    """Rows are worked on alone, so the last ones have the bits that they have by themselves, and so have the vectors'
    gradients where only the last row has one to give."""
    from cign_amd.fused_block_ops import fused_gated_residual_norm as op

    n, D, last = 530_000, 8192, 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    big = {k: torch.zeros(n, D, dtype=B, device="cuda") for k in ("branch", "residual")}
    big["gate"] = torch.zeros(n, 1, dtype=B, device="cuda")
    for t in big.values():
        t[-last:] = torch.randn(last, t.shape[1], generator=gen, device="cuda").to(B)
    vec = {k: torch.randn(D, generator=gen, device="cuda").to(B)
           for k in ("post_weight", "post_bias", "scale", "next_weight", "next_bias")}
    g = [torch.zeros(n, D, dtype=B, device="cuda") for _ in range(2)]
    for t in g:
        t[-1] = torch.randn(D, generator=gen, device="cuda").to(B)

    def run(rows):
        leaves = {k: v[-rows:].detach().requires_grad_() for k, v in big.items()}
        leaves.update({k: v.detach().requires_grad_() for k, v in vec.items()})
        out = op(**leaves)
        grads = torch.autograd.grad(out, list(leaves.values()), [t[-rows:] for t in g])
        return [t.detach()[-last:].clone() if t.shape[0] == rows else t for t in (*out, *grads)]

    assert all(torch.equal(p, q) for p, q in zip(run(n), run(last)))


def test_norm_of_a_tensor_beyond_32_bits():
    from cign_amd.grad_norm import clip_grad_norm, global_grad_norm

    n = (1 << 32) + 13
    g = torch.zeros(n, dtype=B, device="cuda")
    at = torch.tensor([0, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1], device="cuda")
    g[at] = torch.tensor([3.0, 5.0, 7.0, 11.0, 13.0, 4.0], dtype=B, device="cuda")
    want = (9 + 25 + 49 + 121 + 169 + 16) ** 0.5
    assert abs(float(global_grad_norm([g])) - want) <= 2 * U * want
    before = g[at].double()
    norm = clip_grad_norm([g], want / 2)
    assert abs(float(norm) - want) <= 2 * U * want
    assert bool(((g[at].double() - before / 2).abs() <= (2.0 ** -8 + 4 * U + 1e-6 / want) * before / 2).all())
    assert int(torch.count_nonzero(g)) == 6


@pytest.mark.parametrize("n", [5, 80])
def test_classes_beyond_31_bits(n):
    """2^20 classes of 2112 values; few rows are streamed, more come in tiles. The loss, the rows' gradient and the
    first and last classes' against float64, within the bounds of the smaller tests: products exact, their sums and
    the exponentials in float32, the logits' gradient rounded to bfloat16 once."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    V, D = 1 << 20, 2112
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, D, generator=gen, device="cuda").to(B)
    w = torch.randn(V, D, generator=gen, device="cuda", dtype=B).mul_(2 / D ** 0.5)
    labels = torch.randint(0, V, (n,), generator=gen, device="cuda")
    labels[: n // 2] = torch.randint(V - 100, V, (n // 2,), generator=gen, device="cuda")
    g = torch.rand(n, generator=gen, device="cuda") + 0.5
    p, q = x.detach().requires_grad_(), w.detach().requires_grad_()
    r = linear_cross_entropy(p, q, labels)
    gx, gw = torch.autograd.grad(r.loss, (p, q), g)

    X, G = x.double(), g.double()[:, None]

    def chunk(a, b):
        W = w[a:b].double()
        z = X @ W.t()
        return W, z, (D / 4 + 32) * U * (X.abs() @ W.abs().t()) + 2 * U * z.abs()

    parts = [chunk(a, a + 65536)[1:] for a in range(0, V, 65536)]
    lse = torch.logsumexp(torch.stack([torch.logsumexp(z, 1) for z, _ in parts]), 0)
    top = torch.stack([dz.amax(1) for _, dz in parts]).amax(0)
    at = torch.cat([z for z, _ in parts], 1).gather(1, labels[:, None])[:, 0]
    del parts
    tol = 2 * top + 300 * U + 4 * U * lse.abs()
    assert bool(((r.logsumexp.double() - lse).abs() <= tol + U * lse.abs()).all())
    loss = lse - at
    assert bool(((r.loss.double() - loss).abs() <= tol + top + 4 * U * at.abs() + U * loss.abs()).all())

    def terms(a, b):
        W, z, dz = chunk(a, b)
        hot = torch.zeros_like(z)
        here = (labels >= a) & (labels < b)
        hot[here, labels[here] - a] = g.double()[here]
        e = (z - lse[:, None]).exp()
        d = G * e - hot
        err = G * e * (2 * top[:, None] + 2 * dz + ((z - lse[:, None]).abs() + 8) * 2 * U) + 2 * U * hot + 2 * U * G * e
        return W, d, err + 2.0 ** -8 * d.abs()

    wx, tx = torch.zeros_like(X), torch.zeros_like(X)
    for a in range(0, V, 65536):
        W, d, e = terms(a, a + 65536)
        wx += d @ W
        tx += (e + (V / 4 + 96) * U * d.abs()) @ W.abs()
        if a in (0, V - 65536):
            val, t = d.t() @ X, e.t() @ X.abs() + (n / 4 + 96) * U * (d.abs().t() @ X.abs())
            got = gw[a: a + 65536].double()
            assert bool(((got - val).abs() <= t + 2.0 ** -8 * val.abs() + 1e-37).all()), a
    assert bool(((gx.double() - wx).abs() <= tx + 2.0 ** -8 * wx.abs()).all())
