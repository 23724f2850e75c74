"""GPU parity of class_logprobs with its definition in float64: log
probabilities, entropy, top classes and the gradient, over widths, masks,
ties, strides, streams and graphs.

Bounds, u = 2^-24, z = (x - m) / T (m the row's largest logit), s = sum e^z:
- a term e^z is off by at most (3 |z| + 2) u of itself (the difference, the
  factor and their product; the exponential), a sum by a chain of at most 64
  values of a thread, 6 + 2 lane and wavefront steps and 6 joining slices: s by
  u (80 + 2 + 3 mean|z|) of itself, means taken with the weights p; log s by
  that, plus 2 u |log s| of its own: E_lse = u (100 + 4 mean|z| + 4 |log s|);
- log p = z - log s: E_lse + 4 u |z|;
- entropy = log s - mean z: E_lse + u (100 mean|z| + 4 mean z^2);
- p in the gradient: relative E_p = E_lse + u (4 |z| + 4 |log s| + 4);
- grad = (g ([label] - p) - h p (log p + H)) / T: p (|g| + |h| (|log p| + H))
  (E_p + 8 u) + p |h| (E_H + 4 u (|z| + |log s|)) + 2 u |g| at the label, then
  half a step of the logits' type;
- a p below 2^-126 comes out of the hardware exponential as 0: an error of up
  to 2^-126 in p, so 2^-126 (|g| + |h| (|log p| + H)) / T in grad (at T = 0.01,
  |log p| = 80: 10^4 times 2^-126, which a bare 2^-126 does not cover)."""
import math

import numpy as np
import pytest
import torch

from tests.conftest import assert_within

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


def _n(t):
    return t.detach().double().cpu().numpy()


def _oracle(x, T, labels=None, ignore=-100, g=None, h=None):
    """Everything in float64 from [n, V] logits, with the bounds above."""
    n, V = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(axis=1, keepdims=True)
        none = (m == -np.inf)[:, 0]
        z = (x - np.where(m == -np.inf, 0.0, m)) / T
        e = np.exp(z)
        s = e.sum(axis=1, keepdims=True)
        ls = np.log(s)
        p = np.where(none[:, None], 0.0, e / s)
        lp = np.where(none[:, None], -np.inf, z - ls)
        zf = np.where(p > 0, z, 0.0)
        H = np.where(none, 0.0, ls[:, 0] - (p * zf).sum(axis=1))
        az, az2 = (p * np.abs(zf)).sum(axis=1), (p * zf * zf).sum(axis=1)
        als = np.where(none, 0.0, np.abs(ls[:, 0]))
        e_lse = U * (100 + 4 * az + 4 * als)
        e_h = e_lse + U * (100 * az + 4 * az2)
        e_lp = np.where(np.isfinite(lp), e_lse[:, None] + 4 * U * np.abs(np.where(np.isfinite(z), z, 0.0)), 0.0)
        o = dict(lp=lp, H=H, e_lp=e_lp, e_h=e_h)
        if labels is not None:
            rows = np.arange(n)
            ok = (labels >= 0) & (labels < V)
            at = np.where(ok, labels, 0)
            given = labels != ignore
            o["logprob"] = np.where(given, np.where(ok, lp[rows, at], np.nan), 0.0)
            o["e_logprob"] = np.where(given & ok, e_lp[rows, at], 0.0)
        if g is not None or h is not None:
            gg = np.zeros(n) if g is None else np.where(given, np.where(ok, g, np.nan), 0.0)
            hh = np.zeros(n) if h is None else h
            gg, hh = np.where(none, 0.0, gg)[:, None], np.where(none, 0.0, hh)[:, None]
            lpf = np.where(p > 0, lp, 0.0)
            grad = -p * (gg + hh * (lpf + H[:, None]))
            e_p = e_lse[:, None] + U * (4 * np.abs(zf) + 4 * als[:, None] + 4)
            weight = np.abs(gg) + np.abs(hh) * (np.abs(lpf) + H[:, None])
            err = p * weight * (e_p + 8 * U) + 2.0 ** -126 * weight \
                + p * np.abs(hh) * (e_h[:, None] + 4 * U * (np.abs(zf) + als[:, None]))
            if labels is not None:
                hit = np.where(given & ok & ~none, np.where(np.isnan(gg[:, 0]), 0.0, gg[:, 0]), 0.0)
                grad[rows, at] += hit
                err[rows, at] += 2 * U * np.abs(hit)
            o["grad"], o["e_grad"] = grad / T, (err + 4 * U * np.abs(grad)) / T
    return o


def _top(x, k):
    """Falling order, the lowest index first among equals, NaN as -inf."""
    v = np.where(np.isnan(x), -np.inf, x) + 0.0
    return np.argsort(-v, axis=1, kind="stable")[:, :k]


def _check(x, labels, top_k=0, T=1.0, g=None, h=None, ignore=-100, name=""):
    from cign_amd.class_logprobs import class_logprobs

    xr = x.detach().requires_grad_(g is not None or h is not None)
    r = class_logprobs(xr, labels, top_k=top_k, temperature=T, ignore_index=ignore)
    xn = _n(x)
    T = float(np.float32(T))
    o = _oracle(xn, T, None if labels is None else labels.cpu().numpy(), ignore, None if g is None else _n(g),
                None if h is None else _n(h))
    assert_within(_n(r.entropy), o["H"], o["e_h"], f"entropy {name}")
    if labels is None:
        assert r.logprob is None
    else:
        _within(_n(r.logprob), o["logprob"], o["e_logprob"], f"logprob {name}")
    if top_k:
        want = _top(xn, top_k)
        assert r.top_index.dtype == torch.int64
        assert np.array_equal(r.top_index.cpu().numpy(), want), f"top_index {name}"
        _within(_n(r.top_logprobs), np.take_along_axis(o["lp"], want, 1), np.take_along_axis(o["e_lp"], want, 1),
                f"top_logprobs {name}")
    else:
        assert r.top_index is None and r.top_logprobs is None
    if xr.requires_grad:
        outs, gs = zip(*[(a, b) for a, b in ((r.logprob, g), (r.entropy, h)) if b is not None])
        grad, = torch.autograd.grad(outs, xr, gs)
        assert grad.dtype == x.dtype and grad.shape == x.shape
        half = HALF[x.dtype]
        # a bf16 or float32 subnormal result rounds to a step of 2^-133 or 2^-149
        _within(_n(grad), o["grad"], o["e_grad"] + half * (np.abs(o["grad"]) + o["e_grad"]) + 2.0 ** -126,
                f"grad {name}")
    with torch.no_grad():  # without the statistics: the same values
        r2 = class_logprobs(x.detach(), labels, top_k=top_k, temperature=T, ignore_index=ignore)
    assert all(a is b is None or _same(a, b) for a, b in zip(r, r2))


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=7e33), b.nan_to_num(nan=7e33)) if a.is_floating_point() else torch.equal(a, b)


def _within(a, e, bound, name):
    """assert_within with infinities equal to themselves."""
    inf = np.isinf(e)
    assert np.array_equal(a[inf], e[inf]), name
    assert_within(np.where(inf, 0.0, a), np.where(inf, 0.0, e), bound, name)


def _logits(n, V, dtype, seed, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, V, generator=gen, device="cuda") * scale + torch.randn(n, 1, generator=gen, device="cuda")
    labels = torch.randint(0, V, (n,), generator=gen, device="cuda")
    g, h = torch.randn(2, n, generator=gen, device="cuda")
    return x.to(dtype), labels, g, h


# every width at which the kernels' shapes change, and odd ones around them
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 16, 18, 33, 64, 100, 255, 256, 257, 511, 512, 513, 1000, 1025, 2047, 2048, 2049, 4096,
          4097, 5001, 8192, 16385, 32000, 50001]


@pytest.mark.parametrize("V", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logprobs_match_the_definition(V, dtype):
    print(f"class_logprobs V={V} {dtype}", flush=True)
    n = 37 if V < 5000 else 5
    x, labels, g, h = _logits(n, V, dtype, V)
    labels[::3] = -100
    _check(x, labels, 0, 1.0, g, h, name=f"V={V}")
    _check(x, labels, min(V, 5), 0.7, g, None, name=f"V={V} T=0.7")
    _check(x, None, min(V, 1), 2.0, None, h, name=f"V={V} T=2")


@pytest.mark.parametrize("V", [3, 40, 128, 200, 512, 700, 5000, 20011, 70001])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [3, 700])
def test_top_lists_of_every_length(V, dtype, n):
    if n * V > 4_000_000:
        n = 4_000_000 // V
    print(f"top lists V={V} {dtype} n={n}", flush=True)
    x, labels, _, _ = _logits(n, V, dtype, V + n)
    for k in {1, 2, min(V, 17), min(V, 64), min(V, 128)} | ({V} if V <= 128 else set()):
        _check(x, labels, k, name=f"V={V} k={k}")


@pytest.mark.parametrize("V", [100, 3000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_lists_with_ties_and_orders(V, dtype):
    """Equal rows, few distinct values, sorted rows, all large values in one
    thread's chunks (more candidates than a slice keeps), signed zeros."""
    print(f"ties V={V} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(V)
    k = min(V, 128)
    idx = torch.arange(V, device="cuda", dtype=F32)
    rows = [torch.zeros(V, device="cuda"), torch.full((V,), -3.0, device="cuda"),
            torch.randint(0, 3, (V,), generator=gen, device="cuda").float(),
            idx / 64, -idx / 64, torch.where(idx.long() // 8 % 256 < 3, 5.0, -5.0),
            torch.where(idx.long() // 4 % 256 == 7, 4.0, 0.0) + (idx % 5) / 8,
            torch.where(idx.long() % 2 == 0, -0.0, 0.0)]
    x = torch.stack(rows).to(dtype)
    for kk in {1, 3, k}:
        _check(x, None, kk, name=f"V={V} k={kk}")
    many = x.repeat(150, 1)
    _check(many, None, 20, name="many rows")


@pytest.mark.parametrize("V", [5, 100, 3000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masks(V, dtype):
    """Masked classes, rows with one class left and with none, masks of the
    type's lowest value, masked labels, and top lists longer than what is
    left."""
    print(f"masks V={V} {dtype}", flush=True)
    x, labels, g, h = _logits(9, V, dtype, V)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, V // 2] = 2.0
    x[2, : V // 2] = -math.inf
    x[3, labels[3]] = -math.inf
    x[4] = torch.finfo(dtype).min
    x[5, 1:] = torch.finfo(dtype).min
    x[6, ::2] = torch.finfo(dtype).min
    x[6, 1::2] = -math.inf
    _check(x, labels, min(V, 30), 1.0, g, h, name=f"V={V}")
    _check(x, labels, min(V, 3), 1.5, g, None, name=f"V={V} T=1.5")
    from cign_amd.class_logprobs import class_logprobs

    r = class_logprobs(x[:1].requires_grad_(), labels[:1], top_k=min(V, 30))
    assert r.logprob.item() == -math.inf and r.entropy.item() == 0.0
    assert r.top_index[0].tolist() == list(range(min(V, 30))) and (r.top_logprobs == -math.inf).all()


@pytest.mark.parametrize("V", [6, 3000, 40000])
def test_nonfinite_logits_stay_in_their_rows(V):
    from cign_amd.class_logprobs import class_logprobs

    x, labels, g, h = _logits(8, V, F32, V)
    bad = x.clone()
    bad[2, V - 1] = math.nan
    bad[5, 0] = math.inf
    labels[6] = -100
    bad[6] = math.nan
    bad.requires_grad_()
    clean = class_logprobs(x.requires_grad_(), labels, top_k=3)
    got = class_logprobs(bad, labels, top_k=3)
    keep = [0, 1, 3, 4, 7]
    for a, b in zip(got, clean):
        assert torch.equal(a[keep], b[keep])
    assert got.logprob[[2, 5]].isnan().all() and got.entropy[[2, 5, 6]].isnan().all()
    assert got.logprob[6] == 0 and got.top_index[5, 0] == 0 and got.top_index[6].tolist() == [0, 1, 2]
    want = _top(_n(bad)[2:3], 3)
    assert np.array_equal(got.top_index[2:3].cpu().numpy(), want)
    ga, = torch.autograd.grad(got.logprob, bad, g)
    gb, = torch.autograd.grad(clean.logprob, x, g)
    assert torch.equal(ga[keep], gb[keep]) and ga[2].isnan().all()
    assert not ga[6].any()  # an ignored row: zeros, whatever its logits hold


@pytest.mark.parametrize("V", [6, 300, 3000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_top_lists_beside_nan(V, dtype):
    """A NaN, of either sign, ranks as -inf and hides none of the classes read
    with it."""
    x = _logits(12, V, dtype, V)[0]
    k = min(V, 20)
    best = x.float().topk(min(3, V), dim=1).indices
    for r in range(12):
        # next to the row's best classes, and elsewhere
        for i in {int(best[r, r % best.shape[1]]) ^ (1 + r % 3), (r * 37) % V}:
            if i < V and i not in best[r].tolist()[:1]:
                x[r, i] = math.nan if r % 2 else -math.nan
    if dtype == BF16:  # the sign bit as well
        x.view(torch.int16)[::2][x[::2].isnan()] = -64
    from cign_amd.class_logprobs import class_logprobs

    assert x.isnan().any(dim=1).sum() >= 8
    got = class_logprobs(x, top_k=k).top_index.cpu().numpy()
    assert np.array_equal(got, _top(_n(x), k))


def test_labels_out_of_range_are_seen():
    from cign_amd.class_logprobs import class_logprobs

    for V in (5, 3000, 40000):
        x, _, g, _ = _logits(5, V, F32, 1)
        labels = torch.tensor([0, V, -1, -100, V - 1], device="cuda")
        _check(x, labels, 0, 1.0, g, None, name=f"V={V}")
        _check(x, labels, 0, 1.0, g, None, ignore=V, name=f"V={V}, ignore V")
        r = class_logprobs(x, labels.int())
        assert r.logprob[[1, 2]].isnan().all() and r.logprob[3] == 0 and r.logprob[[0, 4]].isfinite().all()


def test_strides_shapes_and_offsets():
    from cign_amd.class_logprobs import class_logprobs

    gen = torch.Generator(device="cuda").manual_seed(4)
    for dtype in (F32, BF16):
        big = torch.randn(6, 4, 5100, generator=gen, device="cuda").to(dtype)
        views = [big[:, 1, 3:5004], big[:, :, :4999], big[2, :, 1:8], big[::2, 3, 7:607], big[:, :, ::3], big[1, 2, 5:105],
                 big[:1, 0, :50].expand(7, 50), big[:, 0, :6].t()]
        for v in views:
            a = v.detach().clone().contiguous().requires_grad_()
            s = v.detach().requires_grad_()
            labels = torch.randint(0, v.shape[-1], v.shape[:-1], generator=gen, device="cuda")
            ra, rs = (class_logprobs(t, labels, top_k=3) for t in (a, s))
            for p, q in zip(ra, rs):
                assert p.shape[: v.dim() - 1] == v.shape[:-1] and torch.equal(p, q)
            w = torch.randn(*labels.shape, 2, generator=gen, device="cuda")[..., 1]  # a strided gradient
            assert torch.equal(torch.autograd.grad(ra.logprob, a, w.contiguous())[0],
                               torch.autograd.grad(rs.logprob, s, w)[0])
        a, s = (big[:, 1, 3:5004].detach().requires_grad_() for _ in range(2))
        labels = torch.zeros(6, dtype=torch.int64, device="cuda")
        assert torch.equal(torch.autograd.grad(class_logprobs(a, labels).logprob.sum(), a)[0],
                           torch.autograd.grad(class_logprobs(s, labels).logprob, s, torch.ones(6, device="cuda"))[0])
    none = class_logprobs(torch.empty(0, 7, device="cuda").requires_grad_(),
                          torch.empty(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert none.logprob.shape == (0,) and none.top_index.shape == (0, 2)
    assert torch.autograd.grad(none.entropy.sum() + none.logprob.sum(), [none.entropy])[0].shape == (0,)


def test_gradient_against_differences():
    from cign_amd.class_logprobs import class_logprobs

    x, labels, g, h = _logits(4, 23, F32, 9, scale=1.0)
    labels[1] = -100
    x.requires_grad_()
    r = class_logprobs(x, labels, temperature=1.5)
    got, = torch.autograd.grad([r.logprob, r.entropy], x, [g, h])
    a, ln, gn, hn = _n(x), labels.cpu().numpy(), _n(g), _n(h)

    def f():
        o = _oracle(a, 1.5, ln)
        return (o["logprob"] * gn).sum() + (o["H"] * hn).sum()

    num = np.empty_like(a)
    step = 1e-5
    for i in np.ndindex(a.shape):
        v = a[i]
        a[i] = v + step
        up = f()
        a[i] = v - step
        num[i] = (up - f()) / (2 * step)
        a[i] = v
    assert_within(_n(got), num, 2e-6 + 1e-5 * np.abs(num), "gradient")


def test_large_offsets_and_temperatures():
    for dtype, off in ((F32, 1000.0), (F32, -3e4), (BF16, 512.0)):
        x, labels, g, h = _logits(20, 3001, F32, 3)
        _check((x + off).to(dtype), labels, 4, 1.0, g, h, name=f"offset {off}")
    x, labels, g, h = _logits(20, 301, F32, 5)
    for T in (0.01, 0.25, 8.0, 100.0):
        _check(x, labels, 4, T, g, h, name=f"T={T}")


@pytest.mark.parametrize("V", [40, 3000, 40000])
def test_rows_far_from_zero(V):
    """Logits whose steps are 2^-4, 1, 64 and 2^13 (spreads of a few steps), and
    rows half of which lies on either side of where the shift's rounded product
    is given up for the difference (|x| log2(e) / T = 10^6)."""
    for off, step in ((6.5e5, 0.0625), (-6.9314e5, 0.0625), (1e7, 1.0), (-1e9, 64.0), (1e11, 8192.0)):
        x, labels, g, h = _logits(12, V, F32, V)
        x = off + (x * 2).round() * step
        T = max(1.0, step)
        _check(x, labels, min(V, 4), T, g, h, name=f"offset {off}")
    x, labels, g, h = _logits(12, V, F32, V + 1)
    edge = 1e6 / 1.4426950408889634
    x = edge + x.round()  # half of the values beyond
    x[6:] *= -1
    _check(x, labels, min(V, 4), 1.0, g, h, name="at the edge")


def test_large_gradients_beside_masks():
    """Gradients of the entropy of 10^9 and more, as a scaled loss or a small
    temperature makes them: a masked class's stays 0."""
    for V in (6, 300, 3000, 40000):
        for dtype in (F32, BF16):
            print(f"large gradients V={V} {dtype}", flush=True)
            x, labels, g, h = _logits(6, V, dtype, V + 3)
            x[:, 1::3] = -math.inf
            x[1, 2::3] = torch.finfo(dtype).min
            labels = torch.zeros_like(labels)
            _check(x, labels, 0, 1.0, g * 1e9, h * 1e12, name=f"V={V}")
            _check(x, labels, 0, 2.0 ** -6, g, h * 1e9, name=f"V={V}, small T")


def test_more_rows_than_a_grid_dimension():
    """131,100 rows of a slice each: the grid's second dimension ends at 65,535."""
    from cign_amd.class_logprobs import class_logprobs

    n, V = 131100, 601
    x, labels, _, _ = _logits(n, V, BF16, 1)
    r = class_logprobs(x, labels, top_k=3)
    for a in (0, 65530, 131066):
        xn, at = _n(x[a:a + 34]), labels[a:a + 34].cpu().numpy()
        o = _oracle(xn, 1.0, at)
        want = _top(xn, 3)
        assert_within(_n(r.entropy[a:a + 34]), o["H"], o["e_h"], f"entropy from row {a}")
        assert_within(_n(r.logprob[a:a + 34]), o["logprob"], o["e_logprob"], f"logprob from row {a}")
        assert np.array_equal(r.top_index[a:a + 34].cpu().numpy(), want)


def test_row_results_do_not_depend_on_the_call():
    """A row's values and gradient are the same in a call of its own, where
    its kernel shape is the same, and runs agree bit for bit."""
    from cign_amd.class_logprobs import class_logprobs

    for V in (18, 3000):
        x, labels, g, h = _logits(300, V, BF16, V)
        x.requires_grad_()
        outs = []
        for _ in range(2):
            r = class_logprobs(x, labels, top_k=2 if V < 512 else 0)
            outs.append((*[t for t in r if t is not None], *torch.autograd.grad([r.logprob, r.entropy], x, [g, h])))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        one = class_logprobs(x[77:78], labels[77:78])
        assert torch.equal(one.logprob, outs[0][0][77:78]) and torch.equal(one.entropy, outs[0][1][77:78])


def test_offsets_beyond_32_bits():
    """More than 2^32 values: rows near the end."""
    from cign_amd.class_logprobs import class_logprobs

    V = 1 << 16
    n = (1 << 16) + 3
    x = torch.zeros(n, V, dtype=BF16, device="cuda")
    x[n - 1, 5] = 3.0
    x[n - 2, V - 1] = 4.0
    x[0, 1] = 5.0
    labels = torch.full((n,), V - 1, device="cuda")
    x.requires_grad_()
    r = class_logprobs(x, labels, top_k=1)
    assert r.top_index[[0, n - 2, n - 1], 0].tolist() == [1, V - 1, 5]
    want = math.log(math.exp(4.0) / (V - 1 + math.exp(4.0)))
    assert abs(r.logprob[n - 2].item() - want) < 1e-4
    assert abs(r.logprob[n - 3].item() + math.log(V)) < 1e-4
    g = torch.zeros(n, device="cuda")
    g[n - 1] = 1.0
    grad, = torch.autograd.grad(r.logprob, x, g)
    assert abs(grad[n - 1].float().sum().item()) < 1e-2 and grad[n - 1, V - 1] > 0.99
    assert not grad[0].any() and not grad[n - 2].any()


def test_side_stream_and_graph():
    from cign_amd.class_logprobs import class_logprobs

    cases = []
    for n, V, dtype, k in ((500, 18, F32, 3), (30, 50001, BF16, 20), (2, 40000, F32, 128)):
        x, labels, g, h = _logits(n, V, dtype, V)
        cases.append((x.requires_grad_(), labels, g, h, k))

    def step():
        out = []
        for x, labels, g, h, k in cases:
            r = class_logprobs(x, labels, top_k=k)
            # detached: no eager graph of the leaves lives on while a step is captured
            out += [t.detach() for t in (*r, *torch.autograd.grad([r.logprob, r.entropy], x, [g, h]))]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    graphs, held = [], []
    for _ in range(2):  # two graphs of the same calls, replayed in turn
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    for i in range(4):
        with torch.no_grad():
            for x, *_ in cases:
                x.mul_(0.9)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held[i % 2]]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_refusals():
    from cign_amd.class_logprobs import class_logprobs

    x = torch.randn(4, 10, device="cuda")
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (x.double(), x.half(), x.cpu(), None):
        with pytest.raises(TypeError, match="logits must be CUDA"):
            class_logprobs(bad, y)
    for bad in (x[:, :0], torch.zeros((), device="cuda"), torch.zeros(1, device="cuda").expand(1 << 20 | 1)):
        with pytest.raises(ValueError, match="logits must be"):
            class_logprobs(bad)
    for k in (-1, 11):
        with pytest.raises(ValueError, match="top_k"):
            class_logprobs(x, y, top_k=k)
    with pytest.raises(ValueError, match="top_k"):
        class_logprobs(torch.zeros(1, 1000, device="cuda"), top_k=129)
    for t in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            class_logprobs(x, y, temperature=t)
    with pytest.raises(TypeError, match="labels"):
        class_logprobs(x, y.float())
    with pytest.raises(ValueError, match="labels must have shape"):
        class_logprobs(x, y[:3])
    with pytest.raises(ValueError, match="labels must be on"):
        class_logprobs(x, y.cpu())
    xr = x.clone().requires_grad_()
    r = class_logprobs(xr, y, top_k=2)
    assert r.logprob.requires_grad and not r.top_logprobs.requires_grad
    grad, = torch.autograd.grad(r.logprob.pow(2).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


@pytest.mark.parametrize("V", [2, 3, 5, 37, 100, 129, 300, 1000, 1025, 3001, 5001, 20011, 50001, 131071])
def test_logarithms_of_the_sums(V):
    """Classes that are all equal: every sum is a whole number, exact in
    float32, so log p = -log V and the entropy log V up to a logarithm's error of
    at most 2^-24, however large it is, and half a step of the result."""
    from cign_amd.class_logprobs import class_logprobs

    want = math.log(V)
    bound = U + float(np.spacing(np.float32(want))) / 2
    for n in (3, 700):
        for dtype in (F32, BF16):
            x = torch.full((n, V), 0.75, dtype=dtype, device="cuda")
            r = class_logprobs(x, torch.full((n,), V - 1, device="cuda"), top_k=2)
            for v in (-r.logprob, r.entropy, -r.top_logprobs):
                assert (v.double() - want).abs().max() <= bound, (V, n, dtype)


def test_log_probabilities_further_off_than_float32_differences():
    """log p = -1.5e38 at T = 4 of a class at one end of the type's range beside
    one at the other: their difference alone overflows."""
    from cign_amd.class_logprobs import class_logprobs

    for V in (5, 300, 3000, 40000):
        x = torch.full((2, V), -3.0e38, device="cuda")
        x[:, 1] = 3.0e38
        r = class_logprobs(x, torch.tensor([0, 1], device="cuda"), top_k=3, temperature=4.0)
        assert abs(r.logprob[0].item() + 1.5e38) <= 4 * U * 1.5e38 and r.logprob[1] == 0
        assert r.top_index[0].tolist() == [1, 0, 2] and (r.top_logprobs[:, 1:] + 1.5e38).abs().max() <= 4 * U * 1.5e38
        assert not r.entropy.any()


def test_zero_rows():
    from cign_amd.class_logprobs import class_logprobs

    for V in (7, 300, 40000):
        x = torch.empty(0, V, device="cuda").requires_grad_()
        labels = torch.empty(0, dtype=torch.int64, device="cuda")
        r = class_logprobs(x, labels, top_k=2)
        assert r.logprob.shape == (0,) and r.top_logprobs.shape == (0, 2)
        e = torch.empty(0, device="cuda")
        for outs in ([r.logprob, r.entropy], [r.logprob], [r.entropy]):
            grad, = torch.autograd.grad(outs, x, [e] * len(outs), retain_graph=True)
            assert grad.shape == x.shape
