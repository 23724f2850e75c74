"""GPU parity of distill_topk_loss with its definition in float64: loss and
gradient over widths, list lengths, tails, empty places, masks, strides and
graphs, and the operators at the model's output together.

Bounds, u = 2^-24, z = (x - m) / T, over all classes and over those outside
the list (the statistics the kernel keeps): log of a sum is off by E = u (100 +
4 mean|z| + 4 |log s|) (a term by (3 |z| + 2) u, a chain of additions of at
most 80, the logarithm's own rounding); log q_i by E + 4 u |z_i|, a probability by that
and 4 u (|z| + |log s| + 1) of itself. So
- loss: T^2 [sum p (2 E + 4 u |z|) + r (2 E + 4 u |z_rest|)] + u |loss|, the
  sums over the list being float64;
- gradient of a class outside the list, C r_j with C = A q_rest - r and r_j its
  share of q_rest: C by A q_rest (3 E + 8 u (|z| + |log s|)), in q_j's terms A q_j
  (...), r_j by E_rest + 4 u (|z_j - m_rest| + |log s_rest| + 1) of itself, so of
  the value (where q_rest is 1e-60 the value is -r r_j and A q_j bounds none of
  it), and 16 u |value|; of a listed one g T [A q_j (...) + 4 u p_j]; 2^-126 g T
  (A + r) where an exponential flushes to 0, then half a step of the logits'
  type."""
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


def _lse(z, axis=1):
    """(log sum e^(z - max), mean |z - max|, its magnitude, max) of rows that
    may be all -inf (max 0 then). The logarithm is kept apart from the largest
    value: at the type's lowest value, -3e38, their sum would lose it, and a KL
    of equal logits came out negative."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(axis=axis, keepdims=True)
        m0 = np.where(m == -np.inf, 0.0, m)
        e = np.exp(z - m0)
        s = e.sum(axis=axis, keepdims=True)
        away = np.where(e > 0, e * np.where(e > 0, m0 - z, 0.0), 0.0).sum(axis=axis, keepdims=True) / np.where(s > 0, s, 1)
        ls = np.log(s)
        return ls[:, 0], away[:, 0], np.where(s > 0, np.abs(ls), 0.0)[:, 0], m0


def _oracle(x, t, index, T, tail, g):
    n, V = x.shape
    K = index.shape[1]
    z = x / T
    loss, eloss = np.zeros(n), np.zeros(n)
    grad, egrad = np.zeros((n, V)), np.zeros((n, V))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        lse, away, als, m0 = _lse(z)
        E = U * (100 + 4 * away + 4 * als)
        for r in range(n):
            present = index[r] >= 0
            j, v = index[r][present], t[r][present]
            if (j >= V).any():
                loss[r] = np.nan
                grad[r] = egrad[r] = np.nan
                continue
            if not present.any():
                continue
            if tail:
                p = np.exp(v)
            else:
                top = v.max()
                p = np.exp(v - top) / np.exp(v - top).sum() if top > -np.inf else np.zeros_like(v)
            member = np.zeros(V, bool)
            member[j] = True
            lq = (z[r] - m0[r, 0]) - lse[r] if lse[r] > -np.inf else np.full(V, -np.inf)
            q = np.exp(lq)
            on = p > 0
            az = np.abs(np.where(np.isfinite(z[r]), z[r] - m0[r, 0], 0.0))
            terms = p[on] * (np.log(p[on]) - lq[j][on])
            el = (p[on] * (2 * E[r] + 4 * U * az[j][on])).sum()
            left, lrest, Er = 0.0, 0.0, 0.0
            e_share = np.zeros(V)
            if tail and not member.all():
                left = max(0.0, 1.0 - p.sum())
                lr, ar, alr, mr = _lse(z[r][None, ~member])
                Er = U * (100 + 4 * ar[0] + 4 * alr[0])
                lrest = (mr[0, 0] - m0[r, 0]) + lr[0] - lse[r] if lse[r] > -np.inf else -np.inf
                e_share = Er + 4 * U * (np.abs(np.where(np.isfinite(z[r]), z[r] - mr[0, 0], 0.0)) + alr[0] + 1)
                if left > 0:
                    terms = np.append(terms, left * (np.log(left) - lrest))
                    el += left * (2 * E[r] + 2 * Er + 4 * U * np.abs(mr[0, 0] - m0[r, 0]) if lrest > -np.inf else 0)
            loss[r] = T * T * terms.sum()
            eloss[r] = T * T * el + U * np.abs(loss[r]) + T * T * 1e-13 * np.abs(terms).sum()
            A = p.sum() + left
            mass = np.zeros(V)
            np.add.at(mass, j, p)
            rest = np.where(member, 0.0, np.exp(lq - lrest)) if lrest > -np.inf else np.zeros(V)
            grad[r] = g[r] * T * (A * q - mass - left * rest)
            e = A * q * (3 * (E[r] + Er) + 8 * U * (az + als[r] + 4)) + 4 * U * mass \
                + np.abs(A * q - left * rest) * (16 * U + np.where(member, 0.0, e_share))
            egrad[r] = np.abs(g[r]) * T * (e + 2.0 ** -126 * (A + left)) + 4 * U * np.abs(grad[r])
    return loss, eloss, grad, egrad


def _within(a, e, bound, name):
    inf = np.isinf(e)
    assert np.array_equal(a[inf], e[inf]), name
    assert_within(np.where(inf, 0.0, a), np.where(inf, 0.0, e), np.where(inf | np.isnan(bound), 0.0, bound), name)


def _inputs(n, V, K, dtype, seed, padded=0.2, mass=0.9):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, V, generator=gen, device="cuda") * 3 + torch.randn(n, 1, generator=gen, device="cuda")
    cpu = np.random.default_rng(seed)
    index = torch.from_numpy(np.stack([cpu.permutation(V)[:K] if K <= V else cpu.integers(0, V, K) for _ in range(n)]))
    index = index.cuda()
    t = torch.log_softmax(2 * torch.randn(n, K, generator=gen, device="cuda"), dim=1) + math.log(mass)
    empty = torch.rand(n, K, generator=gen, device="cuda") < padded
    index = torch.where(empty, -1, index)
    t = torch.where(empty, math.nan, t)  # an empty place's value is not looked at
    return x.to(dtype), t, index, torch.rand(n, generator=gen, device="cuda") + 0.5


def _check(x, t, index, g, T=1.0, tail=False, name=""):
    from cign_amd.distill import distill_topk_loss

    xr = x.detach().requires_grad_()
    loss = distill_topk_loss(xr, t, index, temperature=T, tail=tail)
    assert loss.dtype == F32 and loss.shape == x.shape[:-1]
    grad, = torch.autograd.grad(loss, xr, g)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    with torch.no_grad():
        again = distill_topk_loss(x.detach(), t, index, temperature=T, tail=tail)
    assert torch.equal(loss.nan_to_num(nan=7e33), again.nan_to_num(nan=7e33))
    el, bl, eg, bg = _oracle(_n(x), _n(t), index.cpu().numpy(), float(np.float32(T)), tail, _n(g))
    _within(_n(loss), el, bl, f"loss {name}")
    _within(_n(grad), eg, bg + HALF[x.dtype] * (np.abs(eg) + bg) + 2.0 ** -126, f"grad {name}")
    return loss, grad


WIDTHS = [1, 2, 3, 5, 7, 8, 9, 18, 33, 64, 100, 256, 257, 511, 1000, 1025, 2049, 4097, 8200, 16385, 50001]


@pytest.mark.parametrize("V", WIDTHS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [False, True])
def test_loss_and_gradient_match_the_definition(V, dtype, tail):
    n = 23 if V < 5000 else 4
    for K in sorted({1, min(V, 5), min(V, 64), min(V, 128)}):
        print(f"distill V={V} K={K} {dtype} tail={tail}", flush=True)
        x, t, index, g = _inputs(n, V, K, dtype, V + K)
        _check(x, t, index, g, 1.0 if K % 2 else 2.0, tail, f"V={V} K={K}")


@pytest.mark.parametrize("V", [2, 18, 300, 3000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_lists(V, tail):
    """Full lists, lists longer than the classes, a class named twice, empty
    rows, lists at the row's ends, and teacher values of -inf."""
    print(f"lists V={V} tail={tail}", flush=True)
    for dtype in (F32, BF16):
        K = min(V, 128)
        x, t, index, g = _inputs(12, V, K, dtype, V, padded=0.0, mass=1.0)
        _check(x, t, index, g, 1.0, tail, "whole list")
        if V < 128:
            _check(*_inputs(12, V, 128, dtype, V, padded=0.5, mass=0.7), 1.5, tail, "longer than the classes")
        x, t, index, g = _inputs(12, V, 4, dtype, V + 1, mass=0.6) if V >= 4 else _inputs(12, V, 2, dtype, V, mass=0.6)
        index[0] = -1
        index[1] = 0
        t[1] = -1.75
        index[2] = V - 1
        t[2] = math.log(0.2)
        index[3, 0], t[3, 0] = V - 1, -0.5
        index[4, 0], t[4, 0] = 0, -math.inf
        index[5], t[5] = index[5].abs() % V, -math.inf
        _check(x, t, index, g, 1.0, tail, "special rows")
        loss, grad = _check(x, t, index.int().long(), g, 4.0, tail, "special rows, T=4")
        assert loss[0] == 0 and not grad[0].any()


@pytest.mark.parametrize("V", [300, 5000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_repeats_in_long_lists(V, tail):
    """Lists that name one class 128 times, some classes a few times, two places
    one class, and none twice, among classes far apart and next to each other."""
    for dtype in (F32, BF16):
        for K in (64, 65, 128):
            print(f"repeats V={V} K={K} {dtype} tail={tail}", flush=True)
            x, t, index, g = _inputs(12, V, K, dtype, V + K, padded=0.05, mass=0.7)
            empty = index < 0
            index[0] = V - 1
            index[1] = index[1] % 60
            index[2] = index[2] % 2 * (V - 1)
            index[3, -1], index[4, 1], index[5, 63] = index[3, 0], index[4, 0], index[5, K - 1]
            index[6] = torch.arange(K, device="cuda") + 7
            index[7] = torch.arange(K, device="cuda") * (V // K)
            index[8] = torch.arange(K, device="cuda").flip(0) // 2
            # places of one class agree on its probability
            p = torch.zeros(12, V, device="cuda").scatter_(1, index.clamp_min(0), t.nan_to_num(nan=-9.0))
            count = torch.zeros(12, V, device="cuda").scatter_add_(1, index.clamp_min(0), torch.ones_like(t))
            t = (p - count.clamp_min(1).log()).gather(1, index.clamp_min(0)) - 1
            index, t = torch.where(empty, -1, index), torch.where(empty, math.nan, t)
            _check(x, t, index, g, 1.0, tail, f"V={V} K={K}")


@pytest.mark.parametrize("V", [6, 300, 3000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_masked_and_confident_students(V, tail):
    """Masked classes, listed ones among them, rows without a class left,
    masks of the type's lowest value, and students whose mass outside the list
    is 1e-30 or 1e-60 of the whole."""
    print(f"masked V={V} tail={tail}", flush=True)
    for dtype in (F32, BF16):
        x, t, index, g = _inputs(10, V, 4, dtype, V, padded=0.0, mass=0.8)
        x[0] = -math.inf
        x[1, index[1, 2]] = -math.inf
        member = torch.zeros(V, dtype=torch.bool, device="cuda").scatter_(0, index[2], True)
        x[2] = torch.where(member, x[2], -math.inf)
        x[3] = torch.where(torch.zeros_like(member).scatter_(0, index[3], True), x[3] + 70, x[3])
        x[4] = torch.where(torch.zeros_like(member).scatter_(0, index[4], True), x[4] + 140, x[4])
        x[5] = torch.finfo(dtype).min
        x[6] = torch.where(torch.zeros_like(member).scatter_(0, index[6], True), torch.finfo(dtype).min, x[6])
        _check(x, t, index, g, 1.0, tail, f"V={V}")


@pytest.mark.parametrize("V", [40, 3000, 40000])
@pytest.mark.parametrize("tail", [False, True])
def test_rows_far_from_zero(V, tail):
    """As in the log probabilities' tests: large steps, and rows on both sides
    of |x| log2(e) / T = 10^6, the listed classes beyond it or not."""
    for off, step in ((6.5e5, 0.0625), (1e7, 1.0), (-1e9, 64.0)):
        x, t, index, g = _inputs(8, V, 5, F32, V)
        _check(off + (x * 2).round() * step, t, index, g, max(1.0, step), tail, f"offset {off}")
    x, t, index, g = _inputs(8, V, 5, F32, V + 1)
    x = 1e6 / 1.4426950408889634 + x.round()
    x[1] = x[1].scatter(0, index[1].clamp_min(0), x[1].max().item() + 5)
    x[4:] *= -1
    _check(x, t, index, g, 1.0, tail, "at the edge")


@pytest.mark.parametrize("V", [6, 3000, 40000])
def test_bad_rows_stay_in_their_rows(V):
    from cign_amd.distill import distill_topk_loss

    for tail in (False, True):
        x, t, index, g = _inputs(8, V, 3, F32, V, padded=0.0)
        bad, tb, ib = x.clone(), t.clone(), index.clone()
        bad[2, V - 1] = math.nan
        ib[4, 1] = V
        ib[5] = -1
        bad[5] = math.nan  # a row without a listed class: zeros, whatever its logits hold
        tb[6, 0] = math.nan
        ok = [0, 1, 3, 7]
        xr, br = x.requires_grad_(), bad.requires_grad_()
        want, got = distill_topk_loss(xr, t, index, tail=tail), distill_topk_loss(br, tb, ib, tail=tail)
        gw, = torch.autograd.grad(want, xr, g)
        gg, = torch.autograd.grad(got, br, g)
        assert torch.equal(want[ok], got[ok]) and torch.equal(gw[ok], gg[ok])
        assert got[[2, 4, 6]].isnan().all() and gg[[2, 4]].isnan().all()
        assert got[5] == 0 and not gg[5].any()


def test_strides_and_shapes():
    from cign_amd.distill import distill_topk_loss

    gen = torch.Generator(device="cuda").manual_seed(4)
    for dtype in (F32, BF16):
        big = torch.randn(6, 4, 5100, generator=gen, device="cuda").to(dtype)
        for v in (big[:, 1, 3:5004], big[:, :, :4999], big[2, :, 1:8], big[:, :, ::3], big[:, 0, :6].t(),
                  big[0, 0, 7:600], big[:1, 0, :50].expand(7, 50)):
            V = v.shape[-1]
            K = min(V, 6)
            lists = torch.randn(*v.shape[:-1], 2 * K, generator=gen, device="cuda")
            index = torch.randint(0, V, (*v.shape[:-1], 2 * K), generator=gen, device="cuda")
            a = v.detach().clone().contiguous().requires_grad_()
            s = v.detach().requires_grad_()
            la = distill_topk_loss(a, lists[..., ::2].contiguous(), index[..., ::2].contiguous(), 2.0)
            ls = distill_topk_loss(s, lists[..., ::2], index[..., ::2].int(), 2.0)
            assert la.shape == v.shape[:-1] and torch.equal(la, ls)
            assert torch.equal(torch.autograd.grad(la.sum(), a)[0],
                               torch.autograd.grad(ls, s, torch.ones_like(ls))[0])
    e = distill_topk_loss(torch.empty(0, 7, device="cuda").requires_grad_(), torch.empty(0, 2, device="cuda"),
                          torch.empty(0, 2, dtype=torch.int64, device="cuda"))
    assert e.shape == (0,)


def test_shift_of_a_renormalised_list():
    """Teacher logits or log probabilities: the same loss but for the rounding
    of the shift (values near 100 have steps of 2^-17, an error of at most 2^-17
    in each log p and in p; 4 log p terms bounded by |log p - log q| < 30)."""
    from cign_amd.distill import distill_topk_loss

    x, t, index, _ = _inputs(50, 400, 16, F32, 1, padded=0.0)
    a = distill_topk_loss(x, t, index, 2.0)
    b = distill_topk_loss(x, t + 100.0, index, 2.0)
    assert (a - b).abs().max() <= 4 * 2 * 2.0 ** -17 * 30


def test_gradient_against_differences():
    from cign_amd.distill import distill_topk_loss

    step = 1e-5
    for tail in (False, True):
        x, t, index, g = _inputs(4, 19, 5, F32, 3, mass=0.7)
        xr = x.requires_grad_()
        got, = torch.autograd.grad(distill_topk_loss(xr, t, index, 1.5, tail), xr, g)
        a, tn, jn, gn = _n(x), _n(t), index.cpu().numpy(), _n(g)
        num = np.empty_like(a)
        for i in np.ndindex(a.shape):
            v = a[i]
            ends = []
            for d in (step, -step):
                a[i] = v + d
                ends.append((_oracle(a, tn, jn, 1.5, tail, gn)[0] * gn).sum())
            a[i] = v
            num[i] = (ends[0] - ends[1]) / (2 * step)
        assert_within(_n(got), num, 2e-6 + 1e-5 * np.abs(num), "gradient")


def test_more_rows_than_a_grid_dimension():
    """65,600 rows of a slice each: the grid's second dimension ends at 65,535."""
    from cign_amd.distill import distill_topk_loss

    n, V, K = 65600, 4105, 3
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, V, generator=gen, device="cuda", dtype=BF16)
    index = torch.randint(0, V // K, (n, K), generator=gen, device="cuda") * K + torch.arange(K, device="cuda")
    t = torch.log_softmax(torch.randn(n, K, generator=gen, device="cuda"), dim=1) - 0.1
    loss = distill_topk_loss(x, t, index, tail=True)
    for a in (0, 65520, 65580):
        at = slice(a, a + 20)
        el, bl, _, _ = _oracle(_n(x[at]), _n(t[at]), index[at].cpu().numpy(), 1.0, True, np.ones(20))
        _within(_n(loss[at]), el, bl, f"loss from row {a}")


def test_offsets_beyond_32_bits():
    from cign_amd.distill import distill_topk_loss

    V, n = 1 << 16, (1 << 16) + 3
    x = torch.zeros(n, V, dtype=BF16, device="cuda").requires_grad_()
    index = torch.full((n, 2), -1, device="cuda")
    index[n - 1] = torch.tensor([V - 1, 3], device="cuda")
    t = torch.full((n, 2), math.log(0.5), device="cuda")
    loss = distill_topk_loss(x, t, index)
    assert not loss[: n - 1].any() and abs(loss[n - 1].item() - math.log(V / 2)) < 1e-4
    grad, = torch.autograd.grad(loss, x, torch.ones(n, device="cuda"))
    assert grad[n - 1, [3, V - 1]].tolist() == [-0.5, -0.5]
    assert (grad[n - 1, 4:V - 1] > 0).all() and not grad[n - 2].any() and not grad[0].any()


def test_side_stream_graphs_and_determinism():
    from cign_amd.distill import distill_topk_loss

    cases = []
    for n, V, K, dtype, tail in ((500, 18, 5, F32, True), (9, 50001, 64, BF16, True), (3, 40000, 128, F32, False)):
        x, t, index, g = _inputs(n, V, K, dtype, V)
        cases.append((x.requires_grad_(), t, index, g, tail))

    def step():
        out = []
        for x, t, index, g, tail in cases:
            loss = distill_topk_loss(x, t, index, 2.0, tail)
            # detached: no eager graph of the leaves lives on while a step is captured
            out += [loss.detach(), torch.autograd.grad(loss, x, g)[0]]
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    graphs, held = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step())
    for i in range(4):
        with torch.no_grad():
            for x, *_ in cases:
                x.mul_(0.9)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in held[i % 2]]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_refusals():
    from cign_amd.distill import distill_topk_loss

    x = torch.randn(4, 10, device="cuda")
    t = torch.zeros(4, 3, device="cuda")
    j = torch.zeros(4, 3, dtype=torch.int64, device="cuda")
    for bad in (x.double(), x.half(), x.cpu()):
        with pytest.raises(TypeError, match="logits must be CUDA"):
            distill_topk_loss(bad, t, j)
    with pytest.raises(TypeError, match="teacher_logprobs"):
        distill_topk_loss(x, t.double(), j)
    with pytest.raises(TypeError, match="teacher_index"):
        distill_topk_loss(x, t, j.float())
    with pytest.raises(ValueError, match="teacher_index must have shape"):
        distill_topk_loss(x, t, j[:, :2])
    for bad in (t[:3], t[0], torch.zeros(4, 0, device="cuda"), torch.zeros(4, 129, device="cuda"), t[0, 0]):
        with pytest.raises(ValueError, match="teacher_logprobs must be"):
            distill_topk_loss(x, bad, j)
    with pytest.raises(ValueError, match="must be on"):
        distill_topk_loss(x, t.cpu(), j)
    with pytest.raises(ValueError, match="must be on"):
        distill_topk_loss(x, t, j.cpu())
    with pytest.raises(ValueError, match="detach"):
        distill_topk_loss(x, t.requires_grad_(), j)
    with torch.no_grad():
        distill_topk_loss(x, t, j)
    for T in (0.0, -2.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="temperature"):
            distill_topk_loss(x, t.detach(), j, T)
    xr = x.clone().requires_grad_()
    grad, = torch.autograd.grad(distill_topk_loss(xr, t.detach(), j).pow(2).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


def test_operators_together():
    """Norm, teacher's list, student's loss with labels, gradients through the
    norm: the composition equals torch's float64 autograd of the same model
    within the sum of the parts' bounds, a few 1e-6 of each tensor's scale."""
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    gen = torch.Generator(device="cuda").manual_seed(8)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    n, D, V, K, T = 300, 1280, 18, 5, 2.0
    h, w, b, W = rn(n, D), 1 + 0.1 * rn(D), 0.1 * rn(D), rn(V, D) / 36
    labels = torch.where(rn(n) > 0, torch.randint(0, V, (n,), generator=gen, device="cuda"), -100)
    with torch.no_grad():
        teacher = class_logprobs(3 * rn(n, V), top_k=K, temperature=T)
    leaves = [v.requires_grad_() for v in (h, w, b, W)]
    logits = fused_layernorm(h, w, b) @ W.t()
    kl = distill_topk_loss(logits, teacher.top_logprobs, teacher.top_index, T, tail=True)
    r = class_logprobs(logits, labels)
    loss = 0.7 * kl.mean() - 0.3 * r.logprob.sum() / (labels >= 0).sum() - 0.01 * r.entropy.mean()
    got = torch.autograd.grad(loss, leaves)

    ref = [v.detach().double().requires_grad_() for v in leaves]
    z = torch.nn.functional.layer_norm(ref[0], (D,), ref[1], ref[2], 1e-5) @ ref[3].t()
    lq = torch.log_softmax(z / T, 1)
    lp = teacher.top_logprobs.double()
    left = (1 - lp.exp().sum(1)).clamp_min(0)
    lrest = lq.scatter(1, teacher.top_index, -math.inf).logsumexp(1)
    kl64 = T * T * ((lp.exp() * (lp - lq.gather(1, teacher.top_index))).sum(1) + left * (left.log() - lrest))
    l1 = torch.log_softmax(z, 1)
    nll = torch.nn.functional.nll_loss(l1, labels, ignore_index=-100)
    loss64 = 0.7 * kl64.mean() + 0.3 * nll + 0.01 * (l1.exp() * l1).sum(1).mean()
    want = torch.autograd.grad(loss64, ref)
    assert abs(loss.item() - loss64.item()) <= 1e-5 * abs(loss64.item())
    for a, e in zip(got, want):
        assert (a.double() - e).norm() <= 2e-5 * e.norm()


@pytest.mark.parametrize("V", [6, 300, 3000, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unlisted_classes_at_the_lowest_value(V, dtype):
    """A mask of the type's lowest value and a list of the classes that are not
    masked: the others lie further off, in units of log 2, than float32 holds
    for T < log2(e), and the loss is finite."""
    from cign_amd.distill import distill_topk_loss

    for T in (1.0, 0.75, 2.0):
        print(f"lowest outside the list V={V} {dtype} T={T}", flush=True)
        x, t, index, g = _inputs(6, V, 4, dtype, V, padded=0.0, mass=0.8)
        member = torch.zeros(6, V, dtype=torch.bool, device="cuda").scatter_(1, index, True)
        x = torch.where(member, x, torch.finfo(dtype).min)
        x[1, int((~member[1]).nonzero()[-1])] = 0.5  # one class outside the list is not masked
        x[2, index[2, 0]] = torch.finfo(dtype).min  # a masked class in the list
        xr = x.requires_grad_()
        loss = distill_topk_loss(xr, t, index, T, tail=True)
        grad, = torch.autograd.grad(loss, xr, g)
        el, bl, _, bg = _oracle(_n(x), _n(t), index.cpu().numpy(), T, True, _n(g))
        # T^2 times 3e38 may pass float32's largest value: infinity is its rounding
        el = np.where(el > np.finfo(np.float32).max, np.inf, el)
        _within(_n(loss), el, bl, f"loss V={V} T={T}")
        # the oracle's share of a class outside the list is exp(log q - log q_rest), where 3e38 hides log 2:
        # here the softmax of the classes outside the list
        z, p = x.detach().double() / T, t.double().exp()
        mass = torch.zeros_like(z).scatter_(1, index, p)
        left = 1 - p.sum(1, keepdim=True)
        eg = g.double()[:, None] * T * (torch.softmax(z, 1) - mass - left * torch.softmax(
            z.masked_fill(member, -math.inf), 1))
        eg = _n(eg)
        _within(_n(grad), eg, bg + HALF[dtype] * (np.abs(eg) + bg) + 2.0 ** -126, f"grad V={V} T={T}")
        assert loss[[0, 1, 3, 4, 5]].isfinite().all()


@pytest.mark.parametrize("V", [6, 100, 300, 40000])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_renormalised_lists_far_from_zero(V, dtype):
    """Any constant may be added to a row of the teacher's values: rows at the
    type's lowest value and others so large that log K is below their step."""
    for K in {4, min(V, 100)}:
        print(f"far lists V={V} K={K} {dtype}", flush=True)
        x, t, index, g = _inputs(8, V, K, dtype, V + K)
        present = index >= 0
        place = torch.arange(K, device="cuda")
        rows = (torch.full((K,), torch.finfo(F32).min, device="cuda"), torch.full((K,), -1e30, device="cuda"),
                torch.full((K,), 1e18, device="cuda"), torch.full((K,), 3e38, device="cuda"),
                torch.where(place % 2 == 0, -3.4e38, -3.0e38), torch.where(place % 2 == 0, 2.0 ** 60, -math.inf))
        for r, v in enumerate(rows):
            t[r] = torch.where(present[r], v.to(F32), math.nan)
        _check(x, t, index, g, 1.0, False, f"V={V} K={K}")


def _whole(V, n=3):
    return torch.full((n, V), 0.75, device="cuda")


@pytest.mark.parametrize("V", [3, 37, 100, 129, 300, 1000, 1025, 5001, 20011, 50001])
def test_logarithms_of_the_sums(V):
    """Classes that are all equal: every sum is a whole number, exact in
    float32, so what is left is the logarithms' error, each at most 2^-24 (of
    log s, however large), and the result's half step. The teacher's own
    float32 values are what the definition takes; its masses agree with it to
    1e-12, or to 2^-22 of themselves where they are renormalised."""
    for K in sorted({1, min(V, 5), min(V, 100), min(V, 128)}):
        index = torch.arange(K, device="cuda").mul(max(1, V // K)).expand(3, K).contiguous()
        t = torch.full((3, K), -math.log(V), device="cuda")
        from cign_amd.distill import distill_topk_loss

        p, t0 = math.exp(t[0, 0].item()), t[0, 0].item()
        left = 0.0 if K == V else 1.0 - K * p
        want = K * p * (t0 + math.log(V)) + (left * (math.log(left) - math.log((V - K) / V)) if left else 0.0)
        got = distill_topk_loss(_whole(V), t, index, tail=True)
        assert (got.double() - want).abs().max() <= 2 * U * K * p + 4 * U * left + U * abs(want), (V, K)
        want = math.log(V) - math.log(K)
        got = distill_topk_loss(_whole(V), t, index)
        half = float(np.spacing(np.float32(max(want, 1.0)))) / 2
        assert (got.double() - want).abs().max() <= 2 * U + half + 2.0 ** -22 * want, (V, K)


@pytest.mark.parametrize("V", [5, 100, 300, 40000])
def test_a_class_named_twice_counts_place_by_place(V):
    """Sum over places of p_i (log p_i - log q of its class): below the KL of
    the joined masses by sum p_i log(mass of the class / p_i), a constant of the
    logits, so the gradient is that of the joined masses."""
    from cign_amd.distill import distill_topk_loss

    x = torch.zeros(3, V, device="cuda")
    x[:, 2] = 60.0  # sure of the class, up to e^-60
    index = torch.full((3, 2), 2, device="cuda")
    t = torch.log(torch.tensor([[0.5, 0.5], [0.25, 0.75], [0.125, 0.25]], device="cuda"))
    loss = distill_topk_loss(x, t, index, temperature=2.0)
    p = torch.tensor([[0.5, 0.5], [0.25, 0.75], [1 / 3, 2 / 3]], dtype=torch.float64, device="cuda")
    lq = torch.log_softmax(x.double() / 2, 1)[:, 2]
    want = 4 * ((p * p.log()).sum(1) - lq)
    assert (loss.double() - want).abs().max() <= 4 * 2.0 ** -22
    one, joined = (v.clone().requires_grad_() for v in (x, x))
    g = torch.ones(3, device="cuda")
    a, = torch.autograd.grad(distill_topk_loss(one, t, index, 2.0, tail=True), one, g)
    b, = torch.autograd.grad(distill_topk_loss(joined, t.exp().sum(1, keepdim=True).log(), index[:, :1], 2.0, tail=True),
                             joined, g)
    # the masses agree to 2^-22 of themselves; 2 is the temperature
    assert (a.double() - b.double()).abs().max() <= 2 * 2 * 2.0 ** -22


def test_zero_rows():
    from cign_amd.distill import distill_topk_loss

    for V in (7, 300, 40000):
        x = torch.empty(0, V, device="cuda").requires_grad_()
        loss = distill_topk_loss(x, torch.empty(0, 2, device="cuda"), torch.empty(0, 2, dtype=torch.int64, device="cuda"))
        grad, = torch.autograd.grad(loss, x, torch.empty(0, device="cuda"))
        assert loss.shape == (0,) and grad.shape == x.shape
        assert torch.autograd.grad(distill_topk_loss(x, torch.empty(0, 2, device="cuda"), torch.empty(
            0, 2, dtype=torch.int32, device="cuda"), tail=True).sum(), x)[0].shape == x.shape
