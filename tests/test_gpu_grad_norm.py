"""GPU: global_grad_norm and clip_grad_norm against float64.

Squares and sums are float64 (relative error below 1e-9 for these counts), the
norm is rounded once: within 2^-24 of itself, 2^-23 asserted. A clipped value is a
product with a float32 factor: two roundings of 2^-24 for float32, 2^-8 and
2^-23 for bf16, and half of the smallest subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _grads(sizes, types, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=gen, device="cuda") * scale * (1 + i % 5)).to(t)
            for i, (s, t) in enumerate(zip(sizes, types))]


def _norm(grads):
    return math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def _factor(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))


def _check(grads, max_norm):
    from cign_amd.grad_norm import clip_grad_norm, global_grad_norm

    want = _norm(grads)
    norm = global_grad_norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(float(norm) - want) <= 2 * U * want
    by = _factor(want, max_norm)
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, float("nan")) for g in grads]
    n2 = clip_grad_norm(grads, max_norm, out=out)
    assert torch.equal(n2, norm)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))  # read only
    version = [g._version for g in grads]
    n3 = clip_grad_norm(grads, max_norm)
    assert torch.equal(n3, norm) and all(g._version > v for g, v in zip(grads, version))
    for g, o, b in zip(grads, out, before):
        assert torch.equal(g, o)
        ref = b.double() * by
        half = 2 * U if g.dtype == torch.float32 else 2.0 ** -8 + 2 * U
        tiny = 2.0 ** -149 if g.dtype == torch.float32 else 2.0 ** -133
        assert bool(((g.double() - ref).abs() <= half * 1.01 * ref.abs() + tiny).all())
    return norm


F, B = torch.float32, torch.bfloat16


@pytest.mark.parametrize("size", [1, 2, 7, 8, 9, 255, 2047, 2048, 8191, 8192, 8193, 16385, 100003])
@pytest.mark.parametrize("dtype", [F, B])
def test_one_tensor(size, dtype):
    _check(_grads([size], [dtype]), 0.5)
    _check(_grads([size], [dtype]), 1e6)


@pytest.mark.parametrize("count", [2, 127, 128, 129, 300])
def test_many_tensors(count):
    sizes = [(i * 7919) % 5003 for i in range(count)]  # one of them empty
    assert 0 in sizes
    _check(_grads(sizes, [F if i % 3 else B for i in range(count)]), 1.0)


def test_large_tensors():
    _check(_grads([30_000_001, 5, 12_345_678], [B, F, F]), 2.0)


def test_values_past_float32_squares():
    """Squares of 1e25 and 1e-30 lie outside float32; float64 holds them."""
    from cign_amd.grad_norm import global_grad_norm

    for scale in (1e25, 1e-30):
        g = _grads([5000], [F], scale=scale)
        want = _norm(g)
        assert abs(float(global_grad_norm(g)) - want) <= 2 * U * want
    _check(_grads([5000, 300], [F, B], scale=1e25), 1.0)


def test_shapes_and_strides():
    from cign_amd.grad_norm import clip_grad_norm, global_grad_norm

    gen = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(64, 90, generator=gen, device="cuda")
    grads = [base.clone().t(), base.clone()[:, 3:50], base.clone()[::2], torch.randn((), generator=gen, device="cuda"),
             torch.randn(4, 0, device="cuda"), torch.randn(3, 4, 5, generator=gen, device="cuda").permute(2, 0, 1)]
    want, before = _norm(grads), [g.clone() for g in grads]
    rest = [g._base.clone() if g._base is not None else None for g in grads]
    assert abs(float(global_grad_norm(grads)) - want) <= 2 * U * want
    clip_grad_norm(grads, 0.25)
    for g, b in zip(grads, before):
        assert bool(((g.double() - b.double() * (0.25 / (want + 1e-6))).abs() <= 2.1 * U * b.abs()).all())
    assert torch.equal(grads[1]._base[:, :3], rest[1][:, :3]) and torch.equal(grads[2]._base[1::2], rest[2][1::2])
    out = [torch.empty(g.shape, device="cuda").t().contiguous().t() if g.dim() == 2 else torch.empty_like(g) for g in grads]
    clip_grad_norm(before, 0.25, out=out)
    assert all(torch.equal(o, g) for o, g in zip(out, grads))
    one = torch.ones(1, device="cuda").expand(1000)  # a broadcast gradient
    assert abs(float(global_grad_norm([one])) - math.sqrt(1000)) <= 2 * U * 32
    out = [torch.empty(1000, device="cuda")]
    clip_grad_norm([one], 1.0, out=out)
    assert out[0].unique().numel() == 1 and abs(float(out[0][0]) - 1 / math.sqrt(1000)) <= 1e-8
    flat = torch.zeros(1 + 7 + 9, device="cuda")  # outputs side by side in one buffer, at odd places
    a, b = torch.randn(7, generator=gen, device="cuda"), torch.randn(9, generator=gen, device="cuda")
    clip_grad_norm([a, b], 0.1, out=[flat[1:8], flat[8:]])
    assert flat[0] == 0 and torch.equal(flat[1:8] > 0, a > 0) and torch.equal(flat[8:] > 0, b > 0)


def test_norms_that_are_not_finite():
    from cign_amd.grad_norm import clip_grad_norm

    g = _grads([100, 50], [F, B])
    g[0][3] = float("nan")
    assert clip_grad_norm(g, 1.0).isnan() and all(t.isnan().all() for t in g)
    g = _grads([100, 50], [F, B])
    g[1][3] = float("inf")
    assert clip_grad_norm(g, 1.0).isinf() and g[1][3].isnan() and not g[0].any() and int(g[1].isnan().sum()) == 1
    g = _grads([100], [F])
    before = g[0].clone()
    clip_grad_norm(g, float("inf"))
    assert torch.equal(g[0], before)
    clip_grad_norm(g, 0.0)
    assert not g[0].any()
    z = [torch.zeros(10, device="cuda")]
    assert float(clip_grad_norm(z, 1.0)) == 0.0 and not z[0].any()
    e = [torch.empty(0, device="cuda")]
    assert float(clip_grad_norm(e, 1.0)) == 0.0


def test_as_torch_clips():
    """torch's clip_grad_norm_ on the same gradients: its float32 norm is within
    1e-5 of ours for 30,000 values, and so are the factors."""
    from cign_amd.grad_norm import clip_grad_norm

    sizes = [10000, 1, 20000]
    a, b = _grads(sizes, [F] * 3), _grads(sizes, [F] * 3)
    params = [torch.nn.Parameter(torch.zeros_like(t)) for t in b]
    for p, t in zip(params, b):
        p.grad = t
    n1, n2 = clip_grad_norm(a, 3.0), torch.nn.utils.clip_grad_norm_(params, 3.0)
    assert abs(float(n1) - float(n2)) <= 1e-5 * float(n2)
    assert all((x - y).abs().max() <= 2e-5 * y.abs().max() for x, y in zip(a, b))


def test_streams_and_graphs():
    from cign_amd.grad_norm import clip_grad_norm

    sets = [_grads([5000 + k, 70001, 3], [F, B, F], seed=k) for k in range(2)]
    outs = [[torch.empty_like(g) for g in s] for s in sets]
    want = []
    for s, o in zip(sets, outs):
        n = clip_grad_norm(s, 1.0, out=o)
        want.append([n.clone(), *[t.clone() for t in o]])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    norms = []
    for s, o, st in zip(sets, outs, streams):
        with torch.cuda.stream(st):
            for t in o:
                t.zero_()
            norms.append(clip_grad_norm(s, 1.0, out=o))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for n, o, w in zip(norms, outs, want) for p, q in zip([n, *o], w))
    graphs, held = [], []
    for s, o in zip(sets, outs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(clip_grad_norm(s, 1.0, out=o))
    for i in range(3):
        for s in sets:
            for t in s:
                t.mul_(0.75)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, o, h in zip(sets, outs, held):
            fresh = [torch.empty_like(t) for t in s]
            n = clip_grad_norm(s, 1.0, out=fresh)
            assert torch.equal(n, h) and all(torch.equal(p, q) for p, q in zip(o, fresh)), i


def test_refusals():
    from cign_amd.grad_norm import clip_grad_norm, global_grad_norm

    g = torch.ones(20, device="cuda")
    for grads, kw, err in (([], {}, ValueError), ([g, None], {}, TypeError), ([g.double()], {}, TypeError),
                           ([g.cpu()], {}, TypeError), ([g.half()], {}, TypeError), ([g, g], {}, ValueError),
                           ([g[:12], g[8:]], {}, ValueError), ([g], dict(max_norm=-1.0), ValueError),
                           ([g], dict(max_norm=float("nan")), ValueError), ([g], dict(out=[]), ValueError),
                           ([g], dict(out=[g[:5]]), ValueError), ([g], dict(out=[g.bfloat16()]), TypeError),
                           ([g], dict(out=[g, g]), ValueError), ([g[:10]], dict(out=[g[5:15]]), ValueError),
                           ([g[:5], g[5:10]], dict(out=[g[10:15], g[:5]]), ValueError),
                           ([g[:1].expand(20)], {}, ValueError)):
        with pytest.raises(err):
            clip_grad_norm(grads, **(dict(max_norm=1.0) | kw))
    assert float(g.sum()) == 20.0
    assert abs(float(global_grad_norm([g, g])) - math.sqrt(40)) <= 1e-6  # read only: the same tensor twice counts twice
    r = torch.ones(3, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no_grad"):
        clip_grad_norm([r], 1.0)
    with torch.no_grad():
        clip_grad_norm([r], 1.0)
    assert not global_grad_norm([r]).requires_grad
    assert torch.equal(clip_grad_norm(g, 100.0), global_grad_norm(g))  # one tensor without a list
