"""GPU: linear_cross_entropy against the definition in float64.

Tolerances, u = 2^-24. A logit is a float32 sum of D products: for bf16 the products
are exact and 32 enter a matrix instruction, whose inner roundings are taken as one
for every four, so at most D / 4 + 32 roundings of the sum of absolute terms; for
float32 six such products of 8-bit parts, the larger ones D / 4 roundings each and
2^-22 for the parts left out: (D / 2 + 96) u. Call it dz. Then
  logsumexp, loss: 2 max dz of the row, 300 u for the sum of exponentials (32 values
  a lane, joins, exponentials to 2 u |difference|, differences weighed by p <= 1 and
  |d| e^d <= 1), 4 u of the values;
  p: relative 2 dz + (|z - lse| + 8) 2 u; a logit's gradient g p - g [label]: that
  of p, 2 u of both terms, and for bf16 its rounding, 2^-8 of itself;
  grad_x, grad_weight: those errors through the products (in absolute values), the
  sum's own (terms / 4 + 96) u of its absolute terms, the result's rounding;
  grad_bias: the same with ones (summed before the gradient's rounding).
The roundings to bf16 are independent of each other, so a product's error has at
most 2^-8 of the root of its squared terms as its root mean square: the norm of the
whole error is held to twice that and the result's own 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F, B = torch.float32, torch.bfloat16
HALF = {F: U, B: 2.0 ** -8}


def _inputs(n, D, V, dtype, bias=True, seed=0, ignored=0.2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w = rn(n, D).to(dtype), (rn(V, D) * (2 / math.sqrt(D))).to(dtype)
    b = rn(V).to(dtype) if bias else None
    labels = torch.randint(0, V, (n,), generator=gen, device="cuda")
    labels[torch.rand(n, generator=gen, device="cuda") < ignored] = -100
    return x, w, labels, b, torch.rand(n, generator=gen, device="cuda") + 0.5, 0.1 * rn(n)


def _bounds(x, w, labels, b, gl, gs, dtype):
    """Values in float64 and their tolerances."""
    X, W = x.double(), w.double()
    D, V, n = X.shape[1], W.shape[0], X.shape[0]
    z = X @ W.t() + (0 if b is None else b.double())
    masked = z == -math.inf
    dz = (D / 4 + 32 if dtype == B else D / 2 + 96) * U * (X.abs() @ W.abs().t()) + 2 * U * z.abs().masked_fill(masked, 0)
    dz = dz.masked_fill(masked, 0)
    lse = torch.logsumexp(z, 1)
    valid = labels >= 0
    at = labels.clamp_min(0)[:, None]
    loss = torch.where(valid, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    top = dz.amax(1)
    tol_lse = 2 * top + 300 * U + 4 * U * lse.abs()
    tol_loss = torch.where(valid, tol_lse + top + 4 * U * z.gather(1, at)[:, 0].abs(), 0)
    out = dict(loss=(loss, tol_loss), lse=(lse, tol_lse))
    p = (z - lse[:, None]).exp()
    g = torch.where(valid, gl.double(), 0) if gl is not None else torch.zeros_like(lse)
    s = gs.double() if gs is not None else torch.zeros_like(lse)
    hot = torch.zeros_like(z).scatter_(1, at, g[:, None])
    d = (g + s)[:, None] * p - hot
    away = (z - lse[:, None]).abs().masked_fill(masked, 0)
    base = (g + s).abs()[:, None] * p * (2 * top[:, None] + 2 * dz + (away + 8) * 2 * U) + 2 * U * hot.abs()
    base = base + 2 * U * ((g.abs() + s.abs())[:, None] * p)
    e = base + (HALF[B] * d.abs() if dtype == B else 2 * U * d.abs())
    sum_u = lambda k: (k / 4 + 96) * U * (1 if dtype == B else 2)
    clean = torch.where(masked.all(0)[:, None], torch.zeros_like(W), W)
    out["x"] = (d @ clean, e @ clean.abs() + sum_u(V) * (d.abs() @ clean.abs()))
    out["weight"] = (d.t() @ X, e.t() @ X.abs() + sum_u(n) * (d.abs().t() @ X.abs()))
    out["bias"] = (d.sum(0), base.sum(0) + sum_u(n) * d.abs().sum(0))
    rms = {"x": (d.square() @ clean.square()).sum(), "weight": (d.square().t() @ X.square()).sum()}
    return out, rms


def _check(x, w, labels, b, gl, gs, want=None):
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    dtype = x.dtype
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()] + ([] if b is None else [b.detach().requires_grad_()])
    r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2] if b is not None else None)
    outs, ups = zip(*[(o, g) for o, g in ((r.loss, gl), (r.logsumexp, gs)) if g is not None])
    got = dict(zip(("x", "weight", "bias"), torch.autograd.grad(outs, leaves, ups)))
    ref, rms = _bounds(x, w, labels, b, gl, gs, dtype)
    for name, v in (("loss", r.loss), ("lse", r.logsumexp), *got.items()):
        val, tol = ref[name]
        err = (v.double() - val).abs()
        tol = tol + HALF[v.dtype] * val.abs() + 1e-37
        assert v.shape == val.shape and bool((err <= tol).all()), (name, float((err / tol).max()))
        if dtype == B and name in rms:
            most = HALF[B] * (2 * math.sqrt(float(rms[name])) + float(val.norm())) + float((ref[name][1] * U / HALF[B]).norm())
            assert float((v.double() - val).norm()) <= most, name
    for g, t in zip(got.values(), leaves):
        assert g.dtype == t.dtype
    with torch.no_grad():
        q = linear_cross_entropy(x, w, labels, bias=b)
    assert torch.equal(q.loss, r.loss) and torch.equal(q.logsumexp, r.logsumexp)
    return r, got


SHAPES = [(1, 1, 1), (1, 64, 300), (3, 7, 2), (16, 33, 257), (17, 128, 1000), (33, 100, 70), (64, 64, 4097),
          (65, 64, 255), (130, 65, 511), (255, 192, 256), (257, 1, 600), (300, 1001, 777), (513, 320, 2049),
          (1000, 64, 33), (66, 32, 65), (100, 96, 1000), (128, 160, 4100), (129, 96, 700),
          (1, 1024, 300), (40, 2048, 129), (200, 1024, 200), (70, 1056, 1100), (150, 288, 5000), (2000, 64, 5)]


@pytest.mark.parametrize("n,D,V", SHAPES)
@pytest.mark.parametrize("dtype", [F, B])
def test_shapes(n, D, V, dtype):
    k = SHAPES.index((n, D, V))
    x, w, labels, b, gl, gs = _inputs(n, D, V, dtype, bias=k % 2 == 0, seed=k)
    _check(x, w, labels, b, gl, gs if k % 3 else None)


@pytest.mark.parametrize("dtype", [F, B])
def test_pieces_of_the_vocabulary(dtype):
    """Rows so many that the classes come in several pieces, the last one shorter."""
    x, w, labels, b, gl, _ = _inputs(9000, 40, 16000, dtype, seed=5)
    _check(x, w, labels, b, gl, None)


@pytest.mark.parametrize("dtype", [F, B])
def test_long_sums_in_slots(dtype):
    """Few rows over many classes: the rows' gradient is cut along the classes."""
    x, w, labels, b, gl, gs = _inputs(90, 200, 30011, dtype, seed=6)
    _check(x, w, labels, b, gl, gs)


@pytest.mark.parametrize("dtype", [F, B])
def test_gradients_alone(dtype):
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, gs = _inputs(200, 70, 900, dtype, seed=2)
    _check(x, w, labels, b, gl, None)
    _check(x, w, labels, b, None, gs)
    every = None
    for pick in (7, 1, 2, 4, 3, 5, 6):
        leaves = [t.detach().requires_grad_(bool(pick >> i & 1)) for i, t in enumerate((x, w, b))]
        r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
        got = iter(torch.autograd.grad([r.loss, r.logsumexp], [t for t in leaves if t.requires_grad], [gl, gs]))
        if pick == 7:
            every = list(got)
        else:
            assert all(torch.equal(next(got), every[i]) for i in range(3) if pick >> i & 1), pick


def test_bias_types_and_label_types():
    x, w, labels, b, gl, gs = _inputs(100, 64, 500, B, seed=3)
    _check(x, w, labels, b.float(), gl, gs)
    _check(x, w, labels.int(), b, gl, gs)


@pytest.mark.parametrize("n", [20, 150])
@pytest.mark.parametrize("dtype", [F, B])
def test_masks(n, dtype):
    """Masked classes, with NaN in their weights; ignored rows, with NaN; a row count
    of one left; no row left; no class left."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, gs = _inputs(n, 96, 700, dtype, seed=4)
    b[100:400] = -math.inf
    labels[(labels >= 100) & (labels < 400)] = 5
    ref, _ = _bounds(x, w, labels, b, gl, None, dtype)
    _, clean = _check(x, w, labels, b, gl, None)
    w2, x2 = w.clone(), x.clone()
    w2[100:400] = math.nan
    x2[labels < 0] = math.nan
    leaves = [t.detach().requires_grad_() for t in (x2, w2, b)]
    r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
    got = torch.autograd.grad(r.loss, leaves, gl)
    assert all(torch.equal(p, q) for p, q in zip(got, clean.values()))
    assert not got[1][100:400].any() and not got[2][100:400].any() and not got[0][labels < 0].any()
    assert torch.equal(r.loss[labels < 0], torch.zeros_like(r.loss[labels < 0]))
    for keep in (0, 1):  # rows that take part
        few = torch.full_like(labels, -100)
        few[:keep] = 7
        _check(x, w, few, b, gl, None)
    none = torch.full_like(b, -math.inf).requires_grad_()
    few = torch.full_like(labels, 3)
    few[0] = -100
    r = linear_cross_entropy(leaves[0].detach().nan_to_num().requires_grad_(), leaves[1], few, bias=none)
    assert bool((r.logsumexp == -math.inf).all()) and r.loss[0] == 0 and bool((r.loss[1:] == math.inf).all())
    assert not torch.autograd.grad(r.loss, leaves[1], gl)[0].any()
    masked = torch.full_like(labels, 200)  # a masked label: the loss is infinite, the others' gradient is not
    q = [t.detach().requires_grad_() for t in (x, w, b)]
    r = linear_cross_entropy(q[0], q[1], masked, bias=q[2])
    assert bool((r.loss == math.inf).all()) and all(g.isfinite().all() for g in torch.autograd.grad(r.loss, q, gl))


@pytest.mark.parametrize("dtype", [F, B])
@pytest.mark.parametrize("n,D,V", [(3000, 700, 5000), (2100, 1984, 2500)])
def test_turned_operands_at_odd_edges(n, D, V, dtype):
    """Products along the rows and along the classes whose last lines and columns end inside a tile."""
    x, w, labels, b, gl, gs = _inputs(n, D, V, dtype, bias=D == 700, seed=12)
    _check(x, w, labels, b, gl, gs)


def test_masked_classes_that_are_read_where_they_lie():
    """bfloat16 rows of a multiple of 64 values, in a wider storage of NaN; the masked classes NaN too, the last ones
    among them. The weight's gradient alone reads them where they lie, the rows' packs them."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, _ = _inputs(300, 128, 1000, B, seed=13)
    off = torch.zeros(1000, dtype=torch.bool, device="cuda")
    off[64:130] = off[700:] = True
    b[off] = -math.inf
    labels[(labels >= 64) & (labels < 130) | (labels >= 700)] = 5
    _, clean = _check(x, w, labels, b, gl, None)
    wide = torch.full((1000, 192), math.nan, dtype=B, device="cuda")
    wide[:, :128] = w
    wide[off] = math.nan
    for pick in (1, 2, 3):
        xs, ws = x.detach().requires_grad_(bool(pick & 1)), wide[:, :128].detach().requires_grad_(bool(pick & 2))
        r = linear_cross_entropy(xs, ws, labels, bias=b)
        got = torch.autograd.grad(r.loss, [t for t in (xs, ws) if t.requires_grad], gl)
        for g, name in zip(got, ("x",) * (pick & 1) + ("weight",)):
            assert torch.equal(g, clean[name])


@pytest.mark.parametrize("n", [10, 200])
def test_labels_out_of_range_and_nonfinite_rows(n):
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, _ = _inputs(n, 40, 300, F, seed=8, ignored=0.0)
    clean = linear_cross_entropy(x, w, labels, bias=b)
    labels2, x2 = labels.clone(), x.clone()
    labels2[1], labels2[2], labels2[3] = 300, -1, 1 << 40
    x2[5, 3] = math.inf
    x2[6, 0] = math.nan
    q = x2.requires_grad_()
    r = linear_cross_entropy(q, w, labels2, bias=b)
    keep = [i for i in range(n) if i not in (1, 2, 3, 5, 6)]
    assert torch.equal(r.loss[keep], clean.loss[keep]) and torch.equal(r.logsumexp[keep], clean.logsumexp[keep])
    assert r.loss[[1, 2, 3, 5, 6]].isnan().all() and torch.equal(r.logsumexp[[1, 2, 3]], clean.logsumexp[[1, 2, 3]])
    gx, = torch.autograd.grad(r.loss, q, gl)
    assert gx[[1, 2, 3, 5, 6]].isnan().all() and gx[keep].isfinite().all()


@pytest.mark.parametrize("n", [30, 180])
@pytest.mark.parametrize("dtype", [F, B])
def test_masks_of_the_lowest_value(n, dtype):
    """Biases of the type's lowest value: of some classes, which then have no part in anything; of all of them, whose
    logits are that value (a step of it is 2e31), so that logsumexp is too and the loss log 500."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, gs = _inputs(n, 64, 500, dtype, seed=14, ignored=0.0)
    low = torch.finfo(dtype).min
    labels = labels % 100
    b[200:350] = low
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
    got = torch.autograd.grad((r.loss, r.logsumexp), leaves, (gl, gs))
    assert not got[1][200:350].any() and not got[2][200:350].any()
    b2 = b.clone()
    b2[200:350] = -math.inf
    others = [t.detach().requires_grad_() for t in (x, w, b2)]
    q = linear_cross_entropy(others[0], others[1], labels, bias=others[2])
    assert torch.equal(q.loss, r.loss) and torch.equal(q.logsumexp, r.logsumexp)
    assert all(torch.equal(s, t) for s, t in zip(got, torch.autograd.grad((q.loss, q.logsumexp), others, (gl, gs))))
    r = linear_cross_entropy(x, w, labels, bias=torch.full_like(b, low))
    assert bool((r.logsumexp == low).all()) and bool(((r.loss - math.log(500)).abs() <= 4 * U * math.log(500)).all())


def test_launches_beyond_32_bits_of_threads():
    """Rows so many that a launch of all their tiles, or of a thread for each eight of their values, would pass 2^32
    threads: 2^23 rows against 70,000 classes, read where they lie; 2^23 rows of 2050 values, one row throughout, packed."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    n = 1 << 23
    gen = torch.Generator(device="cuda").manual_seed(15)
    x = torch.randn(n, 64, generator=gen, device="cuda", dtype=B)
    w = torch.randn(70000, 64, generator=gen, device="cuda", dtype=B)
    labels = torch.randint(0, 70000, (n,), generator=gen, device="cuda")
    with torch.no_grad():
        r = linear_cross_entropy(x, w, labels)
    some = torch.cat([torch.randint(0, n, (300,), generator=gen, device="cuda"), torch.arange(n - 3, n, device="cuda")])
    ref, _ = _bounds(x[some], w, labels[some], None, None, None, B)
    for name, v in (("loss", r.loss[some]), ("lse", r.logsumexp[some])):
        val, tol = ref[name]
        assert bool(((v.double() - val).abs() <= tol + U * val.abs()).all()), name
    assert bool(r.loss.isfinite().all())
    del x, w, r, ref
    row, w = torch.randn(1, 2050, generator=gen, device="cuda", dtype=B), torch.randn(2, 2050, generator=gen, device="cuda", dtype=B)
    with torch.no_grad():
        few = linear_cross_entropy(row.expand(200, 2050), w, labels[:200] % 2)
        r = linear_cross_entropy(row.expand(n, 2050), w, labels % 2)
    assert bool((r.logsumexp == few.logsumexp[0]).all())
    one = (labels % 2).bool()
    ref = [linear_cross_entropy(row.expand(200, 2050), w, torch.full((200,), k, device="cuda")).loss[0] for k in (0, 1)]
    assert bool((r.loss == torch.where(one, ref[1], ref[0])).all())


def test_large_logits():
    """Differences of a thousand: one class has all the mass, others none."""
    x, w, labels, b, gl, gs = _inputs(150, 64, 400, F, seed=9)
    _check(x * 30, w * 10, labels, b, gl, gs)
    _check(x * 1e-3, w, labels, None, gl, None)


def test_float32_beyond_bf16():
    """Values that differ in their last bits only: the parts hold all 24."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x = torch.full((100, 64), 1.0, device="cuda")
    w = (1.0 + torch.arange(300, device="cuda")[:, None] * 2.0 ** -23).expand(300, 64).contiguous()
    r = linear_cross_entropy(x, w, torch.arange(100, device="cuda"))
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1) - z[torch.arange(100), torch.arange(100)]
    assert (r.loss.double() - want).abs().max() <= 64 * 2 * 128 * U + 300 * U
    d = r.loss[0].double() - r.loss[99].double()  # 99 steps of 64 * 2^-23
    assert abs(float(d) - 99 * 64 * 2.0 ** -23) <= 64 * 8 * U + 8 * U * 70


@pytest.mark.parametrize("dtype", [F, B])
def test_strides_and_shapes(dtype):
    from cign_amd.linear_cross_entropy import linear_cross_entropy as op

    x, w, labels, b, gl, _ = _inputs(120, 128, 400, dtype, seed=10)
    wide_x, wide_w = torch.zeros(120, 200, device="cuda", dtype=dtype), torch.zeros(400, 136, device="cuda", dtype=dtype)
    for ox, ow in ((0, 0), (8, 8), (3, 5)):
        vx, vw = wide_x[:, ox: ox + 128], wide_w[:, ow: ow + 128]
        vx.copy_(x)
        vw.copy_(w)
        p, q = vx.detach().requires_grad_(), vw.detach().requires_grad_()
        r = op(p, q, labels, bias=b)
        want = op(x, w, labels, bias=b)
        assert torch.equal(r.loss, want.loss) and torch.equal(r.logsumexp, want.logsumexp)
        g = torch.autograd.grad(r.loss, [p, q], gl)
        a, c = x.detach().requires_grad_(), w.detach().requires_grad_()
        assert all(torch.equal(s, t) for s, t in zip(g, torch.autograd.grad(op(a, c, labels, bias=b).loss, [a, c], gl)))
    r = op(x.view(4, 30, 128), w, labels.view(4, 30))
    assert r.loss.shape == (4, 30)
    t = op(x, w.t().contiguous().t(), labels)
    assert torch.equal(t.loss, r.loss.view(-1))
    one = op(x[0], w, labels[0])
    assert one.loss.shape == () and abs(float(one.loss) - float(r.loss.view(-1)[0])) <= 1e-4
    same = op(x[:1].expand(120, 128), w, labels)
    assert torch.equal(same.logsumexp, same.logsumexp[:1].expand(120))


def test_empty():
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w = torch.zeros(0, 64, device="cuda").requires_grad_(), torch.ones(50, 64, device="cuda").requires_grad_()
    b = torch.ones(50, device="cuda").requires_grad_()
    r = linear_cross_entropy(x, w, torch.zeros(0, dtype=torch.int64, device="cuda"), bias=b)
    assert r.loss.shape == r.logsumexp.shape == (0,)
    gx, gw, gb = torch.autograd.grad(r.loss.sum(), [x, w, b])
    assert gx.shape == (0, 64) and gw.shape == (50, 64) and not gw.any() and not gb.any()


def test_gradient_against_differences():
    """Central differences of the float64 loss along random directions."""
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, gs = _inputs(70, 24, 90, F, seed=11)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
    grads = torch.autograd.grad([r.loss, r.logsumexp], leaves, [gl, gs])

    def value(x, w, b):
        z = x @ w.t() + b
        lse = torch.logsumexp(z, 1)
        loss = torch.where(labels >= 0, lse - z.gather(1, labels.clamp_min(0)[:, None])[:, 0], 0)
        return (loss * gl.double()).sum() + (lse * gs.double()).sum()

    gen = torch.Generator(device="cuda").manual_seed(1)
    base = [t.double() for t in (x, w, b)]
    for i in range(3):
        d = torch.randn(base[i].shape, generator=gen, device="cuda").double()
        at = lambda t: value(*[v + (t * d if j == i else 0) for j, v in enumerate(base)])
        slope = (at(1e-6) - at(-1e-6)) / 2e-6
        assert abs(slope - (grads[i].double() * d).sum()) <= 1e-4 * (grads[i].double() * d).abs().sum(), i


def test_agrees_with_class_logprobs():
    """The same classifier through stored float32 logits."""
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x, w, labels, b, gl, _ = _inputs(100, 64, 500, F, seed=12)
    r = linear_cross_entropy(x, w, labels, bias=b)
    lp = class_logprobs((x.double() @ w.double().t() + b.double()).float(), labels).logprob
    assert (r.loss + lp).abs().max() <= 1e-4


@pytest.mark.parametrize("dtype", [F, B])
def test_deterministic_on_streams_and_in_graphs(dtype):
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    sets = [_inputs(300 + k, 130, 3000 + 100 * k, dtype, seed=20 + k) for k in range(2)]

    def step(s):
        x, w, labels, b, gl, gs = s
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        r = linear_cross_entropy(leaves[0], leaves[1], labels, bias=leaves[2])
        grads = torch.autograd.grad([r.loss, r.logsumexp], leaves, [gl, gs])
        return [t.detach() for t in (*r, *grads)]

    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(2):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(s))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, v in zip(got, want) for p, q in zip(g, v))
    del got
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(step(s))
    for i in range(3):
        for s in sets:
            s[0].mul_(0.9)
            s[2][i::7] = -100
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, h in zip(sets, held):
            kept = [t.clone() for t in h]
            assert all(torch.equal(p, q) for p, q in zip(kept, step(s))), i


def test_refusals():
    from cign_amd.linear_cross_entropy import linear_cross_entropy as op

    x, w = torch.zeros(6, 32, device="cuda"), torch.zeros(50, 32, device="cuda")
    y, b = torch.zeros(6, dtype=torch.int64, device="cuda"), torch.zeros(50, device="cuda")
    for a, err in (((x.half(), w, y), TypeError), ((x, w.bfloat16(), y), TypeError), ((x, None, y), TypeError),
                   ((x, w[:, :31], y), ValueError), ((x, w[:0], y), ValueError), ((x, w[0], y), ValueError),
                   ((x, w, y[:5]), ValueError), ((x, w, y.float()), TypeError), ((x, w, None), TypeError),
                   ((x, w.cpu(), y), ValueError), ((x, w, y.cpu()), ValueError), ((x, w, y, b[:49]), ValueError),
                   ((x, w, y, b.bfloat16()), TypeError), ((x, w, y, b.cpu()), ValueError), ((x[:, :0], w, y), ValueError),
                   ((torch.zeros(1, 65537, device="cuda"), torch.zeros(2, 65537, device="cuda"), y[:1]), ValueError)):
        with pytest.raises(err):
            op(*a)
    q = torch.randn(6, 32, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(op(q, w + 0.1, y).loss.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
