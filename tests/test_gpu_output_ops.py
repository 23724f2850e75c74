"""GPU: the output operators as the model and the training driver use them:
the fused output norm in GraphCliffordNet, predictions, a teacher's targets and
distillation steps on a small graph.

Two float32 evaluations of the same norm differ by a few u = 2^-24 of each
normalised value (tests/test_gpu_layernorm.py: at most 72 u); a logit sums 96 of them
with weights of at most 0.11 (nn.Linear's 1 / sqrt(96)) and values of at most 5,
so by at most 96 * 0.11 * 5 * 72 u = 2.3e-4, 3e-4 with the sum's own rounding; a
gradient, two such passes apart, by 1e-4 of its tensor's norm."""
import types

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from tests.test_train_driver import _write_npz

pytestmark = pytest.mark.gpu


def _setup(tmp_path, layers=2, hidden=32, classes=5, seed=0, **kw):
    from cign_amd import train_cign as T
    from cign_amd.model_cign import GraphCliffordNet

    rng = np.random.default_rng(3)
    _write_npz(tmp_path / "roman_empire" / "raw" / "roman_empire.npz", rng, n=300, f=20, e=1500, classes=classes)
    _, data = T.load_dataset("Roman-empire", str(tmp_path))
    data = T.apply_split(data, types.SimpleNamespace(split_mode="original", split_index=2))
    torch.manual_seed(seed)
    model = GraphCliffordNet(20, hidden, classes, num_layers=layers, order_set=(1, 2, 3), gat_heads=4, dropout=0.0,
                             gat_dropout=0.0, **kw).cuda()
    pg = T.prepare_graph(model, data, torch.device("cuda"), hop_scales=(1, 2, 3))
    data = data.to("cuda")
    data.edge_index = pg.edge_index
    return T, model, data, pg.graph_operator


def test_fused_output_norm_in_the_model(tmp_path):
    T, plain, data, op = _setup(tmp_path)
    _, fused, _, op2 = _setup(tmp_path, use_fused_output_norm=True)
    fused.load_state_dict(plain.state_dict())  # the same parameter names
    assert type(plain.output_norm) is torch.nn.LayerNorm and plain.use_fused_output_norm is False
    seen = []
    fused.output_norm.register_forward_hook(lambda m, i, o: seen.append(tuple(o.shape)))
    a, b = T.evaluate_logits(plain, data, op), T.evaluate_logits(fused, data, op2)
    assert seen == [(300, 96)]
    assert (a - b).abs().max().item() <= 3e-4
    grads = []
    for m, o in ((plain, op), (fused, op2)):
        m.train()
        loss = F.cross_entropy(T.forward_model(m, data, o)[data.train_mask], data.y[data.train_mask])
        grads.append(torch.autograd.grad(loss, list(m.parameters())))
    for (name, _), x, y in zip(plain.named_parameters(), *grads):
        assert (x - y).norm() <= 1e-4 * x.norm() + 1e-7, name


def test_fused_layernorm_module_refusals():
    from cign_amd.model_cign import FusedLayerNorm

    for bad in ((4, 8), 0, 16385):
        with pytest.raises(ValueError, match="FusedLayerNorm"):
            FusedLayerNorm(bad)
    norm = FusedLayerNorm(48).cuda()
    with pytest.raises(ValueError, match="rows of 48"):
        norm(torch.zeros(3, 47, device="cuda"))
    x = torch.randn(2, 3, 48, device="cuda")
    assert (norm(x) - F.layer_norm(x, (48,))).abs().max() <= 72 * 2.0 ** -24 * 2 * 5
    assert FusedLayerNorm(48, elementwise_affine=False).cuda()(x).shape == x.shape


def test_predictions(tmp_path):
    T, model, data, op = _setup(tmp_path)
    r = T.predict_nodes(model, data, op, top_k=3)
    logits = T.evaluate_logits(model, data, op)
    lp = torch.log_softmax(logits.double(), 1)
    assert torch.equal(r.top_index[:, 0], logits.argmax(1))
    assert T.accuracy(logits, data.y, data.val_mask) == (
        (r.top_index[:, 0] == data.y) & data.val_mask).sum().item() / data.val_mask.sum().item()
    # log probabilities of 5 classes whose logits stay below 10: within 100 u of the definition
    tol = 100 * 2.0 ** -24 * 10
    assert (r.logprob - lp.gather(1, data.y[:, None])[:, 0]).abs().max() <= tol
    assert (r.entropy + (lp.exp() * lp).sum(1)).abs().max() <= tol
    assert (r.top_logprobs - lp.gather(1, r.top_index)).abs().max() <= tol


@pytest.mark.parametrize("tail", [False, True])
def test_distillation_steps(tmp_path, tail):
    """A wide teacher's top 3 of 5 classes into a narrow student: the loss a
    step reports is torch's on the same logits, parameters move, and the
    teacher's and the student's graphs stay apart."""
    T, teacher, data, op = _setup(tmp_path, seed=1)
    _, student, _, sop = _setup(tmp_path, layers=1, hidden=16, seed=2, use_fused_output_norm=True)
    targets = T.teacher_targets(teacher, data, op, top_k=3, temperature=2.0)
    assert targets.index.shape == targets.logprobs.shape == (300, 3) and not targets.logprobs.requires_grad
    opt = torch.optim.Adam(student.parameters(), lr=3e-3)
    for _ in range(3):
        with torch.no_grad():
            student.train()
            z = T.forward_model(student, data, sop).double()
        lq, lp = torch.log_softmax(z / 2.0, 1), targets.logprobs.double()
        if tail:
            left = (1 - lp.exp().sum(1)).clamp_min(0)
            rest = lq.scatter(1, targets.index, -torch.inf).logsumexp(1)
            kl = (lp.exp() * (lp - lq.gather(1, targets.index))).sum(1) + left * (left.log() - rest)
        else:
            lp = torch.log_softmax(lp, 1)
            kl = (lp.exp() * (lp - lq.gather(1, targets.index))).sum(1)
        want = 0.7 * F.cross_entropy(z[data.train_mask], data.y[data.train_mask]) + 0.3 * 4.0 * kl.mean()
        before = [p.detach().clone() for p in student.parameters()]
        loss, secs = T.distill_one_epoch(student, data, sop, opt, torch.device("cuda"), targets, weight=0.3, tail=tail)
        # the logits are the same float32 values: 300 terms below 20, float32 sums
        assert abs(loss - want.item()) <= 1e-5 * max(1.0, abs(want.item())) and secs > 0
        assert any(not torch.equal(a, b) for a, b in zip(before, student.parameters()))
    assert all(p.grad is None for p in teacher.parameters())
    with pytest.raises(ValueError, match="weight"):
        T.distill_one_epoch(student, data, sop, opt, torch.device("cuda"), targets, weight=1.5)
    with pytest.raises(RuntimeError, match="GPU only"):
        T.distill_one_epoch(student, data, sop, opt, torch.device("cpu"), targets)


def test_distillation_step_in_a_graph(tmp_path):
    """Teacher's targets, then a captured pass of norm, losses and gradients,
    replayed against the eager one."""
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    gen = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    teacher = class_logprobs(3 * rn(500, 700), top_k=10, temperature=2.0)
    h, w, b = rn(500, 700).requires_grad_(), rn(700).requires_grad_(), rn(700).requires_grad_()
    labels = torch.randint(0, 700, (500,), generator=gen, device="cuda")
    up = rn(500), rn(500), rn(500)

    def step():
        z = fused_layernorm(h, w, b)
        kl = distill_topk_loss(z, teacher.top_logprobs, teacher.top_index, 2.0, tail=True)
        r = class_logprobs(z, labels, top_k=4)
        grads = torch.autograd.grad([kl, r.logprob, r.entropy], [h, w, b], up)
        # detached: no eager graph of the leaves lives on while a step is captured
        return [t.detach() for t in (kl, *r, *grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            h.mul_(0.8)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), i


def test_calls_at_once_on_two_streams_and_in_two_graphs():
    """Long rows (slices, joins and their workspaces) on two streams at a time,
    then in two captured graphs replayed in turn: each has the values of a call of
    its own."""
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    gen = torch.Generator(device="cuda").manual_seed(11)
    sets = []
    for V in (20011, 40000):
        x = torch.randn(60, V, generator=gen, device="cuda")
        index = torch.randint(0, V, (60, 128), generator=gen, device="cuda")
        t = torch.log_softmax(torch.randn(60, 128, generator=gen, device="cuda"), dim=1)
        sets.append((x, index[:, 0].contiguous(), t, index))

    def calls(x, labels, t, index):
        x = x.detach().requires_grad_()
        r = class_logprobs(x, labels, top_k=20)
        loss = distill_topk_loss(x, t, index, tail=True)
        gx, = torch.autograd.grad([r.logprob, r.entropy, loss], x, [torch.ones_like(loss)] * 3)
        return [*r, loss, gx, fused_layernorm(x.detach()[:, :9001])]

    want = [calls(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(calls(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    del got
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(calls(*s))
    for _ in range(3):
        for o in outs:
            for v in o:
                v.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(outs, want) for a, b in zip(g, w))


def _operators():
    """name -> (function of rows, the rows' width)."""
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    gen = torch.Generator(device="cuda").manual_seed(21)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    w, b, t = rn(40), rn(40), torch.log_softmax(rn(6, 3), 1)
    labels = torch.randint(0, 40, (6,), generator=gen, device="cuda")
    index = torch.randint(0, 40, (6, 3), generator=gen, device="cuda")
    return {
        "norm": lambda x: fused_layernorm(x, w, b),
        "norm, no parameters": lambda x: fused_layernorm(x),
        "log probabilities": lambda x: class_logprobs(x, labels).logprob,
        "entropy": lambda x: class_logprobs(x).entropy,
        "list": lambda x: distill_topk_loss(x, t, index),
        "list and tail": lambda x: distill_topk_loss(x, t, index, 2.0, tail=True),
    }


def test_forward_mode_derivatives_are_refused():
    """Not zero: with and without gradients, of every input that has one."""
    import torch.autograd.forward_ad as fwd

    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    x = torch.randn(6, 40, device="cuda")
    tangent = torch.ones_like(x)
    with fwd.dual_level():
        for name, f in _operators().items():
            for leaf in (x, x.clone().requires_grad_()):
                dual = fwd.make_dual(leaf, tangent)
                with pytest.raises(RuntimeError, match="jvp"):
                    f(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                    f(dual)
            assert f(x).isfinite().all(), name
        w = fwd.make_dual(torch.ones(40, device="cuda"), torch.ones(40, device="cuda"))
        for args in ((w, None), (None, w)):
            with pytest.raises(RuntimeError, match="jvp"):
                fused_layernorm(x, *args)
        t = fwd.make_dual(torch.zeros(6, 3, device="cuda"), torch.ones(6, 3, device="cuda"))
        with pytest.raises(RuntimeError, match="jvp"):
            distill_topk_loss(x, t, torch.zeros(6, 3, dtype=torch.int64, device="cuda"))
    for name, f in _operators().items():
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (tangent,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: f(v).sum())(x)


def test_traced_calls_compute():
    """A traced call computes what the call does, on other values, with and
    without a gradient, after a save as well; so does a graph of tensor
    operations."""
    import io

    from torch.fx.experimental.proxy_tensor import make_fx

    x, other = torch.randn(6, 40, device="cuda"), torch.randn(6, 40, device="cuda")
    for name, f in _operators().items():
        want = f(other)
        leaf = other.clone().requires_grad_()
        up = torch.randn_like(want)
        grad, = torch.autograd.grad(f(leaf), leaf, up)
        for example in (x, x.clone().requires_grad_()):
            traced = torch.jit.trace(f, (example,))
            buffer = io.BytesIO()
            torch.jit.save(traced, buffer)
            buffer.seek(0)
            for g in (traced, torch.jit.load(buffer)):
                assert torch.equal(g(other), want), name
                leaf = other.clone().requires_grad_()
                assert torch.equal(torch.autograd.grad(g(leaf), leaf, up)[0], grad), name
        assert torch.equal(make_fx(f)(x)(other), want), name
        if not name.startswith("norm") and name != "entropy":  # labels and lists of six rows
            with pytest.raises(RuntimeError, match="must have shape"):
                traced(other[:4])
    from cign_amd.model_cign import FusedLayerNorm

    norm = FusedLayerNorm(40).cuda()
    with torch.no_grad():
        norm.weight.normal_()
    assert torch.equal(torch.jit.trace(norm, (x,))(other), norm(other))


def test_memory_errors_are_torch_s():
    """A result that no memory holds: the error other calls of torch raise."""
    for name, f in {"norm": lambda x: _operators()["norm, no parameters"](x),
                    "entropy": lambda x: _operators()["entropy"](x)}.items():
        with pytest.raises(torch.OutOfMemoryError):
            f(torch.zeros(1, 40, device="cuda").expand(1 << 44, 40))


def test_predictions_outside_inference_mode(tmp_path):
    """Logits of the evaluation forward are inference tensors; what is read from
    them is not."""
    T, model, data, op = _setup(tmp_path)
    r = T.predict_nodes(model, data, op, top_k=2)
    assert not any(v.is_inference() or v.requires_grad for v in r)
    from cign_amd.distill import distill_topk_loss

    x = torch.randn(300, 5, device="cuda").requires_grad_()
    assert torch.autograd.grad(distill_topk_loss(x, r.top_logprobs, r.top_index).sum(), x)[0].isfinite().all()


def test_transforms_agree_or_refuse():
    """vmap over rows of rows: the values of the calls one by one, or an error."""
    xs = torch.randn(3, 6, 40, device="cuda")
    for name, f in _operators().items():
        want = torch.stack([f(x) for x in xs])
        try:
            got = torch.func.vmap(f)(xs)
        except RuntimeError:
            continue
        assert torch.equal(got, want), name


def test_distillation_without_labelled_nodes(tmp_path):
    """weight = 1 leaves the labels out, also where no node has one; weight = 0
    leaves the lists out."""
    T, model, data, op = _setup(tmp_path, seed=1)
    targets = T.teacher_targets(model, data, op, top_k=3)
    opt = torch.optim.SGD(model.parameters(), lr=0.0)
    step = lambda weight: T.distill_one_epoch(model, data, op, opt, torch.device("cuda"), targets, weight=weight)[0]
    both = step(0.25), step(0.0), step(1.0)
    # 300 float32 terms below 20, as in test_distillation_steps
    assert abs(both[0] - 0.75 * both[1] - 0.25 * both[2]) <= 1e-5 * max(1.0, abs(both[0]))
    mask = data.train_mask
    data.train_mask = torch.zeros_like(mask)
    assert step(1.0) == both[2]
    assert all(p.grad is None or p.grad.isfinite().all() for p in model.parameters())
    data.train_mask = mask
    targets.index[:] = data.y[:, None].new_full(targets.index.shape, 5)  # out of range: a loss of NaN
    assert step(0.0) == both[1] and step(0.5) != step(0.5)
