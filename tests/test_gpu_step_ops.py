"""GPU: a training step's operators together: blocks with their boundaries, the
loss over many classes and the clipped gradients, as a model uses them and as the
training driver does."""
import types

import pytest
import torch
import torch.nn.functional as F

from tests.test_gpu_output_ops import _setup

pytestmark = pytest.mark.gpu


class _Deep(torch.nn.Module):
    """Blocks of one product each between fused boundaries, and a classifier."""

    def __init__(self, width, depth, classes):
        super().__init__()
        v = lambda m: torch.nn.Parameter(torch.full((width,), m))
        self.inner = torch.nn.ParameterList([torch.nn.Parameter(torch.randn(width, width) / width ** 0.5) for _ in range(depth)])
        self.vectors = torch.nn.ModuleList([torch.nn.ParameterDict(
            dict(post_weight=v(1.0), post_bias=v(0.0), scale=v(0.4), next_weight=v(1.0), next_bias=v(0.0)))
            for _ in range(depth)])
        self.gates = torch.nn.ParameterList([torch.nn.Parameter(torch.randn(width) / width ** 0.5) for _ in range(depth)])
        self.head = torch.nn.Parameter(torch.randn(classes, width) / width ** 0.5)
        self.head_bias = torch.nn.Parameter(torch.zeros(classes))

    def features(self, x, boundary):
        y = h = x
        for w, vec, a in zip(self.inner, self.vectors, self.gates):
            h, y = boundary(torch.tanh(y @ w), h, gate=(y @ a)[:, None], **dict(vec))
        return y


def _plain_boundary(branch, residual, gate, post_weight, post_bias, scale, next_weight, next_bias):
    v = F.layer_norm(branch, branch.shape[-1:], post_weight, post_bias)
    h = residual + scale * torch.sigmoid(gate) * v
    return h, F.layer_norm(h, h.shape[-1:], next_weight, next_bias)


def test_a_deep_model_steps_as_its_float64_form():
    """Three steps of SGD with clipping: losses, norms and parameters against the
    same steps in float64. Four blocks each multiply a relative rounding of at most
    1e-5 (norms of 96 values, products of 96 terms) by a small factor; 1e-3 of a
    tensor's norm leaves room for 100."""
    from cign_amd.fused_block_ops import fused_gated_residual_norm
    from cign_amd.grad_norm import clip_grad_norm
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    torch.manual_seed(0)
    mine = _Deep(96, 4, 5003).cuda()
    ref = _Deep(96, 4, 5003).cuda()
    ref.load_state_dict(mine.state_dict())
    ref = ref.double()
    x = torch.randn(333, 96, device="cuda")
    labels = torch.randint(0, 5003, (333,), device="cuda")
    labels[::5] = -100
    count = (labels >= 0).sum()
    for step in range(3):
        r = linear_cross_entropy(mine.features(x, fused_gated_residual_norm), mine.head, labels, bias=mine.head_bias)
        loss = r.loss.sum() / count + 1e-3 * r.logsumexp.square().mean()
        z = ref.features(x.double(), _plain_boundary) @ ref.head.t() + ref.head_bias
        want = F.cross_entropy(z, labels) + 1e-3 * torch.logsumexp(z, 1).square().mean()
        assert abs(float(loss) - float(want)) <= 1e-5 * float(want), step
        norms = []
        for m, l in ((mine, loss), (ref, want)):
            params = list(m.parameters())
            grads = list(torch.autograd.grad(l, params))
            if m is mine:
                norms.append(float(clip_grad_norm(grads, 0.1)))
            else:
                norms.append(float(torch.cat([g.flatten() for g in grads]).norm()))
                grads = [g * min(1.0, 0.1 / (norms[-1] + 1e-6)) for g in grads]
            with torch.no_grad():
                for p, g in zip(params, grads):
                    p.sub_(g)
        assert abs(norms[0] - norms[1]) <= 1e-4 * norms[1] and norms[1] > 0.1
        for (name, p), q in zip(mine.named_parameters(), ref.parameters()):
            assert (p.double() - q).norm() <= 1e-3 * 0.1 + 1e-6 * q.norm(), (step, name)


def test_a_step_in_a_graph():
    """Boundary, loss and clipping captured once, replayed against eager steps."""
    from cign_amd.fused_block_ops import fused_gated_residual_norm
    from cign_amd.grad_norm import clip_grad_norm
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    gen = torch.Generator(device="cuda").manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    u, h, a, w, head = rn(400, 256), rn(400, 256), rn(400, 256), rn(256), 0.1 * rn(3001, 256)
    labels = torch.randint(0, 3001, (400,), generator=gen, device="cuda")

    def step():
        leaves = [t.detach().requires_grad_() for t in (u, h, a, w, head)]
        _, y = fused_gated_residual_norm(leaves[0], leaves[1], gate=leaves[2], next_weight=leaves[3], norm="rms")
        loss = linear_cross_entropy(y, leaves[4], labels).loss
        grads = list(torch.autograd.grad(loss.mean(), leaves))
        return [loss.detach(), clip_grad_norm(grads, 0.01), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        for t in (u, head):
            t.mul_(0.9)
        labels.copy_(torch.where(labels % 5 == i, -100, labels))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(kept, want)), i


def test_node_losses_and_clipped_steps(tmp_path):
    """The driver's step with the fused loss and clipping: the loss of the logits'
    cross-entropy, and parameters moved by gradients of at most the given norm."""
    T, model, data, op = _setup(tmp_path, classes=5)
    labels = torch.where(data.train_mask, data.y, -100)
    z = T.evaluate_logits(model, data, op)
    with torch.no_grad():
        r = model.node_losses(data.x, data.edge_index, op, labels)
    # two float32 evaluations of one classifier over 96 values: 3e-4 as for the fused norm
    assert (r.loss - F.cross_entropy(z, labels, reduction="none")).abs().max() <= 6e-4
    assert (r.logsumexp - torch.logsumexp(z, 1)).abs().max() <= 3e-4
    model.train()
    a = F.cross_entropy(T.forward_model(model, data, op)[data.train_mask], data.y[data.train_mask])
    b = model.node_losses(data.x, data.edge_index, op, labels).loss.sum() / data.train_mask.sum()
    params = list(model.parameters())
    for (name, _), p, q in zip(model.named_parameters(), torch.autograd.grad(a, params), torch.autograd.grad(b, params)):
        assert (p - q).norm() <= 1e-4 * p.norm() + 1e-7, name
    before = [p.detach().clone() for p in params]
    sgd = torch.optim.SGD(params, lr=1.0)
    loss, secs = T.train_one_epoch(model, data, op, sgd, torch.device("cuda"), max_grad_norm=1e-3, fused_loss=True)
    assert abs(loss - float(a)) <= 1e-4 * abs(float(a)) and secs > 0
    moved = torch.cat([(p.detach() - q).flatten() for p, q in zip(params, before)]).double().norm()
    assert 0.9e-3 <= float(moved) <= 1.1e-3  # parameters of up to 3 move by float32 steps of 2^-23
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
    before = [p.detach().clone() for p in params]
    T.train_one_epoch(model, data, op, sgd, torch.device("cuda"), grad_scaler=scaler, max_grad_norm=1e-3)
    moved = torch.cat([(p.detach() - q).flatten() for p, q in zip(params, before)]).double().norm()
    assert 0.9e-3 <= float(moved) <= 1.1e-3
    targets = T.teacher_targets(model, data, op, top_k=3)
    before = [p.detach().clone() for p in params]
    T.distill_one_epoch(model, data, op, sgd, torch.device("cuda"), targets, max_grad_norm=1e-3)
    moved = torch.cat([(p.detach() - q).flatten() for p, q in zip(params, before)]).double().norm()
    assert float(moved) <= 1.1e-3
    with pytest.raises(ValueError, match="graph operator"):
        model.node_losses(data.x, data.edge_index, None, labels)


def _operators():
    from cign_amd.fused_block_ops import fused_gated_residual_norm
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    labels = torch.tensor([1, 2, -100, 0], device="cuda")
    w = torch.randn(7, 48, device="cuda")
    return {"boundary": lambda t: fused_gated_residual_norm(t, t)[1], "loss": lambda t: linear_cross_entropy(t, w, labels).loss}


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwAD

    x, t = torch.randn(4, 48, device="cuda"), torch.randn(4, 48, device="cuda")
    for name, f in _operators().items():
        with fwAD.dual_level(), pytest.raises(RuntimeError, match="jvp|forward"):
            f(fwAD.make_dual(x, t))


def test_traced_calls_compute():
    """A trace holds the calls: other values, and shapes that are checked."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, y = torch.randn(4, 48, device="cuda"), torch.randn(4, 48, device="cuda")
    for name, f in _operators().items():
        traced = make_fx(f)(x)
        assert torch.equal(traced(y), f(y)), name
