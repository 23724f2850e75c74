"""GPU: the output operators at sizes where their results, and from 320 MiB on
their logits, pass the cache (kernels of their own: 112 MiB of rows for LayerNorm,
144 and 320 MiB of logits for the gradients and slices). Rows are sampled, the
first and last among them, and compared value by value with the oracles of the
operators' own tests, under their bounds; LayerNorm's parameter gradients, which
every row enters, are compared whole."""
import math

import numpy as np
import pytest
import torch

from tests import test_gpu_class_logprobs as lp
from tests import test_gpu_distill as ds
from tests import test_gpu_layernorm as ln
from tests.conftest import assert_within

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
MIB = 1 << 20


def _rows(bytes_, width, dtype):
    """The least number of rows of this many bytes, made odd."""
    size = 2 if dtype == BF16 else 4
    return -(-bytes_ // (width * size)) | 1


def _sample(n, seed):
    at = np.random.default_rng(seed).integers(0, n, 24)
    return np.unique(np.concatenate([at, [0, 1, n // 2, n - 2, n - 1]]))


@pytest.mark.parametrize("D,dtype,wdtype", [(1001, BF16, BF16), (1283, F32, F32), (8193, F32, F32), (12290, BF16, F32),
                                            (3, F32, F32), (7, BF16, F32), (40, BF16, BF16)])
def test_layernorm_past_the_cache(D, dtype, wdtype):
    from cign_amd.fused_block_ops import fused_layernorm

    n = _rows(112 * MIB, D, dtype)
    print(f"layernorm {n} x {D} {dtype}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(D)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g = rn(n, D).to(dtype), rn(n, D).to(dtype)
    w, b = (1 + 0.3 * rn(D)).to(wdtype), (0.3 * rn(D)).to(wdtype)
    eps = 1e-2 if D < 16 else 1e-5
    for t in (x, w, b):
        t.requires_grad_()
    y = fused_layernorm(x, w, b, eps)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), g)
    at = _sample(n, D)
    pick = torch.from_numpy(at).cuda()
    a = [lp._n(t) for t in (x.detach()[pick], w, b, g[pick])]
    o = ln._oracle(a[0], a[1], a[2], eps, a[3])
    bound = ln._bounds(*a, o, dtype, wdtype)
    assert_within(lp._n(y.detach()[pick]), o["y"], bound["y"], f"y n={n} D={D}")
    assert_within(lp._n(gx[pick]), o["gx"], bound["gx"], f"gx n={n} D={D}")
    # the parameters': sums over all rows in float64, a block of them at a time, with the bounds of
    # test_gpu_layernorm.py: each xh off by 72 u (|xh| + max|x| rstd), a chain of additions of a workgroup's
    # rows (n / 256 at most) and 64 more
    U = 2.0 ** -24
    want = torch.zeros(4, D, dtype=torch.float64, device="cuda")  # gw, gb, and what their bounds add
    with torch.no_grad():
        for r in range(0, n, max(1, (1 << 24) // D)):
            xd, gd = (t[r:r + max(1, (1 << 24) // D)].double() for t in (x, g))
            centred = xd - xd.mean(1, keepdim=True)
            rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + eps)
            xh = centred * rstd
            exh = 72 * U * (xh.abs() + xd.abs().amax(1, keepdim=True) * rstd)
            want += torch.stack([(gd * xh).sum(0), gd.sum(0), (gd.abs() * (exh + (n / 256 + 64) * U * xh.abs())).sum(0),
                                 gd.abs().sum(0) * (n / 256 + 64) * U])
    half = ln.HALF[wdtype]
    for name, got, e, err in (("gw", gw, want[0], want[2]), ("gb", gb, want[1], want[3])):
        assert_within(lp._n(got), lp._n(e), lp._n(err + half * (e.abs() + err)), f"{name} n={n} D={D}")


SHAPES = [(32001, BF16), (50001, F32), (601, BF16), (1003, F32), (4105, BF16), (2051, F32)]


@pytest.mark.parametrize("mib", [150, 330])
@pytest.mark.parametrize("V,dtype", SHAPES)
def test_logprobs_gradient_past_the_cache(V, dtype, mib):
    from cign_amd.class_logprobs import class_logprobs

    n = _rows(mib * MIB, V, dtype)
    print(f"class_logprobs {n} x {V} {dtype}", flush=True)
    x, labels, g, h = lp._logits(n, V, dtype, V + mib)
    labels[::7] = -100
    labels[n - 1] = V - 1
    x[:, V - 3] = -math.inf
    labels = torch.where(labels == V - 3, 0, labels)
    x.requires_grad_()
    at = _sample(n, V)
    pick = torch.from_numpy(at).cuda()
    xn = lp._n(x.detach()[pick])
    half = lp.HALF[dtype]
    for gg, hh, k in ((g, h, 3), (g, None, 0)):
        r = class_logprobs(x, labels, top_k=k)
        outs, ups = zip(*[(o, u) for o, u in ((r.logprob, gg), (r.entropy, hh)) if u is not None])
        grad, = torch.autograd.grad(outs, x, ups)
        o = lp._oracle(xn, 1.0, labels[pick].cpu().numpy(), -100, lp._n(gg[pick]), None if hh is None else lp._n(hh[pick]))
        lp._within(lp._n(r.logprob[pick]), o["logprob"], o["e_logprob"], f"logprob {n} x {V}")
        lp._within(lp._n(r.entropy[pick]), o["H"], o["e_h"], f"entropy {n} x {V}")
        if k:
            want = lp._top(xn, k)
            assert np.array_equal(r.top_index[pick].cpu().numpy(), want)
        lp._within(lp._n(grad[pick]), o["grad"], o["e_grad"] + half * (np.abs(o["grad"]) + o["e_grad"]) + 2.0 ** -126,
                   f"grad {n} x {V}")
        assert not grad[::7].any() or hh is not None  # ignored rows without an entropy's gradient


@pytest.mark.parametrize("mib", [150, 330])
@pytest.mark.parametrize("V,dtype", SHAPES)
def test_list_gradient_past_the_cache(V, dtype, mib):
    """Lists with the row's last class (in its ragged last chunk), a class
    named twice, empty places and rows without any."""
    from cign_amd.distill import distill_topk_loss

    n, K = _rows(mib * MIB, V, dtype), 12
    print(f"distill {n} x {V} {dtype}", flush=True)
    x = lp._logits(n, V, dtype, V + mib + 1)[0]
    gen = torch.Generator(device="cuda").manual_seed(V)
    index = torch.randint(0, V - 2, (n, K), generator=gen, device="cuda")
    index[:, 0], index[:, 1] = V - 1, V - 2
    t = torch.log_softmax(torch.randn(n, K, generator=gen, device="cuda"), 1) - 0.2
    index[1::3, 5], t[1::3, 5] = index[1::3, 4], t[1::3, 4]  # twice, both places alike
    index[::5, 7:] = -1
    index[n // 2] = -1
    g = torch.rand(n, generator=gen, device="cuda") + 0.5
    x.requires_grad_()
    at = _sample(n, V)
    pick = torch.from_numpy(at).cuda()
    a = [lp._n(v[pick]) for v in (x.detach(), t)]
    half = ds.HALF[dtype]
    for tail in (False, True):
        loss = distill_topk_loss(x, t, index, tail=tail)
        grad, = torch.autograd.grad(loss, x, g)
        el, bl, eg, bg = ds._oracle(*a, index[pick].cpu().numpy(), 1.0, tail, lp._n(g[pick]))
        ds._within(lp._n(loss[pick]), el, bl, f"loss {n} x {V}")
        ds._within(lp._n(grad[pick]), eg, bg + half * (np.abs(eg) + bg) + 2.0 ** -126, f"grad {n} x {V}")
        assert not grad[n // 2].any()
