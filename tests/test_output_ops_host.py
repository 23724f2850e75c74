"""CPU tests of the output operators (LayerNorm of any width, class_logprobs,
distill_topk_loss): what the C-ABI and the Python functions refuse before any
launch, workspace sizes, and the places the row kernels read."""
import math

import numpy as np
import pytest
import torch

from cign_amd import _lib

BIG = 1 << 40  # an address no check looks behind


def _refused(name, args, match):
    lib = _lib.load_library(require_gpu=False)
    with pytest.raises(RuntimeError, match=match):
        lib.call(name, *args)


def _with(args, **changes):
    out = list(args)
    for k, v in changes.items():
        out[int(k[1:])] = v
    return out


def test_layernorm_refusals():
    #      stream n  D   xt wt  x    ldx  w    b   eps   y   mean  rstd
    fwd = (None, 4, 32, 0, 0, BIG, 32, BIG, BIG, 1e-5, BIG, BIG, BIG)
    for change, match in (({"_1": -1}, "negative row count"), ({"_2": 0}, "1<=D<=16384"), ({"_2": 16385}, "1<=D<=16384"),
                          ({"_3": 2}, "dtypes"), ({"_4": 1}, "dtypes"), ({"_3": 1, "_4": 2}, "dtypes"),
                          ({"_5": None}, "null"), ({"_10": None}, "null"), ({"_11": None}, "null"),
                          ({"_12": None}, "null"), ({"_6": -1}, "stride")):
        _refused("cign_layernorm_fwd", _with(fwd, **change), match)
    lib = _lib.load_library(require_gpu=False)
    ws = lib.cign_layernorm_bwd_workspace_bytes(4, 32)
    #      stream n  D   xt wt  gy  ldg  x   ldx  w   mean rstd  gx   gw   gb   ws   bytes
    bwd = (None, 4, 32, 0, 0, BIG, 32, BIG, 32, BIG, BIG, BIG, BIG, BIG, BIG, BIG, ws)
    for change, match in (({"_1": -1}, "negative row count"), ({"_2": 16385}, "1<=D<=16384"), ({"_3": 3}, "dtypes"),
                          ({"_5": None}, "null"), ({"_7": None}, "null"), ({"_10": None}, "null"), ({"_6": -1}, "stride"),
                          ({"_8": -1}, "stride"), ({"_15": None}, "workspace"), ({"_16": ws - 1}, "workspace")):
        _refused("cign_layernorm_bwd", _with(bwd, **change), match)
    lib.call("cign_layernorm_fwd", *_with(fwd, _1=0))  # no rows: nothing to do
    lib.call("cign_layernorm_bwd", *_with(bwd, _12=None, _13=None, _14=None))  # no gradient asked for
    assert lib.cign_layernorm_bwd_workspace_bytes(-1, 32) == lib.cign_layernorm_bwd_workspace_bytes(4, 0) == 0
    assert lib.cign_layernorm_bwd_workspace_bytes(1, 7) == 2 * 4 * 7
    assert lib.cign_layernorm_bwd_workspace_bytes(10**6, 16384) == 2 * 4 * 512 * 16384


def test_class_logprobs_refusals():
    lib = _lib.load_library(require_gpu=False)
    #      stream t  n   V     x    ldx   T    label ignore K  lp   H    tlp  tix  stats ws  bytes
    fwd = (None, 0, 4, 5000, BIG, 5000, 1.0, BIG, -100, 3, BIG, BIG, BIG, BIG, BIG, BIG, 1 << 30)
    for change, match in (({"_1": 2}, "dtype"), ({"_2": -1}, "negative row count"), ({"_3": 0}, "1<=V"),
                          ({"_3": (1 << 20) + 1}, "1<=V"), ({"_5": -1}, "stride"), ({"_6": 0.0}, "temperature"),
                          ({"_6": math.inf}, "temperature"), ({"_6": math.nan}, "temperature"), ({"_9": -1}, "top_k"),
                          ({"_9": 129}, "top_k"), ({"_3": 2}, "top_k"), ({"_4": None}, "null"), ({"_10": None}, "null"),
                          ({"_11": None}, "null"), ({"_12": None}, "null"), ({"_13": None}, "null"),
                          ({"_16": 15}, "workspace too small"), ({"_15": None}, "workspace too small")):
        _refused("cign_class_logprobs_fwd", _with(fwd, **change), match)
    #      stream t  n   V     x    ldx   T    label ignore stats gl   ge   gx
    bwd = (None, 0, 4, 5000, BIG, 5000, 1.0, BIG, -100, BIG, BIG, BIG, BIG)
    for change, match in (({"_1": 2}, "dtype"), ({"_4": None}, "null"), ({"_9": None}, "null"), ({"_12": None}, "null"),
                          ({"_7": None}, "null"), ({"_6": -1.0}, "temperature")):
        _refused("cign_class_logprobs_bwd", _with(bwd, **change), match)
    lib.call("cign_class_logprobs_fwd", *_with(fwd, _2=0))
    lib.call("cign_class_logprobs_bwd", *_with(bwd, _2=0))
    size = lib.cign_class_logprobs_workspace_bytes
    assert size(0, 0, 5000, 0) == size(0, 4, 0, 0) == size(0, 4, 5000, 129) == 0
    assert size(0, 4, 5, 5) == 0  # rows that lane groups hold need none


def test_distill_refusals():
    lib = _lib.load_library(require_gpu=False)
    #      stream t  n   V     x    ldx   T   tail K  t    index loss stats mass ws   bytes
    fwd = (None, 0, 4, 5000, BIG, 5000, 1.0, 1, 3, BIG, BIG, BIG, BIG, BIG, BIG, 1 << 30)
    for change, match in (({"_1": 2}, "dtype"), ({"_2": -1}, "negative row count"), ({"_3": 0}, "1<=V"),
                          ({"_5": -1}, "stride"), ({"_6": 0.0}, "temperature"), ({"_8": 0}, "1<=K"), ({"_8": 129}, "1<=K"),
                          ({"_4": None}, "null"), ({"_9": None}, "null"), ({"_10": None}, "null"), ({"_11": None}, "null"),
                          ({"_12": None}, "null"), ({"_13": None}, "null"), ({"_15": 7}, "workspace too small"),
                          ({"_14": None}, "workspace too small")):
        _refused("cign_distill_topk_fwd", _with(fwd, **change), match)
    #      stream t  n   V     x    ldx   T   K  index stats mass g    gx
    bwd = (None, 0, 4, 5000, BIG, 5000, 1.0, 3, BIG, BIG, BIG, BIG, BIG)
    for change, match in [({"_1": 2}, "dtype"), ({"_7": 0}, "1<=K"), ({"_6": math.nan}, "temperature")] + \
            [({f"_{i}": None}, "null") for i in (4, 8, 9, 10, 11, 12)]:
        _refused("cign_distill_topk_bwd", _with(bwd, **change), match)
    lib.call("cign_distill_topk_fwd", *_with(fwd, _2=0))
    lib.call("cign_distill_topk_bwd", *_with(bwd, _2=0))


def test_functions_refuse_host_tensors():
    from cign_amd.class_logprobs import class_logprobs
    from cign_amd.distill import distill_topk_loss
    from cign_amd.fused_block_ops import fused_layernorm

    x = torch.zeros(3, 8)
    for call in (lambda t: fused_layernorm(t), lambda t: class_logprobs(t),
                 lambda t: distill_topk_loss(t, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64))):
        for bad in (x, x.bfloat16(), x.numpy(), None):
            with pytest.raises(TypeError, match="must be CUDA float32 or bfloat16"):
                call(bad)


def _slicing(V, n, W):
    """rowsoftmax.h slicing()."""
    nc = -(-V // W)
    slices = lambda u: -(-nc // (256 * u))
    U = 8 if slices(8) <= 64 else 16
    while U > 1 and n * slices(U) < 1024 and slices(U // 2) <= 64:
        U //= 2
    S = slices(U)
    cps = -(-nc // S)
    while U > 1 and 256 * (U // 2) >= cps:
        U //= 2
    return U, S, cps


@pytest.mark.parametrize("W", [4, 8])
@pytest.mark.parametrize("n", [1, 3, 100, 5000])
def test_slices_cover_every_class_once_in_bounds(W, n):
    """The chunks of a sliced row: reads inside the row, each value owned by
    one chunk of one slice, lists of slices within what the join holds, and the
    workspace the library asks for."""
    lib = _lib.load_library(require_gpu=False)
    for V in (513, 1000, 2049, 4097, 5001, 8200, 16385, 50001, 131072, 524288, 524289, 1 << 20):
        U, S, cps = _slicing(V, n, W)
        nc = -(-V // W)
        assert 1 <= S <= 64 and cps <= 256 * U and (S - 1) * cps < nc <= S * cps and U <= (16 if W == 4 else 8)
        assert S * -(-128 // S) < 256  # the samples of join_top_kernel
        owned = 0
        for s in range(S):
            end = min((s + 1) * cps, nc)
            for c in {s * cps, end - 1, min(s * cps + 256 * U - 1, s * cps + 255)}:
                at = min(min(c, end - 1) * W, V - W)
                assert 0 <= at and at + W <= V
            first = min(s * cps * W, V)
            owned += min(end * W, V) - first
        assert owned == V
        want = 0 if S == 1 else n * S * (16 + 8 * 5)
        assert lib.cign_class_logprobs_workspace_bytes(int(W == 8), n, V, 5) == want
        long = V > 512 * W
        assert lib.cign_distill_topk_workspace_bytes(int(W == 8), n, V) == (n * S * 8 if long and S > 1 else 0)


def _meta_operators():
    """The operators as a trace repeats them, on meta tensors: name -> (call,
    its tensors by name)."""
    from cign_amd._rows import load_output_ops

    load_output_ops()
    ops = torch.ops.cign_amd
    m = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="meta")
    long = torch.int64
    return {
        "layernorm": (lambda x, w, b: ops.layernorm(x, w, b, 1e-5), dict(x=m(4, 6, 32), w=m(32), b=m(32))),
        "layernorm_backward": (lambda g, x, w, s: ops.layernorm_backward(g, x, w, s, torch.float32, True, True, True),
                               dict(g=m(4, 32), x=m(4, 32), w=m(32), s=m(2, 4))),
        "class_logprobs": (lambda x, y: ops.class_logprobs(x, y, 3, 1.0, -100), dict(x=m(4, 6, 32), y=m(4, 6, t=long))),
        "class_logprobs_backward": (lambda h, g, x, y, s: ops.class_logprobs_backward(h, g, x, y, s, 1.0, -100),
                                    dict(h=m(4), g=m(4), x=m(4, 32), y=m(4, t=long), s=m(4, 4))),
        "distill_topk": (lambda x, t, j: ops.distill_topk(x, t, j, 1.0, True),
                         dict(x=m(4, 6, 32), t=m(4, 6, 3), j=m(4, 6, 3, t=long))),
        "distill_topk_backward": (lambda g, x, j, s: ops.distill_topk_backward(g, x, j, s, 1.0),
                                  dict(g=m(4), x=m(4, 32), j=m(4, 3, t=long), s=m(4 * 11))),
    }


def test_operators_check_what_their_accesses_rest_on():
    """A trace repeats the operators without the Python functions' checks: a
    tensor of another shape, type or device is refused by the operator itself."""
    for name, (call, args) in _meta_operators().items():
        first = next(iter(args))
        out = call(**args)
        out = list(out) if isinstance(out, (list, tuple)) else [out]
        assert out[0].shape[: args[first].dim() - 1] == args[first].shape[:-1] or name.endswith("backward"), name
        for key, t in args.items():
            shorter = t[:-1] if key != "s" or name != "layernorm_backward" else t[:, :-1]
            if (name, key) == ("layernorm", "x"):  # nothing else has its rows
                shorter = t[..., :-1]
            for bad in (shorter, t[..., None], t.double(), t.half(), torch.zeros(t.shape, dtype=t.dtype)):
                with pytest.raises((RuntimeError, TypeError, ValueError)):
                    call(**{**args, key: bad})
        if "w" in args:
            with pytest.raises((RuntimeError, TypeError, ValueError)):
                call(**{**args, "w": args["w"].bfloat16()})
    ops, x = torch.ops.cign_amd, torch.zeros(4, 32, device="meta")
    for k in (-1, 33, 1 << 32):
        with pytest.raises(ValueError, match="top_k"):
            ops.class_logprobs(x, None, k, 1.0, -100)
    for t in (torch.zeros(4, 0, device="meta"), torch.zeros((), device="meta")):
        with pytest.raises(ValueError):
            ops.layernorm(t, None, None, 1e-5)
    with pytest.raises(ValueError, match="detach"):
        ops.distill_topk(x, torch.zeros(4, 3, device="meta").requires_grad_(),
                         torch.zeros(4, 3, dtype=torch.int64, device="meta"), 1.0, True)
    for call, args in _meta_operators().values():  # on the host: no kernel
        with pytest.raises((RuntimeError, TypeError)):
            call(**{k: torch.zeros(t.shape, dtype=t.dtype) for k, t in args.items()})


def test_traces_and_forward_mode_on_the_host():
    """A trace holds the call, with and without a gradient, and a forward-mode
    derivative raises."""
    import torch.autograd.forward_ad as fwd

    for name, (call, args) in _meta_operators().items():
        if name.endswith("backward"):
            continue
        rest = {k: t for k, t in args.items() if k != "x"}
        f = lambda x: call(x=x, **rest)
        for x in (args["x"], args["x"].clone().requires_grad_()):
            graph = torch.jit.trace(f, (x,), check_trace=False).graph
            assert f"cign_amd::{name}(" in str(graph) and "aten::empty" not in str(graph)
            with fwd.dual_level():
                dual = fwd.make_dual(x, torch.zeros_like(args["x"]))
                with pytest.raises(RuntimeError, match="jvp"):
                    f(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                    f(dual)
        for key, t in rest.items():
            if t.is_floating_point():
                with fwd.dual_level(), pytest.raises(RuntimeError, match="jvp"):
                    call(**{**args, key: fwd.make_dual(t, torch.zeros_like(t))})
        leaf = args["x"].clone().requires_grad_()
        out = call(**{**args, "x": leaf})
        grad, = torch.autograd.grad(out[0].sum() if name == "class_logprobs" else out.sum(), leaf)
        assert grad.shape == leaf.shape


def _owners(V, W, first, stride, end, threads, U):
    """How often each value of a row of V is some thread's own: Share::place of
    `threads` threads whose chunks lie `stride` apart from `first` on, below
    chunk `end`; every access inside the row."""
    i = (first + np.arange(threads)[:, None] + stride * np.arange(U)[None, :]) * W
    at = np.minimum(i, min(end * W, V) - W)
    own = np.minimum(i - at, W)
    assert at.min() >= 0 and at.max() + W <= V
    value = at[..., None] + np.arange(W)
    return np.bincount(value[np.arange(W) >= own[..., None]], minlength=V)


def _ragged():
    """Widths at, just below and just past what chunks, slices and their numbers
    of chunks a thread end at."""
    edges = {512, 1024, 2048, 4096, 8192, 16384, 32768, 50001, 65536, 131072, 300007, 524288, 1 << 20}
    return sorted(v for e in edges for v in (e - 9, e - 1, e, e + 1, e + 3, e + 4, e + 9) if v <= 1 << 20)


@pytest.mark.parametrize("W", [4, 8])
@pytest.mark.parametrize("n", [1, 3, 100, 5000])
def test_each_value_of_a_sliced_row_has_one_owner(W, n):
    """slice_kernel of both operators, as rowsoftmax.h places it."""
    for V in _ragged():
        U, S, cps = _slicing(V, n, W)
        nc = -(-V // W)
        count = sum(_owners(V, W, s * cps, 256, min((s + 1) * cps, nc), 256, U) for s in range(S))
        assert (count == 1).all(), (V, np.flatnonzero(count != 1)[:5])


@pytest.mark.parametrize("W", [4, 8])
def test_each_value_of_a_gradient_has_one_owner(W):
    """grad_kernel: slices of 32 values a thread, and the rows of lane groups."""
    for V in _ragged() + list(range(1, 600)):
        nc = -(-V // W)
        if nc > 512:
            U = 32 // W
            S = -(-nc // (256 * U))
            cps = -(-nc // S)
            count = sum(_owners(V, W, s * cps, 256, min((s + 1) * cps, nc), 256, U) for s in range(S))
        else:  # with_lanes
            w = W if V >= W else 1
            chunks = -(-V // w)
            lanes = min(64, 1 << (chunks - 1).bit_length())
            U = 1 << (-(-chunks // lanes) - 1).bit_length()
            count = _owners(V, w, 0, lanes, chunks, lanes, U)
        assert (count == 1).all(), (V, np.flatnonzero(count != 1)[:5])
