"""CPU tests of a training step's operators (block boundary, cross entropy of a
linear classifier, global gradient norm): what the C-ABI and the Python functions
refuse before any launch, workspace sizes, shapes on meta tensors, and the tables
and segments the kernels follow."""
import ctypes as C
import math

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


def test_block_boundary_refusals():
    #      stream n D  xt wt ly gk u    ldu h    ldh a    lda w1   b1   c    w2   b2   eps   hid  y    stats
    fwd = (None, 4, 32, 0, 0, 1, 2, BIG, 32, BIG, 32, BIG, 32, BIG, BIG, BIG, BIG, BIG, 1e-5, BIG, BIG, BIG)
    for change, match in (({"_1": -1}, "negative row count"), ({"_2": 0}, "1<=D<=8192"), ({"_2": 8193}, "1<=D<=8192"),
                          ({"_3": 2}, "dtypes"), ({"_4": 1}, "dtypes"), ({"_5": 2}, "layer"), ({"_6": 3}, "gate"),
                          ({"_6": -1}, "gate"), ({"_7": None}, "null"), ({"_9": None}, "null"), ({"_11": None}, "null"),
                          ({"_19": None}, "null"), ({"_20": None}, "null"), ({"_8": -1}, "stride"), ({"_10": -1}, "stride"),
                          ({"_12": -1}, "stride")):
        _refused("cign_block_boundary_fwd", _with(fwd, **change), match)
    lib = _lib.load_library(require_gpu=False)
    ws = lib.cign_block_boundary_bwd_workspace_bytes(4, 32)
    assert ws == 5 * 4 * 4 * 32
    assert lib.cign_block_boundary_bwd_workspace_bytes(10**6, 8192) == 5 * 4 * 1024 * 8192
    assert lib.cign_block_boundary_bwd_workspace_bytes(-1, 32) == lib.cign_block_boundary_bwd_workspace_bytes(1, 8193) == 0
    #      stream n D  xt wt ly gk g1  ld1 g2  ld2 u   ldu h   ldh a   lda
    bwd = (None, 4, 32, 0, 0, 1, 2, BIG, 32, BIG, 32, BIG, 32, BIG, 32, BIG, 32,
           # w1 b1 c w2 stats gu gh ga gw1 gb1 gc gw2 gb2 ws bytes
           BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, BIG, ws)
    for change, match in (({"_1": -1}, "negative row count"), ({"_2": 8193}, "1<=D<=8192"), ({"_3": 3}, "dtypes"),
                          ({"_7": None, "_9": None}, "null"), ({"_11": None}, "null"), ({"_13": None}, "null"),
                          ({"_15": None}, "null"), ({"_21": None}, "null"), ({"_8": -1}, "stride"), ({"_16": -1}, "stride"),
                          ({"_30": None}, "workspace"), ({"_31": ws - 1}, "workspace")):
        _refused("cign_block_boundary_bwd", _with(bwd, **change), match)
    lib.call("cign_block_boundary_fwd", *_with(fwd, _1=0))
    none = {f"_{i}": None for i in range(22, 30)}
    lib.call("cign_block_boundary_bwd", *_with(bwd, **none))  # no gradient asked for


def test_linear_xent_refusals():
    lib = _lib.load_library(require_gpu=False)
    size = lib.cign_linear_xent_workspace_bytes
    #      stream t n  V     D   x   ldx  w    ldw  b   bt label ignore loss lse ws   bytes
    fwd = (None, 0, 4, 5000, 64, BIG, 64, BIG, 64, BIG, 0, BIG, -100, BIG, BIG, BIG, 1 << 40)
    for change, match in (({"_1": 2}, "dtype"), ({"_2": -1}, "negative row count"), ({"_2": (1 << 23) + 1}, "rows"),
                          ({"_3": 0}, "1<=V"), ({"_3": (1 << 20) + 1}, "1<=V"), ({"_4": 0}, "1<=D"),
                          ({"_4": 65537}, "1<=D"), ({"_10": 1}, "bias dtype"), ({"_1": 1, "_10": 2}, "bias dtype"),
                          ({"_5": None}, "null"), ({"_7": None}, "null"), ({"_14": None}, "null"), ({"_13": None}, "null"),
                          ({"_11": None}, "null"), ({"_6": -1}, "stride"), ({"_8": -1}, "stride"),
                          ({"_16": size(0, 4, 5000, 64, BIG, 64, BIG, 64, 0) - 1}, "workspace"),
                          ({"_15": None}, "workspace")):
        _refused("cign_linear_xent_fwd", _with(fwd, **change), match)
    #      stream t n  V     D   x   ldx  w    ldw  b   bt label ignore lse gl   gs   gx   gw   gb   ws  bytes
    bwd = (None, 0, 4, 5000, 64, BIG, 64, BIG, 64, BIG, 0, BIG, -100, BIG, BIG, BIG, BIG, BIG, BIG, BIG, 1 << 40)
    for change, match in (({"_1": 2}, "dtype"), ({"_2": 0}, "no rows"), ({"_5": None}, "null"), ({"_13": None}, "null"),
                          ({"_14": None, "_15": None}, "null"), ({"_11": None}, "null"), ({"_8": -1}, "stride"),
                          ({"_20": size(0, 4, 5000, 64, BIG, 64, BIG, 64, 7) - 1}, "workspace"),
                          ({"_19": None}, "workspace")):
        _refused("cign_linear_xent_bwd", _with(bwd, **change), match)
    lib.call("cign_linear_xent_fwd", *_with(fwd, _2=0))
    lib.call("cign_linear_xent_bwd", *_with(bwd, _16=None, _17=None, _18=None))  # no gradient asked for
    assert size(0, 0, 5000, 64, BIG, 64, BIG, 64, 0) == size(2, 4, 5000, 64, BIG, 64, BIG, 64, 0) == 0
    assert size(0, 4, 5000, 64, BIG, 64, BIG, 64, 8) == 0
    # packed rows of x and weight only where the tiles cannot read them in place
    inside, odd, far = (size(1, 500, 5000, 64, BIG, ld, BIG + a, 64, 0) for ld, a in ((64, 0), (65, 2), (1 << 25, 0)))
    assert odd - inside >= 2 * 64 * (500 + 5000) and far - inside >= 2 * 64 * 500
    # the gradient of 2^20 classes by rows is held a piece at a time
    assert size(1, 8192, 1 << 20, 512, BIG, 512, BIG, 512, 7) < 8192 * (1 << 20)


def _arrays(sizes, dtypes, at=BIG):
    n = len(sizes)
    return ((C.c_void_p * n)(*[at + (i << 36) for i in range(n)]), (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*dtypes))


def test_grad_norm_refusals():
    lib = _lib.load_library(require_gpu=False)
    p, s, t = _arrays([5, 7], [0, 1])
    a = C.addressof
    ws = lib.cign_grad_norm_workspace_bytes(2, a(s))
    assert ws == 16
    clip = (None, 2, a(p), a(s), a(t), 1.0, a(p), BIG, BIG, ws)
    bad_s, bad_t = (C.c_int64 * 2)(5, -1), (C.c_int32 * 2)(0, 2)
    hole = (C.c_void_p * 2)(BIG, None)
    for change, match in (({"_1": -1}, "count"), ({"_2": None}, "null"), ({"_3": None}, "null"), ({"_4": None}, "null"),
                          ({"_3": a(bad_s)}, "negative size"), ({"_4": a(bad_t)}, "dtypes"), ({"_2": a(hole)}, "is null"),
                          ({"_6": None}, "null"), ({"_6": a(hole)}, "is null"), ({"_7": None}, "null"),
                          ({"_5": -1.0}, "max_norm"), ({"_5": math.nan}, "max_norm"), ({"_8": None}, "workspace"),
                          ({"_9": ws - 1}, "workspace")):
        _refused("cign_clip_grad_norm", _with(clip, **change), match)
    norm = (None, 2, a(p), a(s), a(t), BIG, BIG, ws)
    for change, match in (({"_1": -1}, "count"), ({"_5": None}, "null"), ({"_6": None}, "workspace"),
                          ({"_7": ws - 1}, "workspace")):
        _refused("cign_grad_norm", _with(norm, **change), match)
    many = (C.c_int64 * 3)(0, 1, 10**9)
    # chunks of 10^9 / 4096 values, to the next multiple of 2048
    assert lib.cign_grad_norm_workspace_bytes(3, a(many)) == 8 * (1 + -(-10**9 // (-(-(-(-(10**9 + 1) // 4096)) // 2048) * 2048)))
    few = (C.c_int64 * 2)(8192, 8193)  # chunks of at least 8192
    assert lib.cign_grad_norm_workspace_bytes(2, a(few)) == 8 * 3
    assert lib.cign_grad_norm_workspace_bytes(0, a(many)) == lib.cign_grad_norm_workspace_bytes(3, None) == 0


def test_functions_refuse_host_tensors():
    from cign_amd.fused_block_ops import fused_gated_residual_norm
    from cign_amd.grad_norm import clip_grad_norm, global_grad_norm
    from cign_amd.linear_cross_entropy import linear_cross_entropy

    x = torch.zeros(3, 8)
    for call in (lambda t: fused_gated_residual_norm(t, t), lambda t: linear_cross_entropy(t, t, torch.zeros(3).long()),
                 lambda t: global_grad_norm([t]), lambda t: clip_grad_norm([t], 1.0)):
        for bad in (x, x.bfloat16(), x.numpy(), None):
            with pytest.raises(TypeError, match="must be CUDA float32 or bfloat16"):
                call(bad)
    for call in (lambda: global_grad_norm([]), lambda: clip_grad_norm([], 1.0)):
        with pytest.raises(ValueError, match="empty"):
            call()


def test_operators_on_meta_tensors():
    """Shapes and types without a device, and the checks that a kernel's accesses rest on."""
    from cign_amd._rows import load_output_ops

    load_output_ops()
    ops = torch.ops.cign_amd
    m = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device="meta")
    hidden, y = ops.block_boundary(m(2, 3, 8), m(2, 3, 8), m(8), None, m(8), m(2, 3, 1), None, m(8), 1e-5, True)
    assert hidden.shape == y.shape == (2, 3, 8)
    *_, stats = ops.block_boundary_forward(m(2, 3, 8), m(2, 3, 8), None, None, None, None, None, None, 1e-5, False)
    assert stats.shape == (4, 6)
    grads = ops.block_boundary_backward(m(2, 3, 8), None, m(2, 3, 8), m(2, 3, 8), m(8), None, None, m(2, 3, 1), None,
                                        m(4, 6), torch.float32, True, 0b1111)
    assert [tuple(g.shape) for g in grads] == [(2, 3, 8), (2, 3, 8), (2, 3, 1), (8,)]
    for bad in (dict(residual=m(2, 3, 7)), dict(gate=m(2, 1, 8)), dict(w1=m(7)), dict(w1=m(8, dtype=torch.bfloat16))):
        a = dict(branch=m(2, 3, 8), residual=m(2, 3, 8), w1=None, b1=None, c=None, gate=None, w2=None, b2=None) | bad
        with pytest.raises((ValueError, TypeError)):
            ops.block_boundary(*a.values(), 1e-5, True)
    with pytest.raises(ValueError, match="no gate"):
        ops.block_boundary_backward(m(6, 8), None, m(6, 8), m(6, 8), None, None, None, None, None, m(4, 6),
                                    torch.float32, True, 4)
    labels = m(2, 3, dtype=torch.int64)
    loss, lse = ops.linear_xent(m(2, 3, 8), m(50, 8), labels, m(50), -100)
    assert loss.shape == lse.shape == (2, 3) and loss.dtype == lse.dtype == torch.float32
    grads = ops.linear_xent_backward(loss, None, m(2, 3, 8), m(50, 8), labels, m(50), lse, -100, True, True, True)
    assert [tuple(g.shape) for g in grads] == [(2, 3, 8), (50, 8), (50,)]
    for w, l, b in ((m(50, 7), labels, None), (m(50, 8, dtype=torch.bfloat16), labels, None),
                    (m(50, 8), m(2, 2, dtype=torch.int64), None), (m(50, 8), m(2, 3, dtype=torch.int32), None),
                    (m(50, 8), labels, m(49))):
        with pytest.raises((ValueError, TypeError)):
            ops.linear_xent(m(2, 3, 8), w, l, b, -100)
    with pytest.raises(ValueError, match="no bias"):
        ops.linear_xent_backward(loss, None, m(2, 3, 8), m(50, 8), labels, None, lse, -100, True, True, True)
    assert ops.global_grad_norm([m(3), m(4, 5)]).shape == ()
    assert ops.clip_grad_norm([m(3)], 1.0, [m(3)]).shape == ()
    for grads, out in (([m(3)], []), ([m(3)], [m(4)]), ([m(3)], [m(3, dtype=torch.bfloat16)])):
        with pytest.raises((ValueError, TypeError)):
            ops.clip_grad_norm(grads, 1.0, out)


def test_segments_of_split_products():
    """nt_gemm.h seg_a, seg_b: three parts a side, the six products above 2^-26,
    the smallest first."""
    seg = lambda code: [(code >> (4 * s)) & 0xF for s in range(6)]
    pairs = list(zip(seg(0x001102), seg(0x010120)))
    assert sorted(pairs) == sorted((i, j) for i in range(3) for j in range(3) if i + j <= 2)
    assert [i + j for i, j in pairs] == sorted((i + j for i, j in pairs), reverse=True)


@pytest.mark.parametrize("ta,tb", [(1, 1), (3, 5), (8, 8), (125, 32), (7, 9), (1, 100), (100, 1)])
def test_every_tile_has_one_workgroup(ta, tb):
    """nt_gemm.h tile_of: workgroups 0..ta*tb-1 to all tiles, each once."""
    seen = set()
    total = ta * tb
    for wg in range(total):
        x, k = wg & 7, wg >> 3
        each, more = total >> 3, total & 7
        t = x * each + min(x, more) + k
        band, rest = divmod(t, 8 * ta)
        wide = min(8, tb - band * 8)
        seen.add((rest // wide, band * 8 + rest % wide))
    assert seen == {(a, b) for a in range(ta) for b in range(tb)}
