"""Gradients of yolo_amd.layers.linear held to what a computation in 32 bits with one rounding at its end gives: neither
the pre-activation nor its gradient loses bits on the way that the caller's types would have kept."""
import ctypes

import pytest
import torch

import layer_reference as ref
from layer_reference import EPS32, TINY, U, assert_within, d, rounded, slope64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# few rows, whole tiles, ragged ends and odd rows, split reductions in the forward product
KEPT = [(1, 40, 64), (3, 984, 64), (5, 114, 4680), (64, 128, 64), (130, 75, 261), (333, 761, 4104), (200, 1030, 520), (1990, 2048, 264)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", KEPT)
def test_linear_slopes_are_of_the_unrounded_preactivation(m, n, k, dtype):
    """The bias gradient sums dy * act'(p) without any rounding to x's type; the slope is off by |act''| times what the fp32
    sum p is off (its bound, 0.8 for all three) and EPS32 of its own size."""
    from yolo_amd.layers import linear
    g = torch.Generator().manual_seed(m + 3 * n + 5 * k)
    x, w = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype)
    for act in ("gelu", "gelu_tanh", "silu"):
        b = _rand(g, n, scale=0.3).requires_grad_()
        dy = _rand(g, m, n, dtype=dtype)
        db, = torch.autograd.grad(linear(x, w, b, activation=act), b, dy)
        _, _, p, ep = ref.linear_ref(x, w, b, None, act, dtype)
        s, dy = slope64(p, act), d(dy)
        edp = dy.abs() * (0.8 * ep + EPS32 * (1 + s.abs())) + 2.0 ** -23 * (dy * s).abs()
        want = (dy * s).sum(0)
        assert_within(db, want, rounded(want, edp.sum(0) + 512 * 2.0 ** -24 * (dy * s).abs().sum(0), F32), f"db {act}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", KEPT)
def test_linear_entry_keeps_either_preactivation(m, n, k, dtype):
    """At the C entry: in fp32 as summed, or rounded to x's type; either way nothing behind it is written, and the
    backward entry reads what it is told that it is."""
    from yolo_amd import _lib
    from yolo_amd._lib import lib
    g = torch.Generator().manual_seed(m + n + k)
    x, w, b = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype), _rand(g, n, dtype=dtype)
    dy = _rand(g, m, n, dtype=dtype)
    _, _, p, ep = ref.linear_ref(x, w, b, None, None, dtype)
    stream, code = _lib.current_stream_ptr(), {BF16: _lib.TYPE_BF16, F16: _lib.TYPE_F16}[dtype]

    def scratch(desc, nbytes):
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
        desc.workspace, desc.workspace_bytes = ws.data_ptr(), nbytes
        return ws
    for f32 in (0, 1):
        kept = torch.full((m * n + 16,), 7.0, dtype=F32 if f32 else dtype, device="cuda")
        y, db = torch.empty(m, n, dtype=dtype, device="cuda"), torch.empty(n, device="cuda")
        f = _lib.LinearDesc()
        f.x, f.weight, f.bias, f.y, f.pre = x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), kept.data_ptr()
        f.m, f.n, f.k, f.ldx, f.ldw, f.ldy, f.type, f.activation, f.pre_f32 = m, n, k, k, k, n, code, _lib.ACT_CODES["silu"], f32
        ws = scratch(f, lib.yolo_amd_linear_workspace_bytes(ctypes.byref(f)))          # noqa: F841
        _lib.check(lib.yolo_amd_linear_forward(ctypes.byref(f), stream), "forward")
        assert_within(kept[:m * n].reshape(m, n), p, rounded(p, ep, kept.dtype), "pre")
        assert (kept[m * n:] == 7).all()
        r = _lib.LinearBackwardDesc()
        r.dy, r.pre, r.dbias, r.m, r.n, r.k, r.lddy = dy.data_ptr(), kept.data_ptr(), db.data_ptr(), m, n, k, n
        r.type, r.dbias_f32, r.activation, r.pre_f32 = code, 1, _lib.ACT_CODES["silu"], f32
        ws = scratch(r, lib.yolo_amd_linear_backward_workspace_bytes(ctypes.byref(r)))
        _lib.check(lib.yolo_amd_linear_backward(ctypes.byref(r), stream), "backward")
        own = d(kept[:m * n].reshape(m, n))                  # the slope of what was kept
        want = (d(dy) * slope64(own, "silu")).sum(0)
        assert_within(db, want, rounded(want, (EPS32 * 2 + 512 * 2.0 ** -24) * d(dy).abs().sum(0) * 1.1, F32), "db")


def _gradients(x, w, p, ep, dy, kind, bias_dtype):
    """((dx, bound), (dw, bound), (db, bound)) with p kept in 32 bits (ep: its bound) and d(loss)/dp given to the products in
    two parts of x's type t.

    Bounds.  The slope is off by |act''| ep <= 0.8 ep and EPS32 of its own size; leaky and relu take the other slope only
    where the sum's own rounding can change p's sign.  The first part is off by U[t] relative, the second part, which
    holds the rest, by U[t] of that: U[t]^2 in all.  Below their normal range the parts of bf16 are off by TINY; those of fp16
    are scaled by a power of two that puts the largest of them at 2^14 or above, so that their steps of 2^-24 are at most
    2^-38 of it, and a rounding half of that.  A product of r terms in two parts adds 2 r of them."""
    t = x.dtype
    x, w, dy = d(x), d(w), d(dy)
    s = slope64(p, kind)
    if kind is None:
        es = torch.zeros_like(p)
    elif kind in ("leaky", "relu"):
        es = (p.abs() <= ep).to(p.dtype) + EPS32 * s
    else:
        es = 0.8 * ep + EPS32 * (1 + s.abs())
    dp = dy * s
    edp = dy.abs() * es + 2.0 ** -23 * dp.abs()
    largest = float(dp.abs().max()) if dp.numel() else 0.0
    eop = edp + U[t] ** 2 * (dp.abs() + edp) + (largest * 2.0 ** -39 if t is F16 else TINY[t])
    m, n = dp.shape
    dx, dw, db = dp @ w, dp.t() @ x, dp.sum(0)
    edx = eop @ w.abs() + 1.01 * (2 * n + 4) * 2.0 ** -23 * (dp.abs() @ w.abs())
    edw = eop.t() @ x.abs() + 1.01 * (2 * m + 4) * 2.0 ** -23 * (dp.abs().t() @ x.abs())
    edb = edp.sum(0) + 512 * 2.0 ** -24 * dp.abs().sum(0)
    return ((dx, rounded(dx, edx, t)), (dw, rounded(dw, edw, t)), (db, rounded(db, edb, bias_dtype)))


def _check(x, w, b, act, dy, out):
    from yolo_amd.layers import linear
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    got = torch.autograd.grad(linear(*leaves, activation=act, out_dtype=out), leaves, dy)
    _, _, p, ep = ref.linear_ref(x, w, b, None, act, out)
    for name, a, (want, bound) in zip(("dx", "dw", "db"), got, _gradients(x, w, p, ep, dy, act, b.dtype)):
        # from half a step past the type's largest number on, a value rounds to an infinity
        end = (2 - U[a.dtype]) * 2.0 ** (15 if a.dtype is F16 else 127)
        past, may = want.abs() - bound > end, (want.abs() + bound >= end) & torch.isinf(d(a))
        assert torch.equal(d(a)[past], want[past].sign() * float("inf")), f"{name} {act}"
        assert_within(torch.where(past | may, 0.0, d(a)), torch.where(past | may, 0.0, want), bound, f"{name} {act}")


# few rows, whole tiles, ragged ends and odd rows of every tile, a split reduction in dX and in dW
SHAPES = [(1, 40, 64), (3, 984, 64), (64, 128, 64), (130, 75, 261), (333, 136, 1021), (200, 1030, 520), (16, 4096, 1024), (2500, 40, 48),
          (1990, 2048, 264)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_gradients_lose_no_bits(m, n, k, dtype):
    g = torch.Generator().manual_seed(m + 3 * n + 5 * k)
    x, w = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype)
    b = _rand(g, n, scale=0.3)
    for act, out in ((None, F32), ("gelu", dtype), ("gelu_tanh", F32), ("silu", dtype), ("leaky", dtype), ("relu", dtype)):
        _check(x, w, b, act, _rand(g, m, n, dtype=out), out)


@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("size,of_x,of_w", [(1e-9, 1e3, 1e3), (1e6, 1e-2, 1e-4), (1e-30, 1e4, 1e4)])
def test_linear_gradients_past_the_range_of_fp16(size, of_x, of_w, act):
    """fp16 operands with an fp32 result: its gradient may lie where fp16 has no numbers (a mean loss over wide scores, a
    scaled loss), while the gradients of x and weight do not."""
    g = torch.Generator().manual_seed(5)
    m, n, k = 70, 520, 64
    x, w, b = _rand(g, m, k, scale=of_x, dtype=F16), _rand(g, n, k, scale=of_w, dtype=F16), _rand(g, n)
    dy = _rand(g, m, n, scale=size)
    dy[3] = 0
    dy[5] *= 2.0 ** -20
    _check(x, w, b, act, dy, F32)


def test_linear_gradients_of_zeros_and_infinities():
    """An incoming gradient of zeros gives zeros; an infinity or NaN in one row leaves the gradients of the other rows as they
    would be without it."""
    from yolo_amd.layers import linear
    g = torch.Generator().manual_seed(6)
    for dtype in (F16, BF16):
        x, w = _rand(g, 70, 64, dtype=dtype).requires_grad_(), _rand(g, 136, 64, dtype=dtype).requires_grad_()
        y = linear(x, w, activation="silu", out_dtype=F32)
        zeros = torch.autograd.grad(y, (x, w), torch.zeros(70, 136, device="cuda"), retain_graph=True)
        assert not zeros[0].any() and not zeros[1].any()
        dy = _rand(g, 70, 136, scale=1e-3)
        clean, = torch.autograd.grad(y, x, dy, retain_graph=True)
        dy[4, 7], dy[9, 100] = float("inf"), float("nan")
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        keep = [i for i in range(70) if i not in (4, 9)]
        assert torch.equal(dx[keep], clean[keep])
        assert not torch.isfinite(dx[[4, 9]]).any() and not torch.isfinite(dw[7]).any() and torch.isnan(dw[100]).all()


def test_linear_gradients_of_the_largest_values():
    """Slopes above one at the type's largest gradients."""
    for dtype, size, weight in ((F16, 65504.0, 2.0 ** -12), (BF16, 2.0 ** 127, 2.0 ** -40)):
        x = torch.full((5, 8), 0.5, dtype=dtype).cuda()
        w = torch.full((24, 8), weight, dtype=dtype).cuda()
        b = torch.full((24,), 1.4).cuda()                     # gelu's slope is 1.13 there
        _check(x, w, b, "gelu", torch.full((5, 24), size, dtype=dtype).cuda(), dtype)


def test_linear_gradients_offsets_past_32_bits():
    """Pre-activations, their gradient and its second part of 2.4e9 values each: the last rows are where they belong."""
    from yolo_amd.layers import linear
    m, n, k = 2 ** 25 + 77, 72, 16
    g = torch.Generator().manual_seed(12)
    x, dy = (torch.full((m, c), v, dtype=BF16, device="cuda") for c, v in ((k, 0.5), (n, 0.25)))
    x[-300:], dy[-300:] = _rand(g, 300, k, dtype=BF16), _rand(g, 300, n, dtype=BF16)
    w = _rand(g, n, k, dtype=BF16)
    x.requires_grad_()
    dx, = torch.autograd.grad(linear(x, w, activation="gelu"), x, dy)
    rows = torch.cat([torch.arange(5), torch.arange(m - 300, m)]).cuda()
    _, _, p, ep = ref.linear_ref(x[rows], w, None, None, "gelu", BF16)
    assert_within(dx[rows], *_gradients(x[rows], w, p, ep, dy[rows], "gelu", F32)[0], "dx")
    assert torch.equal(dx[m - 400], dx[0])


def test_linear_gradients_repeat_on_two_streams_and_in_a_graph():
    """fp16 with its scale, on two streams at once and replayed from a graph with other gradients, bit for bit."""
    from yolo_amd.layers import linear
    g = torch.Generator().manual_seed(13)
    w = _rand(g, 136, 72, dtype=F16).requires_grad_()
    xs = [_rand(g, m, 72, dtype=F16).requires_grad_() for m in (90, 700)]
    dys = [_rand(g, m, 136, scale=s) for m, s in ((90, 1e-9), (700, 1e6))]

    def step(x, dy):
        return torch.autograd.grad(linear(x, w, activation="silu", out_dtype=F32), (x, w), dy)
    want = [step(x, dy) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, x, dy in zip(streams, xs, dys):
            with torch.cuda.stream(st):
                got.append(step(x, dy))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for u, v in zip(got, want) for a, b in zip(u, v))
    x, dy = xs[0].detach().clone(), dys[0].clone()
    graph = torch.cuda.CUDAGraph()
    leaf = w.detach().clone()

    def captured():
        a, b = x.detach().requires_grad_(), leaf.detach().requires_grad_()
        return torch.autograd.grad(linear(a, b, activation="silu", out_dtype=F32), (a, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = captured()
    for size in (1.0, 1e-12, 3e7, 0.0):
        dy.copy_(dys[0] / 1e-9 * size)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, captured()))
