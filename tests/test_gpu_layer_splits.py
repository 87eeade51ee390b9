"""Products of yolo_amd.layers.linear whose reduction is cut into slices, on every tile that can be: forward, dX and dW, with
operands in one part and in two.  Which tile a size takes, and whether it is split, is asked of the library first."""
import ctypes

import pytest
import torch

from layer_reference import EPS32, TINY, U, act64, assert_within, rounded, slope64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _choices(m, n, k, dtype, act, backward):
    """[(tile, steps ahead, split?)] of y, or of dX and dW, for operands without gaps."""
    from yolo_amd import _lib
    code = {BF16: _lib.TYPE_BF16, F16: _lib.TYPE_F16}[dtype]
    if not backward:
        f, c = _lib.LinearDesc(), _lib.LinearChoice()
        f.x, f.weight, f.y, f.m, f.n, f.k, f.ldx, f.ldw, f.ldy = 256, 256, 256, m, n, k, k, k, n
        f.type, f.activation = code, _lib.ACT_CODES[act]
        _lib.check(_lib.lib.yolo_amd_linear_query(ctypes.byref(f), ctypes.byref(c)), "query")
        return [(c.bm, c.steps_ahead, c.k_slices > 1)]
    b, c = _lib.LinearBackwardDesc(), (_lib.LinearChoice(), _lib.LinearChoice())
    b.dy, b.x, b.weight, b.pre, b.dx, b.dweight = 256, 256, 256, 256, 256, 256
    b.m, b.n, b.k, b.lddy, b.ldx, b.ldw = m, n, k, n, k, k
    b.type, b.activation, b.pre_f32 = code, _lib.ACT_CODES[act], 1
    _lib.check(_lib.lib.yolo_amd_linear_backward_query(ctypes.byref(b), ctypes.byref(c[0]), ctypes.byref(c[1])), "query")
    return [(v.bm, v.steps_ahead, v.k_slices > 1) for v in c]


def _band(size):
    return torch.cat([torch.arange(min(size, 40)), torch.arange(max(0, size - 140), size)]).cuda()


FORWARD = [((41, 40, 1174), None, (64, 4)), ((38, 41, 1175), "gelu", (64, 4)), ((143, 85, 1073), "gelu", (64, 4)),
           ((8621, 8, 4664), "silu", (128, 4)), ((8621, 5, 4666), None, (128, 4)), ((8992, 8, 4608), None, (128, 2)),
           ((8965, 5, 6113), "gelu_tanh", (128, 2)), ((8216, 137, 6320), None, (256, 2)), ((2943, 1764, 3687), "gelu", (256, 2)),
           ((8216, 136, 6320), "leaky", (256, 2))]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,act,tile", FORWARD)
def test_linear_forward_split(shape, act, tile, dtype):
    from yolo_amd.layers import linear
    m, n, k = shape
    assert _choices(m, n, k, dtype, act, False) == [tile + (True,)]
    g = torch.Generator("cuda").manual_seed(m + n + k)
    x, w, b, r = (_rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype), _rand(g, n, dtype=dtype),
                  _rand(g, m, n, dtype=dtype))
    y = linear(x, w, b, activation=act, residual=r)
    for rows, cols in ((_band(m), torch.arange(n).cuda()), (torch.arange(m).cuda(), _band(n))):
        x64, w64, b64, r64 = x[rows].double(), w[cols].double(), b[cols].double(), r[rows][:, cols].double()
        p, mag = x64 @ w64.t() + b64, x64.abs() @ w64.abs().t() + b64.abs()
        a = act64(p, act)
        # |act'| <= 1.13; GELU's 1 + erf cancels: |p| 2^-22 absolute; one more addition for the residual
        e = 1.13 * (k + 4) * 2.0 ** -23 * mag + (EPS32 * a.abs() + 2.0 ** -22 * p.abs() if act else 0) + 2.0 ** -23 * (a.abs() + r64.abs())
        assert_within(y[rows][:, cols], (a + r64).cpu(), rounded(a + r64, e, dtype).cpu(), f"{shape} {act}")


# (m, n, k), activation, (tile, steps ahead) and split of dX, the same of dW
BACKWARD = [((8, 1120, 8), None, (64, 4, True), (64, 4, False)), ((1096, 8, 16), None, (64, 4, False), (64, 4, True)),
            ((16, 4096, 1024), "gelu", (64, 4, True), None), ((333, 4104, 760), "gelu", None, None), ((333, 4101, 761), "silu", None, None),
            ((686, 5, 6), "silu", (64, 4, False), (64, 4, True)),
            ((8864, 4920, 8), None, (128, 4, True), None), ((8604, 2925, 5), "silu", (128, 4, True), None),
            ((8944, 5984, 8), None, (128, 2, True), None), ((8626, 4464, 5), "gelu", (128, 2, True), None),
            ((152, 7432, 8968), None, (256, 2, True), None), ((160, 4520, 5536), "gelu", (256, 2, True), None),
            ((8334, 3125, 143), "gelu_tanh", (256, 2, True), None), ((2312, 5920, 3064), "gelu", None, None),
            ((4592, 8, 8664), None, None, (128, 4, True)), ((5088, 8368, 8), "silu", None, (128, 4, True)),
            ((2098, 8748, 5), "gelu", None, (128, 4, True)), ((8184, 8568, 16), None, None, (128, 2, True)),
            ((2660, 8968, 5), "silu", None, (128, 2, True)), ((3296, 472, 8208), None, None, (256, 2, True)),
            ((4925, 134, 5736), "gelu", None, (256, 2, True)), ((3280, 8640, 144), "gelu", None, (256, 2, True))]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,act,dx_tile,dw_tile", BACKWARD)
def test_linear_backward_split(shape, act, dx_tile, dw_tile, dtype):
    """Bounds: the incoming gradient in one part is exact without an activation; else d(loss)/dp is off by its slope (0.8 times
    the bound of p, and EPS32) and by the second part's rounding, and a product of r terms adds 2 r of them."""
    from yolo_amd.layers import linear
    m, n, k = shape
    took = _choices(m, n, k, dtype, act, True)
    assert any(split for _, _, split in took)
    for want, c in zip((dx_tile, dw_tile), took):
        assert want is None or c == want
    g = torch.Generator("cuda").manual_seed(m + n + k)
    x, w = _rand(g, m, k, dtype=dtype).requires_grad_(), _rand(g, n, k, scale=k ** -0.5, dtype=dtype).requires_grad_()
    dy = _rand(g, m, n, dtype=dtype)
    dx, dw = torch.autograd.grad(linear(x, w, activation=act), (x, w), dy)
    x64, w64, dp = x.detach().double(), w.detach().double(), dy.double()
    off, parts = torch.zeros_like(dp), 1
    if act:
        p, ep = x64 @ w64.t(), (k + 4) * 2.0 ** -23 * (x64.abs() @ w64.abs().t())
        s = slope64(p, act)
        off = dp.abs() * (0.8 * ep + EPS32 * (1 + s.abs())) + 2.0 ** -23 * (dp * s).abs()
        dp = dp * s
        off += U[dtype] ** 2 * (dp.abs() + off) + (float(dp.abs().max()) * 2.0 ** -39 if dtype is F16 else TINY[dtype])
        parts = 2
    rows, cols = _band(m), _band(n)
    for got, a, e, b, terms in ((dx[rows], dp[rows], off[rows], w64, n), (dw[cols], dp[:, cols].t(), off[:, cols].t(), x64, m)):
        want = a @ b
        bound = e @ b.abs() + 1.01 * (parts * terms + 4) * 2.0 ** -23 * (a.abs() @ b.abs())
        assert_within(got, want.cpu(), rounded(want, bound, dtype).cpu(), f"{shape} {act}")
