"""yolo_amd.layers on the GPU against 64-bit definitions (layer_reference.py): products, epilogues and gradients of
`linear`, norms, gates and gradients of `block_norm`, at the sizes, strides and masks where they can go wrong."""
import itertools

import pytest
import torch

import layer_reference as ref
from layer_reference import assert_within, rounded

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(g, *shape, scale=1.0, dtype=F32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _choice(x, w, **kw):
    """The kernel the library picks for x @ w.T."""
    import ctypes
    from yolo_amd import _lib
    dsc = _lib.LinearDesc()
    y = torch.empty(x.shape[0], w.shape[0], dtype=x.dtype, device=x.device)
    dsc.x, dsc.weight, dsc.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
    dsc.m, dsc.n, dsc.k = x.shape[0], w.shape[0], w.shape[1]
    dsc.ldx, dsc.ldw, dsc.ldy = x.stride(0), w.stride(0), w.shape[0]
    dsc.type = {BF16: _lib.TYPE_BF16, F16: _lib.TYPE_F16}[x.dtype]
    c = _lib.LinearChoice()
    _lib.check(_lib.lib.yolo_amd_linear_query(ctypes.byref(dsc), ctypes.byref(c)), "query")
    return _lib.LINEAR_KERNEL_NAMES[c.kernel], c


# ------------------------------------------------------------------ linear, forward
SHAPES = [  # (m, n, k)
    (1, 1, 1), (1, 16, 8), (1, 1000, 1024), (2, 40, 72), (15, 17, 129), (16, 256, 512), (17, 33, 64), (32, 264, 1000),
    (33, 64, 64), (64, 512, 448), (65, 130, 65), (128, 128, 128), (129, 127, 200), (255, 255, 72), (300, 1030, 520),
    (513, 257, 1021), (1024, 96, 2304), (40, 128, 8192),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_forward(m, n, k, dtype):
    from yolo_amd.layers import linear
    g = _gen(m * 7 + n * 3 + k)
    x, w = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype)
    b, r = _rand(g, n, scale=0.3, dtype=dtype), _rand(g, m, n, dtype=dtype)
    for act, bias, res, out in ((None, None, None, dtype), ("leaky", b, r, dtype), ("gelu", b.float(), None, F32),
                                ("silu", None, r.float(), dtype)):
        y = linear(x, w, bias, activation=act, residual=res, out_dtype=out)
        want, bound, _, _ = ref.linear_ref(x, w, bias, res, act, out)
        assert y.dtype == out
        assert_within(y, want, bound, f"{m}x{n}x{k} {act}")


@pytest.mark.parametrize("act", [None, "leaky", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m", [5, 70])
def test_linear_activations(m, act):
    from yolo_amd.layers import linear
    g = _gen(3)
    x, w, b = _rand(g, m, 64, scale=3, dtype=F16), _rand(g, 72, 64, scale=0.4, dtype=F16), _rand(g, 72, dtype=F16)
    for out in (F16, F32):
        y = linear(x, w, b, activation=act, out_dtype=out)
        want, bound, _, _ = ref.linear_ref(x, w, b, None, act, out)
        assert_within(y, want, bound, str(act))


def test_linear_activation_far_out():
    """Pre-activations far into both tails: no overflow turns a finite result into NaN."""
    from yolo_amd.layers import linear
    v = torch.tensor([-3e38, -1e30, -1e5, -200.0, -90.0, -30.0, 0.0, 30.0, 200.0, 1e5, 1e30, 3e38], device="cuda")
    x = v.to(BF16).reshape(-1, 1)
    w = torch.ones(1, 1, dtype=BF16, device="cuda")
    for act in ("leaky", "relu", "gelu", "silu"):
        y = linear(x, w, activation=act, out_dtype=F32).double().cpu()[:, 0]
        want = ref.act64(x.double().cpu()[:, 0], act)
        assert torch.isfinite(y).all(), act
        assert torch.allclose(y, want, rtol=1e-5, atol=1e-6), act
    y = linear(x, w, activation="gelu_tanh", out_dtype=F32).double().cpu()[:, 0]
    assert not torch.isnan(y).any()


@pytest.mark.parametrize("m", [3, 200])
def test_linear_reads_views_and_nothing_beyond_them(m):
    """Row views of wider tensors whose other columns and rows hold NaN: none of it reaches the result."""
    from yolo_amd.layers import linear
    g = _gen(9)
    for k, pad, off in ((64, 16, 0), (64, 16, 8), (60, 20, 0), (61, 3, 1), (200, 8, 4)):
        wide_x = torch.full((m + 4, k + pad + off), float("nan"), dtype=BF16, device="cuda")
        wide_w = torch.full((50 + 4, k + pad + off), float("nan"), dtype=BF16, device="cuda")
        x, w = wide_x[2:2 + m, off:off + k], wide_w[2:52, off:off + k]
        x.copy_(_rand(g, m, k, dtype=BF16))
        w.copy_(_rand(g, 50, k, scale=k ** -0.5, dtype=BF16))
        y = linear(x, w)
        want, bound, _, _ = ref.linear_ref(x, w, None, None, None, BF16)
        assert_within(y, want, bound, f"k={k} pad={pad} off={off}")
    base = _rand(g, 64, m, dtype=BF16)                       # a transposed operand is copied
    y = linear(base.t(), w[:, :64].contiguous())
    want, bound, _, _ = ref.linear_ref(base.t(), w[:, :64], None, None, None, BF16)
    assert_within(y, want, bound, "transposed x")
    x3 = _rand(g, 4, 6, 5, 64, dtype=BF16)
    wt = _rand(g, 24, 64, dtype=BF16)
    y = linear(x3[:, 1:3], wt, residual=_rand(g, 1, 1, 1, 24, dtype=BF16).expand(4, 2, 5, 24))
    assert y.shape == (4, 2, 5, 24)


def test_linear_last_token_is_read_in_place():
    """x[:, -1:] of a (batch, tokens, channels) tensor is rows at one stride: no copy."""
    from yolo_amd.layers import _rows, linear
    g = _gen(91)
    x, w = _rand(g, 6, 50, 64, dtype=BF16), _rand(g, 40, 64, dtype=BF16)
    for view in (x[:, -1:], x[:, 7], x[2:3, :, :], x[:, -1:].transpose(0, 1), x[::2, 3:4]):
        assert _rows(view)[0].data_ptr() == view.data_ptr()
        want, bound, _, _ = ref.linear_ref(view.reshape(-1, 64), w, None, None, None, BF16)
        assert_within(linear(view, w).reshape(-1, 40), want, bound, str(tuple(view.shape)))
    far = torch.empty(20, 1 << 23, dtype=BF16, device="cuda")[:, 5:69]        # rows 16 MiB apart
    far.copy_(_rand(g, 20, 64))
    for rows in (far, far[:1]):
        want, bound, _, _ = ref.linear_ref(rows, w, None, None, None, BF16)
        assert_within(linear(rows, w), want, bound, "far apart")
    odd = x[:, :3]                                           # three of fifty tokens each: copied
    want, bound, _, _ = ref.linear_ref(odd.reshape(-1, 64), w, None, None, None, BF16)
    assert_within(linear(odd, w).reshape(-1, 40), want, bound, "copied")


@pytest.mark.parametrize("m,n,k", [(3, 40, 64), (200, 41, 72), (64, 520, 8192), (300, 1000, 100)])
def test_linear_residual_in_place(m, n, k):
    """At the C entry y may be the residual itself."""
    import ctypes
    from yolo_amd import _lib
    from yolo_amd._lib import lib
    g = _gen(92)
    x, w, r = _rand(g, m, k, dtype=BF16), _rand(g, n, k, scale=k ** -0.5, dtype=BF16), _rand(g, m, n, dtype=BF16)
    y = r.clone()
    d = _lib.LinearDesc()
    d.x, d.weight, d.residual, d.y = x.data_ptr(), w.data_ptr(), y.data_ptr(), y.data_ptr()
    d.m, d.n, d.k, d.ldx, d.ldw, d.ldr, d.ldy, d.type = m, n, k, k, k, n, n, _lib.TYPE_BF16
    need = lib.yolo_amd_linear_workspace_bytes(ctypes.byref(d))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    _lib.check(lib.yolo_amd_linear_forward(ctypes.byref(d), _lib.current_stream_ptr()), "linear")
    want, bound, _, _ = ref.linear_ref(x, w, None, r, None, BF16)
    assert_within(y, want, bound, "in place")


@pytest.mark.parametrize("m", [4, 150])
def test_linear_nan_and_inf_stay_in_their_row(m):
    from yolo_amd.layers import linear
    g = _gen(10)
    x, w = _rand(g, m, 96, dtype=BF16), _rand(g, 40, 96, dtype=BF16)
    clean = linear(x, w)
    x[1, 5], x[3, 7] = float("nan"), float("inf")
    y = linear(x, w)
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any()
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("act", ["leaky", "relu", "gelu", "gelu_tanh", "silu"])
def test_linear_slopes_past_the_type(act):
    """Pre-activations beyond fp16's range, with an fp32 result: kept as infinities, where every slope has its limit."""
    from yolo_amd.layers import linear
    x = torch.full((3, 8), 200.0, dtype=F16, device="cuda")
    w = torch.stack([torch.full((8,), 200.0), torch.full((8,), -200.0), torch.full((8,), 100.0)]).to(F16).cuda()
    w[2, :4] *= -1                                          # 320000, -320000, 0
    b = torch.zeros(3, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = linear(x, w, b, activation=act, out_dtype=F32)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.ones_like(y))
    low, zero = (0.1, 0.1) if act == "leaky" else (0.0, 0.0 if act == "relu" else 0.5)
    # rows of three: sums of at most three roundings of a slope to fp16
    want = torch.tensor([1.0, low, zero], device="cuda")
    torch.testing.assert_close(db, 3 * want, rtol=2.0 ** -22, atol=2.0 ** -22)
    torch.testing.assert_close(dw.float(), 3 * 200 * want.to(F16).float()[:, None].expand(3, 8), rtol=2.0 ** -10, atol=1e-6)
    assert torch.isfinite(dx).all()
    assert torch.equal(y[:, 0].detach(), torch.full((3,), 320000.0, device="cuda"))


def test_linear_empty():
    from yolo_amd.layers import linear
    g = _gen(11)
    w, b = _rand(g, 24, 16, dtype=BF16), _rand(g, 24, dtype=BF16)
    assert linear(torch.empty(0, 16, dtype=BF16, device="cuda"), w, b).shape == (0, 24)
    assert linear(torch.empty(5, 16, dtype=BF16, device="cuda"), w[:0], b[:0]).shape == (5, 0)
    for m in (5, 70):                                       # a sum over nothing: bias and residual alone
        x0 = torch.empty(m, 0, dtype=BF16, device="cuda")
        r = _rand(g, m, 24, dtype=BF16)
        y = linear(x0, w[:, :0], b, activation="relu", residual=r)
        want = torch.relu(b.float()) + r.float()
        assert torch.equal(y, want.to(BF16))
    xs = [t.requires_grad_() for t in (torch.empty(0, 16, dtype=BF16, device="cuda"), w.clone(), b.clone())]
    dx, dw, db = torch.autograd.grad(linear(*xs, activation="silu"), xs, torch.empty(0, 24, dtype=BF16, device="cuda"))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    xs = [torch.zeros(3, 0, dtype=BF16, device="cuda").requires_grad_(), w[:, :0].clone().requires_grad_(), b.clone().requires_grad_()]
    dy = _rand(g, 3, 24, dtype=BF16)
    dx, dw, db = torch.autograd.grad(linear(*xs), xs, dy)
    assert dx.shape == (3, 0) and dw.shape == (24, 0)
    assert_within(db, dy.double().sum(0).cpu(), rounded(dy.double().sum(0).cpu(), 1e-6 * dy.double().abs().sum(0).cpu(), BF16), "db")


def test_linear_offsets_past_32_bits():
    from yolo_amd.layers import linear
    m, k = 2 ** 25 + 77, 72                                  # x holds 2.4e9 elements
    x = torch.empty(m, k, dtype=BF16, device="cuda").fill_(0.5)
    g = _gen(12)
    tail = _rand(g, 300, k, dtype=BF16)
    x[-300:] = tail
    w = _rand(g, 72, k, dtype=BF16)
    y = linear(x, w)                                         # and so does y
    want, bound, _, _ = ref.linear_ref(tail, w, None, None, None, BF16)
    assert_within(y[-300:], want, bound, "last rows")
    want, bound, _, _ = ref.linear_ref(x[:300], w, None, None, None, BF16)
    assert_within(y[:300], want, bound, "first rows")
    assert torch.equal(y[5000], y[m - 400])


def _band_check(x, w, b, r, y, act, dtype):
    """A band of rows and a band of columns of y, both with the ragged edge: the 64-bit product of all is slow here."""
    m, n = y.shape
    rows = torch.cat([torch.arange(0, min(m, 40)), torch.arange(max(0, m - 300), m)]).cuda()
    want, bound, _, _ = ref.linear_ref(x[rows], w, b, r[rows], act, dtype)
    assert_within(y[rows], want, bound, "rows")
    cols = torch.cat([torch.arange(0, min(n, 40)), torch.arange(max(0, n - 300), n)]).cuda()
    want, bound, _, _ = ref.linear_ref(x, w[cols], b[cols], r[:, cols], act, dtype)
    assert_within(y[:, cols], want, bound, "columns")


# (m, n, k), and the tile and split the library takes for it: every kernel of its choice, whole and ragged
TILES = [((4096, 4096, 2048), 256, 1, 2), ((1266, 6976, 4624), 256, 1, 2), ((4090, 4093, 2051), 256, 1, 2),
         ((2048, 4096, 256), 128, 1, 2), ((1990, 4072, 264), 128, 1, 2), ((1990, 4070, 265), 128, 1, 2),
         ((2048, 2048, 1024), 128, 1, 4), ((1999, 2024, 1096), 128, 1, 4), ((2048, 1024, 8192), 128, 2, 4),
         ((1024, 1024, 256), 64, 1, 4), ((333, 760, 200), 64, 1, 4), ((333, 759, 200), 64, 1, 4),
         ((333, 760, 4104), 64, 3, 4), ((333, 761, 4104), 64, 3, 4), ((1100, 1000, 1000), 64, 1, 4)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,bm,slices,ahead", TILES)
def test_linear_tiles(shape, bm, slices, ahead, dtype):
    from yolo_amd.layers import linear
    m, n, k = shape
    g = _gen(m + n + k)
    x, w, b = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype), _rand(g, n, dtype=dtype)
    r = _rand(g, m, n, dtype=dtype)
    c = _choice(x, w)[1]
    assert (c.bm, c.k_slices > 1, c.steps_ahead) == (bm, slices > 1, ahead)
    _band_check(x, w, b, r, linear(x, w, b, activation="gelu_tanh", residual=r), "gelu_tanh", dtype)


# (m, n, k), rows and columns of y per workgroup, and whether K is split
ROWS = [((1, 307, 40), 16, 16, False), ((11, 130, 2152), 16, 16, False), ((5, 114, 4680), 16, 16, True),
        ((7, 41, 11753), 16, 16, True), ((9, 15112, 72), 16, 32, False), ((7, 9080, 2544), 16, 32, False),
        ((13, 19760, 64), 16, 64, False), ((31, 132, 72), 32, 16, False),
        ((19, 64, 1056), 32, 16, False), ((20, 24, 3400), 32, 16, True), ((21, 16, 8216), 32, 16, True),
        ((27, 5850, 72), 32, 32, False), ((31, 4912, 1056), 32, 32, False), ((25, 20003, 136), 32, 64, False)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape,bm,bn,split", ROWS)
def test_linear_few_rows(shape, bm, bn, split, dtype):
    from yolo_amd.layers import linear
    m, n, k = shape
    g = _gen(m + n + k)
    x, w, b = _rand(g, m, k, dtype=dtype), _rand(g, n, k, scale=k ** -0.5, dtype=dtype), _rand(g, n, dtype=dtype)
    r = _rand(g, m, n, dtype=dtype)
    name, c = _choice(x, w)
    assert (name, c.bm, c.bn, c.k_slices > 1) == ("rows", bm, bn, split)
    _band_check(x, w, b, r, linear(x, w, b, activation="silu", residual=r), "silu", dtype)


# ------------------------------------------------------------------ linear, backward
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 24, 40), (7, 33, 65), (64, 128, 64), (130, 72, 264), (300, 130, 61),
                                   (1000, 256, 96), (513, 520, 264), (2500, 40, 48), (600, 1030, 520)])
def test_linear_backward(m, n, k, dtype):
    from yolo_amd.layers import linear
    g = _gen(m + n * 5 + k)
    x = _rand(g, m, k, dtype=dtype).requires_grad_()
    w = _rand(g, n, k, scale=k ** -0.5, dtype=dtype).requires_grad_()
    for act, bias_dtype, res_dtype, out in ((None, dtype, None, dtype), ("leaky", dtype, dtype, dtype), ("gelu", F32, None, F32),
                                            ("silu", None, F32, dtype), ("gelu_tanh", dtype, dtype, dtype), ("relu", F32, None, dtype)):
        b = _rand(g, n, scale=0.3, dtype=bias_dtype).requires_grad_() if bias_dtype else None
        r = _rand(g, m, n, dtype=res_dtype).requires_grad_() if res_dtype else None
        y = linear(x, w, b, activation=act, residual=r, out_dtype=out)
        dy = _rand(g, m, n, dtype=out)
        leaves = [t for t in (x, w, b, r) if t is not None]
        got = dict(zip([n_ for n_, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
        _, _, p, ep = ref.linear_ref(x, w, b, r, act, out)
        dx, dw, db = ref.linear_grad_ref(x, w, p, ep, dy, act, bias_dtype)
        assert_within(got["x"], *dx, f"dx {act}")
        assert_within(got["w"], *dw, f"dw {act}")
        if b is not None:
            assert got["b"].dtype == bias_dtype
            assert_within(got["b"], *db, f"db {act}")
        if r is not None:
            assert torch.equal(got["r"], dy.to(res_dtype))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,n,k", [(4096, 2048, 4096), (4100, 2056, 4104), (2048, 2048, 2048), (4100, 1032, 2056), (2048, 4096, 4096), (2060, 264, 4104)])
def test_linear_backward_large(m, n, k, dtype):
    """The products of the backward pass on the larger tiles: bands of dx and dweight."""
    from yolo_amd.layers import linear
    g = _gen(m + n * 5 + k)
    x = _rand(g, m, k, dtype=dtype).requires_grad_()
    w = _rand(g, n, k, scale=k ** -0.5, dtype=dtype).requires_grad_()
    dy = _rand(g, m, n, dtype=dtype)
    dx, dw = torch.autograd.grad(linear(x, w), (x, w), dy)
    rows, cols = torch.tensor([0, 1, 130, m - 257, m - 2, m - 1]).cuda(), torch.tensor([0, 1, 130, n - 257, n - 2, n - 1]).cuda()
    d64, w64, x64 = dy.double(), w.detach().double(), x.detach().double()
    for got, a, c, terms in ((dx[rows], d64[rows], w64, n), (dw[cols], d64[:, cols].t(), x64, m)):
        want, mag = a @ c, a.abs() @ c.abs()
        assert_within(got, want.cpu(), rounded(want, (terms + 4) * 2.0 ** -23 * mag, dtype).cpu(), "band")


def test_linear_backward_one_gradient_at_a_time():
    """Every subset of wanted gradients gives the gradients of the full set, bit for bit."""
    from yolo_amd.layers import linear
    g = _gen(21)
    x, w, b, r = _rand(g, 70, 48, dtype=BF16), _rand(g, 56, 48, dtype=BF16), _rand(g, 56, dtype=BF16), _rand(g, 70, 56, dtype=BF16)
    dy = _rand(g, 70, 56, dtype=BF16)
    full = None
    for want in sorted(itertools.product((True, False), repeat=4), reverse=True):
        if not any(want):
            continue
        ts = [t.detach().clone().requires_grad_(f) for t, f in zip((x, w, b, r), want)]
        y = linear(ts[0], ts[1], ts[2], activation="gelu", residual=ts[3])
        got = iter(torch.autograd.grad(y, [t for t, f in zip(ts, want) if f], dy))
        got = [next(got) if f else None for f in want]
        if full is None:
            full = got
        for a, c in zip(got, full):
            assert a is None or torch.equal(a, c)


def test_linear_padding_is_not_written():
    """Rows behind the last one and columns behind the row's end keep what they held (a strided y at the C entry)."""
    import ctypes
    from yolo_amd import _lib
    from yolo_amd._lib import lib
    g = _gen(93)
    for m, n, k, ld in ((3, 40, 64, 48), (70, 41, 64, 50), (300, 250, 72, 251), (40, 24, 4680, 33)):
        for f32 in (0, 1):
            x, w = _rand(g, m, k, dtype=BF16), _rand(g, n, k, scale=k ** -0.5, dtype=BF16)
            y = torch.full((m + 2, ld), 7.0, dtype=F32 if f32 else BF16, device="cuda")
            d = _lib.LinearDesc()
            d.x, d.weight, d.y = x.data_ptr(), w.data_ptr(), y.data_ptr()
            d.m, d.n, d.k, d.ldx, d.ldw, d.ldy, d.type, d.y_f32 = m, n, k, k, k, ld, _lib.TYPE_BF16, f32
            need = lib.yolo_amd_linear_workspace_bytes(ctypes.byref(d))
            ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
            d.workspace, d.workspace_bytes = ws.data_ptr(), need
            _lib.check(lib.yolo_amd_linear_forward(ctypes.byref(d), _lib.current_stream_ptr()), "linear")
            want, bound, _, _ = ref.linear_ref(x, w, None, None, None, y.dtype)
            assert_within(y[:m, :n], want, bound, "inside")
            assert (y[m:] == 7).all() and (y[:m, n:] == 7).all()


def test_linear_backward_views():
    """Strided x and weight, and an incoming gradient that is expanded, sliced or transposed."""
    from yolo_amd.layers import linear
    g = _gen(22)
    base_x, base_w = _rand(g, 90, 80, dtype=BF16), _rand(g, 60, 80, dtype=BF16)
    for c0, k in ((0, 64), (8, 40), (3, 33)):
        x, w = base_x[:, c0:c0 + k].detach().requires_grad_(), base_w[:, c0:c0 + k].detach().requires_grad_()
        wide = _rand(g, 90, 100, dtype=BF16)
        for dy in (wide[:, :60], wide[:, 1:61], _rand(g, 1, 60, dtype=BF16).expand(90, 60), _rand(g, 60, 90, dtype=BF16).t()):
            y = linear(x, w, activation="silu")
            dx, dw = torch.autograd.grad(y, [x, w], dy)
            _, _, p, ep = ref.linear_ref(x, w, None, None, "silu", BF16)
            wx, ww, _ = ref.linear_grad_ref(x, w, p, ep, dy, "silu", None)
            assert_within(dx, *wx, "dx")
            assert_within(dw, *ww, "dw")


def test_linear_gradient_against_differences():
    """d/dt of sum(dy * linear(x + t a, w + t c, b + t e)) by central differences of the 64-bit forward pass."""
    from yolo_amd.layers import linear
    g = _gen(23)
    x, w, b = (_rand(g, *s, scale=0.5, dtype=F16).requires_grad_() for s in ((40, 24), (32, 24), (32,)))
    dy = _rand(g, 40, 32, dtype=F16)
    for act in ("gelu", "gelu_tanh", "silu"):
        grads = torch.autograd.grad(linear(x, w, b, activation=act), (x, w, b), dy)
        dirs = [_rand(g, *t.shape).double().cpu() for t in (x, w, b)]

        def value(t):
            p = (ref.d(x) + t * dirs[0]) @ (ref.d(w) + t * dirs[1]).t() + ref.d(b) + t * dirs[2]
            return (ref.act64(p, act) * ref.d(dy)).sum()
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        _, _, p, ep = ref.linear_ref(x, w, b, None, act, F16)
        bounds = ref.linear_grad_ref(x, w, p, ep, dy, act, F16)
        got = sum((ref.d(a) * e).sum() for a, e in zip(grads, dirs))
        tol = sum((bd[1] * e.abs()).sum() for bd, e in zip(bounds, dirs)) + 1e-6 * slope.abs()
        assert abs(got - slope) <= tol, act


# ------------------------------------------------------------------ block_norm
def _norm_case(g, lead, dim, dtype, stream, norm, after, gate, par, residual=True):
    layer = norm == "layer"
    t = {"x": (_rand(g, *lead, dim) * 1.5 + 0.3).to(dtype)}
    t["residual"] = (_rand(g, *lead, dim) * 2 - 0.4).to(stream) if residual else None
    shape = {None: None, "channel": (dim,), "sequence": (lead[0],) + (1,) * (len(lead) - 1) + (dim,), "token": tuple(lead) + (dim,)}[gate]
    t["gate"] = None if shape is None else _rand(g, *shape, scale=0.7).to(par)
    t["after_weight"] = (1 + _rand(g, dim, scale=0.3)).to(par) if after else None
    t["after_bias"] = _rand(g, dim, scale=0.3).to(par) if after and layer else None
    t["before_weight"] = (1 + _rand(g, dim, scale=0.3)).to(par)
    t["before_bias"] = _rand(g, dim, scale=0.3).to(par) if layer else None
    return t


def _check_norm(t, norm, after, scale, eps=1e-6, backward=True, before=True, gradients=("both",)):
    from yolo_amd.layers import block_norm
    g = _gen(77)
    x, residual = t["x"], t["residual"]
    stream_dtype = residual.dtype if residual is not None else x.dtype
    leaves = {k: v.detach().requires_grad_() for k, v in t.items() if v is not None}
    args = {k: leaves.get(k) for k in t}
    s, y = block_norm(**args, norm=norm, after=after, residual_scale=scale, eps=eps, before=before)
    assert s.dtype == stream_dtype and s.shape == x.shape
    conf = (norm, after, before, scale, eps)
    params = {k: t[k] for k in ("gate", "after_weight", "after_bias", "before_weight", "before_bias")}
    out = ref.norm_ref(x, residual, conf, params)
    assert_within(s, out["stream"][0], rounded(*out["stream"], stream_dtype), "stream")
    if before:
        assert y.dtype == x.dtype
        assert_within(y, out["normed"][0], rounded(*out["normed"], x.dtype), "normed")
    else:
        assert y is None
    with torch.no_grad():                                    # the same bits without a graph
        s2, y2 = block_norm(**t, norm=norm, after=after, residual_scale=scale, eps=eps, before=before)
        assert torch.equal(s2, s) and (y is None or torch.equal(y2, y))
    for which in gradients if backward else ():
        ds = _rand(g, *x.shape, dtype=stream_dtype) if which in ("both", "stream") else None
        dy = _rand(g, *x.shape, dtype=x.dtype) if which in ("both", "normed") and before else None
        outs, grads = zip(*[(o, d_) for o, d_ in ((s, ds), (y, dy)) if d_ is not None])
        got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads, retain_graph=True, allow_unused=True)))
        want = ref.norm_ref(x, residual, conf, params, (ds, dy))
        for name, leaf in leaves.items():
            if name == "gate":
                v, e = ref.reduce_gate(want["gate_rows"], tuple(leaf.shape))
            elif name not in want:
                assert not got[name].any()                   # the norm before, when only the stream's gradient came in
                continue
            else:
                v, e = want[name]
            assert got[name].dtype == leaf.dtype
            assert_within(got[name], v, rounded(v, e, leaf.dtype), f"d{name} ({which})")


@pytest.mark.parametrize("dim", [1, 3, 8, 64, 100, 512, 520, 769, 1024, 1032, 2048, 2050, 4096, 8192])
@pytest.mark.parametrize("dtype,stream,par", [(BF16, BF16, F32), (F16, F32, F16), (F32, F32, F32)])
def test_block_norm_widths(dim, dtype, stream, par):
    g = _gen(dim)
    for norm, after, gate, lead in (("rms", True, "channel", (2, 5)), ("layer", True, "sequence", (3, 7)),
                                    ("layer", False, "token", (2, 3))):
        if norm == "layer" and dim < 8:
            continue                                         # one or three values: their variance is near eps, not near 1
        _check_norm(_norm_case(g, lead, dim, dtype, stream, norm, after, gate, par), norm, after, 0.5)


@pytest.mark.parametrize("dim", [2, 7, 9, 511, 1025, 1528, 1536, 2056, 2560, 2561, 3584, 4104, 5504, 6144, 6145, 6501, 7168, 8184, 8191, 8200])
def test_block_norm_widths_between(dim):
    """Rows that fill some of a workgroup's waves, whole or not, and that end anywhere in a run of eight."""
    g = _gen(dim + 1)
    _check_norm(_norm_case(g, (2, 3), dim, BF16, BF16, "rms", True, "token", F32), "rms", True, 0.5)
    _check_norm(_norm_case(g, (3, 2), dim, F16, F32, "rms", False, "channel", F16), "rms", False, 2.0)
    if dim >= 8:
        _check_norm(_norm_case(g, (2, 5), dim, F32, F32, "layer", True, "sequence", F32), "layer", True, 0.5)


@pytest.mark.parametrize("dim", [16384, 12001])
def test_block_norm_widest(dim):
    g = _gen(5)
    _check_norm(_norm_case(g, (3, 2), dim, BF16, F32, "rms", True, "sequence", BF16), "rms", True, 1.0)
    _check_norm(_norm_case(g, (3, 2), dim, BF16, BF16, "layer", True, "channel", F32), "layer", True, 1.0)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("after", [True, False])
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "token"])
def test_block_norm_forms(norm, after, gate):
    g = _gen(6)
    for residual in (True, False):
        t = _norm_case(g, (4, 3, 5), 136, BF16, F32 if residual else BF16, norm, after, gate, F32, residual)
        if not residual and not after and gate is None:
            _check_norm(t, norm, after, 0.5, gradients=("both", "stream", "normed"))
        else:
            _check_norm(t, norm, after, -1.25, gradients=("both", "stream", "normed"))
    t = _norm_case(g, (4, 3, 5), 136, F16, F16, norm, after, gate, F16)
    t["before_weight"] = t["before_bias"] = None
    _check_norm(t, norm, after, 1.0, before=False)           # the residual add alone
    t["after_weight"] = t["after_bias"] = None
    _check_norm(t, norm, after, 1.0)                         # norms without weights


@pytest.mark.parametrize("lead", [(1, 1), (1, 700), (700, 1), (600, 3), (5, 333), (40, 50), (1300, 2)])
def test_block_norm_row_counts(lead):
    """Rows that end inside a block's share, sequences cut into chunks, several sequences to a block."""
    g = _gen(lead[0] * 1000 + lead[1])
    for gate in ("channel", "sequence"):
        _check_norm(_norm_case(g, lead, 72, BF16, BF16, "rms", True, gate, F32), "rms", True, 0.5)
    _check_norm(_norm_case(g, lead, 1100, F32, F32, "layer", True, "sequence", F32), "layer", True, 0.5)


def test_block_norm_plain_norm_returns_its_input():
    from yolo_amd.layers import block_norm
    g = _gen(31)
    x, w = _rand(g, 6, 96, dtype=BF16).requires_grad_(), _rand(g, 96).requires_grad_()
    s, y = block_norm(x, before_weight=w)
    assert s is x
    out = ref.norm_ref(x, None, ("rms", False, True, 1.0, 1e-6), {"before_weight": w})
    assert_within(y, out["normed"][0], rounded(*out["normed"], BF16), "normed")
    dy, ds = _rand(g, 6, 96, dtype=BF16), _rand(g, 6, 96, dtype=BF16)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = ref.norm_ref(x, None, ("rms", False, True, 1.0, 1e-6), {"before_weight": w}, (None, dy))
    assert_within(dx, want["x"][0], rounded(*want["x"], BF16), "dx")
    assert_within(dw, want["before_weight"][0], rounded(*want["before_weight"], F32), "dw")
    s, y = block_norm(x, before=False)
    assert s is x and y is None


def test_block_norm_views_and_far_values():
    from yolo_amd.layers import block_norm
    g = _gen(32)
    wide = torch.full((40, 300), float("nan"), dtype=BF16, device="cuda")
    for c0, dim in ((0, 128), (8, 64), (3, 65)):
        x, r = wide[::2, c0:c0 + dim], _rand(g, 40, 200, dtype=F32)[::2, 5:5 + dim]
        x.copy_(_rand(g, 20, dim))
        s, y = block_norm(x, r, after=True)
        out = ref.norm_ref(x, r, ("rms", True, True, 1.0, 1e-6), {})
        assert_within(s, out["stream"][0], rounded(*out["stream"], F32), "stream")
        assert_within(y, out["normed"][0], rounded(*out["normed"], BF16), "normed")
    # rows of zeros, of one value, of a large offset, with NaN and inf: each row by itself
    x = _rand(g, 6, 64)
    x[0], x[1], x[2] = 0, 7.0, x[2] + 1000.0
    clean = {n: block_norm(x, norm=n)[1] for n in ("rms", "layer")}
    for n, y in clean.items():
        out = ref.norm_ref(x, None, (n, False, True, 1.0, 1e-6), {})
        assert_within(y, out["normed"][0], rounded(*out["normed"], F32), n)
        bad = x.clone()
        bad[3, 5], bad[4, 6] = float("nan"), float("inf")
        z = block_norm(bad, norm=n)[1]
        assert torch.isnan(z[3]).all() and torch.isnan(z[4]).any()
        assert torch.equal(z[[0, 1, 2, 5]], y[[0, 1, 2, 5]])


@pytest.mark.parametrize("dim", [5, 256, 520, 769, 1024, 1500, 2050, 7168, 8193])
def test_block_norm_rows_do_not_meet(dim):
    """NaN and infinities in one row leave every other row's values and gradients alone, whole rows or not."""
    from yolo_amd.layers import block_norm
    g = _gen(dim + 7)
    x, r, ds, dy = (_rand(g, 11, dim, dtype=BF16) for _ in range(4))
    w, b = _rand(g, dim), _rand(g, dim)
    for norm in ("rms", "layer"):
        def run(x, r):
            leaves = [x.clone().requires_grad_(), r.clone().requires_grad_()]
            out = block_norm(*leaves, norm=norm, after_weight=w, after_bias=b if norm == "layer" else None,
                             gate=w, before_weight=b)
            return [*out, *torch.autograd.grad(out, leaves, (ds, dy))]
        clean = run(x, r)
        bad_x, bad_r = x.clone(), r.clone()
        bad_x[3, dim - 1], bad_x[6, 0], bad_r[8, dim // 2] = float("nan"), float("inf"), float("nan")
        keep = [i for i in range(11) if i not in (3, 6, 8)]
        for got, want in zip(run(bad_x, bad_r), clean):
            assert torch.equal(got[keep], want[keep]), (norm, dim)


def test_block_norm_offsets_past_32_bits():
    from yolo_amd.layers import block_norm
    rows, dim = 2 ** 20 + 333, 2056                          # 2.16e9 values
    g = _gen(13)
    ends = torch.cat([torch.arange(100), torch.arange(rows - 100, rows)]).cuda()
    def filled(value):
        t = torch.empty(rows, dim, dtype=BF16, device="cuda").fill_(value)
        t[ends] = _rand(g, 200, dim, dtype=BF16)
        return t
    x, r, ds, dy = filled(0.5).requires_grad_(), filled(-0.25).requires_grad_(), filled(1.0), filled(0.125)
    params = {"after_weight": 1 + _rand(g, dim, scale=0.3), "before_weight": 1 + _rand(g, dim, scale=0.3), "gate": _rand(g, dim)}
    s, y = block_norm(x, r, after=True, **params)
    dx, dr = torch.autograd.grad((s, y), (x, r), (ds, dy))
    conf = ("rms", True, True, 1.0, 1e-6)
    small = [t.detach()[ends] for t in (x, r, ds, dy)]
    all_params = {"gate": params["gate"], "after_weight": params["after_weight"], "after_bias": None,
                  "before_weight": params["before_weight"], "before_bias": None}
    out = ref.norm_ref(small[0], small[1], conf, all_params, (small[2], small[3]))
    assert_within(s[ends], out["stream"][0], rounded(*out["stream"], BF16), "stream")
    assert_within(y[ends], out["normed"][0], rounded(*out["normed"], BF16), "normed")
    assert_within(dx[ends], out["x"][0], rounded(*out["x"], BF16), "dx")
    assert_within(dr[ends], out["residual"][0], rounded(*out["residual"], BF16), "dresidual")
    for t in (s, y, dx, dr):                                 # the rows in between are all alike
        assert torch.equal(t[5000], t[rows - 5000])


def test_block_norm_empty():
    from yolo_amd.layers import block_norm
    x = torch.empty(0, 32, dtype=BF16, device="cuda", requires_grad=True)
    w = torch.ones(32, device="cuda", requires_grad=True)
    gate = torch.ones(32, device="cuda", requires_grad=True)
    s, y = block_norm(x, x.detach(), after_weight=w, gate=gate, before_weight=w)
    assert s.shape == y.shape == (0, 32)
    dx, dw = torch.autograd.grad((s, y), (x, w), (torch.empty_like(s), torch.empty_like(y)))
    assert dx.shape == (0, 32) and not dw.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_block_norm_empty_gate_gradient(dtype):
    """No rows at all: the gradient of a gate that outlives them (one row, one for each sequence) is zero."""
    from yolo_amd.layers import block_norm
    for shape, gate_shape in (((0, 32), (32,)), ((4, 0, 32), (32,)), ((4, 0, 32), (4, 1, 32)), ((0, 7, 32), (0, 1, 32))):
        x = torch.empty(shape, dtype=dtype, device="cuda")
        gate = torch.full(gate_shape, 2.0, dtype=dtype, device="cuda", requires_grad=True)
        torch.full(gate_shape, float("nan"), dtype=dtype, device="cuda")     # what freed memory may hold
        s, y = block_norm(x, x, gate=gate, before_weight=torch.ones(32, device="cuda"))
        dg, = torch.autograd.grad((s, y), gate, (torch.empty_like(s), torch.empty_like(y)))
        assert dg.shape == gate.shape and torch.equal(dg, torch.zeros_like(dg)), (shape, gate_shape)


def test_block_norm_gradient_against_differences():
    from yolo_amd.layers import block_norm
    g = _gen(33)
    for norm in ("rms", "layer"):
        t = _norm_case(g, (3, 4), 40, F32, F32, norm, True, "sequence", F32)
        leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
        s, y = block_norm(**t, norm=norm, after=True, residual_scale=0.7)
        ds, dy = _rand(g, 3, 4, 40), _rand(g, 3, 4, 40)
        grads = torch.autograd.grad((s, y), list(leaves.values()), (ds, dy))
        dirs = {k: _rand(g, *v.shape).double().cpu() for k, v in leaves.items()}

        def value(h):
            m = {k: ref.d(v) + h * dirs[k] for k, v in leaves.items()}
            o = ref.norm_ref(m["x"], m["residual"], (norm, True, True, 0.7, 1e-6), m)
            return (o["stream"][0] * ref.d(ds)).sum() + (o["normed"][0] * ref.d(dy)).sum()
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        got = sum((ref.d(a) * dirs[k]).sum() for a, k in zip(grads, leaves))
        mag = sum((ref.d(a) * dirs[k]).abs().sum() for a, k in zip(grads, leaves))
        assert abs(got - slope) <= 1e-5 * mag, norm


# ------------------------------------------------------------------ together, streams, graphs
def _block(x, stream, p):
    """One residual block between its two norms."""
    from yolo_amd.layers import block_norm, linear
    _, n = block_norm(stream, before_weight=p["w0"])
    up = linear(n, p["w1"], p["b1"], activation="gelu_tanh")
    out = linear(up, p["w2"], p["b2"])
    return block_norm(out, stream, after_weight=p["w3"], gate=p["gate"], residual_scale=0.5, before_weight=p["w4"])


def _block_params(g, dtype, dim=72, hidden=136, batch=3):
    return {"w0": 1 + _rand(g, dim, scale=0.1), "w1": _rand(g, hidden, dim, scale=dim ** -0.5, dtype=dtype),
            "b1": _rand(g, hidden, scale=0.1, dtype=dtype), "w2": _rand(g, dim, hidden, scale=hidden ** -0.5, dtype=dtype),
            "b2": _rand(g, dim, scale=0.1, dtype=dtype), "w3": 1 + _rand(g, dim, scale=0.1),
            "gate": _rand(g, batch, 1, dim, dtype=dtype), "w4": 1 + _rand(g, dim, scale=0.1)}


def _block64(stream, p):
    import torch.nn.functional as F
    rms = lambda v, w: v / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6) * w     # noqa: E731
    n = rms(stream, p["w0"])
    out = F.gelu(n @ p["w1"].t() + p["b1"], approximate="tanh") @ p["w2"].t() + p["b2"]
    h = stream + 0.5 * p["gate"] * rms(out, p["w3"])
    return h, rms(h, p["w4"])


@pytest.mark.parametrize("tokens", [1, 50])
def test_block_of_all_operators(tokens):
    """Norm, widening layer, narrowing layer, norm and add, forward and backward, against 64 bits.  Relative error in
    the 2-norm: four bf16 roundings in a chain forward (n, up, out, the result) and about as many again backward, each
    at most 2^-8 relative in that norm; the norms' factors are near 1 and the weights' norms below 2, so that 16 * 2^-8
    bounds the sum."""
    g = _gen(41)
    p = _block_params(g, BF16)
    stream = _rand(g, 3, tokens, 72, dtype=BF16)
    leaves = [stream.requires_grad_()] + [t.requires_grad_() for t in p.values()]
    s, y = _block(None, stream, p)
    ds, dy = _rand(g, 3, tokens, 72, dtype=BF16), _rand(g, 3, tokens, 72, dtype=BF16)
    got = [s, y, *torch.autograd.grad((s, y), leaves, (ds, dy))]
    l64 = [ref.d(t).requires_grad_() for t in leaves]
    s6, y6 = _block64(l64[0], dict(zip(p, l64[1:])))
    want = [s6, y6, *torch.autograd.grad((s6, y6), l64, (ref.d(ds), ref.d(dy)))]
    for a, b in zip(got, want):
        a, b = ref.d(a), b.detach()
        assert (a - b).norm() <= 16 * 2.0 ** -8 * b.norm()


def test_layers_repeat_bit_for_bit_and_on_other_streams():
    g = _gen(42)
    p = {k: v.requires_grad_() for k, v in _block_params(g, BF16).items()}
    inputs = [_rand(g, 3, n, 72, dtype=BF16).requires_grad_() for n in (90, 41)]
    ds = [torch.randn_like(t) for t in inputs]

    def step(i):
        s, y = _block(None, inputs[i], p)
        return [s.detach(), y.detach(), *torch.autograd.grad((s, y), [inputs[i], *p.values()], (ds[i], ds[i]))]
    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(3):
        for i, st in enumerate(streams):                     # queued side by side
            with torch.cuda.stream(st):
                got[i] = step(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_layers_in_captured_graphs():
    """Two graphs captured one after the other and replayed side by side, with eager work between the replays."""
    g = _gen(43)
    p = _block_params(g, F16)
    for t in p.values():
        t.requires_grad_()
    ins = [_rand(g, 3, n, 72, dtype=F16) for n in (1, 64)]
    dys = [_rand(g, 3, n, 72, dtype=F16) for n in (1, 64)]

    def step(x, dy):
        x = x.detach().requires_grad_()
        s, y = _block(None, x, p)
        return [s, y, *torch.autograd.grad((s, y), [x, *p.values()], (dy, dy))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, dy in zip(ins, dys):
            step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, dy in zip(ins, dys):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append([t.detach() for t in step(x, dy)])
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for x in ins:
            x.copy_(_rand(g, *x.shape, dtype=F16))
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for x, dy, o in zip(ins, dys, outs):
            assert all(torch.equal(a, b) for a, b in zip(o, step(x, dy))), f"replay {rep}"


def test_layers_refuse_a_second_derivative():
    from yolo_amd.layers import linear
    g = _gen(44)
    x, w = _rand(g, 4, 16, dtype=BF16).requires_grad_(), _rand(g, 8, 16, dtype=BF16).requires_grad_()
    dx, = torch.autograd.grad(linear(x, w, activation="silu").float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.float().sum(), w)


def test_layers_refuse_on_the_gpu():
    """What the checks of shapes, types and devices refuse, nothing launched."""
    from yolo_amd._lib import YoloAmdError
    from yolo_amd.layers import block_norm, linear
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device="cuda")     # noqa: E731
    x, w = z(4, 16), z(8, 16)
    for bad in (lambda: linear(z(4, 16, t=F32), z(8, 16, t=F32)), lambda: linear(x, z(8, 16, t=F16)),
                lambda: linear(x, w, out_dtype=F16), lambda: block_norm(x.long()), lambda: block_norm(x, gate=z(16, t=F16)),
                lambda: block_norm(x, residual_scale=z(1)), lambda: block_norm(x, eps=z(1))):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: linear(x, z(8, 15)), lambda: linear(x, z(16)), lambda: linear(x, w, z(7)), lambda: linear(x, w, z(8, t=F16)),
                lambda: linear(x, w, residual=z(4, 7)), lambda: linear(x, w, residual=z(1, 8)), lambda: linear(x, w, activation="tanh"),
                lambda: block_norm(x, norm="batch"), lambda: block_norm(x, z(4, 8)), lambda: block_norm(x, z(4, 16, t=F16)),
                lambda: block_norm(x, before_bias=z(16)), lambda: block_norm(x, after=False, after_weight=z(16)),
                lambda: block_norm(x, before=False, before_weight=z(16)), lambda: block_norm(x, before_weight=z(15)),
                lambda: block_norm(x, norm="layer", before_weight=z(16), before_bias=z(16, t=F32)), lambda: block_norm(x, gate=z(3, 16)),
                lambda: block_norm(z(2, 4, 16), gate=z(1, 4, 16)), lambda: block_norm(z(2, 4, 16), gate=z(2, 4, 1)),
                lambda: block_norm(z(4, 0))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(YoloAmdError):
        block_norm(z(2, 16392))
    with pytest.raises(YoloAmdError):
        linear(x, w.cpu())
    with pytest.raises(YoloAmdError):
        block_norm(x, x, gate=z(16).cpu())
