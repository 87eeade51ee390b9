"""yolo_amd.layers and its C entry points on a machine without a GPU: struct layouts, what is refused before anything
is launched, and the dispatch of the product."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from helpers import ROOT

BF16 = torch.bfloat16


def _linear_desc(m=4, n=8, k=16, **kw):
    from yolo_amd import _lib
    d = _lib.LinearDesc()
    d.x, d.weight, d.y = 0x10000, 0x20000, 0x30000          # never dereferenced: the checks read the numbers only
    d.m, d.n, d.k, d.ldx, d.ldw, d.ldy = m, n, k, k, k, n
    d.type = _lib.TYPE_BF16
    for name, v in kw.items():
        setattr(d, name, v)
    return d


def _query(d):
    from yolo_amd import _lib
    c = _lib.LinearChoice()
    rc = _lib.lib.yolo_amd_linear_query(ctypes.byref(d), ctypes.byref(c))
    return rc, c


def test_struct_layouts_match_the_header():
    from yolo_amd import _lib
    structs = {"yolo_amd_linear_desc": _lib.LinearDesc, "yolo_amd_linear_choice": _lib.LinearChoice,
               "yolo_amd_linear_backward_desc": _lib.LinearBackwardDesc, "yolo_amd_block_norm_desc": _lib.BlockNormDesc,
               "yolo_amd_block_norm_backward_desc": _lib.BlockNormBackwardDesc}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = "#include <stdio.h>\n#include <stddef.h>\n#include \"yolo_amd.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n"
    with tempfile.TemporaryDirectory() as tmp:
        c, exe = os.path.join(tmp, "t.c"), os.path.join(tmp, "t")
        with open(c, "w") as fh:
            fh.write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        got = [int(v) for v in subprocess.check_output([exe]).split()]
    assert got == want


def test_codes_match_the_header():
    from yolo_amd import _lib
    text = open(os.path.join(ROOT, "include", "yolo_amd.h")).read()

    def value(name):
        return int(text.split(f"#define {name} ")[1].split()[0])
    for act, code in _lib.ACT_CODES.items():
        assert value(f"YOLO_AMD_ACT_{(act or 'none').upper()}") == code
    for norm, code in _lib.NORM_CODES.items():
        assert value(f"YOLO_AMD_NORM_{norm.upper()}") == code
    assert (value("YOLO_AMD_TYPE_F32"), value("YOLO_AMD_TYPE_BF16"), value("YOLO_AMD_TYPE_F16")) == (0, 1, 2)
    assert _lib.LINEAR_KERNEL_NAMES[value("YOLO_AMD_LINEAR_ROWS")] == "rows"
    assert _lib.LINEAR_KERNEL_NAMES[value("YOLO_AMD_LINEAR_TILE")] == "tile"


@pytest.mark.parametrize("change,word", [
    (dict(type=0), "type"), (dict(type=3), "type"), (dict(activation=6), "activation"), (dict(activation=-1), "activation"),
    (dict(m=-1), "m="), (dict(k=1 << 22, ldx=1 << 22, ldw=1 << 22), "k="), (dict(n=1 << 22, ldy=1 << 22), "n="),
    (dict(m=1 << 31), "m="), (dict(x=None), "x is null"), (dict(weight=None), "weight is null"), (dict(y=None), "y is null"),
    (dict(ldx=15), "row stride"), (dict(ldw=0), "row stride"), (dict(ldy=7), "row stride"),
    (dict(residual=0x40000, ldr=4), "residual"), (dict(x=0x10001), "aligned"), (dict(y=0x30002, y_f32=1), "aligned"),
    (dict(bias=0x40002, bias_f32=1), "bias"),
])
def test_linear_refusals(change, word):
    from yolo_amd._lib import lib
    d = _linear_desc(**change)
    rc, _ = _query(d)
    assert rc < 0 and word in lib.yolo_amd_last_error().decode()
    assert lib.yolo_amd_linear_forward(ctypes.byref(d), None) == rc
    assert lib.yolo_amd_linear_workspace_bytes(ctypes.byref(d)) == 0


def test_linear_workspace_is_checked():
    from yolo_amd._lib import lib
    d = _linear_desc(m=300, n=60, k=61)                     # rows of 61: both operands are copied
    need = lib.yolo_amd_linear_workspace_bytes(ctypes.byref(d))
    assert need >= (300 + 60) * 64 * 2
    assert lib.yolo_amd_linear_forward(ctypes.byref(d), None) < 0 and b"workspace" in lib.yolo_amd_last_error()
    d.workspace, d.workspace_bytes = 0x100000, need - 1
    assert lib.yolo_amd_linear_forward(ctypes.byref(d), None) == -3 and b"needed" in lib.yolo_amd_last_error()
    d.workspace, d.workspace_bytes = 0x100010, need
    assert lib.yolo_amd_linear_forward(ctypes.byref(d), None) == -1 and b"aligned" in lib.yolo_amd_last_error()


def test_linear_null_descriptors():
    from yolo_amd._lib import lib
    for fn in (lib.yolo_amd_linear_forward, lib.yolo_amd_linear_backward, lib.yolo_amd_block_norm_forward,
               lib.yolo_amd_block_norm_backward):
        assert fn(None, None) < 0 and b"null descriptor" in lib.yolo_amd_last_error()
    assert lib.yolo_amd_linear_workspace_bytes(None) == 0


def test_linear_dispatch():
    """Few rows stream the weights; operands the tiles cannot read in place are copied; a long reduction with few
    output tiles is split."""
    from yolo_amd import _lib
    assert _query(_linear_desc(1, 1024, 1024))[1].kernel == 1
    c = _query(_linear_desc(8192, 16384, 4096))[1]
    assert (c.kernel, c.bm, c.bn, c.k_slices) == (2, 256, 256, 1)
    c = _query(_linear_desc(256, 256, 65536))[1]
    assert c.kernel == 2 and c.k_slices > 1
    c = _query(_linear_desc(300, 60, 61))[1]
    assert (c.copies_x, c.copies_weight) == (1, 1)
    c = _query(_linear_desc(300, 60, 64, ldx=65))[1]
    assert (c.copies_x, c.copies_weight) == (1, 0)
    c = _query(_linear_desc(1, 60, 64, ldx=65))[1]          # one row has no stride
    assert (c.copies_x, c.copies_weight) == (0, 0)
    c = _query(_linear_desc(300, 60, 64, ldx=1 << 23))[1]   # the last token of long sequences
    assert (c.copies_x, c.copies_weight) == (1, 0)
    c = _query(_linear_desc(300, 60, 64, weight=0x20002))[1]
    assert (c.copies_x, c.copies_weight) == (0, 1)
    assert _query(_linear_desc(0, 8, 16, x=None, y=None))[0] == 0
    assert _lib.lib.yolo_amd_linear_forward(ctypes.byref(_linear_desc(0, 8, 16, x=None, y=None)), None) == 0


@pytest.mark.parametrize("change,word", [
    (dict(type=3), "type"), (dict(norm=2), "norm"), (dict(d=0), "rows of"), (dict(d=16385, ldx=16385), "rows of"),
    (dict(rows=-1), "rows of"), (dict(eps=-1.0), "eps"), (dict(x=None), "x is null"), (dict(x=0x10001), "aligned"),
    (dict(ldx=31), "row stride"), (dict(residual=0x40000, ldr=8), "residual"), (dict(gate=0x50000), "rows_per_gate"),
    (dict(after_weight=0x50000), "after"), (dict(before=0, before_weight=0x50000, normed=None), "before"),
    (dict(before_bias=0x50000), "bias"), (dict(before_weight=0x50002, before_f32=1), "aligned"), (dict(normed=None), "normed"),
    (dict(before=0), "normed"), (dict(stream=0x60002, stream_f32=1), "aligned"), (dict(eps=float("nan")), "eps"),
])
def test_block_norm_refusals(change, word):
    from yolo_amd import _lib
    d = _lib.BlockNormDesc()
    d.x, d.normed, d.rows, d.d, d.ldx, d.type, d.norm, d.before, d.eps, d.scale = 0x10000, 0x20000, 4, 32, 32, 1, 0, 1, 1e-6, 1.0
    for name, v in change.items():
        setattr(d, name, v)
    assert _lib.lib.yolo_amd_block_norm_forward(ctypes.byref(d), None) < 0
    assert word in _lib.lib.yolo_amd_last_error().decode()


def test_block_norm_backward_refusals():
    from yolo_amd import _lib
    lib = _lib.lib

    def desc(**kw):
        b = _lib.BlockNormBackwardDesc()
        d = b.forward
        d.x, d.rows, d.d, d.ldx, d.type, d.before, d.eps, d.scale = 0x10000, 6, 32, 32, 1, 1, 1e-6, 1.0
        b.dnormed, b.dx = 0x20000, 0x30000
        for name, v in kw.items():
            setattr(d if hasattr(d, name) else b, name, v)
        return b
    for change, word in ((dict(dgate=0x40000), "gate"), (dict(dafter_weight=0x40000), "after"), (dict(dbefore_bias=0x40000), "bias"),
                         (dict(gate=0x50000, rows_per_gate=4, dgate=0x40000), "whole runs"), (dict(dx=0x30001), "aligned"),
                         (dict(before=0), "dnormed"), (dict(dbefore_weight=0x40000), "workspace")):
        b = desc(**change)
        assert lib.yolo_amd_block_norm_backward(ctypes.byref(b), None) < 0, change
        assert word in lib.yolo_amd_last_error().decode(), change
    assert lib.yolo_amd_block_norm_backward_workspace_bytes(ctypes.byref(desc())) == 0
    assert lib.yolo_amd_block_norm_backward_workspace_bytes(ctypes.byref(desc(dbefore_weight=0x40000))) >= 32 * 4


def test_layers_refuse_cpu_tensors():
    from yolo_amd._lib import YoloAmdError
    from yolo_amd.layers import block_norm, linear
    x, w = torch.zeros(4, 16, dtype=BF16), torch.zeros(8, 16, dtype=BF16)
    with pytest.raises(YoloAmdError, match="CPU"):
        linear(x, w)
    with pytest.raises(YoloAmdError, match="CPU"):
        block_norm(x)
    with pytest.raises(TypeError):
        linear([1.0], w)


def test_reference_bounds_catch_planted_mistakes():
    """The oracle's bounds are tight enough to be worth something: a correct fp32 computation passes, small mistakes of
    the kind a kernel makes do not."""
    import layer_reference as ref
    g = torch.Generator().manual_seed(1)
    x, w, b = (torch.randn(*s, generator=g).to(BF16) for s in ((20, 64), (24, 64), (24,)))
    y = (x.float() @ w.float().t() + b.float()).to(BF16)
    want, bound, _, _ = ref.linear_ref(x, w, b, None, None, BF16)
    ref.assert_within(y, want, bound, "right")
    short = (x[:, :63].float() @ w[:, :63].float().t() + b.float()).to(BF16)       # one term missing
    twice = y.float().to(torch.float16).to(BF16) * (1 + 2.0 ** -6)                 # a scale that is off
    for bad in (short, twice, y.roll(1, 0)):
        with pytest.raises(AssertionError):
            ref.assert_within(bad, want, bound, "wrong")
    v = torch.randn(5, 33, generator=g)
    conf = ("layer", False, True, 1.0, 1e-6)
    out = ref.norm_ref(v, None, conf, {})["normed"]
    good = torch.nn.functional.layer_norm(v, (33,), eps=1e-6)
    ref.assert_within(good, out[0], ref.rounded(*out, torch.float32), "right")
    unbiased = (v - v.mean(-1, keepdim=True)) / v.std(-1, keepdim=True)
    with pytest.raises(AssertionError):
        ref.assert_within(unbiased, out[0], ref.rounded(*out, torch.float32), "wrong")


def test_rows_of_views():
    from yolo_amd.layers import _rows
    t = torch.zeros(4, 6, 8)
    assert _rows(t)[1] == 8 and _rows(t[:, -1:])[1] == 48 and _rows(t[:, 2])[1] == 48 and _rows(t[..., :5])[1] == 8
    assert _rows(t[0])[1] == 8 and _rows(t[1:2, ::2])[1] == 16 and _rows(t[:, :, ::2])[1] == 4 and _rows(t[:, :2])[1] == 8
    assert _rows(t[:, :2])[0].is_contiguous() and _rows(t[:1].expand(4, 6, 8))[0].is_contiguous()
    assert _rows(t[0, 0].expand(3, 8))[1] == 8 and _rows(t[0, 0, ::2])[0].is_contiguous()
    assert _rows(t[..., :1])[1] == 8 and _rows(t.transpose(0, 1))[0].is_contiguous()


def test_gate_rows():
    from yolo_amd.layers import _gate_rows
    e = lambda *s: torch.empty(s)     # noqa: E731
    assert _gate_rows(e(2, 3, 8), e(8)) == 6
    assert _gate_rows(e(2, 3, 8), e(1, 1, 8)) == 6
    assert _gate_rows(e(2, 3, 8), e(2, 1, 8)) == 3
    assert _gate_rows(e(2, 3, 8), e(2, 3, 8)) == 1
    assert _gate_rows(e(2, 3, 5, 8), e(2, 3, 1, 8)) == 5
    assert _gate_rows(e(2, 3, 5, 8), e(2, 1, 1, 8)) == 15
    assert _gate_rows(e(1, 3, 8), e(1, 1, 8)) == 3
    assert _gate_rows(e(3, 8), e(3, 8)) == 1
    assert _gate_rows(e(8), e(8)) == 1
    for bad in ((3, 8), (1, 3, 8), (2, 3, 4), (2, 1, 3, 8), ()):
        with pytest.raises(ValueError):
            _gate_rows(e(2, 3, 8), e(*bad))
