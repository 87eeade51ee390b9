"""The largest products of yolo_amd.layers.linear: what a launch cannot hold is refused before anything runs, by every entry
that plans it; what it can hold takes a tile that fits."""
import ctypes

import pytest

from test_layers_cpu import _linear_desc, _query


@pytest.mark.parametrize("m,n", [(1 << 30, 1 << 10), (1 << 30, 1 << 20), (1 << 21, 1 << 21)])
def test_linear_with_too_many_tiles(m, n):
    from yolo_amd._lib import lib
    d = _linear_desc(m, n, 61)                               # rows of 61: operands that would be copied first
    rc, _ = _query(d)
    assert rc < 0 and b"tiles" in lib.yolo_amd_last_error()
    assert lib.yolo_amd_linear_workspace_bytes(ctypes.byref(d)) == 0
    d.workspace, d.workspace_bytes = 0x100000, 1 << 62
    assert lib.yolo_amd_linear_forward(ctypes.byref(d), None) == rc and b"tiles" in lib.yolo_amd_last_error()


@pytest.mark.parametrize("m,n,k,wants", [(1 << 30, 64, 1 << 10, "dx"), (64, 1 << 21, 1 << 21, "dweight")])
def test_linear_backward_with_too_many_tiles(m, n, k, wants):
    from yolo_amd import _lib
    lib = _lib.lib
    d = _lib.LinearBackwardDesc()
    d.dy, d.x, d.weight = 0x10000, 0x20000, 0x30000          # never dereferenced
    d.m, d.n, d.k, d.lddy, d.ldx, d.ldw, d.type, d.dy_f32 = m, n, k, n, k, k, _lib.TYPE_BF16, 1
    setattr(d, wants, 0x40000)
    assert lib.yolo_amd_linear_backward_workspace_bytes(ctypes.byref(d)) == 0
    d.workspace, d.workspace_bytes = 0x100000, 1 << 62
    assert lib.yolo_amd_linear_backward(ctypes.byref(d), None) < 0 and b"tiles" in lib.yolo_amd_last_error()


@pytest.mark.parametrize("m,n,k", [(1 << 30, 1, 8), (1 << 30, 64, 64), (1 << 30, 256, 8), (1 << 30, 700, 8), ((1 << 30) - 1, 768, 4096),
                                   (1 << 21, 1 << 18, 64)])
def test_linear_with_as_many_tiles_as_fit(m, n, k):
    rc, c = _query(_linear_desc(m, n, k))
    assert rc == 0 and c.kernel == 2 and -(-m // c.bm) * -(-n // c.bn) < 1 << 24
