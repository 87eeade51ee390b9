"""yolo_amd.layers under torch's forward mode, traces and compiler, on the GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from test_layers_modes_cpu import CALLS, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("call", list(CALLS))
def test_tangents_and_traces_are_refused_on_the_gpu(call):
    from yolo_amd._lib import YoloAmdError
    x, w = _inputs("cuda")
    want = CALLS[call](x, w)
    with fw.dual_level():
        with pytest.raises(NotImplementedError):
            CALLS[call](x, fw.make_dual(w, torch.ones_like(w)))
        assert torch.equal(CALLS[call](x, w), want)          # without tangents: as ever
    with pytest.raises(YoloAmdError):
        torch.jit.trace(CALLS[call], (x, w), check_trace=False)
    with pytest.raises(YoloAmdError):
        make_fx(CALLS[call])(x, w)
    assert torch.equal(CALLS[call](x, w), want)


@pytest.mark.parametrize("call", list(CALLS))
def test_tangents_and_traces_are_refused_in_the_backward_pass(call):
    """The gradient that comes in carries a tangent, or is traced, where the forward call saw neither."""
    from yolo_amd._lib import YoloAmdError
    x, w = (t.requires_grad_() for t in _inputs("cuda"))
    y = CALLS[call](x, w)
    dy = torch.ones_like(y).detach()

    def backward(g):
        return torch.autograd.grad(y, x, g, retain_graph=True)[0]
    want = backward(dy)
    with fw.dual_level():
        with pytest.raises(NotImplementedError):
            backward(fw.make_dual(dy, torch.ones_like(dy)))
        assert torch.equal(backward(dy), want)
    with pytest.raises(YoloAmdError):
        make_fx(backward)(dy)
    with pytest.raises(RuntimeError):                        # torch's own, or YoloAmdError
        torch.jit.trace(backward, (dy,), check_trace=False)
    assert torch.equal(backward(dy), want)


@pytest.mark.parametrize("call", list(CALLS))
def test_compiled_callers_run_the_kernels(call):
    x, w = _inputs("cuda")
    f = torch.compile(lambda x, w: CALLS[call](x * 2, w) + 1, backend="eager")
    assert torch.equal(f(x, w), CALLS[call](x * 2, w) + 1)
    assert torch.equal(f(x * 3, w), CALLS[call](x * 6, w) + 1)
