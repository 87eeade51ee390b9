"""Ways of calling yolo_amd.layers in which torch would have to look into the kernels: forward-mode derivatives and traces.
They are refused, whatever the tensors' device, before anything is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

CALLS = {"linear": lambda x, w: _layers().linear(x, w), "linear residual": lambda x, w: _layers().linear(x, w, residual=x),
         "block_norm": lambda x, w: _layers().block_norm(x, before_weight=w[0])[1],
         "block_norm residual": lambda x, w: _layers().block_norm(x, x, gate=w[0], before=False)[0]}


def _layers():
    from yolo_amd import layers
    return layers


def _inputs(device="cpu"):
    return torch.ones(4, 16, dtype=torch.bfloat16, device=device), torch.ones(16, 16, dtype=torch.bfloat16, device=device)


@pytest.mark.parametrize("call", list(CALLS))
def test_tangents_are_refused(call):
    x, w = _inputs()
    with fw.dual_level():
        for dual in (0, 1):
            args = [x, w]
            args[dual] = fw.make_dual(args[dual], torch.ones_like(args[dual]))
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    CALLS[call](*args)


@pytest.mark.parametrize("call", list(CALLS))
def test_traces_are_refused(call):
    from yolo_amd._lib import YoloAmdError
    x, w = _inputs()
    for needs in (False, True):
        w.requires_grad_(needs)
        with pytest.raises(YoloAmdError, match="trace"):
            torch.jit.trace(CALLS[call], (x, w), check_trace=False)
        with pytest.raises(YoloAmdError, match="trace"):
            make_fx(CALLS[call])(x, w.detach())


def test_other_tensors_in_a_dual_level_are_not_minded():
    from yolo_amd._lib import YoloAmdError
    x, w = _inputs()
    with fw.dual_level():
        fw.make_dual(torch.ones(3), torch.ones(3))
        with pytest.raises(YoloAmdError, match="CPU"):       # the next check
            CALLS["linear"](x, w)
