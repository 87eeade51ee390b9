"""GELU of yolo_amd.layers.linear in fp32 against its definition, at pre-activations that are exact."""
import pytest
import torch

import layer_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,columns", [("rows", 1), ("tile", 40)])
def test_gelu_of_exact_values(kernel, columns):
    """x of one column times 1: the sum is x itself.  With twelve roundings of 2^-24 in a chain (seven in the polynomial, the
    reciprocal's and the exponential's two each, two products, the last addition less one), |p| erfc / 2 <= 0.17 and a fit
    that adds 2.7e-8, GELU is off by at most 0.17 * 13 * 2^-24 + 2.7e-8 = 1.6e-7 below 0.  Relative to its own size: the fit's
    5.4e-6, the same roundings (8e-7), and the exponent's own rounding, p^2 / 2 * 2^-24 * 2 <= 4.9e-6 down to -9: 1.2e-5.
    Above 0 GELU is p less the same error, with one more rounding of the result."""
    from yolo_amd.layers import linear
    values = torch.linspace(-9, 9, 6000).to(torch.float16).cuda()
    for p in values.split(30 if kernel == "rows" else 6000):
        y = linear(p[:, None], torch.ones(columns, 1, dtype=torch.float16, device="cuda"), activation="gelu", out_dtype=torch.float32)
        p64, y64 = p.double().cpu(), y.double().cpu()
        want = ref.act64(p64, "gelu")
        off = (y64 - want[:, None]).abs()
        assert (off <= 1.6e-7 + 2.0 ** -24 * want.abs()[:, None]).all(), f"{float(off.max())}"
        low = p64 < 0
        assert (off[low] <= 1.2e-5 * want[low].abs()[:, None]).all(), f"{float((off[low] / want[low].abs()[:, None]).max())}"


def test_gelu_slopes_of_exact_values():
    """The bias gradient of one row is dy act'(p): off by half of erfc's error (14 roundings, 5.4e-8 of the fit), by that of
    p exp(-p^2/2) / sqrt(2 pi) <= 0.242 (six roundings and the exponent's at most 0.25 * 2^-24 there) and by the last one."""
    from yolo_amd.layers import linear
    p = torch.linspace(-9, 9, 4001).to(torch.float16).cuda()
    b = torch.zeros(p.numel(), device="cuda", requires_grad=True)
    y = linear(torch.ones(1, 1, dtype=torch.float16, device="cuda"), p[:, None], b, activation="gelu", out_dtype=torch.float32)
    db, = torch.autograd.grad(y, b, torch.ones_like(y))
    want = ref.slope64(p.double().cpu(), "gelu")
    bound = 0.5 * (14 * 2.0 ** -24 + 5.4e-8) + 0.242 * 8 * 2.0 ** -24 + 2.0 ** -24 * 1.13
    assert ((db.double().cpu() - want).abs() <= bound).all()
