"""The 4-bit operators at the edges of what numbers can be: scales of one feature far apart, infinities, numbers near the largest, and
what the host refuses.

Tolerances: weights formed in half precision are rounded once, to 2^-11 of themselves; 32-bit sums and what is held as exact as in
test_fourbit_gpu.py."""
import math

import pytest
import torch

from test_fourbit_gpu import gen, made_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, False)])
def test_weights_of_many_rows_are_rounded_once_however_small_their_scale_is(group, zeros):
    """A row of x that is one number alone gives back one weight: no other group hides what a small scale loses.  Scales down to 2^-24 of
    their feature's largest."""
    from hos_b200.parts.weights4 import Weight4
    n, k = 80, 512
    groups = k // group
    codes, _, z, _ = made_weights(n, k, group, zeros, 11)
    exponent = -torch.round(torch.arange(groups) * 24 / (groups - 1))
    scales = ((1 + torch.rand(n, groups, generator=gen(12))) * torch.exp2(exponent)).to(BF).to(DEV)
    at = torch.arange(k, device=DEV) // group
    w = (codes.double() - (z.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    got = Weight4.from_codes(codes, scales, z, group).product(torch.eye(k, device=DEV, dtype=BF), F32)
    assert bool(((got.double() - w.T).abs() <= 2.0 ** -11 * w.T.abs()).all())
