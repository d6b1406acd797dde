"""4-bit calls with activations at both ends of bf16's range, against 64-bit products."""
import pytest
import torch

import float_ref as R
from forge_b200 import _forge_C as C

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# tokens of every kernel: few, 17 to 32, to 64, to 128, more
TOKENS = [1, 8, 9, 16, 17, 40, 100, 150]


def _product(x, w, s, group):
    """With more than 128 tokens the weights are rounded to bf16 first. Integers are multiplied as such times 2^-12 (few
    tokens) or 2^-11, which is taken off behind the sums or with the scale: fp32's smallest steps, 2^-149, count as 2^-137 of
    a group's sum, which the scale multiplies, and half of one for each addition of scaled sums (one a group, and one for
    each of up to 24 warps)."""
    M, K = x.shape
    wts = R.unpack_int4(w, s, K, group)
    y, err = R.linear(x, wts, None, R.int4_sizes(s, K, group, x.dtype) if M <= 16 else None)
    if M > 128:
        err = err + x.double().abs() @ R.half_step(wts, x.dtype).t()
    return y, err + K * 2.0 ** -137 * s.max().double() + (K / group + 32) * 2.0 ** -138


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", TOKENS)
@pytest.mark.parametrize("size", [3.3e38, 1e37, 1e36, 1e-30, 2e-36])
def test_no_sum_overflows_before_its_scale(M, size, group):
    """Every activation is the largest finite number, or near it. Weights of up to 1e-3 (their integers up to 7) with
    signs that alternate every four inputs keep the results below it; the integers' own sums are far above."""
    K, N = 392, 40
    g = torch.Generator().manual_seed(M)
    wts = torch.rand(N, K, generator=g) * 1e-3 * torch.where(torch.arange(K) % 8 < 4, 1.0, -1.0)
    w, s = C.prepare_weight_int4(wts.to(DEV), group)
    x = torch.full((M, K), size, device=DEV).bfloat16()
    assert x.isfinite().all()
    want, err = _product(x, w, s, group)
    assert want.abs().max() < 3e38
    R.close_rounded(C.int4_linear(x, w, s, None, group), want, err, "linear")
    # one input alone
    x = torch.zeros(M, K, device=DEV).bfloat16()
    x[:, 387] = size
    want, err = _product(x, w, s, group)
    R.close_rounded(C.int4_linear(x, w, s, None, group), want, err, "one input")
    # the gate: SiLU's argument large, the other factor small, their product finite
    wu, su = C.prepare_weight_int4(wts.to(DEV).flip(0) * 1e-3, group)
    small = torch.zeros_like(x)
    small[:, 387] = min(size, 1e18)
    gate, up = _product(small, w, s, group), _product(small, wu, su, group)
    R.close_rounded(C.int4_gated_linear(small, w, wu, s, su, None, None, group), *R.gate_of(gate, up), "gate")
    torch.cuda.synchronize()
    assert C.device_status() == 0
