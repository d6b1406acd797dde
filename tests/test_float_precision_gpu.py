"""Root-mean-square errors of the 4-bit and gated calls against 64 bits at thousands of inputs, where a bound on the worst case
allows far more than the roundings that are documented.

What is allowed: the rounding of the result, and of the operands where a call rounds them, both measured here by making the
same roundings in 64 bits (independent errors: their squares add, 2 % for the samples' scatter), and the fp32 sums. A chain
of tensor instructions cuts its sum off behind the 24th bit or later once every 16 inputs, so over K inputs it loses at most
K / 16 * 2^-23 of the largest running sum, which for random signs is about the result's size; 2^-21 covers the rest."""
import pytest
import torch

import float_ref as R
from forge_b200 import _forge_C as C

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rms(t):
    return t.double().square().mean().sqrt().item()


def _check(got, want, rounded_operands, chain, what):
    """`rounded_operands`: the 64-bit result from operands rounded as the call rounds them; `chain`: inputs of a sum."""
    size = _rms(want)
    result = _rms(want.to(got.dtype).double() - want)
    operands = _rms(rounded_operands - want)
    allowed = 1.02 * (result ** 2 + operands ** 2) ** 0.5 + (2 * chain / 16 * 2.0 ** -23 + 2.0 ** -21) * size
    off = _rms(got.double() - want)
    assert off <= allowed, f"{what}: {off / size:.3g} of the result's size, allowed {allowed / size:.3g}"


def _new(gen, dtype, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def _silu(g):
    return g * torch.sigmoid(g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("M", [8, 16, 30, 64, 100, 300])
def test_int4(M, group, dtype):
    gen, t, K, N = torch.Generator().manual_seed(M + group), TYPES[dtype], 4096, 1024
    x = _new(gen, t, M, K)
    ops = [C.prepare_weight_int4(_new(gen, torch.float32, N, K, scale=K ** -0.5), group) for _ in range(2)]
    wg, wu = (R.unpack_int4(w, s, K, group) for w, s in ops)
    xd = x.double()
    # beyond 128 tokens the weights of plain calls are rounded first; those of gated calls are not
    want = xd @ wg.t()
    rounded = xd @ wg.to(t).double().t() if M > 128 else want
    _check(C.int4_linear(x, *ops[0], None, group), want, rounded, K if M > 128 else group, "linear")
    want = _silu(xd @ wg.t()) * (xd @ wu.t())
    got = C.int4_gated_linear(x, ops[0][0], ops[1][0], ops[0][1], ops[1][1], None, None, group)
    _check(got, want, want, 2 * K if M > 128 else group, "gate")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [4, 16, 300])
def test_gate(M, dtype):
    gen, t, K, N = torch.Generator().manual_seed(M), TYPES[dtype], 4096, 1024
    x, wg, wu = _new(gen, t, M, K), _new(gen, t, N, K, scale=K ** -0.5), _new(gen, t, N, K, scale=K ** -0.5)
    want = _silu(x.double() @ wg.double().t()) * (x.double() @ wu.double().t())
    _check(C.gated_linear(x, wg, wu), want, want, 2 * K, "h")


@pytest.mark.parametrize("size", [0.1, 1e-5])
@pytest.mark.parametrize("dtype", TYPES)
def test_gradients(dtype, size):
    """The gradients of gate and up are rounded to 11 (bf16: 8) bits, whatever their size."""
    gen, t, M, K, N = torch.Generator().manual_seed(1), TYPES[dtype], 1000, 520, 1032
    x, wg, wu = _new(gen, t, M, K), _new(gen, t, N, K, scale=K ** -0.5), _new(gen, t, N, K, scale=K ** -0.5)
    dh = _new(gen, t, M, N, scale=size)
    got = C.gated_linear_backward(dh, x, wg, wu, *C.gated_linear(x, wg, wu, save=True)[1:])
    xd, gd, ud = x.double(), wg.double(), wu.double()
    g, u, d = xd @ gd.t(), xd @ ud.t(), dh.double()
    s = torch.sigmoid(g)
    exact = d * u * s * (1 + g * (1 - s)), d * g * s

    def outputs(dg, du):
        return dg @ gd + du @ ud, dg.t() @ xd, du.t() @ xd, dg.sum(0), du.sum(0)
    large = 2.0 ** 10 / size   # well inside the type's range
    rounded = outputs(*((v * large).to(t).double() / large for v in exact))
    for i, (name, v) in enumerate(zip(("dx", "dwg", "dwu", "dbg", "dbu"), outputs(*exact))):
        # the bias gradients are summed before that rounding
        _check(got[i], v, rounded[i] if i < 3 else v, (2 * N, M, M, M, M)[i], name)
