"""4-bit weights on the CPU: the recipe against exact rational arithmetic, the packed layout against its description, the
conversion of models, and the refusals of the C entry points (which come before any device call)."""
from fractions import Fraction

import pytest
import torch
import torch.nn as nn

import float_ref as R
from forge_b200 import _lib
from forge_b200.nn import GatedLinear, Int4GatedLinear, Int4Linear, QuantizedLinear, quantize_weight_int4
from forge_b200.quant import quantize

BAD_SHAPE, BAD_POINTER = 1, 2


def _round_to_half(v):
    """A positive rational rounded to the nearest fp16, ties to even."""
    e = -24
    while v >= Fraction(2) ** (e + 11):
        e += 1
    n = v / Fraction(2) ** e
    low = n.numerator // n.denominator
    up = n - low > Fraction(1, 2) or (n - low == Fraction(1, 2) and low % 2 == 1)
    return (low + up) * Fraction(2) ** e


def _round_even(v):
    low = v.numerator // v.denominator
    d = v - low
    return low + (d > Fraction(1, 2) or (d == Fraction(1, 2) and low % 2 == 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_recipe_in_rational_arithmetic(group, dtype):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(6, 200, generator=g).to(dtype)
    w[1] *= 1e-6
    w[2] = torch.round(w[2] * 4) / 4   # many quotients on a border
    packed, scale = quantize_weight_int4(w, group)
    assert packed.shape == (6, 128) and scale.shape == (-(-200 // group), 6) and scale.dtype == torch.float16
    q = R.unpack_int4(packed, torch.ones_like(scale), 200, group)
    for n in range(6):
        for j in range(scale.shape[0]):
            ks = range(j * group, min(200, j * group + group))
            vals = [Fraction(float(w[n, k])) for k in ks]
            s = _round_to_half(max(abs(v) for v in vals) / 7)
            assert Fraction(float(scale[j, n])) == s
            for k, v in zip(ks, vals):
                assert q[n, k] == (max(-7, min(7, _round_even(v / s))) if s else 0)


def test_layout_of_one_weight():
    """Weight 77 of a block: run 9 of eight, so word 4 * 1 + 2; weight 5 of the run, so nibble 6."""
    w = torch.zeros(2, 256)
    w[1, 128 + 77] = 7.0
    packed, _ = quantize_weight_int4(w, 128)
    words = packed.view(torch.int32)[1]
    eights = 0x88888888 - (1 << 32)
    want = torch.full((32,), eights, dtype=torch.int32)
    want[16 + 6] = eights + (7 << 24)
    assert torch.equal(words, want)


def test_weights_past_the_last_input_are_zero():
    packed, _ = quantize_weight_int4(torch.ones(1, 8), 32)
    assert packed.shape == (1, 64) and (packed[0, 4:] == 0x88).all() and (packed[0, :4] == 0xFF).all()


class Net(nn.Module):
    def __init__(self):
        super().__init__()
        self.a = nn.Linear(64, 24)
        self.b = nn.Linear(24, 20, bias=False)
        self.odd = nn.Linear(20, 5)
        self.gate = GatedLinear(16, 40, bias=True, dtype=torch.bfloat16)


def test_quantize_to_4_bits():
    torch.manual_seed(0)
    net = Net()
    out = quantize(net, scheme="weight_only_int4", group_size=32, verbose=False)
    assert isinstance(out.a, Int4Linear) and isinstance(out.b, Int4Linear) and isinstance(out.gate, Int4GatedLinear)
    assert isinstance(out.odd, QuantizedLinear)         # 20 inputs: no multiple of 8
    assert isinstance(net.a, nn.Linear) and isinstance(net.gate, GatedLinear)
    w, s = quantize_weight_int4(net.a.weight, 32)
    assert torch.equal(out.a.w_int4, w) and torch.equal(out.a.w_scale, s)
    assert torch.equal(out.a.bias, net.a.bias.half()) and out.b.bias is None
    w, s = quantize_weight_int4(net.gate.w_up, 32)
    assert torch.equal(out.gate.w_up_int4, w) and torch.equal(out.gate.w_up_scale, s)
    assert out.gate.b_gate.dtype == torch.bfloat16 and torch.equal(out.gate.b_gate, net.gate.b_gate)
    # the INT8 schemes leave the gate as it is
    assert isinstance(quantize(net, verbose=False).gate, GatedLinear)
    with pytest.raises(ValueError):
        quantize(net, scheme="weight_only_int4", sparse=True, verbose=False)
    with pytest.raises(ValueError):
        quantize(net, scheme="weight_only_int4", group_size=48, verbose=False)


def test_module_refusals():
    for make in (lambda: Int4Linear(60, 8), lambda: Int4Linear(64, 8, group_size=256), lambda: Int4GatedLinear(4, 8),
                 lambda: Int4GatedLinear(64, 8, group_size=0), lambda: GatedLinear(64, 60), lambda: GatedLinear(60, 64)):
        with pytest.raises(ValueError):
            make()
    m = Int4Linear(64, 8)
    with pytest.raises(ValueError):   # there is no CPU path
        m(torch.randn(2, 64))
    assert (R.unpack_int4(m.w_int4, m.w_scale, 64, 128) == 0).all()


def test_c_refusals():
    lib = _lib.load()
    p, odd = 0x10000, 0x10008   # never read: every call is refused, or has nothing to do

    def lin(x=p, w=p, s=p, o=p, M=4, K=64, N=16, group=64, dtype=1):
        return lib.forge_int4_linear(x, w, s, 0, o, M, K, N, group, dtype, 0)
    assert [lin(M=0), lin(K=0), lin(N=-3)] == [0, 0, 0]
    assert [lin(x=0), lin(w=0), lin(s=0), lin(o=0)] == [BAD_POINTER] * 4
    assert [lin(K=60), lin(group=16), lin(group=0), lin(dtype=0), lin(dtype=3), lin(x=odd), lin(w=odd),
            lin(s=p + 2)] == [BAD_SHAPE] * 8

    def gated(x=p, g=p, u=p, sg=p, su=p, o=p, M=4, K=64, N=16, group=64, dtype=2):
        return lib.forge_int4_gated_linear(x, g, u, sg, su, 0, 0, o, M, K, N, group, dtype, 0)
    assert [gated(M=0), gated(x=0), gated(g=0), gated(u=0), gated(sg=0), gated(su=0), gated(o=0)] == [0] + [BAD_POINTER] * 6
    assert [gated(K=4), gated(group=8), gated(dtype=0), gated(x=odd), gated(g=odd), gated(u=odd),
            gated(sg=p + 2), gated(su=p + 2)] == [BAD_SHAPE] * 8

    def prep(w=p, dtype=0, o=p, s=p, N=4, K=64, group=64):
        return lib.forge_prepare_weight_int4(w, dtype, o, s, N, K, group, 0)
    assert [prep(N=0), prep(w=0), prep(o=0), prep(s=0)] == [0] + [BAD_POINTER] * 3
    assert [prep(K=12), prep(group=1), prep(dtype=-1), prep(dtype=3), prep(w=odd), prep(o=odd)] == [BAD_SHAPE] * 6

    def fwd(x=p, g=p, u=p, h=p, go=0, uo=0, M=4, K=64, N=16, dtype=1):
        return lib.forge_gated_linear(x, g, u, 0, 0, h, go, uo, M, K, N, dtype, 0)
    assert [fwd(M=0), fwd(x=0), fwd(g=0), fwd(u=0), fwd(h=0), fwd(go=p), fwd(uo=p)] == [0] + [BAD_POINTER] * 6
    assert [fwd(K=12), fwd(N=12), fwd(dtype=0), fwd(x=odd), fwd(g=odd), fwd(u=odd), fwd(h=odd), fwd(go=odd, uo=p),
            fwd(go=p, uo=odd)] == [BAD_SHAPE] * 9

    def bwd(dh=p, x=p, wg=p, wu=p, g=p, u=p, dx=p, dwg=p, dwu=p, M=4, K=64, N=16, dtype=1, ws=p):
        return lib.forge_gated_linear_backward(dh, x, wg, wu, g, u, dx, dwg, dwu, p, p, M, K, N, dtype, ws, 0)
    assert [bwd(M=0), bwd(K=0)] == [0, 0]
    assert [bwd(**{k: 0}) for k in ("dh", "x", "wg", "wu", "g", "u", "ws", "dwg", "dwu")] == [BAD_POINTER] * 9
    assert [bwd(**{k: odd}) for k in ("dh", "x", "wg", "wu", "g", "u", "dx", "dwg", "dwu")] == [BAD_SHAPE] * 9
    assert [bwd(K=12), bwd(N=4), bwd(dtype=0), bwd(ws=p + 128)] == [BAD_SHAPE] * 4
    size = lib.forge_gated_linear_backward_workspace_bytes
    assert size(0, 16) == 0 and size(4, 0) == 0 and size(8192, 14336) >= 2 * 2 * 8192 * 14336


def test_c_refusals_of_sizes():
    lib, p, big = _lib.load(), 0x10000, (1 << 30) + 8
    for M, K, N in ((big, 64, 16), (4, big, 16), (4, 64, big)):
        assert lib.forge_int4_linear(p, p, p, 0, p, M, K, N, 64, 1, 0) == BAD_SHAPE
        assert lib.forge_int4_gated_linear(p, p, p, p, p, 0, 0, p, M, K, N, 64, 1, 0) == BAD_SHAPE
        assert lib.forge_gated_linear(p, p, p, 0, 0, p, 0, 0, M, K, N, 1, 0) == BAD_SHAPE
        assert lib.forge_gated_linear_backward(p, p, p, p, p, p, p, p, p, 0, 0, M, K, N, 1, p, 0) == BAD_SHAPE
        if M != big:
            assert lib.forge_prepare_weight_int4(p, 0, p, p, N, K, 64, 0) == BAD_SHAPE


def test_weights_of_another_shape_are_refused():
    """A row that would be broadcast over all outputs, among them."""
    m, gm = Int4Linear(64, 8), Int4GatedLinear(64, 8)
    good = torch.randn(8, 64)
    for w in (good[:1], good[:, :8], good.t(), good[0], torch.randn(16, 64)):
        with pytest.raises(ValueError):
            m.quantize_weight(w)
        with pytest.raises(ValueError):
            gm.quantize_weight(good, w)
    for w, group in ((good, 16), (good[:, :60], 64), (good[:, :0], 64), (good[0], 64)):
        with pytest.raises(ValueError):
            quantize_weight_int4(w, group)
    m.quantize_weight(good)
    gm.quantize_weight(good, good)
