"""4-bit weights with group scales on the GPU: preparation bit for bit, the linear and the gated layer against 64-bit
products, at the sizes, groups and values where they can go wrong, and the calls they refuse."""
import pytest
import torch

import float_ref as R
from forge_b200 import _forge_C as C
from forge_b200 import _lib
from forge_b200.nn import Int4GatedLinear, Int4Linear, quantize_weight_int4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _ok():
    torch.cuda.synchronize()
    assert C.device_status() == 0


def _weight(N, K, group, gen, scale=0.05):
    """Packed weight with every nibble value, prepared on the CPU."""
    w, s = quantize_weight_int4(torch.randn(N, K, generator=gen) * scale, group)
    w = torch.where(torch.rand(w.shape, generator=gen) < 0.1, torch.randint(0, 256, w.shape, generator=gen).to(torch.uint8), w)
    tail = K % 128   # inputs past K are stored as zeros
    if tail:
        blk = w[:, -64:].view(N, 4, 4, 4)
        run = 4 * torch.arange(4)[None, :] + torch.arange(4)[:, None]   # [t][j]
        blk[:, run * 8 >= tail] = 0x88
    return w.to(DEV), s.to(DEV)


# ------------------------------------------------------------------------------------------------ preparation

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 8), (3, 120), (17, 128), (40, 136), (130, 1000), (5, 4096)])
def test_prepare_equals_the_cpu_recipe(N, K, group, dtype):
    g = torch.Generator().manual_seed(N * 7 + K + group)
    w = (torch.randn(N, K, generator=g) * torch.rand(N, 1, generator=g)).to(dtype)
    w[0, :min(K, 40)] = 0
    want = quantize_weight_int4(w, group)
    got = C.prepare_weight_int4(w.to(DEV), group)
    _ok()
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().view(torch.int16), want[1].view(torch.int16))


def test_prepare_on_rounding_borders():
    """Weights exactly on and one step beside every border n + 1/2 of every scale."""
    rows = []
    for i, s in enumerate([0.0078125, 0.00731, 0.9, 1.7e-5, 3.0]):
        s = torch.tensor(s).half().float()
        n = torch.arange(-7, 7).float() + 0.5
        w = torch.cat([n * s, torch.nextafter(n * s, torch.tensor(9.0)), torch.nextafter(n * s, torch.tensor(-9.0))])
        row = torch.zeros(128)
        row[: len(w)] = w
        row[-1] = 7 * s
        rows.append(row)
    w = torch.stack(rows)
    want, got = quantize_weight_int4(w, 128), C.prepare_weight_int4(w.to(DEV), 128)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_prepare_of_unusual_values():
    w = torch.zeros(6, 64)
    w[0, 3] = float("inf")
    w[1, 40] = float("nan")
    w[2, 0] = 7 * 65504.0
    w[3, 0] = 3e38
    w[4, 0] = 1e-12                 # the scale rounds to zero: all weights are zero
    w[5] = torch.linspace(-1e-6, 1e-6, 64)   # a subnormal scale
    want, got = quantize_weight_int4(w, 32), C.prepare_weight_int4(w.to(DEV), 32)
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().isnan(), want[1].isnan()) and torch.equal(got[1].cpu().nan_to_num(), want[1].nan_to_num())
    nan = got[1].cpu().isnan()
    assert nan[0, 0] and not nan[1, 0] and nan[1, 1] and not nan[0, 1] and not nan[0, 2] and nan[0, 3]


def test_prepare_of_views():
    big = torch.randn(300, 264, device=DEV)
    want = C.prepare_weight_int4(big[10:40, 8:200].clone(), 64)
    got = C.prepare_weight_int4(big[10:40, 8:200], 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.randn(30 * 64 + 1, device=DEV)[1:].view(30, 64)   # contiguous, not 16-byte aligned
    want, got = C.prepare_weight_int4(odd.clone(), 64), C.prepare_weight_int4(odd, 64)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------ linear, gated

SHAPES = [(1, 8, 1), (1, 64, 17), (1, 4096, 100), (2, 120, 16), (5, 2056, 33), (7, 520, 272), (8, 1000, 15), (9, 136, 48),
          (16, 256, 31), (17, 384, 130), (33, 520, 64), (64, 1024, 256), (100, 72, 257), (129, 648, 300), (300, 2048, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_int4_linear(M, K, N, group, dtype):
    g = torch.Generator().manual_seed(M + 3 * K + 5 * N + group)
    x = (torch.randn(M, K, generator=g) * (1 + 9 * (torch.rand(K, generator=g) < 0.05))).to(TYPES[dtype]).to(DEV)
    w, s = _weight(N, K, group, g)
    bias = torch.randn(N, generator=g).to(TYPES[dtype]).to(DEV) if (M + N) % 2 else None
    y = C.int4_linear(x, w, s, bias, group)
    _ok()
    R.close_rounded(y, *linear_bound(x, w, s, bias, group))


def linear_bound(x, w, s, b, group, gated=False):
    """Up to 16 tokens as R.int4_sizes says; up to 128 integers and exact scales, a group at a time; above, a plain call's
    weight is rounded once to the activations' type, a gated one's is in two parts, whose sum is exact."""
    K = x.shape[1]
    weight = R.unpack_int4(w, s, K, group)
    if x.shape[0] <= 16:
        return R.linear(x, weight, b, R.int4_sizes(s, K, group, x.dtype), group)
    if x.shape[0] <= 128:
        return R.linear(x, weight, b, None, group)
    if gated:
        y, err = R.linear(x, weight, b, weight.abs() * (1 + torch.finfo(x.dtype).eps))
        return y, err + 2.0 ** -24 * (y.abs() + err)   # the sum of the two
    y, err = R.linear(x, weight, b)
    return y, err + x.double().abs() @ R.half_step(weight, x.dtype).t()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_int4_gated_linear(M, K, N, group, dtype):
    g = torch.Generator().manual_seed(2 * M + 3 * K + 5 * N + group)
    x = torch.randn(M, K, generator=g).to(TYPES[dtype]).to(DEV)
    (wg, sg), (wu, su) = _weight(N, K, group, g), _weight(N, K, group, g)
    bg, bu = ((torch.randn(N, generator=g) * 0.3).to(TYPES[dtype]).to(DEV) if (M + N) % 2 else None for _ in range(2))
    h = C.int4_gated_linear(x, wg, wu, sg, su, bg, bu, group)
    _ok()
    R.close_rounded(h, *R.gate_of(linear_bound(x, wg, sg, bg, group, True), linear_bound(x, wu, su, bu, group, True)))


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("M,K,N", [(1, 16384, 20000), (9, 8200, 13001), (40, 4104, 30001), (97, 1160, 20001), (150, 4104, 30001)])
def test_several_passes_over_the_rows(M, K, N, group):
    """More rows than the SMs hold at a time, more columns than a ring."""
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g).half().to(DEV)
    w = torch.randint(0, 256, (N, -(-K // 128) * 64), generator=g).to(torch.uint8).to(DEV)
    s = (torch.rand(-(-K // group), N, generator=g) * 0.01 + 0.001).half().to(DEV)
    y = C.int4_linear(x, w, s, None, group)
    _ok()
    R.close_rounded(y, *linear_bound(x, w, s, None, group))
    h = C.int4_gated_linear(x, w, w.flip(0), s, s, None, None, group)
    _ok()
    R.close_rounded(h, *R.gate_of(linear_bound(x, w, s, None, group, True), linear_bound(x, w.flip(0), s, None, group, True)))


EDGES = [(16, 8, 1), (17, 8, 1), (17, 64, 129), (32, 4096, 40), (33, 136, 1), (40, 8200, 130), (64, 14336, 72), (64, 264, 300),
         (65, 4104, 129), (65, 8, 24), (96, 520, 1000), (128, 2056, 40), (128, 128, 257), (129, 8, 1), (129, 8208, 65), (200, 264, 7),
         (256, 136, 513), (257, 1024, 136), (100, 2056, 9500), (70, 6152, 4100)]


@pytest.mark.parametrize("dtype,group", [("fp16", 32), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("M,K,N", EDGES)
def test_both_sides_of_every_choice(M, K, N, dtype, group):
    """16 | 17, 64 | 65 and 128 | 129 tokens, inputs that are divided over a cluster, tiles with one row or one output."""
    g = torch.Generator().manual_seed(M + 3 * K + 5 * N + group)
    x = torch.randn(M, K, generator=g).to(TYPES[dtype]).to(DEV)
    (wg, sg), (wu, su) = _weight(N, K, group, g), _weight(N, K, group, g)
    bias = torch.randn(N, generator=g).to(TYPES[dtype]).to(DEV)
    y = C.int4_linear(x, wg, sg, bias, group)
    h = C.int4_gated_linear(x, wg, wu, sg, su, bias, None, group)
    _ok()
    R.close_rounded(y, *linear_bound(x, wg, sg, bias, group), "linear")
    R.close_rounded(h, *R.gate_of(linear_bound(x, wg, sg, bias, group, True), linear_bound(x, wu, su, None, group, True)), "gated")


def test_several_streams_at_once():
    """Kernels of every kind side by side, none of which keeps anything that another one writes."""
    g = torch.Generator().manual_seed(11)
    w, s = _weight(1100, 2056, 64, g)
    xs = [torch.randn(M, 2056, generator=g).half().to(DEV) for M in (1, 12, 40, 100, 300)]
    run = lambda x: (C.int4_linear(x, w, s, None, 64), C.int4_gated_linear(x, w, w, s, s, None, None, 64))  # noqa: E731
    want = [run(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for k in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                n = (i + k) % len(xs)
                got.append((n, run(xs[n])))
    _ok()
    for n, (y, h) in got:
        assert torch.equal(y, want[n][0]) and torch.equal(h, want[n][1])


_FIRST_CALL_CAPTURED = """
import torch
from forge_b200 import _forge_C as C
from forge_b200.nn import quantize_weight_int4
dev = torch.device("cuda:0")
g = torch.Generator().manual_seed(0)
w, s = (t.to(dev) for t in quantize_weight_int4(torch.randn(48, 136, generator=g) * 0.1, 64))
W = torch.randn(48, 136, generator=g).half().to(dev) * 0.1
xs = [torch.randn(M, 136, generator=g).half().to(dev) for M in (1, 40, 100, 200)]
dh = torch.ones(200, 48, device=dev).half()

def run():
    out = []
    for x in xs:
        out += [C.int4_linear(x, w, s, None, 64), C.int4_gated_linear(x, w, w, s, s, None, None, 64), C.gated_linear(x, W, W)]
    h, gate, up = C.gated_linear(xs[-1], W, W, save=True)
    return out + [h, *C.gated_linear_backward(dh, xs[-1], W, W, gate, up)]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run())) and C.device_status() == 0
"""


def test_a_first_call_may_be_captured():
    """In a process of its own, where no kernel has been loaded or set up."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _FIRST_CALL_CAPTURED], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("M", [1, 8, 40])
def test_repeated_calls_give_the_same_bits(M):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, 4096, generator=g).half().to(DEV)
    w, s = _weight(200, 4096, 64, g)
    y = C.int4_linear(x, w, s, None, 64)
    for _ in range(5):
        assert torch.equal(C.int4_linear(x, w, s, None, 64), y)


@pytest.mark.parametrize("M", [3, 40])
def test_infinities_and_nans_stay_where_they_belong(M):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(M, 264, generator=g).half().to(DEV)
    w, s = _weight(50, 264, 32, g)
    y = C.int4_linear(x, w, s, None, 32)
    xn, sn = x.clone(), s.clone()
    xn[1, 263] = float("nan")
    xn[2, 0] = float("inf")
    sn[8, 7] = float("nan")
    z = C.int4_linear(xn, w, sn, None, 32)
    assert z[1].isnan().all() and not z[2].isfinite().any() and z[:, 7].isnan().all()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[1:3] = False
    keep[:, 7] = False
    assert torch.equal(z[keep], y[keep])


def test_large_results_overflow_only_at_the_end():
    """Products beyond fp16 that cancel: sums are fp32."""
    x = torch.full((2, 64), 300.0, device=DEV).half()
    x[1, 32:] = -300.0
    q = torch.full((4, 64), 7.0) * 60
    w, s = quantize_weight_int4(q, 32)
    y = C.int4_linear(x, w.to(DEV), s.to(DEV), None, 32)
    assert y[0].isinf().all() and (y[1] == 0).all()


def test_no_tokens_no_outputs():
    w, s = C.prepare_weight_int4(torch.randn(24, 64, device=DEV), 64)
    assert C.int4_linear(torch.empty(0, 64, device=DEV).half(), w, s, None, 64).shape == (0, 24)
    x = torch.randn(3, 64, device=DEV).half()
    assert C.int4_linear(x, w[:0], s[:, :0].contiguous(), None, 64).shape == (3, 0)
    assert C.int4_gated_linear(x[:0], w, w, s, s, None, None, 64).shape == (0, 24)


def test_weight_past_32_bit_offsets():
    """A weight of more than 2^31 bytes: its last rows are read where they are."""
    K, N = 65536, 70000
    g = torch.Generator().manual_seed(0)
    w = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device=DEV)
    s = torch.ones(K // 128, N, dtype=torch.float16, device=DEV)
    tail, st = _weight(16, K, 128, g)
    w[-16:], s[:, -16:] = tail, st
    for M in (1, 40):
        x = torch.randn(M, K, generator=g).half().to(DEV)
        y = C.int4_linear(x, w, s)
        _ok()
        R.close_rounded(y[:, -16:], *linear_bound(x, tail, st, None, 128))
        # zeros, within the bound of a product whose parts are q + 8 and 8
        zero, err = linear_bound(x, w[:1], s[:, :1], None, 128)
        R.close_rounded(y[:, :-16], zero.expand(M, N - 16), err.expand(M, N - 16))


def test_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(9)
    x = torch.randn(4, 512, generator=g).half().to(DEV)
    big = torch.randn(80, 512, generator=g).half().to(DEV)
    w, s = _weight(300, 512, 64, g)
    want, want_big = C.int4_linear(x, w, s, None, 64), C.int4_gated_linear(big, w, w, s, s, None, None, 64)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = C.int4_linear(x, w, s, None, 64)
        got_big = C.int4_gated_linear(big, w, w, s, s, None, None, 64)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_big, want_big)
    graph = torch.cuda.CUDAGraph()
    xin = torch.zeros_like(x)
    bin_ = torch.zeros_like(big)
    with torch.cuda.graph(graph):
        y = C.int4_linear(xin, w, s, None, 64)
        z = C.int4_gated_linear(bin_, w, w, s, s, None, None, 64)
    for scale in (1, 2):
        xin.copy_(x * scale)
        bin_.copy_(big * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, C.int4_linear(x * scale, w, s, None, 64))
        assert torch.equal(z, C.int4_gated_linear(big * scale, w, w, s, s, None, None, 64))


def test_rows_behind_the_output_stay():
    """Through the C ABI, into the middle of a larger buffer."""
    g = torch.Generator().manual_seed(3)
    w, s = _weight(37, 256, 128, g)
    for M in (3, 50):
        x = torch.randn(M, 256, generator=g).half().to(DEV)
        out = torch.full((M + 2, 37), 7.0, device=DEV).half()
        _lib.call("forge_int4_linear", x.data_ptr(), w.data_ptr(), s.data_ptr(), 0, out[1:].data_ptr(), M, 256, 37, 128, 1,
                  torch.cuda.current_stream().cuda_stream)
        assert (out[0] == 7).all() and (out[-1] == 7).all()
        assert torch.equal(out[1:-1], C.int4_linear(x, w, s))


def test_an_unaligned_activation_is_taken():
    g = torch.Generator().manual_seed(5)
    w, s = _weight(40, 128, 32, g)
    buf = torch.randn(4 * 128 + 3, generator=g).half().to(DEV)
    x = buf[3:].view(4, 128)
    assert torch.equal(C.int4_linear(x, w, s, None, 32), C.int4_linear(x.clone(), w, s, None, 32))


def test_refusals():
    x = torch.randn(4, 128, device=DEV).half()
    w, s = C.prepare_weight_int4(torch.randn(32, 128, device=DEV), 64)
    call = lambda x=x, w=w, s=s, b=None, g=64: C.int4_linear(x, w, s, b, g)  # noqa: E731
    call()
    with pytest.raises(TypeError):
        call(x=x.float())
    with pytest.raises(TypeError):
        call(s=s.float())
    with pytest.raises(TypeError):
        call(b=torch.zeros(32, device=DEV))
    with pytest.raises(ValueError):
        call(x=x[:, :124].contiguous())            # not a multiple of 8
    with pytest.raises(ValueError):
        call(x=x[:, :0])
    with pytest.raises(ValueError):
        call(x=x[0])
    with pytest.raises(ValueError):
        call(x=x.t().contiguous().t())             # strided
    with pytest.raises(ValueError):
        call(g=96)
    with pytest.raises(ValueError):
        call(g=128)                                # the scales are of another group size
    with pytest.raises(ValueError):
        call(w=w[:, :32].contiguous())
    with pytest.raises(ValueError):
        call(b=torch.zeros(31, device=DEV).half())
    with pytest.raises(ValueError):
        call(x=x.cpu())
    with pytest.raises(ValueError):
        C.int4_gated_linear(x, w, w[:16], s, s[:, :16].contiguous(), None, None, 64)
    with pytest.raises(ValueError):
        C.prepare_weight_int4(torch.randn(32, 100, device=DEV), 64)
    with pytest.raises(ValueError):
        C.prepare_weight_int4(torch.randn(32, 128, device=DEV), 16)
    _ok()


# ------------------------------------------------------------------------------------------------ modules

@pytest.mark.parametrize("dtype", TYPES)
def test_modules(dtype):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 3, 264, generator=g).to(TYPES[dtype]).to(DEV)
    w, w2 = torch.randn(2, 48, 264, generator=g).mul(0.05).to(DEV)
    m = Int4Linear(264, 48, group_size=32, dtype=TYPES[dtype]).to(DEV)
    m.quantize_weight(w)
    m.bias.data.normal_()
    y = m(x)
    assert y.shape == (2, 3, 48) and y.dtype == x.dtype
    R.close_rounded(y.view(6, 48), *linear_bound(x.view(6, 264), m.w_int4, m.w_scale, m.bias, 32))
    gm = Int4GatedLinear(264, 48, group_size=32, dtype=TYPES[dtype]).to(DEV)
    gm.quantize_weight(w, w2)
    h = gm(x.transpose(0, 1))
    x2 = x.transpose(0, 1).reshape(6, 264)
    R.close_rounded(h.reshape(6, 48), *R.gate_of(linear_bound(x2, gm.w_gate_int4, gm.w_gate_scale, None, 32),
                                                 linear_bound(x2, gm.w_up_int4, gm.w_up_scale, None, 32)))
    other = Int4Linear(264, 48, group_size=32, dtype=TYPES[dtype]).to(DEV)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), y)
