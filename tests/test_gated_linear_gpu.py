"""The gated linear layer on 16-bit weights, forward and backward, against 64-bit products and against differences; its use
in a model that is trained and then quantized; the calls it refuses."""
import pytest
import torch
import torch.nn as nn

import float_ref as R
from forge_b200 import _forge_C as C
from forge_b200 import _lib
from forge_b200.nn import GatedLinear, Int4GatedLinear, Int4Linear, gated_linear
from forge_b200.quant import quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 8, 8), (1, 512, 264), (2, 72, 16), (8, 264, 200), (9, 1000, 48), (16, 64, 136), (17, 64, 64), (33, 200, 128),
          (128, 256, 256), (130, 328, 264), (257, 512, 520), (300, 1032, 136), (513, 136, 1032), (700, 640, 1288), (3, 4104, 20008), (12, 1160, 9480)]


def _ok():
    torch.cuda.synchronize()
    assert C.device_status() == 0


def _case(M, K, N, dtype, bias, seed=0):
    g = torch.Generator().manual_seed(seed + M + 3 * K + 5 * N)
    new = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(TYPES[dtype]).to(DEV)  # noqa: E731
    x, wg, wu, dh = new(M, K), new(N, K, scale=K ** -0.5), new(N, K, scale=K ** -0.5), new(M, N, scale=0.1)
    bg, bu = (new(N, scale=0.2), new(N, scale=0.2)) if bias else (None, None)
    return x, wg, wu, bg, bu, dh


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_forward(M, K, N, bias, dtype):
    x, wg, wu, bg, bu, _ = _case(M, K, N, dtype, bias)
    want, err, (g, eg, u, eu) = R.gate(x, wg, wu, bg, bu)
    R.close_rounded(C.gated_linear(x, wg, wu, bg, bu), want, err, "h")
    h, gk, uk = C.gated_linear(x, wg, wu, bg, bu, save=True)
    _ok()
    R.close_rounded(h, want, err, "h in training")
    R.close(gk, g, eg + 2.0 ** -23 * g.abs(), "g")
    R.close(uk, u, eu + 2.0 ** -23 * u.abs(), "u")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_backward(M, K, N, bias, dtype):
    x, wg, wu, bg, bu, dh = _case(M, K, N, dtype, bias, 1)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    h = gated_linear(x, wg, wu, bg, bu)
    grads = torch.autograd.grad(h, leaves, dh)
    _ok()
    with torch.no_grad():
        saved = R.gate(x, wg, wu, bg, bu)[2]
        want = R.gate_backward(dh, x, wg, wu, saved, TYPES[dtype])
    for name, got in zip(want, grads):
        assert got.dtype == x.dtype
        R.close(got, *want[name], name)


def test_gradients_against_differences():
    """Directional derivatives of the 64-bit forward by central differences. With a step of 1e-4 along a direction of the
    inputs' size the third-order term is below 1e-7 of the sum of sizes, against the gradient's own bound of about 1e-3."""
    x, wg, wu, bg, bu, dh = _case(40, 72, 64, "fp16", True, 2)
    args = [x, wg, wu, bg, bu]
    for t in args:
        t.requires_grad_()
    grads = torch.autograd.grad(gated_linear(*args), args, dh)
    a = [t.detach().double() for t in args]
    want = R.gate_backward(dh, *a[:3], R.gate(*a)[2], torch.float16)
    loss = lambda v: (R.gate(*v)[0] * dh.double()).sum()  # noqa: E731
    gen = torch.Generator().manual_seed(3)
    for i, name in enumerate(want):
        v = (torch.randn(a[i].shape, generator=gen).double().to(DEV)) * a[i].abs().mean()
        step = lambda e: loss([t + e * v if j == i else t for j, t in enumerate(a)])  # noqa: B023, E731
        diff = (step(1e-4) - step(-1e-4)) / 2e-4
        got = (grads[i].double() * v).sum()
        size = (want[name][0].abs() * v.abs()).sum()
        assert abs(got - diff) <= (want[name][1] * v.abs()).sum() + 1e-6 * size, name


@pytest.mark.parametrize("needs", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 1), (0, 0, 0, 1, 0), (1, 0, 0, 1, 1)])
def test_only_the_wanted_gradients(needs):
    x, wg, wu, bg, bu, dh = _case(50, 64, 72, "bf16", True)
    args = [x, wg, wu, bg, bu]
    full = [t.clone().requires_grad_() for t in args]
    want = torch.autograd.grad(gated_linear(*full), full, dh)
    some = [t.clone().requires_grad_(bool(n)) for t, n in zip(args, needs)]
    gated_linear(*some).backward(dh)
    for t, n, w in zip(some, needs, want):
        assert (t.grad is not None) == bool(n)
        if n:
            assert torch.equal(t.grad, w)


def test_repeated_steps_give_the_same_bits_and_accumulate():
    x, wg, wu, bg, bu, dh = _case(300, 128, 136, "fp16", True)
    args = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    one = torch.autograd.grad(gated_linear(*args), args, dh)
    two = torch.autograd.grad(gated_linear(*args), args, dh)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    for _ in range(2):
        gated_linear(*args).backward(dh)
    for t, g in zip(args, one):
        assert torch.equal(t.grad, g + g)


def test_a_broadcast_gradient_and_leading_sizes():
    x, wg, wu, _, _, _ = _case(24, 64, 72, "fp16", False)
    a = x.view(2, 3, 4, 64).clone().requires_grad_()
    h = gated_linear(a, wg, wu)
    assert h.shape == (2, 3, 4, 72)
    h.sum().backward()   # the gradient of h has strides of zero
    b = x.clone().requires_grad_()
    gated_linear(b, wg, wu).backward(torch.ones(24, 72, device=DEV).half())
    assert torch.equal(a.grad.view(24, 64), b.grad)
    t = x.t().contiguous().t().requires_grad_()   # strided
    assert torch.equal(gated_linear(t, wg, wu), h.view(24, 72))


def test_no_tokens():
    x, wg, wu, bg, bu, _ = _case(4, 64, 72, "fp16", True)
    x = x[:0].clone().requires_grad_()
    for t in (wg, wu, bg, bu):
        t.requires_grad_()
    h = gated_linear(x, wg, wu, bg, bu)
    assert h.shape == (0, 72)
    h.sum().backward()
    assert x.grad.shape == (0, 64) and all((t.grad == 0).all() for t in (wg, wu, bg, bu))


@pytest.mark.parametrize("M", [3, 40])
def test_infinities_and_nans_stay_in_their_rows(M):
    x, wg, wu, _, _, _ = _case(M, 264, 72, "fp16", False)
    h = C.gated_linear(x, wg, wu)
    y = x.clone()
    y[1, 263] = float("nan")
    z = C.gated_linear(y, wg, wu)
    assert z[1].isnan().all()
    y[1] = x[1]
    keep = [i for i in range(M) if i != 1]
    assert torch.equal(z[keep], h[keep])


def test_a_very_negative_gate_is_zero():
    x = torch.full((2, 64), 30.0, device=DEV).half().requires_grad_()
    wg = torch.full((8, 64), -30.0, device=DEV).half().requires_grad_()   # g = -57600
    wu = torch.full((8, 64), 1.0, device=DEV).half()
    h = gated_linear(x, wg, wu)
    assert (h == 0).all()
    h.sum().backward()
    assert (x.grad == 0).all() and (wg.grad == 0).all()


def test_a_captured_step_replays():
    x, wg, wu, bg, bu, dh = _case(200, 128, 136, "bf16", True)
    eager = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = [torch.autograd.grad(gated_linear(*eager), eager, dh), None]
    with torch.no_grad():
        eager[0].mul_(2)
    want[1] = torch.autograd.grad(gated_linear(*eager), eager, dh)
    static = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(gated_linear(*static), static, dh)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(gated_linear(*static), static, dh)
    for k in range(2):
        with torch.no_grad():
            static[0].copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_two_streams_at_once():
    cases = [_case(300, 256, 264, "fp16", False, s) for s in (5, 6)]
    want = []
    for x, wg, wu, _, _, dh in cases:
        a = [t.clone().requires_grad_() for t in (x, wg, wu)]
        want.append(torch.autograd.grad(gated_linear(*a), a, dh))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for st, (x, wg, wu, _, _, dh) in zip(streams, cases):
        with torch.cuda.stream(st):
            a = [t.clone().requires_grad_() for t in (x, wg, wu)]
            got.append([torch.autograd.grad(gated_linear(*a), a, dh) for _ in range(5)])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for step in g:
            assert all(torch.equal(p, q) for p, q in zip(step, w))


def test_rows_behind_the_outputs_stay():
    x, wg, wu, bg, bu, dh = _case(70, 72, 136, "fp16", True)
    ptr = lambda t: t.data_ptr()  # noqa: E731
    st = torch.cuda.current_stream().cuda_stream
    for M in (5, 70):
        h = torch.full((M + 1, 136), 7.0, device=DEV).half()
        g, u = torch.full((2, M + 1, 136), 7.0, device=DEV)
        _lib.call("forge_gated_linear", ptr(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), ptr(h), 0, 0, M, 72, 136, 1, st)
        assert (h[M] == 7).all() and torch.equal(h[:M], C.gated_linear(x[:M], wg, wu, bg, bu))
        _lib.call("forge_gated_linear", ptr(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), ptr(h), ptr(g), ptr(u), M, 72, 136, 1, st)
        assert (h[M] == 7).all() and (g[M] == 7).all() and (u[M] == 7).all()
        dx = torch.full((M + 1, 72), 7.0, device=DEV).half()
        dw = torch.full((2, 137, 72), 7.0, device=DEV).half()
        db = torch.full((2, 144), 7.0, device=DEV).half()
        ws = torch.empty(_lib.load().forge_gated_linear_backward_workspace_bytes(M, 136), dtype=torch.uint8, device=DEV)
        _lib.call("forge_gated_linear_backward", ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g), ptr(u), ptr(dx), ptr(dw[0]),
                  ptr(dw[1]), ptr(db[0]), ptr(db[1]), M, 72, 136, 1, ptr(ws), st)
        _ok()
        assert (dx[M] == 7).all() and (dw[:, 136] == 7).all() and (db[:, 136:] == 7).all()
        assert dw[:, :136].isfinite().all() and (dx[:M] != 7).any()


def test_refusals():
    x, wg, wu, bg, bu, dh = _case(4, 64, 72, "fp16", True)
    with pytest.raises(TypeError):
        gated_linear(x.float(), wg, wu)
    with pytest.raises(TypeError):
        gated_linear(x, wg, wu.bfloat16())
    with pytest.raises(TypeError):
        gated_linear(x, wg, wu, bg.float(), bu)
    with pytest.raises(ValueError):
        gated_linear(x[:, :60], wg[:, :60], wu[:, :60])
    with pytest.raises(ValueError):
        gated_linear(x, wg[:70], wu[:70])
    with pytest.raises(ValueError):
        gated_linear(x, wg, wu[:64])
    with pytest.raises(ValueError):
        gated_linear(x, wg, wu, bg[:8], bu)
    with pytest.raises(ValueError):
        gated_linear(x.cpu(), wg, wu)
    with pytest.raises(ValueError):
        GatedLinear(60, 64)
    h = gated_linear(x.requires_grad_(), wg, wu)
    (gx,) = torch.autograd.grad(h, x, dh.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):   # no second derivative
        gx.sum().backward()
    with torch.no_grad():
        wg2 = wg.clone().requires_grad_()
    h = gated_linear(x, wg2, wu)
    with torch.no_grad():
        wg2.add_(1)
    with pytest.raises(RuntimeError):   # a weight changed between forward and backward
        h.sum().backward()


class Block(nn.Module):
    """A Llama-style feed-forward block."""

    def __init__(self, d, f, dtype):
        super().__init__()
        self.gate_up = GatedLinear(d, f, bias=True, dtype=dtype, device=DEV)
        self.down = nn.Linear(f, d, dtype=dtype, device=DEV)

    def forward(self, x):
        return x + self.down(self.gate_up(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_block_is_trained_then_served_with_4_bit_weights(dtype):
    torch.manual_seed(0)
    t = TYPES[dtype]
    block = Block(128, 264, t)
    x = torch.randn(3, 40, 128, device=DEV).to(t)
    block(x).float().pow(2).mean().backward()
    # the gate's gradients for the gradient that autograd hands it
    xg = x.clone().requires_grad_()
    hidden = block.gate_up(xg)
    dh = torch.autograd.grad(block.down(hidden).float().pow(2).mean(), hidden, retain_graph=True)[0]
    m = block.gate_up
    grads = torch.autograd.grad(hidden, [xg, m.w_gate, m.w_up, m.b_gate, m.b_up], dh)
    with torch.no_grad():
        x2 = x.view(-1, 128)
        saved = R.gate(x2, m.w_gate, m.w_up, m.b_gate, m.b_up)[2]
        want = R.gate_backward(dh.reshape(120, 264), x2, m.w_gate, m.w_up, saved, t)
    for name, got in zip(want, grads):
        R.close(got.reshape(want[name][0].shape), *want[name], name)
    assert all(p.grad is not None and p.grad.isfinite().all() for p in block.parameters())
    with torch.no_grad():
        for p in block.parameters():
            p.sub_(p.grad, alpha=0.1)
    served = quantize(block, scheme="weight_only_int4", group_size=32, verbose=False)
    assert isinstance(served.gate_up, Int4GatedLinear) and isinstance(served.down, Int4Linear)
    assert isinstance(block.gate_up, GatedLinear)
    one = x[0, :1]
    g4, d4 = served.gate_up, served.down
    h = g4(one)

    def product(v, w, sc, b):
        K = v.shape[1]
        return R.linear(v, R.unpack_int4(w, sc, K, 32), b, R.int4_sizes(sc, K, 32, t), 32)
    R.close_rounded(h, *R.gate_of(product(one, g4.w_gate_int4, g4.w_gate_scale, block.gate_up.b_gate),
                                  product(one, g4.w_up_int4, g4.w_up_scale, block.gate_up.b_up)))
    R.close_rounded(d4(h), *product(h, d4.w_int4, d4.w_scale, d4.bias))
    assert torch.equal(served(one), one + d4(h))
