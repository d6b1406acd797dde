"""The gated linear layer at the ends of its range (no outputs, gradients far from one in size), compiled, and called first
from several threads."""
import os
import subprocess
import sys

import pytest
import torch
import torch.nn as nn

import float_ref as R
from forge_b200 import _forge_C as C
from forge_b200.nn import GatedLinear, gated_linear
from forge_b200.quant import quantize

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_no_outputs():
    """The gradient of x is an empty sum: zeros, whatever the memory held before."""
    for M, lead in ((5, (5,)), (6, (2, 3)), (0, (0,))):
        x = torch.randn(*lead, 64, device=DEV).half().requires_grad_()
        trash = torch.full((M, 64), 7.0, device=DEV).half()
        del trash   # what the allocator hands out next
        m = GatedLinear(64, 0, bias=True, device=DEV)
        h = m(x)
        assert h.shape == (*lead, 0)
        h.sum().backward()
        assert x.grad.shape == x.shape and (x.grad == 0).all()
        assert m.w_gate.grad.shape == (0, 64) and m.b_up.grad.shape == (0,)
    torch.cuda.synchronize()
    assert C.device_status() == 0


def _gradients(dh, x, wg, wu):
    """{name: (value, bound)} in 64 bits for fp16 calls without biases. dg and du are rounded to 11 bits, or where one lies
    more than 2^29 below the call's largest, in steps of 2^-24 of the power of two below 2^-14 of the latter: half of one
    is at most 2^-39 of the largest. The other terms are those of float_ref.gate_backward."""
    g, eg, u, eu = R.gate(x, wg, wu, None, None)[2]
    dh, x, wg, wu = (t.double() for t in (dh, x, wg, wu))
    s = torch.sigmoid(g)
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    eg, eu = (dh.abs() * (1.1 * eu + 0.5 * eg * (u.abs() + eu))
              + R._fn_rel(g) * 2 * (dh * u * s).abs() * (1 + (g * (1 - s)).abs()) + 2.0 ** -120,
              dh.abs() * 1.1 * eg + R._fn_rel(g) * du.abs() + 2.0 ** -120)
    finite = lambda t: t.nan_to_num(0, 0, 0)  # noqa: E731
    floor = 2.0 ** -39 * torch.maximum(finite(dg.abs() + eg).max(), finite(du.abs() + eu).max())
    rg, ru = (e + (d.abs() + e) * 2.0 ** -11 + floor for d, e in ((dg, eg), (du, eu)))
    (M, N), acc = dh.shape, 2.0 ** -23
    a, b = dg.abs() + rg, du.abs() + ru
    out = {
        "dx": (dg @ wg + du @ wu, rg @ wg.abs() + ru @ wu.abs() + (2 * N + 64) * acc * (a @ wg.abs() + b @ wu.abs())),
        "dwg": (dg.t() @ x, rg.t() @ x.abs() + (M + 64) * acc * (a.t() @ x.abs())),
        "dwu": (du.t() @ x, ru.t() @ x.abs() + (M + 64) * acc * (b.t() @ x.abs())),
    }
    return {k: (v, e + R.half_step(v.abs() + e, torch.float16)) for k, (v, e) in out.items()}


def _fp16_case(M, K, N, seed, x_size, wg_size, wu_size):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, wg, wu, dh = new(M, K) * x_size, new(N, K) * wg_size, new(N, K) * wu_size, new(M, N)
    return [t.half().to(DEV).requires_grad_() for t in (x, wg, wu)], dh.to(DEV)


# gradients as they are behind a mean over many tokens, and as a scaled loss makes them; all subnormal in the last
@pytest.mark.parametrize("size", [1e-2, 1e-4, 1e-5, 1e-6, 1e-7, 100.0, 3000.0])
@pytest.mark.parametrize("M,K,N", [(64, 64, 72), (1000, 72, 264), (2048, 64, 64)])
def test_gradients_of_any_size(M, K, N, size):
    args, dh = _fp16_case(M, K, N, M, 0.3, 0.6 * K ** -0.5, 0.6 * K ** -0.5)
    dh = (dh * size).half()
    got = torch.autograd.grad(gated_linear(*args), args, dh)
    with torch.no_grad():
        want = _gradients(dh, *args)
    for name, t in zip(want, got):
        R.close(t, *want[name], name)


def test_gradients_of_the_gate_beyond_fp16():
    """dh u is up to half a million, the gradients of x and the weights are within fp16's range."""
    args, dh = _fp16_case(48, 64, 64, 5, 2.0 ** -6, 2.0 ** -6, 1000.0)
    dh = (dh * 700).half()
    got = torch.autograd.grad(gated_linear(*args), args, dh)
    with torch.no_grad():
        x, wg, wu = args
        assert (dh.double() * (x.double() @ wu.double().t())).abs().max() > 4 * 65504
        want = _gradients(dh, *args)
        assert all(v.abs().max() < 65504 for v, _ in want.values())
    for name, t in zip(want, got):
        assert t.isfinite().all()
        R.close(t, *want[name], name)


def test_gradients_of_tokens_far_apart_in_size():
    """Token m's gradient is 2^-m of the first one's, down to 2^-24 (subnormal numbers themselves)."""
    args, dh = _fp16_case(25, 64, 72, 7, 1.0, 0.125, 0.125)
    dh = (dh * 2.0 ** -torch.arange(25.0, device=DEV)[:, None]).half()
    got = torch.autograd.grad(gated_linear(*args), args, dh)
    with torch.no_grad():
        want = _gradients(dh, *args)
    for name, t in zip(want, got):
        R.close(t, *want[name], name)


def test_no_gradient_and_infinite_gradients():
    args, dh = _fp16_case(40, 64, 72, 9, 1.0, 0.125, 0.125)
    dh = (dh * 1e-6).half()
    h = gated_linear(*args)
    assert all((t == 0).all() for t in torch.autograd.grad(h, args, torch.zeros_like(dh), retain_graph=True))
    dh[3] = 0
    want = torch.autograd.grad(h, args, dh, retain_graph=True)
    for bad in (float("inf"), float("nan")):
        dh[3, 70] = bad
        dx, dwg, dwu = torch.autograd.grad(h, args, dh, retain_graph=True)
        rows = [m for m in range(40) if m != 3]
        outs = [n for n in range(72) if n != 70]
        assert torch.equal(dx[rows], want[0][rows]) and not dx[3].isfinite().any()
        assert torch.equal(dwg[outs], want[1][outs]) and torch.equal(dwu[outs], want[2][outs])
        assert not dwg[70].isfinite().any() and not dwu[70].isfinite().any()


def test_a_compiled_block_is_the_block():
    """Dynamo breaks its graph around the library's calls; results and gradients are those of the uncompiled module."""
    torch.manual_seed(0)
    block = nn.Sequential(nn.Linear(128, 64, device=DEV, dtype=torch.float16), GatedLinear(64, 264, bias=True, device=DEV),
                          nn.Linear(264, 128, device=DEV, dtype=torch.float16))
    x = torch.randn(3, 40, 128, device=DEV).half()

    def step(f):
        block.zero_grad()
        y = f(x)
        y.float().square().sum().backward()
        return [y.detach(), *(p.grad for p in block.parameters())]
    want = step(block)
    torch._dynamo.reset()
    fast = torch.compile(block, backend="eager")
    assert all(torch.equal(a, b) for a, b in zip(step(fast), want))
    served = quantize(block, scheme="weight_only_int4", group_size=32, verbose=False)
    with torch.no_grad():
        assert torch.equal(torch.compile(served, backend="eager")(x), served(x))
    torch._dynamo.reset()


_THREADS = """
import sys, threading, torch
sys.path.insert(0, sys.argv[1])
from forge_b200 import _forge_C as C
from forge_b200.nn import gated_linear
def step(seed):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=gen).half().cuda()
    x, wg, wu, dh = new(40, 64), new(72, 64), new(72, 64), new(40, 72)
    a = [t.requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(gated_linear(*a), a, dh)
    with torch.no_grad():
        w, s = C.prepare_weight_int4(wg, 32)
        few = C.int4_linear(x[:3], w, s, None, 32)
        return [*grads, gated_linear(x[:3], wg, wu), few, C.int4_linear(x, w, s, None, 32),
                C.int4_gated_linear(x[:3], w, w, s, s, None, None, 32)]
start, got = threading.Barrier(4), [None] * 4
def work(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        got[i] = step(i)
        torch.cuda.current_stream().synchronize()
torch.zeros(1, device="cuda")
threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[t.start() for t in threads]
[t.join() for t in threads]
for i in range(4):
    assert all(torch.equal(a, b) for a, b in zip(got[i], step(i))), i
torch.cuda.synchronize()
assert C.device_status() == 0
print("threads ok")
"""


def test_first_calls_of_several_threads():
    """A process whose first calls come from four threads at once."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", _THREADS, root], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "threads ok" in run.stdout, run.stderr[-2000:]
