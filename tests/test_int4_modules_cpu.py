"""The 4-bit and gated modules and their conversion on the CPU: calls that have to be refused before the kernels see them,
with the entry points replaced by stand-ins where a call would reach them."""
import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from forge_b200 import _forge_C as C
from forge_b200.nn import GatedLinear, Int4GatedLinear, Int4Linear, QuantizedLinear, gated_linear
from forge_b200.quant import finalize_qat, quantize


@pytest.fixture
def entry_points(monkeypatch):
    """The forward calls answer with zeros of the right shape and remember what they were given."""
    calls = []

    def answer(name):
        def call(x, w, *args, save=False):
            calls.append((name, x, w, args))
            y = x.new_zeros((x.shape[0], w.shape[0]))
            return (y, y.float(), y.float()) if save else y
        return call
    for name in ("int4_linear", "int4_gated_linear", "gated_linear"):
        monkeypatch.setattr(C, name, answer(name))
    return calls


@pytest.mark.parametrize("features", [64, 72, 136, 264])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("make", [Int4Linear, Int4GatedLinear])
def test_inputs_of_another_width_are_refused(entry_points, make, group, features):
    """Widths in the same last group and block as well, which the packed weight's shape cannot tell from the right one."""
    m = make(features, 24, group_size=group)
    for lead in ((), (3,), (2, 3)):
        assert m(torch.zeros(*lead, features).half()).shape == (*lead, 24)
    seen = len(entry_points)
    for width in (0, 8, features - 8, features - 1, features + 1, features + 8, -(-features // 128) * 128 + 8):
        for lead in ((), (3,), (2, 3), (0,)):
            with pytest.raises(ValueError):
                m(torch.zeros(*lead, width).half())
    with pytest.raises(ValueError):
        m(torch.tensor(1.0).half())
    assert len(entry_points) == seen


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad_mode", [False, True])
@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_tangent_is_not_dropped_by_the_gate(entry_points, which, grad_mode, requires_grad):
    """There is no forward-mode formula: a tangent on any argument raises instead of giving a derivative of zero."""
    args = [torch.zeros(3, 64), torch.zeros(16, 64), torch.zeros(16, 64), torch.zeros(16), torch.zeros(16)]
    args = [t.half().requires_grad_(requires_grad) for t in args]
    with torch.set_grad_enabled(grad_mode):
        gated_linear(*args)
        with forward_ad.dual_level():
            gated_linear(*args)   # no tangent among them
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(NotImplementedError):
                gated_linear(*args)


@pytest.mark.parametrize("grad_mode", [False, True])
def test_a_tangent_is_not_dropped_by_the_gate_module(entry_points, grad_mode):
    m = GatedLinear(64, 16, bias=True)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(2, 3, 64).half(), torch.ones(2, 3, 64).half())
        with pytest.raises(NotImplementedError):
            m(x)


def _layers():
    for make in (Int4Linear, Int4GatedLinear):
        for bias in (False, True):
            yield make(64, 16, bias=bias)


def test_no_gradient_ends_silently_at_a_4_bit_layer(entry_points):
    for m in _layers():
        x = torch.zeros(2, 64).half()
        assert not m(x).requires_grad           # nothing asks for a gradient: the parameters do not by default
        y = m(x.requires_grad_())
        assert y.requires_grad and y.shape == (2, 16)
        with pytest.raises(NotImplementedError):
            y.sum().backward()
        with pytest.raises(NotImplementedError):   # converted on the way
            m(torch.zeros(3, 2, 64, requires_grad=True)).sum().backward()
        with torch.no_grad():
            assert not m(x).requires_grad
        with torch.inference_mode():
            assert not m(x.detach()).requires_grad
        assert all(not p.requires_grad for p in m.parameters())
        for p in m.parameters():
            p.requires_grad_()
            with pytest.raises(NotImplementedError):
                m(x.detach()).sum().backward()
            p.requires_grad_(False)


def test_a_tangent_is_not_dropped_by_a_4_bit_layer(entry_points):
    for m in _layers():
        for grad_mode in (False, True):
            with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
                x = torch.zeros(2, 64).half()
                m(x)
                with pytest.raises(NotImplementedError):
                    m(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("M,N", [(0, 16), (3, 0), (0, 0)])
def test_gradients_that_the_library_does_not_write_are_zero(monkeypatch, M, N):
    """Without tokens or outputs an entry point returns at once; fresh memory may hold anything."""
    monkeypatch.setattr(C, "_act_shape", lambda x: (1, *x.shape))
    monkeypatch.setattr(C, "_chk", lambda *a, **k: None)
    monkeypatch.setattr(C, "_run", lambda *a: None)
    monkeypatch.setattr(torch, "empty_like", lambda t: torch.full_like(t, 7))
    new = lambda *s: torch.zeros(*s).half()  # noqa: E731
    saved = torch.zeros(M, N), torch.zeros(M, N)
    grads = C.gated_linear_backward(new(M, N), new(M, 64), new(N, 64), new(N, 64), *saved)
    assert [tuple(g.shape) for g in grads] == [(M, 64), (N, 64), (N, 64), (N,), (N,)]
    assert all((g == 0).all() for g in grads)


def test_a_model_that_is_a_single_layer_is_converted():
    for layer, scheme, want in ((nn.Linear(64, 24), "weight_only_int4", Int4Linear),
                                (GatedLinear(64, 24, bias=True), "weight_only_int4", Int4GatedLinear),
                                (nn.Linear(20, 24), "weight_only_int4", QuantizedLinear),
                                (nn.Linear(64, 24), "dynamic_int8", QuantizedLinear)):
        out = quantize(layer, scheme=scheme, verbose=False)
        assert type(out) is want and out.out_features == 24
        assert not list(layer.children()) and not list(out.children())
        with pytest.raises(ValueError):   # the caller's object cannot change its class
            quantize(layer, scheme=scheme, inplace=True, verbose=False)
        assert not list(layer.children())
    gate = GatedLinear(64, 24)
    assert quantize(gate, inplace=True, verbose=False) is gate   # which the INT8 schemes leave as it is
    wrapper = nn.Module()
    wrapper.linear, wrapper.weight_fq, wrapper.input_fq = nn.Linear(64, 24), nn.Identity(), nn.Identity()
    assert type(finalize_qat(wrapper, verbose=False)) is QuantizedLinear


def test_an_entry_point_runs_on_its_tensors_device_and_stream(monkeypatch):
    """Tensors of GPU 1 while GPU 0 is current, and of the current one; without a GPU the device switch is a stand-in."""
    from contextlib import contextmanager
    from types import SimpleNamespace
    state, calls = {"device": 0}, []

    @contextmanager
    def device(d):
        before, state["device"] = state["device"], d.index
        yield
        state["device"] = before

    def call(name, *args):
        calls.append((name, state["device"], args))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(C._lib, "call", call)
    monkeypatch.setattr(C._lib, "load", lambda: SimpleNamespace(entry=lambda *a: call("entry", *a) or 0))
    for index in (1, 0):
        C._run(SimpleNamespace(device=SimpleNamespace(index=index)), "entry", 7, 8)
    assert calls == [("entry", 1, (7, 8, 101)), ("entry", 0, (7, 8, 100))] and state["device"] == 0
