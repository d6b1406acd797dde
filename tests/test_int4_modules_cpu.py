"""The 4-bit and gated modules and their conversion on the CPU: calls that have to be refused before the kernels see them,
with the entry points replaced by stand-ins where a call would reach them."""
import pytest
import torch

from forge_b200 import _forge_C as C
from forge_b200.nn import Int4GatedLinear, Int4Linear


@pytest.fixture
def entry_points(monkeypatch):
    """The inference calls answer with zeros of the right shape and remember what they were given."""
    calls = []

    def answer(name, outputs):
        def call(x, *args):
            calls.append((name, x, args))
            return x.new_zeros((x.shape[0], outputs(args)))
        return call
    monkeypatch.setattr(C, "int4_linear", answer("int4_linear", lambda a: a[0].shape[0]))
    monkeypatch.setattr(C, "int4_gated_linear", answer("int4_gated_linear", lambda a: a[0].shape[0]))
    monkeypatch.setattr(C, "gated_linear", answer("gated_linear", lambda a: a[0].shape[0]))
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
