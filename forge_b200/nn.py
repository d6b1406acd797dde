"""Drop-in INT8 linear modules on the forge_b200 kernels.

Mirror of the reference's `forge.nn.QuantizedLinear` and `forge.nn.SparseLinear`
(python/forge/nn/linear.py:135-254): same constructor arguments, same registered buffers and
parameters with the same names, dtypes and layouts (`w_int8`, `w_scale`, `bias`; `W_comp`,
`w_meta` int32, `w_scale`, `bias`), so state_dicts written by either implementation load into
the other. Weight quantisation is the reference's recipe (per output channel, absmax / 127,
round half to even, clamp to +-127, scale stored as fp16).

Without a counterpart there: `Int4Linear` (4-bit weights with group scales, for decoding), `GatedLinear` (the
gate of a Llama-style MLP on unquantized weights, trainable) and `Int4GatedLinear`, which serves the latter.

Beyond the reference: inputs with more than two dimensions are flattened over the leading
dimensions, non-contiguous inputs are made contiguous, and `SparseLinear.from_dense_weight`
prunes on the module's own device instead of assuming "cuda".
"""
import math

import numpy as np
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _forge_C as _C


def quantize_weight_per_channel(weight_fp):
    """(N, K) float weight -> (int8 (N, K), fp16 scales (N)); linear.py:167-173."""
    w = weight_fp.detach().to(torch.float32)
    scale = w.abs().amax(dim=1).clamp(min=1e-8) / 127.0
    q = torch.clamp(torch.round(w / scale.unsqueeze(1)), -127, 127).to(torch.int8)
    return q, scale.to(torch.float16)


class _Int8LinearFn(torch.autograd.Function):
    """Forward on the INT8 tensor-core path; backward through the dequantised weight in fp16,
    as the reference does (linear.py:123-132)."""

    @staticmethod
    def forward(ctx, x, w_int8, w_scale, bias, scratch_q, scratch_s):
        out = _C.int8_linear(x, w_int8, w_scale, bias, scratch_q, scratch_s)
        ctx.save_for_backward(x, w_int8, w_scale)
        ctx.has_bias = bias is not None
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x, w_int8, w_scale = ctx.saved_tensors
        g = grad_out.to(torch.float16)
        w = w_int8.to(torch.float16) * w_scale.unsqueeze(1)
        grad_bias = g.sum(dim=0) if ctx.has_bias else None
        return g @ w, None, None, grad_bias, None, None


class _ScratchMixin:
    def _scratch(self, M, K, device):
        q = getattr(self, "_scratch_q", None)
        if q is None or q.shape[0] < M or q.shape[1] != K or q.device != device:
            self._scratch_q = torch.empty((M, K), dtype=torch.int8, device=device)
            self._scratch_s = torch.empty((M,), dtype=torch.float32, device=device)
        return self._scratch_q, self._scratch_s

    @staticmethod
    def _as_rows(x):
        lead = x.shape[:-1]
        x2 = x.reshape(-1, x.shape[-1])
        if x2.dtype != torch.float16:
            x2 = x2.to(torch.float16)
        return x2.contiguous(), lead


class QuantizedLinear(nn.Module, _ScratchMixin):
    """W8A8 linear layer: per-token activation quantisation + dense INT8 GEMM + dequant + bias."""

    def __init__(self, in_features, out_features, bias=True):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("w_int8", torch.zeros(out_features, in_features, dtype=torch.int8))
        self.w_scale = nn.Parameter(torch.ones(out_features, dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=torch.float16))
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        x2, lead = self._as_rows(x)
        q, s = self._scratch(x2.shape[0], x2.shape[1], x2.device)
        y = _Int8LinearFn.apply(x2, self.w_int8, self.w_scale, self.bias, q, s)
        return y.reshape(*lead, self.out_features)

    @torch.no_grad()
    def quantize_weight(self, weight_fp):
        if self.w_int8.is_cuda and weight_fp.shape[1] % 32 == 0:
            # one kernel on the module's device (IEEE arithmetic: bit-identical to torch on the CPU)
            q, _, _, scale = _C.prepare_weight(weight_fp.detach().to(self.w_int8.device), sparse=False)
        else:
            # any in_features, as the reference accepts (linear.py:167-173); the kernel walks 32-wide runs
            q, scale = quantize_weight_per_channel(weight_fp.detach().to(self.w_int8.device))
        self.w_int8.copy_(q)
        self.w_scale.data.copy_(scale)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class SparseLinear(nn.Module, _ScratchMixin):
    """W8A8 linear layer with a 2:4 structured-sparse weight (inference only)."""

    def __init__(self, in_features, out_features, bias=True):
        super().__init__()
        if in_features % 64 != 0 or out_features % 16 != 0:
            raise ValueError("SparseLinear needs in_features % 64 == 0 and out_features % 16 == 0")
        self.in_features, self.out_features = in_features, out_features
        self.register_buffer("W_comp", torch.zeros(out_features, in_features // 2, dtype=torch.int8))
        self.register_buffer("w_meta", torch.zeros(out_features, in_features // 32, dtype=torch.int32))
        self.w_scale = nn.Parameter(torch.ones(out_features, dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=torch.float16))
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        x2, lead = self._as_rows(x)
        q, s = self._scratch(x2.shape[0], x2.shape[1], x2.device)
        y = _C.sparse_int8_linear(x2, self.W_comp, self.w_meta, self.w_scale.detach(),
                                  None if self.bias is None else self.bias.detach(), q, s, None, 0)
        return y.reshape(*lead, self.out_features)

    @torch.no_grad()
    def from_dense_weight(self, weight_fp):
        """Quantise, prune 2:4 by magnitude, compress and pack (linear.py:234-249)."""
        dev = self.W_comp.device
        if dev.type != "cuda":
            raise RuntimeError("move the module to a CUDA device before from_dense_weight()")
        # one kernel: per-channel quantisation + 2:4 prune + compress + metadata pack
        _, comp, meta, scale = _C.prepare_weight(weight_fp.detach().to(dev), sparse=True)
        self.W_comp.copy_(comp)
        self.w_meta.copy_(meta)
        self.w_scale.data.copy_(scale)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, sparse=2:4")


def quantize_weight_int4(weight_fp, group_size=128):
    """(N, K) float weight -> (w_int4, w_scale) as `_forge_C.prepare_weight_int4` gives them, on any device."""
    w = weight_fp.detach()
    if w.is_cuda:
        return _C.prepare_weight_int4(w, group_size)
    _C._check_group(group_size)
    if w.dim() != 2 or w.size(1) == 0 or w.size(1) % 8 != 0:
        raise ValueError(f"weight: expected (outputs, inputs) with inputs a positive multiple of 8, got {tuple(w.shape)}")
    N, K = w.shape
    groups = -(-K // group_size)
    w = torch.nn.functional.pad(w.to(torch.float32).to(torch.float64), (0, groups * group_size - K)).view(N, groups, group_size)
    with np.errstate(over="ignore"):   # beyond fp16: infinity, which becomes NaN below
        s = torch.from_numpy((w.abs().amax(2) / 7).numpy().astype(np.float16))   # one rounding
    s[~torch.isfinite(s)] = float("nan")
    q = torch.clamp(torch.round(w / s.to(torch.float64)[:, :, None]), -7, 7)
    q[~(s > 0)] = 0
    q = torch.nn.functional.pad(q.to(torch.int64).view(N, -1)[:, :K], (0, -K % 128)) + 8
    # blocks of 128: run 4j + t of eight weights is word 4t + j; weight 2i in nibble i, weight 2i + 1 in nibble i + 4
    q = q.view(N, -1, 4, 4, 4, 2).transpose(2, 3).transpose(4, 5).reshape(N, -1, 2)
    return (q[..., 0] | q[..., 1] << 4).to(torch.uint8), s.t().contiguous()


def _check_weight(module, *weights):
    for w in weights:
        if w.shape != (module.out_features, module.in_features):
            raise ValueError(f"weight: expected shape {(module.out_features, module.in_features)}, got {tuple(w.shape)}")


def _as_16bit_rows(x, features, dtype):
    """x as contiguous (rows, features) in fp16 or bf16 (other types are converted to `dtype`), and its leading sizes.
    The packed weight does not tell the number of inputs, only that of its groups and blocks: it is checked here."""
    if x.shape[-1:] != (features,):
        raise ValueError(f"x: expected (..., {features}), got {tuple(x.shape)}")
    if x.dtype not in (torch.float16, torch.bfloat16):
        x = x.to(dtype)
    return x.reshape(-1, x.shape[-1]).contiguous(), x.shape[:-1]


def _has_tangent(tensors):
    """Whether forward-mode differentiation is under way and one of `tensors` (or None) carries a tangent."""
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _InferenceOnlyFn(torch.autograd.Function):
    """A call that has no derivative, kept in the graph so that a backward pass through it raises (as forward mode does, for
    want of a formula) instead of ending there and leaving every gradient before it out."""

    @staticmethod
    def forward(ctx, call, *args):
        return call(*args)

    @staticmethod
    def backward(ctx, dy):
        raise NotImplementedError("4-bit layers are for inference only: no gradient passes through them")


def _inference_only(call, x, *args):
    """call(x, *args) for the tensors or None in `args`."""
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, *args))) or _has_tangent((x, *args)):
        return _InferenceOnlyFn.apply(call, x, *args)
    return call(x, *args)


class Int4Linear(nn.Module):
    """Linear layer on 4-bit weights with one fp16 scale per `group_size` inputs; activations stay fp16 or bf16. Inference
    only: a backward pass through it raises, and its bias asks for no gradient. Built for few tokens, where its time is
    that of reading the weight; any number runs."""

    def __init__(self, in_features, out_features, bias=True, group_size=128, dtype=torch.float16):
        super().__init__()
        if in_features % 8 != 0:
            raise ValueError("Int4Linear needs in_features % 8 == 0")
        if group_size not in (32, 64, 128):
            raise ValueError("Int4Linear needs group_size 32, 64 or 128")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        self.dtype = dtype
        self.register_buffer("w_int4", torch.full((out_features, -(-in_features // 128) * 64), 0x88, dtype=torch.uint8))
        self.register_buffer("w_scale", torch.ones(-(-in_features // group_size), out_features, dtype=torch.float16))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, dtype=dtype), requires_grad=False)
        else:
            self.register_parameter("bias", None)

    def forward(self, x):
        x2, lead = _as_16bit_rows(x, self.in_features, self.dtype)
        bias = None if self.bias is None else self.bias.to(x2.dtype)
        y = _inference_only(self._run, x2, bias)
        return y.reshape(*lead, self.out_features)

    def _run(self, x, bias):
        return _C.int4_linear(x, self.w_int4, self.w_scale, bias, self.group_size)

    @torch.no_grad()
    def quantize_weight(self, weight_fp):
        _check_weight(self, weight_fp)
        w, s = quantize_weight_int4(weight_fp.to(self.w_int4.device), self.group_size)
        self.w_int4.copy_(w)
        self.w_scale.copy_(s)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, group_size={self.group_size}")


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up):
        h, g, u = _C.gated_linear(x, w_gate, w_up, b_gate, b_up, save=True)
        ctx.save_for_backward(x, w_gate, w_up, g, u)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, g, u = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _C.gated_linear_backward(dh.contiguous(), x, w_gate, w_up, g, u, need[0], need[1] or need[2],
                                         need[3] or need[4])
        return tuple(d if n else None for d, n in zip(grads, need))


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None):
    """SiLU(x w_gate^T + b_gate) * (x w_up^T + b_up), differentiable in every argument by backward passes (forward mode
    raises). x (..., K), weights (N, K), biases (N), all fp16 or all bf16, K and N multiples of 8. In training the two
    products are kept in fp32.

    A step can be captured into a CUDA graph. As with every autograd operation, no graph recorded outside the capture may
    then still be alive for the same leaves: its gradient accumulators belong to the stream it was recorded on."""
    flat = x.dim() == 2   # no reshapes then: each would be a node of its own in the backward pass
    x2 = (x if flat else x.reshape(-1, x.shape[-1])).contiguous()
    w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    args = (x2, w_gate, w_up, b_gate, b_up)
    # with a tangent `apply` raises, as there is no forward-mode formula; the bare call would drop it
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args)) or _has_tangent(args):
        h = _GatedLinearFn.apply(*args)
    else:
        h = _C.gated_linear(*args)
    return h if flat else h.reshape(*x.shape[:-1], w_gate.shape[0])


class GatedLinear(nn.Module):
    """The gate of a Llama-style MLP, SiLU(gate(x)) * up(x), on fp16 / bf16 weights: one kernel forward, trainable.
    `forge_b200.quant.quantize(model, scheme="weight_only_int4")` turns it into an `Int4GatedLinear`."""

    def __init__(self, in_features, out_features, bias=False, dtype=torch.float16, device=None):
        super().__init__()
        if in_features % 8 != 0 or out_features % 8 != 0:
            raise ValueError("GatedLinear needs in_features % 8 == 0 and out_features % 8 == 0")
        self.in_features, self.out_features = in_features, out_features
        new = lambda *s: nn.Parameter(torch.empty(*s, dtype=dtype, device=device))  # noqa: E731
        self.w_gate, self.w_up = new(out_features, in_features), new(out_features, in_features)
        if bias:
            self.b_gate, self.b_up = new(out_features), new(out_features)
        else:
            self.register_parameter("b_gate", None)
            self.register_parameter("b_up", None)
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1 / math.sqrt(self.in_features)   # as nn.Linear
        for p in self.parameters():
            nn.init.uniform_(p, -bound, bound)

    def forward(self, x):
        return gated_linear(x.to(self.w_gate.dtype), self.w_gate, self.w_up, self.b_gate, self.b_up)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.b_gate is not None}"


class Int4GatedLinear(nn.Module):
    """SiLU(gate(x)) * up(x) on 4-bit weights, one kernel. Inference only: a backward pass through it raises, and its biases
    ask for no gradient."""

    def __init__(self, in_features, out_features, bias=False, group_size=128, dtype=torch.float16):
        super().__init__()
        if in_features % 8 != 0:
            raise ValueError("Int4GatedLinear needs in_features % 8 == 0")
        if group_size not in (32, 64, 128):
            raise ValueError("Int4GatedLinear needs group_size 32, 64 or 128")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        self.dtype = dtype
        for k in ("gate", "up"):
            self.register_buffer(f"w_{k}_int4",
                                 torch.full((out_features, -(-in_features // 128) * 64), 0x88, dtype=torch.uint8))
            self.register_buffer(f"w_{k}_scale",
                                 torch.ones(-(-in_features // group_size), out_features, dtype=torch.float16))
            if bias:
                self.register_parameter(f"b_{k}", nn.Parameter(torch.zeros(out_features, dtype=dtype), requires_grad=False))
            else:
                self.register_parameter(f"b_{k}", None)

    def forward(self, x):
        x2, lead = _as_16bit_rows(x, self.in_features, self.dtype)
        bg, bu = (None if b is None else b.to(x2.dtype) for b in (self.b_gate, self.b_up))
        h = _inference_only(self._run, x2, bg, bu)
        return h.reshape(*lead, self.out_features)

    def _run(self, x, bg, bu):
        return _C.int4_gated_linear(x, self.w_gate_int4, self.w_up_int4, self.w_gate_scale, self.w_up_scale, bg, bu,
                                    self.group_size)

    @torch.no_grad()
    def quantize_weight(self, w_gate_fp, w_up_fp):
        _check_weight(self, w_gate_fp, w_up_fp)
        for k, w in (("gate", w_gate_fp), ("up", w_up_fp)):
            q, s = quantize_weight_int4(w.to(self.w_gate_int4.device), self.group_size)
            getattr(self, f"w_{k}_int4").copy_(q)
            getattr(self, f"w_{k}_scale").copy_(s)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.b_gate is not None}, "
                f"group_size={self.group_size}")
