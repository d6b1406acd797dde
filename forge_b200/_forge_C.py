"""Python-level mirror of the reference's `forge._forge_C` extension functions for the
quantized-inference path (reference python/forge/csrc/bindings.cpp:446-575): same names,
argument lists and return values, taking torch CUDA tensors and running on torch's current
stream. Each function forwards to the C ABI of libforge_b200.so through ctypes.
"""
import contextlib

import torch

from . import _lib

_NULL = contextlib.nullcontext()


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _stream():
    # the handle itself: building a torch.cuda.Stream object first takes 3 us
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _on(t):
    """Context in which `t`'s GPU is the current device: the library launches on the current
    device and keys its per-device state (SM count, status word, kernel attributes) on it."""
    if t.device.index == torch.cuda.current_device():
        return _NULL
    return torch.cuda.device(t.device)


def _chk(first, **named):
    """Every tensor argument must be a contiguous CUDA tensor of the stated dtype on `first`'s device
    (None is allowed for optional ones). The C ABI takes raw pointers, so a wrong dtype or a strided
    view would be reinterpreted silently; the reference binding's typed data_ptr<T>() raises instead."""
    if not first.is_cuda:
        raise ValueError("forge_b200 runs on CUDA tensors only (there is no CPU path)")
    for name, (t, dtype) in named.items():
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
        if t.device != first.device:
            raise ValueError(f"{name}: on {t.device}, expected {first.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name}: must be contiguous")


_f16, _f32, _i8, _i32, _u8 = torch.float16, torch.float32, torch.int8, torch.int32, torch.uint8


def fused_quantize_activation(input, M, K):
    """bindings.cpp:448-459 -> (int8 (M,K), float32 (M,))."""
    _chk(input, input=(input, _f16))
    output = torch.empty((M, K), dtype=torch.int8, device=input.device)
    scales = torch.empty((M,), dtype=torch.float32, device=input.device)
    with _on(input):
        _lib.call("forge_fused_quantize_activation", _ptr(input), _ptr(output), _ptr(scales), M, K, _stream())
    return output, scales


def fused_dequantize_bias(input, act_scale, w_scale, bias, M, N):
    """bindings.cpp:461-476 -> float16 (M,N)."""
    _chk(input, input=(input, _i32), act_scale=(act_scale, _f32), w_scale=(w_scale, _f16), bias=(bias, _f16))
    output = torch.empty((M, N), dtype=torch.float16, device=act_scale.device)
    with _on(input):
        _lib.call("forge_fused_dequantize_bias", _ptr(input), _ptr(act_scale), _ptr(w_scale), _ptr(bias),
                  _ptr(output), M, N, _stream())
    return output


def int8_linear(x, w_int8, w_scale, bias, scratch_a_int8, scratch_a_scale):
    """bindings.cpp:498-519 -> float16 (M,N)."""
    _chk(x, x=(x, _f16), w_int8=(w_int8, _i8), w_scale=(w_scale, _f16), bias=(bias, _f16),
         scratch_a_int8=(scratch_a_int8, _i8), scratch_a_scale=(scratch_a_scale, _f32))
    M, K, N = x.size(0), x.size(1), w_int8.size(0)
    output = torch.empty((M, N), dtype=x.dtype, device=x.device)
    with _on(x):
        _lib.call("forge_int8_linear", _ptr(x), _ptr(w_int8), _ptr(w_scale), _ptr(bias), _ptr(output), M, K, N,
                  _ptr(scratch_a_int8), _ptr(scratch_a_scale), _stream())
    return output


def sparse_int8_linear(x, W_comp, w_meta, w_scale, bias, scratch_x_int8, scratch_x_scale, splitk_workspace=None,
                       split_k=1, path=-1):
    """bindings.cpp:521-554 -> float16 (M,N_out). The workspace is accepted for compatibility;
    this implementation never splits K, so none is allocated."""
    _chk(x, x=(x, _f16), W_comp=(W_comp, _i8), w_meta=(w_meta, _i32), w_scale=(w_scale, _f16), bias=(bias, _f16),
         scratch_x_int8=(scratch_x_int8, _i8), scratch_x_scale=(scratch_x_scale, _f32),
         splitk_workspace=(splitk_workspace, _f32))
    M, K, N_out = x.size(0), x.size(1), W_comp.size(0)
    output = torch.empty((M, N_out), dtype=x.dtype, device=x.device)
    with _on(x):
        _lib.call("forge_sparse_int8_linear", _ptr(x), _ptr(W_comp), _ptr(w_meta), _ptr(w_scale), _ptr(bias),
                  _ptr(output), M, K, N_out, _ptr(scratch_x_int8), _ptr(scratch_x_scale), _ptr(splitk_workspace),
                  split_k, _stream(), path)
    return output


def prune_compress_24(weight, compressed, metadata_raw, N, K):
    """bindings.cpp:558-566."""
    _chk(weight, weight=(weight, _i8), compressed=(compressed, _i8), metadata_raw=(metadata_raw, _u8))
    with _on(weight):
        _lib.call("forge_prune_compress_24", _ptr(weight), _ptr(compressed), _ptr(metadata_raw), N, K, _stream())


def pack_metadata(meta_raw, meta_packed, N, K):
    """bindings.cpp:568-575."""
    _chk(meta_raw, meta_raw=(meta_raw, _u8), meta_packed=(meta_packed, _i32))
    with _on(meta_raw):
        _lib.call("forge_pack_metadata", _ptr(meta_raw), _ptr(meta_packed), N, K, _stream())


# ---- additive entry points (no counterpart in the reference extension) ----

def int8_gemm_dequant(A, B, act_scale, w_scale, bias=None):
    M, K, N = A.size(0), A.size(1), B.size(0)
    _chk(A, A=(A, _i8), B=(B, _i8), act_scale=(act_scale, _f32), w_scale=(w_scale, _f16), bias=(bias, _f16))
    output = torch.empty((M, N), dtype=torch.float16, device=A.device)
    with _on(A):
        _lib.call("forge_int8_gemm_dequant", _ptr(A), _ptr(B), _ptr(act_scale), _ptr(w_scale), _ptr(bias),
                  _ptr(output), M, K, N, _stream())
    return output


def int8_gemm_s32(A, B):
    M, K, N = A.size(0), A.size(1), B.size(0)
    _chk(A, A=(A, _i8), B=(B, _i8))
    output = torch.empty((M, N), dtype=torch.int32, device=A.device)
    with _on(A):
        _lib.call("forge_int8_gemm_s32", _ptr(A), _ptr(B), _ptr(output), M, K, N, _stream())
    return output


def sparse_int8_gemm(W_comp, x_int8, w_meta, act_scale, w_scale, bias=None, tile=-1):
    M, K, N_out = x_int8.size(0), x_int8.size(1), W_comp.size(0)
    _chk(x_int8, W_comp=(W_comp, _i8), x_int8=(x_int8, _i8), w_meta=(w_meta, _i32), act_scale=(act_scale, _f32),
         w_scale=(w_scale, _f16), bias=(bias, _f16))
    output = torch.empty((M, N_out), dtype=torch.float16, device=x_int8.device)
    with _on(x_int8):
        _lib.call("forge_sparse_int8_gemm", _ptr(W_comp), _ptr(x_int8), _ptr(w_meta), _ptr(act_scale), _ptr(w_scale),
                  _ptr(bias), _ptr(output), M, K, N_out, 0, 1, _stream(), tile)
    return output


def sparse_int8_gemm_s32(W_comp, x_int8, w_meta):
    M, K, N_out = x_int8.size(0), x_int8.size(1), W_comp.size(0)
    _chk(x_int8, W_comp=(W_comp, _i8), x_int8=(x_int8, _i8), w_meta=(w_meta, _i32))
    output = torch.empty((M, N_out), dtype=torch.int32, device=x_int8.device)
    with _on(x_int8):
        _lib.call("forge_sparse_int8_gemm_s32", _ptr(W_comp), _ptr(x_int8), _ptr(w_meta), _ptr(output), M, K, N_out,
                  _stream())
    return output


def prepare_weight(weight, sparse):
    """Float weight (N, K), fp32 or fp16, on a GPU -> (w_int8 or None, W_comp or None, w_meta or None,
    w_scale fp16) in one kernel: per-channel quantisation and, with sparse=True, 2:4 prune +
    compress + metadata pack."""
    if weight.dtype not in (torch.float32, torch.float16):
        weight = weight.to(torch.float32)
    weight = weight.contiguous()
    N, K = weight.shape
    dev = weight.device
    w_scale = torch.empty((N,), dtype=torch.float16, device=dev)
    w_int8 = None if sparse else torch.empty((N, K), dtype=torch.int8, device=dev)
    W_comp = torch.empty((N, K // 2), dtype=torch.int8, device=dev) if sparse else None
    w_meta = torch.empty((N, K // 32), dtype=torch.int32, device=dev) if sparse else None
    with _on(weight):
        _lib.call("forge_prepare_weight", _ptr(weight), 1 if weight.dtype == torch.float16 else 0, _ptr(w_int8),
                  _ptr(W_comp), _ptr(w_meta), _ptr(w_scale), N, K, _stream())
    return w_int8, W_comp, w_meta, w_scale


def int8_conv2d_forward(input, weight, w_scale, bias, kernel_size, padding=(0, 0), stride=(1, 1), dilation=(1, 1)):
    """INT8 conv2d (forge::nn::int8_conv2d_forward; the reference has no Python binding for it): input
    (N,C_in,H,W) fp16, weight (C_out, C_in*kH*kW) int8, w_scale / bias (C_out) fp16 -> (N,C_out,H_out,W_out)
    fp16, each output position's patch quantized per row."""
    N, C_in, H, W = input.shape
    C_out = weight.shape[0]
    (kH, kW), (pH, pW), (sH, sW), (dH, dW) = kernel_size, padding, stride, dilation
    Ho = (H + 2 * pH - dH * (kH - 1) - 1) // sH + 1
    Wo = (W + 2 * pW - dW * (kW - 1) - 1) // sW + 1
    out = torch.empty((N, C_out, Ho, Wo), dtype=torch.float16, device=input.device)
    _chk(input, input=(input, _f16), weight=(weight, _i8), w_scale=(w_scale, _f16), bias=(bias, _f16))
    with _on(input):
        _lib.call("forge_int8_conv2d_forward", _ptr(input), _ptr(weight), _ptr(w_scale), _ptr(bias), _ptr(out), N, C_in,
                  H, W, C_out, kH, kW, pH, pW, sH, sW, dH, dW, None, _stream())
    return out


def int8_conv_transpose2d_k2s2_forward(input, weight, w_scale, bias):
    """2x2 stride-2 INT8 transposed conv (forge::nn::int8_conv_transpose2d_k2s2_forward): weight
    (4*C_out, C_in) int8 with row co*4 + kh*2 + kw -> (N,C_out,2H,2W) fp16."""
    N, C_in, H, W = input.shape
    C_out = weight.shape[0] // 4
    out = torch.empty((N, C_out, 2 * H, 2 * W), dtype=torch.float16, device=input.device)
    _chk(input, input=(input, _f16), weight=(weight, _i8), w_scale=(w_scale, _f16), bias=(bias, _f16))
    with _on(input):
        _lib.call("forge_int8_conv_transpose2d_k2s2_forward", _ptr(input), _ptr(weight), _ptr(w_scale), _ptr(bias),
                  _ptr(out), N, C_in, H, W, C_out, None, _stream())
    return out


_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # FORGE_DTYPE_*
_DTYPES16 = {torch.float16: 1, torch.bfloat16: 2}
_GROUPS = (32, 64, 128)
_BYTES_PER_BLOCK = 64   # packed 4-bit weights: 128 inputs
_MAX_SIZE = 1 << 30      # of one dimension, as the library checks it


def _act_shape(x):
    """FORGE_DTYPE_* and shape of a contiguous 2-D fp16 / bf16 CUDA activation whose row length the kernels take."""
    dtype = _DTYPES16.get(x.dtype)
    if dtype is None:
        raise TypeError(f"x: expected torch.float16 or torch.bfloat16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError("forge_b200 runs on CUDA tensors only (there is no CPU path)")
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0 or shape[1] % 8 != 0:
        raise ValueError(f"x: expected (tokens, inputs) with inputs a positive multiple of 8, got {tuple(shape)}")
    if shape[0] > _MAX_SIZE or shape[1] > _MAX_SIZE:
        raise ValueError(f"x: at most {_MAX_SIZE} rows and columns, got {tuple(shape)}")
    if not x.is_contiguous():
        raise ValueError("x: must be contiguous")
    return dtype, shape[0], shape[1]


def _run(t, name, *args):
    """An entry point on `t`'s GPU and its current stream, which goes in as the last argument."""
    index = t.device.index
    if index == torch.cuda.current_device():
        status = getattr(_lib.load(), name)(*args, torch._C._cuda_getCurrentRawStream(index))
        if status:
            _lib.check(status, name)
    else:
        with torch.cuda.device(t.device):
            _lib.call(name, *args, _stream())


def _shape(**named):
    for name, (t, shape) in named.items():
        if t is not None and t.shape != shape:
            raise ValueError(f"{name}: expected shape {shape}, got {tuple(t.shape)}")


def _aligned(t):
    """`t` at a 16-byte aligned address (a view into a larger buffer may start anywhere)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_group(group_size):
    if group_size not in _GROUPS:
        raise ValueError(f"group_size: expected 32, 64 or 128, got {group_size}")


def prepare_weight_int4(weight, group_size=128):
    """Float weight (N, K) on a GPU -> (w_int4 uint8 (N, ceil(K / 128) * 64), w_scale fp16 (ceil(K / group_size), N)):
    4-bit integers in the layout of include/forge_b200.h with one scale per group of 32, 64 or 128 inputs."""
    if weight.dtype not in _DTYPES:
        weight = weight.to(torch.float32)
    weight = weight.contiguous()
    _chk(weight)
    _check_group(group_size)
    if weight.dim() != 2 or weight.size(1) == 0 or weight.size(1) % 8 != 0:
        raise ValueError(f"weight: expected (outputs, inputs) with inputs a positive multiple of 8, got {tuple(weight.shape)}")
    weight = _aligned(weight)
    N, K = weight.shape
    w_int4 = torch.empty((N, (K + 127) // 128 * _BYTES_PER_BLOCK), dtype=_u8, device=weight.device)
    w_scale = torch.empty(((K + group_size - 1) // group_size, N), dtype=_f16, device=weight.device)
    _run(weight, "forge_prepare_weight_int4", _ptr(weight), _DTYPES[weight.dtype], _ptr(w_int4), _ptr(w_scale), N, K,
         group_size)
    return w_int4, w_scale


def _int4_operand(x, K, name, w, s, b, N, group_size):
    """Checks one 4-bit weight with its scales and bias against x (M, K) and N outputs; returns their addresses."""
    if w.dtype is not _u8 or s.dtype is not _f16 or (b is not None and b.dtype is not x.dtype):
        raise TypeError(f"{name}_int4, {name}_scale, bias: expected {_u8}, {_f16}, {x.dtype}, "
                        f"got {w.dtype}, {s.dtype}, {None if b is None else b.dtype}")
    if w.shape != (N, (K + 127) // 128 * _BYTES_PER_BLOCK) or s.shape != ((K + group_size - 1) // group_size, N) or (
            b is not None and b.shape != (N,)):
        raise ValueError(f"{name}_int4 {tuple(w.shape)}, {name}_scale {tuple(s.shape)}, bias "
                         f"{None if b is None else tuple(b.shape)} do not fit {K} inputs in groups of {group_size}, {N} outputs")
    dev = x.device
    if w.device != dev or s.device != dev or (b is not None and b.device != dev):
        raise ValueError(f"{name}_int4, {name}_scale and bias must be on {dev}")
    if not (w.is_contiguous() and s.is_contiguous() and (b is None or b.is_contiguous())):
        raise ValueError(f"{name}_int4, {name}_scale and bias must be contiguous")
    pw, ps = w.data_ptr(), s.data_ptr()
    if pw & 15 or ps & 3:
        raise ValueError(f"{name}_int4 must start at a 16-byte aligned address, {name}_scale at a 4-byte aligned one")
    return pw, ps, 0 if b is None else b.data_ptr()


def int4_linear(x, w_int4, w_scale, bias=None, group_size=128):
    """x (M, K) fp16 / bf16 times a 4-bit weight (prepare_weight_int4) plus bias (N) of x's type -> (M, N)."""
    dtype, M, K = _act_shape(x)
    _check_group(group_size)
    N = w_int4.shape[0]
    w, s, b = _int4_operand(x, K, "w", w_int4, w_scale, bias, N, group_size)
    x = _aligned(x)
    output = x.new_empty((M, N))
    _run(x, "forge_int4_linear", x.data_ptr(), w, s, b, output.data_ptr(), M, K, N, group_size, dtype)
    return output


def int4_gated_linear(x, wg_int4, wu_int4, wg_scale, wu_scale, bg=None, bu=None, group_size=128):
    """SiLU(x Wg^T + bg) * (x Wu^T + bu) for 4-bit weights, one kernel -> (M, N)."""
    dtype, M, K = _act_shape(x)
    _check_group(group_size)
    N = wg_int4.shape[0]
    wg, sg, pg = _int4_operand(x, K, "wg", wg_int4, wg_scale, bg, N, group_size)
    wu, su, pu = _int4_operand(x, K, "wu", wu_int4, wu_scale, bu, N, group_size)
    x = _aligned(x)
    output = x.new_empty((M, N))
    _run(x, "forge_int4_gated_linear", x.data_ptr(), wg, wu, sg, su, pg, pu, output.data_ptr(), M, K, N, group_size, dtype)
    return output


def gated_linear(x, Wg, Wu, bg=None, bu=None, save=False):
    """SiLU(x Wg^T + bg) * (x Wu^T + bu) for fp16 / bf16 weights (N, K) -> (M, N). save=True: also the two products in
    fp32, (h, g, u), which gated_linear_backward takes. No autograd; see forge_b200.nn.gated_linear."""
    dtype, M, K = _act_shape(x)
    N = Wg.shape[0]
    _chk(x, Wg=(Wg, x.dtype), Wu=(Wu, x.dtype), bg=(bg, x.dtype), bu=(bu, x.dtype))
    _shape(Wg=(Wg, (N, K)), Wu=(Wu, (N, K)), bg=(bg, (N,)), bu=(bu, (N,)))
    if N % 8 != 0 or N > _MAX_SIZE:
        raise ValueError(f"Wg, Wu: the number of outputs must be a multiple of 8, at most {_MAX_SIZE}, got {N}")
    x, Wg, Wu = _aligned(x), _aligned(Wg), _aligned(Wu)
    h = x.new_empty((M, N))
    g = u = None
    if save:
        g = x.new_empty((M, N), dtype=_f32)
        u = torch.empty_like(g)
    _run(x, "forge_gated_linear", x.data_ptr(), Wg.data_ptr(), Wu.data_ptr(), _ptr(bg), _ptr(bu), h.data_ptr(), _ptr(g),
         _ptr(u), M, K, N, dtype)
    return (h, g, u) if save else h


def gated_linear_backward(dh, x, Wg, Wu, g, u, need_x=True, need_w=True, need_b=True):
    """Gradients of gated_linear for dh (M, N): (dx, dWg, dWu, dbg, dbu) in x's type, None where not asked for."""
    dtype, M, K = _act_shape(x)
    N = Wg.shape[0]
    _chk(x, dh=(dh, x.dtype), x=(x, x.dtype), Wg=(Wg, x.dtype), Wu=(Wu, x.dtype), g=(g, _f32), u=(u, _f32))
    _shape(dh=(dh, (M, N)), Wg=(Wg, (N, K)), Wu=(Wu, (N, K)), g=(g, (M, N)), u=(u, (M, N)))
    if N % 8 != 0 or N > _MAX_SIZE:
        raise ValueError(f"Wg, Wu: the number of outputs must be a multiple of 8, at most {_MAX_SIZE}, got {N}")
    # without tokens or outputs the library writes nothing: the gradients of the weights, or of x, are empty sums
    like = torch.zeros_like if M == 0 or N == 0 else torch.empty_like
    dx = like(x) if need_x else None
    dWg, dWu = (like(Wg), like(Wu)) if need_w else (None, None)
    dbg = dbu = None
    if need_b:
        dbg = x.new_zeros((N,)) if M == 0 else x.new_empty((N,))
        dbu = like(dbg)
    dh, x, Wg, Wu = _aligned(dh), _aligned(x), _aligned(Wg), _aligned(Wu)
    g, u = _aligned(g), _aligned(u)
    size = _lib.load().forge_gated_linear_backward_workspace_bytes(M, N)
    workspace = torch.empty((size,), dtype=_u8, device=x.device)
    _run(x, "forge_gated_linear_backward", _ptr(dh), _ptr(x), _ptr(Wg), _ptr(Wu), _ptr(g), _ptr(u), _ptr(dx), _ptr(dWg),
         _ptr(dWu), _ptr(dbg), _ptr(dbu), M, K, N, dtype, _ptr(workspace))
    return dx, dWg, dWu, dbg, dbu


def device_status(reset=True):
    """FORGE_B200_OK (0) unless a kernel on the current device gave up on a bounded wait since the last
    reset (then FORGE_B200_DEVICE_TIMEOUT, 5); `device_status_raw` returns the recorded code."""
    return _lib.load().forge_b200_device_status(1 if reset else 0)


def device_status_raw(reset=True):
    return _lib.load().forge_b200_device_status_raw(1 if reset else 0)
