"""Plain 64-bit forms of the 4-bit and gated linear operators, with bounds on what the kernels may be off by.

Bounds: a tensor-core instruction adds at most 17 numbers aligned to the largest with at least 24 bits, so it is off by at
most 17 * 2^-23 of the sum of their sizes; over K / 16 of them (and the few fp32 additions of the partial sums behind) a dot
product is off by at most (K + 64) * 2^-23 * sum |x w|. A rounding to a type is off by half a step, eps / 2 of the value
(half the smallest subnormal where the value is below the normal range).
"""
import torch


def half_step(v, dtype):
    f = torch.finfo(dtype)
    return torch.clamp(v.abs() * (f.eps / 2), min=f.smallest_normal * f.eps / 2)


def unpack_int4(w_int4, w_scale, K, group):
    """The layout of include/forge_b200.h, read one weight at a time: (N, K) float64."""
    N = w_int4.shape[0]
    k = torch.arange(K, device=w_int4.device)
    block, run, i = k // 128, k % 128 // 8, k % 8
    word = block * 16 + run % 4 * 4 + run // 4
    nibble = i % 2 * 4 + i // 2
    byte = w_int4[:, word * 4 + nibble // 2].to(torch.int64)
    q = (byte >> (nibble % 2 * 4)) & 15
    return (q - 8).double() * w_scale.double().t()[:, k // group].reshape(N, K)


def int4_sizes(w_scale, K, group, dtype):
    """What `linear` takes as the sizes of 4-bit weights: few tokens are multiplied with q + 8 (bf16: q + 24), from which
    as much is taken off again, so a product's parts are as large as (|q| + 16) s (bf16: 48), |q| <= 8."""
    s = w_scale.double().abs().t()[:, torch.arange(K, device=w_scale.device) // group]
    return s.reshape(w_scale.shape[1], K) * (24 if dtype == torch.float16 else 56)


def linear(x, w, b, sizes=None, chain=None):
    """y and a bound on the fp32 evaluation's error, before any rounding of y. `sizes`: of the products' parts, where they
    are larger than |w|; `chain`: inputs that are summed at a time, where that is not all of them (then the sums of the
    K / chain pieces are added in fp32, each addition off by half a step of at most the sum of sizes)."""
    x, w = x.double(), w.double()
    y = x @ w.t()
    K = x.shape[1]
    err = ((chain or K) + 64) * 2.0 ** -23 * (x.abs() @ (w if sizes is None else sizes).abs().t())
    if chain:
        err = err + (K / chain + 64) * 2.0 ** -24 * (x.abs() @ w.abs().t())
    if b is not None:
        y = y + b.double()
        err = err + 2.0 ** -24 * y.abs()
    return y, err


def _fn_rel(g):
    """Relative error of 1 / (1 + exp(-g)) in fp32: the fast exponential is off by 2 + 1.173 |g| steps, the sum by half a
    step, the fast division by 2, the products around it by half a step each (4 of them)."""
    return (2 + 1.173 * g.abs() + 5) * 2.0 ** -23


def gate_of(gate, up):
    """SiLU(g) u and its bound from (g, bound) and (u, bound)."""
    (g, eg), (u, eu) = gate, up
    silu = g * torch.sigmoid(g)
    # |SiLU'| <= 1.1
    return silu * u, 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + _fn_rel(g) * (silu * u).abs() + 2.0 ** -120


def gate(x, wg, wu, bg, bu):
    g, u = linear(x, wg, bg), linear(x, wu, bu)
    return (*gate_of(g, u), (*g, *u))


def gate_backward(dh, x, wg, wu, saved, dtype):
    """{name: (value, bound)} of the gradients; dg and du are rounded to `dtype` before the products."""
    g, eg, u, eu = saved
    dh, x, wg, wu = (t.double() for t in (dh, x, wg, wu))
    s = torch.sigmoid(g)
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    # SiLU' is at most 1.1 and its slope at most 0.5; 1 + g (1 - s) loses to cancellation at most what |1| + |g (1 - s)| has
    eg_ = (dh.abs() * (1.1 * eu + 0.5 * eg * (u.abs() + eu))
           + _fn_rel(g) * 2 * (dh * u * s).abs() * (1 + (g * (1 - s)).abs()) + 2.0 ** -120)
    eu_ = dh.abs() * 1.1 * eg + _fn_rel(g) * du.abs() + 2.0 ** -120
    rg, ru = eg_ + half_step(dg.abs() + eg_, dtype), eu_ + half_step(du.abs() + eu_, dtype)
    M, N = dh.shape
    acc = 2.0 ** -23
    out = {
        "dx": (dg @ wg + du @ wu, rg @ wg.abs() + ru @ wu.abs()
               + (2 * N + 64) * acc * ((dg.abs() + rg) @ wg.abs() + (du.abs() + ru) @ wu.abs())),
        "dwg": (dg.t() @ x, rg.t() @ x.abs() + (M + 64) * acc * ((dg.abs() + rg).t() @ x.abs())),
        "dwu": (du.t() @ x, ru.t() @ x.abs() + (M + 64) * acc * ((du.abs() + ru).t() @ x.abs())),
        "dbg": (dg.sum(0), eg_.sum(0) + M * acc * (dg.abs() + eg_).sum(0)),
        "dbu": (du.sum(0), eu_.sum(0) + M * acc * (du.abs() + eu_).sum(0)),
    }
    return {k: (v, e + half_step(v.abs() + e, dtype)) for k, (v, e) in out.items()}


def close(got, want, bound, what=""):
    off = (got.double() - want).abs() - bound
    assert got.shape == want.shape and bool((off <= 0).all()), \
        f"{what}: {int((~(off <= 0)).sum())} of {off.numel()} outside the bound, worst by {off.max().item():.3g}"


def close_rounded(got, want, err, what=""):
    """A result evaluated within `err` and rounded once to its type."""
    close(got, want, err + half_step(want.abs() + err, got.dtype), what)
