"""Cases of the 4-bit weight and gated feed-forward operators, for timing and for comparing outputs.

Operators (x (M, K); weights (N, K), one row per output channel):

  int4_linear        y = x W^T + b, W in 4-bit integers with one fp16 scale per group of 32 / 64 / 128 inputs
  int4_gated_linear  h = SiLU(x Wg^T + bg) * (x Wu^T + bu), both weights in that form
  gated_linear       the same gate on 16-bit weights, inference
  gated_linear_train forward and backward of gated_linear: h, dx, dWg, dWu, dbg, dbu for a given dh

`run` computes them in elementary torch operations in 32 bits, or, with `own` set, by the library's calls.
"""
import math

import torch

own = False

_DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16}
_GATED = ("int4_gated_linear", "gated_linear", "gated_linear_train")


def listed():
    return [
        # one token through the benchmark's 11008 x 4096 weight: decoding, where the weight's bytes and the latency count
        {"name": "int4_m1_11008x4096", "op": "int4_linear", "M": 1, "K": 4096, "N": 11008, "group": 128, "dtype": "fp16", "bias": False},
        # eight sequences decoding together, the down projection of the benchmark's MLP
        {"name": "int4_m8_4096x14336", "op": "int4_linear", "M": 8, "K": 14336, "N": 4096, "group": 64, "dtype": "bf16", "bias": True},
        # a short ragged batch on a weight with an odd number of rows and a last group cut short
        {"name": "int4_m37_4099x4104", "op": "int4_linear", "M": 37, "K": 4104, "N": 4099, "group": 32, "dtype": "bf16", "bias": True},
        # a prompt of 2048 tokens on the same benchmark weight
        {"name": "int4_m2048_11008x4096", "op": "int4_linear", "M": 2048, "K": 4096, "N": 11008, "group": 128, "dtype": "fp16", "bias": False},
        # one token through the gate and up projections of the benchmark's MLP
        {"name": "int4_gated_m1", "op": "int4_gated_linear", "M": 1, "K": 4096, "N": 14336, "group": 128, "dtype": "fp16", "bias": False},
        # a ragged batch of prompts through the same projections
        {"name": "int4_gated_m333", "op": "int4_gated_linear", "M": 333, "K": 4096, "N": 14336, "group": 64, "dtype": "bf16", "bias": True},
        # four sequences decoding with unquantized weights
        {"name": "gated_m4", "op": "gated_linear", "M": 4, "K": 4096, "N": 14336, "dtype": "bf16", "bias": False},
        # the benchmark's 8192 tokens through the unquantized projections
        {"name": "gated_m8192", "op": "gated_linear", "M": 8192, "K": 4096, "N": 14336, "dtype": "fp16", "bias": True},
        # a small layer's training step, ragged in every size
        {"name": "gated_train_m1001", "op": "gated_linear_train", "M": 1001, "K": 1032, "N": 2744, "dtype": "fp16", "bias": True},
        # the benchmark's MLP in training
        {"name": "gated_train_m8192", "op": "gated_linear_train", "M": 8192, "K": 4096, "N": 14336, "dtype": "bf16", "bias": False},
    ]


def _log(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["int4_linear", "int4_linear", "int4_gated_linear", "gated_linear", "gated_linear_train"])
    case = {"op": op, "M": _log(rng, 1, 4096), "K": _log(rng, 64, 14336, 8), "dtype": rng.choice(["fp16", "bf16"]),
            "bias": rng.random() < 0.5}
    if op.startswith("int4"):
        case["N"] = _log(rng, 64, 14336)
        case["group"] = rng.choice([32, 64, 128])
    else:
        case["N"] = _log(rng, 64, 14336, 8)
    while case["M"] * case["K"] * case["N"] > 8192 * 4096 * 14336:
        case["M"] //= 2
    return case


def _inputs(case, seed):
    """The numbers of a case: activations with 1 % of the channels 20 times larger, weights of a trained
    layer's size, rounded to 4 bits against per-group scales where the operator wants that."""
    M, K, N, dt = case["M"], case["K"], case["N"], _DTYPE[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    d = {}
    train = case["op"] == "gated_linear_train"
    x = normal(M, K)
    if not train:
        x *= 1 + 19 * (torch.rand(K, generator=g, device="cuda") < 0.01)
    d["x"] = x.to(dt)
    # the gate's argument has a standard deviation near one, as behind a norm
    for k in ("g", "u") if case["op"] in _GATED else ("w",):
        w = normal(N, K) * min(0.02, 1.3 / math.sqrt(K))
        if case["op"].startswith("int4"):
            G = case["group"]
            groups = -(-K // G)
            w = torch.nn.functional.pad(w, (0, groups * G - K)).view(N, groups, G)
            s = (w.abs().amax(2) / 7).half()
            q = torch.round(w / s.float()[:, :, None]).clamp_(-7, 7).to(torch.int8).view(N, groups * G)[:, :K]
            # the four-bit range is -8 .. 7: files of other programs use its lowest value too
            q[torch.rand(N, K, generator=g, device="cuda") < 0.01] = -8
            d["q" + k], d["s" + k] = q.contiguous(), s.t().contiguous()
        else:
            d["w" + k] = w.to(dt)
        d["b" + k] = (normal(N) * 0.01).to(dt) if case["bias"] else None
    if train:
        d["dh"] = (normal(M, N) * 0.01).to(dt)
    return d


def _pack(q):
    """(N, K) integers -8 .. 7 -> (N, ceil(K / 128) * 64) bytes. 8 neighbouring weights make one 32-bit word, weight 2i in
    its nibble i, weight 2i + 1 in its nibble i + 4, each as the integer + 8; of the 16 words of a block of 128 weights
    word 4t + j is the block's run 4j + t. Weights past K are zero."""
    N, K = q.shape
    pad = -K % 128
    n = torch.nn.functional.pad(q, (0, pad)).to(torch.int32).add_(8)
    n = n.view(N, (K + pad) // 128, 4, 4, 4, 2).transpose(2, 3)  # row, block, t, j, i, odd
    i = torch.arange(4, device=q.device, dtype=torch.int32)
    shift = torch.stack((4 * i, 4 * i + 16), 1)
    word = (n.to(torch.int64) << shift).sum((4, 5))
    return torch.stack([(word >> (8 * b)) & 255 for b in range(4)], -1).to(torch.uint8).view(N, -1)


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"op": case["op"], "group": case.get("group")}
    for k, v in d.items():
        if k[0] == "q":
            state["w" + k[1:]] = _pack(v)
        else:
            state[k] = v
    if case["op"] == "gated_linear_train":
        for k in ("x", "wg", "wu", "bg", "bu"):
            if state[k] is not None:
                state[k].requires_grad_()
    return state


def _unpack(w, s, K, group):
    """The packed weight as 32-bit numbers (N, K)."""
    N = w.shape[0]
    nib = torch.stack((w & 15, w >> 4), -1).view(N, -1, 4, 4, 2, 4)  # row, block, t, j, odd, i
    q = nib.permute(0, 1, 3, 2, 5, 4).reshape(N, -1)[:, :K].float() - 8
    return q * s.float().repeat_interleave(group, 0)[:K].t()


def _linear(x, w, b):
    y = x @ w.t()
    return y if b is None else y + b.float()


@torch.no_grad()
def _plain(s):
    x = s["x"].float()
    dt = s["x"].dtype
    K = x.shape[1]
    if s["op"] == "int4_linear":
        return _linear(x, _unpack(s["ww"], s["sw"], K, s["group"]), s["bw"]).to(dt)
    if s["op"] == "int4_gated_linear":
        wg, wu = _unpack(s["wg"], s["sg"], K, s["group"]), _unpack(s["wu"], s["su"], K, s["group"])
    else:
        wg, wu = s["wg"].float(), s["wu"].float()
    gate, up = _linear(x, wg, s["bg"]), _linear(x, wu, s["bu"])
    sig = 1 / (1 + torch.exp(-gate))
    h = (gate * sig * up).to(dt)
    if s["op"] != "gated_linear_train":
        return h
    dh = s["dh"].float()
    dgate = dh * up * sig * (1 + gate * (1 - sig))
    dup = dh * gate * sig
    out = {"h": h, "dx": (dgate @ wg + dup @ wu).to(dt), "dwg": (dgate.t() @ x).to(dt), "dwu": (dup.t() @ x).to(dt)}
    if s["bg"] is not None:
        out["dbg"], out["dbu"] = dgate.sum(0).to(dt), dup.sum(0).to(dt)
    return out


def run(state):
    s = state
    if not own:
        return _plain(s)
    from forge_b200 import _forge_C as C
    if s["op"] == "int4_linear":
        return C.int4_linear(s["x"], s["ww"], s["sw"], s["bw"], s["group"])
    if s["op"] == "int4_gated_linear":
        return C.int4_gated_linear(s["x"], s["wg"], s["wu"], s["sg"], s["su"], s["bg"], s["bu"], s["group"])
    if s["op"] == "gated_linear":
        return C.gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"])
    from forge_b200.nn import gated_linear
    h = gated_linear(s["x"], s["wg"], s["wu"], s["bg"], s["bu"])
    names = ["x", "wg", "wu"] + (["bg", "bu"] if s["bg"] is not None else [])
    grads = torch.autograd.grad(h, [s[k] for k in names], s["dh"])
    return {"h": h.detach(), **{"d" + k: v for k, v in zip(names, grads)}}


def work(case):
    M, K, N = case["M"], case["K"], case["N"]
    mats = 2 if case["op"] in _GATED else 1
    bias = mats * N * 2 if case["bias"] else 0
    acts = 2 * (M * K + M * N) + bias
    if case["op"].startswith("int4"):
        weights = mats * (N * K // 2 + N * -(-K // case["group"]) * 2)
    else:
        weights = mats * N * K * 2
    if case["op"] == "gated_linear_train":
        # read x, Wg, Wu, dh and the biases; write h, dx and the gradients of the weights and biases
        return {"bytes": 2 * weights + 2 * acts, "flops": 12 * M * K * N}
    return {"bytes": weights + acts, "flops": 2 * mats * M * K * N}


def exact(case, seed):
    d = _inputs(case, seed)
    f = lambda t: None if t is None else t.to(torch.float64)  # noqa: E731
    lin = torch.nn.functional.linear
    x = f(d["x"])

    def weight(k):
        if not case["op"].startswith("int4"):
            return f(d["w" + k])
        which = torch.arange(case["K"], device="cuda") // case["group"]
        return f(d["q" + k]) * f(d["s" + k])[which].t()

    if case["op"] == "int4_linear":
        return lin(x, weight("w"), f(d["bw"]))
    wg, wu = weight("g"), weight("u")
    a, u = lin(x, wg, f(d["bg"])), lin(x, wu, f(d["bu"]))
    sig = (torch.tanh(a / 2) + 1) / 2
    silu = a * sig
    if case["op"] != "gated_linear_train":
        return silu * u
    dh = f(d["dh"])
    du = dh * silu
    da = dh * u * (sig + silu * (1 - sig))
    out = {"h": silu * u, "dx": torch.addmm(du @ wu, da, wg), "dwg": torch.mm(da.mT, x), "dwu": torch.mm(du.mT, x)}
    if case["bias"]:
        out["dbg"], out["dbu"] = torch.einsum("mn->n", da), torch.einsum("mn->n", du)
    return out
