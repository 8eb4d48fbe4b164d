"""The 8-bit activation path as it is measured: RMS norm and row quantisation into int8, the int8 matrix
product with scales for each token and channel, and a gated feed-forward half of a layer made of them.

`run` computes the operators in their plain form (elementary torch operations) where `own` is false, and
makes a user's calls of the library where it is true.  Sizes are those of the library's benchmark layers
(K = 4096 / 8192 / 11008 / 28672 and their feature counts) and generic odd ones.
"""
import math
from types import SimpleNamespace as State

import torch

own = False

EPS = 1e-5
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one new token enters a layer: the norm in front of its projections (latency)
        dict(name="norm_token", op="norm", M=1, K=4096, type="f16", residual=True),
        # a long prompt through the norm of a layer of width 8192
        dict(name="norm_prompt", op="norm", M=4096, K=8192, type="bf16", residual=True),
        # a first norm without residual, rows of odd length at odd addresses
        dict(name="norm_odd", op="norm", M=1000, K=5001, type="f16", residual=False),
        # the input of a down projection, a batch of 16 tokens
        dict(name="quant_batch", op="quant", M=16, K=11008, type="f16"),
        # ... and a prompt, width 28672
        dict(name="quant_prompt", op="quant", M=2048, K=28672, type="bf16"),
        # one token through a 4096 x 4096 projection with bias (latency)
        dict(name="gemm_token", op="gemm", M=1, N=4096, K=4096, type="f16", scales="f16", bias=True, act="none"),
        # 16 tokens through a fused gate/up layer
        dict(name="gemm_batch_gated", op="gemm", M=16, N=22016, K=4096, type="bf16", scales="f32", bias=False, act="gated"),
        # a short prompt through a fused query/key/value projection
        dict(name="gemm_chunk", op="gemm", M=131, N=12288, K=4096, type="f16", scales="f16", bias=True, act="none"),
        # odd token and feature counts, a reduction that ends inside every tile, padded rows
        dict(name="gemm_odd", op="gemm", M=777, N=4099, K=11003, type="f16", scales="f32", bias=True, act="silu"),
        # a prompt through a down projection
        dict(name="gemm_prompt_down", op="gemm", M=2048, N=8192, K=28672, type="f16", scales="f16", bias=False, act="none"),
        # the largest: a long prompt through a fused gate/up layer
        dict(name="gemm_prompt_gated", op="gemm", M=4096, N=57344, K=8192, type="bf16", scales="f32", bias=False, act="gated"),
        # norm, gate/up, quantisation and down projection of a layer in a row, as a server runs them
        dict(name="layer_half", op="layer", M=256, K=4096, H=11008, type="bf16"),
    ]


def draw(rng):
    size = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["norm", "quant", "gemm", "gemm", "layer"])
    dtype = rng.choice(["f16", "bf16"])
    if kind in ("norm", "quant"):
        K = size(64, 32768)
        if rng.random() < 0.6:
            K = -(-K // 16) * 16
        M = max(1, min(size(1, 16384), (1 << 26) // K))
        return dict(op=kind, M=M, K=K, type=dtype, **({"residual": rng.random() < 0.7} if kind == "norm" else {}))
    if kind == "layer":
        K, H = size(256, 8192), size(512, 28672)
        M = max(1, min(size(1, 4096), int(2e12 / (6 * K * H))))
        return dict(op="layer", M=M, K=-(-K // 16) * 16, H=-(-H // 16) * 16, type=dtype)
    act = rng.choice(["none", "relu", "silu", "gated"])
    N, K = size(128, 57344), size(256, 28672)
    if rng.random() < 0.6:
        N, K = -(-N // 64) * 64, -(-K // 64) * 64
    if act == "gated":
        N += N % 2
    M = max(1, min(size(1, 8192), int(2e12 / (2.0 * N * K))))
    return dict(op="gemm", M=M, N=N, K=K, type=dtype, scales=rng.choice(["f16", "bf16", "f32"]), bias=rng.random() < 0.5, act=act)


def _noise(*shape, gen):
    return torch.randn(*shape, generator=gen, device="cuda")


def _int8(rows, cols, gen):
    """int8 [rows, cols] of normally distributed values, each row 16-byte aligned as the product wants it."""
    ld = -(-cols // 16) * 16
    q = torch.empty(rows, ld, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // ld)
    for r in range(0, rows, step):
        q[r:r + step] = (_noise(min(step, rows - r), ld, gen=gen) * 32).round_().clamp_(-127, 127).to(torch.int8)
    return q[:, :cols]


def _layer_weights(N, K, s, gen, scales, dtype, bias):
    """Weights of an int8 layer whose outputs are of the order of its inputs."""
    w = _int8(N, K, gen)
    ws = ((torch.rand(N, generator=gen, device="cuda") + 0.5) * (s / (32 * math.sqrt(K)))).to(scales)
    b = (_noise(N, gen=gen) * 0.1).to(dtype) if bias else None
    return w, ws, b


def _activations(M, K, gen, dtype):
    """Hidden states: normal, with rows and a few channels that stand out."""
    x = _noise(M, K, gen=gen) * (0.5 + 2 * torch.rand(M, 1, generator=gen, device="cuda"))
    x[:, :: max(1, K // 8)] *= 6
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, M, K, op = TYPES[case["type"]], case["M"], case["K"], case["op"]
    s = State(op=op, case=case)
    new = lambda *shape, dtype=t: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    row8 = lambda rows, cols: new(rows, -(-cols // 16) * 16, dtype=torch.int8)[:, :cols]  # noqa: E731
    if op in ("norm", "quant", "layer"):
        s.x = _activations(M, K, gen, t)
        s.q, s.scale = row8(M, K), new(M, dtype=torch.float32)
    if op in ("norm", "layer"):
        s.weight = (1 + 0.2 * _noise(K, gen=gen)).to(t)
        s.residual = _activations(M, K, gen, t) if op == "layer" or case["residual"] else None
        s.h = new(M, K) if s.residual is not None else None
    if op in ("norm", "quant"):
        s.back = new(M, K)
    if op == "gemm":
        N, s.act = case["N"], case["act"]
        s.x = _int8(M, K, gen)
        s.x_scale = (torch.rand(M, generator=gen, device="cuda") + 0.5) / 32
        s.w, s.w_scale, s.bias = _layer_weights(N, K, 1.0, gen, TYPES[case["scales"]], t, case["bias"])
        s.out = new(M, N // 2 if s.act == "gated" else N)
    if op == "layer":
        H = case["H"]
        s.w1, s.s1, _ = _layer_weights(2 * H, K, 1.0, gen, torch.float32, t, False)
        s.w2, s.s2, _ = _layer_weights(K, H, 1.0, gen, torch.float32, t, False)
        s.mid, s.q2, s.scale2, s.out = new(M, H), row8(M, H), new(M, dtype=torch.float32), new(M, K)
    if own:
        _plan(s)
    return s


def _plan(s):
    """The operators a program keeps for its buffers: arguments checked, launches planned."""
    from mixed_gemv_b200 import _lib, api

    pdl = _lib.FLAG_PDL
    acts = {"none": 0, "relu": _lib.FLAG_ACT_RELU, "silu": _lib.FLAG_ACT_SILU, "gated": _lib.FLAG_GATED_SILU}
    s.ops = []

    def keep(op, args):
        op.initialize(args)
        s.ops.append(op)

    if s.op in ("norm", "layer"):
        keep(api.RmsNormQuantizer(), api.RmsNormQuantizeArguments(
            x=s.x, weight=s.weight, q=s.q, scale=s.scale, residual=s.residual, residual_out=s.h, eps=EPS, flags=pdl))
    if s.op == "quant":
        keep(api.RowQuantizer(), api.RowQuantizeArguments(x=s.x, q=s.q, scale=s.scale, flags=pdl))
    if s.op in ("norm", "quant"):
        keep(api.RowDequantizer(), api.RowDequantizeArguments(q=s.q, scale=s.scale, out=s.back, flags=pdl))
    if s.op == "gemm":
        keep(api.GemmI8Adaptor(), api.GemmI8Arguments(
            x=s.x, x_scale=s.x_scale, weights=s.w, weight_scale=s.w_scale, bias=s.bias, out=s.out, flags=pdl | acts[s.act]))
    if s.op == "layer":
        keep(api.GemmI8Adaptor(), api.GemmI8Arguments(
            x=s.q, x_scale=s.scale, weights=s.w1, weight_scale=s.s1, out=s.mid, flags=pdl | _lib.FLAG_GATED_SILU))
        keep(api.RowQuantizer(), api.RowQuantizeArguments(x=s.mid, q=s.q2, scale=s.scale2, flags=pdl))
        keep(api.GemmI8Adaptor(), api.GemmI8Arguments(
            x=s.q2, x_scale=s.scale2, weights=s.w2, weight_scale=s.s2, out=s.out, flags=pdl))


def _plain_quantise(y):
    """(values in -127..127, scale of each row) of float rows."""
    amax = y.abs().amax(dim=1, keepdim=True)
    scale = amax / 127
    q = torch.where(amax > 0, (y * (127 / amax)).round(), torch.zeros_like(y))
    return q, scale


def _plain_norm(x, residual, weight):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(dim=1, keepdim=True) + EPS) * weight.float()
    return h, y


def _plain_product(q, scale, w, w_scale, bias, act, dtype):
    z = (q.float() @ w.float().t()) * scale.reshape(-1, 1) * w_scale.float()
    if bias is not None:
        z = z + bias.float()
    if act == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif act == "silu":
        z = z / (1 + torch.exp(-z))
    elif act == "gated":
        g, u = z[:, 0::2], z[:, 1::2]
        z = g / (1 + torch.exp(-g)) * u
    return z.to(dtype)


def run(s):
    if own:
        for op in s.ops:
            op.run()
        if s.op in ("norm", "quant"):
            out = {"values": s.back, "scale": s.scale}
        else:
            out = {"out": s.out}
        if s.op in ("norm", "layer") and s.h is not None:
            out["residual"] = s.h
        return out
    t = TYPES[s.case["type"]]
    if s.op == "gemm":
        return {"out": _plain_product(s.x, s.x_scale, s.w, s.w_scale, s.bias, s.act, t)}
    h, y = (None, s.x.float()) if s.op == "quant" else _plain_norm(s.x, s.residual, s.weight)
    q, scale = _plain_quantise(y)
    if s.op == "layer":
        mid = _plain_product(q, scale, s.w1, s.s1, None, "gated", t)
        q2, scale2 = _plain_quantise(mid.float())
        out = {"out": _plain_product(q2, scale2, s.w2, s.s2, None, "none", t)}
    else:
        out = {"values": (q * scale).to(t), "scale": scale[:, 0]}
    if s.op in ("norm", "layer") and s.residual is not None:
        out["residual"] = h
    return out


def exact(case, seed):
    """The definition in 64 bits: out[m, n] = act(sum_k q[m, k] w[n, k] s[m] t[n] + b[n]); a row's scale is the largest
    magnitude / 127 and its values the nearest multiples of it.  Sums that the operators round to 16 bits on the way (the
    residual, the activations between the two products) are rounded here too: they are outputs of their own."""
    s = prepare(case, seed)
    t = TYPES[case["type"]]

    def quantised(rows):
        top = torch.linalg.vector_norm(rows, ord=float("inf"), dim=1)
        step = top / 127.0
        level = torch.round(rows / torch.where(step > 0, step, torch.ones_like(step))[:, None])
        return level, step

    def product(level, step, w, w_step, bias, act):
        z = torch.einsum("mk,nk->mn", level, w.double())
        z.mul_(step[:, None]).mul_(w_step.double()[None, :])
        if bias is not None:
            z.add_(bias.double())
        if act == "relu":
            return torch.clamp_min(z, 0.0)
        if act == "silu":
            return z * torch.sigmoid(z)
        if act == "gated":
            z = z.reshape(z.shape[0], -1, 2)
            return z[..., 0] * torch.sigmoid(z[..., 0]) * z[..., 1]
        return z

    if s.op == "gemm":
        return {"out": product(s.x.double(), s.x_scale.double(), s.w, s.w_scale, s.bias, s.act)}
    rows, out = s.x.double(), {}
    if s.op in ("norm", "layer"):
        if s.residual is not None:
            out["residual"] = rows + s.residual.double()
            rows = out["residual"].to(t).double()
        mean = torch.einsum("mk,mk->m", rows, rows) / rows.shape[1]
        rows = rows / torch.sqrt(mean + EPS)[:, None] * s.weight.double()
    level, step = quantised(rows)
    if s.op == "layer":
        mid = product(level, step, s.w1, s.s1, None, "gated").to(t).double()
        level, step = quantised(mid)
        out["out"] = product(level, step, s.w2, s.s2, None, "none")
    else:
        out["values"], out["scale"] = level * step[:, None], step
    return out


def work(case):
    M, K, op, e = case["M"], case["K"], case["op"], SIZE[case["type"]]
    if op == "quant":
        return {"bytes": M * K * 2 * e + 4 * M, "flops": 4 * M * K}
    if op == "norm":
        return {"bytes": M * K * e * (4 if case["residual"] else 2) + K * e + 4 * M, "flops": 8 * M * K}
    if op == "gemm":
        N, gated = case["N"], case["act"] == "gated"
        columns = N * SIZE[case["scales"]] + (N * e if case["bias"] else 0)
        return {"bytes": M * K + N * K + 4 * M + columns + M * (N // 2 if gated else N) * e, "flops": 2 * M * N * K}
    H = case["H"]
    return {"bytes": 4 * M * K * e + K * e + 3 * H * K + 4 * (2 * H + K), "flops": 6 * M * K * H}
