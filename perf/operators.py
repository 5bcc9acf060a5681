"""The MXFP4 and grouped-product operators as cases that can be timed and compared.

Four kinds of work, each what a program that serves or trains a mixture of experts does with
rows sorted by expert:
  encode   weights or activations to MXFP4 (blocks of 32 along the last axis, one power-of-two
           scale a block, E2M1 elements) and back to bf16 values
  mx       rows times their expert's MXFP4 matrix: bf16 rows, or rows quantised to MXFP4 first
  dense    rows times their expert's bf16 or fp16 matrix
  train    the same with its backward pass: output, gradient of the rows and of every matrix
A case's routing (how many rows each expert has) comes from the case itself, its values from
the seed.  ``own`` False computes them in elementary torch operations in 32 bits, ``own`` True
by the library's entry points.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
STD = 0.02                                     # weights N(0, STD), activations N(0, 1)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LARGEST = 2 * 8192 * 28672 * 4096              # operations of the largest listed product

# an expert's gate/up matrix: rows M = 2 x intermediate, columns K = hidden; experts, top-k
QWEN = dict(M=2816, K=2048, E=60, k=4)         # Qwen1.5-MoE-A2.7B
DEEPSEEK = dict(M=2816, K=2048, E=64, k=6)     # DeepSeek-V2-Lite
MIXTRAL = dict(M=28672, K=4096, E=8, k=2)      # Mixtral-8x7B


def _product(kind, T, shape, dtype="bf16", out="bf16", skew=0.0, pad=0, pick=1, x4=False, **more):
    """T tokens, each to k of E experts; ``skew``: Zipf exponent of the experts' popularity;
    ``pad``: rows behind the last group; ``x4``: rows quantised to MXFP4 before the product."""
    return dict(kind=kind, T=T, dtype=dtype, out=out, skew=skew, pad=pad, pick=pick, x4=x4, **shape, **more)


def listed():
    return [
        # one token's hidden state quantised before an expert's product: latency
        dict(kind="encode", rows=1, K=2048, dtype="bf16", name="encode_one_token"),
        # a large expert's matrix quantised when a checkpoint is converted
        dict(kind="encode", rows=4096, K=14336, dtype="f32", name="encode_expert_matrix"),
        # one token of one sequence: its four experts
        _product("mx", 1, QWEN, name="mx_decode_t1"),
        # one token times one matrix (a down projection), the single-expert form
        _product("mx", 1, dict(M=4096, K=14336, E=1, k=1), out="f32", name="mx_gemv_4096x14336"),
        # a decode batch, two or three rows an expert, fp32 results
        _product("mx", 32, QWEN, out="f32", skew=0.6, pick=2, name="mx_decode_t32"),
        # a short prompt of odd length, activations kept in bf16
        _product("mx", 333, QWEN, skew=0.4, pick=3, name="mx_prefill_t333"),
        # a long prompt, activations quantised too
        _product("mx", 2048, DEEPSEEK, x4=True, pick=4, name="mx_x4_prefill_t2048"),
        # few large experts, a long prompt, activations quantised
        _product("mx", 4096, MIXTRAL, x4=True, pick=5, name="mx_x4_prefill_t4096"),
        # experts left in 16 bits, a decode batch, fp16
        _product("dense", 12, MIXTRAL, dtype="f16", out="f16", pick=6, name="dense_decode_t12"),
        # the largest product: few large experts in bf16, a long prompt
        _product("dense", 4096, MIXTRAL, pick=7, name="dense_prefill_t4096"),
        # experts trained before they are quantised: a step's products, forward and backward
        _product("train", 2048, DEEPSEEK, skew=0.4, pick=8, name="train_t2048"),
        # a small odd step: uneven sizes, an expert nobody took, padded rows, fp16
        _product("train", 259, dict(M=712, K=1000, E=9, k=3), dtype="f16", out="f16", skew=1.5, pad=23, pick=9,
                 name="train_small_odd"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["encode", "mx", "mx", "mx", "dense", "dense", "train", "train"])
    if kind == "encode":
        K = 32 * _log(rng, 1, 448)
        return dict(kind=kind, rows=_log(rng, 1, max(1, 4096 * 14336 // K)), K=K,
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    E = _log(rng, 1, 64)
    k = rng.randint(1, min(8, E))
    if kind == "mx":
        M, K = _log(rng, 48, 20000), 32 * _log(rng, 2, 448)
        dtype, out, x4 = "bf16", rng.choice(["bf16", "f32"]), rng.random() < 0.5
    else:
        M, K = 8 * _log(rng, 8, 2000), 8 * _log(rng, 8, 1000)
        dtype, x4 = rng.choice(["bf16", "f16"]), False
        out = rng.choice([dtype, "f32"]) if kind == "dense" else dtype
    E = min(E, max(1, 8 * 28672 * 4096 // (M * K)))
    k = min(k, E)
    most = LARGEST // (2 * M * K * k * (3 if kind == "train" else 1))
    T = _log(rng, 1, max(1, min(4096, most)))
    return _product(kind, T, dict(M=M, K=K, E=E, k=k), dtype, out, skew=rng.choice([0.0, 0.5, 1.2]),
                    pad=rng.choice([0, 0, rng.randint(1, 70)]), pick=rng.randrange(1 << 20), x4=x4)


def _counts(case):
    """Rows of each expert: every token takes k different ones, by popularity."""
    rng = np.random.default_rng(case["pick"])
    pop = -case["skew"] * np.log(rng.permutation(case["E"]) + 1.0)
    keys = pop + rng.gumbel(size=(case["T"], case["E"]))
    ids = np.argpartition(-keys, case["k"] - 1, axis=1)[:, : case["k"]]
    return np.bincount(ids.reshape(-1), minlength=case["E"])


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "encode":
        std = 1.0 if case["rows"] < 64 else STD
        return dict(case=case, x=(_randn(gen, case["rows"], case["K"]) * std).to(dtype))
    n = _counts(case)
    E, M, K, P = case["E"], case["M"], case["K"], int(n.sum()) + case["pad"]
    s = dict(case=case, x=_randn(gen, P, K).to(dtype))
    s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device=DEV)
    # the row lists of the experts that have rows, as a batched product takes them
    act = np.flatnonzero(n)
    first = np.concatenate([[0], np.cumsum(n)])[act]
    at = np.minimum(np.arange(n.max()), n[act][:, None] - 1)
    s["active"] = torch.tensor(act, device=DEV)
    s["rows"] = torch.tensor(first[:, None] + at, device=DEV)
    s["valid"] = torch.tensor(np.arange(n.max()) < n[act][:, None], device=DEV)
    if case["kind"] == "mx":
        # quantised one expert at a time (the 32-bit temporaries are large)
        parts = [_encode(_randn(gen, 1, M, K) * STD) for _ in range(E)]
        s["codes"] = torch.cat([c for c, _ in parts])
        s["scales"] = torch.cat([b for _, b in parts])
        if own:   # the handle that a program builds once beside its weights
            from block_lut_amd.formats import MXFP4Stack
            s["stack"] = MXFP4Stack(s["codes"], s["scales"])
    else:
        s["w"] = torch.empty((E, M, K), dtype=dtype, device=DEV)
        for e in range(E):
            s["w"][e] = _randn(gen, M, K) * STD
    if case["kind"] == "train":
        s["dy"] = _randn(gen, P, M).to(dtype)
        s["x"].requires_grad_()
        s["w"].requires_grad_()
    return s


# ------------------------------------------------------------- plain forms

def _power_of_two(byte):
    """2^(byte - 127) for bytes of 1 to 254: the exponent of a 32-bit float (a byte of 0 is a
    block of zeros here)."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _encode(x):
    """MXFP4 codes (two a byte, the even element in the low four bits) and scale bytes: the
    largest power of two not above the block's largest magnitude, divided by 4; elements
    rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even code, past 6 to 6."""
    x = x.float()
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    exponent = torch.frexp(amax).exponent - 1
    byte = torch.where(amax > 0, (exponent - 2 + 127).clamp(0, 254), 0)
    t = (b * _power_of_two(254 - byte)).abs()
    code = ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5))
    code = (code + 8 * torch.signbit(b)).to(torch.uint8).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], byte[..., 0].to(torch.uint8)


def _decode(codes, scales):
    """The values of MXFP4 codes in 32 bits."""
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    levels = torch.cat([levels, -levels])
    v = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], -1).flatten(-2)
    return (v.unflatten(-1, (-1, 32)) * _power_of_two(scales)[..., None]).flatten(-2)


def _batched(rows, s):
    """Each active expert's rows, padded with zeros to the longest list."""
    return torch.where(s["valid"][..., None], rows[s["rows"]], 0.0)


def _scatter(y, s, P, dtype):
    """The batched rows back at their places; rows of no expert are zero."""
    out = torch.zeros((P, y.shape[-1]), dtype=dtype, device=y.device)
    out[s["rows"][s["valid"]]] = y[s["valid"]].to(dtype)
    return out


def run(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "encode":
        return _run_encode(x)
    if case["kind"] == "mx":
        return _run_mx(state, x, DTYPES[case["out"]])
    if case["kind"] == "dense":
        return _run_dense(state, x, DTYPES[case["out"]])
    return _run_train(state, x)


def _run_encode(x):
    if own:
        from block_lut_amd import ops
        from block_lut_amd.formats import MXFP4Stack
        return ops.dequant(MXFP4Stack(*ops.mxfp4_encode(x)))[0]
    return _decode(*_encode(x)).to(torch.bfloat16)


def _run_mx(s, x, out):
    case = s["case"]
    if own:
        from block_lut_amd import ops
        if case["E"] == 1 and not case["x4"] and not case["pad"]:
            return ops.gemv(s["stack"], x, out_dtype=out)
        if case["x4"]:
            codes, scales = ops.mxfp4_encode(x)
            return ops.grouped_gemm(codes, s["stack"], s["offsets"], x_scales=scales, out_dtype=out)
        return ops.grouped_gemm(x, s["stack"], s["offsets"], out_dtype=out)
    rows = _decode(*_encode(x)) if case["x4"] else x.float()
    w = _decode(s["codes"][s["active"]], s["scales"][s["active"]])
    y = torch.bmm(_batched(rows, s), w.transpose(1, 2).contiguous())
    return _scatter(y, s, x.shape[0], out)


def _run_dense(s, x, out):
    if own:
        from block_lut_amd import ops
        return ops.grouped_gemm(x, s["w"], s["offsets"], out_dtype=out)
    w = s["w"][s["active"]].float()
    y = torch.bmm(_batched(x.float(), s), w.transpose(1, 2).contiguous())
    return _scatter(y, s, x.shape[0], out)


def _run_train(s, x):
    if own:
        from block_lut_amd import ops
        y = ops.grouped_linear(x, s["w"], s["offsets"])
        dx, dw = torch.autograd.grad(y, (x, s["w"]), s["dy"])
        return dict(y=y.detach(), dx=dx, dw=dw)
    with torch.no_grad():
        w = s["w"][s["active"]].float()
        xb, dyb = _batched(x.float(), s), _batched(s["dy"].float(), s)
        y = _scatter(torch.bmm(xb, w.transpose(1, 2).contiguous()), s, x.shape[0], x.dtype)
        dx = _scatter(torch.bmm(dyb, w), s, x.shape[0], x.dtype)
        dw = torch.zeros_like(s["w"])
        dw[s["active"]] = torch.bmm(dyb.transpose(1, 2).contiguous(), xb).to(x.dtype)
        return dict(y=y, dx=dx, dw=dw)


# ------------------------------------------------------------- work, exact

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["kind"] == "encode":
        n = case["rows"] * case["K"]
        # the values read; codes and scales written, and read for the values written
        return dict(bytes=n * (size[case["dtype"]] + 2 * (1 / 2 + 1 / 32) + 2), flops=0)
    n = _counts(case)
    rows, P, M, K = int(n.sum()), int(n.sum()) + case["pad"], case["M"], case["K"]
    touched = int(np.count_nonzero(n))
    flops = 2 * rows * M * K
    if case["kind"] == "mx":
        return dict(bytes=rows * K * 2 + touched * M * K * (1 / 2 + 1 / 32) + P * M * size[case["out"]], flops=flops)
    if case["kind"] == "dense":
        return dict(bytes=rows * K * 2 + touched * M * K * 2 + P * M * size[case["out"]], flops=flops)
    return dict(bytes=2 * (rows * (K + M) + touched * M * K + P * (M + K) + case["E"] * M * K), flops=3 * flops)


def _nearest_e2m1(x):
    """64-bit values of the MXFP4 code nearest to each element, by the distance to every
    level (of two equally near ones the one with the even code)."""
    b = x.double().reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(amax.clamp(min=2.0 ** -125))) - 2)
    t = b.abs() / scale
    levels = torch.tensor([0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0], dtype=torch.float64, device=x.device)   # even codes first
    value = levels[(t[..., None] - levels).abs().argmin(-1)]
    return (torch.sign(b) * value * scale).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].detach()
        if case["kind"] == "encode":
            return torch.cat([_nearest_e2m1(p) for p in x.split(256)])
        ends = np.cumsum(_counts(case))
        x = torch.cat([_nearest_e2m1(p) for p in x.split(1024)]) if case["x4"] else x.double()
        y = torch.zeros((x.shape[0], case["M"]), dtype=torch.float64, device=DEV)
        dx = torch.zeros_like(x)
        dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=DEV) if case["kind"] == "train" else None
        grid = np.array([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12]) / 2.0
        for e, (a, b) in enumerate(zip(np.concatenate([[0], ends[:-1]]).tolist(), ends.tolist())):
            if a == b:
                continue
            if case["kind"] == "mx":
                c = s["codes"][e].long()
                w = torch.empty((case["M"], case["K"]), dtype=torch.float64, device=DEV)
                w[:, 0::2], w[:, 1::2] = (torch.tensor(grid, device=DEV)[i] for i in (c % 16, c // 16))
                w *= (2.0 ** (s["scales"][e].double() - 127)).repeat_interleave(32, 1)
            else:
                w = s["w"][e].double()
            y[a:b] = x[a:b] @ w.T
            if case["kind"] == "train":
                dy = s["dy"][a:b].double()
                dx[a:b] = dy @ w
                dw[e] = dy.T @ x[a:b]
        return dict(y=y, dx=dx, dw=dw) if case["kind"] == "train" else y
