"""The int8 and expert-grouped products that perf measurements run, in their plain form and as calls.

``own`` selects the side: False computes each operator with elementary torch operations in FP32,
True calls the library.  A case is a dict of plain values; ``op`` names the operator:

    linear_int8     activations quantized per token on the way, int8 weights with channel scales
    gemm_int8       the product of codes that are at hand (several projections of one activation)
    weights_int8    weights to int8 codes with one scale per output channel
    grouped         rows grouped by expert times the expert's weights (16-bit types)
    grouped_mxfp8   the same with MXFP8 activations and MXFP8 results
    grouped_int8    the same with int8 codes
    grouped_grad    both gradients of the grouped product
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _case(name, op, M, N, K, E=1, dtype="bf16", out="bf16", bias=False, nk=False):
    return {"name": name, "op": op, "M": M, "N": N, "K": K, "E": E, "dtype": dtype, "out": out, "bias": bias,
            "nk": nk}


def listed():
    return [
        # one token being generated, a wide projection: latency and the weights' bytes
        _case("linear_int8_token", "linear_int8", 1, 12288, 4096),
        # a decoding batch of odd size, odd widths, FP16 with a bias
        _case("linear_int8_odd", "linear_int8", 37, 5003, 2051, dtype="f16", out="f16", bias=True),
        # a prompt through the dense projection
        _case("linear_int8_prompt", "linear_int8", 4096, 12288, 4096),
        # a wide projection of activations quantized once for several of them, weights [N][K]
        _case("gemm_int8_wide", "gemm_int8", 2048, 28672, 8192, nk=True),
        # a model's weights quantized when they are loaded
        _case("weights_int8", "weights_int8", 1, 12288, 4096),
        # a small projection's weights kept in FP32, odd sizes
        _case("weights_int8_odd", "weights_int8", 1, 1001, 515, dtype="f32"),
        # a few tokens through many experts: the chosen experts' weights are all that counts
        _case("grouped_tokens", "grouped", 16, 2048, 2048, E=64),
        # a batch spread unevenly over experts, some of them empty
        _case("grouped_batch", "grouped", 4099, 2816, 2048, E=32),
        # a chunk of a long prompt through few large experts in the framework's own format
        _case("grouped_mxfp8", "grouped_mxfp8", 8192, 4096, 2048, E=8),
        # a serving batch through int8 experts
        _case("grouped_int8", "grouped_int8", 1000, 4096, 2048, E=16),
        # a training step's gradients, small experts, FP32 weight gradients
        _case("grouped_grad", "grouped_grad", 2050, 1408, 1024, E=16, out="f32"),
        # a training step's gradients, few large experts
        _case("grouped_grad_large", "grouped_grad", 16384, 8192, 4096, E=8),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["linear_int8", "linear_int8", "gemm_int8", "weights_int8", "grouped", "grouped",
                     "grouped_mxfp8", "grouped_int8", "grouped_grad", "grouped_grad"])
    M, N, K, E = size(1, 16384), size(64, 12288), size(64, 8192), 1
    if rng.random() < 0.7:  # most models' widths are round, some are not
        N, K = max(64, N // 64 * 64), max(64, K // 64 * 64)
    if op.startswith("grouped"):
        E = size(1, 96)
        N, K = min(N, 8192), min(K, 4096)
    # no more weights than 2 GiB in BF16, no more work than the largest listed case
    while E * N * K > 1 << 30:
        E = max(1, E // 2)
        N = N if E > 1 else max(64, N // 2)
    while M * N * K > 16384 * 8192 * 4096:
        M = max(1, M // 2)
    dtype = "bf16" if op == "grouped_mxfp8" else rng.choice(["bf16", "bf16", "f16"])
    out = "bf16" if op == "grouped_mxfp8" else dtype
    if op == "weights_int8":
        dtype = rng.choice(["bf16", "f16", "f32"])
        M = 1
    case = _case("", op, M, N, K, E=E, dtype=dtype, out=out, bias=op == "linear_int8" and rng.random() < 0.5,
                 nk=op in ("linear_int8", "gemm_int8", "grouped") and rng.random() < 0.3)
    del case["name"]
    return case


def _active(case):
    """Experts that get rows: one in eight stays without, and a few rows reach as few experts."""
    return min(case["M"], case["E"] - case["E"] // 8)


def _padded(shape, dtype, device="cuda"):
    """An empty tensor whose rows start on 16-byte boundaries, as weights and codes are kept."""
    per = 16 // torch.empty((), dtype=dtype).element_size()
    ld = (shape[-1] + per - 1) // per * per
    return torch.empty(tuple(shape[:-1]) + (ld,), dtype=dtype, device=device)[..., :shape[-1]]


def _activations(M, K, gen):
    """Normal values with a scale of their own per row and a few channels that stand out."""
    x = torch.randn((M, K), generator=gen, device="cuda")
    x *= 0.5 + 2.0 * torch.rand((M, 1), generator=gen, device="cuda")
    return x * (1.0 + 15.0 * (torch.rand((1, K), generator=gen, device="cuda") > 0.995))


def _codes_of_columns(w):
    """int8 codes and scales of w [..., K, N] for each column."""
    a = w.abs().amax(-2, keepdim=True).clamp_min(2.0 ** -100)
    return torch.round(w * (torch.full_like(a, 127.0) / a)).to(torch.int8), (a / torch.full_like(a, 127.0)).squeeze(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, M, N, K, E = (case[k] for k in ("op", "M", "N", "K", "E"))
    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if op.startswith("grouped"):
        active = _active(case)
        chosen = torch.randperm(E, generator=gen, device="cuda")[:active]
        share = torch.rand((active,), generator=gen, device="cuda") ** 2 + 0.02
        more = torch.multinomial(share, max(M - active, 1), replacement=True, generator=gen)[:M - active]
        sizes = torch.zeros(E, dtype=torch.int64, device="cuda")
        sizes[chosen] = 1 + torch.bincount(more, minlength=active)
        state["offsets"] = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
        state["most"] = int(sizes.max())  # the largest group, known to the router's program
    if op == "weights_int8":
        state["w"] = (torch.randn((K, N), generator=gen, device="cuda") / math.sqrt(K)).to(dtype)
        return state
    w = torch.randn((E, K, N), generator=gen, device="cuda")
    w /= math.sqrt(K)
    x = _activations(M, K, gen)
    if op in ("linear_int8", "gemm_int8", "grouped_int8"):
        codes, scales = _codes_of_columns(w)
        del w
        if case["nk"]:
            kept = _padded((E, N, K), torch.int8)
            kept.copy_(codes.transpose(1, 2))
        else:
            kept = _padded((E, K, N), torch.int8)
            kept.copy_(codes)
        grouped = op == "grouped_int8"
        state["w"], state["w_scales"] = (kept, scales) if grouped else (kept[0], scales[0])
        state["bias"] = torch.randn((N,), generator=gen, device="cuda") if case["bias"] else None
        if op == "linear_int8":
            state["x"] = x.to(dtype)
        else:
            codes, scales = _codes_of_columns(x.t())
            state["x"] = _padded((M, K), torch.int8)
            state["x"].copy_(codes.t())
            state["x_scales"] = scales.contiguous()
        return state
    shape = (E, N, K) if case["nk"] else (E, K, N)
    state["w"] = _padded(shape, dtype)
    state["w"].copy_(w.transpose(1, 2) if case["nk"] else w)
    del w
    if op == "grouped_mxfp8":
        codes, scales = _mxfp8_of_rows(x)
        state["x"], state["x_scales"] = codes.view(torch.uint8).contiguous(), scales.contiguous()
        return state
    state["x"] = _padded((M, K), dtype)
    state["x"].copy_(x)
    if op == "grouped_grad":
        state["dy"] = _padded((M, N), dtype)
        state["dy"].copy_(torch.randn((M, N), generator=gen, device="cuda") / 8)
    return state


def _mxfp8_of_rows(x):
    """E4M3 codes and power-of-two scale bytes of blocks of 32 values along the rows of FP32 x."""
    M, K = x.shape
    blocks = (K + 31) // 32
    v = torch.nn.functional.pad(x, (0, 32 * blocks - K)).view(M, blocks, 32)
    amax = v.abs().amax(-1)
    mantissa, exponent = torch.frexp((amax / torch.full_like(amax, 448.0)).clamp_min(2.0 ** -126))
    exponent = exponent - (mantissa == 0.5).to(exponent.dtype)
    codes = torch.ldexp(v, -exponent.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.view(M, 32 * blocks)[:, :K], (exponent + 127).to(torch.uint8)


def _mxfp8_values(codes, scales):
    """The FP32 values that MXFP8 rows stand for."""
    exponent = scales.to(torch.int32).repeat_interleave(32, dim=1)[:, :codes.shape[1]] - 127
    return torch.ldexp(codes.to(torch.float32), exponent)


def _places(state, M):
    """(expert, place within its group) of each row."""
    rows = torch.arange(M, device="cuda")
    expert = torch.bucketize(rows, state["offsets"][1:].to(torch.int64), right=True)
    return expert, rows - state["offsets"].to(torch.int64)[expert]


def _by_expert(x, places, E, most):
    """Rows laid out as one zero-padded block per expert."""
    blocks = x.new_zeros((E, most, x.shape[1]))
    blocks[places] = x
    return blocks


def _plain(state):
    case = state["case"]
    op, M, E, out = case["op"], case["M"], case["E"], TYPES[case["out"]]
    if op == "weights_int8":
        return _codes_of_columns(state["w"].float())
    w = state["w"].float()
    if case["nk"]:
        w = w.transpose(-1, -2)
    if op == "linear_int8":
        codes, scales = _codes_of_columns(state["x"].float().t())
        y = (codes.float().t() @ w) * scales.unsqueeze(1) * state["w_scales"]
        return (y if state["bias"] is None else y + state["bias"]).to(out)
    if op == "gemm_int8":
        return ((state["x"].float() @ w) * state["x_scales"].unsqueeze(1) * state["w_scales"]).to(out)
    places = _places(state, M)
    if op == "grouped_mxfp8":
        x = _mxfp8_values(state["x"].view(torch.float8_e4m3fn), state["x_scales"])
    else:
        x = state["x"].float()
    blocks = _by_expert(x, places, E, state["most"])
    if op == "grouped_grad":
        dy = _by_expert(state["dy"].float(), places, E, state["most"])
        return (dy @ w.transpose(1, 2))[places].to(TYPES[case["dtype"]]), (blocks.transpose(1, 2) @ dy).to(out)
    y = (blocks @ w)[places]
    if op == "grouped_int8":
        y = y * state["x_scales"].unsqueeze(1) * state["w_scales"][places[0]]
    if op == "grouped_mxfp8":
        return _mxfp8_values(*_mxfp8_of_rows(y)).to(torch.bfloat16)
    return y.to(out)


def _calls(state):
    import mix_precision_kernel_b200 as mpk

    case = state["case"]
    op, out = case["op"], TYPES[case["out"]]
    if op == "weights_int8":
        return mpk.quantize_int8_cols(state["w"])
    if op == "linear_int8":
        return mpk.linear_int8(state["x"], state["w"], state["w_scales"], bias=state["bias"], out_dtype=out,
                               b_layout=mpk.B_NK if case["nk"] else mpk.B_KN)
    if op == "gemm_int8":
        return mpk.gemm_int8(state["x"], state["x_scales"], state["w"], state["w_scales"], out_dtype=out,
                             b_layout=mpk.B_NK if case["nk"] else mpk.B_KN)
    if op == "grouped_int8":
        return mpk.gemm_grouped_int8(state["x"], state["x_scales"], state["w"], state["w_scales"],
                                     state["offsets"], out_dtype=out)
    if op == "grouped_mxfp8":
        d, s = mpk.gemm_grouped_mxfp8(state["x"], state["x_scales"], state["w"], state["offsets"])
        y = torch.empty(d.shape, dtype=torch.bfloat16, device=d.device)
        mpk.mxfp8_dequantize_bf16_gpu(d, s, y, d.shape[0], d.shape[1])
        return y
    if op == "grouped":
        return mpk.gemm_grouped(state["x"], state["w"], state["offsets"], out_dtype=out,
                                b_layout=mpk.B_NK if case["nk"] else mpk.B_KN)
    # the weights [E][K][N] of the product are, for the gradient of its rows, [E][N'][K'] with N' = K
    dx = mpk.gemm_grouped(state["dy"], state["w"], state["offsets"], out_dtype=TYPES[case["dtype"]],
                          b_layout=mpk.B_NK)
    return dx, mpk.gemm_grouped_wgrad(state["x"], state["dy"], state["offsets"], out_dtype=out)


def run(state):
    return _calls(state) if own else _plain(state)


def work(case):
    op, M, N, K = (case[k] for k in ("op", "M", "N", "K"))
    b, o = BYTES[case["dtype"]], BYTES[case["out"]]
    if op == "weights_int8":
        return {"bytes": K * N * (b + 1) + 4 * N, "flops": 2 * K * N}
    E = _active(case)
    flops = 2 * M * N * K
    if op == "linear_int8":
        n = M * K * b + K * N + 4 * N + M * N * o + (4 * N if case["bias"] else 0)
    elif op == "gemm_int8":
        n = M * K + 4 * M + K * N + 4 * N + M * N * o
    elif op == "grouped_int8":
        n = M * K + 4 * M + E * (K * N + 4 * N) + M * N * o
    elif op == "grouped_mxfp8":
        n = M * K + M * ((K + 31) // 32) + E * K * N * b + M * N * 2
    elif op == "grouped":
        n = M * K * b + E * K * N * b + M * N * o
    else:
        # activations, gradients and weights read, the rows' gradients and every expert's weights' written
        n = M * K * b + M * N * b + E * K * N * b + M * K * b + case["E"] * K * N * o
        flops *= 2
    return {"bytes": n, "flops": flops}


def exact(case, seed):
    """The definitions in 64 bits, one expert after the other, on the inputs of ``seed``."""
    state = prepare(case, seed)
    op = case["op"]

    def codes(v, dim):
        top = v.double().abs().amax(dim, keepdim=True)
        top = torch.maximum(top, torch.full_like(top, 2.0 ** -100))
        return torch.round(127.0 * v.double() / top), top.squeeze(dim) / 127.0

    if op == "weights_int8":
        return None, codes(state["w"], 0)[1]
    w = state["w"].double()
    if case["nk"]:
        w = w.transpose(-1, -2)
    if op in ("linear_int8", "gemm_int8"):
        a, s = codes(state["x"], 1) if op == "linear_int8" else (state["x"].double(), state["x_scales"].double())
        y = torch.einsum("mk,kn->mn", a, w) * s[:, None] * state["w_scales"].double()[None, :]
        return y if state["bias"] is None else y + state["bias"].double()
    ends = state["offsets"].tolist()
    groups = [slice(lo, hi) for lo, hi in zip(ends, ends[1:])]
    if op == "grouped_mxfp8":
        a = state["x"].view(torch.float8_e4m3fn).double()
        factor = torch.pow(2.0, state["x_scales"].double() - 127.0)
        a = a * factor[:, torch.arange(a.shape[1], device="cuda") // 32]
    else:
        a = state["x"].double()
    if op == "grouped_grad":
        dy = state["dy"].double()
        dx = torch.cat([dy[g] @ w[e].t() for e, g in enumerate(groups)])
        return dx, torch.stack([a[g].t() @ dy[g] for g in groups])
    y = torch.cat([a[g] @ w[e] for e, g in enumerate(groups)])
    if op == "grouped_int8":
        y = y * state["x_scales"].double()[:, None]
        y = torch.cat([y[g] * state["w_scales"][e].double() for e, g in enumerate(groups)])
    if op == "grouped_mxfp8":
        top = torch.zeros((y.shape[0], (y.shape[1] + 31) // 32), dtype=torch.float64, device="cuda")
        block = (torch.arange(y.shape[1], device="cuda") // 32).expand_as(y)
        top.scatter_reduce_(1, block, y.abs(), "amax")
        scale = torch.pow(2.0, torch.ceil(torch.log2(torch.clamp(top / 448.0, min=2.0 ** -126)))).gather(1, block)
        v = y / scale
        # E4M3: three bits of fraction above 2^-6, steps of 2^-9 below; ties to even
        step = torch.pow(2.0, torch.clamp(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -20))), min=-6.0) - 3.0)
        y = torch.round(v / step) * step * scale
    return y
