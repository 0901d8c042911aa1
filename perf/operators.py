"""Operators on 8-bit floating-point blocks: the calls that a training step or a server makes of them.

Values are held as OCP e4m3 codes with one float32 scale for every 128 consecutive values of a row
(the last block of a row may be shorter), or for every 128 x 128 block of a weight matrix.

  quantize   values to codes and scales: activations of a step (one scale per row block), or a layer's
             weights (one per 128 x 128 block).  The scale is the smallest power of two that brings the
             block's largest magnitude to 448, the largest e4m3 value, or below.
  dense      act(x w + bias) over blocks; x comes as codes and scales, or as float values that the call
             itself brings into that form.  w is [out, in] ("oi", as checkpoints hold it) or [in, out]
             ("io", the form of the input gradient dy W^T over the same weights).
  wgrad      the weight gradient x^T dy from x kept in 8 bits.
  agrad      the gradient of an activation (or of the gated product act(z) * up) from z (and up) kept
             in 8 bits.

Sizes are those of this repository's benchmark workloads and tests, and sizes around them.
Activations are normal with rows and channels of different magnitudes, weights N(0, 0.02).
"""
from __future__ import annotations

import math

import torch

own = False  # False: the plain forms below; True: the framework's operators

BLOCK = 128
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2, "f8": 1}
ACTIVATIONS = {"none": 0, "gelu": 1, "relu": 2, "silu": 3, "hardswish": 4, "tanh": 5}
MAX_MULTIPLY_ADDS = 2048 * 4096 * 14336  # of a drawn case: the largest listed one's
MAX_VALUES = 2048 * 14336                # of a drawn elementwise case


def _blocks(n):
    return -(-n // BLOCK)


# -------------------------------------------------------------------------------------------------
# Cases.
# -------------------------------------------------------------------------------------------------
def _quantize(M, K, x="bf16", rows=1):
    return {"kind": "quantize", "M": M, "K": K, "x": x, "rows": rows}


def _dense(M, K, N, x="f8", layout="oi", out="bf16", bias=False, act="none"):
    return {"kind": "dense", "M": M, "K": K, "N": N, "x": x, "layout": layout, "out": out, "bias": bias, "act": act}


def _wgrad(M, K, N, dy="bf16", layout="oi", out="f32"):
    return {"kind": "wgrad", "M": M, "K": K, "N": N, "dy": dy, "layout": layout, "out": out}


def _agrad(M, N, act, dy="bf16", gated=False):
    return {"kind": "agrad", "M": M, "N": N, "act": act, "dy": dy, "gated": gated}


def listed():
    cases = {
        # The activations of eight decoding sequences before a projection: the smallest call.
        "quantize_decode8": _quantize(8, 4096),
        # A prompt's activations, odd length, float32, kept for the backward pass.
        "quantize_prompt1333_f32": _quantize(1333, 11008, "f32"),
        # A layer's master weights brought into 8 bits again after an optimizer step.
        "quantize_weights_f32": _quantize(14336, 4096, "f32", BLOCK),
        # One token through an up projection: autoregressive decode of one sequence.
        "dense_decode": _dense(1, 4096, 11008, x="bf16"),
        # A serving step that mixes decoding sequences and short prompt pieces: an odd row count.
        "dense_mixed97_silu": _dense(97, 4096, 14336, x="bf16", act="silu"),
        # Prompt processing (prefill) with the exact GELU and a bias.
        "dense_prefill_gelu": _dense(2048, 4096, 4096, bias=True, act="gelu"),
        # The input gradient of a down projection of 2048 tokens: dy in bf16, the weights as the forward pass has them.
        "dense_input_gradient": _dense(2048, 14336, 4096, x="bf16", layout="io"),
        # A vocabulary head of odd width over sixteen sequences, float32 logits.
        "dense_head16_odd": _dense(16, 2048, 32001, x="bf16", out="f32"),
        # The weight gradient of a small projection of an embedding model, float32, an odd token count.
        "wgrad_333_f32": _wgrad(333, 1536, 384, dy="f32", layout="io"),
        # The weight gradient of an up projection over 2048 tokens: the largest case.
        "wgrad_2048": _wgrad(2048, 4096, 14336),
        # The gradient of a GELU layer of an embedding model, float32.
        "agrad_333_gelu_f32": _agrad(333, 1536, "gelu", dy="f32"),
        # The gradient of a gated MLP's product over 2048 tokens.
        "agrad_gated_silu": _agrad(2048, 14336, "silu", gated=True),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of the range: a multiple of 128, of 16, or any."""
    unit = rng.choice([128, 128, 16, 1])
    return unit * max(1, _log_int(rng, lo, hi) // unit)


def draw(rng):
    kind = rng.choice(["quantize", "dense", "dense", "dense", "wgrad", "wgrad", "agrad"])
    act = rng.choice(["none", "silu", "gelu", "relu", "hardswish", "tanh"])
    K, N = _size(rng, 256, 14336), _size(rng, 256, 14336)
    rows = min(_log_int(rng, 1, 4096), max(1, MAX_MULTIPLY_ADDS // (K * N)))
    if kind == "quantize":
        M = min(_log_int(rng, 1, 8192), max(1, MAX_VALUES // K))
        return _quantize(M, K, rng.choice(["f32", "bf16"]), rng.choice([1, 1, BLOCK]))
    if kind == "dense":
        return _dense(rows, K, N, rng.choice(["f8", "bf16", "f32"]), rng.choice(["oi", "oi", "io"]), rng.choice(["bf16", "f32"]),
                      rng.random() < 0.3, act)
    if kind == "wgrad":
        return _wgrad(rows, K, N, rng.choice(["bf16", "bf16", "f32"]), rng.choice(["oi", "io"]), rng.choice(["bf16", "f32"]))
    M = min(_log_int(rng, 1, 8192), max(1, MAX_VALUES // N))
    return _agrad(M, N, act, rng.choice(["bf16", "f32"]), rng.random() < 0.5)


# -------------------------------------------------------------------------------------------------
# Inputs, made on the GPU from the seed alone.
# -------------------------------------------------------------------------------------------------
def _activations(g, M, K, dtype="f32"):
    """Normal values whose rows and channels differ in magnitude, as those of a network do."""
    def spread(*shape):
        return torch.exp(0.5 * torch.randn(*shape, generator=g, device="cuda"))

    return (torch.randn(M, K, generator=g, device="cuda") * spread(M, 1) * spread(1, K)).to(TORCH[dtype])


def _kept(g, M, K):
    """Activations in 8 bits, as an earlier call left them."""
    return _plain_quantize(_activations(g, M, K), 1)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))
    kind, M = case["kind"], case["M"]
    t = {}
    if kind == "quantize":
        std = 0.02 if case["rows"] > 1 else 1.0
        t["x"] = (std * _activations(g, M, case["K"])).to(TORCH[case["x"]])
    elif kind == "dense":
        K, N = case["K"], case["N"]
        if case["x"] == "f8":
            t["x"], t["x_scale"] = _kept(g, M, K)
        else:
            t["x"] = _activations(g, M, K, case["x"])
        shape = (N, K) if case["layout"] == "oi" else (K, N)
        t["w"], t["w_scale"] = _plain_quantize(0.02 * torch.randn(*shape, generator=g, device="cuda"), BLOCK)
        # Scales as a trained checkpoint has them: any float32 value.
        t["w_scale"] = t["w_scale"] * (0.75 + 0.5 * torch.rand(t["w_scale"].shape, generator=g, device="cuda"))
        if case["bias"]:
            t["bias"] = 0.1 * torch.randn(N, generator=g, device="cuda")
    elif kind == "wgrad":
        t["x"], t["x_scale"] = _kept(g, M, case["K"])
        t["dy"] = (0.01 * _activations(g, M, case["N"])).to(TORCH[case["dy"]])
    else:
        t["z"], t["z_scale"] = _kept(g, M, case["N"])
        if case["gated"]:
            t["up"], t["up_scale"] = _kept(g, M, case["N"])
        t["dy"] = (0.01 * _activations(g, M, case["N"])).to(TORCH[case["dy"]])
    return {"case": case, "tensors": t}


# -------------------------------------------------------------------------------------------------
# The operators in plain form: float32 values, rounded once at the end.
# -------------------------------------------------------------------------------------------------
def _tiles(x, rows):
    """x [M, K], padded with zeros, as [row blocks, rows, column blocks, 128]."""
    M, K = x.shape
    m, k = -(-M // rows), _blocks(K)
    padded = torch.zeros(m * rows, k * BLOCK, dtype=x.dtype, device=x.device)
    padded[:M, :K] = x
    return padded.reshape(m, rows, k, BLOCK)


def _plain_quantize(x, rows):
    M, K = x.shape
    t = _tiles(x.float(), rows)
    finite = torch.isfinite(t)
    largest = torch.where(finite, t.abs(), 0.0).amax((1, 3))
    mantissa, exponent = torch.frexp(largest)  # mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.clamp(torch.where(mantissa <= 0.875, exponent - 9, exponent - 8), min=-126)
    scale = torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), exponent), 1.0)
    v = torch.where(finite, t / scale[:, None, :, None], float("nan"))
    codes = v.reshape(-1, t.shape[2] * BLOCK)[:M, :K].contiguous().to(torch.float8_e4m3fn)
    return codes, scale


def _spread(scale, rows, shape):
    """A scale for every value: [ceil(M / rows), ceil(K / 128)] to [M, K]."""
    s = scale.repeat_interleave(rows, 0) if rows > 1 else scale
    return s[:shape[0]].repeat_interleave(BLOCK, 1)[:, :shape[1]]


def _values(codes, scale, rows=1):
    return codes.float() * _spread(scale, rows, codes.shape)


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "hardswish":
        return v * torch.clamp(v / 6 + 0.5, 0, 1)
    return torch.clamp(v, min=0) if act == "relu" else torch.tanh(v) if act == "tanh" else v


def _act_slope(v, act):
    one = torch.ones_like(v)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * math.sqrt(0.5 / math.pi)
    if act == "silu":
        s = 1 / (1 + torch.exp(-v))
        return s * (1 + v * (1 - s))
    if act == "hardswish":
        return torch.where(v <= -3, 0 * one, torch.where(v >= 3, one, v / 3 + 0.5))
    if act == "tanh":
        return 1 - torch.tanh(v) ** 2
    return (v > 0).to(v.dtype) if act == "relu" else one


def _plain(case, t):
    kind = case["kind"]
    if kind == "quantize":
        codes, scale = _plain_quantize(t["x"], case["rows"])
        return {"codes": codes, "scale": scale}
    if kind == "dense":
        x, scale = (t["x"], t["x_scale"]) if case["x"] == "f8" else _plain_quantize(t["x"], 1)
        w = _values(t["w"], t["w_scale"], BLOCK)
        y = _values(x, scale) @ (w.t() if case["layout"] == "oi" else w)
        if case["bias"]:
            y = y + t["bias"]
        return _act(y, case["act"]).to(TORCH[case["out"]])
    if kind == "wgrad":
        x, dy = _values(t["x"], t["x_scale"]), t["dy"].float()
        return (dy.t() @ x if case["layout"] == "oi" else x.t() @ dy).to(TORCH[case["out"]])
    z, dy = _values(t["z"], t["z_scale"]), t["dy"].float()
    if not case["gated"]:
        return (dy * _act_slope(z, case["act"])).to(t["dy"].dtype)
    up = _values(t["up"], t["up_scale"])
    return {"dz": (dy * up * _act_slope(z, case["act"])).to(t["dy"].dtype), "dup": (dy * _act(z, case["act"])).to(t["dy"].dtype)}


# -------------------------------------------------------------------------------------------------
# The framework's operators, over device pointers.
# -------------------------------------------------------------------------------------------------
_open = []


def _bind(state):
    """The call's argument block and output buffers, as a program keeps them for a layer."""
    import compute_amd as ca

    if not _open:
        _open.append(ca.New("mi355x"))
    backend, lib = _open[0], ca._lib
    case, t = state["case"], state["tensors"]
    kind, M = case["kind"], case["M"]
    dtypes = {"f32": int(ca.Float32), "bf16": int(ca.BFloat16), "f8": int(ca.F8E4M3FN)}
    ptr = {n: v.data_ptr() for n, v in t.items()}

    def empty(*shape, dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if kind == "quantize":
        K, rows = case["K"], case["rows"]
        out = {"codes": empty(M, K, dtype=torch.float8_e4m3fn), "scale": empty(-(-M // rows), _blocks(K), dtype=torch.float32)}
        a = lib.mx_f8_quantize_args(x=ptr["x"], codes=out["codes"].data_ptr(), scale=out["scale"].data_ptr(), M=M, K=K,
                                    x_dtype=dtypes[case["x"]], block_rows=rows)
        return backend.F8Quantize, a, out
    if kind == "dense":
        K, N = case["K"], case["N"]
        out = empty(M, N, dtype=TORCH[case["out"]])
        a = lib.mx_f8_dense_args(x=ptr["x"], x_scale=ptr.get("x_scale"), w=ptr["w"], w_scale=ptr["w_scale"], bias=ptr.get("bias"),
                                 out=out.data_ptr(), M=M, K=K, N=N, x_dtype=dtypes[case["x"]], bias_dtype=dtypes["f32"],
                                 out_dtype=dtypes[case["out"]], weight_layout=int(case["layout"] == "oi"), activation=ACTIVATIONS[case["act"]])
        return backend.F8Dense, a, out
    if kind == "wgrad":
        K, N = case["K"], case["N"]
        out = empty(*((N, K) if case["layout"] == "oi" else (K, N)), dtype=TORCH[case["out"]])
        a = lib.mx_f8_weight_grad_args(x=ptr["x"], x_scale=ptr["x_scale"], dy=ptr["dy"], out=out.data_ptr(), M=M, K=K, N=N,
                                       dy_dtype=dtypes[case["dy"]], out_dtype=dtypes[case["out"]], weight_layout=int(case["layout"] == "oi"))
        return backend.F8WeightGradient, a, out
    N, dtype = case["N"], t["dy"].dtype
    out = {"dz": empty(M, N, dtype=dtype), "dup": empty(M, N, dtype=dtype)} if case["gated"] else empty(M, N, dtype=dtype)
    dz = out["dz"] if case["gated"] else out
    a = lib.mx_f8_act_grad_args(z=ptr["z"], z_scale=ptr["z_scale"], up=ptr.get("up"), up_scale=ptr.get("up_scale"), dy=ptr["dy"],
                                dz=dz.data_ptr(), dup=out["dup"].data_ptr() if case["gated"] else None, M=M, N=N,
                                dy_dtype=dtypes[case["dy"]], activation=ACTIVATIONS[case["act"]])
    return backend.F8ActivationGradient, a, out


def run(state):
    if own:
        if "bound" not in state:
            state["bound"] = _bind(state)
        call, args, out = state["bound"]
        call(args)
        return out
    return _plain(state["case"], state["tensors"])


# -------------------------------------------------------------------------------------------------
# What a pass cannot do without, and what it has to give.
# -------------------------------------------------------------------------------------------------
def work(case):
    kind, M = case["kind"], case["M"]
    if kind == "quantize":
        K = case["K"]
        return {"bytes": M * K * (BYTES[case["x"]] + 1) + 4 * -(-M // case["rows"]) * _blocks(K), "flops": 0}
    if kind == "dense":
        K, N = case["K"], case["N"]
        x = M * K * BYTES[case["x"]] + (4 * M * _blocks(K) if case["x"] == "f8" else 0)
        w = K * N + 4 * _blocks(K) * _blocks(N)
        return {"bytes": x + w + M * N * BYTES[case["out"]] + 4 * N * case["bias"], "flops": 2 * M * K * N}
    if kind == "wgrad":
        K, N = case["K"], case["N"]
        return {"bytes": M * K + 4 * M * _blocks(K) + M * N * BYTES[case["dy"]] + K * N * BYTES[case["out"]], "flops": 2 * M * K * N}
    N = case["N"]
    kept = (M * N + 4 * M * _blocks(N)) * (2 if case["gated"] else 1)
    return {"bytes": kept + M * N * BYTES[case["dy"]] * (3 if case["gated"] else 2), "flops": 0}


def _decode64(codes):
    """e4m3 codes by their bits: sign, four exponent bits (bias 7), three of mantissa; 0x7f is NaN."""
    b = codes.view(torch.uint8).long()
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2((e - 10).double()))
    v = torch.where((b & 127) == 127, float("nan"), v)
    return torch.where(b > 127, -v, v)


def _wide64(codes, scale, rows):
    i = torch.arange(codes.shape[0], device=codes.device) // rows
    j = torch.arange(codes.shape[1], device=codes.device) // BLOCK
    return _decode64(codes) * scale.double()[i][:, j]


def _quantize64(x, rows):
    """(code values, scales) of a matrix, by the definition, block column by block column."""
    x = x.double()
    M, K = x.shape
    values, scales = torch.empty_like(x), []
    for k in range(0, K, BLOCK):
        part = x[:, k:k + BLOCK]
        top = torch.where(torch.isfinite(part), part.abs(), 0.0).amax(1)
        if rows > 1:
            top = torch.stack([p.amax() for p in top.split(rows)])
        e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -160) / 448))
        e = torch.where(448 * torch.exp2(e - 1) >= top, e - 1, e)
        e = torch.where(448 * torch.exp2(e) < top, e + 1, e)
        s = torch.where(top > 0, torch.exp2(torch.clamp(e, min=-126)), 1.0)
        scales.append(s)
        v = part / s.repeat_interleave(rows)[:M, None]
        step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -20))), min=-6) - 3)
        r = torch.round(v / step) * step  # ties to even
        values[:, k:k + BLOCK] = torch.where(torch.isfinite(part), r, float("nan"))
    return values, torch.stack(scales, 1)


def exact(case, seed):
    t = prepare(case, seed)["tensors"]
    kind, act = case["kind"], case.get("act")
    if kind == "quantize":
        values, scale = _quantize64(t["x"], case["rows"])
        return {"codes": values, "scale": scale}
    if kind == "dense":
        if case["x"] == "f8":
            x = _wide64(t["x"], t["x_scale"], 1)
        else:
            v, s = _quantize64(t["x"], 1)
            x = v * s.repeat_interleave(BLOCK, 1)[:, :case["K"]]
        w = _wide64(t["w"], t["w_scale"], BLOCK)
        y = x @ (w.t() if case["layout"] == "oi" else w)
        return _act64(y + t["bias"].double() if case["bias"] else y, act)
    if kind == "wgrad":
        g = _wide64(t["x"], t["x_scale"], 1).t() @ t["dy"].double()
        return g.t().contiguous() if case["layout"] == "oi" else g
    z, dy = _wide64(t["z"], t["z_scale"], 1), t["dy"].double()
    slope = _slope64(z, act)
    if not case["gated"]:
        return dy * slope
    return {"dz": dy * slope * _wide64(t["up"], t["up_scale"], 1), "dup": dy * _act64(z, act)}


def _normal_cdf64(v):
    return 0.5 * torch.erfc(-v / math.sqrt(2))


def _act64(v, act):
    if act == "gelu":
        return v * _normal_cdf64(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "hardswish":
        return v * torch.minimum(torch.maximum(v + 3, torch.zeros_like(v)), torch.full_like(v, 6)) / 6
    return {"none": lambda u: u, "relu": torch.relu, "tanh": torch.tanh}[act](v)


def _slope64(v, act):
    if act == "gelu":
        return _normal_cdf64(v) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        return torch.sigmoid(v) + v * torch.sigmoid(v) * torch.sigmoid(-v)
    if act == "hardswish":
        return torch.where(v.abs() < 3, (2 * v + 3) / 6, (v > 0).double())
    if act == "tanh":
        return 1 / torch.cosh(v) ** 2
    return (v > 0).double() if act == "relu" else torch.ones_like(v)
