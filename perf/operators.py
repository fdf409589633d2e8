"""Cases of the feed-forward operators: quantisation of tokens, the scaled 8-bit product, the gated block in 16 and
8 bits and the gated block's gradient, each with its plain form in elementary torch operations.

Tensors are row-major with a row per token or channel, which is the column-major matrix of the library's calls with a
column per token or channel: x is [tokens, k], a weight is [rows, k] ("across" false) or [k, rows] ("across" true), an
output is [tokens, rows].  `pad` elements lie behind each row of the inputs.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16", torch.float32: "float32", torch.int8: "int8"}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}

# Most floating operations and bytes that a drawn case may ask for: the largest listed case's.
_MOST_FLOPS = 8.0 * 21504 * 1024 * 4096
_MOST_BYTES = 3.0 * 21504 * 4096


def listed():
    return [
        # the activations of 48 sequences in one decode step, before an 8-bit projection: a call of few microseconds
        dict(name="quantize 48x4096 bf16", op="quantize", n=48, k=4096, dtype="bf16", pad=0),
        # the hidden activations of a whole batch of long sequences
        dict(name="quantize 21504x4096 bf16", op="quantize", n=21504, k=4096, dtype="bf16", pad=0),
        # one token against a vocabulary: nothing but the weights' way out of memory
        dict(name="i8 1x4096->50400 f32", op="scaled", n=1, k=4096, m=50400, dtype="f32", across=False, pad=0),
        # a ragged batch on widths that no tile divides
        dict(name="i8 223x1000->4099 f16", op="scaled", n=223, k=1000, m=4099, dtype="f16", across=False, pad=0),
        # a prefill's down projection
        dict(name="i8 1712x16384->4096 bf16", op="scaled", n=1712, k=16384, m=4096, dtype="bf16", across=False, pad=0),
        # the block in one decode step of 48 sequences
        dict(name="gated 48x4096->16384 bf16", op="gated", n=48, k=4096, m=16384, dtype="bf16", act="silu", keep=False, across=False, pad=0),
        # a ragged prefill, odd number of tokens and of features
        dict(name="gated 2239x1024->2731 f16", op="gated", n=2239, k=1024, m=2731, dtype="f16", act="gelu_tanh", keep=False, across=False, pad=0),
        # the forward pass of a training step: the pre-activations are kept for the backward pass
        dict(name="gated 21504x1024->4096 bf16", op="gated", n=21504, k=1024, m=4096, dtype="bf16", act="silu", keep=True, across=False, pad=0),
        # one token through the 8-bit block
        dict(name="gated i8 1x4096->16384 bf16", op="gated_scaled", n=1, k=4096, m=16384, dtype="bf16", act="silu", across=False, pad=0),
        # a prefill through the 8-bit block
        dict(name="gated i8 1712x4096->16384 f16", op="gated_scaled", n=1712, k=4096, m=16384, dtype="f16", act="silu", across=False, pad=0),
        # a small training step on odd sizes
        dict(name="grad 1119x1000->2730 f16", op="grad", n=1119, k=1000, m=2730, dtype="f16", act="gelu", across=False, pad=0),
        # the backward pass of the training step above
        dict(name="grad 21504x1024->4096 bf16", op="grad", n=21504, k=1024, m=4096, dtype="bf16", act="silu", across=False, pad=0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "scaled", "scaled", "gated", "gated", "gated_scaled", "grad"])
    case = dict(op=op, n=_log_uniform(rng, 1, 21504), k=_log_uniform(rng, 64, 16384), pad=rng.choice([0, 0, 16, 3]))
    if rng.random() < 0.6:  # widths are mostly multiples of 64
        case["k"] = max(64, case["k"] // 64 * 64)
    if op == "quantize":
        case["dtype"] = rng.choice(["bf16", "f16", "f32"])
        while case["n"] * case["k"] * (_BYTES[case["dtype"]] + 1) > _MOST_BYTES:
            case["n"] = case["n"] // 2
        return case
    case["m"] = _log_uniform(rng, 64, 50400 if op == "scaled" else 16384)
    if rng.random() < 0.6:
        case["m"] = max(64, case["m"] // 64 * 64)
    case["dtype"] = rng.choice(["bf16", "f16", "f32"] if op == "scaled" else ["bf16", "f16"])
    case["across"] = rng.random() < 0.2
    if op != "scaled":
        case["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])
    if op == "gated":
        case["keep"] = rng.random() < 0.4
    while case["n"] > 1 and work(case)["flops"] > _MOST_FLOPS:
        case["n"] = case["n"] // 2
    return case


def work(case):
    n, k = case["n"], case["k"]
    e = _BYTES[case["dtype"]]
    if case["op"] == "quantize":
        return {"bytes": float(n * k * (e + 1) + 4 * n), "flops": 3.0 * n * k}
    m = case["m"]
    if case["op"] == "scaled":
        return {"bytes": float(n * k + m * k + 4 * (n + m) + e * n * m), "flops": 2.0 * n * k * m}
    if case["op"] == "gated":
        return {"bytes": float(e * (n * k + 2 * m * k + n * m * (3 if case["keep"] else 1))), "flops": 4.0 * n * k * m}
    if case["op"] == "gated_scaled":
        return {"bytes": float(n * k + 2 * m * k + 4 * (n + 2 * m) + e * n * m), "flops": 4.0 * n * k * m}
    # x, the weights, the pre-activations and the output's gradient in; the gradients of x and of the weights out
    return {"bytes": float(e * (2 * n * k + 4 * m * k + 3 * n * m)), "flops": 8.0 * n * k * m}


# ------------------------------------------------------------------- inputs
def _padded(t, pad):
    """The same matrix with `pad` elements of room behind each row."""
    if not pad:
        return t.contiguous()
    room = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=t.dtype, device=t.device)
    room[:, : t.shape[1]] = t
    return room[:, : t.shape[1]]


def _activations(gen, n, k):
    """Normal values of another size from token to token, some channels much larger than the rest, as hidden states have."""
    x = torch.randn(n, k, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(n, 1, generator=gen, device="cuda"))
    x *= torch.where(torch.rand(1, k, generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    n, k, op, pad = case["n"], case["k"], case["op"], case["pad"]
    state = dict(case)
    if op == "quantize":
        x = _activations(gen, n, k)
        if n > 8:
            x[n // 2] = 0.0  # a padding token
        state["x"] = _padded(x.to(_DTYPES[case["dtype"]]), pad)
        return state
    dtype = _DTYPES[case["dtype"]]
    m = case["m"]
    rows = m if op == "scaled" else 2 * m
    if op in ("scaled", "gated_scaled"):
        x = torch.clamp(torch.round(24.0 * torch.randn(n, k, generator=gen, device="cuda")), -127, 127).to(torch.int8)
        w = torch.clamp(torch.round(32.0 * torch.randn(rows, k, generator=gen, device="cuda")), -127, 127).to(torch.int8)
        state["x_scale"] = 0.03 * torch.exp(0.5 * torch.randn(n, generator=gen, device="cuda"))
        state["w_scale"] = torch.exp(0.3 * torch.randn(rows, generator=gen, device="cuda")) / (32.0 * math.sqrt(k))
    else:
        x = _activations(gen, n, k).to(dtype)
        w = (torch.randn(rows, k, generator=gen, device="cuda") / math.sqrt(k)).to(dtype)
    state["x"] = _padded(x, pad)
    state["w"] = _padded(w.t() if case["across"] else w, pad)
    if op == "grad":
        state["p"] = torch.randn(n, 2 * m, generator=gen, device="cuda").to(dtype)
        state["dh"] = (0.01 * torch.randn(n, m, generator=gen, device="cuda")).to(dtype)
        # where the gradient of the pre-activations goes between the two halves of the backward pass
        ld = (2 * m + 7) // 8 * 8
        state["dp"] = torch.empty(n, ld, dtype=dtype, device="cuda")
    return state


# -------------------------------------------------------------- plain forms
def _act(g, act):
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    if act == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
    return torch.where(g > 0, g, torch.zeros_like(g))


def _act_slope(g, act):
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return s * (1.0 + g * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5))) + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g * g * g))
        return 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * g * g)
    return (g > 0).to(g.dtype)


def _plain_quantize(x):
    largest = x.float().abs().amax(dim=1, keepdim=True)
    # 127 x / largest next to a half has to round as the real number does
    r = torch.round(127.0 * x.double() / torch.where(largest > 0, largest, torch.ones_like(largest)).double())
    return r.to(torch.int8), (largest / 127.0).reshape(-1)


def _plain(s):
    op = s["op"]
    if op == "quantize":
        return _plain_quantize(s["x"])
    x = s["x"].float()
    w = s["w"].float() if s["across"] else s["w"].float().t()  # [k, rows]
    dtype, m = _DTYPES[s["dtype"]], s["m"]
    if op == "scaled":
        return (x @ w * s["x_scale"][:, None] * s["w_scale"][None, :]).to(dtype)
    if op == "grad":
        p, dh = s["p"].float(), s["dh"].float()
        g, u = p[:, :m], p[:, m:]
        dp = torch.cat([dh * u * _act_slope(g, s["act"]), dh * _act(g, s["act"])], dim=1)
        dw = x.t() @ dp if s["across"] else dp.t() @ x
        return dw.to(dtype), (dp @ w.t()).to(dtype)
    p = x @ w
    if op == "gated_scaled":
        p = p * s["x_scale"][:, None] * s["w_scale"][None, :]
    h = (_act(p[:, :m], s["act"]) * p[:, m:]).to(dtype)
    return (h, p.to(dtype)) if op == "gated" and s["keep"] else h


# ------------------------------------------------------ the framework's calls
_handle = None


def _library():
    """The package and the handle that the program keeps, on torch's default stream."""
    global _handle
    import sycl_blas_amd as sb

    if _handle is None:
        _handle = sb.SB_Handle(torch.cuda.current_device(), stream=1)  # 1 names the device's default stream (hipStreamLegacy)
    return sb, _handle


def _run_own(s):
    sb, handle = _library()

    def buf(t):
        return sb.DeviceBuffer.from_pointer(t.data_ptr(), _NAMES[t.dtype], t.numel())

    op, n, k, x = s["op"], s["n"], s["k"], s["x"]
    ldx = x.stride(0)
    if op == "quantize":
        q = torch.empty(n, k, dtype=torch.int8, device="cuda")
        scale = torch.empty(n, dtype=torch.float32, device="cuda")
        sb._quantize(handle, k, n, buf(x), ldx, buf(q), k, buf(scale))
        return q, scale
    w, m, dtype = s["w"], s["m"], _DTYPES[s["dtype"]]
    trans, ldw = ("n" if s["across"] else "t"), w.stride(0)
    if op == "grad":
        dw = torch.empty(w.shape, dtype=dtype, device="cuda")
        dx = torch.empty(n, k, dtype=dtype, device="cuda")
        dp = s["dp"]
        sb._gated_gemm_grad(handle, sb.activation_t[s["act"]], trans, "n", m, n, k, buf(w), ldw, buf(x), ldx, buf(s["p"]), 2 * m,
                            buf(s["dh"]), m, buf(dp), dp.shape[1], 0.0, buf(dw), w.shape[1], 0.0, buf(dx), k)
        return dw, dx
    c = torch.empty(n, m, dtype=dtype, device="cuda")
    if op == "scaled":
        sb._gemm_scaled(handle, trans, "n", m, n, k, 1.0, buf(w), ldw, buf(s["w_scale"]), buf(x), ldx, buf(s["x_scale"]), 0.0,
                        buf(c), m)
        return c
    act = sb.activation_t[s["act"]]
    if op == "gated_scaled":
        sb._gated_gemm_scaled(handle, act, trans, "n", m, n, k, buf(w), ldw, buf(s["w_scale"]), buf(x), ldx, buf(s["x_scale"]),
                              buf(c), m)
        return c
    if s["keep"]:
        p = torch.empty(n, 2 * m, dtype=dtype, device="cuda")
        sb._gated_gemm(handle, act, trans, "n", m, n, k, buf(w), ldw, buf(x), ldx, buf(c), m, buf(p), 2 * m)
        return c, p
    sb._gated_gemm(handle, act, trans, "n", m, n, k, buf(w), ldw, buf(x), ldx, buf(c), m)
    return c


def run(state):
    return _run_own(state) if own else _plain(state)


# ------------------------------------------------------------------- in 64 bits
def _gate64(p, m, act):
    g, u = p[:, :m], p[:, m:]
    if act == "silu":
        return g * torch.sigmoid(g) * u
    if act == "gelu":
        return 0.5 * g * torch.special.erfc(-g / math.sqrt(2.0)) * u
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(g, approximate="tanh") * u
    return torch.clamp(g, min=0.0) * u


def exact(case, seed):
    s = prepare(case, seed)
    x, op = s["x"].to(torch.float64), case["op"]
    if op == "quantize":
        largest = torch.linalg.vector_norm(x, ord=math.inf, dim=1)
        q = torch.round(x * 127.0 / torch.clamp(largest, min=torch.finfo(torch.float64).tiny)[:, None])
        return q.to(torch.int8), largest / 127.0
    w = s["w"].to(torch.float64)
    w = w.transpose(0, 1) if case["across"] else w  # [rows, k]
    m = case["m"]
    if op == "grad":
        p = s["p"].to(torch.float64).requires_grad_(True)
        (dp,) = torch.autograd.grad(_gate64(p, m, case["act"]), p, s["dh"].to(torch.float64))
        dw = torch.mm(dp.transpose(0, 1), x)
        return (dw.transpose(0, 1).contiguous() if case["across"] else dw), torch.mm(dp, w)
    p = torch.mm(x, w.transpose(0, 1))
    if "x_scale" in s:
        p *= torch.outer(s["x_scale"].to(torch.float64), s["w_scale"].to(torch.float64))
    if op == "scaled":
        return p
    h = _gate64(p, m, case["act"])
    return (h, p) if op == "gated" and case["keep"] else h
