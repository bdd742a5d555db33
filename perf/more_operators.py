"""The operators of a forward with 8-bit activations and 4-bit weights, as calls of the public Python
binding (qattn.py) that can be timed and compared: rows into 8 bits (a plain row, or a residual sum and its
norm) and the products of such rows with 4-bit weights.

A case is a dict of plain values.  `kind` names the call:

  norm      Context.rmsnorm_q8: residual sum, RMSNorm, 8-bit codes and a scale for each row
  quantize  Context.quantize_q8: rows as 8-bit codes and scales
  product   Context.w4_matmul: 8-bit rows times 4-bit weights with group scales
  swiglu    Context.w4_matmul_swiglu: the gate and up products of an FFN and SwiGLU of them"""
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-6
GROUP = 32  # columns that share a multiplier and a zero point
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST_VALUES, MOST_FLOPS, MOST_ROWS = 16_384_000, 2.3e11, 20000


def listed():
    return [
        # The rows of a step of 16 requests, as the model's layers normalise them: latency.
        {"name": "norm_16", "kind": "norm", "rows": 16, "width": 1024, "residual": True, "dtype": "f16"},
        # A full batch of 16 requests of 500 tokens.
        {"name": "norm_8000", "kind": "norm", "rows": 8000, "width": 1024, "residual": True, "dtype": "f16"},
        # A ragged batch of a wider model, the first norm of a forward: no residual yet.
        {"name": "norm_1419_wide", "kind": "norm", "rows": 1419, "width": 2560, "residual": False, "dtype": "bf16"},
        # The attention output of a step of 64 tokens on its way into the output projection.
        {"name": "quantize_64", "kind": "quantize", "rows": 64, "width": 2048, "dtype": "f16"},
        # That of a full batch.
        {"name": "quantize_8000", "kind": "quantize", "rows": 8000, "width": 2048, "dtype": "f16"},
        # One token through a wide projection: a matrix-vector product.
        {"name": "vector_4096", "kind": "product", "rows": 1, "k": 4096, "n": 8192, "dtype": "bf16"},
        # A step of 16 tokens through the QKV projection.
        {"name": "qkv_16", "kind": "product", "rows": 16, "k": 1024, "n": 4096, "dtype": "f16"},
        # 16 ragged requests through the output projection.
        {"name": "output_1419", "kind": "product", "rows": 1419, "k": 2048, "n": 1024, "dtype": "f16"},
        # A few requests through a projection whose sizes fill no tile.
        {"name": "odd_333", "kind": "product", "rows": 333, "k": 2592, "n": 1001, "dtype": "bf16"},
        # A full batch through the QKV projection.
        {"name": "qkv_8000", "kind": "product", "rows": 8000, "k": 1024, "n": 4096, "dtype": "f16"},
        # One request of 50 tokens through an FFN's first half.
        {"name": "gate_up_50", "kind": "swiglu", "rows": 50, "k": 1024, "n": 2816, "dtype": "f16"},
        # Four documents of 5,000 tokens through it: the largest.
        {"name": "gate_up_20000", "kind": "swiglu", "rows": 20000, "k": 1024, "n": 2816, "dtype": "f16"},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("norm", "quantize", "product", "product", "product", "swiglu", "swiglu"))
    case = {"kind": kind, "rows": _log_int(rng, 1, MOST_ROWS), "dtype": rng.choice(("f16", "bf16"))}
    if kind in ("norm", "quantize"):
        case["width"] = 8 * _log_int(rng, 1, 2048)
        case["rows"] = min(case["rows"], MOST_VALUES // case["width"])
        return {**case, "residual": rng.random() < 0.7} if kind == "norm" else case
    case["k"] = 32 * _log_int(rng, 1, 256)
    # Outputs of any count; SwiGLU's features in whole tiles of 32.
    case["n"] = _log_int(rng, 1, 8192) if kind == "product" else 32 * _log_int(rng, 1, 128)
    per_row = 2 * case["k"] * case["n"] * (2 if kind == "swiglu" else 1)
    case["rows"] = max(1, min(case["rows"], int(MOST_FLOPS) // per_row))
    return case


# ---- the library ----------------------------------------------------------------------------


def _binding():
    if "qattn" not in sys.modules:
        path = os.path.join(ROOT, "qwen3-embedding-webgpu-prepacked_amd", "qattn.py")
        spec = importlib.util.spec_from_file_location("qattn", path)
        sys.modules["qattn"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["qattn"])
    return sys.modules["qattn"]


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        _ctx = _binding().Context(0)
    return _ctx


# ---- inputs ---------------------------------------------------------------------------------


class State:
    """What a program holds between calls."""

    def __init__(self, **parts):
        self.__dict__.update(parts)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(g, dtype, rows, width):
    """Activations as a residual stream or an attention holds them: rows of unlike sizes, and channels that
    are larger than the others."""
    size = torch.exp(0.5 * _randn(g, rows, 1)) * torch.exp(0.7 * _randn(g, 1, width))
    return (_randn(g, rows, width) * size).to(dtype)


def _row_inputs(case, seed):
    """(rows, residual or None, gains or None)"""
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    x = _rows(g, dtype, case["rows"], case["width"])
    if case["kind"] == "quantize":
        return x, None, None
    residual = _rows(g, dtype, case["rows"], case["width"]) if case["residual"] else None
    return x, residual, 1.0 + 0.2 * _randn(g, case["width"])


def _product_inputs(case, seed):
    """8-bit rows and their scales; weights as codes (two to a byte, even columns low), a byte for each group
    (multiplier low, zero point high) and a scale for each row."""
    g = _generator(seed)
    k, n = case["k"], case["n"] * (2 if case["kind"] == "swiglu" else 1)
    x = _randn(g, case["rows"], k)
    most = x.abs().amax(-1, keepdim=True)
    codes_x = torch.round(x * (127.0 / most)).to(torch.int8)
    scale_x = (most[:, 0] / 127.0) * torch.exp(0.3 * _randn(g, case["rows"]))
    zero = 7 + torch.randint(0, 2, (n, k // GROUP), generator=g, device="cuda")
    mult = torch.randint(5, 16, (n, k // GROUP), generator=g, device="cuda")
    codes = torch.round(2.7 * _randn(g, n, k)).to(torch.int64) + zero.repeat_interleave(GROUP, 1)
    codes = codes.clamp(0, 15).to(torch.uint8)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    groups = (mult | (zero << 4)).to(torch.uint8)
    scale_w = torch.exp(0.2 * _randn(g, n)) / (27.0 * math.sqrt(k))  # results of about unit size
    return codes_x, scale_x, packed, groups, scale_w


def prepare(case, seed):
    dtype = DTYPES[case["dtype"]]
    if case["kind"] in ("norm", "quantize"):
        x, residual, gains = _row_inputs(case, seed)
        state = State(case=case, x=x, residual=residual, gains=gains,
                      codes=torch.zeros(x.shape, device="cuda", dtype=torch.int8),
                      scales=torch.zeros(len(x), device="cuda"),
                      total=None if residual is None else torch.zeros_like(x))
    else:
        codes, scales, packed, groups, scale_w = _product_inputs(case, seed)
        state = State(case=case, codes=codes, scales=scales, packed=packed, groups=groups, scale_w=scale_w)
        # Rows of the result stand a multiple of eight elements apart, as the library takes them.
        state.y = torch.zeros(case["rows"], -(-case["n"] // 8) * 8, device="cuda", dtype=dtype)
    if own:
        state.ctx, state.dtype = _context(), _binding().BF16 if case["dtype"] == "bf16" else _binding().F16
        if case["kind"] in ("product", "swiglu"):
            image = _binding().w4_pack(packed.cpu().numpy(), groups.cpu().numpy(), scale_w.cpu().numpy())
            state.weights = torch.from_numpy(image).cuda()
    return state


# ---- a pass ---------------------------------------------------------------------------------


def run(state):
    case, kind = state.case, state.case["kind"]
    if not own:
        return {"norm": _plain_norm, "quantize": _plain_quantize, "product": _plain_product,
                "swiglu": _plain_swiglu}[kind](state)
    if kind == "norm":
        state.ctx.rmsnorm_q8(state.x.data_ptr(), state.gains.data_ptr(), state.codes.data_ptr(), state.scales.data_ptr(),
                             case["rows"], case["width"], eps=EPS, dtype=state.dtype,
                             **({} if state.residual is None else
                                {"residual_ptr": state.residual.data_ptr(), "sum_ptr": state.total.data_ptr()}))
        return [state.codes, state.scales, state.total]
    if kind == "quantize":
        state.ctx.quantize_q8(state.x.data_ptr(), state.codes.data_ptr(), state.scales.data_ptr(), case["rows"],
                              case["width"], dtype=state.dtype)
        return [state.codes, state.scales]
    call = state.ctx.w4_matmul if kind == "product" else state.ctx.w4_matmul_swiglu
    call(state.codes.data_ptr(), state.scales.data_ptr(), case["rows"], case["k"], state.weights.data_ptr(),
         state.weights.numel(), case["n"], state.y.data_ptr(), dtype=state.dtype, ldy=state.y.shape[1])
    return state.y[:, :case["n"]]


# ---- the plain forms ------------------------------------------------------------------------


def _codes(t):
    """(codes, largest value) of rows."""
    most = t.abs().amax(-1)
    full = torch.full_like(most, 127.0)
    factor = torch.where(most > 0, full / most, torch.zeros_like(most))
    return torch.round(t * factor[:, None]).to(torch.int8), most


def _plain_norm(state):
    v = state.x.float()
    total = None
    if state.residual is not None:
        v = v + state.residual.float()
        total = v.to(state.x.dtype)
    codes, most = _codes((v if total is None else total.float()) * state.gains)
    inverse = 1.0 / torch.sqrt((v * v).mean(-1) + EPS)
    return [codes, most / 127.0 * inverse, total]


def _plain_quantize(state):
    codes, most = _codes(state.x.float())
    return [codes, most / 127.0]


def _plain_weights(state):
    codes = torch.stack([state.packed & 15, state.packed >> 4], -1).flatten(-2)
    zero = (state.groups >> 4).float().repeat_interleave(GROUP, 1)
    mult = (state.groups & 15).float().repeat_interleave(GROUP, 1)
    return (codes.float() - zero) * mult * state.scale_w[:, None]


def _plain_rows(state):
    return (state.codes.float() * state.scales[:, None]) @ _plain_weights(state).T


def _plain_product(state):
    return _plain_rows(state).to(state.y.dtype)


def _plain_swiglu(state):
    gate, up = _plain_rows(state).split(state.case["n"], -1)
    return (gate / (1.0 + torch.exp(-gate)) * up).to(state.y.dtype)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    rows = case["rows"]
    if case["kind"] == "quantize":
        return {"bytes": rows * (3 * case["width"] + 4), "flops": 3 * rows * case["width"]}
    if case["kind"] == "norm":
        moved = 7 if case["residual"] else 3  # x, the residual, their sum, the codes
        return {"bytes": rows * (moved * case["width"] + 4) + 4 * case["width"], "flops": 7 * rows * case["width"]}
    k, n = case["k"], case["n"] * (2 if case["kind"] == "swiglu" else 1)
    weights = n * k // 2 + n * (k // GROUP) + 4 * n
    return {"bytes": weights + rows * (k + 4) + 2 * rows * case["n"], "flops": 2 * rows * n * k}


# ---- the same calls in 64 bits --------------------------------------------------------------


def _exact_rows(case, seed):
    x, residual, gains = _row_inputs(case, seed)
    total = x.double() if residual is None else x.double() + residual.double()
    # The stored sum: two 16-bit numbers add up exactly in 64 bits, and round to 16 once.
    stored = x if residual is None else total.to(x.dtype)
    weighted = stored.double() if gains is None else stored.double() * gains.double()
    scale = torch.linalg.vector_norm(weighted, ord=math.inf, dim=1) / 127
    if gains is None:
        return [None, scale]
    return [None, scale * torch.rsqrt(torch.linalg.vector_norm(total, dim=1).square() / case["width"] + EPS),
            None if residual is None else stored.double()]


def _exact_product(case, seed):
    codes, scale, packed, groups, scale_w = _product_inputs(case, seed)
    n, half = packed.shape
    nibble = torch.empty(n, 2 * half, dtype=torch.float64, device="cuda")
    nibble[:, 0::2], nibble[:, 1::2] = packed.remainder(16).double(), packed.div(16, rounding_mode="floor").double()
    byte = groups.double()[..., None]
    high = torch.floor(byte / 16)
    weight = ((nibble.view(n, -1, GROUP) - high) * (byte - 16 * high)).view(n, -1)
    y = torch.mm(codes.double(), weight.T.contiguous())
    y = y * scale.double()[:, None] * scale_w.double()
    if case["kind"] == "product":
        return y
    return y[:, :case["n"]] * torch.sigmoid(y[:, :case["n"]]) * y[:, case["n"]:]


def exact(case, seed):
    return (_exact_rows if case["kind"] in ("norm", "quantize") else _exact_product)(case, seed)
