"""Cases of the block-scaled FP8 operators: what they compute and what it has to move.

A pre-norm transformer block with 8-bit linears runs four kinds of step:

  norm      h = x + r, y = h * rsqrt(mean(h^2) + eps) * w, y held in 8 bits
  quantize  y = x held in 8 bits
  mm        out = A . W^T + bias (+ residual), A and W held in 8 bits
  swiglu    y = silu(A . Wg^T + bg) * (A . Wu^T + bu) held in 8 bits

"Held in 8 bits" is E4M3 codes with one power-of-two scale (an E8M0 byte e,
2^(e-127)) for each row's blocks of 128 columns: the smallest exponent e >= 1
with amax <= 448 * 2^(e-127). Weights have one scale for each 128 x 128 block,
stored for each row as the activations' are. Scale bytes lie in atoms of 128
rows x 4 blocks (row 32 i + j, block k at byte 16 j + 4 i + k), zero where the
matrix has none. A gate | up weight alternates 128 gate and 128 up rows.

run() computes in plain torch operations in 32 bits, or (own) calls the library.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MOST_PRODUCT = 7040 * 3072 * 14336      # multiply-adds of the largest listed product
MOST_VALUES = 7040 * 14336              # values of the largest listed quantization


def _norm(name, m, n, dtype, residual):
    return {"name": name, "op": "norm", "m": m, "n": n, "dtype": dtype, "residual": residual}


def _quantize(name, m, n, dtype):
    return {"name": name, "op": "quantize", "m": m, "n": n, "dtype": dtype}


def _mm(name, m, n, k, bias, residual, dtype="bf16"):
    return {"name": name, "op": "mm", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "residual": residual}


def _swiglu(name, m, h, k):
    return {"name": name, "op": "swiglu", "m": m, "h": h, "k": k}


def listed():
    return [
        # one token through the decoder's width: the latency of the smallest call
        _norm("norm token 1x512", 1, 512, "bf16", True),
        # one latent frame of the decoder at 704x1280 after its four-fold temporal expansion is 44 x 80 tokens
        _norm("norm frame 3520x512", 3520, 512, "bf16", True),
        # a long batch of rows with an fp32 residual stream, its row count not a multiple of the tile
        _norm("norm rows 14081x2048 fp32", 14081, 2048, "fp32", True),
        # the attention output of a refinement step, ready for its output projection
        _quantize("quantize frames 14080x512", 14080, 512, "bf16"),
        # hidden activations of the wide feed-forward layer over four body blocks
        _quantize("quantize wide 7040x14336", 7040, 14336, "bf16"),
        # a conditioning vector through one linear of the DiT's width: one row, bound by the weight's bytes
        _mm("mm token 1x3072x3072", 1, 3072, 3072, True, False),
        # a few rows through the long down projection: the weight is read once, K is long
        _mm("mm few 24x3072x14336", 24, 3072, 14336, True, False),
        # query | key | value of one latent frame of the decoder: short K
        _mm("mm frame 3520x768x512", 3520, 768, 512, True, False),
        # an output projection of one body block less a token, added to the residual stream
        _mm("mm block 1759x3072x3072", 1759, 3072, 3072, True, True),
        # the down projection over four body blocks: the largest product
        _mm("mm large 7040x3072x14336", 7040, 3072, 14336, True, True),
        # gate and up of a handful of rows in the decoder
        _swiglu("swiglu few 16x2048x512", 16, 2048, 512),
        # gate and up of a refinement step of the decoder: four frames of 3520 tokens
        _swiglu("swiglu frames 14080x2048x512", 14080, 2048, 512),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _log_16(rng, low, high):
    return 16 * _log_int(rng, low // 16, high // 16)


def draw(rng):
    op = rng.choice(("norm", "quantize", "mm", "mm", "swiglu"))
    m = _log_int(rng, 1, 14081)
    if op == "norm":
        n = _log_16(rng, 64, 8192)
        m = max(1, min(m, MOST_VALUES // (3 * n)))
        return {"op": op, "m": m, "n": n, "dtype": rng.choice(("bf16", "fp16", "fp32")), "residual": rng.random() < 0.7}
    if op == "quantize":
        n = _log_16(rng, 64, 14336)
        m = max(1, min(m, MOST_VALUES // (2 * n)))
        return {"op": op, "m": m, "n": n, "dtype": rng.choice(("bf16", "fp16", "fp32"))}
    if op == "mm":
        n, k = _log_int(rng, 48, 14336), _log_16(rng, 64, 14336)
        m = max(1, min(m, MOST_PRODUCT // (n * k)))
        return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(("bf16", "bf16", "fp16")),
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.4}
    h, k = _log_16(rng, 128, 8192), _log_16(rng, 64, 4096)
    m = max(1, min(m, MOST_PRODUCT // (4 * h * k)))
    return {"op": op, "m": m, "h": h, "k": k}


# ------------------------------------------------------------------ layouts
def _ceil(a, b):
    return -(-a // b)


def _lay_out(scale_bytes):
    """[rows, blocks] scale bytes -> the flat atoms, zeros where there are none."""
    rows, kb = scale_bytes.shape
    full = torch.zeros(_ceil(rows, 128) * 128, _ceil(kb, 4) * 4, dtype=torch.uint8, device=scale_bytes.device)
    full[:rows, :kb] = scale_bytes
    return full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _taken_out(flat, rows, kb):
    """The [rows, blocks] scale bytes of flat atoms."""
    mb, kt = _ceil(rows, 128), _ceil(kb, 4)
    return flat.view(mb, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(mb * 128, kt * 4)[:rows, :kb]


def _padded(y, multiple, dim):
    short = -y.shape[dim] % multiple
    if not short:
        return y
    size = list(y.shape)
    size[dim] = short
    return torch.cat([y, torch.zeros(size, dtype=y.dtype, device=y.device)], dim)


def _scale_bytes(amax):
    """amax (fp32) -> the smallest byte e >= 1 with amax <= 448 * 2^(e - 127), 255 where it is not finite."""
    bits = amax.view(torch.int32)
    e = ((bits + 0x1FFFFF) >> 23) - 8
    return torch.where(bits >= 0x7F800000, 255, e.clamp(min=1)).to(torch.uint8)


def _power(scale_bytes):
    """2^(e - 127) of scale bytes, in 32 bits."""
    return torch.exp2(scale_bytes.to(torch.float32) - 127.0)


def _plain_quantize(y):
    """fp32 [rows, cols] -> (E4M3 codes [rows, cols], scale bytes [rows, blocks])."""
    rows, cols = y.shape
    blocks = _padded(y, 128, 1).view(rows, -1, 128)
    e = _scale_bytes(blocks.abs().amax(-1))
    codes = (blocks * torch.exp2(127.0 - e.to(torch.float32))[..., None]).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).reshape(rows, -1)[:, :cols].contiguous().view(torch.float8_e4m3fn), e


def _plain_weight(w):
    """fp32 [N, K] -> (E4M3 codes, scale bytes [N, blocks]) with one scale for each 128 x 128 block."""
    n, k = w.shape
    p = _padded(_padded(w, 128, 0), 128, 1)
    blocks = p.view(p.shape[0] // 128, 128, p.shape[1] // 128, 128)
    e = _scale_bytes(blocks.abs().amax((1, 3)))
    codes = (blocks * torch.exp2(127.0 - e.to(torch.float32))[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.view(torch.uint8).reshape(p.shape)[:n, :k].contiguous().view(torch.float8_e4m3fn)
    return codes, e.repeat_interleave(128, 0)[:n].contiguous()


def _values(codes, flat):
    """The values that codes and laid-out scale bytes stand for, in 32 bits."""
    rows, cols = codes.shape
    s = _power(_taken_out(flat, rows, _ceil(cols, 128)))
    return codes.to(torch.float32) * s.repeat_interleave(128, 1)[:, :cols]


# ------------------------------------------------------------------ inputs
def _rows(g, m, n, device):
    """Activations as a residual network has them: a magnitude of its own for
    each row, a few channels far above the others."""
    x = torch.randn(m, n, generator=g, device=device)
    channel = torch.exp(0.5 * torch.randn(n, generator=g, device=device))
    channel = torch.where(torch.rand(n, generator=g, device=device) < 0.01, channel * 12.0, channel)
    return x * channel * torch.exp(0.3 * torch.randn(m, 1, generator=g, device=device))


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    op, m = case["op"], case["m"]
    state = {"op": op}
    if op in ("norm", "quantize"):
        dtype = DTYPES[case["dtype"]]
        state["x"] = _rows(g, m, case["n"], device).to(dtype)
        if op == "norm":
            state["w"] = 1 + 0.1 * torch.randn(case["n"], generator=g, device=device)
            state["r"] = _rows(g, m, case["n"], device).to(dtype) if case["residual"] else None
        return state
    k = case["k"]
    codes, e = _plain_quantize(_rows(g, m, k, device))
    state["a"], state["sa"] = codes, _lay_out(e)
    if op == "mm":
        n = case["n"]
        codes, e = _plain_weight(torch.randn(n, k, generator=g, device=device) / k ** 0.5)
        state["b"], state["sb"] = codes, _lay_out(e)
        dtype = state["dtype"] = DTYPES[case["dtype"]]
        state["bias"] = 0.1 * torch.randn(n, generator=g, device=device) if case["bias"] else None
        state["r"] = _rows(g, m, n, device).to(dtype) if case["residual"] else None
        return state
    h, hp = case["h"], _ceil(case["h"], 128) * 128
    gate_up = torch.randn(2, h, k, generator=g, device=device) / k ** 0.5
    bias = 0.1 * torch.randn(2, h, generator=g, device=device)
    gate_up, bias = _padded(gate_up, 128, 1), _padded(bias, 128, 1)
    rows = gate_up.view(2, hp // 128, 128, k).permute(1, 0, 2, 3).reshape(2 * hp, k)
    codes, e = _plain_weight(rows)
    state["b"], state["sb"] = codes, _lay_out(e)
    state["bias"] = bias.view(2, hp // 128, 128).permute(1, 0, 2).reshape(-1).contiguous()
    state["h"] = h
    return state


# ------------------------------------------------------------------ one pass
def _run_own(s):
    from recavsr_b200.runtime import fp8_block

    if s["op"] == "norm":
        codes, scales, hidden = fp8_block.rms_norm_quantize(s["x"], s["w"], EPS, residual=s["r"])
    elif s["op"] == "quantize":
        (codes, scales), hidden = fp8_block.quantize(s["x"]), None
    elif s["op"] == "mm":
        return {"out": fp8_block.mm(s["a"], s["b"], s["sa"], s["sb"], s["bias"], residual=s["r"], dtype=s["dtype"])}
    else:
        (codes, scales), hidden = fp8_block.swiglu_mm(s["a"], s["b"], s["sa"], s["sb"], s["bias"], features=s["h"]), None
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu), "hidden": hidden}


def run(state):
    s = state
    if own:
        return _run_own(s)
    hidden = None
    if s["op"] == "norm":
        y = s["x"].to(torch.float32)
        if s["r"] is not None:
            y = y + s["r"].to(torch.float32)
            hidden = y.to(s["x"].dtype)
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["w"]
    elif s["op"] == "quantize":
        y = s["x"].to(torch.float32)
    else:
        y = _values(s["a"], s["sa"]) @ _values(s["b"], s["sb"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["op"] == "mm":
            if s["r"] is not None:
                y = y + s["r"].to(torch.float32)
            return {"out": y.to(s["dtype"])}
        y = y.view(y.shape[0], -1, 2, 128)
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1 + torch.exp(-gate)) * up).reshape(y.shape[0], -1)[:, :s["h"]]
    codes, e = _plain_quantize(y)
    return {"codes": codes, "scales": _lay_out(e).view(torch.float8_e8m0fnu), "hidden": hidden}


def work(case):
    """Every input read once and every output written once; the products'
    multiply-adds, and for the others a few operations for each value."""
    op, m = case["op"], case["m"]
    if op in ("norm", "quantize"):
        n, size = case["n"], torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
        moved = m * n * (size + 1) + m * _ceil(n, 128)
        if op == "norm":
            moved += 4 * n + (2 * m * n * size if case["residual"] else 0)
        return {"bytes": moved, "flops": (8 if op == "norm" else 3) * m * n}
    k = case["k"]
    if op == "mm":
        n = case["n"]
        moved = (m + n) * k + (m + n) * _ceil(k, 128) + 2 * m * n * (2 if case["residual"] else 1)
        return {"bytes": moved + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    h = case["h"]
    moved = (m + 2 * h) * k + (m + 2 * h) * _ceil(k, 128) + m * h + m * _ceil(h, 128) + 8 * h
    return {"bytes": moved, "flops": 4 * m * h * k}


# ------------------------------------------------------------------ in 64 bits
def _exact_codes(y):
    """The definition in 64 bits: codes' values and scale bytes of y [rows, cols]."""
    rows, cols = y.shape
    kb = _ceil(cols, 128)
    p = torch.zeros(rows, kb * 128, dtype=torch.float64, device=y.device)
    p[:, :cols] = y
    p = p.view(rows, kb, 128)
    amax = p.abs().amax(-1)
    mantissa, exponent = torch.frexp(amax / 448.0)          # amax = 448 * mantissa * 2^exponent, mantissa in [0.5, 1)
    e = torch.where(mantissa == 0.5, exponent - 1, exponent)
    e = torch.where(amax == 0, torch.full_like(e, -126), e).clamp(min=-126)
    v = torch.ldexp(p, -e[..., None])
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 4).clamp(min=-9))    # E4M3: four significant bits
    codes = (torch.round(v / step) * step).view(rows, -1)[:, :cols]
    flat = torch.zeros(_ceil(rows, 128) * 128 * _ceil(kb, 4) * 4, dtype=torch.float64, device=y.device) + 2.0 ** -127
    row = torch.arange(rows, device=y.device)[:, None]
    block = torch.arange(kb, device=y.device)[None, :]
    at = ((row // 128) * _ceil(kb, 4) + block // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + block % 4
    flat[at] = torch.ldexp(torch.ones_like(amax), e)
    return codes.to(torch.float8_e4m3fn), flat.to(torch.float32)


def _exact_operand(codes, flat):
    rows, cols = codes.shape
    row = torch.arange(rows, device=codes.device)[:, None]
    block = torch.arange(_ceil(cols, 128), device=codes.device)[None, :]
    at = ((row // 128) * _ceil(_ceil(cols, 128), 4) + block // 4) * 512 + (row % 32) * 16 + (row % 128 // 32) * 4 + block % 4
    power = torch.ldexp(torch.ones(at.shape, dtype=torch.float64, device=codes.device), flat[at].to(torch.int32) - 127)
    return codes.to(torch.float64) * power[:, torch.arange(cols, device=codes.device) // 128]


def exact(case, seed):
    s = prepare(case, seed)
    hidden = None
    if s["op"] == "norm":
        y = s["x"].double()
        if s["r"] is not None:
            y = y + s["r"].double()
            hidden = y
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * s["w"].double()
    elif s["op"] == "quantize":
        y = s["x"].double()
    else:
        y = _exact_operand(s["a"], s["sa"]) @ _exact_operand(s["b"], s["sb"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if s["op"] == "mm":
            return {"out": y if s["r"] is None else y + s["r"].double()}
        cols = torch.arange(s["h"], device=y.device)
        gate, up = y[:, cols // 128 * 256 + cols % 128], y[:, cols // 128 * 256 + 128 + cols % 128]
        y = gate * torch.sigmoid(gate) * up
    codes, scales = _exact_codes(y)
    return {"codes": codes, "scales": scales, "hidden": hidden}
