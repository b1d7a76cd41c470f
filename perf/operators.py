"""Products with matrices in microscaled 4-bit floating point: what is timed and compared.

The format (blocks of 32 neighbouring values of a row share a power of two):

  E2M1, 4 bits, for matrices      0 0.5 1 1.5 2 3 4 6 and their negatives
  E2M3, 6 bits, for rows          0 to 2 in steps of 1/8, to 4 in steps of 1/4, to 7.5 in steps of 1/2, and their negatives

A block's power of two is the smallest 2^e (e from -127 on) with which its largest magnitude is at most 7 (E2M1, where 7 becomes 6: half
a step) or 7.5 (E2M3).  A value is the nearest of the list times 2^e, ties to the even code; a block that holds an infinity or a NaN is NaN.
A row's last block may be short.

  quantise   W' = the matrix W in E2M1, written and read back
  linear     out = X' W'^T + b            X' = the rows X in E2M3; sums in 32 bits, rounded once to the output's type
  swiglu     out = silu(X' G'^T) (X' U'^T)
  experts    out_t = sum over a token's choices (e, w) of w Y'_te D_e'^T,  Y_te = silu(X'_t G_e'^T) (X'_t U_e'^T) rounded to bfloat16,
             Y' = Y in E2M3

The stored form of a matrix `[rows][k]`: codes `[ceil(rows / 16)][ceil(k / 128)][64][16]` bytes, place 16 g + r of a tile holding row r's
values 32 g .. 32 g + 31 of the tile's 128, two to a byte, the lower one in the low half; powers of two `[ceil(rows / 16)][ceil(k / 512)][64][4]`,
place 16 g + r, byte s: row r's block 4 s + g of these 512 values, as e + 127 (255: NaN).  Gate and up matrices stand tile by tile in turn.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_E2M3 = tuple(i / 8 for i in range(16)) + tuple(2 + i / 4 for i in range(8)) + tuple(4 + i / 2 for i in range(8))


# ------------------------------------------------------------------ the cases
def _quantise(rows, k, dtype):
    return dict(op="quantise", rows=rows, k=k, dtype=dtype)


def _linear(m, n, k, dtype="bf16", out="fp32", bias=False):
    return dict(op="linear", m=m, n=n, k=k, dtype=dtype, out=out, bias=bias)


def _swiglu(m, f, k):
    return dict(op="swiglu", m=m, f=f, k=k, dtype="bf16")


def _experts(m, experts, top, f, k):
    return dict(op="experts", m=m, experts=experts, top=top, f=f, k=k, dtype="bf16")


def listed():
    return [
        # a matrix as it is loaded: the key product of the smallest model (two heads of 64), one of odd sizes in 32 bits, gate|up of the 7B one
        dict(_quantise(128, 896, "bf16"), name="quantise 128x896"),
        dict(_quantise(1000, 1111, "fp32"), name="quantise 1000x1111 fp32"),
        dict(_quantise(37888, 3584, "bf16"), name="quantise 37888x3584"),
        # one sequence decoding: attention's output product of the smallest model, where latency counts
        dict(_linear(1, 896, 896), name="linear 1x896x896"),
        # eight sequences decoding: the 7B model's down product, whose time is the matrix
        dict(_linear(8, 3584, 18944), name="linear 8x3584x18944"),
        # a short turn against a matrix of odd sizes
        dict(_linear(37, 1100, 2500, out="bf16", bias=True), name="linear 37x1100x2500"),
        # a prompt of some hundred tokens, rows in 32 bits
        dict(_linear(300, 2048, 2048, dtype="fp32"), name="linear 300x2048x2048 fp32"),
        # a prompt of 2,048 tokens: q|k|v of the 7B model with their biases
        dict(_linear(2048, 4608, 3584, bias=True), name="linear 2048x4608x3584"),
        # gate and up of the 7B model: eight sequences decoding, and a long prompt
        dict(_swiglu(8, 18944, 3584), name="swiglu 8x18944x3584"),
        dict(_swiglu(4096, 18944, 3584), name="swiglu 4096x18944x3584"),
        # routed experts while decoding: one sequence with four of 32 narrow ones, eight with two of eight wide ones
        dict(_experts(1, 32, 4, 1536, 2048), name="experts 1 token 4 of 32"),
        dict(_experts(8, 8, 2, 4096, 2048), name="experts 8 tokens 2 of 8"),
    ]


def _spread(rng, low, high, multiple=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(multiple, v // multiple * multiple)


def draw(rng):
    most = 4096 * 37888 * 3584                      # the largest listed product
    op = rng.choice(("quantise", "linear", "linear", "swiglu", "experts"))
    step = rng.choice((1, 1, 16, 128))              # odd sizes as often as those of models
    if op == "quantise":
        rows, k = _spread(rng, 64, 40000, step), _spread(rng, 128, 20000, step)
        return _quantise(min(rows, 37888 * 3584 // k), k, rng.choice(("bf16", "fp32")))
    if op == "experts":
        experts = rng.choice((4, 8, 16, 32, 64))
        f, k = _spread(rng, 256, 4096, step), _spread(rng, 256, 4096, step)
        return _experts(rng.randint(1, 16), experts, rng.randint(1, 4), max(64, min(f, (1 << 28) // (3 * experts * k))), k)
    m = rng.choice((_spread(rng, 1, 16), _spread(rng, 16, 64), _spread(rng, 64, 4096)))
    n, k = _spread(rng, 128, 40000, step), _spread(rng, 128, 20000, step)
    n = max(16, min(n, (37888 * 3584) // k, most // (m * k)))
    if op == "swiglu":
        return _swiglu(m, max(8, n // 2), k)
    return _linear(m, n, k, rng.choice(("bf16", "bf16", "fp32")), rng.choice(("fp32", "bf16")), rng.random() < 0.5)


def work(case):
    k, size = case["k"], {"bf16": 2, "fp32": 4}
    held = 0.5 + 1 / 32                             # bytes of a value in four bits, with its share of a power of two
    if case["op"] == "quantise":
        n = case["rows"] * k                        # read, stored, the stored form read, written
        return {"bytes": n * (size[case["dtype"]] + 2 * held + 2), "flops": 2 * n}
    m = case["m"]
    if case["op"] == "experts":
        f, e, top = case["f"], case["experts"], case["top"]
        chosen = e * (1 - (1 - top / e) ** m)       # experts that somebody has chosen, on the average
        return {"bytes": chosen * 3 * f * k * held + 2 * m * k * 2 + m * top * 8, "flops": 2 * m * top * 3 * f * k}
    n, out, bias = (2 * case["f"], case["f"] * 2, 0) if case["op"] == "swiglu" else (case["n"], case["n"] * size[case["out"]], case["bias"] * case["n"] * 4)
    return {"bytes": m * k * size[case["dtype"]] + n * k * held + m * out + bias, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the plain form
def _blocks(x):
    """x `[..., k]` as `[..., blocks, 32]`, zeros behind the end."""
    k = x.shape[-1]
    return torch.nn.functional.pad(x, (0, -k % 32)).unflatten(-1, (-1, 32))


def _power(e):
    """2^e exactly, for e from -126 to 127."""
    return ((e + 127) << 23).view(torch.float32)


def _steps(x, top):
    """The multiples (of a block's power of two) that the values of x become, and the exponents; `top`: the largest of the list, 6 or 7.5."""
    b = _blocks(x.float())
    amax = b.abs().amax(-1)
    bits = amax.view(torch.int32)
    e = ((bits + (0x1FFFFF if top == 6 else 0x0FFFFF)) >> 23) - 129       # (a carry where the mantissa is over 1.75, or 1.875)
    e = e.clamp(min=-127)
    # two factors: neither of them leaves the normal numbers
    half = e // 2
    v = b * _power(-half)[..., None] * _power(half - e)[..., None]
    a, finest = v.abs(), 0.5 if top == 6 else 0.125
    step = torch.where(a < 2, finest, torch.where(a < 4, 2 * finest, 4 * finest))
    v = torch.copysign((torch.round(a / step) * step).clamp(max=top), v)
    return torch.where(torch.isfinite(amax)[..., None], v, float("nan")), e


def _values(steps, e, k):
    """32-bit values of multiples and exponents, `[..., k]`."""
    half = e // 2
    return (steps * _power(half)[..., None] * _power(e - half)[..., None]).flatten(-2)[..., :k]


def _rows(x):
    return _values(*_steps(x, 7.5), x.shape[-1])


def _stored(w):
    """The stored form of the matrices `[..., rows, k]` and its powers of two, see above."""
    steps, e = _steps(w, 6)
    bad = torch.isnan(steps).any(-1)
    a = steps.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4))
    code = torch.where(bad[..., None], 0, code).to(torch.uint8) + torch.signbit(steps).to(torch.uint8) * 8
    code = code[..., 0::2] + code[..., 1::2] * 16
    e = torch.where(bad, 255, e + 127).to(torch.uint8)
    rows, blocks = e.shape[-2:]
    code = torch.nn.functional.pad(code, (0, 0, 0, -blocks % 4, 0, -rows % 16)).unflatten(-2, (-1, 4)).unflatten(-4, (-1, 16))
    codes = code.movedim(-4, -2).flatten(-3, -2).contiguous()             # [tile][128s][g][r] -> [tile][128s][64][16]
    e = torch.nn.functional.pad(e, (0, -blocks % 16, 0, -rows % 16)).unflatten(-1, (-1, 4, 4)).unflatten(-4, (-1, 16))
    scales = e.movedim(-4, -1).movedim(-3, -1).flatten(-3, -2).contiguous()     # [tile][512s][s][g][r] -> [tile][512s][g][r][s]
    return codes, scales


def _read(codes, scales, rows, k):
    """Multiples `[..., rows, blocks, 32]` and exponents (255 - 127: NaN) of the stored form."""
    byte = codes.unflatten(-2, (4, 16)).movedim(-2, -4).flatten(-3, -2).flatten(-4, -3)
    byte = byte[..., :rows, : -(-k // 32), :]
    code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
    e = scales.unflatten(-2, (4, 16)).movedim(-1, -3).movedim(-1, -4).flatten(-3, -1).flatten(-3, -2)
    return code, e[..., :rows, : -(-k // 32)].to(torch.int32) - 127


def _matrix(codes, scales, rows, k):
    code, e = _read(codes, scales, rows, k)
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float32, device=codes.device)
    steps = table[code.int()]
    return _values(torch.where((e == 128)[..., None], float("nan"), steps), e.clamp(max=127), k)


def _silu(z):
    return z / (1 + torch.exp(-z))


# ------------------------------------------------------------------ inputs
def _pairs(gate, up):
    return torch.stack([gate, up], dim=-4).flatten(-5, -4)                # tiles in turn


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, k = _TYPES[case["dtype"]], case["k"]

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    if case["op"] == "quantise":
        return dict(case=case, w=normal(case["rows"], k, std=0.02, dtype=dtype))
    # rows as a norm leaves them: some columns larger than the others
    x = (normal(case["m"], k) * (1 + normal(k, std=0.5).abs())).to(dtype)
    if case["op"] == "linear":
        codes, scales = _stored(normal(case["n"], k, std=0.02))
        return dict(case=case, x=x, codes=codes, scales=scales, bias=normal(case["n"], dtype=torch.float32) if case["bias"] else None)
    f = case["f"]
    if case["op"] == "swiglu":
        gate, up = _stored(normal(f, k, std=0.02)), _stored(normal(f, k, std=0.02))
        return dict(case=case, x=x, codes=_pairs(gate[0], up[0]), scales=_pairs(gate[1], up[1]))
    m, e, top = case["m"], case["experts"], case["top"]
    gate, up, down = (_stored(normal(e, *s, std=0.02)) for s in ((f, k), (f, k), (k, f)))
    chosen = torch.rand(m, e, generator=g, device="cuda").argsort(-1)[:, :top].to(torch.int32).contiguous()
    weights = torch.softmax(torch.randn(m, top, generator=g, device="cuda"), -1)
    return dict(case=case, x=x, gate_up=_pairs(gate[0], up[0]), gate_up_scales=_pairs(gate[1], up[1]), down=down[0], down_scales=down[1],
                chosen=chosen, weights=weights)


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    op, k = case["op"], case["k"]
    if own:
        from minfer_amd.kernels import ops
        if op == "quantise":
            w = state["w"]
            codes, scales = (torch.empty(s, dtype=torch.uint8, device=w.device) for s in ops.mx4_shapes(*w.shape))
            ops.mx4_quantise(w, codes, scales)
            out = torch.empty(w.shape, dtype=torch.bfloat16, device=w.device)
            ops.mx4_dequantise(codes, scales, out)
            return out
        x = state["x"]
        if op == "linear":
            out = torch.empty((case["m"], case["n"]), dtype=_TYPES[case["out"]], device=x.device)
            ops.mx4_linear(x, state["codes"], state["scales"], state["bias"], out)
        elif op == "swiglu":
            out = torch.empty((case["m"], case["f"]), dtype=torch.bfloat16, device=x.device)
            ops.mx4_linear_swiglu(x, state["codes"], state["scales"], out)
        else:
            out = torch.empty((case["m"], k), dtype=torch.bfloat16, device=x.device)
            ops.mx4_moe_sparse(x, state["gate_up"], state["gate_up_scales"], state["down"], state["down_scales"], state["chosen"],
                               state["weights"], out, case["f"], act=ops.MOE_ACTS["silu"], accumulate=False)
        return out
    if op == "quantise":
        return _values(*_steps(state["w"], 6), k).to(torch.bfloat16)
    x = _rows(state["x"])
    if op == "linear":
        out = x @ _matrix(state["codes"], state["scales"], case["n"], k).T
        return (out if state["bias"] is None else out + state["bias"]).to(_TYPES[case["out"]])
    f = case["f"]
    if op == "swiglu":
        gate, up = (_matrix(state["codes"][i::2], state["scales"][i::2], f, k) for i in (0, 1))
        return (_silu(x @ gate.T) * (x @ up.T)).to(torch.bfloat16)
    chosen, weights = state["chosen"].long(), state["weights"]
    m, e = case["m"], case["experts"]
    gate, up = (_matrix(state["gate_up"][:, i::2], state["gate_up_scales"][:, i::2], f, k).flatten(0, 1) for i in (0, 1))
    y = (_silu(x @ gate.T) * (x @ up.T)).to(torch.bfloat16).view(m, e, f)              # of every expert
    share = torch.zeros(m, e, device=x.device).scatter_add_(1, chosen, weights)        # 0 where it was not chosen
    z = torch.bmm(_rows(y).transpose(0, 1), _matrix(state["down"], state["down_scales"], k, f).transpose(1, 2).contiguous())
    return (z * share.T[..., None]).sum(0).to(torch.bfloat16)


# ------------------------------------------------------------------ in 64 bits
def _power_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(x, levels, full):
    """x `[..., k]` in 64 bits, block by block: the nearest level times the block's power of two; `full`: the most that a block's largest may be."""
    k = x.shape[-1]
    b = torch.nn.functional.pad(x.double(), (0, -k % 32)).unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(amax)                                # amax = mantissa 2^exponent, mantissa from 1/2 to 1
    e = exponent - 3 + (mantissa * 8 > full).to(exponent.dtype)
    unit = _power_64(e.clamp(min=-127))
    v = b / unit
    levels = torch.tensor(levels, dtype=torch.float64, device=x.device)
    middle = (levels[1:] + levels[:-1]) / 2
    at = torch.bucketize(v.abs(), middle)                                 # (on a middle: the lower one)
    tie = (at < len(middle)) & (v.abs() == middle[at.clamp(max=len(middle) - 1)])
    at = at + (tie & (at % 2 == 1)).to(at.dtype)
    return (levels[at] * torch.sign(v) * unit).flatten(-2)[..., :k]


def exact(case, seed):
    state, op, k = prepare(case, seed), case["op"], case["k"]
    if op == "quantise":
        return _nearest(state["w"], _E2M1, 7.0)

    def matrix(codes, scales, rows, k):
        code, e = _read(codes, scales, rows, k)
        magnitude = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)[(code & 7).int()]
        sign = 1.0 - 2.0 * (code >> 3).double()
        return (magnitude * sign * _power_64(e)[..., None]).flatten(-2)[..., :k]

    x = _nearest(state["x"], _E2M3, 7.5)
    if op == "linear":
        out = x @ matrix(state["codes"], state["scales"], case["n"], k).T
        return out if state["bias"] is None else out + state["bias"].double()
    f = case["f"]
    if op == "swiglu":
        gate = x @ matrix(state["codes"][0::2].contiguous(), state["scales"][0::2].contiguous(), f, k).T
        return gate * torch.sigmoid(gate) * (x @ matrix(state["codes"][1::2].contiguous(), state["scales"][1::2].contiguous(), f, k).T)
    out = torch.zeros(case["m"], k, dtype=torch.float64, device=x.device)
    for t, row in enumerate(state["chosen"].tolist()):
        for j, e in enumerate(row):
            gate = matrix(state["gate_up"][e, 0::2].contiguous(), state["gate_up_scales"][e, 0::2].contiguous(), f, k) @ x[t]
            up = matrix(state["gate_up"][e, 1::2].contiguous(), state["gate_up_scales"][e, 1::2].contiguous(), f, k) @ x[t]
            y = _nearest((gate * torch.sigmoid(gate) * up).to(torch.bfloat16), _E2M3, 7.5)
            out[t] += state["weights"][t, j].double() * (matrix(state["down"][e], state["down_scales"][e], k, f) @ y)
    return out
