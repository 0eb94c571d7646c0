"""Channels-last GroupNorm and microscaled 4-bit floating point: the operators' cases, plain forms and 64-bit values.

``own`` chooses the side: False runs the plain torch forms below (32-bit arithmetic, 64 next to rounding borders), True
makes the calls of ``vrhino_b200.ops`` that a user's program makes.  Both take the same state.

Formats.  e2m1 elements (0, .5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte with the even k in the low nibble, rows
padded to 32 elements.  "nvfp4": blocks of 16 with an e4m3 scale and one F32 scale per tensor; "mxfp4": blocks of 32
with a power-of-two scale (e8m0).  Scales lie in tiles of 128 rows x 4 blocks, 512 bytes each:
byte (row % 32) * 16 + (row % 128) // 32 * 4 + block % 4 of tile (row // 128, block // 4).
"""
import math

import torch

own = False

_BLOCK = {"nvfp4": 16, "mxfp4": 32}
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------ cases --
def _gn(name, batch, spatial, channels, groups, activation, dtype):
    return {"name": name, "op": "group_norm", "batch": batch, "spatial": spatial, "channels": channels, "groups": groups,
            "activation": activation, "dtype": dtype}


def _trip(name, format, rows, k, dtype):
    return {"name": name, "op": "round_trip", "format": format, "rows": rows, "k": k, "dtype": dtype}


def _linear(name, format, m, k, n, activation):
    return {"name": name, "op": "linear", "format": format, "m": m, "k": k, "n": n, "activation": activation}


def _product(name, format, m, k, n, out):
    return {"name": name, "op": "product", "format": format, "m": m, "k": k, "n": n, "out": out}


def listed():
    return [
        # the middle block of an image VAE, 16 x 16 positions: latency
        _gn("gn_mid_block", 1, 256, 512, 32, "silu", "bf16"),
        # a video decoder's first stage, 4 frames of 60 x 104
        _gn("gn_video_stage", 1, 24960, 512, 32, "silu", "bf16"),
        # the last stage of a video decoder, 28 frames of 240 x 424
        _gn("gn_decoder_stage", 1, 2849280, 256, 32, "silu", "bf16"),
        # a UNet's transformer input (no activation follows): 10 channels to a group, odd extent, F32
        _gn("gn_unet_f32", 3, 1035, 320, 32, "none", "f32"),
        # a feed-forward weight brought to 4 bits and read back, with its tensor scale
        _trip("trip_weight_nv", "nvfp4", 13824, 5120, "bf16"),
        # a small activation of odd width in F32
        _trip("trip_odd_mx", "mxfp4", 333, 1000, "f32"),
        # the timestep's modulation projection, both guidance branches: two rows through a 4-bit weight
        _linear("linear_two_rows", "nvfp4", 2, 1536, 9216, "none"),
        # the text embedding's first linear, 512 tokens
        _linear("linear_text", "mxfp4", 512, 4096, 1536, "gelu_tanh"),
        # a video DiT's feed-forward, up: 32760 tokens
        _linear("linear_ffn_up", "nvfp4", 32760, 1536, 8960, "gelu_tanh"),
        # and down, from operands already in 4 bits, into the F32 accumulation that an epilogue reads
        _product("product_ffn_down", "nvfp4", 32760, 8960, 1536, "f32"),
        # nothing a multiple of a tile
        _product("product_odd", "mxfp4", 1001, 1000, 1003, "bf16"),
        # the feed-forward of a 14-billion-parameter DiT
        _product("product_large", "nvfp4", 32760, 5120, 13824, "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["group_norm", "group_norm", "round_trip", "linear", "product"])
    if op == "group_norm":
        groups = rng.choice([1, 8, 16, 32])
        channels = groups * rng.choice([1, 2, 3, 4, 6, 8, 10, 12, 16, 20, 32])
        batch = rng.choice([1, 1, 2, 3, 4])
        spatial = _log(rng, 1, 300_000_000 // (channels * batch))
        return {"op": op, "batch": batch, "spatial": spatial, "channels": channels, "groups": groups,
                "activation": rng.choice(["none", "silu", "gelu_tanh"]), "dtype": rng.choice(["bf16", "f32"])}
    format = rng.choice(["nvfp4", "mxfp4"])
    if op == "round_trip":
        k = _log(rng, 1, 16384)
        return {"op": op, "format": format, "rows": _log(rng, 1, 70_000_000 // k), "k": k, "dtype": rng.choice(["bf16", "f32"])}
    m = rng.choice([_log(rng, 1, 64), _log(rng, 1, 32768)])
    k, n = _log(rng, 16, 8192), _log(rng, 8, 8192)
    if rng.random() < 0.5:  # model widths are round more often than not
        k, n = -(-k // 64) * 64, -(-n // 64) * 64
    if op == "linear":
        return {"op": op, "format": format, "m": m, "k": k, "n": n, "activation": rng.choice(["none", "silu", "gelu_tanh"])}
    return {"op": op, "format": format, "m": m, "k": k, "n": n, "out": rng.choice(["bf16", "f32"])}


# ----------------------------------------------------------------------------------------- inputs --
def _normal(generator, *shape):
    return torch.randn(shape, device="cuda", generator=generator)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "group_norm":
        dtype, c = _DTYPES[case["dtype"]], case["channels"]
        # feature maps: every channel with an offset and a spread of its own
        x = _normal(g, case["batch"], case["spatial"], c)
        x.mul_(1.0 + 0.5 * torch.rand((c,), device="cuda", generator=g)).add_(0.5 * _normal(g, c))
        return {"case": case, "x": x.to(dtype), "weight": 1.0 + 0.1 * _normal(g, c), "bias": 0.1 * _normal(g, c)}
    format = case["format"]
    if case["op"] == "round_trip":
        x = _normal(g, case["rows"], case["k"]) * 0.02
        return {"case": case, "x": x.to(_DTYPES[case["dtype"]])}
    m, k, n = case["m"], case["k"], case["n"]
    state = {"case": case, "w": _pack(_normal(g, n, k) * 0.02, format, None)}
    # activations: a few channels are much larger than the rest
    x = _normal(g, m, k) * (1.0 + 7.0 * (torch.rand((k,), device="cuda", generator=g) < 0.02))
    if case["op"] == "linear":
        state["x"] = x.to(torch.bfloat16)
        # the activation's tensor scale is calibrated beforehand, as serving programs keep it
        state["x_scale"] = _tensor_scale(state["x"]) if format == "nvfp4" else None
        state["bias"] = (0.1 * _normal(g, n)).to(torch.bfloat16)
    else:
        state["x"] = _pack(x, format, None)
    return state


# ------------------------------------------------------------------------------------ plain forms --
def _tensor_scale(x):
    # divided in 64 bits: the nearest F32, where a 32-bit product with 1 / 2688 would miss it
    return (x.abs().amax().double() / 2688.0).float().reshape(1)


def _e2m1(v):
    """The e2m1 code of every value of v (64-bit), ties to the even code, saturating."""
    a = v.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).to(v.dtype)
    a = torch.round(a / step) * step  # rounds half to even: the even multiple has the even code
    code = torch.where(a <= 2.0, a * 2.0, torch.where(a <= 4.0, a + 2.0, torch.full_like(a, 7.0)))
    return code.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)


def _scales_and_codes(x, format, tensor_scale):
    """x [rows, k] -> scale values [rows, blocks] and scale bytes, codes [rows, blocks, block], in 64 bits."""
    rows, k = x.shape
    block = _BLOCK[format]
    blocks = -(-k // block)
    x = torch.nn.functional.pad(x.double(), (0, blocks * block - k)).view(rows, blocks, block)
    amax = x.abs().amax(dim=2)
    if format == "nvfp4":
        q = torch.where(amax > 0, amax / (6.0 * tensor_scale.double()), torch.zeros_like(amax)).clamp(max=448.0)
        exponent = torch.floor(torch.log2(q.clamp(min=2.0 ** -6)))
        exponent = exponent - (torch.exp2(exponent) > q.clamp(min=2.0 ** -6)).double()
        step = torch.exp2(exponent - 3.0)
        s = torch.round(q / step) * step
        bytes_ = s.to(torch.float8_e4m3fn).view(torch.uint8)
        scale = s * tensor_scale.double()
    else:
        exponent = (torch.frexp(amax).exponent - 3).clamp(min=-127)
        exponent = torch.where(amax > 0, exponent, torch.full_like(exponent, -127))
        bytes_ = (exponent + 127).to(torch.uint8)
        scale = torch.exp2(exponent.double())
    codes = _e2m1(torch.where(scale[:, :, None] > 0, x / scale[:, :, None], torch.zeros_like(x)))
    return bytes_, codes


def _pack(x, format, tensor_scale):
    """(codes, scale tiles, tensor scale) of x [rows, k], rows a slab at a time so that the 64-bit temporaries stay small."""
    if format == "nvfp4" and tensor_scale is None:
        tensor_scale = _tensor_scale(x)
    rows, k = x.shape
    slab = max(1, (1 << 26) // k)
    parts = [_scales_and_codes(x[i:i + slab], format, tensor_scale) for i in range(0, rows, slab)]
    bytes_, codes = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    codes = torch.nn.functional.pad(codes.view(rows, -1), (0, -codes[0].numel() % 32))
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    row_tiles, block_tiles = -(-rows // 128), -(-bytes_.shape[1] // 4)
    padded = torch.nn.functional.pad(bytes_, (0, block_tiles * 4 - bytes_.shape[1], 0, row_tiles * 128 - rows))
    tiles = padded.view(row_tiles, 4, 32, block_tiles, 4).permute(0, 3, 2, 1, 4).contiguous()
    return packed.contiguous(), tiles.view(-1), tensor_scale


def _unpack(operand, format, rows, k):
    """The values of a packed operand, [rows, k] in 32 bits."""
    packed, tiles, tensor_scale = operand
    block = _BLOCK[format]
    blocks = -(-k // block)
    row_tiles, block_tiles = -(-rows // 128), -(-blocks // 4)
    bytes_ = tiles.view(row_tiles, block_tiles, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(row_tiles * 128, block_tiles * 4)[:rows, :blocks]
    codes = torch.stack((packed & 15, packed >> 4), dim=2).view(rows, -1)[:, :k]
    magnitude = (codes & 7).float()
    value = torch.where(magnitude <= 4.0, magnitude * 0.5, torch.where(magnitude < 7.0, magnitude - 2.0, torch.full_like(magnitude, 6.0)))
    value = torch.where(codes >= 8, -value, value)
    if format == "nvfp4":
        s = bytes_.contiguous().view(torch.float8_e4m3fn).float()
    else:
        s = torch.exp2(bytes_.float() - 127.0)
    value = value * s.repeat_interleave(block, dim=1)[:, :k]
    return value if tensor_scale is None else value * tensor_scale


def _activate(y, activation):
    if activation == "silu":
        return y / (1.0 + torch.exp(-y))
    if activation == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain(state):
    case = state["case"]
    if case["op"] == "group_norm":
        x = state["x"]
        b, s, c = x.shape
        v = x.float().view(b, s, case["groups"], c // case["groups"])
        mean = v.mean(dim=(1, 3), keepdim=True)
        d = v - mean
        inverse = 1.0 / torch.sqrt((d * d).mean(dim=(1, 3), keepdim=True) + 1e-6)
        y = (d * inverse).view(b, s, c) * state["weight"] + state["bias"]
        return _activate(y, case["activation"]).to(x.dtype)
    format = case["format"]
    if case["op"] == "round_trip":
        x = state["x"]
        return _unpack(_pack(x, format, None), format, *x.shape).to(x.dtype)
    m, k, n = case["m"], case["k"], case["n"]
    w = _unpack(state["w"], format, n, k)
    if case["op"] == "product":
        return (_unpack(state["x"], format, m, k) @ w.t()).to(_DTYPES[case["out"]])
    x = _unpack(_pack(state["x"], format, state["x_scale"]), format, m, k)
    return _activate(x @ w.t() + state["bias"].float(), case["activation"]).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------- runs --
_backend = None


def _own(state):
    global _backend
    from vrhino_b200 import ops
    if _backend is None:
        _backend = ops.B200Backend()
    be, case = _backend, state["case"]
    kinds = {"none": None, "silu": ops.SILU, "gelu_tanh": ops.GELU_TANH}
    if case["op"] == "group_norm":
        return be.group_norm_channels_last(state["x"], case["groups"], state["weight"], state["bias"], 1e-6,
                                           activation=kinds[case["activation"]])
    format = {"nvfp4": ops.NVFP4, "mxfp4": ops.MXFP4}[case["format"]]
    if case["op"] == "round_trip":
        x = state["x"]
        scale = be.fp4_tensor_scale(x) if format == ops.NVFP4 else None
        return be.fp4_dequantize(be.fp4_quantize(x, format, scale), x.dtype)
    w = ops.Fp4Tensor(*state["w"], format, (case["n"], case["k"]))
    if case["op"] == "product":
        return be.fp4_linear(ops.Fp4Tensor(*state["x"], format, (case["m"], case["k"])), w, dtype=_DTYPES[case["out"]])
    x = be.fp4_quantize(state["x"], format, state["x_scale"])
    return be.fp4_linear(x, w, state["bias"], kinds[case["activation"]])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    if case["op"] == "group_norm":
        elements = case["batch"] * case["spatial"] * case["channels"]
        return {"bytes": 2 * elements * (2 if case["dtype"] == "bf16" else 4) + 8 * case["channels"], "flops": 8 * elements}
    if case["op"] == "round_trip":
        elements = case["rows"] * case["k"]
        return {"bytes": 2 * elements * (2 if case["dtype"] == "bf16" else 4), "flops": 4 * elements}
    m, k, n = case["m"], case["k"], case["n"]
    packed = 0.5 + 1.0 / _BLOCK[case["format"]]
    if case["op"] == "linear":
        return {"bytes": int(2 * m * k + n * k * packed + 2 * n + 2 * m * n), "flops": 2 * m * n * k}
    return {"bytes": int((m + n) * k * packed + m * n * (2 if case["out"] == "bf16" else 4)), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------- values in 64 bits --
_E2M1_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# non-negative finite e4m3 values in code order
_E4M3_VALUES = tuple(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8))[:127]


def _nearest(v, grid):
    """The index of the grid value nearest to every v >= 0: counts the midpoints below v; on a midpoint the even index."""
    grid = torch.tensor(grid, dtype=torch.float64, device=v.device)
    middle = (grid[1:] + grid[:-1]) / 2
    low = torch.searchsorted(middle, v.contiguous(), right=False)  # midpoints < v
    high = torch.searchsorted(middle, v.contiguous(), right=True)  # midpoints <= v
    return torch.where(low % 2 == 0, low, high)


def _exact_values(x, format, tensor_scale):
    """What x [rows, k] stands for after quantisation: the definition on the real line."""
    e2m1 = torch.tensor(_E2M1_VALUES, dtype=torch.float64, device=x.device)
    block, (rows, k) = _BLOCK[format], x.shape
    out = torch.empty((rows, k), dtype=torch.float64, device=x.device)
    for i in range(0, rows, max(1, (1 << 25) // k)):
        v = x[i:i + max(1, (1 << 25) // k)].double()
        v = torch.nn.functional.pad(v, (0, -k % block)).unflatten(1, (-1, block))
        top = v.abs().amax(dim=2, keepdim=True)
        if format == "nvfp4":
            e4m3 = torch.tensor(_E4M3_VALUES, dtype=torch.float64, device=x.device)
            g = tensor_scale.double()
            s = e4m3[_nearest(torch.nan_to_num(top / g / 6.0, nan=0.0), _E4M3_VALUES)] * g
        else:
            s = torch.ldexp(torch.ones_like(top), (torch.frexp(top).exponent - 3).clamp(min=-127))
        ratio = torch.nan_to_num(v.abs() / s, nan=0.0, posinf=0.0)
        value = torch.sign(v) * e2m1[_nearest(ratio, _E2M1_VALUES)] * s
        out[i:i + v.shape[0]] = value.flatten(1)[:, :k]
    return out


def _exact_operand(operand, format, rows, k):
    packed, tiles, tensor_scale = operand
    table = torch.tensor(_E2M1_VALUES + tuple(-v for v in _E2M1_VALUES), dtype=torch.float64, device=packed.device)
    block = _BLOCK[format]
    row, b = torch.arange(rows, device=packed.device)[:, None], torch.arange(-(-k // block), device=packed.device)[None, :]
    at = ((row // 128) * (-(-b.shape[1] // 4)) + b // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + b % 4
    code = tiles[at].long()
    if format == "nvfp4":
        s = torch.tensor(_E4M3_VALUES, dtype=torch.float64, device=packed.device)[code] * tensor_scale.double()
    else:
        s = torch.ldexp(torch.ones_like(code, dtype=torch.float64), code - 127)
    out = torch.empty((rows, packed.shape[1] * 2), dtype=torch.float64, device=packed.device)
    out[:, 0::2], out[:, 1::2] = table[(packed & 15).long()], table[(packed >> 4).long()]
    return out[:, :k] * s.repeat_interleave(block, dim=1)[:, :k]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "group_norm":
        x = state["x"]
        v = x.double().unflatten(2, (case["groups"], -1))
        variance, mean = torch.var_mean(v, dim=(1, 3), correction=0, keepdim=True)
        y = ((v - mean) / torch.sqrt(variance + 1e-6)).flatten(2) * state["weight"].double() + state["bias"].double()
        return _exact_activation(y, case["activation"])
    format = case["format"]
    if case["op"] == "round_trip":
        x = state["x"]
        g = (x.double().abs().max() / 2688.0).float() if format == "nvfp4" else None  # an F32 value by definition
        return _exact_values(x, format, g)
    m, k, n = case["m"], case["k"], case["n"]
    w = _exact_operand(state["w"], format, n, k)
    if case["op"] == "product":
        return _exact_operand(state["x"], format, m, k) @ w.t()
    y = _exact_values(state["x"], format, state["x_scale"]) @ w.t() + state["bias"].double()
    return _exact_activation(y, case["activation"])


def _exact_activation(y, activation):
    if activation == "silu":
        return y * torch.sigmoid(y)
    if activation == "gelu_tanh":
        return y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    return y
