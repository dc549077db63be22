"""The framework's microscaled 4-bit linear and its fused norms, as cases that can be timed and compared.

Three operators of a diffusion transformer's block with MXFP4 weights:

    "quantise"  16- or 32-bit rows -> MXFP4 (blocks of 32, E2M1 elements, one E8M0 scale) -> the values they stand for
    "product"   MXFP4 activations @ MXFP4 weights^T + bias -> 16 bits; the activations are MXFP4 already, or 16-bit rows that the
                call quantises
    "norm"      r = x + residual_scale * gate * post(y), h = (norm(r) * weight + bias) * (1 + scale) + shift
"""

import importlib
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token's activations before a linear of width 5120 (the repository's hidden size): latency
        {"name": "quantise one token", "op": "quantise", "rows": 1, "k": 5120, "dtype": "bf16"},
        # the activations of 4096 tokens before the down projection of a 13824-wide FFN
        {"name": "quantise activations", "op": "quantise", "rows": 4096, "k": 13824, "dtype": "bf16"},
        # an fp32 checkpoint weight on its way into the layer (loader) and back (LoRA merge)
        {"name": "quantise a weight", "op": "quantise", "rows": 13824, "k": 5120, "dtype": "fp32"},
        # ragged rows, K a multiple of 32 only
        {"name": "quantise ragged rows", "op": "quantise", "rows": 777, "k": 1056, "dtype": "fp16"},
        # one token through the FFN's up projection: the weight's bytes are the cost
        {"name": "product one token", "op": "product", "m": 1, "n": 13824, "k": 5120, "dtype": "bf16", "bias": True, "packed": False},
        # a handful of tokens through the down projection, activations already in MXFP4
        {"name": "product 16 tokens", "op": "product", "m": 16, "n": 5120, "k": 13824, "dtype": "bf16", "bias": False, "packed": True},
        # a ragged prompt in a narrow model: every tile edge is inside a tile
        {"name": "product ragged", "op": "product", "m": 520, "n": 2811, "k": 1056, "dtype": "fp16", "bias": True, "packed": False},
        # an image's tokens through the FFN's up projection: the tensor cores are the cost
        {"name": "product 8192 tokens", "op": "product", "m": 8192, "n": 13824, "k": 5120, "dtype": "bf16", "bias": True, "packed": True},
        # the norm between two blocks for one token
        {"name": "norm one token", "op": "norm", "batch": 1, "length": 1, "c": 5120, "dtype": "bf16", "y_dtype": "bf16", "kind": "rms", "post": True, "modulated": "sample"},
        # two samples of a diffusion transformer, shift / scale / gate for each
        {"name": "norm two samples", "op": "norm", "batch": 2, "length": 8192, "c": 5120, "dtype": "bf16", "y_dtype": "bf16", "kind": "layer", "post": False, "modulated": "sample"},
        # fp32 residual stream, norms before and after the block, weights only
        {"name": "norm fp32 stream", "op": "norm", "batch": 4, "length": 520, "c": 1024, "dtype": "fp32", "y_dtype": "fp16", "kind": "rms", "post": True, "modulated": "none"},
        # an odd width and a modulation for each token
        {"name": "norm odd width", "op": "norm", "batch": 3, "length": 333, "c": 1027, "dtype": "fp16", "y_dtype": "fp16", "kind": "layer", "post": True, "modulated": "token"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "norm"])
    if op == "quantise":
        k = 32 * _log(rng, 1, 432)
        rows = _log(rng, 1, max(1, min(16384, (13824 * 5120) // k)))
        return {"op": op, "rows": rows, "k": k, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "product":
        m, n, k = _log(rng, 1, 8192), _log(rng, 8, 13824), 32 * _log(rng, 1, 160)
        return {"op": op, "m": m, "n": n, "k": k, "dtype": rng.choice(["bf16", "fp16"]), "bias": rng.random() < 0.5, "packed": rng.random() < 0.5}
    c = _log(rng, 8, 8192)
    if rng.random() < 0.5:
        c = 8 * max(1, c // 8)
    batch = rng.choice([1, 2, 3, 4])
    length = _log(rng, 1, max(1, min(8192, (2 * 8192 * 5120) // (c * batch))))
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    return {"op": op, "batch": batch, "length": length, "c": c, "dtype": dtype, "y_dtype": dtype if dtype != "fp32" else rng.choice(["fp32", "bf16", "fp16"]),
            "kind": rng.choice(["rms", "layer"]), "post": rng.random() < 0.5, "modulated": rng.choice(["none", "sample", "token"])}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _activations(gen, rows, k, dtype):
    """Rows as a block sees them: normal, a few channels many times larger than the rest, the last row of several all zero (padding)."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x *= torch.exp2(torch.randint(-2, 3, (rows, 1), generator=gen, device="cuda").float())
    x[:, torch.randint(0, k, (max(1, k // 256),), generator=gen, device="cuda")] *= 20.0
    if rows > 4:
        x[-1] = 0.0
    return x.to(DTYPES[dtype])


def _packed(x):
    """MXFP4 bytes and scales of fp32 rows, in the layout the linear keeps: two codes to a byte, scales in tiles of 128 rows x 4 blocks."""
    rows, k = x.shape
    e, q = _mxfp4(x)
    code = torch.where(q.abs() <= 2, q.abs() * 2, torch.where(q.abs() <= 4, q.abs() + 2, torch.full_like(q, 7.0))).to(torch.uint8)
    code += torch.where(q < 0, 8, 0).to(torch.uint8)
    code = code.view(rows, k // 2, 2)
    data = code[..., 0] + 16 * code[..., 1]
    return data, _tiled((e + 127).to(torch.uint8))


def _tiled(scales):
    rows, blocks = scales.shape
    tr, tk = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros((tr * 128, tk * 4), dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(tr, 4, 32, tk, 4).permute(0, 3, 2, 1, 4).reshape(tr, tk, 512).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "quantise":
        x = _activations(gen, case["rows"], case["k"], case["dtype"])
        if case["dtype"] == "fp32":                                # a weight: no outliers, 1/sqrt(K) wide
            x = torch.randn(x.shape, generator=gen, device="cuda") / case["k"] ** 0.5
        return {"case": case, "x": x}
    if case["op"] == "product":
        m, n, k, dtype = case["m"], case["n"], case["k"], DTYPES[case["dtype"]]
        x = _activations(gen, m, k, case["dtype"])
        w, ws = _packed(torch.randn((n, k), generator=gen, device="cuda") / k ** 0.5)
        bias = torch.randn((n,), generator=gen, device="cuda").to(dtype) if case["bias"] else None
        state = {"case": case, "w": w, "ws": ws, "bias": bias, "dtype": dtype}
        if case["packed"]:
            state["a"], state["as"] = _packed(x.float())
        else:
            state["x"] = x
        return state
    b, l, c, dtype = case["batch"], case["length"], case["c"], DTYPES[case["dtype"]]

    def vector(*shape, spread=0.2, about=0.0, dt=torch.bfloat16):
        return (about + spread * torch.randn(shape, generator=gen, device="cuda")).to(dt)

    state = {"case": case, "x": (2.0 * torch.randn((b, l, c), generator=gen, device="cuda") + 0.25).to(dtype),
             "y": torch.randn((b, l, c), generator=gen, device="cuda").to(DTYPES[case["y_dtype"]]),
             "gate": None, "scale": None, "shift": None, "weight": None, "bias": None, "post_weight": None, "residual_scale": 1.0, "eps": 1e-6}
    if case["post"]:
        state["post_weight"] = vector(c, about=1.0)
    if case["modulated"] == "none":
        state["weight"], state["bias"], state["residual_scale"] = vector(c, about=1.0), vector(c) if case["kind"] == "layer" else None, 0.5
    else:
        # one projection gives all three, as in a diffusion transformer: slices of a wider fp32 tensor
        per = l if case["modulated"] == "token" else 1
        state["shift"], state["scale"], state["gate"] = vector(b, per, 3 * c, dt=torch.float32).chunk(3, dim=-1)
    return state


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def _mxfp4(x):
    """(scale exponents, elements) of fp32 rows; elements are the E2M1 values, still to be multiplied by 2^exponent."""
    blocks = x.reshape(x.shape[0], -1, 32)
    _, exponent = torch.frexp(blocks.abs().amax(dim=-1))                   # amax = f * 2^exponent, f in [0.5, 1)
    e = torch.where(blocks.abs().amax(dim=-1) > 0, (exponent - 3).clamp(min=-127), torch.full_like(exponent, -127))
    v = torch.ldexp(blocks, -e.unsqueeze(-1))
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)                      # torch.round: ties to even, as the elements' codes
    return e, torch.where(v < 0, -q, q).view(x.shape)


def _values(e, q):
    """fp32 values of elements and exponents; two steps, since 2^-127 alone is not a normal fp32 number."""
    scale = torch.ldexp(torch.ones_like(e, dtype=torch.float32), e).repeat_interleave(32, dim=1)
    return q * scale


def _unpacked(data, scales, k):
    rows = data.shape[0]
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=data.device)
    code = torch.stack((data & 15, data >> 4), dim=-1).view(rows, k)
    tr, tk = scales.shape[:2]
    flat = scales.view(tr, tk, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tr * 128, tk * 4)[:rows, : k // 32]
    return _values(flat.to(torch.int32) - 127, lut[code.int()])


def _norm32(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    return v * torch.rsqrt(v.square().mean(dim=-1, keepdim=True) + eps)


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "quantise":
        return _values(*_mxfp4(state["x"].float())).to(state["x"].dtype)
    if case["op"] == "product":
        a = _unpacked(state["a"], state["as"], case["k"]) if case["packed"] else _values(*_mxfp4(state["x"].float()))
        y = a @ _unpacked(state["w"], state["ws"], case["k"]).t()
        if state["bias"] is not None:
            y = y + state["bias"].float()
        return y.to(state["dtype"])
    z = state["y"].float()
    if state["post_weight"] is not None:
        z = _norm32(z, case["kind"], state["eps"]) * state["post_weight"].float()
    if state["gate"] is not None:
        z = z * state["gate"].float()
    r = state["x"].float() + state["residual_scale"] * z
    h = _norm32(r, case["kind"], state["eps"])
    if state["weight"] is not None:
        h = h * state["weight"].float()
    if state["bias"] is not None:
        h = h + state["bias"].float()
    if state["scale"] is not None:
        h = h * (1.0 + state["scale"].float()) + state["shift"].float()
    return {"r": r.to(state["x"].dtype), "h": h.to(state["y"].dtype)}


def _run_own(state):
    import __graft_entry__

    __graft_entry__.load_package()
    case = state["case"]
    if case["op"] == "norm":
        norm = importlib.import_module("feather_b200.kernel.norm")
        r, h = norm.gated_residual_norm(state["x"], state["y"], gate=state["gate"], residual_scale=state["residual_scale"], post_norm=state["post_weight"] is not None,
                                        post_weight=state["post_weight"], weight=state["weight"], bias=state["bias"], scale=state["scale"], shift=state["shift"],
                                        kind=case["kind"], eps=state["eps"], out_dtype=state["y"].dtype)
        return {"r": r, "h": h}
    mx = importlib.import_module("feather_b200.kernel.mxfp4")
    if case["op"] == "quantise":
        data, scales = mx.quantize_mxfp4(state["x"])
        return mx.dequantize_mxfp4(data, scales, state["x"].dtype)
    if case["packed"]:
        return mx.scaled_mm_mxfp4(state["a"], state["as"], state["w"], state["ws"], state["bias"], state["dtype"])
    return mx.linear_mxfp4(state["x"], state["w"], state["ws"], state["bias"], state["dtype"])


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    packed = 0.5 + 1 / 32
    if case["op"] == "quantise":                                           # rows in, MXFP4 out; MXFP4 in, values out
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * size[case["dtype"]] + 2 * packed), "flops": 4 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k * (packed if case["packed"] else 2)
        return {"bytes": a + n * k * packed + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    n, c = case["batch"] * case["length"] * case["c"], case["c"]
    extra = {"none": 0, "sample": 12 * case["batch"] * c, "token": 12 * n}[case["modulated"]] + 2 * c
    return {"bytes": 2 * n * (size[case["dtype"]] + size[case["y_dtype"]]) + extra, "flops": 20 * n}


# ------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_round(x):
    """MXFP4 values of fp64 rows: the nearest grid point of each scaled element by its borders, ties to the even code."""
    rows, k = x.shape
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    border = (grid[1:] + grid[:-1]) / 2
    out = torch.empty_like(x)
    chunk = max(1, (1 << 26) // k)
    for at in range(0, rows, chunk):
        block = x[at:at + chunk].reshape(-1, 32)
        top = block.abs().max(dim=1, keepdim=True).values
        unit = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2.0, min=-127.0))
        unit = torch.where(unit * 8.0 <= top, unit * 2.0, unit)             # log2 next to a power of two
        unit = torch.where(unit * 4.0 > top, torch.clamp(unit / 2.0, min=2.0 ** -127), unit)
        size = block.abs() / unit
        low, high = torch.bucketize(size, border), torch.bucketize(size, border, right=True)    # differ on a border: codes i and i + 1
        code = torch.where(low % 2 == 0, low, high)
        out[at:at + chunk] = (torch.sign(block) * grid[code] * unit).view(-1, k)
    return out


def _exact_unpacked(data, scales, k):
    """Byte by byte from the layout's definition: row r, element j."""
    rows = data.shape[0]
    grid = torch.tensor(_GRID, dtype=torch.float64, device=data.device)
    r, j = torch.arange(rows, device=data.device).unsqueeze(1), torch.arange(k, device=data.device).unsqueeze(0)
    code = (data[r, j // 2].long() >> (4 * (j % 2))) & 15
    value = grid[code & 7] * (1.0 - 2.0 * (code >> 3).double())
    b = j // 32
    power = scales[r // 128, b // 4, (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].double() - 127.0
    return value * torch.exp2(power)


def _exact_norm(v, kind, eps):
    mean = v.sum(dim=-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
    d = v - mean
    return d / torch.sqrt((d * d).sum(dim=-1, keepdim=True) / v.shape[-1] + eps)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantise":
        return _exact_round(state["x"].double())
    if case["op"] == "product":
        w = _exact_unpacked(state["w"], state["ws"], case["k"])
        a = _exact_unpacked(state["a"], state["as"], case["k"]) if case["packed"] else _exact_round(state["x"].double())
        y = torch.einsum("mk,nk->mn", a, w)
        return y if state["bias"] is None else y + state["bias"].double()
    r, h = torch.empty(state["x"].shape, dtype=torch.float64, device="cuda"), torch.empty(state["x"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["batch"]):
        z = state["y"][i].double()
        if case["post"]:
            z = _exact_norm(z, case["kind"], state["eps"]) * state["post_weight"].double()
        if state["gate"] is not None:
            z = z * state["gate"][i].double()
        r[i] = state["x"][i].double() + state["residual_scale"] * z
        v = _exact_norm(r[i], case["kind"], state["eps"])
        if state["weight"] is not None:
            v = v * state["weight"].double()
        if state["bias"] is not None:
            v = v + state["bias"].double()
        if state["scale"] is not None:
            v = v * (1.0 + state["scale"][i].double()) + state["shift"][i].double()
        h[i] = v
    return {"r": r, "h": h}
