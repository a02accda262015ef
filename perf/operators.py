"""The microscaled 4-bit operators and the mixture-of-experts layer over 4-bit experts: what is measured of them.

A case runs one of three operators:

  quantize   rows of f32 / bf16 / f16 values -> 4-bit codes and block scales -> the values they stand for. The codes are
             e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives). Format "e8m0_32": blocks of 32 share a power of two.
             Format "e4m3_16": blocks of 16 share an e4m3 number, a matrix shares one f32 number on top.
  product    C[m, n] = sum over k of A[m, k] * B[n, k], both operands held in one of the two formats.
  moe        a router, the top_k experts of each token, and their gated two-layer networks with 4-bit weights.

With `own` false `run` is plain torch; with `own` true it calls minicompiler_b200.
"""

import math

import torch

own = False

DEVICE = "cuda"
BLOCK = {"e8m0_32": 32, "e4m3_16": 16}
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------------------------------------ the cases


def listed():
    return [
        # one token's activations before a projection: latency
        dict(name="quantize_one_row", op="quantize", fmt="e8m0_32", dtype="bf16", rows=1, cols=2048),
        # a ragged matrix whose rows end inside a block
        dict(name="quantize_ragged_e4m3", op="quantize", fmt="e4m3_16", dtype="f16", rows=509, cols=1021),
        # a weight matrix as it is loaded, with its own f32 scale
        dict(name="quantize_weights_e4m3", op="quantize", fmt="e4m3_16", dtype="f32", rows=8192, cols=4096),
        # the activations of the MLP stack's batch
        dict(name="quantize_batch", op="quantize", fmt="e8m0_32", dtype="bf16", rows=65536, cols=2048),
        # one token through a large projection: the weights are streamed once
        dict(name="product_one_row", op="product", fmt="e8m0_32", dtype="bf16", m=1, n=8192, k=8192),
        # nothing divides anything
        dict(name="product_ragged_e4m3", op="product", fmt="e4m3_16", dtype="f16", m=77, n=1003, k=1501),
        # a serving batch
        dict(name="product_batch_128_e4m3", op="product", fmt="e4m3_16", dtype="bf16", m=128, n=8192, k=8192),
        # one layer of the MLP stack
        dict(name="product_mlp_layer_e4m3", op="product", fmt="e4m3_16", dtype="f16", m=65536, n=2048, k=2048),
        # the large square product
        dict(name="product_8192", op="product", fmt="e8m0_32", dtype="bf16", m=8192, n=8192, k=8192),
        # one token of a decode step
        dict(name="moe_one_token", op="moe", fmt="e8m0_32", dtype="bf16", tokens=1, experts=64, top_k=8, d=2048, f=1024, renormalize=True),
        # a few tokens, ragged widths
        dict(name="moe_ragged_e4m3", op="moe", fmt="e4m3_16", dtype="f16", tokens=7, experts=13, top_k=3, d=1000, f=721, renormalize=False),
        # a decode batch that reaches nearly every expert
        dict(name="moe_batch", op="moe", fmt="e4m3_16", dtype="bf16", tokens=32, experts=128, top_k=8, d=2048, f=768, renormalize=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high):
    """Spread over the logarithm; half of them multiples of 32."""
    v = _log(rng, low, high)
    return v if v < 64 or rng.random() < 0.5 else v // 32 * 32


def draw(rng):
    op = rng.choice(("quantize", "product", "moe"))
    fmt = rng.choice(("e8m0_32", "e4m3_16"))
    if op == "quantize":
        cols = _size(rng, 16, 16384)
        rows = _size(rng, 1, max(1, min(65536, (1 << 27) // cols)))
        return dict(op=op, fmt=fmt, dtype=rng.choice(("f32", "bf16", "f16")), rows=rows, cols=cols)
    if op == "product":
        n, k = _size(rng, 64, 16384), _size(rng, 64, 16384)
        m = _size(rng, 1, max(1, min(65536, (1 << 39) // (n * k), (1 << 28) // n, (1 << 28) // k)))
        return dict(op=op, fmt=fmt, dtype=rng.choice(("bf16", "f16")), m=m, n=n, k=k)
    experts = _log(rng, 4, 160)
    d = _size(rng, 64, 4096)
    f = _size(rng, 32, min(2048, (1 << 28) // (experts * d)))
    return dict(op=op, fmt=fmt, dtype=rng.choice(("bf16", "f16")), tokens=_log(rng, 1, 64), experts=experts,
                top_k=rng.randint(1, min(8, experts)), d=d, f=f, renormalize=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------- the stored format
# codes: uint8 [batch, rows, pitch], two per byte, the even column in the low bits, pitch = 16 bytes per 32 columns,
# zero behind the last column. scales: uint8 [batch, ceil(rows / 128), ceil(blocks / 4), 512], the byte of row r and
# block b at (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of its tile.


def _tiled(scales):
    batch, rows, blocks = scales.shape
    rt, kt = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros(batch, rt * 128, kt * 4, dtype=torch.uint8, device=scales.device)
    full[:, :rows, :blocks] = scales
    return full.view(batch, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5).reshape(batch, rt, kt, 512).contiguous()


def _untiled(tiles, rows, blocks):
    batch, rt, kt, _ = tiles.shape
    return tiles.view(batch, rt, kt, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(batch, rt * 128, kt * 4)[:, :rows, :blocks]


def _scale_values(tiles, fmt, rows, blocks):
    s = _untiled(tiles, rows, blocks).contiguous()
    if fmt == "e8m0_32":  # 2^(byte - 127); a byte of 0 does not occur beside codes other than 0
        return (s.to(torch.int32) << 23).view(torch.float32)
    return s.view(torch.float8_e4m3fn).to(torch.float32)


def _decoded(matrix, fmt, rows, cols):
    """f32 [batch, rows, cols] without the matrix's own f32 scale."""
    codes, tiles = matrix["codes"], matrix["scales"]
    blocks = -(-cols // BLOCK[fmt])
    magnitudes = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), device=codes.device)
    nibbles = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :cols]
    scales = _scale_values(tiles, fmt, rows, blocks)
    return magnitudes[nibbles.to(torch.int32)] * scales.repeat_interleave(BLOCK[fmt], dim=-1)[..., :cols]


def _rounded(x, fmt, g):
    """Block scales (f32) and magnitude numbers 0..7 of f32 x [batch, rows, cols]; g: f32 [batch] or None."""
    block = BLOCK[fmt]
    batch, rows, cols = x.shape
    blocks = -(-cols // block)
    padded = torch.nn.functional.pad(x, (0, blocks * block - cols)).view(batch, rows, blocks, block)
    amax = padded.abs().amax(dim=-1)
    if fmt == "e8m0_32":
        exponent = (torch.frexp(amax)[1] - 3).clamp(min=-127)  # floor(log2 amax) - 2
        exponent = torch.where(amax == 0, torch.full_like(exponent, -127), exponent)
        stored = (exponent + 127).to(torch.uint8)
        y = torch.ldexp(padded, -exponent[..., None])
    else:
        six_g = (6.0 * g).view(batch, 1, 1)
        stored8 = (amax / six_g).clamp(max=448.0).to(torch.float8_e4m3fn)
        stored = stored8.view(torch.uint8)
        step = stored8.to(torch.float32) * g.view(batch, 1, 1)
        inverse = torch.where(step == 0, torch.zeros_like(step), 1.0 / step)
        y = padded * inverse[..., None]
    a = y.abs()  # to the nearest of the eight magnitudes, ties to the even code
    number = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    number = number + 8 * torch.signbit(y).to(torch.uint8)
    return stored, number.view(batch, rows, blocks * block)[..., :cols]


def _own_scale(x):
    """The f32 scale of each matrix of x [batch, rows, cols]: its largest magnitude goes to 6 * 448."""
    amax = x.abs().amax(dim=(1, 2))
    return amax / torch.full_like(amax, 2688.0)  # a division: by a plain number torch multiplies with the reciprocal


def _held(x, fmt):
    """A matrix in hand in the stored format: f32 [batch, rows, cols] -> dict."""
    g = _own_scale(x) if fmt == "e4m3_16" else None
    stored, number = _rounded(x, fmt, g)
    batch, rows, cols = x.shape
    width = -(-cols // 32) * 32
    number = torch.nn.functional.pad(number, (0, width - cols)).view(batch, rows, width // 2, 2)
    return {"codes": (number[..., 0] | (number[..., 1] << 4)).contiguous(), "scales": _tiled(stored), "g": g}


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _activations(gen, rows, cols):
    """Normal values with the few wide channels that activations have."""
    x = torch.randn(rows, cols, generator=gen, device=DEVICE)
    wide = torch.rand(cols, generator=gen, device=DEVICE) < 0.01
    return torch.where(wide, x * 8.0, x)


# -------------------------------------------------------------------------------------------------------------- prepare


def prepare(case, seed):
    gen = _generator(seed)
    fmt, dtype = case["fmt"], DTYPE[case["dtype"]]
    if case["op"] == "quantize":
        x = _activations(gen, case["rows"], case["cols"]).to(dtype)
        state = {"case": case, "x": x}
    elif case["op"] == "product":
        a = _held(_activations(gen, case["m"], case["k"])[None], fmt)
        b = _held(torch.randn(1, case["n"], case["k"], generator=gen, device=DEVICE) * case["k"] ** -0.5, fmt)
        state = {"case": case, "a": a, "b": b}
    else:
        e, d, f = case["experts"], case["d"], case["f"]
        parts = ([], [])
        for _ in range(e):
            parts[0].append(_held(torch.randn(1, 2 * f, d, generator=gen, device=DEVICE) * d ** -0.5, fmt))
            parts[1].append(_held(torch.randn(1, d, f, generator=gen, device=DEVICE) * f ** -0.5, fmt))
        stacked = [{key: None if p[0][key] is None else torch.cat([q[key] for q in p]) for key in ("codes", "scales", "g")} for p in parts]
        x = torch.randn(case["tokens"], d, generator=gen, device=DEVICE).to(dtype)
        router = (torch.randn(e, d, generator=gen, device=DEVICE) * d ** -0.5).to(dtype)
        state = {"case": case, "x": x, "router": router, "gate_up": stacked[0], "down": stacked[1]}
    if own:
        _plan(state)
    return state


def _plan(state):
    """What a program keeps beside its data: descriptors of the device memory, result buffers, workspace."""
    import minicompiler_b200 as mc

    case = state["case"]
    fmt, dtype = case["fmt"], case["dtype"]

    def empty(shape, t):
        return torch.empty(shape, dtype=t, device=DEVICE)

    def described(held, rows, cols, batch=1):
        g = held["g"]
        return mc.Fp4Matrix(fmt, rows, cols, held["codes"].data_ptr(), held["scales"].data_ptr(), 0 if g is None else g.data_ptr(), batch)

    state["mc"] = mc
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        sizes = mc.fp4_sizes(fmt, rows, cols)
        held = {"codes": empty(sizes.codes_bytes, torch.uint8), "scales": empty(sizes.scales_bytes, torch.uint8),
                "g": empty(1, torch.float32) if fmt == "e4m3_16" else None}
        state.update(held=held, matrix=described(held, rows, cols), values=empty((rows, cols), DTYPE[dtype]))
    elif case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        need = mc.fp4_gemm_workspace_bytes(fmt, m, n, k)
        state.update(c=empty((m, n), DTYPE[dtype]), workspace=empty(max(1, need), torch.uint8))
        state["plan"] = mc.Fp4Gemm(described(state["a"], m, k), described(state["b"], n, k), state["c"].data_ptr(), dtype,
                                   workspace=state["workspace"].data_ptr(), workspace_bytes=need)
    else:
        t, e, d, f, top_k = case["tokens"], case["experts"], case["d"], case["f"], case["top_k"]
        need = mc.moe_workspace_bytes(t, e, top_k, d, f)
        state.update(y=empty((t, d), DTYPE[dtype]), chosen=empty((t, top_k), torch.int32), weights=empty((t, top_k), torch.float32),
                     workspace=empty(max(1, need), torch.uint8))
        state["plan"] = mc.MoeLayer(described(state["gate_up"], 2 * f, d, e), described(state["down"], d, f, e), state["x"].data_ptr(), dtype,
                                    state["router"].data_ptr(), state["y"].data_ptr(), tokens=t, top_k=top_k, renormalize=case["renormalize"],
                                    chosen=state["chosen"].data_ptr(), weights=state["weights"].data_ptr(),
                                    workspace=state["workspace"].data_ptr(), workspace_bytes=need)


# ------------------------------------------------------------------------------------------------------------------ run


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"quantize": _plain_quantize, "product": _plain_product, "moe": _plain_moe}[case["op"]](case, state)


def _run_own(case, state):
    mc, stream = state["mc"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "quantize":
        x, matrix, g = state["x"], state["matrix"], state["held"]["g"]
        if g is not None:
            mc.fp4_tensor_scale(x.data_ptr(), case["dtype"], case["rows"], case["cols"], g.data_ptr(), stream=stream)
        mc.fp4_quantize(x.data_ptr(), case["dtype"], matrix, stream=stream)
        mc.fp4_dequantize(matrix, state["values"].data_ptr(), case["dtype"], stream=stream)
        return {"values": state["values"]} if g is None else {"values": state["values"], "scale": g}
    state["plan"].enqueue(stream)
    if case["op"] == "product":
        return {"c": state["c"]}
    return {"y": state["y"], "chosen": state["chosen"], "weights": state["weights"]}


def _plain_quantize(case, state):
    fmt, rows, cols = case["fmt"], case["rows"], case["cols"]
    x = state["x"].to(torch.float32)[None]
    held = _held(x, fmt)
    values = _decoded(held, fmt, rows, cols)[0]
    if held["g"] is None:
        return {"values": values.to(DTYPE[case["dtype"]])}
    return {"values": (values * held["g"]).to(DTYPE[case["dtype"]]), "scale": held["g"]}


def _plain_product(case, state):
    fmt, m, n, k = case["fmt"], case["m"], case["n"], case["k"]
    a, b = _decoded(state["a"], fmt, m, k)[0], _decoded(state["b"], fmt, n, k)[0]
    c = a @ b.T
    if fmt == "e4m3_16":
        c = c * (state["a"]["g"] * state["b"]["g"])
    return {"c": c.to(DTYPE[case["dtype"]])}


def _plain_moe(case, state):
    fmt, tokens, experts, top_k, d, f = (case[key] for key in ("fmt", "tokens", "experts", "top_k", "d", "f"))
    x = state["x"].to(torch.float32)
    logits = x.to(torch.float64) @ state["router"].to(torch.float64).T
    order = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :top_k]
    weights = torch.softmax(logits, dim=-1).gather(1, order).to(torch.float32)
    if case["renormalize"]:
        weights = weights / weights.sum(dim=-1, keepdim=True)

    def part(matrix, slots):
        return {key: None if v is None else v[slots] for key, v in matrix.items()}

    def scaled(matrix, rows, cols):
        w = _decoded(matrix, fmt, rows, cols)
        return w if matrix["g"] is None else w * matrix["g"].view(-1, 1, 1)

    if tokens * top_k <= experts:  # only the chosen experts, once for each (token, expert)
        slots = order.flatten()
        xs = x.repeat_interleave(top_k, dim=0)[:, :, None]
        h = (scaled(part(state["gate_up"], slots), 2 * f, d) @ xs)[..., 0]
        h = h[:, :f] * torch.sigmoid(h[:, :f]) * h[:, f:]
        y = (scaled(part(state["down"], slots), d, f) @ h[:, :, None])[..., 0].view(tokens, top_k, d)
    else:  # every expert on every token, then the chosen ones
        h = torch.matmul(x, scaled(state["gate_up"], 2 * f, d).transpose(1, 2))
        h = h[..., :f] * torch.sigmoid(h[..., :f]) * h[..., f:]
        every = torch.matmul(h, scaled(state["down"], d, f).transpose(1, 2)).transpose(0, 1)
        y = every.gather(1, order[:, :, None].expand(tokens, top_k, d))
    y = (y * weights[:, :, None]).sum(dim=1)
    return {"y": y.to(DTYPE[case["dtype"]]), "chosen": order.to(torch.int32), "weights": weights}


# ----------------------------------------------------------------------------------------------------------------- work


def _held_bytes(fmt, rows, cols):
    return rows * (cols / 2 + -(-cols // BLOCK[fmt]))


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * n * size + 2 * _held_bytes(case["fmt"], case["rows"], case["cols"]), "flops": 4 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _held_bytes(case["fmt"], m, k) + _held_bytes(case["fmt"], n, k) + m * n * size, "flops": 2 * m * n * k}
    t, e, d, f, top_k = (case[key] for key in ("tokens", "experts", "d", "f", "top_k"))
    reached = e * (1.0 - (1.0 - top_k / e) ** t)  # experts that get a token, on average
    weights = _held_bytes(case["fmt"], 2 * f, d) + _held_bytes(case["fmt"], d, f)
    return {"bytes": reached * weights + (e + 2 * t) * d * size, "flops": 2 * t * e * d + t * top_k * 6 * d * f}


# ---------------------------------------------------------------------------------------------------------------- exact
# From the definitions, in 64 bits; numbers are taken apart with floor and log2 of exact powers instead of the bits.


def _exact_grid(y):
    """The nearest e2m1 number: a step of 0.5 below 2, of 1 below 4, of 2 up to 6; ties to the even multiple."""
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).to(torch.float64)
    return torch.copysign(torch.round(a / step) * step, y)


def _power_below(x):
    """The largest power of two that is not above x > 0: log2 may be off by its last bit, so its floor is put right."""
    e = torch.floor(torch.log2(x))
    e = torch.where(torch.exp2(e + 1.0) <= x, e + 1.0, e)
    return torch.exp2(torch.where(torch.exp2(e) > x, e - 1.0, e))


def _exact_e4m3(t):
    """The nearest e4m3 number of t >= 0, at most 448."""
    t = t.clamp(max=448.0)
    step = _power_below(t.clamp(min=2.0 ** -6)) / 8.0
    return (torch.round(t / step) * step).clamp(max=448.0)


def _exact_f32(x):
    return x.to(torch.float32).to(torch.float64)


def _exact_decoded(held, fmt, rows, cols):
    codes = held["codes"].to(torch.int16)
    width = codes.shape[-1] * 2
    c = torch.empty(*codes.shape[:-1], width, dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        nibble = (codes // 16 if half else codes % 16).to(torch.float64)
        sign = 1.0 - 2.0 * torch.floor(nibble / 8.0)
        three = nibble % 8.0
        exponent, mantissa = torch.floor(three / 2.0), three % 2.0
        c[..., half::2] = sign * torch.where(exponent == 0, mantissa / 2.0, (1.0 + mantissa / 2.0) * torch.exp2(exponent - 1.0))
    block = BLOCK[fmt]
    column = torch.arange(cols, device=codes.device) // block
    row = torch.arange(rows, device=codes.device)
    place = (row % 32 * 16 + row // 32 % 4 * 4)[:, None] + (column % 4)[None, :]
    byte = held["scales"][:, (row // 128)[:, None], (column // 4)[None, :], place].to(torch.float64)
    if fmt == "e8m0_32":
        scale = torch.exp2(byte - 127.0)
    else:
        exponent, mantissa = torch.floor(byte / 8.0), byte % 8.0
        scale = torch.where(exponent == 0, mantissa / 8.0 * 2.0 ** -6, (1.0 + mantissa / 8.0) * torch.exp2(exponent - 7.0))
        scale = scale * held["g"].to(torch.float64).view(-1, 1, 1)
    return c[..., :cols] * scale


def exact(case, seed):
    state = prepare(case, seed)
    fmt = case["fmt"]
    if case["op"] == "quantize":
        return _exact_quantize(fmt, state["x"].to(torch.float64))
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        b = _exact_decoded(state["b"], fmt, n, k)[0]
        return {"c": _exact_decoded(state["a"], fmt, m, k)[0] @ b.T}
    return _exact_moe(case, state)


def _exact_quantize(fmt, x):
    block = BLOCK[fmt]
    rows, cols = x.shape
    blocks = -(-cols // block)
    padded = torch.zeros(rows, blocks * block, dtype=torch.float64, device=x.device)
    padded[:, :cols] = x
    padded = padded.view(rows, blocks, block)
    amax = padded.abs().max(dim=-1, keepdim=True)[0]
    if fmt == "e8m0_32":
        step = _power_below(amax.clamp(min=2.0 ** -125)) / 4.0
        return {"values": (_exact_grid(padded / step) * step).view(rows, -1)[:, :cols]}
    # the format defines its scales with f32 steps: g, amax / (6 g), the step s g and its reciprocal are f32 numbers
    g = _exact_f32(x.abs().max() / 2688.0)
    s = _exact_e4m3(_exact_f32(amax / _exact_f32(6.0 * g)))
    step = _exact_f32(s * g)
    inverse = torch.where(step == 0, torch.zeros_like(step), _exact_f32(1.0 / step))
    values = _exact_grid(_exact_f32(padded * inverse)) * s * g
    return {"values": values.view(rows, -1)[:, :cols], "scale": g.view(1)}


def _exact_moe(case, state):
    fmt, tokens, top_k, d, f = (case[key] for key in ("fmt", "tokens", "top_k", "d", "f"))
    x = state["x"].to(torch.float64)
    logits = (x[:, None, :] * state["router"].to(torch.float64)[None]).sum(dim=-1)
    p = torch.exp(logits - logits.max(dim=-1, keepdim=True)[0])
    p = p / p.sum(dim=-1, keepdim=True)
    rest = logits.clone()
    rows = torch.arange(tokens, device=x.device)
    chosen = torch.empty(tokens, top_k, dtype=torch.int64, device=x.device)
    for j in range(top_k):
        chosen[:, j] = rest.argmax(dim=-1)
        rest[rows, chosen[:, j]] = -math.inf
    weights = p[rows[:, None], chosen]
    if case["renormalize"]:
        weights = weights / weights.sum(dim=-1, keepdim=True)
    y = torch.zeros(tokens, d, dtype=torch.float64, device=x.device)
    for e in sorted(set(chosen.flatten().tolist())):
        t, j = torch.nonzero(chosen == e, as_tuple=True)

        def one(held, r, c):
            return _exact_decoded({key: None if v is None else v[e:e + 1] for key, v in held.items()}, fmt, r, c)[0]

        h = x[t] @ one(state["gate_up"], 2 * f, d).T
        h = h[:, :f] / (1.0 + torch.exp(-h[:, :f])) * h[:, f:]
        y.index_add_(0, t, (h @ one(state["down"], d, f).T) * weights[t, j][:, None])
    return {"y": y, "chosen": chosen.to(torch.int32), "weights": weights}
