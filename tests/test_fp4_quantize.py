"""Rounding to the microscaled 4-bit formats and back, against the definition in 64 bits (oracle/fp4_reference.py).

Codes and scales are whole numbers that the definition fixes, so they have to be equal, bytes of padding included. A value
read back is code * scale, exact in f32 (at most 6 significant bits); E4M3_16 multiplies with the f32 tensor scale (one
rounding, 2^-24 relative) and a 16-bit result is rounded once more (half a step: bf16 2^-8, f16 2^-11)."""

import ctypes as C

import numpy as np
import pytest

FORMATS = ("e8m0_32", "e4m3_16")


@pytest.fixture(scope="module")
def ref():
    from oracle import fp4_reference

    return fp4_reference


# ------------------------------------------------------------------------------------------------- without a GPU


def test_sizes_follow_the_layout(mc):
    for rows, cols in [(1, 1), (1, 32), (127, 33), (128, 128), (129, 4097)]:
        for fmt, block in (("e8m0_32", 32), ("e4m3_16", 16)):
            s = mc.fp4_sizes(fmt, rows, cols, 3)
            assert s.code_pitch == -(-cols // 32) * 16
            assert s.codes_bytes == 3 * rows * s.code_pitch
            assert s.scales_bytes == 3 * -(-rows // 128) * -(-(-(-cols // block)) // 4) * 512


def test_reference_tables(ref):
    import torch

    table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.E4M3, table)
    # ties go to the even code, past the end is the end
    assert ref.nearest_even([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 1e30], ref.MAGNITUDES).tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7]


def _matrix(mc, fmt="e8m0_32", rows=4, cols=64, codes=1 << 20, scales=1 << 21, g=0, batch=1):
    return mc.Fp4Matrix(fmt, rows, cols, codes, scales, g, batch)


@pytest.mark.parametrize("change, message", [
    (dict(rows=0), "empty matrix"),
    (dict(cols=0), "empty matrix"),
    (dict(batch=0), "no matrices"),
    (dict(codes=0), "null codes or scales"),
    (dict(scales=0), "null codes or scales"),
    (dict(codes=(1 << 20) + 8), "16-byte alignment"),
    (dict(scales=(1 << 20) + 4), "16-byte alignment"),
    (dict(g=4096), "no tensor scale"),
    (dict(fmt="e4m3_16", g=4098), "unaligned tensor scale"),
    (dict(rows=1 << 31), "too large"),
    (dict(cols=(1 << 30) + 1), "too large"),
])
def test_a_wrong_matrix_is_refused_by_both_directions(mc, change, message):
    m = _matrix(mc, **change)
    with pytest.raises(mc.McError, match=message):
        mc.fp4_quantize(1 << 22, "f32", m, pitch=1 << 31)
    with pytest.raises(mc.McError, match=message):
        mc.fp4_dequantize(m, 1 << 22, "f32", pitch=1 << 31)


def test_wrong_values_are_refused(mc):
    m = _matrix(mc)
    with pytest.raises(mc.McError, match="null values"):
        mc.fp4_quantize(0, "f32", m)
    with pytest.raises(mc.McError, match="not aligned to their type"):
        mc.fp4_quantize((1 << 22) + 2, "f32", m)
    with pytest.raises(mc.McError, match="not aligned to their type"):
        mc.fp4_dequantize(m, (1 << 22) + 1, "bf16")
    with pytest.raises(mc.McError, match="less than a row"):
        mc.fp4_quantize(1 << 22, "f32", m, pitch=63)
    with pytest.raises(mc.McError, match="unknown type"):
        mc.fp4_quantize(1 << 22, "f64", m)
    with pytest.raises(mc.McError, match="unknown 4-bit format"):
        mc.Fp4Matrix("e5m2", 1, 1, 16, 16)
    lib = mc.lib()
    assert lib.mcd_fp4_quantize(7, 1 << 22, 64, m._ref, 0) != 0 and b"unknown type" in lib.mcd_last_error()
    assert lib.mcd_fp4_quantize(0, 1 << 22, 64, None, 0) != 0 and b"null 4-bit matrix" in lib.mcd_last_error()
    m._c.format = 3
    assert lib.mcd_fp4_quantize(0, 1 << 22, 64, m._ref, 0) != 0 and b"unknown 4-bit format" in lib.mcd_last_error()
    for args, message in [(dict(rows=0), "empty"), (dict(batch=0), "no matrices"), (dict(out=0), "null or unaligned"), (dict(out=2), "null or unaligned"),
                          (dict(src=0), "null values")]:
        a = dict(src=1 << 22, dtype="f32", rows=4, cols=4, out=1 << 20, batch=1) | args
        with pytest.raises(mc.McError, match=message):
            mc.fp4_tensor_scale(a["src"], a["dtype"], a["rows"], a["cols"], a["out"], batch=a["batch"])


# ------------------------------------------------------------------------------------------------------ on a GPU


def _torch_dtype(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _buffers(mc, fmt, rows, cols, batch, fill=0xA5, guard=256):
    import torch

    sizes = mc.fp4_sizes(fmt, rows, cols, batch)
    codes = torch.full((sizes.codes_bytes + guard,), fill, dtype=torch.uint8, device="cuda")
    scales = torch.full((sizes.scales_bytes + guard,), fill, dtype=torch.uint8, device="cuda")
    return codes, scales, sizes


def _values(rng, rows, cols, dtype):
    """Values over many binades, zeros and exact ties among them, as the type holds them (returned in 64 bits)."""
    import torch

    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-6, 7, size=(rows, 1)))
    x = np.where(rng.random((rows, cols)) < 0.1, 0.0, x)
    ties = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -2.5, -5.0], size=(rows, cols))
    x = np.where(rng.random((rows, cols)) < 0.2, ties, x)
    return torch.from_numpy(x).to(_torch_dtype(dtype))


def _round_trip(mc, ref, fmt, dtype, x, *, batch=1, pitch=None, offset=0, stream=0, scale=True):
    """Quantises x [batch, rows, cols] (torch, CPU), checks every byte, reads it back and checks the values."""
    import torch

    b, rows, cols = x.shape
    pitch = pitch or cols
    t = _torch_dtype(dtype)
    src = torch.full((offset + b * rows * pitch,), 3.0, dtype=t, device="cuda")
    view = src[offset:].view(b, rows, pitch)
    view[:, :, :cols] = x.to("cuda")
    codes, scales, sizes = _buffers(mc, fmt, rows, cols, b)
    g = None
    torch.cuda.synchronize()
    if fmt == "e4m3_16" and scale:
        g = torch.full((b,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        mc.fp4_tensor_scale(view.data_ptr(), dtype, rows, cols, g.data_ptr(), pitch=pitch, batch=b, stream=stream)
    m = mc.Fp4Matrix(fmt, rows, cols, codes.data_ptr(), scales.data_ptr(), 0 if g is None else g.data_ptr(), b)
    mc.fp4_quantize(view.data_ptr(), dtype, m, pitch=pitch, stream=stream)
    out = torch.full((offset + b * rows * pitch + 8,), 7.0, dtype=t, device="cuda")
    torch.cuda.synchronize()
    back = out[offset:offset + b * rows * pitch].view(b, rows, pitch)
    mc.fp4_dequantize(m, back.data_ptr(), dtype, pitch=pitch, stream=stream)
    torch.cuda.synchronize()
    assert (codes[sizes.codes_bytes:] == 0xA5).all() and (scales[sizes.scales_bytes:] == 0xA5).all()
    assert (out[:offset] == 7.0).all() and (back[:, :, cols:] == 7.0).all() and (out[offset + b * rows * pitch:] == 7.0).all()
    got_codes = codes[: sizes.codes_bytes].cpu().numpy().reshape(b, rows, sizes.code_pitch)
    got_scales = scales[: sizes.scales_bytes].cpu().numpy().reshape(b, -(-rows // 128), -1, 512)
    half_step = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype] * (1 + 2.0 ** -20)
    smallest = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}[dtype] / 2  # half a subnormal step
    for i in range(b):
        xi = x[i].double().numpy()
        gi = 1.0
        if g is not None:
            gi = float(g[i].item())
            assert gi == ref.tensor_scale(xi)
        code, scale_bytes = ref.quantize(xi, fmt, gi)
        want_codes, want_scales = ref.pack(code, scale_bytes, fmt)
        assert np.array_equal(got_scales[i], want_scales)
        assert np.array_equal(got_codes[i], want_codes)
        want = ref.values(code, scale_bytes, fmt, gi)
        got = back[i, :, :cols].double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        f32_step = 2.0 ** -24 if g is not None else 0.0
        limit = np.finfo(np.float32).max if dtype != "f16" else 65504.0
        fine = ~np.isnan(want) & (np.abs(want) <= limit)
        assert (np.abs(got - want)[fine] <= (np.abs(want) * (half_step + f32_step) + smallest)[fine]).all()
        assert (np.abs(got)[~np.isnan(want) & ~fine] >= limit).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 32), (3, 31), (2, 16), (5, 77), (128, 128), (129, 513), (31, 4100), (260, 96)])
def test_every_byte_is_the_definitions(mc, ref, fmt, dtype, rows, cols):
    rng = np.random.default_rng(rows * 1000 + cols)
    _round_trip(mc, ref, fmt, dtype, _values(rng, rows, cols, dtype)[None])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ("f32", "f16"))
@pytest.mark.parametrize("pitch, offset", [(80, 0), (77, 1), (79, 3), (96, 16), (72, 0), (76, 4), (72, 8)])
def test_strides_and_alignment(mc, ref, fmt, dtype, pitch, offset):
    rng = np.random.default_rng(pitch)
    x = _values(rng, 3 * 130, 70, dtype).view(3, 130, 70)
    _round_trip(mc, ref, fmt, dtype, x, batch=3, pitch=pitch, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_infinity_extremes_and_zero(mc, ref, fmt):
    import torch

    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 160)).astype(np.float32)
    x[0, 3], x[1, 40], x[2, 159] = np.nan, np.inf, -np.inf
    x[3] = 0.0
    x[4] = -0.0
    x[5] = 2.0 ** -149  # the smallest subnormals
    x[6] = rng.standard_normal(160) * 2.0 ** -140
    x[7] = rng.standard_normal(160) * 2.0 ** -126
    x[8] = np.finfo(np.float32).max
    x[9, ::2] = np.finfo(np.float32).max
    x[10] = np.exp2(rng.integers(-120, 120, 160))
    x[11] = 448.0 * 6.0 * np.sign(rng.standard_normal(160))
    x[12, :16] = 6.0 * 448 * 1.5
    _round_trip(mc, ref, fmt, "f32", torch.from_numpy(x)[None], scale=False)
    _round_trip(mc, ref, fmt, "f32", torch.from_numpy(x[11:])[None])


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf"), 2.0 ** -140, 2.0 ** 126, 3.3e38, 0.37])
def test_any_tensor_scale(mc, ref, g):
    import torch

    rng = np.random.default_rng(9)
    x = rng.standard_normal((3, 64)).astype(np.float32)
    codes, scales, sizes = _buffers(mc, "e4m3_16", 3, 64, 1)
    tg = torch.tensor([g], device="cuda", dtype=torch.float32)
    m = mc.Fp4Matrix("e4m3_16", 3, 64, codes.data_ptr(), scales.data_ptr(), tg.data_ptr())
    src = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    mc.fp4_quantize(src.data_ptr(), "f32", m)
    torch.cuda.synchronize()
    code, scale_bytes = ref.quantize(x, "e4m3_16", float(np.float32(g)))
    want_codes, want_scales = ref.pack(code, scale_bytes, "e4m3_16")
    assert np.array_equal(scales[: sizes.scales_bytes].cpu().numpy().reshape(want_scales.shape), want_scales)
    assert np.array_equal(codes[: sizes.codes_bytes].cpu().numpy().reshape(want_codes.shape), want_codes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("batch, rows, cols", [(1, 1, 1), (2, 3, 50), (3, 300, 700), (1, 1500, 1001)])
def test_tensor_scale_passes_over_what_is_not_finite(mc, ref, dtype, batch, rows, cols):
    import torch

    rng = np.random.default_rng(rows)
    x = torch.from_numpy(rng.standard_normal((batch, rows, cols)) * 5).to(_torch_dtype(dtype))
    if rows > 1:
        x[0, 1, 2], x[0, 2, 1] = float("inf"), float("nan")
        x[-1, 2, 3] = -77.0
    d = x.cuda()
    out = torch.full((batch + 1,), 9.0, device="cuda")
    torch.cuda.synchronize()
    mc.fp4_tensor_scale(d.data_ptr(), dtype, rows, cols, out.data_ptr(), batch=batch)
    torch.cuda.synchronize()
    assert out[batch].item() == 9.0
    for i in range(batch):
        assert out[i].item() == ref.tensor_scale(x[i].double().numpy())
    zero = torch.zeros(rows, cols, device="cuda", dtype=_torch_dtype(dtype))
    mc.fp4_tensor_scale(zero.data_ptr(), dtype, rows, cols, out.data_ptr())
    torch.cuda.synchronize()
    assert out[0].item() == 1.0


@pytest.mark.gpu
def test_host_memory_is_refused(mc):
    import torch

    codes, scales, _ = _buffers(mc, "e8m0_32", 4, 64, 1)
    m = mc.Fp4Matrix("e8m0_32", 4, 64, codes.data_ptr(), scales.data_ptr())
    host = np.zeros(256, dtype=np.float32)
    with pytest.raises(mc.McError, match="not device memory"):
        mc.fp4_quantize(host.ctypes.data, "f32", m)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_side_stream_and_replayed_graph(mc, ref, fmt):
    import torch

    rng = np.random.default_rng(2)
    rows, cols = 33, 200
    first, second = (_values(rng, rows, cols, "bf16") for _ in range(2))
    src = first.cuda()
    codes, scales, sizes = _buffers(mc, fmt, rows, cols, 1)
    g = torch.ones(1, device="cuda")
    m = mc.Fp4Matrix(fmt, rows, cols, codes.data_ptr(), scales.data_ptr(), g.data_ptr() if fmt == "e4m3_16" else 0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        if fmt == "e4m3_16":
            mc.fp4_tensor_scale(src.data_ptr(), "bf16", rows, cols, g.data_ptr(), stream=side.cuda_stream)
        mc.fp4_quantize(src.data_ptr(), "bf16", m, stream=side.cuda_stream)
    for x in (first, second):
        src.copy_(x)
        codes.fill_(0xA5)
        scales.fill_(0xA5)
        graph.replay()
        torch.cuda.synchronize()
        gi = float(g.item())
        code, scale_bytes = ref.quantize(x.double().numpy(), fmt, gi)
        want_codes, want_scales = ref.pack(code, scale_bytes, fmt)
        assert np.array_equal(codes[: sizes.codes_bytes].cpu().numpy().reshape(want_codes.shape), want_codes)
        assert np.array_equal(scales[: sizes.scales_bytes].cpu().numpy().reshape(want_scales.shape), want_scales)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, cols", [(4, 96), (1024, 4096)])
def test_a_chain_of_calls_reads_what_the_call_before_wrote(mc, ref, rows, cols):
    """Launches may start before the one in front of them is done: dequantise into x, take x's scale, quantise x, and again."""
    import torch

    rng = np.random.default_rng(1)
    fmt = "e4m3_16"
    sources, keep = [], []
    for i in range(2):
        code = rng.integers(0, 16, size=(rows, cols)).astype(np.uint8)
        scale = np.full((rows, cols // 16), 0x38 + 8 * i, dtype=np.uint8)
        codes, tiles = (torch.from_numpy(v).cuda() for v in ref.pack(code, scale, fmt))
        keep.append((codes, tiles))
        sources.append(mc.Fp4Matrix(fmt, rows, cols, codes.data_ptr(), tiles.data_ptr()))
    x = torch.zeros(rows, cols, device="cuda")
    codes, scales, sizes = _buffers(mc, fmt, rows, cols, 1)
    g = torch.zeros(40, device="cuda")
    back = torch.zeros(40, rows, cols, device="cuda") if rows < 100 else None
    torch.cuda.synchronize()
    for i in range(40):
        m = mc.Fp4Matrix(fmt, rows, cols, codes.data_ptr(), scales.data_ptr(), g.data_ptr() + 4 * i)
        mc.fp4_dequantize(sources[i % 2], x.data_ptr(), "f32")
        mc.fp4_tensor_scale(x.data_ptr(), "f32", rows, cols, g.data_ptr() + 4 * i)
        mc.fp4_quantize(x.data_ptr(), "f32", m)
        if back is not None:
            mc.fp4_dequantize(m, back.data_ptr() + 4 * i * rows * cols, "f32")
    torch.cuda.synchronize()
    want = [float(np.float32(6.0 * (i + 1) / 2688.0)) for i in range(2)]  # the codes hold a 6, the scales are 1 or 2
    assert g.tolist() == [want[i % 2] for i in range(40)]
    if back is not None:
        for i in range(2):
            assert (back[i::2] == back[i]).all() and not torch.equal(back[0], back[1])


@pytest.mark.gpu
def test_more_values_than_32_bits_count(mc, ref):
    """Rows far behind the 2^31st value: sampled rows against the definition."""
    import torch

    rows, cols = 70000, 33000  # 2.3e9 values of 16 bits
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i in range(0, rows, 10000):
        x[i:i + 10000].normal_(generator=gen)
    codes, scales, sizes = _buffers(mc, "e8m0_32", rows, cols, 1)
    m = mc.Fp4Matrix("e8m0_32", rows, cols, codes.data_ptr(), scales.data_ptr())
    torch.cuda.synchronize()
    mc.fp4_quantize(x.data_ptr(), "bf16", m)
    back = torch.empty_like(x)
    mc.fp4_dequantize(m, back.data_ptr(), "bf16")
    torch.cuda.synchronize()
    for r in (0, 65075, 65076, rows - 1):
        code, scale_bytes = ref.quantize(x[r:r + 1].double().cpu().numpy(), "e8m0_32")
        want_codes, _ = ref.pack(code, scale_bytes, "e8m0_32")
        assert np.array_equal(codes[: sizes.codes_bytes].view(rows, -1)[r].cpu().numpy(), want_codes[0])
        assert np.array_equal(back[r].double().cpu().numpy(), ref.values(code, scale_bytes, "e8m0_32")[0])


def _rounded_once(x, dtype):
    """64-bit x to the nearest f16 or bf16, ties to even, subnormals included; past the end infinity."""
    digits, lowest, most = {"f16": (11, -24, 65504.0), "bf16": (8, -133, float(2 - 2.0 ** -7) * 2.0 ** 127), "f32": (24, -149, float(np.finfo(np.float32).max))}[dtype]
    step = np.exp2(np.maximum(np.frexp(x)[1] - digits, lowest).astype(np.float64))
    r = np.rint(x / step) * step
    return np.where(np.abs(r) > most, np.copysign(np.inf, r), r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("cols", (2016, 2015))
def test_values_read_back_are_rounded_once(mc, ref, dtype, cols):
    """code * scale * g has 6 + 24 bits, which 64-bit numbers hold: what is read back is its nearest, however near a tie it lies."""
    import torch

    rng = np.random.default_rng(8)
    # every code under every scale, for tensor scales of any size
    g = np.exp2(rng.uniform(-24, 3, 60)).astype(np.float32)
    g = np.concatenate([g, np.exp2(rng.uniform(-149, 127, 60)).astype(np.float32), np.float32(1) + np.arange(1, 41).astype(np.float32) * np.float32(2.0 ** -23),
                        np.arange(1, 20, dtype=np.float32) * np.float32(2.0 ** -149), np.float32([2.0 ** -126, 3.4e38])])
    # scales that take a product as near to a tie of the result's type as f32 lets them: the f32 product lies on the tie
    digits, lowest = {"f32": (24, -149), "bf16": (8, -133), "f16": (11, -24)}[dtype]
    exponent = np.concatenate([rng.integers(-10, 11, 150), rng.integers(lowest - 2, lowest + digits, 100)])
    tie = (2.0 ** (digits - 1) + rng.integers(0, 2 ** (digits - 1), 250) + 0.5) * np.exp2(np.maximum(exponent - digits + 1.0, lowest))
    g = np.concatenate([g, (tie / rng.choice([1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875, 2.25, 2.625], 250)).astype(np.float32)])
    g = g[g > 0]
    code = np.tile(np.arange(16, dtype=np.uint8), 126)[None, :cols]
    scale = np.minimum(np.arange(126, dtype=np.uint8), 0x7E)[None]
    codes, tiles = ref.pack(code, scale, "e4m3_16")
    batch = len(g)
    dev = [torch.from_numpy(np.repeat(v[None], batch, axis=0)).cuda() for v in (codes, tiles)] + [torch.from_numpy(g).cuda()]
    m = mc.Fp4Matrix("e4m3_16", 1, cols, dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), batch)
    out = torch.empty(batch, cols, dtype=_torch_dtype(dtype), device="cuda")
    torch.cuda.synchronize()
    mc.fp4_dequantize(m, out.data_ptr(), dtype)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    want = np.stack([_rounded_once(ref.values(code, scale, "e4m3_16", float(v))[0], dtype) for v in g])
    if dtype != "f32":
        twice = np.stack([_rounded_once(_rounded_once(ref.values(code, scale, "e4m3_16", float(v))[0], "f32"), dtype) for v in g])
        assert (twice != want).sum() > 200  # what two roundings would give is told apart
    assert np.array_equal(got, want), int((got != want).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("g", [None, 1.0, -0.37, float("nan"), float("inf"), 0.0, 2.0 ** -149, -(2.0 ** 120)])
def test_reading_back_with_any_tensor_scale_and_nan_blocks(mc, ref, dtype, g):
    """The signs of codes and of g multiply, a NaN scale makes its 16 values NaN, zeros of a block under an infinite g are NaN."""
    import torch

    rng = np.random.default_rng(12)
    rows, cols = 5, 200
    code = rng.integers(0, 16, size=(rows, cols)).astype(np.uint8)
    scale = rng.integers(0, 0x7F, size=(rows, -(-cols // 16))).astype(np.uint8)
    scale[2, 4] = 0x7F
    scale[3, 1] = 0
    codes, tiles = (torch.from_numpy(v).cuda() for v in ref.pack(code, scale, "e4m3_16"))
    tg = torch.tensor([1.0 if g is None else g], dtype=torch.float32, device="cuda")
    m = mc.Fp4Matrix("e4m3_16", rows, cols, codes.data_ptr(), tiles.data_ptr(), 0 if g is None else tg.data_ptr())
    out = torch.empty(rows, cols, dtype=_torch_dtype(dtype), device="cuda")
    torch.cuda.synchronize()
    mc.fp4_dequantize(m, out.data_ptr(), dtype)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        values = ref.values(code, scale, "e4m3_16", float(tg.item()))
        fine = np.isfinite(values)
        want = values.copy()
        want[fine] = _rounded_once(values[fine], dtype)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
