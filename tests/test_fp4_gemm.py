"""The product of two microscaled 4-bit matrices against 64-bit sums of the numbers that they stand for.

Two kinds of data. "Exact": scales of few bits, so that every product is a multiple of 2^-8 and every partial sum below
2^15, which f32 holds without rounding in any order: the result has to be equal. "Normal": scales as quantising normal
values gives them; a sum of k terms in f32, in any order and with each addition off by at most 2^-23 relative (truncation),
is off by at most k 2^-23 sum|a b|, the tensor scales add two roundings, the result's type half a step."""

import numpy as np
import pytest

FORMATS = ("e8m0_32", "e4m3_16")
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def ref():
    from oracle import fp4_reference

    return fp4_reference


# ------------------------------------------------------------------------------------------------- without a GPU


def _plan(mc, change=None, fmt_b=None, k_b=None, **gemm):
    a = dict(fmt="e8m0_32", rows=300, cols=512, codes=1 << 20, scales=1 << 21) | (change or {})
    b = dict(fmt=fmt_b or "e8m0_32", rows=200, cols=k_b or 512, codes=1 << 22, scales=1 << 23)
    A = mc.Fp4Matrix(a["fmt"], a["rows"], a["cols"], a["codes"], a["scales"], a.get("g", 0), a.get("batch", 1))
    B = mc.Fp4Matrix(b["fmt"], b["rows"], b["cols"], b["codes"], b["scales"])
    g = dict(c=1 << 24, c_dtype="bf16") | gemm
    return mc.Fp4Gemm(A, B, **g)


@pytest.mark.parametrize("kw, message", [
    (dict(change=dict(rows=0)), "empty matrix"),
    (dict(change=dict(codes=0)), "null codes"),
    (dict(change=dict(scales=(1 << 20) + 8)), "16-byte alignment"),
    (dict(change=dict(batch=2)), "single matrices"),
    (dict(fmt_b="e4m3_16"), "formats differ"),
    (dict(k_b=544), r"columns \(k\) differ"),
    (dict(c=0), "no output buffer"),
    (dict(c=(1 << 24) + 1), "not aligned to its type"),
    (dict(c=(1 << 24) + 2, c_dtype="f32"), "not aligned to its type"),
    (dict(ldc=199), "ldc is less"),
    (dict(status=3), "unaligned status"),
])
def test_wrong_arguments_are_refused(mc, kw, message):
    with pytest.raises(mc.McError, match=message):
        _plan(mc, **kw).enqueue()


def test_a_missing_or_short_workspace_is_refused(mc):
    need = mc.fp4_gemm_workspace_bytes("e8m0_32", 1, 256, 70016)
    assert need > 0
    A = mc.Fp4Matrix("e8m0_32", 1, 70016, 1 << 20, 1 << 21)
    B = mc.Fp4Matrix("e8m0_32", 256, 70016, 1 << 22, 1 << 23)
    for workspace, size, message in [(0, need, "bytes of workspace"), (1 << 25, need - 1, "bytes of workspace"), ((1 << 25) + 4, need, "16-byte")]:
        with pytest.raises(mc.McError, match=message):
            mc.Fp4Gemm(A, B, 1 << 24, "f32", workspace=workspace, workspace_bytes=size).enqueue()
    lib = mc.lib()
    assert lib.mcd_fp4_gemm(None, 0) != 0 and b"null arguments" in lib.mcd_last_error()
    assert lib.mcd_fp4_gemm_workspace(None) == 0


# ------------------------------------------------------------------------------------------------------ on a GPU


class Operand:
    def __init__(self, mc, ref, code, scale, fmt, g=None):
        import torch

        codes, tiles = ref.pack(code, scale, fmt)
        self.codes, self.tiles = torch.from_numpy(codes).cuda(), torch.from_numpy(tiles).cuda()
        self.g = None if g is None else torch.tensor([g], dtype=torch.float32, device="cuda")
        self.m = mc.Fp4Matrix(fmt, code.shape[0], code.shape[1], self.codes.data_ptr(), self.tiles.data_ptr(),
                              0 if g is None else self.g.data_ptr())
        self.values = ref.values(code, scale, fmt, 1.0 if g is None else float(np.float32(g)))


def _exact_operand(mc, ref, rng, rows, k, fmt):
    code = rng.integers(0, 16, size=(rows, k)).astype(np.uint8)
    blocks = -(-k // ref.BLOCK[fmt])
    choices = [126, 127, 128] if fmt == "e8m0_32" else [0x30, 0x34, 0x36, 0x38, 0x3A, 0x3C]  # 0.5 .. 1.5 in steps of 0.125
    return Operand(mc, ref, code, rng.choice(choices, size=(rows, blocks)).astype(np.uint8), fmt)


def _product(mc, a, b, dtype, ldc=None, offset=0, stream=0):
    """The product into a buffer of 7s: (result in 64 bits, whether everything around it was left alone)."""
    import torch

    m, n, k = a.m.rows, b.m.rows, a.m.cols
    ldc = ldc or n
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    buf = torch.full((offset + m * ldc + 64,), 7.0, dtype=t, device="cuda")
    need = mc.fp4_gemm_workspace_bytes(a.m.format, m, n, k)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")  # NaNs: what is read of it has to be written first
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    c = buf[offset:]
    plan = mc.Fp4Gemm(a.m, b.m, c.data_ptr(), dtype, ldc=ldc, workspace=ws.data_ptr(), workspace_bytes=need, status=status.data_ptr())
    plan.enqueue(stream)
    torch.cuda.synchronize()
    assert status.item() == 0
    rows = c[: m * ldc].view(m, ldc)
    around = bool((buf[:offset] == 7).all() and (rows[:, n:] == 7).all() and (c[m * ldc:] == 7).all() and (ws[need:] == 0xFF).all())
    return rows[:, :n].double().cpu().numpy(), around


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m, n, k", [
    (1, 1, 1), (1, 8, 31), (1, 128, 64), (2, 130, 65), (16, 128, 256), (17, 257, 257), (33, 64, 300), (64, 200, 96), (65, 129, 512),
    (128, 128, 128), (128, 300, 1000), (129, 128, 256), (200, 70, 33), (256, 256, 768), (300, 513, 321), (1, 300, 4096), (40, 100, 5000),
    (513, 256, 1024), (512, 512, 2080), (700, 900, 640), (2100, 1300, 700), (1600, 1600, 2304), (10000, 257, 64), (2305, 2304, 1), (3000, 1, 128), (1000, 16, 3100), (700, 100, 257), (513, 128, 2048), (128, 128, 4096), (3, 200, 66000), (70, 650, 66000), (90, 16, 33000), (100, 4300, 1700), (5000, 120, 1100), (17, 2000, 2100), (5, 9000, 2048), (70, 1030, 4100), (1200, 20, 9000), (20, 1201, 9000), (300, 513, 6200), (200, 1000, 7777), (1000, 700, 8200), (1500, 1600, 6500),
    (257, 8100, 6145),
])
def test_exact_data_gives_equal_results(mc, ref, fmt, m, n, k):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    a, b = _exact_operand(mc, ref, rng, m, k, fmt), _exact_operand(mc, ref, rng, n, k, fmt)
    want = a.values @ b.values.T
    got, around = _product(mc, a, b, "f32")
    assert around
    assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("m, n, k", [(1, 512, 2048), (5, 130, 777), (100, 256, 1024), (150, 300, 4096), (1024, 640, 512), (1537, 1800, 1500)])
def test_normal_data_within_the_bound(mc, ref, fmt, dtype, m, n, k):
    rng = np.random.default_rng(k)
    operands, bound = [], []
    for rows, sigma in ((m, 1.0), (n, k ** -0.5)):
        x = (rng.standard_normal((rows, k)) * sigma).astype(np.float32)
        g = ref.tensor_scale(x) if fmt == "e4m3_16" else None
        code, scale = ref.quantize(x, fmt, 1.0 if g is None else g)
        operands.append(Operand(mc, ref, code, scale, fmt, g))
        bound.append(np.abs(operands[-1].values))
    a, b = operands
    want = a.values @ b.values.T
    got, around = _product(mc, a, b, dtype)
    assert around
    sums = bound[0] @ bound[1].T
    allowed = (k + 2) * 2.0 ** -23 * sums + STEP[dtype] * (np.abs(want) + k * 2.0 ** -23 * sums) + 2.0 ** -25
    assert (np.abs(got - want) <= allowed).all()
    # far inside the bound as a whole: errors of a sum's roundings are not all of one sign
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= STEP[dtype] + k * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("f32", "bf16"))
@pytest.mark.parametrize("m, n, ldc, offset", [(20, 100, 101, 1), (20, 100, 104, 8), (200, 100, 131, 3), (300, 256, 264, 16), (200, 128, 128, 1), (2100, 1300, 1301, 1),
                                               (2100, 1300, 1304, 16), (2100, 1300, 1304, 1), (1537, 1285, 1286, 2),
                                               (1537, 1285, 1285, 0), (1537, 1285, 1286, 3), (700, 1100, 1104, 8)])
def test_only_c_is_written(mc, ref, dtype, m, n, ldc, offset):
    rng = np.random.default_rng(ldc)
    a, b = _exact_operand(mc, ref, rng, m, 96, "e8m0_32"), _exact_operand(mc, ref, rng, n, 96, "e8m0_32")
    got, around = _product(mc, a, b, dtype, ldc=ldc, offset=offset)
    assert around
    want = a.values @ b.values.T
    assert (np.abs(got - want) <= (0 if dtype == "f32" else STEP[dtype]) * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("m, n, ldc, offset", [(20, 300, 301, 1), (20, 300, 304, 8), (300, 20, 21, 1), (300, 500, 501, 1), (300, 500, 504, 8), (300, 501, 504, 16),
                                               (300, 500, 502, 2), (257, 4100, 4103, 3)])
def test_slices_of_k_write_c_and_nothing_else(mc, ref, dtype, m, n, ldc, offset):
    rng = np.random.default_rng(ldc)
    a, b = _exact_operand(mc, ref, rng, m, 6200, "e8m0_32"), _exact_operand(mc, ref, rng, n, 6200, "e8m0_32")
    got, around = _product(mc, a, b, dtype, ldc=ldc, offset=offset)
    assert around
    want = a.values @ b.values.T
    assert (np.abs(got - want) <= (0 if dtype == "f32" else STEP[dtype]) * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m, n", [(5, 40), (200, 300)])
def test_a_nan_scale_reaches_its_row_and_no_other(mc, ref, fmt, m, n):
    rng = np.random.default_rng(4)
    k = 200
    code = rng.integers(0, 16, size=(m, k)).astype(np.uint8)
    scale = np.full((m, -(-k // ref.BLOCK[fmt])), 127 if fmt == "e8m0_32" else 0x38, dtype=np.uint8)
    code[3, : ref.BLOCK[fmt]] = 0
    scale[3, 0] = 255 if fmt == "e8m0_32" else 0x7F
    a, b = Operand(mc, ref, code, scale, fmt), _exact_operand(mc, ref, rng, n, k, fmt)
    got, _ = _product(mc, a, b, "f32")
    assert np.isnan(got[3]).all()
    want = np.delete(a.values, 3, axis=0) @ b.values.T
    assert np.array_equal(np.delete(got, 3, axis=0), want)


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(3, 256, 8192), (3, 256, 70000), (100, 1300, 2600), (700, 600, 512), (300, 600, 7000)])
def test_the_same_bits_every_time_and_in_a_replayed_graph(mc, ref, m, n, k):
    import torch

    rng = np.random.default_rng(8)
    x, w = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((n, k)).astype(np.float32)
    a, b = (Operand(mc, ref, *ref.quantize(v, "e4m3_16", 1.0), "e4m3_16") for v in (x, w))
    first, _ = _product(mc, a, b, "f32")
    second, _ = _product(mc, a, b, "f32")
    assert np.array_equal(first, second)
    need = mc.fp4_gemm_workspace_bytes("e4m3_16", m, n, k)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    c = torch.zeros(m, n, device="cuda")
    plan = mc.Fp4Gemm(a.m, b.m, c.data_ptr(), "f32", workspace=ws.data_ptr(), workspace_bytes=need)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan.enqueue(side.cuda_stream)
        plan.enqueue(side.cuda_stream)
    for _ in range(2):
        c.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.double().cpu().numpy(), first)
    assert plan.launches in (1, 2)


@pytest.mark.gpu
def test_two_streams_with_a_workspace_each(mc, ref):
    import torch

    rng = np.random.default_rng(11)
    problems = []
    for m, n, k in ((4, 384, 80000), (9, 256, 70000)):
        a, b = _exact_operand(mc, ref, rng, m, k, "e8m0_32"), _exact_operand(mc, ref, rng, n, k, "e8m0_32")
        need = mc.fp4_gemm_workspace_bytes("e8m0_32", m, n, k)
        assert need > 0
        ws, c = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty(m, n, device="cuda")
        plan = mc.Fp4Gemm(a.m, b.m, c.data_ptr(), "f32", workspace=ws.data_ptr(), workspace_bytes=need)
        problems.append((plan, torch.cuda.Stream(), a, b, c, ws))
    torch.cuda.synchronize()
    for _ in range(20):
        for plan, stream, *_ in problems:
            plan.enqueue(stream.cuda_stream)
    torch.cuda.synchronize()
    for _, _, a, b, c, _ in problems:
        assert np.array_equal(c.double().cpu().numpy(), a.values @ b.values.T)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", (1, 48, 300))
def test_two_layers_as_a_program_runs_them(mc, ref, fmt, tokens):
    """Weights quantised once; per call: quantise activations, product, quantise the result, product."""
    import torch

    rng = np.random.default_rng(tokens)
    widths = (320, 512, 192)
    x = torch.from_numpy(rng.standard_normal((tokens, widths[0]))).to(torch.bfloat16).cuda()
    keep = []

    def held(rows, cols):
        s = mc.fp4_sizes(fmt, rows, cols)
        t = [torch.empty(s.codes_bytes, dtype=torch.uint8, device="cuda"), torch.empty(s.scales_bytes, dtype=torch.uint8, device="cuda"),
             torch.empty(1, device="cuda")]
        keep.append(t)
        return mc.Fp4Matrix(fmt, rows, cols, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr() if fmt == "e4m3_16" else 0), t[2]

    def quantize(src, rows, cols):
        m, g = held(rows, cols)
        if fmt == "e4m3_16":
            mc.fp4_tensor_scale(src.data_ptr(), "bf16", rows, cols, g.data_ptr())
        mc.fp4_quantize(src.data_ptr(), "bf16", m)
        return m

    value, matrix = x.double().cpu().numpy(), quantize(x, tokens, widths[0])
    for k, n in zip(widths, widths[1:]):
        w = torch.from_numpy(rng.standard_normal((n, k)) * k ** -0.5).to(torch.bfloat16).cuda()
        wm = quantize(w, n, k)
        c = torch.empty(tokens, n, dtype=torch.bfloat16, device="cuda")
        need = mc.fp4_gemm_workspace_bytes(fmt, tokens, n, k)
        ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
        keep.append((w, c, ws))
        mc.Fp4Gemm(matrix, wm, c.data_ptr(), "bf16", workspace=ws.data_ptr(), workspace_bytes=need).enqueue()
        torch.cuda.synchronize()

        def stands_for(v):
            g = ref.tensor_scale(v) if fmt == "e4m3_16" else 1.0
            return ref.values(*ref.quantize(v, fmt, g), fmt, g)

        left, right = stands_for(value), stands_for(w.double().cpu().numpy())
        want, sums = left @ right.T, np.abs(left) @ np.abs(right).T
        got = c.double().cpu().numpy()
        assert (np.abs(got - want) <= (k + 2) * 2.0 ** -23 * sums * 1.01 + 2.0 ** -8 * np.abs(want)).all()
        # the next layer starts from what the GPU computed
        value, matrix = got, quantize(c, tokens, n)


@pytest.mark.gpu
def test_host_memory_is_refused(mc):
    import torch

    host = np.zeros(1 << 16, dtype=np.uint8)
    base = (host.ctypes.data + 15) // 16 * 16
    dev = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    a, b = (mc.Fp4Matrix("e8m0_32", 4, 64, p, dev.data_ptr() + 8192) for p in (base, dev.data_ptr()))
    with pytest.raises(mc.McError, match="not device memory"):
        mc.Fp4Gemm(a, b, dev.data_ptr() + 32768, "f32").enqueue()
    torch.cuda.synchronize()


def _far_operand(mc, ref, rng, rows, k, byte, g, zero=None):
    """Codes under one block scale and a tensor scale g; row `zero` has codes 0."""
    code = rng.integers(0, 16, size=(rows, k)).astype(np.uint8)
    if zero is not None:
        code[zero] = 0
    return Operand(mc, ref, code, np.full((rows, -(-k // 16)), byte, dtype=np.uint8), "e4m3_16", g)


# one CTA per tile whole, in a cluster, through the workspace; SM pairs whole and in slices
FORMS = [(5, 40, 200), (3, 256, 8192), (3, 256, 66000), (300, 513, 321), (300, 501, 6400)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", FORMS)
@pytest.mark.parametrize("ga, gb, byte", [(2.0 ** -75, 2.0 ** -75, 0x78), (2.0 ** -120, 2.0 ** -20, 0x78), (2.0 ** 64, 2.0 ** 64, 0x01), (2.0 ** 100, 2.0 ** 35, 0x01),
                                          (2.0 ** -100, 2.0 ** 100, 0x38), (2.0 ** 100, 2.0 ** -100, 0x38), (2.0 ** -130, 2.0 ** 5, 0x78)])
def test_tensor_scales_whose_product_leaves_f32(mc, ref, m, n, k, ga, gb, byte):
    """Powers of two, and sums that f32 holds exactly: so does C, although g_a g_b need not. 0x78 is 2^8, 0x01 2^-9."""
    rng = np.random.default_rng(k)
    a, b = _far_operand(mc, ref, rng, m, k, byte, ga, zero=1), _far_operand(mc, ref, rng, n, k, byte, gb)
    want = a.values @ b.values.T
    want = np.where(np.abs(want) < 2.0 ** 128, want, np.copysign(np.inf, want))
    assert np.isfinite(want).any() and np.count_nonzero(want) > want.size / 2
    got, around = _product(mc, a, b, "f32")
    assert around
    assert np.array_equal(got, want)
    assert (got[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", FORMS)
@pytest.mark.parametrize("ga, gb, byte", [(1.37 * 2.0 ** -70, 1.71 * 2.0 ** -70, 0x78), (1.9 * 2.0 ** -118, 1.3 * 2.0 ** -20, 0x78)])
def test_tensor_scales_whose_product_is_subnormal(mc, ref, m, n, k, ga, gb, byte):
    """The sums are exact; each scale is a rounding of 2^-24, and where C is subnormal one of half of f32's smallest number."""
    rng = np.random.default_rng(k + 1)
    a, b = _far_operand(mc, ref, rng, m, k, byte, ga), _far_operand(mc, ref, rng, n, k, byte, gb)
    want = a.values @ b.values.T
    got, _ = _product(mc, a, b, "f32")
    assert (np.abs(got - want) <= 2.01 * 2.0 ** -24 * np.abs(want) + 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k, launches", [(5, 40, 200, 1), (3, 256, 8192, 1), (3, 256, 70000, 2), (300, 513, 321, 1), (300, 501, 6400, 1)])
def test_the_launches_that_the_plan_says(mc, ref, m, n, k, launches):
    """Whole, in clusters, through the workspace, pairs, pairs in slices: what is said beforehand is what was counted."""
    import torch

    rng = np.random.default_rng(3)
    a, b = _exact_operand(mc, ref, rng, m, k, "e8m0_32"), _exact_operand(mc, ref, rng, n, k, "e8m0_32")
    need = mc.fp4_gemm_workspace_bytes("e8m0_32", m, n, k)
    assert (need > 0) == (launches == 2)
    ws, c = torch.empty(max(16, need), dtype=torch.uint8, device="cuda"), torch.empty(m, n, device="cuda")
    plan = mc.Fp4Gemm(a.m, b.m, c.data_ptr(), "f32", workspace=ws.data_ptr(), workspace_bytes=need)
    torch.cuda.synchronize()
    before = mc.lib().mcd_launch_count()
    plan.enqueue()
    counted = mc.lib().mcd_launch_count() - before
    torch.cuda.synchronize()
    assert plan.launches == launches == counted


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", FORMS)
def test_a_nan_tensor_scale_makes_all_of_c_nan(mc, ref, m, n, k):
    rng = np.random.default_rng(1)
    for scales in ((float("nan"), 2.0 ** 5), (2.0 ** -100, float("nan"))):
        a, b = (_far_operand(mc, ref, rng, rows, k, 0x38, g) for rows, g in zip((m, n), scales))
        got, around = _product(mc, a, b, "bf16")
        assert around and np.isnan(got).all()
