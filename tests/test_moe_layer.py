"""The mixture-of-experts layer against its formula in 64 bits, on the same codes, scales, tokens and router.

The choice of experts and its order have to be equal: logits are sums of exact products in 64 bits, so only logits that
agree to the last bits could differ, and where the tests want ties they are exact. y is held to a bound that follows the
computation: f32 sums of n terms, each addition off by at most 2^-23 relative; silu(g) * u with |silu'| <= 1.1; h rounded
to 11 bits (2^-11 relative, and 2^-40 of the largest in its row: half a step of f16's smallest numbers after the shift);
the weights of the softmax and the joining sum in f32; half a step of y's type."""

import numpy as np
import pytest

FORMATS = ("e8m0_32", "e4m3_16")
STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
U = 2.0 ** -23


@pytest.fixture(scope="module")
def ref():
    from oracle import fp4_reference

    return fp4_reference


# ------------------------------------------------------------------------------------------------- without a GPU


def _layer(mc, **change):
    a = dict(fmt="e8m0_32", experts=8, d=64, f=96, dtype="bf16", tokens=4, top_k=2, x=1 << 24, router=1 << 25, y=1 << 26, rows=None,
             fmt_down=None, experts_down=None, d_down=None, codes=1 << 20, ldx=0, workspace=1 << 27, workspace_bytes=1 << 30, chosen=0, cols=None) | change
    gate_up = mc.Fp4Matrix(a["fmt"], a["rows"] or 2 * a["f"], a["cols"] or a["d"], a["codes"], 1 << 21, 0, a["experts"])
    down = mc.Fp4Matrix(a["fmt_down"] or a["fmt"], a["d_down"] or a["d"], a["f"], 1 << 22, 1 << 23, 0, a["experts_down"] or a["experts"])
    return mc.MoeLayer(gate_up, down, a["x"], a["dtype"], a["router"], a["y"], tokens=a["tokens"], top_k=a["top_k"], ldx=a["ldx"],
                       chosen=a["chosen"], workspace=a["workspace"], workspace_bytes=a["workspace_bytes"])


@pytest.mark.parametrize("change, message", [
    (dict(dtype="f32"), "bf16 or f16"),
    (dict(tokens=0), "1 to 64 tokens"),
    (dict(tokens=65), "1 to 64 tokens"),
    (dict(top_k=0), "top_k is 1 to 8"),
    (dict(top_k=9), "top_k is 1 to 8"),
    (dict(experts=20, top_k=17), "top_k is 1 to 16"),
    (dict(experts=513), "at most 512 experts"),
    (dict(codes=0), "null codes"),
    (dict(codes=(1 << 20) + 8), "16-byte alignment"),
    (dict(rows=190), "2f rows"),
    (dict(rows=193), "2f rows"),
    (dict(d_down=65), r"down's rows \(d\)"),
    (dict(fmt_down="e4m3_16"), "differ in format"),
    (dict(experts_down=7), "different numbers of experts"),
    (dict(x=0), "null x"),
    (dict(router=0), "null x, router"),
    (dict(y=0), "null x, router or y"),
    (dict(y=(1 << 26) + 1), "not aligned to its type"),
    (dict(ldx=63), "leading dimension"),
    (dict(chosen=2), "unaligned chosen"),
    (dict(workspace=0), "bytes of workspace"),
    (dict(workspace_bytes=100), "bytes of workspace"),
    (dict(workspace=(1 << 27) + 8), "16-byte"),
])
def test_wrong_arguments_are_refused(mc, change, message):
    with pytest.raises(mc.McError, match=message):
        _layer(mc, **change).enqueue()


def test_null_arguments_and_workspace_of_refused_sizes(mc):
    lib = mc.lib()
    assert lib.mcd_moe_layer(None, 0) != 0 and b"null arguments" in lib.mcd_last_error()
    assert mc.moe_workspace_bytes(1, 8, 2, 64, 64) > 0
    for sizes in [(0, 8, 2, 64, 64), (65, 8, 2, 64, 64), (1, 0, 2, 64, 64), (1, 8, 17, 64, 64), (1, 8, 2, 0, 64), (1, 8, 2, 64, 0)]:
        assert mc.moe_workspace_bytes(*sizes) == 0


def test_the_workspace_of_every_size_that_the_layer_refuses_is_nothing(mc):
    """The layer's limits are those of its workspace: just inside there is one, just outside there is none."""
    widest = 1 << 24
    for inside, outside in [((1, 512, 2, 64, 64), (1, 513, 2, 64, 64)), ((1, 3, 3, 64, 64), (1, 3, 4, 64, 64)),
                            ((1, 8, 2, widest, 64), (1, 8, 2, widest + 1, 64)), ((1, 8, 2, 64, widest), (1, 8, 2, 64, widest + 1)),
                            ((64, 512, 16, widest, widest), (64, 512, 16, 1 << 62, 1 << 62))]:
        assert mc.moe_workspace_bytes(*inside) > 0 and mc.moe_workspace_bytes(*outside) == 0
    for change, message in [(dict(experts=513), "at most 512 experts"), (dict(experts=3, top_k=4), "top_k is 1 to 3"), (dict(d=widest + 1), "at most 2\\^24")]:
        with pytest.raises(mc.McError, match=message):
            _layer(mc, **change).enqueue()


# ------------------------------------------------------------------------------------------------------ on a GPU


class Problem:
    """Weights, router and tokens on the GPU, and the same numbers in 64 bits."""

    def __init__(self, mc, ref, *, fmt, dtype, tokens, experts, top_k, d, f, renormalize=True, seed=0, sigma=1.0, ldx=None, offset=0,
                 weight_sigma=1.0, x=None, router=None, spoil=None):
        import torch

        self.mc, self.fmt, self.dtype = mc, fmt, dtype
        self.tokens, self.experts, self.top_k, self.d, self.f, self.renormalize = tokens, experts, top_k, d, f, renormalize
        rng = np.random.default_rng(seed)
        t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
        self.t = t
        x = rng.standard_normal((tokens, d)) * sigma if x is None else x
        router = rng.standard_normal((experts, d)) * d ** -0.5 if router is None else router
        x, router = torch.from_numpy(np.asarray(x)).to(t), torch.from_numpy(np.asarray(router)).to(t)
        self.x64, self.router64 = x.double().numpy(), router.double().numpy()
        self.ldx = ldx or d
        self.x = torch.full((offset + tokens * self.ldx + 8,), 5.0, dtype=t, device="cuda")
        self.x_view = self.x[offset:]
        self.x_view[: tokens * self.ldx].view(tokens, self.ldx)[:, :d] = x.cuda()
        self.router = router.cuda()
        self.keep, self.values, self.matrices = [], [], []
        for rows, cols in ((2 * f, d), (d, f)):
            codes, tiles, gs, values = [], [], [], []
            for e in range(experts):
                w = (rng.standard_normal((rows, cols)) * cols ** -0.5 * weight_sigma).astype(np.float32)
                g = ref.tensor_scale(w) if fmt == "e4m3_16" else 1.0
                code, scale = ref.quantize(w, fmt, g)
                if spoil is not None:
                    spoil(len(self.values), e, code, scale)
                c, s = ref.pack(code, scale, fmt)
                codes.append(c), tiles.append(s), gs.append(g), values.append(ref.values(code, scale, fmt, g))
            dev = [torch.from_numpy(np.stack(codes)).cuda(), torch.from_numpy(np.stack(tiles)).cuda(), torch.tensor(gs, dtype=torch.float32, device="cuda")]
            self.keep.append(dev)
            self.values.append(values)
            self.matrices.append(mc.Fp4Matrix(fmt, rows, cols, dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr() if fmt == "e4m3_16" else 0, experts))
        need = mc.moe_workspace_bytes(tokens, experts, top_k, d, f)
        self.need = need
        self.ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        self.ldy = self.ldx
        self.y = torch.full((offset + tokens * self.ldy + 8,), 7.0, dtype=t, device="cuda")
        self.y_view = self.y[offset:]
        self.offset = offset
        self.chosen = torch.full((tokens, top_k), -7, dtype=torch.int32, device="cuda")
        self.weights = torch.full((tokens, top_k), -7.0, device="cuda")
        self.plan = mc.MoeLayer(self.matrices[0], self.matrices[1], self.x_view.data_ptr(), dtype, self.router.data_ptr(), self.y_view.data_ptr(),
                                tokens=tokens, top_k=top_k, renormalize=renormalize, ldx=self.ldx, ldy=self.ldy, chosen=self.chosen.data_ptr(),
                                weights=self.weights.data_ptr(), workspace=self.ws.data_ptr(), workspace_bytes=need)
        torch.cuda.synchronize()

    def run(self, stream=0):
        import torch

        self.plan.enqueue(stream)
        torch.cuda.synchronize()
        return self.result()

    def result(self):
        rows = self.y_view[: self.tokens * self.ldy].view(self.tokens, self.ldy)
        assert (self.y[: self.offset] == 7).all() and (rows[:, self.d:] == 7).all() and (self.y_view[self.tokens * self.ldy:] == 7).all()
        assert (self.ws[self.need:] == 0xFF).all()
        return rows[:, : self.d].double().cpu().numpy()

    def expected(self):
        """(y, bound, chosen, weights) in 64 bits."""
        with np.errstate(all="ignore"):
            return self._expected()

    def _expected(self):
        x = self.x64
        logits = x @ self.router64.T
        chosen = np.stack([np.lexsort((np.arange(self.experts), -np.where(np.isnan(l), -np.inf, l), np.isnan(l)))[: self.top_k] for l in logits])
        p = np.exp(logits - logits.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
        weights = np.take_along_axis(p, chosen, axis=1)
        if self.renormalize:
            weights = weights / weights.sum(axis=1, keepdims=True)
        y, bound = np.zeros((self.tokens, self.d)), np.zeros((self.tokens, self.d))
        d, f = self.d, self.f
        for t in range(self.tokens):
            size = np.zeros(self.d)
            for j in range(self.top_k):
                gu, dn = self.values[0][chosen[t, j]], self.values[1][chosen[t, j]]
                z, z_err = gu @ x[t], (d + 4) * U * (np.abs(gu) @ np.abs(x[t]))
                gate, up = z[:f], z[f:]
                sig = np.where(gate >= 0, 1 / (1 + np.exp(-np.abs(gate))), np.exp(-np.abs(gate)) / (1 + np.exp(-np.abs(gate))))
                h = gate * sig * up
                h_err = 1.1 * z_err[:f] * (np.abs(up) + z_err[f:]) + np.abs(gate * sig) * z_err[f:] + 8 * U * np.abs(h)
                h_err += 2.0 ** -11 * (np.abs(h) + h_err) + 2.0 ** -40 * (np.abs(h) + h_err).max()
                o = dn @ h
                o_size = np.abs(dn) @ (np.abs(h) + h_err)
                o_err = np.abs(dn) @ h_err + (f + 4) * U * o_size
                y[t] += weights[t, j] * o
                # a weight: exp of a rounded difference (|difference| <= 16 in these tests), sum, division
                bound[t] += weights[t, j] * (o_err + 32 * U * np.abs(o))
                size += weights[t, j] * (np.abs(o) + o_err)
            bound[t] += (self.top_k + 8) * U * size
        return y, bound + STEP[self.dtype] * (np.abs(y) + bound) + 2.0 ** -25, chosen, weights

    def check(self, stream=0):
        got = self.run(stream)
        y, bound, chosen, weights = self.expected()
        assert np.array_equal(self.chosen.cpu().numpy(), chosen)
        assert np.allclose(self.weights.double().cpu().numpy(), weights, rtol=64 * U, atol=0)
        assert (np.abs(got - y) <= bound).all(), float((np.abs(got - y) / bound).max())
        # as a whole: the rounding of h and that of y, which are independent of one another
        off = np.linalg.norm(got - y) / np.linalg.norm(y)
        assert off <= STEP[self.dtype] + 2.0 ** -11 + 1e-5
        return got


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("tokens, experts, top_k, d, f", [
    (1, 1, 1, 32, 32), (1, 4, 2, 64, 96), (1, 8, 8, 256, 128), (2, 5, 1, 33, 17), (3, 16, 4, 130, 77), (7, 13, 3, 300, 721), (9, 40, 6, 512, 260),
    (16, 8, 2, 129, 128), (33, 6, 3, 96, 40), (64, 4, 4, 64, 64), (64, 64, 16, 96, 48), (1, 512, 16, 40, 24), (5, 8, 2, 1100, 1300),
    (40, 100, 6, 200, 260), (64, 90, 12, 97, 770), (21, 200, 9, 540, 390), (20, 12, 5, 300, 200), (9, 40, 6, 1100, 260), (6, 30, 5, 1024, 300),
    (3, 63, 8, 448, 700), (37, 40, 8, 1030, 140),
])
def test_layer(mc, ref, fmt, dtype, tokens, experts, top_k, d, f):
    Problem(mc, ref, fmt=fmt, dtype=dtype, tokens=tokens, experts=experts, top_k=top_k, d=d, f=f, renormalize=tokens % 2 == 1, seed=d + f).check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("ldx, offset", [(100, 1), (104, 8), (97, 0)])
def test_strides_and_alignment(mc, ref, dtype, ldx, offset):
    Problem(mc, ref, fmt="e8m0_32", dtype=dtype, tokens=5, experts=6, top_k=2, d=97, f=50, ldx=ldx, offset=offset).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("sigma, weight_sigma", [(2.0 ** 60, 1.0), (2.0 ** -60, 1.0), (1.0, 2.0 ** 40), (1.0, 2.0 ** -40), (2.0 ** -100, 2.0 ** 50)])
def test_values_far_from_one(mc, ref, fmt, sigma, weight_sigma):
    """bf16 reaches further than the 11-bit fragments: the shifts bring every magnitude into their range."""
    rng = np.random.default_rng(3)
    d = 96
    router = rng.standard_normal((6, d)) * d ** -0.5 / sigma
    p = Problem(mc, ref, fmt=fmt, dtype="bf16", tokens=4, experts=6, top_k=2, d=d, f=64, sigma=sigma, weight_sigma=weight_sigma, router=router)
    got = p.run()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen)
    fine = np.abs(y) < 2.0 ** 127
    # below 2^-126 f32 sums lose their relative precision
    assert (np.abs(got - y) <= bound + 2.0 ** -120)[fine].all()


@pytest.mark.gpu
def test_ties_take_the_lowest_index(mc, ref):
    tokens, experts, d = 3, 70, 64
    router = np.zeros((experts, d))
    router[10:] = 1.0 / 64  # experts 10 .. 69 are equal, 0 .. 9 lower for positive x
    x = np.ones((tokens, d))
    x[1] = -1.0   # 0 .. 9 win, all equal
    x[2] = 0.0    # every expert equal
    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=tokens, experts=experts, top_k=4, d=d, f=32, x=x, router=router)
    p.run()
    assert p.chosen.cpu().tolist() == [[10, 11, 12, 13], [0, 1, 2, 3], [0, 1, 2, 3]]
    assert np.array_equal(p.weights.cpu().numpy(), np.full((tokens, 4), 0.25, dtype=np.float32))
    assert (p.result()[2] == 0).all()


@pytest.mark.gpu
def test_every_token_to_the_same_experts(mc, ref):
    rng = np.random.default_rng(1)
    d = 128
    x = np.abs(rng.standard_normal((64, d))) + 0.1
    router = np.zeros((20, d))
    router[17], router[3] = 0.05, 0.04
    p = Problem(mc, ref, fmt="e4m3_16", dtype="bf16", tokens=64, experts=20, top_k=2, d=d, f=160, x=x, router=router)
    p.check()
    assert (p.chosen.cpu().numpy() == [17, 3]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf")))
def test_a_token_that_is_not_finite_stays_alone(mc, ref, bad):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((5, 80))
    x[2, 7] = bad
    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=5, experts=9, top_k=3, d=80, f=48, x=x)
    got = p.run()
    y, bound, chosen, _ = p.expected()
    rest = [0, 1, 3, 4]
    assert np.isnan(got[2]).all()
    assert np.array_equal(p.chosen.cpu().numpy()[rest], chosen[rest])
    assert sorted(set(p.chosen.cpu().numpy()[2])) == sorted(p.chosen.cpu().numpy()[2])  # still experts, each once
    assert (np.abs(got - y) <= bound)[rest].all()
    if np.isnan(bad):
        assert p.chosen.cpu().tolist()[2] == [0, 1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("which", (0, 1))
def test_a_nan_scale_reaches_the_tokens_of_its_expert(mc, ref, fmt, which):
    def spoil(matrix, expert, code, scale):
        if matrix == which and expert == 2:
            scale[5, 0] = 255 if fmt == "e8m0_32" else 0x7F

    p = Problem(mc, ref, fmt=fmt, dtype="bf16", tokens=12, experts=6, top_k=2, d=64, f=48, spoil=spoil)
    got = p.run()
    hit = (p.chosen.cpu().numpy() == 2).any(axis=1)
    assert hit.any() and not hit.all()
    assert np.isfinite(got[~hit]).all()
    y, bound, _, _ = p.expected()
    assert (np.abs(got - y) <= bound)[~hit].all()
    if which == 0:
        assert np.isnan(got[hit]).all()  # one h of the expert is NaN
    else:
        assert np.isnan(got[hit][:, 5]).all() and np.isfinite(np.delete(got[hit], 5, axis=1)).all()


@pytest.mark.gpu
def test_the_same_bits_every_time_and_in_a_replayed_graph(mc, ref):
    import torch

    p = Problem(mc, ref, fmt="e4m3_16", dtype="bf16", tokens=24, experts=10, top_k=4, d=256, f=192)
    first = p.check()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        p.plan.enqueue(side.cuda_stream)
        p.plan.enqueue(side.cuda_stream)
    for _ in range(3):
        p.y_view[: p.tokens * p.d].fill_(float("nan"))
        p.ws[: p.need].fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(p.result(), first)
    # other tokens through the same captured call
    rng = np.random.default_rng(77)
    x = torch.from_numpy(rng.standard_normal((24, 256))).to(p.t)
    p.x_view[: 24 * 256].view(24, 256).copy_(x)
    p.x64 = x.double().numpy()
    graph.replay()
    torch.cuda.synchronize()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen) and (np.abs(p.result() - y) <= bound).all()


@pytest.mark.gpu
def test_two_streams_and_without_the_optional_results(mc, ref):
    import torch

    problems = [Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=n, experts=12, top_k=3, d=160, f=96, seed=n) for n in (2, 11)]
    streams = [torch.cuda.Stream() for _ in problems]
    for p in problems:
        p.plan = mc.MoeLayer(p.matrices[0], p.matrices[1], p.x_view.data_ptr(), "bf16", p.router.data_ptr(), p.y_view.data_ptr(), tokens=p.tokens, top_k=3,
                             workspace=p.ws.data_ptr(), workspace_bytes=p.need)
    for _ in range(20):
        for p, s in zip(problems, streams):
            p.plan.enqueue(s.cuda_stream)
    torch.cuda.synchronize()
    for p in problems:
        y, bound, _, _ = p.expected()
        assert (np.abs(p.result() - y) <= bound).all()
        assert (p.chosen == -7).all()


@pytest.mark.gpu
def test_experts_quantised_by_the_library_in_one_call(mc, ref):
    """The run of a program: stacked weights -> tensor scales -> codes, then layers on tokens, one call's y the next one's x."""
    import torch

    fmt, experts, d, f, tokens = "e4m3_16", 6, 160, 96, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    matrices, keep, values = [], [], []
    for rows, cols in ((2 * f, d), (d, f)):
        w = (torch.randn(experts, rows, cols, generator=gen, device="cuda") * cols ** -0.5).to(torch.bfloat16)
        s = mc.fp4_sizes(fmt, rows, cols, experts)
        codes, scales = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in (s.codes_bytes, s.scales_bytes))
        g = torch.empty(experts, device="cuda")
        m = mc.Fp4Matrix(fmt, rows, cols, codes.data_ptr(), scales.data_ptr(), g.data_ptr(), experts)
        mc.fp4_tensor_scale(w.data_ptr(), "bf16", rows, cols, g.data_ptr(), batch=experts)
        mc.fp4_quantize(w.data_ptr(), "bf16", m)
        matrices.append(m), keep.append((w, codes, scales, g))
        torch.cuda.synchronize()
        wh = w.double().cpu().numpy()
        values.append([ref.values(*ref.quantize(wh[e], fmt, ref.tensor_scale(wh[e])), fmt, ref.tensor_scale(wh[e])) for e in range(experts)])
    p = Problem(mc, ref, fmt=fmt, dtype="bf16", tokens=tokens, experts=experts, top_k=2, d=d, f=f)
    p.values = values
    for _ in range(3):
        p.plan = mc.MoeLayer(matrices[0], matrices[1], p.x_view.data_ptr(), "bf16", p.router.data_ptr(), p.y_view.data_ptr(), tokens=tokens, top_k=2,
                             chosen=p.chosen.data_ptr(), weights=p.weights.data_ptr(), workspace=p.ws.data_ptr(), workspace_bytes=p.need)
        got = p.check()
        p.x_view[: tokens * d].view(tokens, d).copy_(torch.from_numpy(got * 3).to(torch.bfloat16))
        p.x64 = torch.from_numpy(got * 3).to(torch.bfloat16).double().numpy()


@pytest.mark.gpu
def test_host_memory_is_refused(mc, ref):
    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=1, experts=4, top_k=1, d=64, f=32)
    host = np.zeros(64, dtype=np.uint16)
    p.plan._args.x = host.ctypes.data
    with pytest.raises(mc.McError, match="not device memory"):
        p.plan.enqueue()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts, top_k, d, launches", [(1, 8, 2, 64, 3), (16, 8, 2, 64, 3), (17, 8, 2, 64, 4), (6, 30, 5, 1024, 4), (6, 30, 5, 1025, 3), (64, 40, 8, 64, 4)])
def test_three_launches_or_four(mc, ref, tokens, experts, top_k, d, launches):
    """Three for up to 32 slots; a fourth levels h where there are more, or where few rows of y meet 24 experts."""
    import torch

    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=tokens, experts=experts, top_k=top_k, d=d, f=32)
    torch.cuda.synchronize()
    before = mc.lib().mcd_launch_count()
    p.plan.enqueue()
    counted = mc.lib().mcd_launch_count() - before
    torch.cuda.synchronize()
    assert counted == launches
