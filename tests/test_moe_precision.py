"""How exact the mixture-of-experts layer is, where the coarse bounds of test_moe_layer.py would not show it.

h = silu(G x) * (U x) enters the down projection as two f16 numbers: hi, its nearest, and what hi leaves, rounded in turn:
22 bits, 2^-22 of a value, and not less than 2^-36 after the shift that takes the largest of a token and expert to
[2^14, 2^15), 2^-50 of that one. The rest is f32: sums of n terms off by n 2^-23 of their terms' magnitudes, silu by 8 steps."""

import numpy as np
import pytest

from test_moe_layer import FORMATS, STEP, U, Problem, ref  # noqa: F401  (ref: the fixture)


class Tight(Problem):
    """The same layer held to a bound in which h has 22 bits."""

    def _expected(self):
        x, d, f = self.x64, self.d, self.f
        logits = x @ self.router64.T
        chosen = np.stack([np.lexsort((np.arange(self.experts), -l))[: self.top_k] for l in logits])
        p = np.exp(logits - logits.max(axis=1, keepdims=True))
        weights = np.take_along_axis(p / p.sum(axis=1, keepdims=True), chosen, axis=1)
        if self.renormalize:
            weights = weights / weights.sum(axis=1, keepdims=True)
        y, bound = np.zeros((self.tokens, d)), np.zeros((self.tokens, d))
        for t in range(self.tokens):
            size = np.zeros(d)
            for j in range(self.top_k):
                gu, dn = self.values[0][chosen[t, j]], self.values[1][chosen[t, j]]
                z, z_err = gu @ x[t], (d + 4) * U * (np.abs(gu) @ np.abs(x[t]))
                gate, up = z[:f], z[f:]
                small = np.exp(-np.abs(gate))
                sig = np.where(gate >= 0, 1, small) / (1 + small)
                h = gate * sig * up
                h_err = 1.1 * z_err[:f] * (np.abs(up) + z_err[f:]) + np.abs(gate * sig) * z_err[f:] + 8 * U * np.abs(h)
                h_err += 2.0 ** -22 * (np.abs(h) + h_err) + 2.0 ** -50 * (np.abs(h) + h_err).max()
                o, o_size = dn @ h, np.abs(dn) @ (np.abs(h) + h_err)
                o_err = np.abs(dn) @ h_err + (2 * f + 4) * U * o_size  # twice the terms: hi and what it leaves
                y[t] += weights[t, j] * o
                bound[t] += weights[t, j] * (o_err + 32 * U * np.abs(o))
                size += weights[t, j] * (np.abs(o) + o_err)
            bound[t] += (self.top_k + 8) * U * size
        smallest = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}[self.dtype]  # half a step of the subnormal numbers
        return y, bound + STEP[self.dtype] * (np.abs(y) + bound) + smallest, chosen, weights


def _differences(f, d, fmt, seed):
    """A `spoil` that makes a down projection's row the difference of two of h's values: codes 1 and -1 under scales of 1.

    The values are of like size, so what is left of them shows how many bits they had."""
    rng = np.random.default_rng(seed)
    pairs = np.stack([rng.permutation(f)[:2] for _ in range(d)])

    def spoil(matrix, expert, code, scale):
        if matrix == 1:
            code[:] = 0
            code[np.arange(d), pairs[:, 0]] = 2
            code[np.arange(d), pairs[:, 1]] = 10
            scale[:] = 127 if fmt == "e8m0_32" else 0x38
        else:
            # rows of U repeat those of G, and all rows are nearly one another's: h's values lie close together
            code[f:] = code[:f]
            scale[f:] = scale[:f]
            code[:] = code[0]
            scale[:] = scale[0]
            flip = rng.integers(0, code.shape[1], size=2 * f)
            code[np.arange(2 * f), flip] = (code[np.arange(2 * f), flip] + 1) % 8

    return spoil


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("tokens, experts, top_k, d, f", [(1, 1, 1, 64, 40), (1, 6, 2, 48, 300), (5, 7, 3, 96, 33), (9, 2, 1, 64, 48), (20, 4, 2, 1100, 72),
                                                          (40, 30, 5, 64, 140), (64, 3, 3, 80, 64)])
def test_h_has_more_bits_than_f16(mc, ref, fmt, dtype, tokens, experts, top_k, d, f):  # noqa: F811
    p = Tight(mc, ref, fmt=fmt, dtype=dtype, tokens=tokens, experts=experts, top_k=top_k, d=d, f=f, seed=d, spoil=_differences(f, d, fmt, 5))
    got = p.run()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen)
    assert (np.abs(got - y) <= bound).all(), float((np.abs(got - y) / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens, experts, top_k, d, f", [(1, 4, 2, 640, 96), (7, 13, 3, 300, 721), (64, 4, 4, 64, 64), (33, 6, 3, 96, 40), (40, 100, 6, 200, 260),
                                                          (20, 12, 5, 300, 200), (9, 40, 6, 1100, 260), (64, 90, 12, 97, 770)])
def test_the_layer_is_as_exact_as_its_result_type(mc, ref, fmt, tokens, experts, top_k, d, f):  # noqa: F811
    """In the norm the error is that of rounding y alone. An error spread evenly over half a step 2^-11 of a binade has the mean
    square 2^-22 / 3; over mantissas m of density 1 / m the mean of m^2 is 1.5 / ln 2. A third on top for the sample's spread."""
    p = Tight(mc, ref, fmt=fmt, dtype="f16", tokens=tokens, experts=experts, top_k=top_k, d=d, f=f, seed=f)
    got = p.run()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen)
    assert (np.abs(got - y) <= bound).all()
    assert np.linalg.norm(got - y) <= 1.3 * STEP["f16"] * (np.log(2) / 4.5) ** 0.5 * np.linalg.norm(y)


def _silu_problem(mc, ref, gates, up_exponent):
    """One expert whose h is silu(gate) * 2^up_exponent for each of the gates (sums of two numbers of a block), x of ones."""
    f, d = len(gates), 32

    def spoil(matrix, expert, code, scale):
        code[:] = 0
        if matrix == 1:
            code[:f] = 2 * np.eye(f, dtype=np.uint8)  # y[i] = h[i]
            scale[:] = 127
        else:
            for i, (first, second, e) in enumerate(gates):  # -(first + second) * 2^e, first and second magnitudes of the code
                code[i, :2] = 8 + np.searchsorted(ref.MAGNITUDES, [first, second])
                scale[i] = 127 + e
            code[f:, 0] = 2
            scale[f:] = 127 + up_exponent

    x = np.zeros((1, d))
    x[0, :2] = 1.0
    return Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=1, experts=1, top_k=1, d=d, f=f, x=x, spoil=spoil)


@pytest.mark.gpu
def test_silu_of_very_negative_gates(mc, ref):  # noqa: F811
    """silu(v) goes to 0 like v e^v: 1 + e^-v leaves f32 at -88.7 and a fast division gives up at -87.3, but times 2^100 the values
    are ordinary numbers down to v = -150. bf16 rounds by 2^-8 of a value at most, the rest is far below."""
    gates = [(3, 2, 4), (4, 1.5, 4), (4, 0, 0), (6, 0, 4), (6, 0.5, 4), (6, 1, 4), (6, 1.5, 4), (6, 2, 4), (6, 3, 4), (1, 0, 0), (0, 0, 0)]
    gate = np.array([-(a + b) * 2.0 ** e for a, b, e in gates])
    want = gate / (1 + np.exp(-gate)) * 2.0 ** 100
    # values below 2^-50 of the largest of the token and expert are not kept; the large ones are in a layer of their own
    for part in (gate < -20, gate >= -20):
        q = _silu_problem(mc, ref, [v for v, keep in zip(gates, part) if keep], 100)
        mine = q.run()[0][: part.sum()]
        largest = np.abs(want[part]).max()
        assert (np.abs(mine - want[part]) <= 2.0 ** -8 * 1.01 * np.abs(want[part]) + 2.0 ** -46 * largest).all(), (mine, want[part])


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [(6, 1, 4), (4, 1.5, 4), (6, 2, 4)])
def test_silu_of_one_very_negative_gate(mc, ref, gate):  # noqa: F811
    """-112, -88 and -128: alone in its layer each keeps its bits."""
    v = -(gate[0] + gate[1]) * 2.0 ** gate[2]
    got = _silu_problem(mc, ref, [gate], 100).run()[0][0]
    want = v / (1 + np.exp(-v)) * 2.0 ** 100
    assert abs(got - want) <= 2.0 ** -8 * 1.01 * abs(want)


@pytest.mark.gpu
@pytest.mark.parametrize("x_sigma, gate_up_scale, down_scale", [(2.0 ** -40, 1.37 * 2.0 ** -20, 1.37 * 2.0 ** -36), (2.0 ** -40, 1.37 * 2.0 ** -20, 1.9 * 2.0 ** -34),
                                                               (1.0, 1.37 * 2.0 ** -55, 1.37 * 2.0 ** -37), (2.0 ** 10, 1.37 * 2.0 ** 10, 1.37 * 2.0 ** -100)])
@pytest.mark.parametrize("tokens", (2, 40))
def test_tensor_scales_beside_the_shifts(mc, ref, tokens, x_sigma, gate_up_scale, down_scale):  # noqa: F811
    """A tensor scale times the power of two that undoes a shift may be subnormal where the result is an ordinary number."""
    import torch

    d, f, experts = 64, 48, 5
    rng = np.random.default_rng(4)
    router = rng.standard_normal((experts, d)) * d ** -0.5 / x_sigma
    p = Tight(mc, ref, fmt="e4m3_16", dtype="bf16", tokens=tokens, experts=experts, top_k=2, d=d, f=f, sigma=x_sigma, router=router)
    for i, scale in enumerate((gate_up_scale, down_scale)):
        old = p.keep[i][2].double().cpu().numpy()
        new = np.full(experts, np.float32(scale))
        p.keep[i][2].copy_(torch.from_numpy(new))
        p.values[i] = [v / o * float(n) for v, o, n in zip(p.values[i], old, new)]
    got = p.run()
    y, bound, _, _ = p.expected()
    fine = np.abs(y) >= 2.0 ** -122
    assert fine.mean() > 0.9
    assert (np.abs(got - y) <= bound)[fine].all(), float((np.abs(got - y) / bound)[fine].max())


@pytest.mark.gpu
@pytest.mark.parametrize("x_exponent, router_exponent", [(-80, -80), (-100, -30), (-130, -10), (70, 70), (100, 28), (-120, 120), (0, -130)])
@pytest.mark.parametrize("d", (96, 97, 1100))
def test_the_choice_of_experts_at_any_exponent(mc, ref, x_exponent, router_exponent, d):  # noqa: F811
    """Products of two bf16 numbers reach from 2^-266 to 2^256, further than f32: the choice is that of 64 bits all the same."""
    rng = np.random.default_rng(d)
    tokens, experts, top_k = 6, 70, 5
    x = rng.standard_normal((tokens, d)) * 2.0 ** x_exponent
    router = rng.standard_normal((experts, d)) * 2.0 ** router_exponent
    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=tokens, experts=experts, top_k=top_k, d=d, f=32, x=x, router=router, renormalize=False)
    p.run()
    logits = p.x64 @ p.router64.T
    chosen = np.argsort(-logits, axis=1, kind="stable")[:, :top_k]
    assert np.array_equal(p.chosen.cpu().numpy(), chosen)
    weights = np.exp(logits - logits.max(axis=1, keepdims=True))
    weights = np.take_along_axis(weights / weights.sum(axis=1, keepdims=True), chosen, axis=1)
    assert np.allclose(p.weights.double().cpu().numpy(), weights, rtol=64 * U, atol=2.0 ** -126)


@pytest.mark.gpu
def test_products_that_mix_exponents(mc, ref):  # noqa: F811
    """Large values of x that meet zeros of the router: only the products' own size says whether f32 holds them."""
    d, experts = 64, 40
    rng = np.random.default_rng(2)
    x = np.zeros((2, d))
    x[:, :32] = 1.0
    x[0, 32:] = rng.standard_normal(32) * 2.0 ** -80
    x[1, 32:] = rng.standard_normal(32) * 2.0 ** 80
    router = np.zeros((experts, d))
    router[:, 32:] = rng.standard_normal((experts, 32)) * 2.0 ** -70
    p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=2, experts=experts, top_k=4, d=d, f=32, x=x, router=router)
    p.run()
    logits = p.x64 @ p.router64.T
    assert np.array_equal(p.chosen.cpu().numpy(), np.argsort(-logits, axis=1, kind="stable")[:, :4])


@pytest.mark.gpu
def test_weights_of_experts_far_below_the_best(mc, ref):  # noqa: F811
    """Weights of logits some 80 below the best: the difference has more bits than f32, and a rounding of it would be 2^-18 of the
    weight. A weight is off by expf (2 steps of 2^-23), the part that f32 leaves of the difference, the sum and the division: 8 steps."""
    d, experts, top_k = 64, 16, 16
    router = np.zeros((experts, d))
    router[:, 0] = -np.linspace(0, 84, experts)
    router[:, 1] = 2.0 ** -18 * (1 + np.arange(experts) % 3)
    router[:, 2] = 1.01
    x = np.zeros((3, d))
    x[:, :3] = [[1, 1, 0], [1, 1, 3], [0.9, 1.7, 0.3]]
    for renormalize in (False, True):
        p = Problem(mc, ref, fmt="e8m0_32", dtype="bf16", tokens=3, experts=experts, top_k=top_k, d=d, f=32, x=x, router=router, renormalize=renormalize)
        p.run()
        _, _, chosen, weights = p.expected()
        assert np.array_equal(p.chosen.cpu().numpy(), chosen)
        assert np.allclose(p.weights.double().cpu().numpy(), weights, rtol=8 * U, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens, experts, top_k, d, f", [(64, 1, 1, 33, 17), (33, 1, 1, 1025, 256), (40, 3, 2, 300, 1300), (34, 5, 4, 1100, 520), (64, 17, 16, 97, 257),
                                                          (63, 30, 3, 200, 300), (64, 30, 3, 200, 300), (31, 60, 4, 130, 700), (32, 60, 4, 130, 700), (37, 40, 3, 1030, 90),
                                                          (38, 40, 3, 1030, 90)])
def test_every_form_of_the_down_projection(mc, ref, fmt, tokens, experts, top_k, d, f):  # noqa: F811
    """Experts with many slots, on both sides of where the form or the depth of its rings changes."""
    p = Tight(mc, ref, fmt=fmt, dtype="f16", tokens=tokens, experts=experts, top_k=top_k, d=d, f=f, seed=d + f)
    got = p.run()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen)
    assert (np.abs(got - y) <= bound).all(), float((np.abs(got - y) / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts, top_k, d, f", [(40, 160, 3, 256, 192), (33, 40, 2, 1100, 100), (64, 6, 5, 1100, 300), (8, 20, 4, 1100, 300)])
def test_the_same_bits_in_every_form(mc, ref, tokens, experts, top_k, d, f):  # noqa: F811
    import torch

    p = Problem(mc, ref, fmt="e4m3_16", dtype="bf16", tokens=tokens, experts=experts, top_k=top_k, d=d, f=f)
    first = p.run()
    for _ in range(10):
        p.y_view[: tokens * d].fill_(float("nan"))
        p.ws[: p.need].fill_(0xFF)
        torch.cuda.synchronize()
        assert np.array_equal(p.run(), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_tokens_of_zeros_and_an_expert_that_is_not_a_number(mc, ref, dtype):  # noqa: F811
    """A batch padded with zeros: these tokens choose the first experts, with equal weights, and get zeros. A router's row with a NaN
    comes behind every number; the softmax over all experts is NaN then, and so are y and the weights, but not the choice."""
    rng = np.random.default_rng(3)
    tokens, experts, d = 12, 20, 72
    x = rng.standard_normal((tokens, d))
    x[5:] = 0.0
    router = rng.standard_normal((experts, d)) * d ** -0.5
    p = Problem(mc, ref, fmt="e8m0_32", dtype=dtype, tokens=tokens, experts=experts, top_k=3, d=d, f=48, x=x, router=router)
    got = p.run()
    y, bound, chosen, _ = p.expected()
    assert np.array_equal(p.chosen.cpu().numpy(), chosen) and (chosen[5:] == [0, 1, 2]).all()
    assert (np.abs(got - y) <= bound).all() and (got[5:] == 0).all()
    assert (p.weights[5:] == p.weights[5, 0]).all()
    router[7, 3] = np.nan
    p = Problem(mc, ref, fmt="e8m0_32", dtype=dtype, tokens=tokens, experts=experts, top_k=experts - 4, d=d, f=48, x=x, router=router)
    got = p.run()
    logits = p.x64 @ p.router64.T
    logits[:, 7] = -np.inf
    want = np.argsort(-logits, axis=1, kind="stable")[:, : experts - 4]
    assert np.array_equal(p.chosen.cpu().numpy(), want) and not (want == 7).any()
    assert np.isnan(got).all() and np.isnan(p.weights.cpu().numpy()).all()
