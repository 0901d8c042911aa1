"""Precision of the operators on 8-bit blocks where ordinary data does not show it: sums that cancel, tails of activations."""
import numpy as np
import pytest

import compute_amd as ca
from oracle import f8_ref as R
from tests.test_gpu_f8 import BF16, F8, F32, activations, assert_within, dense_bound, dense_problem, run_dense, run_graph, store, to_f64, wgrad_want

pytestmark = pytest.mark.gpu

# The kernel for few rows, tiles of both layouts, tiles whose operands come through registers.
KERNELS = [(2, 256, 40, True), (16, 512, 200, True), (24, 256, 80, False), (300, 512, 272, True), (130, 255, 77, True), (40, 200, 75, False)]


@pytest.mark.parametrize("M,K,N,oi", KERNELS)
def test_sums_that_cancel(backend, M, K, N, oi):
    """In every eight of k: 256, -256 and a small value, against weights of one.

    float32: all partial sums, in any order, are multiples of 2^-6 below 2^15, so the result is exact.
    bfloat16: seven products of an eight are cut at 2^-13 of 256; the eights' sums are then multiples of 2^-9 below
    2^15, and the result is rounded once.
    """
    rng = np.random.default_rng(K)
    x = np.zeros((M, K))
    x[:, 0:K // 8 * 8:8], x[:, 1:K // 8 * 8:8] = 256, -256
    x[:, 2:K // 8 * 8:8] = 2.0 ** -6 * rng.integers(1, 4, (M, K // 8))
    codes, scale = R.encode(x), np.ones((M, R.blocks(K)), np.float32)
    shape = (N, K) if oi else (K, N)
    w, ws = R.encode(np.ones(shape)), np.ones((R.blocks(shape[0]), R.blocks(shape[1])), np.float32)
    want = np.repeat(x.sum(1, keepdims=True), N, 1)
    assert np.array_equal(run_dense(backend, codes, scale, w, ws, oi, 0, F32), want)
    got = run_dense(backend, codes, scale, w, ws, oi, 0, BF16)
    cut = K // 8 * 7 * 2.0 ** -13 * 256
    assert_within(got, want, np.full_like(want, cut) + 2.0 ** -8 * (np.abs(want) + cut), "bfloat16")


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("act", [1, 3])
def test_activation_gradient_tails(backend, act, dt):
    """GELU and SiLU far from zero, each result held against its own size, dz against the terms of its slope.

    bfloat16: GELU's polynomial 3.8e-5, the exponent z^2 / 2 (SiLU: z) rounded twice, z^2 * 2^-24 <= 1.1e-5, and 16 roundings of
    2^-24: below 2^-13; half a step of 2^-8.  float32: erfc's argument is rounded twice, which moves erfc by 1.5 z^2 * 2^-24, the
    exponent's by z^2 * 2^-24 (SiLU: 2 |z| * 2^-24), erfc and exp to 8 ulp, 16 roundings: (3 z^2 + 32) 2^-24.
    """
    z = R.VALUES[[c for c in range(256) if (c & 127) != 127]]
    z = np.concatenate([z * s for s in (2.0 ** -5, 2.0 ** -6, 2.0 ** -7)])
    z = np.unique(z[(z >= -13) & (z != 0)])
    z = np.resize(z, (-(-z.size // 128), 128))
    codes, scale = R.quantize(z)
    exact = R.values(codes, scale)
    rng = np.random.default_rng(1)
    dy = store(rng.uniform(0.5, 2, z.shape).astype(np.float32), dt)
    ones, one = R.quantize(np.ones(z.shape))

    def build(f, p):
        return f.FusedF8ActivationGradient(p["z"], p["zs"], p["dy"], ca.ActivationType(act), p["u"], p["us"])

    dz, dup = run_graph(backend, build, {"z": (codes, F8), "zs": (scale, F32), "dy": (dy, dt), "u": (ones, F8), "us": (one, F32)})
    d = to_f64(dy, dt)
    rel = 2.0 ** -13 if dt == BF16 else (3 * exact ** 2 + 32) * 2.0 ** -24
    half = 2.0 ** -8 if dt == BF16 else 2.0 ** -24
    want = d * R.act(exact, act)
    assert_within(to_f64(dup, dt), want, (rel + half * (1 + rel)) * np.abs(want) + 1e-38, "dup")
    # the slope's terms: the cumulative and z times the density (GELU), g and z g (1 - g) (SiLU)
    if act == 1:
        terms = R.act(exact, 1) / np.where(exact == 0, 1, exact) + np.abs(exact) * np.exp(-exact ** 2 / 2) / np.sqrt(2 * np.pi)
    else:
        g = 1 / (1 + np.exp(-exact))
        terms = g + np.abs(exact) * g * (1 - g)
    want = d * R.slope(exact, act)
    assert_within(to_f64(dz, dt), want, rel * d * terms + half * np.abs(want) * 1.001 + 1e-38, "dz")


@pytest.mark.parametrize("M,K,N", [(37, 130, 70), (37, 144, 72), (700, 131, 45), (64, 144, 72)])
@pytest.mark.parametrize("oi", [True, False])
def test_weight_gradient_of_an_infinite_row(backend, M, K, N, oi):
    """The last token's first block overflows: positive codes times positive dy are infinite there, and the tokens that
    pad the last step, whose codes are zeros, add nothing to them; the second block is as ever."""
    rng = np.random.default_rng(K)
    x, xs = R.encode(np.full((M, K), 1.5)), np.ones((M, 2), np.float32)
    xs[M - 1, 0] = np.inf
    dy = store(rng.uniform(0.5, 1, (M, N)).astype(np.float32), BF16)
    got, = run_graph(backend, lambda f, p: [f.FusedF8WeightGradient(p["x"], p["xs"], p["dy"], ca.DenseLayout(int(oi)), F32)],
                     {"x": (x, F8), "xs": (xs, F32), "dy": (dy, BF16)})
    got = got.T if oi else got
    assert np.all(got[:128] == np.inf)
    want, bound = wgrad_want(x[:, 128:], xs[:, 1:], to_f64(dy, BF16), False, F32, BF16)
    assert_within(got[128:].astype(np.float64), want, bound, "the second block")


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("M,K,N,oi", KERNELS)
def test_dense_of_tiny_rows(backend, M, K, N, oi, out):
    """Row scales from 2^-100 down to 2^-126 against weight scales around 2^-13: products of two scales on both sides of 2^-126.

    Past the usual bound a subnormal product is rounded by half of 2^-149 and meets a block's sum of up to 448^2 * 128 < 2^24.7.
    """
    x, xs, w, ws, _ = dense_problem(M, K, N, oi)
    xs = np.ldexp(1.0, -100 - np.arange(xs.size).reshape(xs.shape) % 27).astype(np.float32)
    want, bound = dense_bound(x, xs, w, ws, oi, K, N, 0, out)
    assert np.abs(want).max() > 2.0 ** -110
    assert_within(run_dense(backend, x, xs, w, ws, oi, 0, out), want, bound + R.blocks(K) * 2.0 ** -150 * 2.0 ** 24.7, "tiny rows")


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(40, 300, 200), (256, 256, 256), (300, 144, 72)])
def test_weight_gradient_of_tiny_rows(backend, M, K, N, dt):
    """Scales from 2^-118 down to 2^-126: from 2^-124 the values are exact in bfloat16, below rounded to multiples of 2^-133."""
    rng = np.random.default_rng(K)
    x, _ = R.quantize(activations(rng, M, K))
    xs = np.ldexp(1.0, -118 - rng.integers(0, 9, (M, R.blocks(K)))).astype(np.float32)
    dy = store(1e6 * activations(rng, M, N), dt)
    got, = run_graph(backend, lambda f, p: [f.FusedF8WeightGradient(p["x"], p["xs"], p["dy"])], {"x": (x, F8), "xs": (xs, F32), "dy": (dy, dt)})
    d = to_f64(dy, dt)
    want, bound = wgrad_want(x, xs, d, False, F32, dt)
    low = R.spread(xs < 2.0 ** -124, 1, x.shape)
    assert_within(got.astype(np.float64), want, bound + 2.0 ** -134 * (low.T @ np.abs(d)), "tiny rows")
