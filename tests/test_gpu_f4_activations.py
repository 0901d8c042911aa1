"""The activations of float32 results of the products over 4-bit blocks, to float32's precision: x is zero, so that a result is the
activation of its bias exactly, in every kernel.

Bounds, in units of 2^-24 of the result.  GELU is x times 0.5 erfc(|x| / sqrt 2) or one minus it, the first exp(-x^2 / 2) times a polynomial of
nine terms in a reciprocal: three roundings of the exponent, each x^2 / 2; two for the exponential, three for the reciprocal and its argument
(of which the polynomial takes no more), nine steps of the polynomial whose parts add up to 2.4 times its value, one for its fit, four for products and the
difference: 1.5 x^2 + 32.  SiLU is x times the reciprocal of one plus an exponential: two roundings of the exponent, each |x|; two, one
and two for exponential, sum and reciprocal and one for the product: 2 |x| + 6.
"""
import math

import numpy as np
import pytest

import compute_amd as ca
from f4_helpers import E8, F32, F4, I32, make_x, run_graph
from oracle import f4_ref as R

pytestmark = pytest.mark.gpu

BOUND = {"gelu": lambda v: 1.5 * v * v + 32, "silu": lambda v: 2 * np.abs(v) + 6}
ACT = {"gelu": ca.ActivationGelu, "silu": ca.ActivationSilu}
LEAST = {"gelu": -12.5, "silu": -80.0}


def exact(act, v):
    if act == "gelu":
        return np.array([t * 0.5 * math.erfc(-t / math.sqrt(2)) for t in v.ravel()]).reshape(v.shape)
    return v / (1 + np.exp(-v))


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("kind", ["f4", "bf16", "f32"])
@pytest.mark.parametrize("M,E", [(1, 0), (4, 0), (40, 0), (300, 0), (6, 3), (90, 3)])
def test_float32_results(backend, M, E, kind, oi, act):
    K, N = 128, 2048
    rng = np.random.default_rng(M + E)
    x, dt, xs, _ = make_x(rng, M, K, kind)
    x[:] = 0
    n = max(E, 1)
    w, ws = R.random_codes(rng, n, *((N, K) if oi else (K, N)))
    b = np.where(rng.random((n, N)) < 0.5, rng.uniform(LEAST[act], 6, (n, N)), 1.5 * rng.standard_normal((n, N))).astype(np.float32)
    inputs = {"x": (x, dt), "w": (w if E else w[0], F4), "ws": (ws if E else ws[0], E8), "b": (b if E else b[0], F32)}
    if xs is not None:
        inputs["xs"] = (xs, E8)
    off = np.linspace(0, M, n + 1).astype(np.int32)
    if E:
        inputs["o"] = (off, I32)
    cfg = ca.F4DenseConfig(Activation=ACT[act], WeightLayout=ca.DenseLayout(int(oi)), OutputDType=F32)

    def build(f, p):
        if E:
            return [f.FusedF4ExpertDense(p["x"], p.get("xs"), p["o"], p["w"], p["ws"], p["b"], cfg)]
        return [f.FusedF4Dense(p["x"], p.get("xs"), p["w"], p["ws"], p["b"], cfg)]

    got, = run_graph(backend, build, inputs)
    for e in range(n):
        v = b[e].astype(np.float64)
        want = exact(act, v)
        steps = np.abs(got[off[e]:off[e + 1]].astype(np.float64) - want) / (np.abs(want) * 2.0 ** -24 + 1e-300)
        assert np.all(steps <= BOUND[act](v)), (steps - BOUND[act](v)).max()


@pytest.mark.parametrize("M", [2, 40])
def test_special_values(backend, M):
    """Zeros, infinities, NaN and very large values; GELU of minus infinity is 0 times infinity, NaN as its formula gives."""
    b = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 3e38, -3e38, 1e20, -1e20, 1e-40, -30.0, 20.0] + [0.0] * 20, np.float32)
    want = np.array([0, 0, np.inf, np.nan, np.nan, 3e38, 0, 1e20, 0, 0.5e-40, 0, 20] + [0] * 20, np.float32)
    w, ws = np.zeros((32, 64), np.uint8), np.full((32, 4), 127, np.uint8)
    cfg = ca.F4DenseConfig(Activation=ca.ActivationGelu, WeightLayout=ca.DenseLayoutOutputsInput)
    got, = run_graph(backend, lambda f, p: [f.FusedF4Dense(p["x"], None, p["w"], p["ws"], p["b"], cfg)],
                     {"x": (np.zeros((M, 128), np.float32), F32), "w": (w, F4), "ws": (ws, E8), "b": (b, F32)})
    assert np.allclose(got, np.tile(want, (M, 1)), rtol=1e-6, atol=1e-44, equal_nan=True)
