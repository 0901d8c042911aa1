"""Float32 x keeps all its bits against weights in 4-bit blocks: every tile for float32 x in both layouts, the kernels for few rows and
for few columns, of one matrix and of experts, on sums that are exact in float32, so that results are known bit for bit."""
import numpy as np
import pytest

import compute_amd as ca
from f4_helpers import E8, F32, F4, I32, run_graph
from f4_tile_cases import CASES, plan_of
from oracle import f4_ref as R

pytestmark = pytest.mark.gpu

POWERS = np.array([1, 2, 4, 6, 9, 10, 12, 14], np.uint8)  # the codes of powers of two and their negatives
SIZES = sorted({c[1:] for c in CASES if c[0] == "f32"}) + [
    (False, M, 1216, 1032, 0, f"f4_columns 512x{r} slices 4") for M, r in ((1, 1), (2, 2), (4, 4))] + [
    (False, 12, 1216, 1032, 3, "f4_columns 512x4 slices 4"), (True, 1, 1216, 8200, 0, "f4_skinny")]


def odd_values(rng, n):
    """float32 values of 24 significant bits, the last of them set, over 13 binades, of both signs."""
    v = (1 << 23 | rng.integers(0, 1 << 22, n) << 1 | 1).astype(np.float64) * 2.0 ** rng.integers(-30, -17, n)
    return np.where(rng.random(n) < 0.5, -v, v).astype(np.float32)


def leading16(v):
    """v without the last 8 of its 24 significant bits."""
    return (v.view(np.uint32) & 0xffffff00).view(np.float32)


def product(backend, x, w, ws, oi, ends):
    cfg = ca.F4DenseConfig(WeightLayout=ca.DenseLayout(int(oi)), OutputDType=F32)
    inputs = {"x": (x, F32), "w": (w if ends else w[0], F4), "ws": (ws if ends else ws[0], E8)}
    if ends:
        inputs["o"] = (np.array([0, *ends], np.int32), I32)
        return run_graph(backend, lambda f, p: [f.FusedF4ExpertDense(p["x"], None, p["o"], p["w"], p["ws"], None, cfg)], inputs)[0]
    return run_graph(backend, lambda f, p: [f.FusedF4Dense(p["x"], None, p["w"], p["ws"], None, cfg)], inputs)[0]


def expert_of(M, ends):
    """The expert of each row (E: those behind the last)."""
    return np.searchsorted(np.array(ends), np.arange(M), side="right") if ends else np.zeros(M, int)


@pytest.mark.parametrize("oi,M,K,N,E,plan", SIZES)
def test_one_term(backend, oi, M, K, N, E, plan):
    """One value of x in a row, at any k, against powers of two: y is that product."""
    assert plan_of(backend, "f32", oi, M, K, N, E) == plan
    rng = np.random.default_rng(M + K + N)
    n, ends = max(E, 1), [M // 5, M // 5, M - M // 7] if E else []
    shape = (n, N, K) if oi else (n, K, N)
    w = R.pack(POWERS[rng.integers(0, 8, shape)])
    ws = rng.integers(120, 135, (*shape[:2], R.blocks(shape[2]))).astype(np.uint8)
    at, v, expert = rng.integers(0, K, M), odd_values(rng, M), expert_of(M, ends)
    x = np.zeros((M, K), np.float32)
    x[np.arange(M), at] = v
    got = product(backend, x, w, ws, oi, ends)
    want = np.zeros((M, N), np.float32)
    for e in range(n):
        wv = R.values(w[e], ws[e]).astype(np.float32)
        mine = expert == e
        want[mine] = v[mine, None] * (wv[:, at[mine]].T if oi else wv[at[mine]])
    assert np.array_equal(got, want)


@pytest.mark.parametrize("oi,M,K,N,E,plan", SIZES)
def test_what_the_last_bits_leave(backend, oi, M, K, N, E, plan):
    """A value and, at another k, its first 16 bits with the other sign, against weights that are the same for all k: every partial
    sum of their parts is a multiple of the value's last bit with 24 bits at most, so y is the last 8 bits exactly."""
    rng = np.random.default_rng(M + K + N + 1)
    n, ends = max(E, 1), [M // 5, M // 5, M - M // 7] if E else []
    codes, blocks = POWERS[rng.integers(0, 8, (n, N))], rng.integers(120, 135, (n, R.blocks(N)))
    if oi:
        w, ws = np.repeat(codes[:, :, None], K, 2), np.repeat(np.repeat(blocks, 32, 1)[:, :N, None], R.blocks(K), 2)
    else:
        w, ws = np.repeat(codes[:, None], K, 1), np.repeat(blocks[:, None], K, 1)
    w, ws = R.pack(w), ws.astype(np.uint8)
    first, v, expert = rng.integers(0, K, M), odd_values(rng, M), expert_of(M, ends)
    second = (first + rng.integers(1, K, M)) % K
    x = np.zeros((M, K), np.float32)
    x[np.arange(M), first] = v
    x[np.arange(M), second] = -leading16(v)
    got = product(backend, x, w, ws, oi, ends)
    last = v - leading16(v)
    assert np.all(last != 0)
    want = np.zeros((M, N), np.float32)
    for e in range(n):
        one = R.values(w[e][:, :1], ws[e][:, :1])[:, 0] if oi else R.values(w[e][0], ws[e][0])
        want[expert == e] = last[expert == e, None] * one.astype(np.float32)
    assert np.array_equal(got, want)
