"""The operators on 8-bit blocks past the counts of a launch (2^24 workgroups of 256 threads) and past 31 bits of offset.

Blocks of one value each keep the first at a gigabyte or less, and their results are exact."""
import numpy as np
import pytest

import compute_amd as ca
from oracle import f8_ref as R
from tests.test_gpu_f8 import (BF16, F8, F32, activations, assert_within, dense_bound, run_dense, run_graph, store, to_f64, wgrad_want)

pytestmark = pytest.mark.gpu

ROWS = (1 << 28) + 37  # 2^24 workgroups take 2^28 blocks of a row


def pieces(n):
    return [slice(i, min(i + (1 << 26), n)) for i in range(0, n, 1 << 26)]


def test_quantize_rows_past_a_launch(backend):
    """Every bfloat16 pattern, again and again: its codes and scales come from a table of all 65536."""
    patterns = np.arange(65536, dtype=np.uint16)
    with np.errstate(invalid="ignore"):  # signalling NaN among the patterns
        codes, scales = R.quantize(ca.bf16_to_f32(patterns).astype(np.float64)[:, None])
    x = np.resize(patterns, (ROWS, 1))
    got, got_scale = run_graph(backend, lambda f, p: f.FusedF8Quantize(p["x"]), {"x": (x, BF16)})
    got, got_scale, x = got.ravel(), got_scale.ravel(), x.ravel()
    nan = (codes.ravel() & 127) == 127
    for s in pieces(ROWS):
        assert np.array_equal(got_scale[s], scales.ravel()[x[s]])
        assert np.all((got[s] == codes.ravel()[x[s]]) | (nan[x[s]] & ((got[s] & 127) == 127)))


def test_activation_gradient_past_a_launch(backend):
    rng = np.random.default_rng(3)
    z = np.resize(np.array([c for c in range(256) if (c & 127) != 127], np.uint8), (ROWS, 1))
    dy = np.resize(ca.bf16_from_f32(rng.standard_normal(9973).astype(np.float32)), (ROWS, 1))
    got, = run_graph(backend, lambda f, p: [f.FusedF8ActivationGradient(p["z"], p["zs"], p["dy"], ca.ActivationRelu)],
                     {"z": (z, F8), "zs": (np.ones((ROWS, 1), np.float32), F32), "dy": (dy, BF16)})
    got, z, dy = got.ravel(), z.ravel(), dy.ravel()
    for s in pieces(ROWS):
        positive = (z[s] >= 1) & (z[s] < 128)
        assert np.array_equal(np.where(positive, got[s], got[s] & 0x7fff), np.where(positive, dy[s], 0))


@pytest.mark.parametrize("M", [1, 3])
def test_dense_columns_past_a_launch(backend, M):
    """One value of k: a product of two codes and a power of two, four significant bits each, exact in bfloat16."""
    N = ROWS
    finite = np.array([c for c in range(256) if (c & 127) != 127], np.uint8)
    x = np.array([[0x38], [0xc5], [0x11]], np.uint8)[:M]
    xs = np.array([[0.5], [2.0], [1.0]], np.float32)[:M]
    w = np.resize(finite, (N, 1))
    ws = np.resize(np.array([0.25, 1.0, 8.0], np.float32), (R.blocks(N), 1))
    got, = run_graph(backend, lambda f, p: [f.FusedF8Dense(p["x"], p["xs"], p["w"], p["ws"], None, ca.F8DenseConfig(0, 1, BF16))],
                     {"x": (x, F8), "xs": (xs, F32), "w": (w, F8), "ws": (ws, F32)})
    values = R.VALUES.astype(np.float32)
    for m in range(M):
        for s in pieces(N):
            want = values[w.ravel()[s]] * np.repeat(ws.ravel()[s.start // 128:R.blocks(s.stop)], 128)[:s.stop - s.start]
            assert np.array_equal(ca.bf16_to_f32(got[m, s]), want * np.float32(values[x[m, 0]] * xs[m, 0]))


# Codes of 2.2e9 bytes: offsets pass 31 bits.
FAR = 1_100_003


@pytest.mark.parametrize("K,out", [(2048, BF16), (2047, F32)])
def test_dense_of_far_rows(backend, K, out):
    """Rows of a prime period: the first 997 against 64 bits, all others the same bits."""
    rng = np.random.default_rng(K)
    N = 24
    block, scale = R.quantize(activations(rng, 997, K))
    w, ws = R.quantize(0.02 * rng.standard_normal((N, K)), 128)
    x, xs = np.resize(block, (FAR, K)), np.resize(scale, (FAR, R.blocks(K)))
    got = run_dense(backend, x, xs, w, ws, True, 0, out)
    want, bound = dense_bound(block, scale, w, ws, True, K, N, 0, out)
    assert_within(got[:997], want, bound, "the first rows")
    assert np.array_equal(got, np.resize(got[:997], got.shape))


@pytest.mark.parametrize("K,oi,dt", [(2048, True, BF16), (2047, False, F32)])
def test_weight_gradient_of_far_tokens(backend, K, oi, dt):
    """dy is zero but for the first and the last 500 tokens, so that their sum alone is left, exact zeros beside it."""
    rng = np.random.default_rng(K)
    N = 16
    block, scale = R.quantize(activations(rng, 997, K))
    x, xs = np.resize(block, (FAR, K)), np.resize(scale, (FAR, R.blocks(K)))
    rows = np.concatenate([np.arange(500), np.arange(FAR - 500, FAR)])
    dy = np.zeros((FAR, N), np.uint16 if dt == BF16 else np.float32)
    dy[rows] = store(activations(rng, 1000, N), dt)
    got, = run_graph(backend, lambda f, p: [f.FusedF8WeightGradient(p["x"], p["xs"], p["dy"], ca.DenseLayout(int(oi)))],
                     {"x": (x, F8), "xs": (xs, F32), "dy": (dy, dt)})
    want, bound = wgrad_want(x[rows], xs[rows], to_f64(dy[rows], dt), oi, F32, dt)
    assert_within(got.astype(np.float64), want, bound, "far tokens")


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_far_rows(backend, rows):
    """bfloat16 x of 4.5e9 bytes; a period of 128 x 13 rows, so that blocks of 128 rows repeat too."""
    K, period = 2047, 128 * 13
    block = store(activations(np.random.default_rng(rows), period, K), BF16)
    x = np.resize(block, (FAR, K))
    codes, scale = run_graph(backend, lambda f, p: f.FusedF8Quantize(p["x"], rows), {"x": (x, BF16)})
    want, ws = R.quantize(to_f64(block, BF16), rows)
    last = FAR // period * period  # the last period is cut short: its last block of 128 rows too
    tail, ts = R.quantize(to_f64(x[last:], BF16), rows)
    for i in range(0, last, period):
        assert np.array_equal(codes[i:i + period], want) and np.array_equal(scale[i // rows:(i + period) // rows], ws)
    assert np.array_equal(codes[last:], tail) and np.array_equal(scale[last // rows:], ts)
