"""The operators on 8-bit blocks at sizes past 2^24 workgroups of 256 threads, more than one launch holds.

Blocks of one value each keep the arrays at a gigabyte or less, and the results are exact."""
import numpy as np
import pytest

import compute_amd as ca
from oracle import f8_ref as R
from tests.test_gpu_f8 import BF16, F8, F32, run_graph

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
