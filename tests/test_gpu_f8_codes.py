"""8-bit floating-point codes in the ops that only move data, and as constants."""
import numpy as np
import pytest

import compute_amd as ca
from tests.test_gpu_f8 import F8, run_graph

pytestmark = pytest.mark.gpu


def test_codes_move_like_bytes(backend):
    """The ops that only move data take codes: constants, transposes, slices, broadcasts, reshapes, bitcasts."""
    rng = np.random.default_rng(2)
    c = rng.integers(0, 256, (130, 70), dtype=np.uint8)

    def build(f, p):
        k = p["c"]
        return [f.Transpose(k, 1, 0), f.Slice(k, [3, 1], [129, 70], [2, 3]), f.BroadcastInDim(k, ca.Shape(F8, 2, 130, 70), [1, 2]),
                f.Reshape(k, 70, 130), f.Identity(k), f.Bitcast(k, ca.Uint8), f.Transpose(f.Constant(c.ravel(), 130, 70, dtype=F8), 1, 0)]

    t, s, b, r, i, u, k = run_graph(backend, build, {"c": (c, F8)})
    assert np.array_equal(t, c.T) and np.array_equal(s, c[3:129:2, 1:70:3]) and np.array_equal(b, np.stack([c, c]))
    assert np.array_equal(r, c.reshape(70, 130)) and np.array_equal(i, c) and np.array_equal(u, c) and np.array_equal(k, c.T)
