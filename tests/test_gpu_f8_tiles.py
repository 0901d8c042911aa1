"""Every tile of the dense product over 8-bit blocks, in one slice of K and in several (test_f8_plans.py holds the plans)."""
import numpy as np
import pytest

import compute_amd as ca
from tests.test_gpu_f8 import BF16, F8, F32, assert_within, dense_bound, dense_problem, to_f64, upload

pytestmark = pytest.mark.gpu

# (M, K, N, [n, k] layout, results, kernel and tile, whether K is cut)
TILES = [(70, 256, 130, True, BF16, "f8_dense_tiles 64x64", False), (70, 2000, 144, False, BF16, "f8_dense_tiles 64x64", True),
         (70, 1008, 130, True, F32, "f8_dense_tiles 64x64", True), (2100, 256, 512, True, BF16, "f8_dense_tiles 64x128", False),
         (2100, 256, 512, False, F32, "f8_dense_tiles 64x128", False), (1500, 2000, 130, True, BF16, "f8_dense_tiles 64x128", True),
         (1500, 1008, 130, True, F32, "f8_dense_tiles 64x128", True), (500, 1024, 640, False, F32, "f8_dense_tiles 64x128", True),
         (400, 256, 4099, True, BF16, "f8_dense_tiles 128x64", False), (700, 2000, 512, False, BF16, "f8_dense_tiles 128x64", True),
         (2100, 256, 1024, False, BF16, "f8_dense_tiles 128x128", False), (1500, 4000, 512, True, BF16, "f8_dense_tiles 128x128", True),
         (2100, 256, 2000, True, BF16, "f8_dense_tiles 256x128", False), (2100, 4000, 1024, False, BF16, "f8_dense_tiles 256x128", True),
         (2100, 2000, 1024, True, F32, "f8_dense_tiles 256x128", True), (2100, 256, 4000, False, BF16, "f8_dense_tiles 256x256", False),
         (2100, 4000, 2000, True, BF16, "f8_dense_tiles 256x256", True), (70, 1000, 130, True, F32, "f8_dense_staged 64x64", True),
         (700, 256, 2001, False, F32, "f8_dense_staged 128x64", False), (1500, 1000, 200, True, F32, "f8_dense_staged 128x64", True),
         (1500, 256, 2001, False, BF16, "f8_dense_staged 128x128", False), (1500, 4001, 512, True, BF16, "f8_dense_staged 128x128", True)]


@pytest.mark.parametrize("M,K,N,oi,out,tile,sliced", TILES)
def test_dense_tile(backend, M, K, N, oi, out, tile, sliced):
    """Sampled rows, the first and the last tile's among them, against 64 bits; four more calls bit for bit."""
    x, xs, w, ws, _ = dense_problem(M, K, N, oi)
    bld = backend.Builder("tile")
    f = bld.Main()
    arrays = {"x": (x, F8), "xs": (xs, F32), "w": (w, F8), "ws": (ws, F32)}
    p = {n: f.Parameter(n, ca.Shape(dt, *a.shape)) for n, (a, dt) in arrays.items()}
    f.Return([f.FusedF8Dense(p["x"], p["xs"], p["w"], p["ws"], None, ca.F8DenseConfig(0, int(oi), out))])
    exe, inputs = bld.Compile(), [upload(backend, a, dt, *a.shape) for a, dt in arrays.values()]
    first = exe.Execute(inputs)[0].ToFlatData().reshape(M, N)
    rows = np.unique(np.concatenate([[0, M // 2, M - 2, M - 1], np.random.default_rng(1).integers(0, M, 12)]))
    want, bound = dense_bound(x[rows], xs[rows], w, ws, oi, K, N, 0, out)
    assert_within(to_f64(first[rows], out), want, bound, tile)
    outs = [exe.Execute(inputs)[0] for _ in range(4)]
    for o in outs:
        assert np.array_equal(o.ToFlatData().reshape(M, N), first)
        o.Finalize()
