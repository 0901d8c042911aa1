"""Products against [out, in] weights in 4-bit blocks whose slices of K begin with odd steps of 64, K a multiple of 128, so that the
scales are loaded as they lie: the last step's are the last two bytes of the array.  The last columns' terms are largest there, and
what lies beside the arrays is NaN.  Bounds of f4_helpers.dense_want."""
import numpy as np
import pytest

from f4_helpers import F32, Memory, assert_within, dense_args, dense_want, make_x
from f4_tile_cases import plan_of
from oracle import f4_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,M,K,N,plan", [
    ("bf16", 17, 4096, 5120, "f4_wide 128x64 slices 6"), ("bf16", 17, 2560, 64, "f4_wide 64x64 slices 8"), ("f32", 16, 4096, 64, "f4_wide 64x64 slices 13"),
    ("f32", 16, 1536, 64, "f4_wide 64x64 slices 8"), ("f32", 16, 1536, 61, "f4_wide 64x64 slices 8"), ("f32", 40, 1408, 130, "f4_wide 64x64 slices 8"),
    ("f32", 17, 896, 4104, "f4_wide 128x64 slices 5"), ("f32", 17, 2176, 8200, "f4_wide 256x64 slices 7"),
    ("f32", 100, 3968, 8200, "f4_wide 256x128 slices 7"), ("bf16", 100, 2048, 8200, "f4_wide 128x128 slices 3"),
    ("bf16", 200, 2176, 8200, "f4_wide 256x128 slices 2")])
def test_last_scales(backend, kind, M, K, N, plan):
    assert plan_of(backend, kind, True, M, K, N, 0) == plan
    slices, steps = int(plan.split()[-1]), K // 64
    assert -(-steps // slices) % 2 == 1
    rng = np.random.default_rng(M + K + N)
    x, dt, _, xv = make_x(rng, M, K, kind)
    w, ws = R.random_codes(rng, N, K)
    ws[-3:, -2:] += 8
    m = Memory(backend)
    ax, aw, aws, ao = m.put(x), m.put(w), m.put(ws), m.room(M * N * 4)
    m.upload(fill=0xff)
    want, bound = dense_want(xv, R.values(w, ws).T, None, 0, F32, kind)
    without = dense_want(xv[:, :-64], R.values(w[:, :-32], ws[:, :-2]).T, None, 0, F32, kind)[0]
    assert (np.abs(want - without) > 4 * bound)[:, -1].any()  # a loss of the last step would show
    for _ in range(2):
        backend.F4Dense(dense_args(m, ax, 0, aw, aws, 0, ao, M, K, N, dt, F32, True))
        assert_within(m.back(ao, np.float32, (M, N)).astype(np.float64), want, bound, plan)
