"""8-bit floating-point codes in the ops that only move data and as constants; which kernels a product launches."""
import numpy as np
import pytest

import compute_amd as ca
from compute_amd import _lib
from tests.test_gpu_f8 import BF16, F8, F32, Memory, run_graph, store

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


@pytest.mark.parametrize("M,K,N,oi", [(1, 512, 256, True), (4, 512, 256, True), (5, 512, 256, True), (16, 300, 256, True), (5, 512, 256, False),
                                      (40, 512, 256, True), (40, 300, 256, True), (300, 512, 256, False)])
@pytest.mark.parametrize("x_dt", [F8, BF16, F32])
@pytest.mark.parametrize("off", [0, 4])
def test_plan_names_the_kernel_that_runs(backend, M, K, N, oi, x_dt, off):
    """The launches that the profile counts: the product's kernel is the plan's, and float x past four rows has its codes made first."""
    rng = np.random.default_rng(M + K)
    m = Memory(backend)
    x = rng.integers(0, 100, (M, K), dtype=np.uint8) if x_dt == F8 else store(rng.standard_normal((M, K)).astype(np.float32), x_dt)
    shape = (N, K) if oi else (K, N)
    ax, axs = m.put(x, off), m.put(np.ones((M, 3 if K == 300 else 4), np.float32))
    aw, aws, ao = m.put(rng.integers(0, 100, shape, dtype=np.uint8)), m.put(np.ones((4, 4), np.float32)), m.room(M * N * 2)
    m.upload()
    a = _lib.mx_f8_dense_args(x=m.base + ax, x_scale=m.base + axs if x_dt == F8 else None, w=m.base + aw, w_scale=m.base + aws,
                              out=m.base + ao, M=M, K=K, N=N, x_dtype=int(x_dt), out_dtype=int(BF16), weight_layout=int(oi))
    plan = backend.F8DensePlan(a)
    backend.Synchronize()
    backend.SetProfiling(True)
    try:
        backend.ProfileReset()
        backend.F8Dense(a)
        ran = set(backend.Profile())
    finally:
        backend.SetProfiling(False)
    makes = x_dt != F8 and not (oi and M <= 4)
    assert ran == {plan.split()[0]} | ({"f8_quantize_rows"} if makes else set())
