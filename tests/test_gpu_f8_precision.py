"""What mxrt.h promises of the sums of the dense product over 8-bit blocks, where ordinary data does not show it."""
import numpy as np
import pytest

from oracle import f8_ref as R
from tests.test_gpu_f8 import BF16, F32, assert_within, run_dense

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
