"""Weight gradients over 8-bit blocks, many steps long: the same bits at every call, next to other calls, from threads and backends.

A wave that met another's buffer, or a slice another's scratch, would show as a difference between two calls.
The first result of each is held against 64 bits with the bounds at the head of test_gpu_f8.py.
"""
import threading

import numpy as np
import pytest

import compute_amd as ca
from oracle import f8_ref as R
from tests.test_gpu_f8 import BF16, F8, F32, SLICED, activations, assert_within, dense_executable, store, to_f64, upload, wgrad_want

pytestmark = pytest.mark.gpu

# (tokens, k, n, [n, k] layout, dy): both tiles of both types, one slice of the tokens and several, whole chunks and odd rows.
SHAPES = [(2048, 1024, 1024, True, BF16), (700, 2048, 2176, False, BF16), (2047, 2000, 1000, True, BF16), (1501, 1001, 777, False, BF16),
          (500, 2001, 1003, True, BF16), (900, 3600, 3488, True, BF16), (900, 3601, 3487, False, BF16), (700, 4101, 4099, False, BF16),
          (2048, 1024, 1024, False, F32), (1501, 1001, 777, True, F32), (700, 3600, 3488, False, F32), (33, 2000, 1000, True, F32)]


def weight_gradient_executable(backend, M, K, N, oi, dt, seed=0):
    """(executable, uploaded inputs, the gradient in 64 bits, its bound)."""
    rng = np.random.default_rng(seed + M + 7 * K + N)
    x, xs = R.quantize(activations(rng, M, K))
    dy = store(0.01 * activations(rng, M, N), dt)
    bld = backend.Builder("wgrad")
    f = bld.Main()
    arrays = {"x": (x, F8), "xs": (xs, F32), "dy": (dy, dt)}
    p = {n: f.Parameter(n, ca.Shape(d, *a.shape)) for n, (a, d) in arrays.items()}
    f.Return([f.FusedF8WeightGradient(p["x"], p["xs"], p["dy"], ca.DenseLayout(int(oi)), F32)])
    want, bound = wgrad_want(x, xs, to_f64(dy, dt), oi, F32, dt)
    return bld.Compile(), [upload(backend, a, d, *a.shape) for a, d in arrays.values()], want, bound


@pytest.mark.parametrize("M,K,N,oi,dt", SHAPES)
def test_weight_gradient_repeats_bit_for_bit(backend, M, K, N, oi, dt):
    """Twenty calls in a row, and ten with a product in slices, whose sums lie in the same scratch, before each."""
    exe, inputs, want, bound = weight_gradient_executable(backend, M, K, N, oi, dt)
    dense, dense_inputs = dense_executable(backend, *SLICED[0], 1)
    first = exe.Execute(inputs)[0].ToFlatData().reshape(want.shape)
    assert_within(first.astype(np.float64), want, bound, f"{M}x{K}x{N}")
    between = dense.Execute(dense_inputs)[0].ToFlatData()
    outs = [exe.Execute(inputs)[0] for _ in range(20)]
    for o in outs:
        assert np.array_equal(o.ToFlatData().reshape(want.shape), first)
        o.Finalize()
    for _ in range(10):
        d, o = dense.Execute(dense_inputs)[0], exe.Execute(inputs)[0]
        assert np.array_equal(o.ToFlatData().reshape(want.shape), first) and np.array_equal(d.ToFlatData(), between)
        d.Finalize()
        o.Finalize()


def test_weight_gradients_from_threads_and_two_backends(backend):
    """Four threads, two on each of two backends, run gradients in slices at once: each gets its own results."""
    other = ca.New("mi355x")
    try:
        runs = [weight_gradient_executable(b, *SHAPES[i], seed=i) for b in (backend, other) for i in (0, 8)]
        first = [exe.Execute(inputs)[0].ToFlatData() for exe, inputs, *_ in runs]
        assert np.array_equal(first[0], first[2]) and np.array_equal(first[1], first[3])
        wrong = []

        def work(exe, inputs, want):
            for _ in range(20):
                o, = exe.Execute(inputs)
                if not np.array_equal(o.ToFlatData(), want):
                    wrong.append(want.shape)
                o.Finalize()

        threads = [threading.Thread(target=work, args=(exe, inputs, w)) for (exe, inputs, *_), w in zip(runs, first)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong
    finally:
        del runs
        other.Finalize()
