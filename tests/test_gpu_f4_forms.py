"""Forms of the operators on 4-bit blocks that other tests leave out: [in, out] weights of an odd number of inputs, offsets that do not
ascend against them, a bias in bf16, as many experts as there may be, and codes through the ops that take them as they are.
Bounds of f4_helpers.dense_want."""
import numpy as np
import pytest

import compute_amd as ca
from f4_helpers import BF16, E8, F32, F4, I32, Memory, assert_within, dense_args, dense_want, make_x, run_graph, store, to_f64
from f4_tile_cases import plan_of
from oracle import f4_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M", [1, 3, 4, 5, 40, 300])
@pytest.mark.parametrize("K,N", [(1, 8), (3, 34), (63, 64), (65, 128), (65, 520), (1001, 130), (1001, 256)])
def test_odd_inputs(backend, M, K, N, kind):
    rng = np.random.default_rng(M + K)
    x, dt, _, xv = make_x(rng, M, K, kind)
    w, ws = R.random_codes(rng, K, N)
    m = Memory(backend)
    ax, aw, aws, ao = m.put(x), m.put(w), m.put(ws), m.room(M * N * 4)
    m.upload(fill=0xff)
    backend.F4Dense(dense_args(m, ax, 0, aw, aws, 0, ao, M, K, N, dt, F32, False))
    assert_within(m.back(ao, np.float32, (M, N)).astype(np.float64), *dense_want(xv, R.values(w, ws), None, 0, F32, kind), "odd")
    assert np.all(m.back(ao + M * N * 4, np.uint8, (64,)) == 0xff)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("M", [12, 90, 300])
@pytest.mark.parametrize("N", [72, 128])
def test_odd_inputs_of_experts(backend, M, N, kind):
    E, K = 3, 131
    rng = np.random.default_rng(M)
    x, dt, _, xv = make_x(rng, M, K, kind)
    w, ws = R.random_codes(rng, E, K, N)
    ends = [M // 3, M // 3, M - 2]
    m = Memory(backend)
    ax, aw, aws, ao, aoff = m.put(x), m.put(w), m.put(ws), m.room(M * N * 4), m.put(np.array([0, *ends], np.int32))
    m.upload(fill=0xff)
    backend.F4ExpertDense(dense_args(m, ax, 0, aw, aws, 0, ao, M, K, N, dt, F32, False, experts=(aoff, E)))
    got, start = m.back(ao, np.float32, (M, N)).astype(np.float64), 0
    for e, end in enumerate(ends):
        if end > start:
            assert_within(got[start:end], *dense_want(xv[start:end], R.values(w[e], ws[e]), None, 0, F32, kind), f"expert {e}")
        start = end
    assert not got[ends[-1]:].any()


@pytest.mark.parametrize("kind,M,K,N,plan", [
    ("bf16", 20, 1024, 64, "f4_columns 512x4 slices 4"), ("f32", 20, 1024, 64, "f4_columns 512x4 slices 4"), ("f4", 20, 1024, 64, "f4_columns 512x4 slices 4"),
    ("bf16", 700, 256, 320, "f4_wide"), ("f32", 700, 256, 320, "f4_wide"), ("f4", 700, 256, 320, "f4_wide")])
def test_offsets_that_do_not_ascend(backend, kind, M, K, N, plan):
    """Whatever offsets hold, nothing outside the result is written, the call ends, and the next one with offsets in order is right."""
    E = 70
    assert plan_of(backend, kind, False, M, K, N, E).startswith(plan)
    rng = np.random.default_rng(M)
    x, dt, xs, xv = make_x(rng, M, K, kind)
    w, ws = R.random_codes(rng, E, K, N)
    ordered = np.sort(rng.integers(0, M + 1, E + 1))
    ordered[0] = 0
    for off in (np.tile([M, 0], E)[:E + 1], np.arange(E, -1, -1) * M // E, np.tile([0x7fffffff, -0x80000000], E)[:E + 1], rng.integers(0, M, E + 1), ordered):
        m = Memory(backend)
        ax, aw, aws, ao, aoff = m.put(x), m.put(w), m.put(ws), m.room(M * N * 4), m.put(off.astype(np.int32))
        axs = m.put(xs) if xs is not None else 0
        m.upload(fill=0x5a)
        backend.F4ExpertDense(dense_args(m, ax, axs, aw, aws, 0, ao, M, K, N, dt, F32, False, experts=(aoff, E)))
        flat = m.buf.ToFlatData()
        end = ao + M * N * 4
        assert np.all(flat[end:aoff] == 0x5a)
        for at, a in m.parts:
            assert np.array_equal(flat[at:at + a.nbytes], np.ascontiguousarray(a).view(np.uint8).ravel())
    got = m.back(ao, np.float32, (M, N)).astype(np.float64)
    for e in np.flatnonzero(ordered[1:] > ordered[:-1]):
        s = slice(ordered[e], ordered[e + 1])
        assert_within(got[s], *dense_want(xv[s], R.values(w[e], ws[e]), None, 0, F32, kind), f"expert {e}")
    assert not got[ordered[-1]:].any()


@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("M", [2, 70])
def test_bias_in_bf16(backend, M, oi):
    E, K, N = 2, 96, 66
    rng = np.random.default_rng(M)
    x, dt, _, xv = make_x(rng, M, K, "bf16")
    w, ws = R.random_codes(rng, E, *((N, K) if oi else (K, N)))
    b = store(rng.standard_normal((E, N)).astype(np.float32), BF16)
    cfg = ca.F4DenseConfig(Activation=ca.ActivationTanh, WeightLayout=ca.DenseLayout(int(oi)), OutputDType=F32)
    ends = np.array([0, M // 2, M], np.int32)
    one, many = run_graph(backend, lambda f, p: [f.FusedF4Dense(p["x"], None, p["w0"], p["s0"], p["b0"], cfg),
                                                 f.FusedF4ExpertDense(p["x"], None, p["o"], p["w"], p["ws"], p["b"], cfg)],
                          {"x": (x, dt), "w0": (w[0], F4), "s0": (ws[0], E8), "b0": (b[0], BF16), "o": (ends, I32), "w": (w, F4), "ws": (ws, E8),
                           "b": (b, BF16)})
    bv = to_f64(b, BF16)
    for e, got in ((0, one), (0, many[:M // 2]), (1, many[M // 2:])):
        wv, part = R.values(w[e], ws[e]), xv if got is one else xv[:M // 2] if e == 0 else xv[M // 2:]
        assert_within(got.astype(np.float64), *dense_want(part, wv.T if oi else wv, bv[e], 5, F32, "bf16"), f"expert {e}")


@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("kind", ["f4", "bf16", "f32"])
@pytest.mark.parametrize("M", [50, 5000])
def test_as_many_experts_as_there_may_be(backend, M, kind, oi):
    E, K, N = ca.MaxExperts, 64, 32
    rng = np.random.default_rng(M)
    x, dt, xs, xv = make_x(rng, M, K, kind)
    w, ws = R.random_codes(rng, E, *((N, K) if oi else (K, N)))
    off = np.sort(rng.integers(0, M + 1, E + 1)).astype(np.int32)
    off[0], off[-1] = 0, M - 3
    off = np.minimum(off, M - 3)
    inputs = {"x": (x, dt), "o": (off, I32), "w": (w, F4), "ws": (ws, E8)}
    if xs is not None:
        inputs["xs"] = (xs, E8)
    cfg = ca.F4DenseConfig(WeightLayout=ca.DenseLayout(int(oi)), OutputDType=F32)
    got, = run_graph(backend, lambda f, p: [f.FusedF4ExpertDense(p["x"], p.get("xs"), p["o"], p["w"], p["ws"], None, cfg)], inputs)
    want, bound = np.zeros((M, N)), np.zeros((M, N))
    for e in np.flatnonzero(off[1:] > off[:-1]):
        s = slice(off[e], off[e + 1])
        wv = R.values(w[e], ws[e])
        want[s], bound[s] = dense_want(xv[s], wv.T if oi else wv, None, 0, F32, kind)
    assert_within(got.astype(np.float64), want, bound, "1024 experts")


def test_codes_through_ops_that_take_them(backend):
    """Identity, Reshape and Bitcast of codes and scales, constants of them, and a parameter as a result."""
    rng = np.random.default_rng(1)
    w, ws = R.random_codes(rng, 6, 64)
    x = rng.standard_normal((2, 64)).astype(np.float32)

    def build(f, p):
        c, s = f.Identity(p["w"]), f.Identity(p["ws"])
        const = f.Constant(w.ravel(), 6, 64, dtype=F4), f.Constant(ws.ravel(), 6, 2, dtype=E8)
        halves = f.Reshape(c, 2, 3, 64), f.Reshape(s, 2, 3, 2)
        bytes_ = f.Bitcast(f.Reshape(c, 6, 32, 2), ca.Uint8)
        cfg = ca.F4DenseConfig(WeightLayout=ca.DenseLayoutOutputsInput)
        return [p["w"], c, s, bytes_, f.FusedF4Dequantize(*halves, F32), f.FusedF4Dense(p["x"], None, c, s, None, cfg),
                f.FusedF4Dense(p["x"], None, *const, None, cfg), f.FusedF4Dequantize(f.Reshape(f.Bitcast(bytes_, F4), 6, 64), s, F32)]

    same, c, s, raw, values, y, yc, back = run_graph(backend, build, {"w": (w, F4), "ws": (ws, E8), "x": (x, F32)})
    assert np.array_equal(same, w) and np.array_equal(c, w) and np.array_equal(s, ws) and np.array_equal(raw, w)
    v = R.values(w, ws).astype(np.float32)
    assert np.array_equal(values, v.reshape(2, 3, 64)) and np.array_equal(back, v) and np.array_equal(y, yc)
    assert_within(y.astype(np.float64), *dense_want(x.astype(np.float64), v.T.astype(np.float64), None, 0, F32, "f32"), "y")
