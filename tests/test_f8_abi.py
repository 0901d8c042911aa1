"""Operators on 8-bit floating-point blocks without a GPU: shapes, refusals, the plans, the oracle."""
import ctypes as C

import numpy as np
import pytest

import compute_amd as ca
from compute_amd import _lib
from oracle import f8_ref as R

F8, F32, BF16 = ca.F8E4M3FN, ca.Float32, ca.BFloat16


def params(host_backend, **shapes):
    bld = host_backend.Builder("f8")
    f = bld.Main()
    return f, {n: f.Parameter(n, s) for n, s in shapes.items()}


def test_capabilities(host_backend):
    caps = host_backend.Capabilities()
    for op in (ca.OpType.F8Quantize, ca.OpType.F8Dense, ca.OpType.F8WeightGradient, ca.OpType.F8ActivationGradient):
        assert caps.Extensions.get(op) and op not in caps.Operations  # those of the reference only
    assert caps.DTypes.get(F8)
    assert ca.Shape(F8, 3, 5).byte_size() == 15


def test_shapes(host_backend):
    f, p = params(host_backend, x=ca.Shape(BF16, 2, 3, 300), w=ca.Shape(F8, 300, 130), ws=ca.Shape(F32, 3, 2),
                  w2=ca.Shape(F32, 130, 300))
    codes, scale = f.FusedF8Quantize(p["x"])
    assert f.Shape(codes) == ca.Shape(F8, 2, 3, 300) and f.Shape(scale) == ca.Shape(F32, 2, 3, 3)
    wc, wsc = f.FusedF8Quantize(p["w2"], 128)
    assert f.Shape(wc) == ca.Shape(F8, 130, 300) and f.Shape(wsc) == ca.Shape(F32, 2, 3)
    y = f.FusedF8Dense(codes, scale, p["w"], p["ws"], None)
    assert f.Shape(y) == ca.Shape(BF16, 2, 3, 130)
    y = f.FusedF8Dense(p["x"], None, wc, wsc, None, ca.F8DenseConfig(WeightLayout=ca.DenseLayoutOutputsInput, OutputDType=F32))
    assert f.Shape(y) == ca.Shape(F32, 2, 3, 130)
    assert f.Shape(f.FusedF8WeightGradient(codes, scale, y)) == ca.Shape(F32, 300, 130)
    assert f.Shape(f.FusedF8WeightGradient(codes, scale, y, ca.DenseLayoutOutputsInput, BF16)) == ca.Shape(BF16, 130, 300)
    dz, dup = f.FusedF8ActivationGradient(codes, scale, p["x"], ca.ActivationSilu, codes, scale)
    assert f.Shape(dz) == f.Shape(dup) == ca.Shape(BF16, 2, 3, 300)


@pytest.mark.parametrize("what,err", [
    ("quantize_int", ca.ErrNotImplemented), ("quantize_f64", ca.ErrNotImplemented), ("quantize_rows", ca.ErrNotImplemented),
    ("quantize_rank3_tiles", ca.ComputeError), ("dense_no_scale", ca.ComputeError), ("dense_float_scale", ca.ComputeError),
    ("dense_scale_shape", ca.ComputeError), ("dense_weight_dtype", ca.ErrNotImplemented), ("dense_weight_shape", ca.ComputeError),
    ("dense_weight_scale", ca.ComputeError), ("dense_layout", ca.ComputeError), ("dense_out", ca.ErrNotImplemented),
    ("dense_bias", ca.ComputeError), ("dense_act", ca.ComputeError), ("wgrad_rows", ca.ComputeError),
    ("wgrad_dtype", ca.ErrNotImplemented), ("wgrad_float_x", ca.ErrNotImplemented), ("agrad_shape", ca.ComputeError),
    ("agrad_up_shape", ca.ComputeError), ("agrad_act", ca.ComputeError), ("convert_to", ca.ErrNotImplemented),
    ("convert_from", ca.ErrNotImplemented), ("dot", ca.ComputeError), ("add", ca.ComputeError), ("neg", ca.ComputeError),
    ("gelu", ca.ErrNotImplemented), ("reduce", ca.ComputeError), ("other_builder", ca.ComputeError)])
def test_graph_refusals(host_backend, what, err):
    f, p = params(host_backend, x=ca.Shape(BF16, 6, 300), c=ca.Shape(F8, 6, 300), s=ca.Shape(F32, 6, 3), w=ca.Shape(F8, 300, 130),
                  ws=ca.Shape(F32, 3, 2), i=ca.Shape(ca.Int32, 6, 300), d=ca.Shape(ca.Float64, 6, 300), dy=ca.Shape(BF16, 6, 130),
                  x3=ca.Shape(F32, 2, 3, 300), b=ca.Shape(F32, 131), dy5=ca.Shape(BF16, 5, 130), c2=ca.Shape(F8, 6, 299),
                  dyi=ca.Shape(ca.Float16, 6, 130))
    x, c, s, w, ws = (p[k] for k in ("x", "c", "s", "w", "ws"))
    _, q = params(host_backend, x=ca.Shape(BF16, 6, 300))
    call = {
        "quantize_int": lambda: f.FusedF8Quantize(p["i"]), "quantize_f64": lambda: f.FusedF8Quantize(p["d"]),
        "quantize_rows": lambda: f.FusedF8Quantize(x, 64), "quantize_rank3_tiles": lambda: f.FusedF8Quantize(p["x3"], 128),
        "dense_no_scale": lambda: f.FusedF8Dense(c, None, w, ws, None), "dense_float_scale": lambda: f.FusedF8Dense(x, s, w, ws, None),
        "dense_scale_shape": lambda: f.FusedF8Dense(c, ws, w, ws, None), "dense_weight_dtype": lambda: f.FusedF8Dense(c, s, x, ws, None),
        "dense_weight_shape": lambda: f.FusedF8Dense(c, s, c, s, None), "dense_weight_scale": lambda: f.FusedF8Dense(c, s, w, s, None),
        "dense_layout": lambda: f.FusedF8Dense(c, s, w, ws, None, ca.F8DenseConfig(WeightLayout=2)),
        "dense_out": lambda: f.FusedF8Dense(c, s, w, ws, None, ca.F8DenseConfig(OutputDType=ca.Float16)),
        "dense_bias": lambda: f.FusedF8Dense(c, s, w, ws, p["b"]), "dense_act": lambda: f.FusedF8Dense(c, s, w, ws, None, ca.F8DenseConfig(9)),
        "wgrad_rows": lambda: f.FusedF8WeightGradient(c, s, p["dy5"]), "wgrad_dtype": lambda: f.FusedF8WeightGradient(c, s, p["dyi"]),
        "wgrad_float_x": lambda: f.FusedF8WeightGradient(x, s, p["dy"]),
        "agrad_shape": lambda: f.FusedF8ActivationGradient(c, s, p["dy"], 1),
        "agrad_up_shape": lambda: f.FusedF8ActivationGradient(c, s, x, 1, p["c2"], s),
        "agrad_act": lambda: f.FusedF8ActivationGradient(c, s, x, -1), "convert_to": lambda: f.ConvertDType(x, F8),
        "convert_from": lambda: f.ConvertDType(c, F32), "dot": lambda: f.DotGeneral(c, [1], [], w, [0], []),
        "add": lambda: f.Add(c, c), "neg": lambda: f.Neg(c), "gelu": lambda: f.FusedGelu(c, True), "reduce": lambda: f.ReduceSum(c, 0),
        "other_builder": lambda: f.FusedF8Quantize(q["x"]),
    }[what]
    with pytest.raises(err):
        call()


def dense_args(**kw):
    a = _lib.mx_f8_dense_args(x=1 << 20, x_scale=2 << 20, w=3 << 20, w_scale=4 << 20, out=5 << 20, M=4, K=256, N=256, x_dtype=int(F8),
                              out_dtype=int(BF16), weight_layout=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def wgrad_args(**kw):
    a = _lib.mx_f8_weight_grad_args(x=1 << 20, x_scale=2 << 20, dy=3 << 20, out=4 << 20, M=4, K=256, N=256, dy_dtype=int(BF16),
                                    out_dtype=int(F32))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [dict(M=-1), dict(K=1 << 30), dict(N=1 << 30), dict(x=0), dict(x_scale=None), dict(w=0), dict(w_scale=0),
                                dict(out=0), dict(out=1 << 20), dict(out=(1 << 20) + 1000), dict(out=4 << 20), dict(out_dtype=int(ca.Int8)),
                                dict(x_dtype=int(ca.Int8)), dict(x_dtype=int(BF16)), dict(weight_layout=2), dict(activation=6),
                                dict(out=(5 << 20) + 1), dict(x_scale=(2 << 20) + 2), dict(bias=(6 << 20) + 1, bias_dtype=int(BF16)),
                                dict(bias=6 << 20, bias_dtype=int(F8)), dict(bias=5 << 20, bias_dtype=int(F32)),
                                dict(M=1 << 29, K=1 << 29)])
def test_dense_arguments_refused(host_backend, kw):
    """The plan checks what the call checks, before anything is launched."""
    assert host_backend.F8DensePlan(dense_args())
    with pytest.raises(ca.ComputeError):
        host_backend.F8DensePlan(dense_args(**kw))


@pytest.mark.parametrize("kw", [dict(M=-1), dict(K=1 << 30), dict(x=0), dict(x_scale=0), dict(dy=0), dict(out=0), dict(out=3 << 20),
                                dict(dy_dtype=int(F8)), dict(out_dtype=int(ca.Float64)), dict(weight_layout=-1), dict(dy=(3 << 20) + 1),
                                dict(out=(4 << 20) + 2)])
def test_weight_gradient_arguments_refused(host_backend, kw):
    assert host_backend.F8WeightGradientPlan(wgrad_args())
    with pytest.raises(ca.ComputeError):
        host_backend.F8WeightGradientPlan(wgrad_args(**kw))


def test_device_calls_fail_host_only(host_backend):
    for call, a in ((host_backend.F8Dense, dense_args()), (host_backend.F8WeightGradient, wgrad_args()),
                    (host_backend.F8Quantize, _lib.mx_f8_quantize_args()), (host_backend.F8ActivationGradient, _lib.mx_f8_act_grad_args())):
        with pytest.raises(ca.ErrNoDevice):
            call(a)
    assert host_backend._lib.mx_f8_dense(None, C.byref(dense_args())) == _lib.MX_ERR_INVALID


def test_float_data_for_codes_refused(host_backend):
    with pytest.raises(ca.ComputeError):
        host_backend.BufferFromFlatData(0, np.zeros(4, np.float32), ca.Shape(F8, 4))


# -- the oracle itself ---------------------------------------------------------------------------
def test_oracle_codes():
    assert R.VALUES[0x7e] == 448 and R.VALUES[0x08] == 2.0 ** -6 and R.VALUES[0x01] == 2.0 ** -9 and R.VALUES[0x38] == 1
    finite = [c for c in range(256) if (c & 127) != 127]
    assert np.array_equal(R.encode(R.VALUES[finite]), np.array(finite, np.uint8))
    # halfway between neighbours: the even code
    for lo in range(126):
        mid = (R.VALUES[lo] + R.VALUES[lo + 1]) / 2
        assert R.encode(np.array([mid]))[0] == (lo if lo % 2 == 0 else lo + 1)


@pytest.mark.parametrize("top,want", [(448.0, 1.0), (np.nextafter(448.0, 449), 2.0), (449.0, 2.0), (224.0, 0.5), (1.75, 2.0 ** -8), (0.0, 1.0),
                                      (1e-45, 2.0 ** -126), (3.4e38, 2.0 ** 120)])
def test_oracle_scales(top, want):
    assert R.scale_of(top) == want


@pytest.mark.parametrize("kind", range(6))
def test_oracle_slopes_are_differences(kind):
    z = np.linspace(-6.03, 6.01, 301)
    h = 1e-5
    d = (R.act(z + h, kind) - R.act(z - h, kind)) / (2 * h)
    # a difference that spans a corner (ReLU at 0, HardSwish at -3 and 3: one point of this grid) is the
    # mean of two slopes and no derivative
    smooth = np.all([np.abs(z - c) > h for c in {2: [0], 4: [-3, 3]}.get(kind, [np.inf])], axis=0)
    assert smooth.sum() >= 300
    # central difference: h^2 / 6 * |third derivative| (below 3 here) + rounding 8 * 2^-53 / h
    assert np.max(np.abs(d - R.slope(z, kind))[smooth]) <= 0.5 * h * h + 8 * 2.0 ** -53 / h
