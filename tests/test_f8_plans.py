"""Which tile and how many slices the operators on 8-bit blocks take: the plans of the GPU tests' cases, without a GPU."""
import pytest

from tests.test_f8_abi import dense_args, wgrad_args
from tests.test_gpu_f8 import BF16, F32, SLICED, WGRAD
from tests.test_gpu_f8_precision import KERNELS
from tests.test_gpu_f8_repeats import SHAPES
from tests.test_gpu_f8_tiles import TILES


def dense_plan(b, M, K, N, oi, out, **kw):
    return b.F8DensePlan(dense_args(x=1 << 40, w=2 << 40, w_scale=3 << 40, x_scale=4 << 40, out=5 << 40, M=M, K=K, N=N,
                                    weight_layout=int(oi), out_dtype=int(out), **kw))


def wgrad_plan(b, M, K, N, oi, dt):
    return b.F8WeightGradientPlan(wgrad_args(x=1 << 40, x_scale=2 << 40, dy=3 << 40, out=4 << 40, M=M, K=K, N=N, weight_layout=int(oi),
                                             dy_dtype=int(dt)))


def test_plan_names(host_backend):
    assert dense_plan(host_backend, 2048, 4096, 4096, True, BF16) == "f8_dense_tiles 256x128 slices 1"
    assert dense_plan(host_backend, 1, 4096, 11008, True, BF16) == "f8_dense_skinny"
    assert dense_plan(host_backend, 97, 4099, 4096, True, BF16).startswith("f8_dense_staged ")
    assert dense_plan(host_backend, 97, 4096, 4099, False, BF16).startswith("f8_dense_staged ")
    assert wgrad_plan(host_backend, 2048, 4096, 14336, True, BF16) == "f8_wgrad_bf16 256x256 slices 1"
    assert wgrad_plan(host_backend, 333, 1536, 384, False, F32) == "f8_wgrad_f32 128x128 slices 4"


@pytest.mark.parametrize("dt", [BF16, F32])
def test_plan_of_float_x_is_that_of_its_codes(host_backend, dt):
    """From five rows on the codes are made first, in memory of the call's own: what counts is the product over them."""
    for M, K, N, oi in [(5, 4096, 11008, True), (16, 4096, 4096, True), (17, 4096, 4096, True), (8, 4096, 4096, False), (97, 4096, 14336, True),
                        (97, 4095, 4096, True)]:
        want = dense_plan(host_backend, M, K, N, oi, BF16)
        for off in (0, 4):
            kw = dict(x=(1 << 40) + off, x_scale=None, x_dtype=int(dt), out=5 << 40, w=2 << 40, w_scale=3 << 40)
            got = host_backend.F8DensePlan(dense_args(**kw, M=M, K=K, N=N, weight_layout=int(oi), out_dtype=int(BF16)))
            assert got == want, (M, K, N, oi, off)
    kw = dict(x=1 << 40, x_scale=None, x_dtype=int(dt), out=5 << 40, w=2 << 40, w_scale=3 << 40)
    assert host_backend.F8DensePlan(dense_args(**kw, M=4, K=4096, N=4096, weight_layout=1)) == "f8_dense_skinny"


def test_sliced_products_are_sliced(host_backend):
    """test_gpu_f8.SLICED: three products cut into slices, and one that is not."""
    slices = [int(dense_plan(host_backend, M, K, N, oi, out).split()[-1]) for M, K, N, oi, out in SLICED]
    assert all(s > 1 for s in slices[:3]) and len(set(slices[:3])) > 1 and slices[3] == 1, slices


@pytest.mark.parametrize("M,K,N,oi,out,tile,sliced", TILES)
def test_tiles_are_the_ones_named(host_backend, M, K, N, oi, out, tile, sliced):
    name, slices = dense_plan(host_backend, M, K, N, oi, out).split(" slices ")
    assert name == tile and (int(slices) > 1) == sliced


def test_repeats_reach_every_weight_gradient_tile(host_backend):
    """Both tiles of both types, in one slice and in several where the rule has such, whole rows and odd ones."""
    plans = set()
    for M, K, N, oi, dt in SHAPES:
        name, slices = wgrad_plan(host_backend, M, K, N, oi, dt).split(" slices ")
        plans.add((name, int(slices) > 1, K % 16 == 0 and N % 8 == 0))
    for name in ("f8_wgrad_bf16 128x128", "f8_wgrad_f32 128x128"):
        assert {(s, w) for n, s, w in plans if n == name} >= {(True, True), (True, False)}, plans
    for name in ("f8_wgrad_bf16 128x128", "f8_wgrad_bf16 256x256"):
        assert {(s, w) for n, s, w in plans if n == name} >= {(False, True), (False, False)}, plans
    assert any(n == "f8_wgrad_f32 256x256" for n, _, _ in plans)
    assert any(wgrad_plan(host_backend, M, K, N, True, dt).endswith("slices 1") for M, K, N in WGRAD for dt in (F32, BF16))


def test_precision_cases_take_the_kernels_they_name(host_backend):
    plans = [dense_plan(host_backend, M, K, N, oi, BF16).split()[0] for M, K, N, oi in KERNELS]
    assert plans == ["f8_dense_skinny"] * 2 + ["f8_dense_tiles"] * 2 + ["f8_dense_staged"] * 2
