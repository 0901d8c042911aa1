"""Plans of products without a result: nothing is launched, and asking is no error.

Whatever kernel the sizes would lead to (few rows in either layout, tiles of each kind), a product without rows or columns has none.
"""
import pytest

from f4_tile_cases import plan_of


@pytest.mark.parametrize("E", [0, 1, 5])
@pytest.mark.parametrize("M,K,N", [(0, 256, 256), (0, 0, 256), (0, 4096, 128), (7, 256, 0), (700, 256, 0), (7, 0, 0), (0, 256, 0), (0, 0, 0)])
@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("x", ["f4", "bf16", "f32"])
def test_nothing_to_compute(host_backend, x, oi, M, K, N, E):
    assert plan_of(host_backend, x, oi, M, K, N, E) == "nothing"


@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("x", ["f4", "bf16", "f32"])
def test_no_terms_is_a_product(host_backend, x, oi):
    """K = 0: act(bias), from a kernel."""
    assert plan_of(host_backend, x, oi, 7, 0, 256, 0).startswith("f4_wide")


@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("M,N", [(7, 256), (700, 4096), (4096, 11008)])
def test_no_terms_have_no_parts(host_backend, oi, M, N):
    """Without terms nothing of x is read, and float32 x is not three arrays: the tile is one of those for a single array."""
    assert plan_of(host_backend, "f32", oi, M, 0, N, 0) == plan_of(host_backend, "bf16", oi, M, 0, N, 0)
