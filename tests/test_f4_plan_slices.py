"""The slices that a plan names are those that K is cut into: whole steps each, as even as they come, none of them empty."""
import pytest

from f4_tile_cases import plan_of

STEP = {"f4_tiles": 256, "f4_wide": 64, "f4_columns": 64}


@pytest.mark.parametrize("M,N,E", [(1, 4096, 0), (2, 11008, 0), (3, 512, 0), (4, 4096, 0), (16, 1536, 0), (33, 776, 0), (6, 4096, 3), (12, 1536, 8)])
@pytest.mark.parametrize("oi", [True, False])
@pytest.mark.parametrize("x", ["f4", "bf16", "f32"])
def test_no_slice_is_empty(host_backend, x, oi, M, N, E):
    for K in (2, 64, 130, 320, 514, 1000, 1216, 2880, 4096, 4160, 5000, 11008, 14336, 33000):
        kernel, *more = plan_of(host_backend, x, oi, M, K, N, E).split()
        if kernel == "f4_skinny":
            continue
        slices, steps = int(more[-1]), -(-K // STEP[kernel])
        per = -(-steps // slices)
        assert -(-steps // per) == slices, (K, kernel, slices)


def test_columns_of_65_steps(host_backend):
    assert plan_of(host_backend, "bf16", False, 1, 4160, 4096, 0) == "f4_columns 512x1 slices 13"  # 5 steps each
    assert plan_of(host_backend, "bf16", False, 1, 4096, 4096, 0) == "f4_columns 512x1 slices 16"
