"""The gated product's planner (csrc/gated_plan.h) on the CPU, for 256 CUs: the faster form of the forward pass where both were
measured, and the forms and tiles that the GPU tests' shapes are there for."""

import pytest

from tests.test_gpu_gated import FEW, LARGE_TILES, ROWS, ROWS_SHAPES, TILES, plan

# rows x channels -> hidden columns, on either side of the rule where the two forms were measured 3% and more apart
FASTER = {
    ROWS: [(49152, 64, 256), (65536, 64, 256), (320000, 64, 256), (24576, 64, 512), (16384, 64, 1024), (81920, 16, 64),
           (49152, 128, 512), (24576, 128, 1024), (196608, 128, 128), (160000, 128, 512)],
    TILES: [(16384, 64, 256), (32768, 64, 256), (40000 - 1, 64, 256), (16384, 64, 512), (8192, 64, 1024), (32768, 128, 512),
            (16384, 128, 1024), (81920, 128, 128), (65, 64, 1 << 20), (8191, 64, 1 << 20), (320000, 136, 256)],
    FEW: [(1, 64, 256), (64, 16, 1 << 20)],
}


@pytest.mark.parametrize("form", FASTER)
def test_forward_form(form):
    for shape in FASTER[form]:
        assert plan(*shape)[0] == form, shape


def test_shapes_of_the_gpu_tests():
    for shape in ROWS_SHAPES:
        assert plan(*shape)[0] == ROWS, shape
    for shape, fields in LARGE_TILES.items():
        assert all(plan(*shape)[i] == v for i, v in fields.items()), shape
