"""CPU test: the sizes that the GPU tests of the matrix kernels run take every tile in every way."""
import ctypes

import pytest

import head_tiles as ht
from collie_amd import _lib


@pytest.mark.parametrize('dtype', [_lib.F32, _lib.BF16, _lib.F16])
def test_the_listed_sizes_take_every_tile_in_every_way(dtype):
    cases = ht.FLOAT32 if dtype == _lib.F32 else ht.SIXTEEN_BITS
    seen = {(name, gated, *ht.plan(dtype, product, gated, m, n_in, n_out))
            for gated, m, n_in, n_out in cases for name, product in ht.PRODUCTS.items()}
    every = {(name, gated, tile, way) for name in ht.PRODUCTS for gated in (0, 1)
             for tile in ht.TILES for way in ('whole', 'cut', 'mixed')}
    assert seen == every


def test_plans_of_few_rows_and_refusals():
    assert ht.plan(_lib.BF16, 0, 0, 64, 100, 100) is None       # streamed weights
    assert ht.plan(_lib.BF16, 1, 0, 64, 100, 100) is not None
    lib, out = _lib.load(), (ctypes.c_int64 * 5)()
    for args in ((9, 0, 0, 100, 8, 8, out), (0, 3, 0, 100, 8, 8, out), (0, 0, 0, 0, 8, 8, out),
                 (0, 0, 0, 100, 0, 8, out), (0, 0, 0, 100, 8, 1 << 20, out), (0, 0, 0, 100, 8, 8, None)):
        assert lib.collie_layer_plan(*args) == -1
        assert lib.collie_last_error()
