"""
Sizes of linear and gated layers whose products between them take every tile of the matrix kernels, in
every way: whole tiles only, tiles cut along the depth only, and whole ones followed by cut ones.
``collie_layer_plan`` says which (``test_head_tiles_cpu.py`` holds this list to it).
"""
import ctypes

from collie_amd import _lib

PRODUCTS = {'forward': 0, 'dx': 1, 'dw': 2}
TILES = [(128, 64), (128, 128), (256, 256)]

# (gated, rows, n_in, n_out)
SIXTEEN_BITS = [
    (0, 65, 65, 65), (1, 65, 65, 65), (1, 65, 6000, 515), (0, 2050, 3001, 65), (0, 130, 1500, 8200),
    (1, 12000, 515, 257), (0, 3001, 1030, 2050), (1, 700, 4100, 1500), (1, 6000, 1500, 700),
    (0, 2050, 6000, 2050), (1, 6000, 2050, 1030), (0, 6000, 3001, 1500), (0, 1500, 3001, 8200),
    (1, 3001, 16390, 1030), (0, 4100, 8200, 4100), (1, 1500, 3001, 16390), (1, 33000, 515, 65),
    (0, 33000, 515, 130), (1, 700, 130, 16390), (0, 33000, 130, 700), (0, 700, 130, 33000),
    (1, 24000, 257, 515),
]
FLOAT32 = [
    (0, 65, 65, 65), (1, 65, 65, 65), (1, 257, 257, 130), (0, 257, 257, 257), (1, 130, 6000, 515),
    (0, 700, 16390, 65), (0, 257, 200, 33000), (1, 33000, 515, 65), (1, 4100, 4100, 200),
    (0, 3001, 4100, 700), (1, 1500, 1500, 3001), (0, 130, 3001, 33000), (1, 257, 130, 16390),
    (0, 24000, 257, 257), (0, 515, 16390, 700), (1, 700, 700, 8200), (0, 1500, 12000, 1500),
    (1, 1500, 1500, 6000), (1, 33000, 130, 130), (0, 257, 130, 33000), (1, 700, 16390, 200),
    (0, 700, 700, 16390), (1, 700, 24000, 700), (0, 24000, 1500, 700),
]


def plan(dtype, product, gated, m, n_in, n_out):
    """((tile rows, tile columns), 'whole' | 'cut' | 'mixed'); None for the kernel without tiles."""
    out = (ctypes.c_int64 * 5)()
    rc = _lib.load().collie_layer_plan(dtype, product, gated, m, n_in, n_out, out)
    assert rc == 0, _lib.load().collie_last_error()
    rows, cols, tiles, whole, parts = out
    if rows == 0:
        return None
    assert 0 <= whole <= tiles and parts >= 1 and (whole == tiles) == (parts == 1)
    return (rows, cols), 'whole' if parts == 1 else 'cut' if whole == 0 else 'mixed'
