"""Scales of the 8-bit products: of one tile and the next, and of magnitudes whose product no fp32 number holds."""
import numpy as np
import pytest

from tests.test_fp8_gpu import E4M3, Eight, check_product, random_codes, up

pytestmark = pytest.mark.gpu
F = np.float32


def operand(lib, rng, r, c, spread, block=1):
    scale = np.exp2(rng.integers(-spread, spread + 1, (up(c, 128) // 128, up(r, block) // block))).astype(F)
    return Eight(lib, r, c, E4M3, block).set(random_codes(rng, r, c, E4M3), scale)


# several tiles for each pair of CTAs, an odd number of K-blocks, a scale for every row on both sides and no two alike: a tile's last scales and the
# next one's first lie in the same place
@pytest.mark.parametrize("m,n,k", [(4100, 4300, 100), (4100, 4300, 300), (4000, 4800, 300), (2100, 9000, 640)])
def test_scales_of_a_tile_and_the_next(lib, m, n, k):
    rng = np.random.default_rng(k)
    check_product(lib, operand(lib, rng, m, k, 12), operand(lib, rng, n, k, 12), 0, rng)
