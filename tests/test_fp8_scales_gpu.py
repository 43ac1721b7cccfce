"""8-bit products: the scales of one tile and the next, and what a product leaves to wait for."""
import subprocess
import sys

import numpy as np
import pytest

from tests.conftest import ROOT
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


def test_waiting_for_the_device_costs_no_more_after_a_product():
    """In a process of its own: the products' time-out flag is not fetched from the device by every later call of eddlb200_sync."""
    code = """
import time
import numpy as np
from eddl_b200 import capi
L = capi.lib()
L.call("init", 0)
def least():
    times = []
    for _ in range(10):
        t = time.perf_counter()
        for _ in range(200):
            L.call("sync", 0)
        times.append((time.perf_counter() - t) / 200 * 1e6)
    return min(times)
L.sync()
before = least()
q, s, c = L.to_device(np.zeros((128, 128)), dtype=np.uint8), L.zeros((1, 128)), L.empty((128, 128))
L.call("fp8_mult2d", 0, q, 128, s, 0, 1, q, 128, s, 0, 1, c, 0, 128, 128, 128)
L.sync()
after = least()
assert after <= before + 5, (before, after)          # 1.6 us; a blocking copy of a word adds 11
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, timeout=300)
