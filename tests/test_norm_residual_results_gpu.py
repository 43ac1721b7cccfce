"""The backward pass of the residual norms for every choice of wanted results, with results and inputs off the 16-byte grid."""
import ctypes

import numpy as np
import pytest

from eddl_b200.capi import DeviceArray
from tests import test_norm_residual_gpu as base

pytestmark = pytest.mark.gpu
F = np.float32


class Piece(DeviceArray):
    """A tensor that begins 4 bytes behind a 16-byte border, as a piece of one flat buffer does; what lies around it has to stay."""

    def __init__(self, lib, arr):
        arr = np.ascontiguousarray(arr, dtype=F)
        self.lib, self.dev, self.shape, self.size, self.dtype = lib, 0, arr.shape, arr.size, arr.dtype
        self.room = lib.to_device(np.concatenate([np.full(1, 5, F), arr.ravel(), np.full(7, 5, F)]))
        self.addr = self.room.addr + 4
        self.ptr = ctypes.c_void_p(self.addr)

    def numpy(self):
        around = np.delete(self.room.numpy(), np.s_[1:1 + self.size])
        assert np.all(around == 5)
        return super().numpy()

    def __del__(self):
        pass


class Pieces:
    """The library as the base tests use it; tensors made after `after` calls of the forward pass are pieces."""

    def __init__(self, lib, after):
        self.lib, self.empty, self.left = lib, lib.empty, after

    def call(self, name, *args):
        self.lib.call(name, *args)
        self.left -= name == "norm_residual_fwd"

    def to_device(self, arr):
        return self.lib.to_device(arr) if self.left > 0 else Piece(self.lib, arr)


# one slice a group: a block writes dgate itself
@pytest.mark.parametrize("dims", [(1, 1, 300), (1, 1, 512), (3, 1, 768), (700, 1, 512), (5, 1, 1028), (2, 1, 1400), (1, 1, 2048), (1, 1, 2304), (2, 1, 4096), (3, 1, 4500), (1, 1, 16384)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("inc_g", [0, 1])
def test_dgate_off_the_grid(lib, monkeypatch, dims, kind, inc_g):
    monkeypatch.setattr(base, "wanted", lambda c: ["dgate", "dg2"])
    base.check(Pieces(lib, 1), base.Case(31, *dims, kind, beta=bool(kind)), inc_g=inc_g)


# the blocks of a cluster write into one another's memory with their first row: as soon as they are there (nothing to read but one gradient), and
# more clusters than the device holds
@pytest.mark.parametrize("dims", [(1, 1, 4097), (1, 2, 16384), (200, 1, 6000)])
@pytest.mark.parametrize("kind", [0, 1])
def test_first_exchange_of_a_cluster(lib, dims, kind):
    c = base.Case(32, *dims, kind).forward()
    dev = base.Device(lib, c).forward()
    c.backward(dh=False)
    got = []
    for _ in range(20):
        out = {"df": lib.empty(c.f.shape), "dr": lib.empty(c.r.shape)}
        dev.backward(out, dh=None)
        got.append([out[k].numpy() for k in ("df", "dr")])
    assert all(np.array_equal(a, b) for g in got for a, b in zip(g, got[0]))
    base.check(lib, c, dh=False)


DIMS = [(3, 5, 96), (2, 33, 256), (2, 30, 512), (3, 4, 768), (2, 6, 1024), (2, 9, 1400), (4, 3, 2048), (2, 41, 2304), (2, 3, 4096), (2, 3, 4500), (2, 300, 6148),
        (3, 5, 97), (40, 1, 130), (2, 9, 701), (1, 1300, 700), (2, 3, 2303), (2, 3, 5001)]


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("wanted", [["dgate"], ["df", "dr", "dgate", "dg1", "dg2"]])
def test_dgate_with_a_shift_that_is_not_trained(lib, monkeypatch, dims, wanted):
    """RMS norms, b1 given, neither db1 nor db2 wanted: dgate is the sum of u (n1 g1 + b1) all the same."""
    monkeypatch.setattr(base, "wanted", lambda c: wanted)
    base.check(lib, base.Case(33, *dims, 0, beta=True))


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("wanted", [["df", "dr"], ["dgate"], ["df", "dr", "dgate", "dg1", "dg2"]])
@pytest.mark.parametrize("beta", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
def test_rms_norms_without_gradients_of_shifts(lib, monkeypatch, dims, wanted, beta, aligned):
    """What a net of RMS norms without trained shifts asks for: three sums a row instead of eight."""
    monkeypatch.setattr(base, "wanted", lambda c: wanted)
    base.check(lib if aligned else Pieces(lib, 0), base.Case(34, *dims, 0, beta=beta))


@pytest.mark.parametrize("dims", [(3, 5, 96), (2, 30, 512), (2, 9, 1400), (2, 3, 4500)])
@pytest.mark.parametrize("wanted", [["dr"], ["dr", "dg2"]])
def test_add_and_rms_norm(lib, monkeypatch, dims, wanted):
    """r + f and its RMS norm, no gate, no norm of f; and the first norm of a net."""
    monkeypatch.setattr(base, "wanted", lambda c: wanted + ["df"] * (c.f is not None))
    for block in (True, False):
        base.check(lib, base.Case(35, *dims, 0, post=0, gate=False, beta=False, block=block, scale=1.0), dr_out=block)
        base.check(Pieces(lib, 0), base.Case(36, *dims, 0, post=0, gate=False, beta=False, block=block, scale=1.0), inc_d=1)


@pytest.mark.parametrize("dims", DIMS)
@pytest.mark.parametrize("kind", [0, 1])
def test_tensors_off_the_grid(lib, dims, kind):
    """Every tensor 4 bytes behind a 16-byte border, columns in fours or not, all gradients."""
    base.check(Pieces(lib, 0), base.Case(37, *dims, kind))
