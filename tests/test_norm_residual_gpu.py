"""GPU parity of the norms around a block (with gate and residual scale), forward and backward, against 64-bit arithmetic."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F, D = np.float32, np.float64
H = 2.0 ** -24                      # half a step of fp32, relative
NAMES = ("dgate", "dg1", "db1", "dg2", "db2")


def norm(x, kind, eps):
    c = x - x.mean(1, keepdims=True) if kind else x
    rstd = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
    return c * rstd, rstd


def norm_back(d, n, rstd, kind):
    b = d - n * (d * n).mean(1, keepdims=True)
    return rstd * (b - d.mean(1, keepdims=True) if kind else b)


class Case:
    def __init__(self, seed, groups, rows, cols, kind, post=1, gate=True, affine=True, beta=True, block=True, scale=0.75, shift=0.0):
        rng = np.random.default_rng(seed)
        self.dims, self.kind, self.post, self.eps = (groups, rows, cols), kind, post, 1e-3
        r = lambda *s: rng.standard_normal(s).astype(F)      # noqa: E731
        n = groups * rows
        self.f = (r(n, cols) * F(0.8) + F(shift)) if block else None
        self.r = r(n, cols) * F(1.3) + F(shift)
        self.scale = scale if block else 1.0
        self.gate = r(groups, cols) if gate and block else None
        self.g1, self.b1 = (r(cols) if affine and post and block else None), (r(cols) if beta and post and block else None)
        self.g2, self.b2 = (r(cols) if affine else None), (r(cols) if beta else None)
        self.dh, self.dr_out = r(n, cols), r(n, cols)

    def forward(self):
        d = lambda a: None if a is None else a.astype(D)      # noqa: E731
        x = d(self.r)
        if self.f is not None:
            self.n1, self.rstd1 = norm(d(self.f), self.kind, self.eps) if self.post else (d(self.f), None)
            self.z = self.n1 * (1 if self.g1 is None else d(self.g1)) + (0 if self.b1 is None else d(self.b1))
            self.G = np.ones_like(x) if self.gate is None else np.repeat(d(self.gate), self.dims[1], 0)
            x = self.scale * x + self.G * self.z
        self.r_out = x
        self.n2, self.rstd2 = norm(x, self.kind, self.eps)
        self.h = self.n2 * (1 if self.g2 is None else d(self.g2)) + (0 if self.b2 is None else d(self.b2))
        return self

    def backward(self, dh=True, dr_out=True):
        a = self.dh.astype(D) if dh else 0 * self.r_out
        u = norm_back(a * (1 if self.g2 is None else self.g2.astype(D)), self.n2, self.rstd2, self.kind) + (self.dr_out if dr_out else 0)
        self.u = u
        out = {"dr": self.scale * u, "dg2": (a * self.n2).sum(0), "db2": a.sum(0)}
        if self.f is not None:
            dz = self.G * u
            dn = dz * (1 if self.g1 is None else self.g1.astype(D))
            out.update(df=norm_back(dn, self.n1, self.rstd1, self.kind) if self.post else dn, dg1=(dz * self.n1).sum(0), db1=dz.sum(0),
                       dgate=(u * self.z).reshape(self.dims + ()).sum(1))
        return out


class Device:
    def __init__(self, lib, c):
        self.lib, self.c = lib, c
        up = lambda a: None if a is None else lib.to_device(a)      # noqa: E731
        for k in ("f", "r", "gate", "g1", "b1", "g2", "b2", "dh", "dr_out"):
            setattr(self, k, up(getattr(c, k)))
        n, cols = c.r.shape
        self.r_out, self.h, self.stats = lib.to_device(np.full((n, cols), np.nan, F)) if c.f is not None else None, lib.to_device(np.full((n, cols), np.nan, F)), lib.empty((n, 4))

    def forward(self, **more):
        c = self.c
        a = dict(f=self.f, r=self.r, gate=self.gate, g1=self.g1, b1=self.b1, g2=self.g2, b2=self.b2, r_out=self.r_out, h=self.h, stats=self.stats)
        a.update(more)
        self.lib.call("norm_residual_fwd", 0, c.kind, c.post if c.f is not None else 0, *c.dims, a["f"], a["r"], a["gate"], a["g1"], a["b1"], c.scale, a["g2"], a["b2"], c.eps, a["r_out"], a["h"], a["stats"])
        return self

    def backward(self, out, inc_d=0, inc_g=0, **more):
        c = self.c
        a = dict(dh=self.dh, dr_out=self.dr_out, r_out=self.r_out if self.r_out is not None else self.r)
        a.update(more)
        self.lib.call("norm_residual_bwd", 0, c.kind, c.post if c.f is not None else 0, *c.dims, a["dh"], a["dr_out"], self.f, a["r_out"], self.gate, self.g1, self.b1, c.scale, self.g2 if a["dh"] else None,
                      self.stats, out.get("df"), out.get("dr"), inc_d, *(out.get(k) for k in NAMES), inc_g)


def steps(c):
    """Roundings between an input and a value of a row, as a factor on the magnitudes: a row's sums are held by up to 1024 threads of 16 values
    (16 + 10 adds in a line), every value then passes some ten operations, and centring magnifies by mean / deviation."""
    def spread(x):
        return (1 + np.abs(x.mean(1)) / x.std(1).clip(1e-30)).max() if c.kind and x.shape[1] > 1 else 1.0
    return 64 * H * max(spread(x.astype(D)) for x in (c.r_out, c.f) if x is not None)


def wanted(c):
    return ["dr", "dg2", "db2"] + (["df"] if c.f is not None else []) + (["dgate"] if c.gate is not None else []) + (["dg1", "db1"] if c.f is not None and c.post else [])


def check(lib, c, dh=True, dr_out=True, inc_d=0, inc_g=0):
    c.forward()
    dev = Device(lib, c).forward()
    e = steps(c)
    G = np.abs(c.G) if c.f is not None else 0
    if c.f is not None:
        z = np.abs(c.n1 * (1 if c.g1 is None else c.g1)) + (0 if c.b1 is None else np.abs(c.b1))
        r_size = np.abs(c.scale * c.r) + G * (z + (1 if c.post else 0))
        assert np.all(np.abs(dev.r_out.numpy() - c.r_out) <= e * r_size)
    else:
        r_size = np.abs(c.r.astype(D))
    # an error of r_out reaches h through its own value, the row's mean and deviation
    n_off = e * (r_size * c.rstd2 + (1 + np.abs(c.n2)) * (1 + (r_size * c.rstd2).max(1, keepdims=True)))
    assert np.all(np.abs(dev.h.numpy() - c.h) <= n_off * (1 if c.g2 is None else np.abs(c.g2)) + e * np.abs(c.h) + 1e-30)
    want = c.backward(dh, dr_out)
    old = {k: np.random.default_rng(3).standard_normal(want[k].shape).astype(F) for k in wanted(c)}
    if not dh:
        for k in ("dg2", "db2"):
            old.pop(k)
    out = {k: lib.to_device(v if (inc_d if k in ("df", "dr") else inc_g) else np.full_like(v, np.nan)) for k, v in old.items()}
    dev.backward(out, inc_d, inc_g, **({} if dh else dict(dh=None)), **({} if dr_out else dict(dr_out=None)))
    n = c.r.shape[0]
    g2 = 1 if c.g2 is None else np.abs(c.g2)
    a = np.abs(c.dh) * g2 if dh else 0 * np.abs(c.dh)
    # magnitudes of the terms of u: its own, and the row's means of dn2 and dn2 n2 (an error of n2 moves both)
    grow = 1 + (n_off / e).max(1, keepdims=True)
    u_size = (np.abs(c.dr_out) if dr_out else 0) + c.rstd2 * (a + (1 + np.abs(c.n2)) * (a * (1 + np.abs(c.n2))).mean(1, keepdims=True)) * grow
    sizes = {"dr": abs(c.scale) * u_size, "dg2": ((np.abs(c.dh)) * (np.abs(c.n2) + grow)).sum(0), "db2": np.abs(c.dh).sum(0)}
    if c.f is not None:
        dz = G * u_size
        dn = dz * (1 if c.g1 is None else np.abs(c.g1))
        n1 = np.abs(c.n1) + 1
        # <dn1> and <dn1 n1> come from sums over dr_out, dn2 and n2 apart: their magnitudes add
        sizes.update(df=c.rstd1 * (dn + n1 * (dn * n1).mean(1, keepdims=True) * 2) if c.post else dn, dg1=(dz * n1).sum(0), db1=dz.sum(0),
                     dgate=(u_size * (z + 1)).reshape(c.dims).sum(1))
    for k, v in out.items():
        inc = inc_d if k in ("df", "dr") else inc_g
        over = n if k not in ("df", "dr") else 0
        got = v.numpy().reshape(want[k].shape)
        w = want[k] + (old[k] if inc else 0)
        # sums over rows: at most one addition for each row in a line
        bound = (e + over * H) * sizes[k] + H * np.abs(w) + 1e-30
        assert np.all(np.abs(got - w) <= bound), (k, np.max(np.abs(got - w) / bound))
        if n * c.dims[2] >= 2000:           # and roundings do not all point the same way
            assert np.linalg.norm(got - w) <= 0.25 * np.linalg.norm(bound), k
    return dev


SHAPES = [(1, 1, 1), (1, 3, 5), (2, 7, 64), (3, 5, 127), (1, 40, 128), (5, 9, 130), (2, 33, 256), (7, 1, 257), (2, 30, 512), (3, 4, 771), (1, 9, 1024), (2, 6, 1028), (4, 3, 2048),
          (1, 5, 2049), (2, 3, 4096), (1, 3, 4100), (2, 2, 5001), (1, 2, 8192), (1, 3, 12000), (1, 2, 16384), (1, 3, 16383), (300, 2, 32), (2, 700, 96), (1, 3000, 260),
          (1, 13000, 100), (1, 1300, 700), (1, 1301, 701), (2, 50, 1400), (1, 60, 1535), (2, 41, 2304), (1, 40, 2303), (1, 500, 4352), (2, 300, 6148), (1, 350, 8192), (1, 200, 12004)]


@pytest.mark.parametrize("dims", SHAPES)
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("beta", [False, True])
def test_forward_and_backward(lib, dims, kind, beta):
    check(lib, Case(sum(dims), *dims, kind, beta=beta))


@pytest.mark.parametrize("dims", [(3, 5, 96), (2, 9, 1000), (2, 3, 4500)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("post,gate,affine,block", [(0, True, True, True), (1, False, True, True), (1, True, False, True), (0, False, False, True), (0, False, True, False)])
def test_parts_left_out(lib, dims, kind, post, gate, affine, block):
    check(lib, Case(11, *dims, kind, post=post, gate=gate, affine=affine, beta=affine, block=block))


@pytest.mark.parametrize("dims", [(3, 5, 96), (2, 9, 1001), (2, 3, 4500), (40, 1, 130), (1, 50, 300)])
@pytest.mark.parametrize("inc_d,inc_g", [(1, 0), (0, 1), (1, 1)])
def test_added_to_what_is_there(lib, dims, inc_d, inc_g):
    check(lib, Case(12, *dims, 1), inc_d=inc_d, inc_g=inc_g)


@pytest.mark.parametrize("dims", [(3, 5, 96), (2, 3, 4500)])
@pytest.mark.parametrize("kind", [0, 1])
def test_one_gradient_missing(lib, dims, kind):
    check(lib, Case(13, *dims, kind), dh=False)
    check(lib, Case(14, *dims, kind), dr_out=False)


def test_rows_far_from_zero(lib):
    check(lib, Case(15, 2, 20, 768, 1, shift=30.0))


def test_inputs_that_are_no_multiple_of_16_bytes_apart(lib):
    c = Case(16, 2, 5, 256, 1).forward()
    dev = Device(lib, c)
    room = lib.empty((c.r.size + 8,))
    lib.call("memcpy_h2d", 0, room.addr + 4, c.r.ctypes.data_as(ctypes.c_void_p), c.r.nbytes)
    dev.forward()
    h, r = dev.h.numpy(), dev.r_out.numpy()
    dev.forward(r=room.addr + 4)
    assert np.allclose(dev.h.numpy(), h, rtol=0, atol=64 * H * 8) and np.allclose(dev.r_out.numpy(), r, rtol=0, atol=4 * H * 8)


def test_in_place(lib):
    """r_out over r, h over f; df over dh, dr over dr_out: the bits of the separate tensors."""
    for cols in (96, 1000, 4500):
        c = Case(17, 2, 6, cols, 1).forward()
        a, b = Device(lib, c).forward(), Device(lib, c)
        b.forward(r_out=b.r)
        assert np.array_equal(a.r_out.numpy(), b.r.numpy()) and np.array_equal(a.h.numpy(), b.h.numpy())
        apart = {k: lib.empty(getattr(c, "r").shape) for k in ("df", "dr")}
        a.backward(apart)
        b.backward(dict(df=b.dh, dr=b.dr_out), r_out=b.r)
        assert np.array_equal(apart["df"].numpy(), b.dh.numpy()) and np.array_equal(apart["dr"].numpy(), b.dr_out.numpy())
        d = Device(lib, c)
        d.forward(h=d.f)
        assert np.array_equal(a.h.numpy(), d.f.numpy())


def test_forward_alone_is_the_same_without_stats(lib):
    c = Case(18, 2, 6, 640, 0).forward()
    a, b = Device(lib, c).forward(), Device(lib, c).forward(stats=None)
    assert np.array_equal(a.h.numpy(), b.h.numpy())
    b.forward(h=None, g2=None, b2=None, stats=None)
    assert np.array_equal(a.r_out.numpy(), b.r_out.numpy())


def test_differences(lib):
    """Every gradient against central differences of the loss <dh, h> + <dr_out, r_out>, evaluated in 64 bits."""
    c = Case(19, 2, 3, 40, 1).forward()
    dev = Device(lib, c).forward()
    out = {k: lib.empty(v) for k, v in dict(df=c.f.shape, dr=c.r.shape, dgate=c.gate.shape, dg1=(40,), db1=(40,), dg2=(40,), db2=(40,)).items()}
    dev.backward(out)
    rng = np.random.default_rng(0)
    for name, g in out.items():
        x0 = getattr(c, name[1:]).astype(D)
        way = rng.standard_normal(x0.shape)
        loss = []
        for s in (1e-4, -1e-4):
            setattr(c, name[1:], x0 + s * way)
            c.forward()
            loss.append((c.dh * c.h).sum() + (c.dr_out * c.r_out).sum())
        setattr(c, name[1:], x0.astype(F))
        slope = (loss[0] - loss[1]) / 2e-4
        # third-order terms of a step of 1e-4, and fp32 gradients over a few hundred terms
        assert abs((g.numpy() * way).sum() - slope) <= 1e-5 * np.abs(g.numpy() * way).sum() + 1e-4, name


def test_infinities_and_nan_stay_in_their_rows(lib):
    c = Case(20, 1, 9, 300, 1)
    c.f[3, 7], c.r[5, 9] = np.inf, np.nan
    with np.errstate(all="ignore"):
        c.forward()
    dev = Device(lib, c).forward()
    bad = ~np.isfinite(dev.h.numpy())
    assert bad[3].all() and bad[5].all() and not np.delete(bad, [3, 5], 0).any()


def test_same_call_same_bits(lib):
    for dims in ((2, 700, 96), (1, 900, 640), (1, 40, 6000)):
        c = Case(21, *dims, 1).forward()
        dev = Device(lib, c).forward()
        got = []
        for _ in range(2):
            out = {k: lib.empty(v) for k, v in dict(df=c.f.shape, dgate=c.gate.shape, dg1=(dims[2],), db1=(dims[2],), dg2=(dims[2],), db2=(dims[2],)).items()}
            dev.backward(out)
            got.append({k: v.numpy() for k, v in out.items()})
        for k in got[0]:
            assert np.array_equal(got[0][k], got[1][k]), k


def test_no_rows(lib):
    v = lib.to_device(np.full(64, 2.0, F))
    w = lib.to_device(np.full(64, 2.0, F))
    e = lib.empty((16,))
    for inc, want in ((1, 2.0), (0, 0.0)):
        lib.call("norm_residual_bwd", 0, 1, 1, 3, 0, 64, e, e, e, e, None, None, None, 1.0, None, e, None, None, 0, None, None, None, v, w, inc)
        assert np.all(v.numpy() == want) and np.all(w.numpy() == want)
    lib.call("norm_residual_fwd", 0, 1, 1, 0, 5, 64, e, e, None, None, None, 1.0, None, None, 1e-5, lib.empty((16,)), lib.empty((16,)), None)


def test_zeros_owed_to_the_deltas(lib):
    c = Case(22, 1, 300, 512, 1).forward()
    dev = Device(lib, c).forward()
    apart = {k: lib.empty(c.r.shape) for k in ("df", "dr")}
    dev.backward(apart)
    lib.call("set_option", b"lazy_zero", 1)
    try:
        owed = {k: lib.to_device(np.full(c.r.shape, 7.0, F)) for k in ("df", "dr")}
        for v in owed.values():
            lib.call("fill", 0, v, v.size, 0.0)
        dev.backward(owed, inc_d=1)
        for k in owed:
            assert np.array_equal(owed[k].numpy(), apart[k].numpy())
    finally:
        lib.call("set_option", b"lazy_zero", 0)
