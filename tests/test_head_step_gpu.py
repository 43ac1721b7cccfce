"""The 8-bit products, the residual norms and the distillation loss as they are used together: a training step of a student's last block and
head, and the same calls captured into a graph."""
import ctypes
import glob
import os

import numpy as np
import pytest

from tests.test_distill_gpu import inputs, reference
from tests.test_fp8_gpu import E4M3, E5M2, Eight
from tests.test_norm_residual_gpu import Case, Device

pytestmark = pytest.mark.gpu
F, D = np.float32, np.float64


class Head:
    """norm(f) gate + r -> norm -> dense in 8 bits -> distillation, and back."""

    def __init__(self, lib, groups=3, rows=50, cols=260, classes=1500, k=9, seed=0):
        self.lib, self.dims = lib, (groups, rows, cols)
        rng = np.random.default_rng(seed)
        n = self.n = groups * rows
        self.case = Case(seed, groups, rows, cols, 1)
        self.classes, self.k, self.T, self.alpha = classes, k, 2.0, 0.25
        self.norm = Device(lib, self.case)
        self.w = (rng.standard_normal((classes, cols)) * 0.1).astype(F)
        _, _, self.ids, self.teacher = inputs(rng, n, classes, k, classes)
        self.labels = rng.integers(0, classes, n).astype(np.int32)
        self.weights = (rng.integers(0, 4, n) > 0).astype(F) / F(n)
        up = lib.to_device
        self.d = dict(w=up(self.w), ids=up(self.ids, dtype=np.int32), teacher=up(self.teacher), labels=up(self.labels, dtype=np.int32), weights=up(self.weights))
        new = lib.empty
        self.logits, self.delta, self.loss = new((n, classes)), new((n, classes)), new((n,))
        self.dw, self.dh, self.moment = new((classes, cols)), new((n, cols)), lib.zeros((classes, cols))
        self.hq, self.ht = Eight(lib, n, cols, E4M3, 1), Eight(lib, cols, n, E4M3, 1)
        self.wq, self.wt = Eight(lib, classes, cols, E4M3, 128), Eight(lib, cols, classes, E4M3, 128)
        self.gq, self.gt = Eight(lib, n, classes, E5M2, 1), Eight(lib, classes, n, E5M2, 1)
        self.out = {k: lib.empty(v) for k, v in dict(df=(n, cols), dr=(n, cols), dgate=(groups, cols), dg1=(cols,), db1=(cols,), dg2=(cols,), db2=(cols,)).items()}

    def quantize(self, a, q, t):
        self.lib.call("fp8_quantize", 0, a, q.rows, q.cols, q.fmt, q.block, 1, q.q, q.ld, q.scale, t.q, t.ld, t.scale)

    def product(self, a, b, c):
        self.lib.call("fp8_mult2d", 0, *a.args(), *b.args(), c, 0, a.rows, b.rows, a.cols)

    def forward(self):
        self.norm.forward()
        self.quantize(self.norm.h, self.hq, self.ht)
        self.quantize(self.d["w"], self.wq, self.wt)
        self.product(self.hq, self.wq, self.logits)
        d = self.d
        self.lib.call("distill", 0, self.logits, d["ids"], d["teacher"], None, d["labels"], d["weights"], self.n, self.classes, self.classes, self.k, self.T, self.alpha, self.loss, self.delta)
        self.quantize(self.delta, self.gq, self.gt)
        self.product(self.gq, self.wt, self.dh)
        self.product(self.gt, self.ht, self.dw)

    def step(self):
        self.forward()
        self.norm.backward(self.out, dh=self.dh)
        self.lib.call("sgd_momentum", 0, self.d["w"], self.dw, self.moment, 1e-3, 0.9, self.w.size)


def near(got, want, size, rel):
    return np.linalg.norm(got - want) <= rel * np.linalg.norm(size)


def test_a_training_step(lib):
    """Every link against 64-bit arithmetic on what the link before left: 2^-20 of the magnitudes is sixteen roundings of fp32."""
    H = Head(lib)
    H.step()
    lib.sync()
    c = H.case.forward()
    h = H.norm.h.numpy()
    assert near(h, c.h, c.h, 2.0 ** -20)
    # 8 bits: within half a step of the value, 2^-4 in e4m3 (2^-3 in e5m2), but for values far below their block's largest
    for q, src, half in ((H.hq, h, 2.0 ** -4), (H.ht, h.T, 2.0 ** -4), (H.gq, H.delta.numpy(), 2.0 ** -3), (H.gt, H.delta.numpy().T, 2.0 ** -3)):
        assert np.all(np.abs(q.real() - src) <= half * np.abs(src) + 2.0 ** -9 * np.repeat(np.repeat(q.scale.numpy().T, q.block, 0)[:q.rows], 128, 1)[:, :q.cols])
    hq, wq, gq = H.hq.real(), H.wq.real(), H.gq.real()
    assert np.array_equal(H.wt.real(), wq.T)                   # one scale for a tile: the transpose stands for the same numbers
    logits = H.logits.numpy()
    assert near(logits, hq @ wq.T, np.abs(hq) @ np.abs(wq).T, 2.0 ** -20)
    loss, delta, l_size, d_size = reference(logits, H.ids, H.teacher, None, H.labels, H.weights, H.T, H.alpha)
    assert near(H.loss.numpy(), loss, l_size, 2.0 ** -18) and near(H.delta.numpy(), delta, d_size, 2.0 ** -18)
    dh = H.dh.numpy()
    assert near(dh, gq @ wq, np.abs(gq) @ np.abs(wq), 2.0 ** -20)
    gt, ht = H.gt.real(), H.ht.real()
    assert near(H.dw.numpy(), gt @ ht.T, np.abs(gt) @ np.abs(ht).T, 2.0 ** -20)
    c.dh = dh
    want = c.backward()
    for k, v in H.out.items():
        assert near(v.numpy().reshape(want[k].shape), want[k], want[k], 2.0 ** -17), k
    assert np.allclose(H.d["w"].numpy(), H.w - F(1e-3) * H.dw.numpy(), rtol=1e-6, atol=1e-9)


def test_two_heads_in_turn(lib):
    """Steps of two nets one after the other, without waiting in between: the bits of each alone."""
    def bits(H):
        return [a.numpy() for a in (H.logits, H.loss, H.delta, H.dw, H.out["df"], H.out["dg2"], H.out["dgate"])]
    alone = []
    for seed in (1, 2):
        H = Head(lib, seed=seed, classes=900 + 700 * seed)
        H.step()
        alone.append(bits(H))
    a, b = Head(lib, seed=1, classes=1600), Head(lib, seed=2, classes=2300)
    a.step()
    b.step()
    for x, y in zip(alone[0] + alone[1], bits(a) + bits(b)):
        assert np.array_equal(x, y)


def _cudart():
    cands = sorted(glob.glob(os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "lib64", "libcudart.so*")))
    rt = ctypes.CDLL(cands[-1])
    rt.cudaStreamBeginCapture.argtypes = [ctypes.c_void_p, ctypes.c_int]
    rt.cudaStreamEndCapture.argtypes = [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]
    rt.cudaGraphInstantiate.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p, ctypes.c_ulonglong]
    rt.cudaGraphLaunch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    rt.cudaGraphExecDestroy.argtypes = rt.cudaGraphDestroy.argtypes = [ctypes.c_void_p]
    return rt


def test_captured_and_replayed(lib):
    """All but the backward norms (which say so) can be captured: nothing of theirs lives in the library's memory."""
    from eddl_b200 import capi
    H = Head(lib, seed=3)
    H.forward()
    H.norm.backward(H.out, dh=H.dh)
    lib.sync()
    keep = [a.numpy() for a in (H.logits, H.loss, H.delta, H.dw, H.dh)]
    rt = _cudart()
    stream, graph, ex = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    lib.call("stream", 0, ctypes.byref(stream))
    assert rt.cudaStreamBeginCapture(stream, 1) == 0
    try:
        H.forward()
        with pytest.raises(capi.Error, match="captured"):
            H.norm.backward(H.out, dh=H.dh)
        with pytest.raises(capi.Error, match="captured"):
            H.norm.backward({"dgate": H.out["dgate"]}, dh=H.dh)
        # without sums over rows nothing is kept: capturable
        H.norm.backward({k: H.out[k] for k in ("df", "dr")}, dh=H.dh)
    finally:
        assert rt.cudaStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert rt.cudaGraphInstantiate(ctypes.byref(ex), graph, 0) == 0
    try:
        df = H.out["df"].numpy()
        for a in (H.logits, H.loss, H.delta, H.dw, H.dh, H.out["df"]):
            lib.call("fill", 0, a, a.size, float("nan"))
        lib.sync()
        for _ in range(2):
            assert rt.cudaGraphLaunch(ex, stream) == 0
        lib.sync()
        for a, k in zip((H.logits, H.loss, H.delta, H.dw, H.dh), keep):
            assert np.array_equal(a.numpy(), k)
        assert np.array_equal(H.out["df"].numpy(), df)
    finally:
        rt.cudaGraphExecDestroy(ex)
        rt.cudaGraphDestroy(graph)
