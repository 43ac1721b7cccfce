"""GPU parity of the distillation loss and its gradient against 64-bit arithmetic."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F, D = np.float32, np.float64
H = 2.0 ** -24


def reference(x, ids, teacher, lse, labels, weights, T, alpha):
    """Row by row, as the definition says.  Returns loss, delta and the magnitudes that their roundings are relative to."""
    T, alpha = D(F(T)), D(F(alpha))                          # what an fp32 argument holds: the rest of the mass, 1 - sum p, magnifies 0.7 - float(0.7)
    rows, cols = x.shape
    loss, delta = np.zeros(rows), np.zeros((rows, cols))
    l_size, d_size = np.zeros(rows), np.zeros((rows, cols))
    for r in range(rows):
        w = 1.0 if weights is None else D(weights[r])
        s = x[r].astype(D)
        if w == 0 or not np.any(s > -np.inf):
            continue
        def softmax(v):
            m = v.max()
            e = np.exp(v - m)
            return e / e.sum(), v - m - np.log(e.sum())
        seen, keep = set(), []
        for j, i in enumerate(ids[r]):
            if 0 <= i < cols and i not in seen:
                seen.add(i)
                keep.append(j)
        at, t = ids[r][keep], teacher[r][keep].astype(D) / T
        if alpha != 1 and (lse is not None or np.any(t > -np.inf)):
            q, logq = softmax(s / T)
            logp = t - D(lse[r]) if lse is not None else softmax(t)[1]
            p = np.exp(logp)
            on = p > 0
            kl = np.sum(p[on] * (logp[on] - logq[at][on]))
            size = np.sum(p[on] * (1 + np.abs(logp[on]) + np.abs(logq[at][on])))
            g, gs = q.copy(), q.copy()
            if lse is not None:
                rest = max(0.0, 1 - p.sum())
                others = np.ones(cols, bool)
                others[at] = False
                q_rest = q[others].sum()
                if rest > 0:
                    with np.errstate(divide="ignore"):
                        kl += rest * np.log(rest / q_rest)
                    size += rest * (1 + abs(np.log(rest)) + (abs(np.log(q_rest)) if q_rest > 0 else 0))
                g = q * (p.sum() + rest)
                ratio = rest / q_rest if q_rest > 0 else 0
                g[others] = q[others] * ((p.sum() + rest) - ratio) if q_rest > 0 else 0
                gs[others] = q[others] * (2 + ratio)
            g[at] -= p
            gs[at] += p
            loss[r] += w * (1 - D(alpha)) * T * T * kl
            l_size[r] += abs(w) * (1 - alpha) * T * T * size
            delta[r] += w * (1 - D(alpha)) * T * g
            d_size[r] += abs(w) * (1 - alpha) * T * gs
        if alpha and 0 <= labels[r] < cols:
            q, logq = softmax(s)
            loss[r] -= w * D(alpha) * logq[labels[r]]
            l_size[r] += abs(w) * alpha * (1 + abs(logq[labels[r]]))
            q[labels[r]] -= 1
            delta[r] += w * D(alpha) * q
            q[labels[r]] += 2
            d_size[r] += abs(w) * alpha * q
    return loss, delta, l_size, d_size


def inputs(rng, rows, cols, k, ld):
    wide = (rng.standard_normal((rows, ld)) * 2).astype(F)
    x = wide[:, :cols]
    teacher_all = (x * F(0.6) + rng.standard_normal((rows, cols)) * 2).astype(F)
    ids = np.argsort(-teacher_all, 1, kind="stable")[:, :k].astype(np.int32)
    return wide, teacher_all, np.ascontiguousarray(ids), np.take_along_axis(teacher_all, ids.astype(np.int64), 1)


def lse_of(teacher_all, T):
    t = teacher_all.astype(D) / D(F(T))
    m = t.max(1, keepdims=True)
    return (m[:, 0] + np.log(np.exp(t - m).sum(1))).astype(F)


def run(lib, wide, cols, ids, teacher, lse, labels, weights, T, alpha, with_delta=True, in_place=False):
    rows, ld = wide.shape
    up = lambda a, t=F: None if a is None else lib.to_device(a, dtype=t)      # noqa: E731
    x = up(wide)
    loss, delta = lib.to_device(np.full(rows, np.nan, F)), x if in_place else lib.to_device(np.full((rows, ld), -77.0, F)) if with_delta else None
    lib.call("distill", 0, x, up(ids, np.int32), up(teacher), up(lse), up(labels, np.int32), up(weights), rows, cols, ld, ids.shape[1], T, alpha, loss, delta)
    return loss.numpy(), delta.numpy() if delta is not None else None


def check(lib, wide, cols, ids, teacher, lse, labels, weights, T, alpha):
    loss, delta = run(lib, wide, cols, ids, teacher, lse, labels, weights, T, alpha)
    want, dwant, l_size, d_size = reference(wide[:, :cols], ids, teacher, lse, labels, weights, T, alpha)
    # Exponentials: 2 steps, an argument rounded twice, relative to it -- |d| e^-|d| is below 1/e, and over a row the mean |d| is at most log cols + 1.
    # Sums: a thread adds at most cols / 128 + 98 values in fp32 (128 threads or more a row from 257 columns on, 32 below), the rest in 64 bits.
    off = (8 + 4 * (np.log(cols) + 1) + (cols / 32 if cols <= 256 else min(98, cols / 128)) + 4) * H
    spread = 1 + np.abs(wide[:, :cols].astype(D) - wide[:, :cols].max(1, keepdims=True)) / min(T, 1.0)
    assert np.all(np.abs(loss - want) <= off * l_size + H * np.abs(want) + 1e-30), np.max(np.abs(loss - want) / (off * l_size + 1e-30))
    assert np.all(np.abs(delta[:, :cols] - dwant) <= (off + 3 * H * np.where(np.isfinite(spread), spread, 1)) * d_size + 1e-37)
    assert np.all(delta[:, cols:] == -77.0)
    alone, _ = run(lib, wide, cols, ids, teacher, lse, labels, weights, T, alpha, with_delta=False)
    assert np.array_equal(alone, loss)
    return loss, delta


SHAPES = [(1, 1, 0, 1), (3, 2, 1, 1), (5, 10, 0, 3), (40, 10, 2, 4), (9, 255, 0, 12), (8, 256, 4, 256), (7, 257, 0, 5), (64, 1000, 0, 10), (3, 1001, 3, 17), (2, 2048, 0, 130), (3, 2049, 0, 64),
          (2, 16384, 0, 600), (2, 16387, 1, 33), (3, 32768, 0, 64), (2, 50001, 0, 1024), (1, 65537, 3, 100), (3, 131071, 1, 128), (1, 344064, 0, 16), (3000, 40, 0, 5), (700, 300, 0, 8), (1300, 1301, 1, 9), (1250, 3000, 2, 40), (3000, 4501, 0, 7), (700, 20000, 2, 6)]


@pytest.mark.parametrize("rows,cols,pad,k", SHAPES)
@pytest.mark.parametrize("T,alpha", [(1.0, 0.0), (2.0, 0.3), (0.7, 0.5), (3.0, 1.0), (1.0, 0.5)])
@pytest.mark.parametrize("tail", [False, True])
def test_loss_and_gradient(lib, rows, cols, pad, k, T, alpha, tail):
    rng = np.random.default_rng(rows + cols + k)
    wide, every, ids, teacher = inputs(rng, rows, cols, min(k, cols), cols + pad)
    labels = rng.integers(0, cols, rows).astype(np.int32) if alpha else None
    if alpha and rows > 2:
        labels[1], labels[2] = -1, cols                      # no label
    weights = rng.random(rows).astype(F) if rows % 2 else None
    if weights is not None and rows > 3:
        weights[3] = 0
    if tail and k >= cols:
        pytest.skip("the entries are all classes: no rest")
    check(lib, wide, cols, ids, teacher, lse_of(every, T) if tail else None, labels, weights, T, alpha)


@pytest.mark.parametrize("rows,cols,k", [(1200, 250, 1), (40, 3458, 3), (30, 8000, 2), (20, 16000, 3), (9, 70000, 4)])
def test_entries_of_little_mass(lib, rows, cols, k):
    """A high temperature leaves the entries P of the teacher's mass and Q of the student's, both small: the loss and the gradient outside the entries are
    differences of the order of P and Q, and as exact as those."""
    T = 8.0
    rng = np.random.default_rng(cols)
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols)
    lse = lse_of(every, T)
    loss, delta = run(lib, wide, cols, ids, teacher, lse, None, None, T, 0.0)
    want, dwant, _, _ = reference(wide, ids, teacher, lse, None, None, T, 0.0)
    at = ids.astype(np.int64)
    x = wide.astype(D) / T
    log_q = x - x.max(1, keepdims=True)
    log_q -= np.log(np.exp(log_q).sum(1, keepdims=True))
    q, log_p = np.exp(log_q), teacher.astype(D) / T - lse[:, None].astype(D)
    P, Q = np.exp(log_p).sum(1), np.take_along_axis(q, at, 1).sum(1)
    assert P.max() < 0.1 and Q.max() < 0.1
    # `off` as in check(): of the sums.  Every term of the entries is p times logarithms of the size L, the two terms of the rest are ln(1 - P) and
    # ln(1 - Q), each as exact as P and Q are.
    off = (8 + 4 * (np.log(cols) + 1) + (cols / 32 if cols <= 256 else min(98, cols / 128)) + 4) * H
    L = 1 + np.abs(log_p).max(1) + np.abs(np.take_along_axis(log_q, at, 1)).max(1)
    assert np.all(np.abs(loss - want) <= T * T * off * (P * L + 2 * Q) + H * np.abs(want)), np.max(np.abs(loss - want) / (T * T * off * (P * L + 2 * Q)))
    outside = np.ones_like(q, bool)
    np.put_along_axis(outside, at, False, 1)
    spread = 1 + np.abs(x - x.max(1, keepdims=True))
    bound = T * q * (P + 2 * Q)[:, None] * (2 * off + 3 * H * spread)
    assert np.all((np.abs(delta - dwant) <= bound)[outside]), np.max((np.abs(delta - dwant) / bound)[outside])


@pytest.mark.parametrize("cols,k", [(20, 6), (600, 9), (5000, 40), (40000, 70)])
@pytest.mark.parametrize("tail", [False, True])
def test_padding_and_repeated_entries(lib, cols, k, tail):
    rng = np.random.default_rng(cols)
    rows = 12
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols)
    ids[0, :] = ids[0, 2]                                    # one class k times
    ids[1, 1::2] = ids[1, 0]
    ids[2, ::2] = -1
    ids[3, 1:] = cols + np.arange(k - 1)
    ids[4, :] = -5                                           # no entry at all
    ids[5, 3], ids[5, 4] = 2 ** 31 - 1, -2 ** 31
    labels = rng.integers(0, cols, rows).astype(np.int32)
    labels[6] = ids[6, 0]
    check(lib, wide, cols, ids, teacher, lse_of(every, 2.0) if tail else None, labels, None, 2.0, 0.25)


@pytest.mark.parametrize("cols", [24, 900, 9000, 70000])
@pytest.mark.parametrize("tail", [False, True])
def test_masks(lib, cols, tail):
    """Masked classes, by -infinity and by the lowest number; rows that a mask leaves empty; NaN behind a weight of zero."""
    rng = np.random.default_rng(cols)
    k, rows = 7, 10
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols + 2)
    lse = lse_of(every, 0.7) if tail else None
    open_ = np.ones((rows, cols), bool)
    np.put_along_axis(open_, ids.astype(np.int64), False, 1)
    wide[1, :cols][open_[1]] = -np.inf                       # only the entries are left: nothing outside
    wide[2, :cols] = -np.inf                                 # nothing is left
    wide[3, :cols][open_[3]] = np.finfo(F).min
    wide[4, :cols] = np.finfo(F).min                         # the lowest number everywhere: uniform
    weights = np.ones(rows, F)
    weights[5], weights[6] = 0, 0
    wide[5, :], wide[6, 0], teacher[6, 1] = np.nan, np.inf, np.nan
    teacher[7, 1:3] = -np.inf
    if not tail:
        teacher[8, :] = -np.inf                              # a teacher without a class
    wide[:, cols:] = np.nan                                  # beyond the columns
    if tail:
        # with nothing outside the entries the loss is infinite, not a number nowhere
        loss, delta = run(lib, wide, cols, ids, teacher, lse, None, weights, 0.7, 0.0)
        assert np.isposinf(loss[1]) and np.all(np.isfinite(delta[1, :cols]))
        weights[1] = weights[3] = 0                          # row 3: nothing outside in fp32 either
    check_rows = check(lib, wide, cols, ids, teacher, lse, None, weights, 0.7, 0.0)
    assert np.all(check_rows[0][[2, 5, 6]] == 0) and np.all(check_rows[1][[2, 5, 6], :cols] == 0)


def test_an_entry_that_the_student_masks(lib):
    rng = np.random.default_rng(1)
    for cols in (30, 3000):
        wide, every, ids, teacher = inputs(rng, 3, cols, 4, cols)
        wide[1, ids[1, 2]] = -np.inf
        loss, delta = run(lib, wide, cols, ids, teacher, None, None, None, 1.0, 0.0)
        assert np.isposinf(loss[1]) and np.all(np.isfinite(delta)) and np.all(np.isfinite(loss[[0, 2]]))


def test_not_a_number_is_not_hidden(lib):
    rng = np.random.default_rng(2)
    for cols in (30, 3000, 40000):
        for value in (np.nan, np.inf):
            wide, every, ids, teacher = inputs(rng, 4, cols, 4, cols)
            wide[1, cols // 2] = value
            teacher[2, 0] = value
            loss, delta = run(lib, wide, cols, ids, teacher, None, None, None, 1.0, 0.0)
            assert np.isnan(loss[1]) and np.isnan(loss[2]) and np.isnan(delta[1]).any() and np.isnan(delta[2]).any()
            assert np.all(np.isfinite(loss[[0, 3]])) and np.all(np.isfinite(delta[[0, 3]]))
        wide[:] = np.nan
        loss, _ = run(lib, wide, cols, ids, teacher, None, None, None, 1.0, 0.0)
        assert np.all(np.isnan(loss))


def test_in_place_and_repeated(lib):
    rng = np.random.default_rng(3)
    for cols in (33, 1000, 20000, 90000):
        wide, every, ids, teacher = inputs(rng, 5, cols, 6, cols + 1)
        labels = rng.integers(0, cols, 5).astype(np.int32)
        a = run(lib, wide, cols, ids, teacher, None, labels, None, 2.0, 0.5)
        for other in (run(lib, wide, cols, ids, teacher, None, labels, None, 2.0, 0.5), run(lib, wide, cols, ids, teacher, None, labels, None, 2.0, 0.5, in_place=True)):
            assert np.array_equal(a[0], other[0]) and np.array_equal(a[1][:, :cols], other[1][:, :cols])


def test_unaligned_logits(lib):
    rng = np.random.default_rng(4)
    rows, cols, k = 3, 512, 5
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols)
    room, out = lib.empty((rows * cols + 4,)), lib.empty((rows * cols + 4,))
    lib.call("memcpy_h2d", 0, room.addr + 4, wide.ctypes.data_as(ctypes.c_void_p), wide.nbytes)
    loss = lib.empty((rows,))
    lib.call("distill", 0, room.addr + 4, lib.to_device(ids, dtype=np.int32), lib.to_device(teacher), None, None, None, rows, cols, cols, k, 1.0, 0.0, loss, out.addr + 8)
    a = run(lib, wide, cols, ids, teacher, None, None, None, 1.0, 0.0)
    assert np.allclose(loss.numpy(), a[0], rtol=1e-5) and np.allclose(out.numpy()[2:2 + rows * cols].reshape(rows, cols), a[1], rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("tail", [False, True])
def test_differences(lib, tail):
    """The gradient against central differences of the reference's loss."""
    rng = np.random.default_rng(5)
    rows, cols, k, T, alpha = 4, 60, 5, 1.5, 0.4
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols)
    lse = lse_of(every, T) if tail else None
    labels = rng.integers(0, cols, rows).astype(np.int32)
    _, delta = run(lib, wide, cols, ids, teacher, lse, labels, None, T, alpha)
    way = rng.standard_normal(wide.shape)
    up, down = (reference(wide.astype(D) + s * way, ids, teacher, lse, labels, None, T, alpha)[0].sum() for s in (1e-4, -1e-4))
    assert abs((up - down) / 2e-4 - (delta * way).sum()) <= 1e-5 * np.abs(delta * way).sum() + 1e-6


def test_no_rows(lib):
    lib.call("distill", 0, None, None, None, None, None, None, 0, 5, 5, 1, 1.0, 0.5, None, None)
