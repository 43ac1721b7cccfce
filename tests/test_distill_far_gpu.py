"""Distillation where the student's mass outside the teacher's entries is below what fp32 holds beside the rest of it: the loss is finite and its
gradient is not zero, as long as the student has a class there at all."""
import numpy as np
import pytest

from tests.test_distill_gpu import inputs, lse_of, run

pytestmark = pytest.mark.gpu
F, D = np.float32, np.float64
H = 2.0 ** -24


def log_sum(a):
    m = a.max(1, keepdims=True)
    return (m + np.log(np.exp(a - m).sum(1, keepdims=True)))


def reference(x, at, teacher, lse, labels, T, alpha):
    """Loss and gradient with every mass as a logarithm, and how far fp32 arithmetic may be off them."""
    T, alpha, x = D(F(T)), D(F(alpha)), x.astype(D)
    log_p = teacher.astype(D) / T - lse.astype(D)[:, None]
    p = np.exp(log_p)
    rest = np.maximum(0, 1 - p.sum(1, keepdims=True))
    log_q = x / T - log_sum(x / T)
    outside = np.ones(x.shape, bool)
    np.put_along_axis(outside, at, False, 1)
    open_log = np.where(outside, log_q, -np.inf)
    log_rest = log_sum(open_log)
    picked = np.take_along_axis(log_q, at, 1)
    with np.errstate(divide="ignore", invalid="ignore"):
        kl = (p * (log_p - picked)).sum(1) + (rest * (np.where(rest > 0, np.log(rest), 0) - log_rest))[:, 0]
    size = (p * (1 + np.abs(log_p) + np.abs(picked))).sum(1) + (rest * (1 + np.abs(log_rest)))[:, 0]
    # a softmax of its own: beside a maximum of 1e38 the logarithm of the sum has no room for that of the number of classes
    share = np.exp(open_log - open_log.max(1, keepdims=True))
    share *= rest / share.sum(1, keepdims=True)
    g = np.exp(log_q) * (p.sum(1, keepdims=True) + rest) - share
    np.put_along_axis(g, at, np.take_along_axis(g, at, 1) - p, 1)
    # an exponential is off by `off` and, its argument being rounded, by four half steps for each unit of that: how far its class is below the
    # largest one it is taken against.  That of the classes outside is their own where they are more than 32 powers of two (23 units) below the row's.
    below, below_out = (x.max(1, keepdims=True) - x), np.where(outside, np.where(outside, x, -np.inf).max(1, keepdims=True) - x, 0)
    soft = lambda v, d: v * (off_of(x.shape[1]) + 4 * H * (1 + d))      # noqa: E731
    apart = np.minimum(below - below_out, 23 * T)
    bound = soft(np.exp(log_q), below / T) * 2 + soft(share, (below_out + apart) / T)
    np.put_along_axis(bound, at, np.take_along_axis(bound, at, 1) + soft(p, 0), 1)
    loss, l_size, delta, bound = (1 - alpha) * T * T * kl, (1 - alpha) * T * T * size, (1 - alpha) * T * g, (1 - alpha) * T * bound
    if alpha:
        log_1 = x - log_sum(x)
        hot = np.eye(x.shape[1])[labels]
        loss, delta = loss - alpha * (log_1 * hot).sum(1), delta + alpha * (np.exp(log_1) - hot)
        l_size, bound = l_size + alpha * (1 - (log_1 * hot).sum(1)), bound + alpha * (soft(np.exp(log_1), below) + 2 * H * hot)
    return loss, delta, off_of(x.shape[1]) * l_size + H * np.abs(loss), bound + H * np.abs(delta) + 1e-37


def off_of(cols):
    """As for ordinary rows: an exponential's two steps and the mean of its argument's roundings over a row, and the sums of a thread."""
    return (8 + 4 * (np.log(cols) + 1) + (cols / 32 if cols <= 256 else min(98, cols / 128)) + 4) * H


@pytest.mark.parametrize("rows,cols,k", [(9, 40, 3), (1300, 40, 3), (9, 1000, 7), (7, 9001, 20), (5, 20000, 64), (4, 70000, 33), (1250, 300, 5)])
@pytest.mark.parametrize("T,alpha", [(1.0, 0.0), (1.0, 0.4), (2.0, 0.3), (4.0, 0.5), (0.5, 0.5), (3.0, 0.0)])
def test_student_without_mass_outside_the_entries(lib, rows, cols, k, T, alpha):
    rng = np.random.default_rng(cols + k)
    wide, every, ids, teacher = inputs(rng, rows, cols, k, cols + 1)
    at = ids.astype(np.int64)
    x = wide[:, :cols]
    # the entries lead by 10 to 4000 temperatures: on both sides of what the smallest normal number holds (87)
    lead = (T * np.exp(rng.uniform(np.log(10), np.log(4000), (rows, 1)))).astype(F)
    lead[0], lead[1] = T * 86, T * 89
    np.put_along_axis(x, at, np.take_along_axis(x, at, 1) + lead, 1)
    labels = rng.integers(0, cols, rows).astype(np.int32)
    labels[::2] = ids[::2, 0]
    lse = lse_of(every, T)
    loss, delta = run(lib, wide, cols, ids, teacher, lse, labels if alpha else None, None, T, alpha)
    want, dwant, l_off, d_off = reference(x, at, teacher, lse, labels, T, alpha)
    assert np.all(np.isfinite(want)) and np.all(np.abs(loss - want) <= l_off), np.max(np.abs(loss - want) / l_off)
    assert np.all(np.abs(delta[:, :cols] - dwant) <= d_off), np.max(np.abs(delta[:, :cols] - dwant) / d_off)
    assert np.all(delta[:, cols:] == -77.0)


@pytest.mark.parametrize("cols", [50, 900, 30000])
def test_masks_of_finite_numbers(lib, cols):
    """All classes but the entries closed by a large finite number: the rest's loss is as large, and its gradient goes to the classes that are closed least."""
    rng = np.random.default_rng(cols)
    wide, every, ids, teacher = inputs(rng, 4, cols, 5, cols)
    at = ids.astype(np.int64)
    keep = np.take_along_axis(wide, at, 1)
    for closed in (-1e4, -1e9, np.finfo(F).min / 2):
        x = np.full_like(wide, closed)
        np.put_along_axis(x, at, keep, 1)
        lse = lse_of(every, 1.0)
        loss, delta = run(lib, x, cols, ids, teacher, lse, None, None, 1.0, 0.0)
        want, dwant, l_off, d_off = reference(x, at, teacher, lse, None, 1.0, 0.0)
        assert np.all(np.abs(loss - want) <= l_off) and np.all(np.abs(delta - dwant) <= d_off)
