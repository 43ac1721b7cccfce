"""The 8-bit, residual-norm and distillation entry points refuse wrong arguments before they touch a device (no GPU needed)."""
import ctypes

import pytest

from eddl_b200 import capi

INVAL, LIMIT = -1, -5
P = [0x10000000 * (i + 1) for i in range(24)]          # addresses far apart that nothing looks behind


def call(name, args):
    conv = [ctypes.c_void_p(a) if isinstance(a, int) and (a - a % 4 in P or a >= 1 << 50) else a for a in args]
    return capi.lib().fn[name](*conv)


def with_changes(names, base, change):
    assert set(change) <= set(names)
    return [change.get(n, b) for n, b in zip(names, base)]


QUANT = "dev a rows cols format block_rows pow2 q ldq scale qt ldqt scale_t".split()
QUANT_OK = [0, P[0], 64, 100, 0, 1, 0, P[1], 112, P[2], P[3], 64, P[4]]


@pytest.mark.parametrize("change", [
    dict(a=None), dict(rows=-1), dict(cols=-1), dict(format=2), dict(format=-1), dict(block_rows=64), dict(pow2=2), dict(q=None, qt=None), dict(scale=None), dict(scale_t=None),
    dict(ldq=100), dict(ldq=96), dict(ldqt=48), dict(q=P[1] + 8), dict(qt=P[3] + 1), dict(q=P[0]), dict(qt=P[0] + 16), dict(qt=P[1]), dict(scale=P[1]), dict(scale_t=P[2]), dict(a=P[0] + 2), dict(scale=P[2] + 1)])
def test_quantize_refuses(change):
    assert call("fp8_quantize", with_changes(QUANT, QUANT_OK, change)) == INVAL
    assert "fp8_quantize" in capi.lib().last_error()


PROD = "dev qa lda sa fa ba qb ldb sb fb bb c inc m n k".split()
PROD_OK = [0, P[0], 112, P[1], 0, 1, P[2], 112, P[3], 1, 128, P[4], 0, 30, 40, 100]


@pytest.mark.parametrize("change", [
    dict(qa=None), dict(qb=None), dict(sa=None), dict(sb=None), dict(c=None), dict(fa=2), dict(fb=-1), dict(ba=2), dict(bb=0), dict(lda=96), dict(lda=100), dict(ldb=104), dict(ldb=1 << 40),
    dict(qa=P[0] + 4), dict(qb=P[2] + 8), dict(m=-1), dict(n=-1), dict(k=-1), dict(c=P[0]), dict(c=P[2] + 64), dict(c=P[3]), dict(c=P[4] + 2), dict(sa=P[1] + 1)])
def test_product_refuses(change):
    assert call("fp8_mult2d", with_changes(PROD, PROD_OK, change)) == INVAL
    assert "fp8_mult2d" in capi.lib().last_error()


FWD = "dev kind post groups rows cols f r gate g1 b1 res_scale g2 b2 eps r_out h stats".split()
FWD_OK = [0, 1, 1, 2, 3, 100, P[0], P[1], P[2], P[3], P[4], 0.5, P[5], P[6], 1e-5, P[7], P[8], P[9]]
NO_BLOCK = dict(f=None, r_out=None, gate=None, g1=None, b1=None, post=0, res_scale=1.0)


@pytest.mark.parametrize("change", [
    dict(kind=2), dict(post=2), dict(groups=-1), dict(rows=-1), dict(cols=0), dict(eps=-1.0), dict(eps=float("nan")), dict(r=None), dict(f=None), dict(r_out=None), dict(post=0), dict(post=0, g1=None), dict(h=None),
    dict(h=None, g2=None), dict(NO_BLOCK, res_scale=0.5), dict(NO_BLOCK, post=1), dict(NO_BLOCK, gate=P[2]), dict(NO_BLOCK, h=None, g2=None, b2=None), dict(stats=P[9] + 4), dict(r_out=P[1] + 4),
    dict(r_out=P[2]), dict(r_out=P[8]), dict(h=P[5]), dict(h=P[0] + 400), dict(stats=P[0]), dict(stats=P[8]), dict(f=P[0] + 1), dict(h=P[8] + 2)])
def test_norm_forward_refuses(change):
    assert call("norm_residual_fwd", with_changes(FWD, FWD_OK, change)) == INVAL
    assert "norm_residual_fwd" in capi.lib().last_error()


BWD = "dev kind post groups rows cols dh dr_out f r_out gate g1 b1 res_scale g2 stats df dr inc_d dgate dg1 db1 dg2 db2 inc_g".split()
BWD_OK = [0, 1, 1, 2, 3, 100, P[0], P[1], P[2], P[3], P[4], P[5], P[6], 0.5, P[7], P[8], P[9], P[10], 0, P[11], P[12], P[13], P[14], P[15], 0]
BWD_NO_BLOCK = dict(f=None, gate=None, g1=None, b1=None, post=0, res_scale=1.0, df=None, dgate=None, dg1=None, db1=None)


@pytest.mark.parametrize("change", [
    dict(kind=-1), dict(post=3), dict(groups=-2), dict(rows=-1), dict(cols=0), dict(dh=None, dr_out=None), dict(dh=None), dict(dh=None, g2=None), dict(f=None), dict(BWD_NO_BLOCK, dgate=P[11]), dict(BWD_NO_BLOCK, df=P[9]),
    dict(BWD_NO_BLOCK, dg1=P[12]), dict(post=0), dict(post=0, g1=None, b1=None), dict(gate=None), dict(stats=None), dict(stats=P[8] + 8), dict(r_out=None), dict(df=P[0] + 4), dict(df=P[4]), dict(df=P[10]),
    dict(dr=P[8]), dict(dr=P[0], inc_d=1), dict(df=P[2], inc_d=1), dict(dgate=P[0]), dict(dg1=P[5]), dict(dg2=P[12]), dict(dh=P[0] + 2), dict(db2=P[15] + 1)])
def test_norm_backward_refuses(change):
    assert call("norm_residual_bwd", with_changes(BWD, BWD_OK, change)) == INVAL
    assert "norm_residual_bwd" in capi.lib().last_error()


DIST = "dev logits ids teacher teacher_lse labels weights rows cols ld k temperature alpha loss delta".split()
DIST_OK = [0, P[0], P[1], P[2], P[3], P[4], P[5], 6, 100, 104, 5, 2.0, 0.5, P[6], P[7]]


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(ids=None), dict(teacher=None), dict(loss=None), dict(labels=None), dict(rows=-1), dict(cols=0), dict(ld=99), dict(k=0), dict(k=-1), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=1e-39),
    dict(temperature=float("inf")), dict(temperature=float("nan")), dict(alpha=-0.1), dict(alpha=1.1), dict(alpha=float("nan")), dict(delta=P[0] + 4), dict(delta=P[1]), dict(loss=P[0]), dict(loss=P[7]), dict(loss=P[5]), dict(logits=P[0] + 2), dict(ids=P[1] + 1)])
def test_distill_refuses(change):
    assert call("distill", with_changes(DIST, DIST_OK, change)) == INVAL
    assert "distill" in capi.lib().last_error()


def test_limits_are_told_apart_from_mistakes():
    assert call("norm_residual_fwd", with_changes(FWD, FWD_OK, dict(cols=16385))) == LIMIT
    assert call("norm_residual_bwd", with_changes(BWD, BWD_OK, dict(cols=16385))) == LIMIT
    assert call("norm_residual_fwd", with_changes(FWD, FWD_OK, dict(rows=2 ** 31 - 1))) == LIMIT
    assert call("norm_residual_bwd", with_changes(BWD, BWD_OK, dict(groups=2 ** 31 - 1))) == LIMIT
    assert call("distill", with_changes(DIST, DIST_OK, dict(cols=344065, ld=344065))) == LIMIT
    assert call("distill", with_changes(DIST, DIST_OK, dict(k=1025))) == LIMIT
    assert call("distill", with_changes(DIST, DIST_OK, dict(rows=2 ** 31 - 1, delta=None, loss=1 << 60))) == LIMIT
    assert call("fp8_quantize", with_changes(QUANT, QUANT_OK, dict(rows=1, cols=2 ** 31 - 1, ldq=(1 << 31) + 16, qt=None, q=1 << 60, scale=1 << 61))) == LIMIT
    assert call("fp8_mult2d", with_changes(PROD, PROD_OK, dict(m=2 ** 31 - 1, c=1 << 60, qb=1 << 61, sb=1 << 62, sa=3 << 60))) == LIMIT


def test_right_arguments_reach_the_device():
    """Without a GPU every well-formed call fails with a device error, not with a refusal: there is no CPU fallback."""
    if capi.lib().device_count() > 0:
        pytest.skip("a GPU is visible: the addresses are made up")
    for name, args in (("fp8_quantize", QUANT_OK), ("fp8_mult2d", PROD_OK), ("norm_residual_fwd", FWD_OK), ("norm_residual_bwd", BWD_OK), ("distill", DIST_OK)):
        assert call(name, args) not in (0, INVAL, LIMIT), name
