"""GPU parity of the 8-bit dense operators against 64-bit arithmetic on the same 8-bit values."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
F = np.float32
E4M3, E5M2 = 0, 1
LARGEST = {E4M3: 448.0, E5M2: 57344.0}


def decode_table(fmt):
    """The 256 values of a format (IEEE-like fields; e4m3 has no infinities, its NaN is 0x7f / 0xff)."""
    bits, bias = (3, 7) if fmt == E4M3 else (2, 15)
    code = np.arange(256)
    sign, exp, man = np.where(code & 128, -1.0, 1.0), (code & 127) >> bits, code & ((1 << bits) - 1)
    v = np.where(exp == 0, man * 2.0 ** (1 - bias - bits), (1 + man * 2.0 ** -bits) * 2.0 ** (exp - bias))
    if fmt == E4M3:
        v = np.where((code & 127) == 127, np.nan, v)
    else:
        v = np.where(exp == 31, np.where(man == 0, np.inf, np.nan), v)
    return sign * v


def round8(x, fmt):
    """Nearest value of the format, ties to even; x within its range."""
    bits, least = (3, -6) if fmt == E4M3 else (2, -14)
    x = np.asarray(x, np.float64)
    e = np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** (least - 10)))), least)
    step = 2.0 ** (e - bits)
    return np.clip(np.round(x / step) * step, -LARGEST[fmt], LARGEST[fmt])


def up(n, to):
    return -(-n // to) * to


def quantize_ref(a, fmt, block, pow2):
    """Values (as 64-bit numbers) and scales [column block][row block] of a matrix, with the roundings of the definition."""
    r, c = a.shape
    nb, nr = up(c, 128) // 128, up(r, block) // block
    vals, scale = np.empty(a.shape), np.empty((nb, nr), F)
    for b in range(nb):
        for i in range(nr):
            at = np.s_[i * block:(i + 1) * block, b * 128:(b + 1) * 128]
            peak = F(max(np.abs(a[at]).max(), 2.0 ** -100))
            if pow2:
                s = 2.0 ** np.ceil(np.log2(np.float64(peak) / LARGEST[fmt]))
                scale[b, i], vals[at] = s, round8(np.float64(a[at]) / s, fmt)
            else:
                scale[b, i] = F(peak / F(LARGEST[fmt]))
                vals[at] = round8((a[at] * F(F(LARGEST[fmt]) / peak)).astype(F), fmt)
    return vals, scale


class Eight:
    """A quantised matrix on the device, its rows `ld` bytes apart and the bytes between them set to `fill`."""

    def __init__(self, lib, rows, cols, fmt, block, ld=None, fill=0x7f):
        self.lib, self.rows, self.cols, self.fmt, self.block = lib, rows, cols, fmt, block
        self.ld = ld or up(max(cols, 1), 16)
        self.q = lib.to_device(np.full((max(rows, 1), self.ld), fill, np.uint8), dtype=np.uint8)
        self.scale = lib.to_device(np.full((up(cols, 128) // 128, up(rows, block) // block), np.nan, F))

    def set(self, codes, scale):
        raw = np.full((self.rows, self.ld), 0x7f, np.uint8)
        raw[:, :self.cols] = codes
        self.q = self.lib.to_device(raw, dtype=np.uint8)
        self.scale = self.lib.to_device(scale)
        return self

    def codes(self):
        return self.q.numpy()

    def values(self):
        return decode_table(self.fmt)[self.codes()[:, :self.cols]]

    def real(self):
        """What it stands for, in 64 bits."""
        s = self.scale.numpy().astype(np.float64)
        return self.values() * np.repeat(np.repeat(s.T, self.block, 0)[:self.rows], 128, 1)[:, :self.cols]

    def args(self):
        return self.q, self.ld, self.scale, self.fmt, self.block


def quantize(lib, a, fmt, block, pow2, which="qt"):
    d, r, c = lib.to_device(a), *a.shape
    q, t = Eight(lib, r, c, fmt, block, up(c, 16) + 32), Eight(lib, c, r, fmt, block)
    lib.call("fp8_quantize", 0, d, r, c, fmt, block, pow2, *((q.q, q.ld, q.scale) if "q" in which else (None, 0, None)),
             *((t.q, t.ld, t.scale) if "t" in which else (None, 0, None)))
    return q, t


def matrix(rng, r, c):
    a = rng.standard_normal((r, c)) * np.exp(rng.standard_normal((1, c))) * np.exp(2 * rng.standard_normal((r, 1)))
    return a.astype(F)


@pytest.mark.parametrize("fmt", [E4M3, E5M2])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("pow2", [0, 1])
@pytest.mark.parametrize("r,c", [(1, 1), (1, 129), (127, 4), (128, 128), (130, 257), (17, 300), (300, 64), (258, 516)])
def test_quantize_gives_the_defined_bits(lib, r, c, block, fmt, pow2):
    rng = np.random.default_rng(r * 1000 + c + fmt)
    a = matrix(rng, r, c)
    a[rng.random(a.shape) < 0.05] = 0
    for which in ("qt", "q", "t"):
        q, t = quantize(lib, a, fmt, block, pow2, which)
        for got, src, there in ((q, a, "q" in which), (t, np.ascontiguousarray(a.T), "t" in which)):
            if not there:
                assert np.all(got.codes() == 0x7f) and np.all(np.isnan(got.scale.numpy()))
                continue
            vals, scale = quantize_ref(src, fmt, block, pow2)
            assert np.array_equal(got.scale.numpy(), scale)
            assert np.array_equal(got.values(), vals)
            assert np.all(got.codes()[:, got.cols:] == 0x7f)          # bytes between the rows stay


@pytest.mark.parametrize("pow2", [0, 1])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_quantize_borders(lib, fmt, pow2):
    """Zeros, the smallest magnitudes, peaks on both sides of a power of two, infinities, NaN."""
    top = F(LARGEST[fmt])
    rows = [np.zeros(128, F), np.full(128, 1e-45, F), np.full(128, 2.0 ** -100, F), np.full(128, 3e38, F)]
    for peak in (top, np.nextafter(top, F(np.inf)), np.nextafter(top, F(0)), F(1), F(2.0 ** -60) * top):
        row = np.linspace(-1, 1, 128).astype(F) * peak
        row[5] = peak
        rows.append(row)
    a = np.stack(rows)
    for block in (1, 128):
        q, _ = quantize(lib, a, fmt, block, pow2)
        vals, scale = quantize_ref(a, fmt, block, pow2)
        assert np.array_equal(q.values(), vals) and np.array_equal(q.scale.numpy(), scale)
    bad = a[4:6].copy()
    bad[0, 7], bad[1, 9] = np.nan, np.inf
    q, _ = quantize(lib, bad, fmt, 1, pow2)
    vals, scale = quantize_ref(np.nan_to_num(bad[:1], nan=0.0), fmt, 1, pow2)
    got = q.values()
    assert np.isnan(got[0, 7]) and np.array_equal(np.delete(got[0], 7), np.delete(vals[0], 7)) and q.scale.numpy()[0, 0] == scale[0, 0]
    assert np.isinf(q.scale.numpy()[0, 1]) and np.isnan(got[1, 9])


def random_codes(rng, r, c, fmt):
    """Any finite codes: every exponent and sign, zeros and subnormals among them."""
    codes = rng.integers(0, 256, (r, c)).astype(np.uint8)
    bad = ~np.isfinite(decode_table(fmt)[codes])
    codes[bad] = rng.integers(0, 0x70, int(bad.sum())).astype(np.uint8)
    return codes


def operand(lib, rng, r, c, fmt, block, ld=None):
    scale = np.exp(rng.standard_normal((up(c, 128) // 128, up(r, block) // block))).astype(F)
    return Eight(lib, r, c, fmt, block, ld).set(random_codes(rng, r, c, fmt), scale)


def check_product(lib, a, b, inc, rng):
    m, n, k = a.rows, b.rows, a.cols
    c0 = rng.standard_normal((m, n)).astype(F) * F(1e3)
    c = lib.to_device(c0)
    lib.call("fp8_mult2d", 0, *a.args(), *b.args(), c, inc, m, n, k)
    lib.sync()
    ra, rb = a.real(), b.real()
    want, size = ra @ rb.T + (c0 if inc else 0), np.abs(ra) @ np.abs(rb).T
    got = c.numpy()
    # Products of 8-bit values are exact.  A block is four instructions of 32 products each; an instruction may drop, from each of its 33
    # terms, what lies below 2^-23 of the largest of them, so a block is off by 4 * 33 * 2^-23 of the sum of its magnitudes at most; scaling
    # rounds twice, the sum over the blocks and the old value once a block.
    blocks = up(k, 128) // 128
    bound = (4 * 33 * 2.0 ** -23 + (blocks + 3) * 2.0 ** -24) * size + 2.0 ** -24 * np.abs(want)
    assert np.all(np.abs(got - want) <= bound), (np.abs(got - want) / (bound + 1e-300)).max()
    # rounding errors do not all point the same way: the whole is far nearer
    off = np.linalg.norm(got - want) / np.linalg.norm(size)
    assert off <= 2.0 ** -22, off


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 300, 1000), (3, 129, 127), (16, 64, 256), (17, 1000, 520), (33, 70, 129), (64, 1000, 2048), (65, 257, 384), (128, 128, 4096),
                                   (129, 1, 700), (200, 333, 1290), (257, 130, 64), (700, 900, 300), (1, 5000, 4100)])
@pytest.mark.parametrize("blocks", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("inc", [0, 1])
def test_product(lib, m, n, k, blocks, inc):
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    check_product(lib, operand(lib, rng, m, k, E4M3, blocks[0]), operand(lib, rng, n, k, E4M3, blocks[1], up(k, 16) + 48), inc, rng)


# many tiles of 256 x 256: whole and ragged ones, one and several rounds of them, few and many K-blocks, an odd number of them
@pytest.mark.parametrize("m,n,k", [(1537, 1601, 260), (300, 9601, 700), (9999, 130, 513), (2048, 1536, 128), (4096, 4352, 64), (1600, 1700, 2000), (2500, 2300, 300), (2100, 2400, 140), (2400, 2100, 140), (4096, 2304, 384)])
@pytest.mark.parametrize("blocks", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("inc", [0, 1])
def test_large_product(lib, m, n, k, blocks, inc):
    test_product(lib, m, n, k, blocks, inc)


@pytest.mark.parametrize("m", [1, 24, 100, 300, 9000])
@pytest.mark.parametrize("formats", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
def test_product_formats(lib, m, formats):
    rng = np.random.default_rng(m)
    check_product(lib, operand(lib, rng, m, 650, formats[0], 1), operand(lib, rng, 210, 650, formats[1], 128), 0, rng)


def test_product_of_nothing(lib):
    rng = np.random.default_rng(0)
    a, b = operand(lib, rng, 5, 16, E4M3, 1), operand(lib, rng, 7, 16, E4M3, 1)
    for inc in (0, 1):
        c = lib.to_device(np.full((5, 7), 3.0, F))
        lib.call("fp8_mult2d", 0, a.q, 16, a.scale, 0, 1, b.q, 16, b.scale, 0, 1, c, inc, 5, 7, 0)
        assert np.all(c.numpy() == (3.0 if inc else 0.0))
        lib.call("fp8_mult2d", 0, a.q, 16, a.scale, 0, 1, b.q, 16, b.scale, 0, 1, c, inc, 0, 7, 16)
        lib.call("fp8_quantize", 0, None, 0, 5, 0, 1, 0, a.q, 16, a.scale, None, 0, None)


def test_values_outside_the_operands_do_not_matter(lib):
    """NaN codes in the bytes between rows, NaN scales of rows that are not there: operands cut out of larger ones."""
    rng = np.random.default_rng(5)
    a, b = operand(lib, rng, 130, 200, E4M3, 1, 512), operand(lib, rng, 140, 200, E4M3, 1, 256)
    c = lib.zeros((100, 90))
    sa, sb = a.scale.numpy(), b.scale.numpy()
    sa2, sb2 = np.ascontiguousarray(sa[:, :100]), np.ascontiguousarray(sb[:, :90])
    lib.call("fp8_mult2d", 0, a.q, 512, lib.to_device(sa2), 0, 1, b.q, 256, lib.to_device(sb2), 0, 1, c, 0, 100, 90, 200)
    want = a.real()[:100] @ b.real()[:90].T
    assert np.linalg.norm(c.numpy() - want) <= 2.0 ** -20 * np.linalg.norm(np.abs(a.real()[:100]) @ np.abs(b.real()[:90]).T)


def test_not_a_number_stays_in_its_row(lib):
    rng = np.random.default_rng(6)
    for m in (4, 300):
        a, b = operand(lib, rng, m, 300, E4M3, 1), operand(lib, rng, 150, 300, E4M3, 128)
        codes = a.codes()[:, :300].copy()
        codes[2, 17] = 0x7f
        a.set(codes, a.scale.numpy())
        c = lib.zeros((m, 150))
        lib.call("fp8_mult2d", 0, *a.args(), *b.args(), c, 0, m, 150, 300)
        bad = np.isnan(c.numpy())
        assert bad[2].all() and not np.delete(bad, 2, 0).any()


def test_same_call_same_bits(lib):
    rng = np.random.default_rng(7)
    for m, n, k in ((3, 500, 3000), (300, 700, 900)):
        a, b = operand(lib, rng, m, k, E4M3, 1), operand(lib, rng, n, k, E4M3, 128)
        out = []
        for _ in range(3):
            c = lib.empty((m, n))
            lib.call("fp8_mult2d", 0, *a.args(), *b.args(), c, 0, m, n, k)
            out.append(c.numpy())
        assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])


def test_gradients_of_a_dense_layer(lib):
    """y = x w^T in 8 bits: with power-of-two scales dx and dw are the products of the same 8-bit values, so <dy, y(x + e) - y(x)> is <dx, e> for
    steps e that keep every quantised value exact (x, w, dy on the 8-bit grid to begin with)."""
    rng = np.random.default_rng(8)
    m, n, k = 72, 136, 200
    grid = lambda *s: (rng.integers(-8, 9, s)).astype(F)      # noqa: E731  small whole numbers are 8-bit values under any power-of-two scale up to 2^4
    x, w, dy = grid(m, k), grid(n, k), grid(m, n)

    def forward(x, w):
        (xq, _), (wq, _) = quantize(lib, x, E4M3, 1, 1), quantize(lib, w, E4M3, 128, 1)
        y = lib.empty((m, n))
        lib.call("fp8_mult2d", 0, *xq.args(), *wq.args(), y, 0, m, n, k)
        return y.numpy().astype(np.float64)
    (xq, xt), (wq, wt), (dq, dt) = quantize(lib, x, E4M3, 1, 1), quantize(lib, w, E4M3, 128, 1), quantize(lib, dy, E5M2, 1, 1)
    dyq = dq.real()
    dx, dw = lib.empty((m, k)), lib.empty((n, k))
    lib.call("fp8_mult2d", 0, *dq.args(), *wt.args(), dx, 0, m, k, n)
    lib.call("fp8_mult2d", 0, *dt.args(), *xt.args(), dw, 0, n, k, m)
    assert np.array_equal(dx.numpy(), dyq @ w.astype(np.float64)) and np.array_equal(dw.numpy(), dt.real() @ x.astype(np.float64))
    ex, ew = grid(m, k), grid(n, k)
    base = forward(x, w)
    assert np.sum(dyq * (forward(ex, w))) == np.sum(dx.numpy().astype(np.float64) * ex)             # y is linear in x and in w
    assert np.sum(dyq * (forward(x, ew))) == np.sum(dt.real().T * forward(x, ew)) == np.sum(dw.numpy().astype(np.float64) * ew)
    assert np.array_equal(base, x.astype(np.float64) @ w.T.astype(np.float64))


def test_zeros_owed_to_the_result(lib):
    rng = np.random.default_rng(9)
    a, b = operand(lib, rng, 300, 256, E4M3, 1), operand(lib, rng, 400, 256, E4M3, 128)
    plain = lib.empty((300, 400))
    lib.call("fp8_mult2d", 0, *a.args(), *b.args(), plain, 0, 300, 400, 256)
    lib.call("set_option", b"lazy_zero", 1)
    try:
        c = lib.to_device(np.full((300, 400), 5.0, F))
        lib.call("fill", 0, c, c.size, 0.0)
        lib.call("fp8_mult2d", 0, *a.args(), *b.args(), c, 1, 300, 400, 256)
        assert np.array_equal(c.numpy(), plain.numpy())
    finally:
        lib.call("set_option", b"lazy_zero", 0)
