"""Quantisation to microscaled 4-bit floats, the way back and the linear layer on such weights, through the C ABI against
numpy in 64 bits (mx4support.py)."""
import numpy as np
import pytest

import hipsupport as H
import mx4support as M
import vtsupport as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    h = H.Hip(kv_max=8)
    yield h
    h.close()


def quantize(hip, x, cols, bf16=False, shift=0):
    """x [rows, stride] on the host; its first `cols` columns -> codes, scales and the values that come back"""
    rows, stride = x.shape
    item = 2 if bf16 else 4
    src = S.f32_to_bf16_trunc(x) if bf16 else x
    dx = H.DevBuf(hip.lib, x.size * item + 64)
    hip.lib.tts_hip_to_device(dx.at(shift * item), np.ascontiguousarray(src).ctypes.data, x.size * item)
    p = M.panels(cols)
    dc, ds, dy = H.DevBuf(hip.lib, rows * p * 64), H.DevBuf(hip.lib, rows * p * 4), H.DevBuf(hip.lib, x.size * 4 + 64)
    hip.lib.tts_hip_memset(dy.ptr, 0x55, x.size * 4 + 64)
    assert hip.lib.tts_hip_mx4_quantize(dc.ptr, ds.ptr, dx.at(shift * item), int(bf16), rows, cols, stride) == 0
    assert hip.lib.tts_hip_mx4_dequantize(dy.at(4 * shift), dc.ptr, ds.ptr, rows, cols, stride) == 0
    got = dc.to_numpy(np.uint8, (rows, 64 * p)), ds.to_numpy(np.uint8, (rows, 4 * p)), dy.to_numpy(np.float32, x.size + 16)
    hip.check()
    for b in (dx, dc, ds, dy):
        b.free()
    return got


@pytest.mark.parametrize("rows,cols,gap,shift", [(1, 1, 0, 0), (3, 31, 0, 0), (2, 33, 7, 1), (5, 127, 1, 0), (4, 128, 0, 0), (7, 129, 3, 3), (37, 1000, 24, 0),
                                                 (300, 96, 0, 0), (9, 3072, 0, 0), (2, 20000, 8, 2), (1, 40000, 0, 0), (1000, 16, 16, 0)])
@pytest.mark.parametrize("bf16", [False, True])
def test_quantize(hip, rows, cols, gap, shift, bf16):
    r = np.random.default_rng(rows * 7 + cols)
    x = (r.standard_normal((rows, cols + gap)) * np.exp2(r.integers(-30, 30, (rows, 1)))).astype(np.float32)
    if bf16:
        x = S.bf16_to_f32(S.f32_to_bf16_trunc(x))
    codes, scales, back = quantize(hip, x, cols, bf16, shift)
    want = M.encode_matrix(x[:, :cols])
    assert np.array_equal(scales, want[1]) and np.array_equal(codes, want[0])
    v = M.decode(*want)[:, :cols].astype(np.float32)
    whole = back[shift:shift + x.size].reshape(x.shape)
    assert np.array_equal(whole[:, :cols], v)
    untouched = np.frombuffer(b"\x55" * 4, np.float32)[0]
    assert np.all(whole[:, cols:] == untouched) and np.all(back[:shift] == untouched) and np.all(back[shift + x.size:] == untouched)


def test_quantize_ties_extremes_and_what_is_not_finite(hip):
    x = np.zeros((12, 64), np.float32)
    x[0, :11] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -5, 7]                         # ties go to the even code
    x[1, :6] = [7.99, 7, 5.01, 1e-30, -0.0, -7.99]                                             # beyond 6, far below half of the first step
    x[2] = np.exp2(-149.0) * np.arange(1, 65)                                                  # subnormal: scale 2^-127
    x[3] = np.float32(3.4028235e38) * np.linspace(-1, 1, 64).astype(np.float32)
    x[4, 3], x[5, 40], x[6, 32], x[7, 31] = np.nan, np.inf, -np.inf, np.nan                    # one block of the two
    x[8] = np.exp2(-126.0) * np.linspace(-2, 2, 64)
    x[9] = np.exp2(-120.0) * np.linspace(-2, 2, 64)
    x[10] = np.exp2(np.linspace(-140, -110, 64))
    codes, scales, back = quantize(hip, x, 64)
    want = M.encode_matrix(x)
    assert np.array_equal(scales, want[1])
    finite = np.repeat(scales != 255, 16, 1)
    assert np.array_equal(codes[finite], want[0][finite])
    v = M.decode(*want)[:, :64].astype(np.float32)
    assert np.array_equal(back[:x.size].reshape(x.shape), v, equal_nan=True)
    assert np.isnan(v[4, :32]).all() and not np.isnan(v[4, 32:]).any() and np.isnan(v[5, 32:]).all() and not np.isnan(v[5, :32]).any()


def linear(hip, x, codes, scales, n, shift=0):
    m, k = x.shape
    dx = H.DevBuf(hip.lib, x.nbytes + 64)
    hip.lib.tts_hip_to_device(dx.at(4 * shift), np.ascontiguousarray(x).ctypes.data, x.nbytes)
    dc, ds, dy = H.DevBuf.from_numpy(hip.lib, codes), H.DevBuf.from_numpy(hip.lib, scales), H.DevBuf(hip.lib, 4 * (m * n + 64))
    hip.lib.tts_hip_memset(dy.ptr, 0x55, 4 * (m * n + 64))
    assert hip.lib.tts_hip_linear_mx4(dy.at(4 * shift), dx.at(4 * shift), dc.ptr, ds.ptr, m, k, n) == 0
    y = dy.to_numpy(np.float32, m * n + 64)
    hip.check()
    for b in (dx, dc, ds, dy):
        b.free()
    untouched = np.frombuffer(b"\x55" * 4, np.float32)[0]
    assert np.all(y[:shift] == untouched) and np.all(y[shift + m * n:] == untouched)
    return y[shift:shift + m * n].reshape(m, n)


def weights(n, k, seed):
    r = np.random.default_rng(seed)
    codes, scales = M.encode_matrix((r.standard_normal((n, k)) * 0.02 * np.exp2(r.integers(-6, 6, (n, 1)))).astype(np.float32))
    return codes, scales, M.decode(codes, scales)[:, :k]


def tolerance(x, w):
    """x enters as a sum of four planes of e2m1's wider relative e2m3, each of which leaves at most 2^-4 of its block's largest
    magnitude (half a step of the top binade over its smallest value); the accumulators of a panel of 128 are cut four or eight times
    at 2^-23, panels and K cuts are added at 2^-24."""
    k = x.shape[1]
    return 2.0 ** -16 * (M.block_max(x) @ np.abs(w).T) + (2.0 ** -20 + 2.0 ** -24 * (k / 64 + 24)) * (np.abs(x).astype(np.float64) @ np.abs(w).T)


@pytest.mark.parametrize("n,k", [(1, 1), (5, 33), (36, 3072), (257, 36), (16, 128), (300, 384), (1000, 1000), (513, 2176), (3072, 9216), (200, 12288)])
@pytest.mark.parametrize("m", [1, 2, 4, 5, 16, 17, 33, 129])
def test_linear(hip, m, n, k):
    codes, scales, w = weights(n, k, n + k)
    x = S.f32_normal((m, k), 900 + m + k)
    y = linear(hip, x, codes, scales, n)
    off = np.abs(y - x.astype(np.float64) @ w.T)
    assert np.all(off <= tolerance(x, w)), float((off / tolerance(x, w)).max())


@pytest.mark.parametrize("m,n,k", [(700, 640, 512), (1531, 300, 1000), (97, 9216, 256)])
def test_linear_many_rows(hip, m, n, k):
    codes, scales, w = weights(n, k, 5)
    x = S.f32_normal((m, k), 77)
    off = np.abs(linear(hip, x, codes, scales, n) - x.astype(np.float64) @ w.T)
    assert np.all(off <= tolerance(x, w))


@pytest.mark.parametrize("m", [1, 3, 20, 70])
def test_linear_rows_that_lie_on_no_16_bytes(hip, m):
    codes, scales, w = weights(130, 203, 6)
    x = S.f32_normal((m, 203), 78)
    off = np.abs(linear(hip, x, codes, scales, 130, shift=1) - x.astype(np.float64) @ w.T)
    assert np.all(off <= tolerance(x, w))


@pytest.mark.parametrize("m", [1, 4, 6, 40, 200])
def test_linear_what_is_not_finite_stays_in_its_row_and_its_column(hip, m):
    n, k = 300, 640
    codes, scales, w = weights(n, k, 7)
    x = S.f32_normal((m, k), 79)
    clean = linear(hip, x, codes, scales, n)
    x[m // 2, 333] = np.inf
    scales[17, 6] = 255
    y = linear(hip, x, codes, scales, n)
    rows, cols = np.arange(m) != m // 2, np.arange(n) != 17
    assert np.array_equal(y[rows][:, cols], clean[rows][:, cols])
    assert not np.isfinite(y[m // 2]).any() and np.isnan(y[:, 17]).all()


@pytest.mark.parametrize("m", [1, 7, 50])
def test_linear_large_and_small_values(hip, m):
    """Blocks of x across the range of floats; the smallest are held to 2^-127 times their planes' steps."""
    n, k = 64, 512
    codes, scales, w = weights(n, k, 8)
    x = S.f32_normal((m, k), 80) * np.repeat(np.exp2(np.linspace(-140, 100, k // 32)), 32).astype(np.float32)
    x[:, 64:96] = 0
    off = np.abs(linear(hip, x, codes, scales, n) - x.astype(np.float64) @ w.T)
    assert np.all(off <= tolerance(x, w) + 2.0 ** -127 * np.abs(w).sum(1))


def test_linear_results_do_not_depend_on_the_call(hip):
    codes, scales, _ = weights(512, 1024, 9)
    for m in (1, 16, 64, 300):
        x = S.f32_normal((m, 1024), 81)
        assert np.array_equal(linear(hip, x, codes, scales, 512), linear(hip, x, codes, scales, 512))


def test_what_is_called_behind_a_memset_runs_behind_it(hip):
    """Large enough that the memory is still being set when the next call is queued."""
    lib, rows, k = hip.lib, 4096, 8192
    dx, dc, ds = H.DevBuf(lib, rows * k * 4), H.DevBuf(lib, rows * k // 2), H.DevBuf(lib, rows * k // 32)
    for fill in (0x55, 0x3f):
        lib.tts_hip_memset(dx.ptr, fill, dx.nbytes)
        assert lib.tts_hip_mx4_quantize(dc.ptr, ds.ptr, dx.ptr, 0, rows, k, 0) == 0
        lib.tts_hip_memset(dx.ptr, 0, dx.nbytes)
        assert lib.tts_hip_mx4_dequantize(dx.ptr, dc.ptr, ds.ptr, rows, k, 0) == 0
        want = M.decode(*M.encode(np.full((1, 32), np.frombuffer(bytes([fill] * 4), np.float32)[0])))
        assert np.all(dx.to_numpy(np.float32, (rows, k)) == np.float32(want[0, 0]))
    hip.check()
    for b in (dx, dc, ds):
        b.free()


@pytest.mark.parametrize("m", [1, 7, 40, 1100])
def test_matrices_past_32_bits(hip, m):
    """4.6 GB of codes, or of results: the last rows are random, the others zeros; quantised from 4.9 GB of values and decoded again."""
    lib, n, k, tail = hip.lib, 1_100_000, 8192, 70
    r = np.random.default_rng(13)
    w = r.standard_normal((tail, k)).astype(np.float32)
    codes, scales = M.encode_matrix(w)
    if m == 1:
        rows = 150_000
        dx, dc, ds = H.DevBuf(lib, rows * k * 4), H.DevBuf(lib, rows * k // 2), H.DevBuf(lib, rows * k // 32)
        lib.tts_hip_memset(dx.ptr, 0, dx.nbytes)
        lib.tts_hip_to_device(dx.at((rows - tail) * k * 4), w.ctypes.data, w.nbytes)
        assert lib.tts_hip_mx4_quantize(dc.ptr, ds.ptr, dx.ptr, 0, rows, k, 0) == 0
        lib.tts_hip_memset(dx.ptr, 0x55, dx.nbytes)
        assert lib.tts_hip_mx4_dequantize(dx.ptr, dc.ptr, ds.ptr, rows, k, 0) == 0
        for b, want in ((dc, codes), (ds, scales), (dx, M.decode(codes, scales).astype(np.float32))):
            for at, have in ((b.nbytes - want.nbytes, want), (0, np.zeros_like(want))):
                got = np.empty_like(want)
                lib.tts_hip_to_host(got.ctypes.data, b.at(at), got.nbytes)
                assert np.array_equal(got, have)
            b.free()
    dc, ds, dy = H.DevBuf(lib, n * k // 2), H.DevBuf(lib, n * k // 32), H.DevBuf(lib, m * n * 4)
    x = S.f32_normal((m, k), 90)
    dx = H.DevBuf.from_numpy(lib, x)
    for b, tail_bytes in ((dc, codes), (ds, scales)):
        lib.tts_hip_memset(b.ptr, 0, b.nbytes)
        lib.tts_hip_to_device(b.at(b.nbytes - tail_bytes.nbytes), tail_bytes.ctypes.data, tail_bytes.nbytes)
    lib.tts_hip_memset(dy.ptr, 0x55, dy.nbytes)
    assert lib.tts_hip_linear_mx4(dy.ptr, dx.ptr, dc.ptr, ds.ptr, m, k, n) == 0
    full = M.decode(codes, scales)
    for row in (0, m // 2, m - 1):
        got = np.empty(n, np.float32)
        lib.tts_hip_to_host(got.ctypes.data, dy.at(row * n * 4), got.nbytes)
        off = np.abs(got[n - tail:] - x[row].astype(np.float64) @ full.T)
        assert not got[:n - tail].any() and np.all(off <= tolerance(x[row:row + 1], full)[0])
    hip.check()
    for b in (dc, ds, dx, dy):
        b.free()


@pytest.mark.parametrize("cols", [1, 40])
def test_quantize_more_rows_than_a_launch_has_threads_for(hip, cols):
    """2^28 rows and a few, 17 GB of codes: rows around the places where a launch ends (2^27 - 8 and 2^28 - 16) and at both
    ends are random, the others zeros."""
    lib, rows, wide = hip.lib, (1 << 28) + 3, 48
    dx, dc, ds = H.DevBuf(lib, rows * cols * 4), H.DevBuf(lib, rows * 64), H.DevBuf(lib, rows * 4)
    lib.tts_hip_memset(dx.ptr, 0, dx.nbytes)
    lib.tts_hip_memset(dc.ptr, 0x55, dc.nbytes)
    lib.tts_hip_memset(ds.ptr, 0x55, ds.nbytes)
    first = [0, (1 << 27) - 8 - wide // 2, (1 << 28) - 16 - wide // 2]
    x = [S.f32_normal((min(wide, rows - f), cols), 95 + i) for i, f in enumerate(first)]
    for f, a in zip(first, x):
        lib.tts_hip_to_device(dx.at(f * cols * 4), a.ctypes.data, a.nbytes)
    assert lib.tts_hip_mx4_quantize(dc.ptr, ds.ptr, dx.ptr, 0, rows, cols, 0) == 0
    lib.tts_hip_memset(dx.ptr, 0x55, dx.nbytes)
    assert lib.tts_hip_mx4_dequantize(dx.ptr, dc.ptr, ds.ptr, rows, cols, 0) == 0
    hip.check()

    def rows_of(b, at, width, n, dtype):
        got = np.empty((n, width), dtype)
        lib.tts_hip_to_host(got.ctypes.data, b.at(at * got.strides[0]), got.nbytes)
        return got

    for f, a in list(zip(first, x)) + [(at, np.zeros((wide, cols), np.float32)) for at in (wide, (1 << 27) + wide, (1 << 28) - 1000)]:
        n = len(a)
        codes, scales = M.encode_matrix(a)
        assert np.array_equal(rows_of(dc, f, 64, n, np.uint8), codes) and np.array_equal(rows_of(ds, f, 4, n, np.uint8), scales)
        assert np.array_equal(rows_of(dx, f, cols, n, np.float32), M.decode(codes, scales)[:, :cols].astype(np.float32))
    for b in (dx, dc, ds):
        b.free()


# rows of x, weight rows, columns -> tile of vt_mx4_plans.h (weight rows x rows of x) and cuts of K on 256 CUs, which test_mx4_plans_cpu.py asserts: one, two and more panels,
# odd and even, and ends inside a tile and a panel
TILES = {(515, 8250, 128): ("256x128", 1), (515, 8250, 200): ("256x128", 1), (515, 8250, 384): ("256x128", 1), (300, 13100, 1300): ("256x128", 1), (515, 8202, 3072): ("256x128", 1),
         (130, 13100, 3190): ("256x128", 2), (2101, 129, 9216): ("256x128", 12), (226, 3072, 9216): ("256x128", 8),
         (200, 11514, 128): ("128x64", 1), (200, 11514, 200): ("128x64", 1), (400, 9000, 300): ("128x64", 1), (400, 9000, 1000): ("128x64", 1), (40, 11514, 3190): ("128x64", 5),
         (40, 8250, 9216): ("128x64", 7),
         (97, 9216, 256): ("128x32", 1), (700, 640, 512): ("128x32", 1), (16, 20000, 1000): ("128x32", 1), (9, 9216, 3072): ("128x32", 6), (64, 9216, 3072): ("128x32", 3)}


def random_weights(n, k, seed):
    """Any codes, scales 2^-12 .. 2^-5: [n, k] -> codes, scales, values"""
    r = np.random.default_rng(seed)
    p = M.panels(k)
    codes, scales = r.integers(0, 256, (n, 64 * p), dtype=np.uint8), r.integers(115, 123, (n, 4 * p), dtype=np.uint8)
    codes[:, (k + 1) // 2:] = 0
    if k % 2:
        codes[:, k // 2] &= 15
    return codes, scales, M.decode(codes, scales)[:, :k]


def sums(x, w):
    """What is left of tolerance() where x's planes are known: the accumulators and the sums of panels."""
    return (2.0 ** -20 + 2.0 ** -24 * (x.shape[1] / 64 + 24)) * (np.abs(x) @ np.abs(w).T)


@pytest.mark.parametrize("m,n,k", TILES)
@pytest.mark.parametrize("shift", [0, 1])
def test_linear_tiles(hip, m, n, k, shift):
    codes, scales, w = random_weights(n, k, n + k)
    x = S.f32_normal((m, k), 910 + m + k)
    y = linear(hip, x, codes, scales, n, shift)
    off = np.abs(y - x.astype(np.float64) @ w.T)
    tol = tolerance(x, w)
    assert np.all(off <= tol), float((off / tol).max())
    assert np.array_equal(y, linear(hip, x, codes, scales, n, shift))


@pytest.mark.parametrize("m,n,k", [(515, 8250, 200), (515, 8250, 384), (130, 13100, 3190), (200, 11514, 200), (400, 9000, 300), (97, 9216, 256), (16, 20000, 1000)])
def test_linear_tiles_what_is_not_finite_stays_in_its_row_and_its_column(hip, m, n, k):
    codes, scales, _ = random_weights(n, k, 17)
    x = S.f32_normal((m, k), 92)
    clean = linear(hip, x, codes, scales, n)
    bad, out = [0, m // 2, m - 1], [5, n // 2, n - 1]
    for i, (s, r) in enumerate(zip(bad, out)):
        x[s, (i * k + k // 2) // 3] = (np.inf, np.nan, -np.inf)[i]
        scales[r, (i * k // 32 + 1) // 3] = 255
    y = linear(hip, x, codes, scales, n)
    rows, cols = np.ones(m, bool), np.ones(n, bool)
    rows[bad], cols[out] = False, False
    assert np.isfinite(clean).all() and np.array_equal(y[rows][:, cols], clean[rows][:, cols])
    assert np.isnan(y[~rows]).all() and np.isnan(y[:, ~cols]).all()


@pytest.mark.parametrize("m,n,k", [(8, 1000, 3072), (8, 36, 9216), (6, 300, 20000), (8, 513, 12288), (8, 5, 33)])
def test_linear_eight_rows(hip, m, n, k):
    codes, scales, w = random_weights(n, k, 18)
    x = S.f32_normal((m, k), 93)
    off = np.abs(linear(hip, x, codes, scales, n) - x.astype(np.float64) @ w.T)
    assert np.all(off <= tolerance(x, w))


@pytest.mark.parametrize("m,n,k", [(1, 9216, 3072), (8, 3072, 9216), (64, 9216, 3072), (226, 3072, 9216), (515, 8202, 3072), (700, 640, 512)])
def test_linear_error_of_a_normal_row(hip, m, n, k):
    """The error as a share of the results' norm on values ~N(0, 1).  Five planes leave 2.0e-8 of x's norm, and so of y's, weights being independent of it.  A panel's sum is
    cut at 2^-23 in its last product and, of a tile, in the one in front of it: 2^-22 of it at most, 2.4e-7 of the norm of P panels that are independent of each other.  Adding
    P of them rounds partial sums of sqrt(i) at up to 2^-24, uniformly, i.e. 2^-24 / sqrt(3): sqrt(P / 2) 2^-24 / sqrt(3) of the norm, 2.1e-7 at 72.  Together, as if they all
    pointed the same way, 4.7e-7 (four planes leave 5.2e-7); and 2 % for what a finite row's planes are off from 2.0e-8."""
    codes, scales, w = random_weights(n, k, 19)
    x = S.f32_normal((m, k), 94)
    want = x.astype(np.float64) @ w.T
    off = np.linalg.norm(linear(hip, x, codes, scales, n) - want) / np.linalg.norm(want)
    bound = 1.02 * 2.0e-8 + 2.0 ** -22 + np.sqrt(M.panels(k) / 2) * 2.0 ** -24 / np.sqrt(3)
    assert off <= bound, off


@pytest.mark.parametrize("m", [1, 4, 7, 40, 300])
@pytest.mark.parametrize("large", [30.0, 1000.0, 1e6])
def test_linear_one_value_far_above_its_neighbours(hip, m, large):
    """A channel of 32 `large` times the others, and no weight on it: what is left of the others by the planes' definition."""
    n, k = 320, 1024
    codes, scales, _ = random_weights(n, k, 20)
    codes = codes.reshape(n, -1, 16)
    codes[:, :, 2] &= 0x0f                                # value 5 of 32
    codes = codes.reshape(n, -1)
    w = M.decode(codes, scales)
    x = S.f32_normal((m, k), 96)
    x[:, 5::32] *= np.float32(large)
    held = M.planes(x)
    off = np.abs(linear(hip, x, codes, scales, n) - held @ w.T)
    # a product may be cut at 2^-23 of the largest that the exponents of its 128 columns could make, a large value's with no weight among them
    top = [np.repeat(np.abs(a).reshape(len(a), -1, 128).max(-1), 128, -1).astype(np.float64) for a in (x, w)]
    tol = sums(held, w) + 2.0 ** -23 * (top[0] @ top[1].T)
    assert np.all(off <= tol), float((off / tol).max())


@pytest.mark.parametrize("m", [1, 4, 7, 40, 600])
def test_linear_holds_every_value(hip, m):
    """Weights that pick one column each: x comes back to 2^-21 of the largest of its block, as its planes hold it, and each of the five planes' products cut at 2^-23 of
    what the block's exponents could make."""
    k = 300
    w = np.eye(k, dtype=np.float32)
    codes, scales = M.encode_matrix(w)
    r = np.random.default_rng(21)
    x = (r.standard_normal((m, k)) * np.exp2(r.integers(-12, 12, (m, k)))).astype(np.float32)
    y = linear(hip, x, codes, scales, k)
    assert np.all(np.abs(y - x.astype(np.float64)) <= (2.0 ** -21 + 5 * 2.0 ** -23) * M.block_max(x))
