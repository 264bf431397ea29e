"""The key/value cache in 4 bits through the C ABI: append, read and attention against numpy in 64 bits (mx4support.py), and a
decoder layer in 4 bits as a program runs it."""
import ctypes as C

import numpy as np
import pytest

import hipsupport as H
import mx4support as M
import vtsupport as S

pytestmark = pytest.mark.gpu
LAYOUTS = [(32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 256), (14, 2, 64), (6, 2, 192), (20, 1, 64)]


@pytest.fixture(scope="module")
def hip():
    h = H.Hip(kv_max=8)
    yield h
    h.close()


@pytest.mark.parametrize("kv_heads,hd", [(8, 128), (1, 64), (3, 192), (2, 256)])
@pytest.mark.parametrize("n,pos,gap,shift", [(1, 0, 0, 0), (1, 301, 0, 0), (37, 5, 12, 0), (200, 100, 3, 1)])
def test_append_and_read(hip, kv_heads, hd, n, pos, gap, shift):
    rows, width = 310, kv_heads * hd
    c = M.Cache(hip, rows, kv_heads, hd)
    for a in c.host.values():
        a[:] = np.random.default_rng(a.size).integers(0, 255, a.shape)
    cache = c.upload()
    x = [S.f32_normal((n, width + gap), 10 + i) * 3 for i in range(2)]
    dev = [H.DevBuf(hip.lib, a.nbytes + 64) for a in x]
    for d, a in zip(dev, x):
        hip.lib.tts_hip_to_device(d.at(4 * shift), a.ctypes.data, a.nbytes)
    k, v = (d.at(4 * shift) for d in dev)
    assert hip.lib.tts_hip_kv4_append(cache, k, v, n, pos, width + gap) == 0
    got = c.download()
    c.fill(*[a[:, :width].reshape(n, kv_heads, hd).transpose(1, 0, 2) for a in x], pos)
    for name in got:
        assert np.array_equal(got[name], c.host[name]), name                                    # the other rows too
    for d, a in zip(dev, x):
        hip.lib.tts_hip_memset(d.ptr, 0x55, a.nbytes + 64)
    assert hip.lib.tts_hip_kv4_read(k, v, cache, n, pos, width + gap) == 0
    for d, a, name in zip(dev, x, "kv"):
        back = d.to_numpy(np.float32, a.size + 16)[shift:shift + a.size].reshape(a.shape)
        want = M.decode(c.host[name + "c"][:, pos:pos + n], c.host[name + "s"][:, pos:pos + n])
        assert np.array_equal(back[:, :width], want.transpose(1, 0, 2).reshape(n, width).astype(np.float32))
        assert np.all(back[:, width:] == np.frombuffer(b"\x55" * 4, np.float32)[0])
        d.free()
    hip.check()
    c.free()


def attend(hip, cache, q, pos, heads, scale):
    dq, do = H.DevBuf.from_numpy(hip.lib, q), H.DevBuf(hip.lib, q.nbytes + 64)
    hip.lib.tts_hip_memset(do.ptr, 0x55, q.nbytes + 64)
    assert hip.lib.tts_hip_kv4_attention(do.ptr, dq.ptr, cache, q.shape[0], pos, heads, scale) == 0
    out = do.to_numpy(np.float32, q.size + 16)
    hip.check()
    dq.free()
    do.free()
    assert np.all(out[q.size:] == np.frombuffer(b"\x55" * 4, np.float32)[0])
    return out[:q.size].reshape(q.shape)


def oracle(q, k, v, pos, heads, scale, absolute=True):
    """-> out, tolerance [rows, heads * hd]; k, v [kv_heads, pos + rows, hd]"""
    rows, hd, n = q.shape[0], k.shape[2], pos + q.shape[0]
    out, tol = np.zeros((rows, heads, hd)), np.zeros((rows, heads, hd))
    seen = np.arange(n)[None] <= pos + np.arange(rows)[:, None]
    for h in range(heads):
        kh, vh = k[h * len(k) // heads], v[h * len(k) // heads]
        qh = q.reshape(rows, heads, hd)[:, h].astype(np.float64)
        s = np.where(seen, qh @ kh.T * scale, -np.inf)
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ vh
        # a score, times the magnitude of the scale (an error has no sign): q enters as five planes, each leaving 2^-4 of its block's largest magnitude, the accumulators are cut at 2^-23
        # ten times, the scale and the difference to the largest score rounded: 2^-24 of each.  The weights' exponential: 2^-22, and
        # what the exponent's rounding to 2^-24 of itself makes.  A weight's error e is a relative one, in the sum of the weights and in that
        # of the values.  Sums over n rows: chains of n / 64 at 2^-24 and the parts'; weights enter as 24 bits, accumulators cut at 2^-23.
        ds = np.where(seen, abs(scale) * (2.0 ** -20 * (M.block_max(qh) @ np.abs(kh).T) + 2.0 ** -19 * (np.abs(qh) @ np.abs(kh).T)) + 2.0 ** -22 * np.abs(np.where(seen, s, 0)), 0)
        far = np.where(seen & (p > 1e-12), m - s, 0).max(1, keepdims=True)
        e = 2 * ds.max(1, keepdims=True) + 2.0 ** -21 + 2.0 ** -23 * far + 2.0 ** -23 * (n / 32 + 40)
        # Besides, in absolute terms: a weight goes in as fp16 planes of p 2^14, p = 1 for the largest, whose smallest step is 2^-24, and so is off by up to
        # 2^-25 2^-14 = 2^-39 of the largest weight however small it is; the largest weight over the sum is at most 1, and n weights meet
        # n values: 2^-39 sum |v|.  A value goes in as fp16 of v 2^13 / 2^E with 2^E at most a quarter of the largest value: off by up to 2^-25 2^-13 / 4 =
        # 2^-40 of that, weights adding up to 1.
        tol[:, h] = e * (p @ np.abs(vh)) + absolute * (2.0 ** -39 * (seen @ np.abs(vh)) + 2.0 ** -40 * np.abs(vh).max()) + 1e-37
    return out.reshape(rows, -1), tol.reshape(rows, -1)


def case(hip, heads, kv_heads, hd, rows, pos, spread=1.0, extra=37):
    c = M.Cache(hip, pos + rows + extra, kv_heads, hd)
    r = np.random.default_rng(heads + 31 * rows + pos)
    for a in c.host.values():
        a[:] = 255                                        # behind the last row: codes of -6, scales of NaN
    c.fill(*[r.standard_normal((kv_heads, pos + rows, hd)).astype(np.float32) * spread for _ in range(2)])
    return c, (r.standard_normal((rows, heads * hd)) * spread).astype(np.float32)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("rows,pos", [(1, 0), (1, 1), (1, 15), (1, 16), (1, 300), (1, 2999), (3, 5), (5, 1000), (16, 0), (17, 130), (65, 0), (130, 70), (33, 2100)])
def test_attention(hip, heads, kv_heads, hd, rows, pos):
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    got = attend(hip, c.upload(), q, pos, heads, 1 / np.sqrt(hd))
    want, tol = oracle(q, *c.values(pos + rows), pos, heads, float(np.float32(1 / np.sqrt(hd))))
    c.free()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("rows,pos", [(1, 40000), (9, 33333), (400, 517)])
def test_attention_long(hip, rows, pos):
    c, q = case(hip, 8, 2, 128, rows, pos)
    got = attend(hip, c.upload(), q, pos, 8, 1 / np.sqrt(128))
    want, tol = oracle(q, *c.values(pos + rows), pos, 8, float(np.float32(1 / np.sqrt(128))))
    c.free()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("rows,pos", [(1, 500), (40, 300)])
@pytest.mark.parametrize("spread,scale", [(8.0, 1.0), (1e-3, 1.0), (1e15, 1e-31), (3.0, -0.5), (1.0, 0.0)])
def test_attention_scores_far_apart_and_equal(hip, rows, pos, spread, scale):
    """One weight takes all; all are equal; values near the ends of the range; a scale that turns the order round."""
    c, q = case(hip, 8, 2, 128, rows, pos, spread)
    got = attend(hip, c.upload(), q, pos, 8, scale)
    want, tol = oracle(q, *c.values(pos + rows), pos, 8, float(np.float32(scale)))
    c.free()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("hd", [64, 128, 192, 256])
@pytest.mark.parametrize("rows,pos,bad", [(1, 200, 77), (50, 20, 40), (200, 0, 100), (3, 90, 91)])
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_attention_nan_reaches_who_sees_it(hip, hd, rows, pos, bad, which):
    """A NaN in one key's or value's block: the queries that see the row answer NaN (all of it, or the block's values), the others what
    they answered without it, bit for bit."""
    c, q = case(hip, 4, 2, hd, rows, pos)
    clean = attend(hip, c.upload(), q, pos, 4, 0.1).reshape(rows, 4, hd)
    c.host[which][1, bad, 1] = 255
    got = attend(hip, c.upload(), q, pos, 4, 0.1).reshape(rows, 4, hd)
    c.free()
    sees = pos + np.arange(rows) >= bad
    assert np.array_equal(got[:, :2], clean[:, :2]) and np.array_equal(got[~sees], clean[~sees])
    hit = got[sees][:, 2:]
    if which == "ks":
        assert np.isnan(hit).all()
    else:
        assert np.isnan(hit[..., 32:64]).all()
        rest = np.delete(np.arange(hd), np.arange(32, 64))
        assert np.array_equal(hit[..., rest], clean[sees][:, 2:][..., rest])


@pytest.mark.parametrize("hd", [64, 128, 192, 256])
@pytest.mark.parametrize("rows,pos", [(1, 0), (1, 32), (1, 332), (6, 1001), (70, 64)])
def test_attention_hidden_rows_change_nothing(hip, hd, rows, pos):
    """Behind the last row, and so in front of the next head's first: zeros, the largest scales, NaN.  The same bits."""
    outs = []
    for fill in (0, 254, 255):
        c, q = case(hip, 6, 3, hd, rows, pos, extra=1 + pos % 2)
        n = pos + rows
        for a in c.host.values():
            a[:, n:] = fill
        outs.append(attend(hip, c.upload(), q, pos, 6, 0.1))
        c.free()
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


def test_attention_results_do_not_depend_on_the_call(hip):
    for rows, pos in ((1, 3000), (50, 700)):
        c, q = case(hip, 32, 8, 128, rows, pos)
        cache = c.upload()
        first = attend(hip, cache, q, pos, 32, 0.1)
        for _ in range(5):
            assert np.array_equal(first, attend(hip, cache, q, pos, 32, 0.1))
        c.free()


BOTH = [(4, 2, 64, 1, 300), (4, 2, 128, 40, 600), (4, 2, 192, 40, 20), (4, 1, 256, 64, 0), (32, 2, 64, 300, 0), (32, 2, 128, 300, 1500), (32, 2, 128, 700, 0)]      # few columns and many


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
def test_attention_scores_of_any_size(hip, heads, kv_heads, hd, rows, pos):
    """All keys the same, queries from 2^-10 to 2^60 and both signs: all weights are the same, results are means of values.  (Products of the
    same numbers in the same order: the scores differ by nothing.)"""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    r, n = np.random.default_rng(5), pos + rows
    k, v = np.repeat(r.standard_normal((kv_heads, 1, hd)), n, 1).astype(np.float32), r.standard_normal((kv_heads, n, hd)).astype(np.float32)
    c.fill(k, v)
    q = (q * 2.0 ** (-10 + 70 * (np.arange(rows) + r.random(rows))[:, None] / rows)).astype(np.float32)
    got = attend(hip, c.upload(), q, pos, heads, 0.1).reshape(rows, heads, hd)
    _, v = c.values(n)
    c.free()
    count = (pos + np.arange(rows) + 1)[:, None]
    for h in range(heads):
        vh = v[h * kv_heads // heads]
        mean, size = np.cumsum(vh, 0)[pos:] / count, np.cumsum(np.abs(vh), 0)[pos:] / count
        # weights alike to 2^-21 and the sums' rounding, as in the oracle; values and small weights to 2^-39 besides
        tol = (2.0 ** -20 + 2.0 ** -23 * (n / 32 + 40)) * size + 2.0 ** -39 * np.abs(vh).max() + 2.0 ** -39 * count * size
        assert np.all(np.abs(got[:, h] - mean) <= tol), (h, float((np.abs(got[:, h] - mean) / tol).max()))


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
@pytest.mark.parametrize("top", [2.0 ** 9, 2.0 ** 24, 2.0 ** 25, 1.5 * 2 ** 25, -1.5 * 2 ** 25, 2.0 ** 26, -1.5 * 2 ** 26, 2.0 ** 28])
@pytest.mark.parametrize("far", [False, True])
def test_attention_scores_a_step_of_fp32_apart(hip, heads, kv_heads, hd, rows, pos, top, far):
    """Scores that are fp32 numbers, one and two of fp32's steps u apart (1 where they are smaller), the larger ones in later tiles, waves and
    parts: weights are 2^-2u, 2^-u and 1, whatever the largest score is.  far: a value 2^-60 times the others, so that some waves go
    their way through fp32."""
    n, u = pos + rows, max(float(np.spacing(np.float32(abs(top)))), 1.0)
    scale = np.float32(0.6931472)
    assert scale * np.float32(1.44269504) == 1                # scores are in units of log2 e: a whole number's weight is a power of two
    r = np.random.default_rng(17)
    step = np.zeros(n)
    step[n * 6 // 10:], step[n * 9 // 10:] = 1, 2
    k, v = np.zeros((kv_heads, n, hd), np.float32), r.standard_normal((kv_heads, n, hd)).astype(np.float32)
    k[..., 0], k[..., 1], k[..., 32] = np.copysign(4, top), 1, step / 2
    if far:
        v[:, n // 5] *= np.float32(2.0 ** -60)
    q = np.zeros((rows, heads, hd), np.float32)
    q[..., 0], q[..., 1], q[..., 32] = abs(top) / 4, u * (np.arange(rows * heads).reshape(rows, heads) % 4), 2 * u      # neighbouring maxima
    c = M.Cache(hip, n + 5, kv_heads, hd)
    c.fill(k, v)
    got = attend(hip, c.upload(), q.reshape(rows, -1), pos, heads, float(scale)).reshape(rows, heads, hd)
    kd, vd = c.values(n)
    c.free()
    assert np.array_equal(kd, k)
    seen = np.arange(n)[None] <= pos + np.arange(rows)[:, None]
    p = np.where(seen, np.exp2(u * step), 0)
    p /= p.sum(1, keepdims=True)
    for h in range(heads):
        vh = vd[h * kv_heads // heads]
        # weights alike to 2^-21 and the sums' rounding, as in the oracle; small weights and values to 2^-39
        tol = (2.0 ** -20 + 2.0 ** -23 * (n / 32 + 40)) * (p @ np.abs(vh)) + 2.0 ** -39 * (seen @ np.abs(vh)) + 2.0 ** -39 * np.abs(vh).max()
        assert np.all(np.abs(got[:, h] - p @ vh) <= tol), (h, float((np.abs(got[:, h] - p @ vh) / tol).max()))


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
@pytest.mark.parametrize("near", [False, True])
def test_attention_values_of_any_size(hip, heads, kv_heads, hd, rows, pos, near):
    """A row 2^100 times as large as the others, and one 2^-60 times: who does not see the first has what it has without it, and so, but for a
    part in the last binades, has who gives it a weight of 2^-110.  No absolute error: nothing counts beside the values seen, each by its weight."""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    r, n = np.random.default_rng(6), pos + rows
    k, v = r.standard_normal((2, kv_heads, n, hd)).astype(np.float32)
    bad = n - 1 - rows // 3
    v[:, bad] *= np.float32(2.0 ** 100)
    v[:, bad // 2] *= np.float32(2.0 ** -60)
    q = q.reshape(rows, heads, hd)
    q[..., 0], k[..., 0], k[:, bad, 0] = 8, 0, 0 if near else -96
    q = q.reshape(rows, -1)
    c.fill(k, v)
    got = attend(hip, c.upload(), q, pos, heads, 0.1)
    want, tol = oracle(q, *c.values(n), pos, heads, float(np.float32(0.1)), absolute=False)
    c.free()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
@pytest.mark.parametrize("small,large", [(-112, -60), (-118, 0), (-118, 100), (-70, 120)])
def test_attention_values_that_only_later_queries_see(hip, heads, kv_heads, hd, rows, pos, small, large):
    """Values of about 2^small, the last row's of 2^large: the queries in front of it have what the small ones make, in 24 bits down to where
    fp32 has no more, and the last query, who gives the row a weight like the others', has its share of it."""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    r, n = np.random.default_rng(8), pos + rows
    k, v = r.standard_normal((2, kv_heads, n, hd)).astype(np.float32)
    v[:, :-1] *= np.float32(2.0 ** small)
    v[:, -1] *= np.float32(2.0 ** large)
    c.fill(k, v)
    got = attend(hip, c.upload(), q, pos, heads, 0.1)
    want, tol = oracle(q, *c.values(n), pos, heads, float(np.float32(0.1)), absolute=False)
    c.free()
    # besides, a column's parts (8 waves, at most 64 workgroups), their products with their shares and the result are rounded to 2^-149 at the lowest, half a step each
    tol += 80 * 2.0 ** -150 - 1e-37
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
@pytest.mark.parametrize("size", [130, 142, 200, -130, -142])
@pytest.mark.parametrize("far", [False, True])
def test_attention_a_score_that_leaves_fp32(hip, heads, kv_heads, hd, rows, pos, size, far):
    """A key whose score is +-2^|size|, of finite queries: who sees it answers NaN, the others what they answered without it.  far: some waves go their
    way through fp32."""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    r, n = np.random.default_rng(9), pos + rows
    k, v = r.standard_normal((2, kv_heads, n, hd)).astype(np.float32)
    k[..., 32:] = 0
    bad = n - 1 - rows // 3
    if far:
        v[:, n // 5] *= np.float32(2.0 ** -60)
    q = q.reshape(rows, heads, hd)
    q[..., 32:] *= np.float32(2.0 ** 80)                     # against keys of 0
    q[..., 33] = np.float32(1.375 * 2.0 ** 80)               # more than one plane
    c.fill(k, v)
    clean = attend(hip, c.upload(), q.reshape(rows, -1), pos, heads, 1.0).reshape(rows, heads, hd)
    k[0, bad, 33] = np.copysign(np.float32(2.0 ** (abs(size) - 80)), size)
    c.fill(k, v)
    got = attend(hip, c.upload(), q.reshape(rows, -1), pos, heads, 1.0).reshape(rows, heads, hd)
    c.free()
    hit = np.zeros(got.shape, bool)
    hit[pos + np.arange(rows) >= bad, :heads // kv_heads] = True
    assert np.isfinite(clean).all() and np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", BOTH)
def test_attention_nan_beside_values_of_any_size(hip, heads, kv_heads, hd, rows, pos):
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    r, n = np.random.default_rng(7), pos + rows
    k, v = r.standard_normal((2, kv_heads, n, hd)).astype(np.float32)
    v[:, n // 3] *= np.float32(2.0 ** -90)
    bad = n - 1 - rows // 3
    v[0, bad, 33] = np.nan
    c.fill(k, v)
    got = attend(hip, c.upload(), q, pos, heads, 0.1).reshape(rows, heads, hd)
    c.free()
    nan = np.zeros(got.shape, bool)
    nan[pos + np.arange(rows) >= bad, :heads // kv_heads, 32:64] = True
    assert np.array_equal(np.isnan(got), nan)


@pytest.mark.parametrize("rows,heads", [(3, 4), (1100, 16)])
def test_a_cache_past_32_bits(hip, rows, heads):
    """Two heads of 34 million rows, 2.2 GB of codes each: rows at the end of what attention reaches and of the cache; all others are zeros
    and get the weight of a score of 0."""
    kv_heads, hd, max_rows, last = 2, 128, 34_000_000, 1 << 24
    buf = [H.DevBuf(hip.lib, kv_heads * max_rows * n) for n in (hd // 2, hd // 32) * 2]
    for b in buf:
        hip.lib.tts_hip_memset(b.ptr, 0, b.nbytes)
    cache = C.byref(hip.pkg.Kv4(*[b.ptr for b in buf], max_rows, kv_heads, hd))
    r = np.random.default_rng(11)
    x = [(r.standard_normal((rows, kv_heads * hd)) * 4).astype(np.float32) for _ in range(2)]
    dev = [H.DevBuf.from_numpy(hip.lib, a) for a in x]
    back = [H.DevBuf(hip.lib, a.nbytes) for a in x]
    decoded = [M.decode(*M.encode(a)) for a in x]
    for pos in (max_rows - rows, last - rows):
        assert hip.lib.tts_hip_kv4_append(cache, dev[0].ptr, dev[1].ptr, rows, pos, 0) == 0
        assert hip.lib.tts_hip_kv4_read(back[0].ptr, back[1].ptr, cache, rows, pos, 0) == 0
        for b, d in zip(back, decoded):
            assert np.array_equal(b.to_numpy(np.float32, d.shape), d.astype(np.float32))
    q = (r.standard_normal((rows, heads * hd)) * 4).astype(np.float32)
    got = attend(hip, cache, q, last - rows, heads, 1.0).reshape(rows, heads, hd)
    seen = np.arange(rows)[None] <= np.arange(rows)[:, None]
    for h in range(heads):
        kh, vh = (d[:, h * kv_heads // heads * hd:][:, :hd] for d in decoded)
        s = q.reshape(rows, heads, hd)[:, h].astype(np.float64) @ kh.T
        m = np.maximum(np.where(seen, s, 0).max(1, keepdims=True), 0)
        p = np.exp(np.where(seen, s - m, -np.inf))
        p /= p.sum(1, keepdims=True) + (last - rows) * np.exp(-m)
        ds = 2.0 ** -20 * (M.block_max(q.reshape(rows, heads, hd)[:, h].astype(np.float64)) @ np.abs(kh).T) + 2.0 ** -18 * (np.abs(q.reshape(rows, heads, hd)[:, h]) @ np.abs(kh).T) + 2.0 ** -21 * np.abs(s)
        # 2^24 weights of one size are added in 64 parts of 8 waves, 1024 tiles of 32 rows each: chains of 8192 at 2^-24
        e = 2 * np.where(seen, ds, 0).max(1, keepdims=True) + 2.0 ** -11 + 2.0 ** -23 * m
        assert np.all(np.abs(got[:, h] - p @ vh) <= e * (p @ np.abs(vh)) + 2.0 ** -38 * np.abs(vh).sum(0)), h
    for b in buf + dev + back:
        b.free()


def test_a_layer_in_4_bits(hip):
    """A prompt and two decode steps through a layer's attention half and its feed-forward half: norms, projections, rotation, cache,
    attention, residuals, all on the device; against the same in 64 bits on the same 4-bit weights.  The rounding of k and v to
    4 bits turns differences of the last bit into steps where a value lies on a border, so the oracle reads the cache's bytes."""
    lib, D, heads, kvh, hd, F, T, n_dec = hip.lib, 512, 8, 2, 64, 768, 21, 2
    r = np.random.default_rng(3)
    names = {"q": (heads * hd, D), "k": (kvh * hd, D), "v": (kvh * hd, D), "o": (D, heads * hd), "g": (F, D), "u": (F, D), "d": (D, F)}
    w, dev = {}, {}
    for i, (name, (n, k)) in enumerate(names.items()):
        full = H.DevBuf.from_numpy(lib, (r.standard_normal((n, k)) * 0.05).astype(np.float32))
        p = M.panels(k)
        dev[name] = H.DevBuf(lib, n * p * 64), H.DevBuf(lib, n * p * 4)
        assert lib.tts_hip_mx4_quantize(dev[name][0].ptr, dev[name][1].ptr, full.ptr, 0, n, k, 0) == 0
        w[name] = M.decode(dev[name][0].to_numpy(np.uint8, (n, 64 * p)), dev[name][1].to_numpy(np.uint8, (n, 4 * p)))[:, :k]
        full.free()
    gain = [np.abs(r.standard_normal(D)).astype(np.float32) * 0.5 + 0.75 for _ in range(2)]
    dgain = [H.DevBuf.from_numpy(lib, g) for g in gain]
    c = M.Cache(hip, T + n_dec, kvh, hd)
    cache = c.upload()
    lin = lambda y, x, name, m: lib.tts_hip_linear_mx4(y.ptr, x.ptr, dev[name][0].ptr, dev[name][1].ptr, m, names[name][1], names[name][0])  # noqa: E731
    size = {n: H.DevBuf(lib, 4 * T * max(F, D)) for n in "x n q k v a o g u f".split()}
    b = size

    def norm(x, g):
        return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * g

    def turn(x, pos, h):
        x = x.reshape(len(x), h, hd // 2, 2)
        f = 1.0 / 1e6 ** (2 * np.arange(hd // 2) / hd)
        a = (pos + np.arange(len(x)))[:, None, None] * f
        return np.stack((x[..., 0] * np.cos(a) - x[..., 1] * np.sin(a), x[..., 0] * np.sin(a) + x[..., 1] * np.cos(a)), -1).reshape(len(x), -1)

    freqs = H.DevBuf(lib, 4 * T * hd)
    for pos, m in ((0, T), (T, 1), (T + 1, 1)):
        x = r.standard_normal((m, D)).astype(np.float32)
        lib.tts_hip_to_device(b["x"].ptr, x.ctypes.data, x.nbytes)
        lib.tts_hip_rms_norm(b["n"].ptr, b["x"].ptr, dgain[0].ptr, m, D, 1e-5)
        lib.tts_hip_compute_rope_freqs(freqs.ptr, pos, m, hd, 1e6)
        status = [lin(b[n], b["n"], n, m) for n in "qkv"]
        lib.tts_hip_apply_rope(b["q"].ptr, freqs.ptr, m, heads, hd)
        lib.tts_hip_apply_rope(b["k"].ptr, freqs.ptr, m, kvh, hd)
        status.append(lib.tts_hip_kv4_append(cache, b["k"].ptr, b["v"].ptr, m, pos, 0))
        status.append(lib.tts_hip_kv4_attention(b["a"].ptr, b["q"].ptr, cache, m, pos, heads, 0.125))
        status.append(lin(b["o"], b["a"], "o", m))
        lib.tts_hip_add_inplace(b["x"].ptr, b["o"].ptr, m * D)
        lib.tts_hip_rms_norm(b["n"].ptr, b["x"].ptr, dgain[1].ptr, m, D, 1e-5)
        status += [lin(b["g"], b["n"], "g", m), lin(b["u"], b["n"], "u", m)]
        lib.tts_hip_silu_mul(b["g"].ptr, b["u"].ptr, m * F)
        status.append(lin(b["f"], b["g"], "d", m))
        lib.tts_hip_add_inplace(b["x"].ptr, b["f"].ptr, m * D)
        assert not any(status)
        got = b["x"].to_numpy(np.float32, (m, D))
        x = x.astype(np.float64)
        y = norm(x, gain[0])
        k = turn(y @ w["k"].T, pos, kvh)
        held = c.download()
        c.host = held
        kv = c.values(pos + m)
        # what was appended is what the projections gave, to a step of 4 bits (a half, or a whole one on a border)
        for have, new in zip(kv, (k, y @ w["v"].T)):
            new = new.reshape(m, kvh, hd).transpose(1, 0, 2)
            assert np.all(np.abs(have[:, pos:pos + m] - new) <= M.block_max(new) / 4 + 1e-5)
        a, _ = oracle(turn(y @ w["q"].T, pos, heads), *kv, pos, heads, 0.125)
        x = x + a @ w["o"].T
        y = norm(x, gain[1])
        g = y @ w["g"].T
        x = x + (g / (1 + np.exp(-g)) * (y @ w["u"].T)) @ w["d"].T
        assert np.abs(got - x).max() <= 1e-4 * np.sqrt((x * x).mean())      # fp32 sums through eight launches of a few 2^-20 each, five times over
    hip.check()
    c.free()
