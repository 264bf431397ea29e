"""What the operators over a paged cache promise of a result's bits, range and rounding, at the places where a kernel that is right on ordinary numbers can
fall short: weights of bf16 calls, scores that only a neighbour in the same wave sees, values near the end of the range, positions near 2^31, shared pages."""
from fractions import Fraction
import math

import numpy as np
import pytest

import hipsupport as H
import pagedsupport as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    h = H.Hip(kv_max=8)
    yield h
    h.close()


def normal(rng, shape, bf16):
    x = rng.standard_normal(shape, np.float32)
    return P.value16(P.bits16(x)) if bf16 else x


MANY = [((32, 8, 128), "1300@0 3@50", 16, 0), ((32, 8, 128), "130@500 1@700 64@64 0@9 900@450", 64, 0), ((32, 8, 128), "2500@1000 1@3000 2@100", 32, 1200),
        ((16, 16, 64), "333@3700 900@1100 1@40 700@0", 256, 0), ((14, 2, 64), "2000@800", 1024, 0), ((12, 4, 256), "1700@30 1@5 40@900", 16, 0)]


@pytest.mark.parametrize("layout,batch,page,window", MANY)
def test_a_bf16_result_is_rounded_and_little_else(hip, layout, batch, page, window):
    """Queries of many columns in bf16: weights enter to 16 bits.  A value's error is its own rounding, of at most half a step h = 2^-8 of the power of two
    below it and uniform within, so that over many values the squares add up to h^2 / 3 each.  Weights (2^-17 of each, independent: 4e-6 of the norm), scores
    (1e-6) and sums are far below 2 % of that; a weight rounded to bf16 (2^-8 / sqrt 3 times 0.74) would be another 80 % beside it."""
    c = P.Cache(hip, batch, page, *layout, window=window, seed=len(batch))
    c.fill()
    c.upload()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), 1)
    scale, keep = 1 / math.sqrt(layout[2]), c.some()
    assert any(P.is_many(c, i, 1) for i in range(len(c.rows)))
    got = P.attention(c, q, 1, scale)[keep].astype(np.float64)
    want, size, most = c.attend(q, scale, keep)
    want, size = want[keep], size[keep]
    off = got - want
    half = 2.0 ** (np.floor(np.log2(np.abs(want))) - 8)
    rel = 2 * (3 * c.hd / 8 + 3) * 2.0 ** -23 * most + 64 * 2.0 ** -23 + 2.0 ** -16
    # the next power of two is nearer than rel to some results: twice the half step there
    assert (np.abs(off) <= 2.0 ** -8 * (np.abs(want) + rel * size) + rel * size).all()
    assert math.sqrt((off ** 2).sum()) <= 1.02 * math.sqrt((half ** 2).sum() / 3)
    c.free()


# layout, batch, page: few columns in parts, few with a wave's rows behind one another, 32 at a time, many in one part and in several, and both in one launch
NEIGHBOURS = [((32, 8, 128), "3@700", 16), ((8, 1, 128), "7@1500", 32), ((32, 8, 128), " ".join(["4@900"] * 40), 16), ((24, 3, 64), " ".join(["9@700"] * 50), 64),
              ((6, 2, 192), " ".join(["5@600"] * 70), 16), ((16, 2, 256), " ".join(["3@800"] * 60), 16), ((32, 8, 128), "300@700 5@5", 64),
              ((16, 16, 64), "512@1500", 16), ((32, 8, 128), "1300@0", 16), ((32, 8, 128), "90@2500 600@1500", 64), ((32, 8, 128), "600@1500 1@2000 2@777", 64),
              ((14, 2, 64), "2000@800", 1024), ((12, 4, 256), "1700@30", 16)]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page", NEIGHBOURS)
def test_keys_that_a_query_does_not_see_leave_its_bits(hip, layout, batch, page, bf16):
    """Queries share waves and tiles with later ones of their sequence.  Keys that only those see - scores far above the others', infinities, NaN - and values
    there change no bit of what came before."""
    c = P.Cache(hip, batch, page, *layout, seed=len(batch))
    c.fill()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16)
    scale, results = 2 / math.sqrt(layout[2]), []
    first = [max(1, (r - 1) // 2 | 1) if r > 1 else r for r in c.rows]                  # queries from this one on see what changes
    before = np.concatenate([np.arange(r) < f for r, f in zip(c.rows, first)])
    for what in ("as it is", "far", "infinite", "NaN"):
        for pool, odd in ((c.k, 0x7F80), (c.v, 0xFF80)):
            for i, t in enumerate(c.tables):
                p = np.arange(c.past[i] + first[i], c.past[i] + c.rows[i])
                x = c.rng.standard_normal((len(p), layout[1], layout[2]), np.float32) * 30
                pool[t[p // page], :, p % page] = P.bits16(x) if what == "far" else odd if what == "infinite" else P.NAN16 if what == "NaN" else P.bits16(x / 30)
        c.upload()
        results.append(P.attention(c, q, bf16, scale))
        for d in c.dev.values():
            d.free()
    c.dev = {}
    assert np.isfinite(results[0]).all() and before.any()
    for other in results[1:]:
        assert np.array_equal(other[before], results[0][before])
        assert len(before) == before.sum() or not np.array_equal(other[~before], results[0][~before])
    c.free()


RANGE = NEIGHBOURS + [((32, 8, 128), "1@0 1@1999 1@40", 16), ((8, 1, 128), "1@20000", 256), ((4, 4, 192), "37@300", 16), ((8, 1, 128), "5300@100", 32),
                      ((32, 8, 128), "1@9000 1500@100", 16)]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("alike", [True, False])
@pytest.mark.parametrize("layout,batch,page", RANGE)
def test_a_mean_is_finite_where_its_values_are(hip, layout, batch, page, alike, bf16):
    """Values up to the largest that bf16 has, over as many rows as there are: what a query answers is a mean of them, however large their sum; from the queries
    on that see the large ones, and without a bit's change for the others in their waves.  Weights are then relative to up to 2^40 times the largest one, and
    the difference to it is off by 2^-19 (of a number below 64, half a step) times log 2: 2^-19 beside what pagedsupport.check counts."""
    c = P.Cache(hip, batch, page, *layout, seed=len(batch))
    c.fill()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16) * np.float32(0 if alike else 1)
    scale, keep = 1 / math.sqrt(layout[2]), c.some()
    c.upload()
    ordinary = P.attention(c, q, bf16, scale)
    for d in c.dev.values():
        d.free()
    first = [r // 3 for r in c.rows]                             # queries from this one on see large values, in the first half of their heads
    for i, t in enumerate(c.tables):
        p = np.arange(c.past[i] + first[i] if c.rows[i] > 1 else 0, c.past[i] + c.rows[i])
        x = c.rng.standard_normal((len(p), layout[1], layout[2] // 2), np.float32)
        x = 3.3e38 * np.clip(1 - 0.01 * np.abs(x), 0.9, 1) if alike else np.clip(x, -1.65, 1.65) * 2e38
        c.v[t[p // page], :, p % page, :layout[2] // 2] = P.bits16(x)
    c.upload()
    got = P.attention(c, q, bf16, scale)
    assert np.isfinite(got).all()
    want, size, most = c.attend(q, scale, keep)
    rel = 2 * (3 * c.hd / 8 + 3) * 2.0 ** -23 * most + 64 * 2.0 ** -23 + 2.0 ** -19 + (2.0 ** -16 if bf16 else 0)
    off, tol = np.abs(got - want)[keep], (rel * size + (2.0 ** -8 * (np.abs(want) + rel * size) if bf16 else 0))[keep]
    assert (off <= tol).all(), float((off / tol).max())
    before = np.concatenate([np.arange(r) < (f if r > 1 else 0) for r, f in zip(c.rows, first)])
    assert np.array_equal(got[before], ordinary[before])
    c.free()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("most", [0.16, 40.0, 5e5])
def test_angles_are_those_of_the_turns_given(hip, most, half, norm):
    """Position times turn in whole numbers of any length, of which the fraction is an angle: at the ends of int, and for turns of many whole ones a position.
    (A product rounded to 64 bits is off by up to 2^-25 of a turn at 2^31 times 0.16, by 1/8 at 2^31 times 5e5.)"""
    rows, heads, hd = 12, 3, 64
    rng = np.random.default_rng(11)
    pos = np.array([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 2 ** 30 + 12345, -2 ** 29 - 1, 2 ** 28 + 1, 10 ** 6 + 7, 4097, 1, 0, -1, -77], np.int32)
    t = most * rng.random(hd // 2)
    left = np.array([[float((Fraction(int(p)) * Fraction(float(f)) + Fraction(1, 2)) % 1 - Fraction(1, 2)) for f in t] for p in pos])
    x = rng.standard_normal((rows, heads, hd), np.float32)
    gain = 1 + 0.1 * rng.standard_normal(hd).astype(np.float32)
    dx, do, dt, dg, dp = (P.Dev(hip.lib, a) for a in (x, np.zeros_like(x), t, gain, pos))
    assert hip.lib.tts_hip_rotary(do.ptr, dx.ptr, 0, rows, heads, hd, 0, 0, dp.ptr, P.how(hip, dt.ptr, hd, half, dg.ptr if norm else None)) == 0
    y = x.astype(np.float64)
    if norm:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(1e-5))) * gain
    a, b = (y[..., :hd // 2], y[..., hd // 2:]) if half else (y[..., 0::2], y[..., 1::2])
    c, s = np.cos(2 * math.pi * left)[:, None], np.sin(2 * math.pi * left)[:, None]
    got = do.get().astype(np.float64)
    u, v = (got[..., :hd // 2], got[..., hd // 2:]) if half else (got[..., 0::2], got[..., 1::2])
    # cosine and sine to 2 ulp of 1, the rest of the angle to 2^-24 of a step, two products and a sum: 2^-23 each; a norm adds its sum and five operations
    tol = (8 * 2.0 ** -23 + ((hd / 8 + 8) * 2.0 ** -24 if norm else 0)) * (np.abs(a) + np.abs(b))
    assert (np.abs(u - (a * c - b * s)) <= tol).all() and (np.abs(v - (a * s + b * c)) <= tol).all()
    for d in (dx, do, dt, dg, dp):
        d.free()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page,common,window", [
    ((32, 8, 128), " ".join(["1@700"] * 64), 16, 30, 0), ((32, 8, 128), "1@2000 1@640 37@900 1@641", 32, 20, 0), ((16, 16, 64), "300@1500 1@5000 9@1500", 64, 23, 0),
    ((32, 8, 128), "600@1500 1@1500 2@1600 1@9000", 16, 93, 1000), ((12, 4, 256), "3@300 1@700", 256, 1, 0), ((32, 8, 128), "1@9000 1@9000 1@9000", 16, 562, 0)])
def test_sequences_that_share_pages(hip, layout, batch, page, common, window, bf16):
    """A common beginning of `common` pages that all read, steps and prompts, and what follows it of each."""
    c = P.Cache(hip, batch, page, *layout, window=window, seed=len(batch))
    c.tables = [np.concatenate((c.tables[0][:common], t[common:])) for t in c.tables]
    assert all(p >= common * page for p in c.past) and c.batch.set(c.past, c.rows, c.tables) == 0
    c.fill()
    c.upload()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16)
    scale, keep = 1 / math.sqrt(layout[2]), c.some()
    got = P.attention(c, q, bf16, scale)
    assert np.isfinite(got).all() and P.check(c, got, *c.attend(q, scale, keep), bf16, keep)
    x = normal(np.random.default_rng(8), (sum(c.rows), layout[1], layout[2]), bf16)
    d = P.Dev(hip.lib, P.bits16(x) if bf16 else x)
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, d.ptr, d.ptr, bf16, 0, None) == 0
    pos = c.positions()
    pages = np.concatenate([t[np.arange(p, p + r) // page] for t, r, p in zip(c.tables, c.rows, c.past)])
    for pool, new in zip((c.k, c.v), c.download()):
        pool[pages, :, pos % page] = P.bits16(x)
        assert np.array_equal(new, pool)                                                # the common pages are as they were
    d.free()
    c.free()
