"""Several sequences over a paged cache through the C ABI: rotary positions, keys and values into pages, attention, against numpy in 64 bits
(pagedsupport.py), and a layer as a program runs it.  Every row of a pool that no sequence has holds NaN."""
import ctypes as C
import math

import numpy as np
import pytest

import hipsupport as H
import pagedsupport as P

pytestmark = pytest.mark.gpu
LAYOUTS = [(32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 256), (14, 2, 64), (6, 2, 192), (20, 1, 64)]


@pytest.fixture(scope="module")
def hip():
    h = H.Hip(kv_max=8)
    yield h
    h.close()


def normal(rng, shape, bf16):
    x = rng.standard_normal(shape, np.float32)
    return P.value16(P.bits16(x)) if bf16 else x


# ---- rotary positions --------------------------------------------------------------------------

@pytest.mark.parametrize("rot,theta,factor,original,low,high",
                         [(128, 1e6, 1.0, 0, 1, 32), (64, 1e4, 8.0, 8192, 1, 32), (2, 5e5, 4.0, 0, 1, 2), (512, 1e6, 32.0, 131072, 0.5, 64),
                          (26, 10.0, 0.5, 100, -3, 3)])
def test_turns(hip, rot, theta, factor, original, low, high):
    d = P.Dev(hip.lib, np.zeros(rot // 2), behind=64)
    assert hip.lib.tts_hip_rotary_turns(d.ptr, rot, theta, factor, original, low, high) == 0
    np.testing.assert_allclose(d.get(), P.turns(rot, theta, factor, original, low, high), rtol=1e-12)
    d.free()


ROTARY = [  # rows, heads, head_dim, rot, half, norm, gaps (out, x), shift (values from a multiple of 16 bytes)
    (1, 32, 128, 128, 0, False, (0, 0), 0), (37, 32, 128, 128, 1, True, (0, 2048), 0), (3, 6, 128, 64, 0, True, (4, 8), 0), (5, 3, 64, 32, 1, False, (0, 0), 0),
    (2, 5, 192, 192, 1, True, (0, 0), 0), (9, 7, 256, 128, 0, True, (0, 0), 0), (4, 2, 512, 512, 1, True, (0, 0), 0), (6, 3, 96, 52, 1, True, (0, 0), 0),
    (6, 3, 96, 52, 0, False, (0, 0), 0), (3, 1, 2, 2, 1, True, (0, 0), 0), (3, 4, 10, 6, 1, False, (1, 3), 1), (70, 5, 80, 80, 1, True, (0, 0), 1),
    (4, 9, 128, 0, 0, True, (0, 0), 0), (300, 64, 128, 128, 1, True, (0, 0), 0), (1100, 33, 64, 64, 0, False, (64, 0), 0),
]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("rows,heads,hd,rot,half,norm,gaps,shift", ROTARY)
def test_rotary(hip, rows, heads, hd, rot, half, norm, gaps, shift, bf16):
    rng = np.random.default_rng(rows + hd)
    size, width = (2 if bf16 else 4), heads * hd
    x = normal(rng, (rows, heads, hd), bf16) * np.float32(1 if bf16 else 3)
    pos = rng.integers(0, 1 << 20, rows).astype(np.int32)
    pos[0] = 0
    if rows > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -5
    gain = 1 + 0.1 * rng.standard_normal(hd).astype(np.float32)
    t = P.turns(rot, 1e6) if rot else np.zeros(0)
    wide = np.zeros((rows, width + gaps[1]), np.uint16 if bf16 else np.float32)
    wide[:, :width] = P.bits16(x).reshape(rows, -1) if bf16 else x.reshape(rows, -1)
    raw = np.zeros(wide.size + shift, wide.dtype)
    raw[shift:] = wide.ravel()
    old = np.full(rows * (width + gaps[0]) + shift, 77, wide.dtype)
    dx, do, dt = P.Dev(hip.lib, raw), P.Dev(hip.lib, old, behind=256), P.Dev(hip.lib, np.concatenate((t, [np.nan])))
    dg, dp = P.Dev(hip.lib, gain), P.Dev(hip.lib, pos)
    how = P.how(hip, dt.ptr if rot else None, rot, half, dg.ptr if norm else None, 1e-5, 1.25)
    args = (bf16, rows, heads, hd)
    assert hip.lib.tts_hip_rotary(do.ptr + shift * size, dx.ptr + shift * size, *args, width + gaps[0] if gaps[0] else 0, width + gaps[1] if gaps[1] else 0,
                                  dp.ptr if rot else None, how) == 0, hip.lib.tts_hip_last_error()
    out = do.get()
    assert (out[:shift] == 77).all()
    out = out[shift:].reshape(rows, -1)
    assert (out[:, width:] == 77).all()                                                             # the room between rows
    got = (P.value16(out[:, :width]) if bf16 else out[:, :width]).reshape(x.shape).astype(np.float64)
    want, both = P.turned(x, pos, t, half, gain if norm else None, 1e-5, 1.25)
    # cosine and sine to 2 ulp of 1 and the rest of the angle to 2^-24 of a step, two products and a sum, times the magnitude: 2^-23 each; a norm adds the sum of
    # head_dim / 8 squares and five operations
    rel = 8 * 2.0 ** -23 + ((hd / 8 + 8) * 2.0 ** -24 if norm else 0)
    tol = rel * both + (2.0 ** -8 * (np.abs(want) + rel * both) if bf16 else 0)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / np.maximum(tol, 1e-300)).max())
    if not norm:
        assert np.array_equal(got[..., rot:], x[..., rot:])
    if gaps == (0, 0):                                                                              # in place
        assert hip.lib.tts_hip_rotary(dx.ptr + shift * size, dx.ptr + shift * size, *args, 0, 0, dp.ptr if rot else None, how) == 0
        assert np.array_equal(dx.get()[shift:], out.ravel())
    for d in (dx, do, dt, dg, dp):
        d.free()


def test_rotary_agrees_with_apply_rope(hip):
    """What the library's table turns (whole heads of pairs side by side), this turns alike."""
    rows, heads, hd = 40, 4, 128
    x = np.random.default_rng(1).standard_normal((rows, heads, hd)).astype(np.float32)
    a, b, table = P.Dev(hip.lib, x), P.Dev(hip.lib, x), P.Dev(hip.lib, np.zeros((rows, hd), np.float32))
    t, pos = P.Dev(hip.lib, np.zeros(hd // 2)), P.Dev(hip.lib, np.arange(7, 7 + rows, dtype=np.int32))
    hip.lib.tts_hip_compute_rope_freqs(table.ptr, 7, rows, hd, 1e6)
    hip.lib.tts_hip_apply_rope(a.ptr, table.ptr, rows, heads, hd)
    assert hip.lib.tts_hip_rotary_turns(t.ptr, hd, 1e6, 1.0, 0, 1, 32) == 0
    assert hip.lib.tts_hip_rotary(b.ptr, b.ptr, 0, rows, heads, hd, 0, 0, pos.ptr, P.how(hip, t.ptr, hd, 0)) == 0
    # the table's angles are products in fp32 of up to 46: off by 46 2^-23 with their frequency's rounding
    np.testing.assert_allclose(b.get(), a.get(), rtol=0, atol=float(np.abs(x).max()) * 2 * (46 * 2.0 ** -23 + 8 * 2.0 ** -23))
    for d in (a, b, table, t, pos):
        d.free()


@pytest.mark.parametrize("width", [128, 26])                      # rows on four values, and not
def test_what_does_not_turn_is_passed_on(hip, width):
    """Every bf16 there is, and fp32 of every exponent, through a call that turns nothing, and as values into pages: the same bits, a NaN as a NaN."""
    every = np.arange(65536, dtype=np.uint32)
    for bits, bf16 in ((every.astype(np.uint16), 1), (every << 16 | every[::-1] ^ 0x5A5A, 0)):
        bits = bits[:len(bits) // (2 * width) * 2 * width]
        dx, do = P.Dev(hip.lib, bits), P.Dev(hip.lib, np.zeros_like(bits))
        assert hip.lib.tts_hip_rotary(do.ptr, dx.ptr, bf16, len(bits) // (2 * width), 2, width, 0, 0, None, P.how(hip, None, 0, 0)) == 0
        value = lambda b: P.value16(b) if bf16 else b.view(np.float32)
        out, nan = do.get(), np.isnan(value(bits))
        assert np.array_equal(out[~nan], bits[~nan]) and np.isnan(value(out)[nan]).all() and nan.any()
        for d in (dx, do):
            d.free()
    if width != 128:
        return
    c = P.Cache(hip, "256@0", 16, 8, 2, 128)
    c.upload()
    bits = every.astype(np.uint16).reshape(256, 2, 128)
    dx = P.Dev(hip.lib, bits)
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, dx.ptr, dx.ptr, 1, 0, None) == 0
    pos = np.arange(256)
    for pool in c.download():
        out, nan = pool[c.tables[0][pos // 16], :, pos % 16], np.isnan(P.value16(bits))
        assert np.array_equal(out[~nan], bits[~nan]) and np.isnan(P.value16(np.ascontiguousarray(out))[nan]).all()
    dx.free()
    c.free()


# ---- keys and values into pages ----------------------------------------------------------------

@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page,rot,half,norm,gap", [
    ((32, 8, 128), "1@301", 16, 128, 0, False, 0), ((32, 8, 128), "37@5 1@16 0@3 1@15 20@0", 16, 128, 1, True, 4096), ((16, 16, 64), "300@40", 64, 32, 0, True, 0),
    ((6, 2, 192), "33@31 1@0", 32, 190, 1, False, 3), ((12, 4, 256), "5@250 100@0", 256, 256, 1, True, 8), ((14, 2, 64), "17@100", 1024, None, 0, False, 0),
    ((32, 8, 128), "700@9 400@0", 16, 128, 0, True, 0)])
def test_append(hip, layout, batch, page, rot, half, norm, gap, bf16):
    heads, kv, hd = layout
    c = P.Cache(hip, batch, page, heads, kv, hd, seed=3)
    c.fill("past")
    c.upload()
    rows, width, rng = sum(c.rows), kv * hd, np.random.default_rng(5)
    k, v = normal(rng, (rows, kv, hd), bf16), normal(rng, (rows, kv, hd), bf16)
    gain = 1 + 0.1 * rng.standard_normal(hd).astype(np.float32)
    wide = [np.zeros((rows, width + gap), np.uint16 if bf16 else np.float32) for _ in "kv"]
    for w, x in zip(wide, (k, v)):
        w[:, :width] = (P.bits16(x) if bf16 else x).reshape(rows, -1)
    t = P.turns(rot, 1e6) if rot else np.zeros(0)
    dk, dv, dt, dg = (P.Dev(hip.lib, a) for a in (*wide, t, gain))
    how = None if rot is None else P.how(hip, dt.ptr, rot, half, dg.ptr if norm else None)
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, dk.ptr, dv.ptr, bf16, width + gap if gap else 0,
                                        how) == 0, hip.lib.tts_hip_last_error()
    got_k, got_v = c.download()
    pos = c.positions()
    pages = np.concatenate([c.tables[i][np.arange(p, p + r) // page] for i, (r, p) in enumerate(zip(c.rows, c.past))])
    want_k, want_v = c.k.copy(), c.v.copy()
    want_v[pages, :, pos % page] = P.bits16(v)
    assert np.array_equal(got_v, want_v)                                                            # the other rows too
    new = P.value16(np.ascontiguousarray(got_k[pages, :, pos % page])).astype(np.float64)
    if rot is None:
        assert np.array_equal(new, P.value16(P.bits16(k)))
    else:
        want, both = P.turned(k, pos, t, half, gain if norm else None, 1e-5)
        rel = 8 * 2.0 ** -23 + ((hd / 8 + 8) * 2.0 ** -24 if norm else 0)
        assert (np.abs(new - want) <= rel * both + 2.0 ** -8 * (np.abs(want) + rel * both)).all()
    got_k[pages, :, pos % page] = want_k[pages, :, pos % page]
    assert np.array_equal(got_k, want_k)
    for d in (dk, dv, dt, dg):
        d.free()
    c.free()


# ---- attention ---------------------------------------------------------------------------------

BATCHES = ["1@0", "1@15 1@16 1@17 1@31 1@32", "1@1999", "5@0", "37@300 1@31 0@40 17@5", "300@0", "130@500 1@700 64@64", "1@9000 3@5000", "2@62"]


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("batch,page,window", [(b, (16, 64, 32, 256)[i % 4], (0, 0, 333, 0, 20, 100, 0, 0, 1)[i]) for i, b in enumerate(BATCHES)])
def test_attention(hip, batch, page, window, layout, bf16):
    c = P.Cache(hip, batch, page, *layout, window=window, seed=len(batch))
    c.fill()
    c.upload()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16)
    scale = 1 / math.sqrt(layout[2])
    got = P.attention(c, q, bf16, scale, q_gap=64)
    assert P.check(c, got, *c.attend(q, scale), bf16)
    again = P.attention(c, q, bf16, scale)
    assert np.array_equal(got, again)                                                               # the same bits, whatever came first
    c.free()


MANY = [  # layout, batch, page, window: enough for the kernel for many columns
    ((32, 8, 128), "1300@0 3@50", 16, 0), ((32, 8, 128), "130@500 1@700 64@64 0@9 900@450", 64, 0), ((32, 8, 128), "7000@0", 16, 90),
    ((32, 8, 128), "37@9000 100@4000", 32, 0), ((16, 16, 64), "333@3700 900@1100 1@40 700@0", 256, 0), ((16, 16, 64), "65@36000 300@2000", 16, 0),
    ((8, 1, 128), "300@9000", 16, 0), ((8, 1, 128), "5300@100 17@800", 32, 500), ((8, 1, 128), "10000@33", 64, 260), ((14, 2, 64), "2000@800", 1024, 0),
    ((20, 1, 64), "1500@733 9@9", 16, 0), ((12, 4, 256), "1700@30 1@5 40@900", 16, 0), ((12, 4, 256), "3@70 600@3000 1300@0", 256, 1700),
    ((8, 1, 256), "100@20000", 64, 0)]
BOTH = [  # and sequences of few columns, in the same launch; more of their rows than the caches hold, or not
    ((32, 8, 128), "1300@0 1@9000 2@300 1@0 3@700", 16, 0), ((32, 8, 128), "600@1500 1@2000 1@11 2@777", 64, 0),
    ((32, 8, 128), "4@9000 2500@1000 1@3000 2@100", 32, 1200), ((16, 16, 64), "900@3000 16@30 9@500 1@0 1@2000", 256, 0),
    ((16, 16, 64), "1@9000 900@3000 3@5000 600@10", 16, 0), ((8, 1, 128), "1@70 1@5000 1@60 1500@3000 2@900", 64, 0)]
WIDE = [  # enough for 32 columns at a time
    ((32, 8, 128), "37@5100 1@300", 16, 0), ((32, 8, 128), "300@700 5@5 0@1", 64, 650), ((32, 8, 128), "90@1111 7@2000", 32, 1000),
    ((16, 16, 64), "512@1500", 16, 0), ((20, 1, 64), "100@4000 2@9000", 256, 0), ((8, 1, 128), "70@9999", 16, 0)]


def large(hip, layout, batch, page, window, bf16, scale=None, size=1.0):
    c = P.Cache(hip, batch, page, *layout, window=window, seed=len(batch))
    c.fill(size=size)
    c.upload()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16)
    scale = scale or 1 / math.sqrt(layout[2])
    keep = c.some()
    got = P.attention(c, q, bf16, scale, q_gap=8)
    assert np.isfinite(got).all()
    assert P.check(c, got, *c.attend(q, scale, keep), bf16, keep)
    assert np.array_equal(got, P.attention(c, q, bf16, scale))
    many = any(P.is_many(c, i, bf16) for i in range(len(c.rows)))
    c.free()
    return many


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page,window", MANY + BOTH)
def test_attention_of_many_columns(hip, layout, batch, page, window, bf16):
    assert large(hip, layout, batch, page, window, bf16) == (layout[2] < 256 or bf16)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page,window", WIDE)
def test_attention_of_32_columns_at_a_time(hip, layout, batch, page, window, bf16):
    assert not large(hip, layout, batch, page, window, bf16)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,batch,page,window", [((4096, 1, 64), "1@40 2@9", 16, 0), ((1, 1, 256), "300@5 1@2", 1 << 20, 0), ((100, 1, 128), "3@100", 64, 17),
                                                      ((7, 7, 192), "20@0", 16, 0)])
def test_attention_of_other_layouts(hip, layout, batch, page, window, bf16):
    test_attention(hip, batch, page, window, layout, bf16)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout,n,apart,window", [((24, 3, 64), 200, 1, 0), ((8, 2, 128), 300, 11, 2000)])
def test_attention_of_many_sequences(hip, layout, n, apart, window, bf16):
    test_attention(hip, " ".join(f"1@{apart * i}" for i in range(n)), 16, window, layout, bf16)


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("layout", [(8, 2, 128), (6, 2, 192), (16, 2, 64), (8, 2, 256)])
@pytest.mark.parametrize("batch,window", [("40@100", 0), ("9@7", 0), ("40@100 1@200", 30), ("300@10", 40), ("200@3000", 0), ("2000@800", 0), ("7500@10", 300),
                                          ("3700@0 1@500", 600), ("25000@0", 100), ("2000@800 1@500 2@40 1@0", 0)])
def test_what_a_query_does_not_see_changes_nothing(hip, batch, window, layout, bf16):
    """Infinities and NaN in keys and values: who sees a key's NaN answers NaN, who sees a value's in that value; nobody else notices.  Who sees a key's
    infinity answers NaN where its score is +infinity or no number, and may where it is -infinity, a weight of 0."""
    c = P.Cache(hip, batch, 16, *layout, window=window, seed=1)
    c.fill()
    rows, past = c.rows[0], c.past[0]
    at = lambda p: (c.tables[0][p // 16], p % 16)
    seen = past + rows // 2
    for p, h, d, what in ((seen, 0, 5, 0x7F80), (seen + 1, 0, 6, 0xFF80), (past + rows - 1, 1, 7, 0x7FC0), (past + 1, 1, 9, 0x7F80)):
        page, r = at(p)
        c.v[page, h, r, d] = what
    page, r = at(past + rows - 3)
    c.k[page, 1, r, 3] = 0x7FC0
    if window:
        page, r = at(past + rows - window - 2)
        c.k[page, 0, r, 3] = 0x7F80
        c.v[page, 0, r, 11] = 0x7FC0
    c.upload()
    q = normal(np.random.default_rng(7), (sum(c.rows), layout[0], layout[2]), bf16)
    scale = 1 / math.sqrt(layout[2])
    got = P.attention(c, q, bf16, scale)
    keep = c.some()
    keep[rows // 2 - 5:rows // 2 + 45] = True
    keep[:60] = keep[max(0, rows - window - 10):rows - window + 40] = keep[rows - 20:rows] = True
    want, size, most = c.attend(q, scale, keep)
    got, want, size = (np.where(keep[:, None, None], x, 0) for x in (got, want, size))
    assert np.isnan(want).any() and not np.isnan(want).all()
    inf = np.isinf(got)
    assert not (inf & ~np.isnan(want)).any()
    if window:
        age = np.arange(past, past + rows) - (past + rows - window - 2)
        sees = np.zeros(want.shape, bool)
        sees[:rows, :layout[0] // layout[1]] = ((age >= 0) & (age < window))[:, None, None]
        assert sees.any() and not sees.all()
        want[sees & np.isnan(got)] = np.nan
    assert P.check(c, np.where(inf, np.nan, got), want, size, most, bf16, keep)
    c.free()


@pytest.mark.parametrize("bf16", [0, 1])
@pytest.mark.parametrize("batch", ["1@700", "100@300", "300@1500", "1500@1000"])
def test_scores_far_apart(hip, batch, bf16):
    """Scores of hundreds: a weight's error is that of its score, and the largest takes all."""
    c = P.Cache(hip, batch, 16, 8, 2, 128, seed=2)
    c.fill(size=6.0)
    c.upload()
    q = normal(np.random.default_rng(8), (sum(c.rows), 8, 128), bf16) * np.float32(8)
    got = P.attention(c, q, bf16, 0.0883883)
    want, size, most = c.attend(q, 0.0883883)
    assert np.isfinite(got).all()
    score = (3 * 128 / 8 + 3) * 2.0 ** -23 * most
    assert (np.abs(got - want) <= (2 * score + 2.0 ** -17 + (2.0 ** -8 if bf16 else 0)) * size * 1.01 + (2.0 ** -8 * np.abs(want) if bf16 else 0)).all()
    c.free()


def test_pages_behind_4_gib(hip):
    """Pools of 9 GB each: rows whose offsets in values and in bytes pass 32 bits."""
    page, kv, hd = 64, 8, 128
    c = P.Cache(hip, "1@130 70@0", page, 32, kv, hd, seed=4, spare=0)
    c.fill()
    one = kv * page * hd * 2
    n_pages = (9 << 30) // one
    c.batch.free()
    c.batch = P.PagedBatch(n_pages, page, 32, kv, hd, max_seqs=2, max_rows=80, max_table=8)
    far = [n_pages - 1 - t for t in c.tables]
    assert c.batch.set(c.past, c.rows, far) == 0
    pools = {n: H.DevBuf(hip.lib, n_pages * one) for n in "kv"}
    for n, host in (("k", c.k), ("v", c.v)):
        for t, f in zip(c.tables, far):
            for a, b in zip(t, f):
                row = np.ascontiguousarray(host[a])
                hip.lib.tts_hip_to_device(pools[n].at(int(b) * one), row.ctypes.data, one)
    c.dev = pools
    q = normal(np.random.default_rng(9), (71, 32, hd), 0)
    assert P.check(c, P.attention(c, q, 0, 0.088), *c.attend(q, 0.088), 0)
    x = normal(np.random.default_rng(10), (71, kv, hd), 0)
    d = P.Dev(hip.lib, x)
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, pools["k"].ptr, pools["v"].ptr, d.ptr, d.ptr, 0, 0, None) == 0
    got = np.empty((kv, page, hd), np.uint16)
    hip.lib.tts_hip_to_host(got.ctypes.data, pools["v"].at(int(far[1][1]) * one), one)
    want = c.v[c.tables[1][1]].copy()
    want[:, :6] = P.bits16(x[65:71]).transpose(1, 0, 2)
    assert np.array_equal(got, want)
    d.free()
    c.free()


@pytest.mark.parametrize("bf16", [0, 1])
def test_more_items_than_a_grid_has(hip, bf16):
    """Tiles of columns past 65535, the most that a grid's second dimension has: the rows around that place."""
    heads, hd, rows, w = 4, 256, 262144 + 600, 3                  # four columns a row, 16 to a tile
    c = P.Cache(hip, f"{rows}@0", 1 << 14, heads, 1, hd, window=w, seed=5, spare=0)
    c.fill(size=0.5)
    c.upload()
    rng = np.random.default_rng(12)
    block = normal(rng, (4096, heads, hd), bf16)
    q = np.tile(block, (-(-rows // 4096), 1, 1))[:rows]
    got = P.attention(c, q, bf16, 0.0625)
    keep = np.zeros(rows, bool)
    for at in (0, 262140, rows):
        keep[max(0, at - 100):at + 100] = True
    assert np.isfinite(got).all()
    assert P.check(c, got, *c.attend(q, 0.0625, keep), bf16, keep)
    c.free()


def test_an_empty_batch_does_nothing(hip):
    c = P.Cache(hip, "0@5 0@0", 16, 8, 2, 64, seed=4)
    c.upload()
    q = P.Dev(hip.lib, np.zeros(64, np.float32), behind=64)
    assert hip.lib.tts_hip_paged_attention(q.ptr, q.ptr + 128, 0, 0, c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, 1.0) == 0
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, q.ptr, q.ptr, 0, 0, None) == 0
    assert hip.lib.tts_hip_rotary(q.ptr, q.ptr, 0, 0, 1, 64, 0, 0, q.ptr, P.how(hip, q.ptr, 0, 0)) == 0
    assert (q.get() == 0).all() and all((x == P.NAN16).all() for x in c.download())
    q.free()
    c.free()


def test_a_refused_batch_leaves_none(hip):
    c = P.Cache(hip, "1@5", 16, 8, 2, 64, seed=4)
    c.upload()
    q = P.Dev(hip.lib, np.zeros((1, 512), np.float32))
    assert c.batch.positions()
    assert c.batch.set([5], [1], [[99]]) == -1 and b"page 0" in hip.lib.tts_hip_last_error()
    assert not c.batch.positions()
    assert hip.lib.tts_hip_paged_attention(q.ptr, q.ptr, 0, 0, c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, 1.0) == -1
    assert hip.lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, q.ptr, q.ptr, 0, 0, None) == -1
    assert c.batch.set([5], [1], [[1]]) == 0 and c.batch.positions()
    q.free()
    c.free()


@pytest.mark.parametrize("bf16", [0, 1])
def test_prompts_and_steps_as_a_program_runs_them(hip, bf16):
    """A layer's attention of three utterances: prompts in chunks, then steps of all of them, from one matrix q|k|v, on one handle.  Each step's cache and
    results against 64 bits, from the cache that the library wrote."""
    heads, kv, hd, page = 8, 2, 128, 16
    width, rng, lib = (heads + 2 * kv) * hd, np.random.default_rng(11), hip.lib
    c = P.Cache(hip, "90@0 70@0 8@0", page, heads, kv, hd, seed=6)
    c.upload()
    gain = [1 + 0.1 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    t = P.turns(hd, 1e6)
    dt, dq, dk = P.Dev(lib, np.zeros(hd // 2)), P.Dev(lib, gain[0]), P.Dev(lib, gain[1])
    assert lib.tts_hip_rotary_turns(dt.ptr, hd, 1e6, 1.0, 0, 1, 32) == 0
    queries, keys = P.how(hip, dt.ptr, hd, 1, dq.ptr), P.how(hip, dt.ptr, hd, 1, dk.ptr)
    past = [0, 0, 0]
    for rows in ([50, 0, 0], [37, 66, 0], [1, 1, 6], [1, 1, 1], [1, 0, 1], [0, 1, 0], [0, 1, 0], [0, 1, 0]):
        x = rng.standard_normal((sum(rows), width)).astype(np.float32)
        x = P.bits16(x) if bf16 else x
        dx = P.Dev(lib, x)
        turned = P.Dev(lib, np.zeros((sum(rows), heads * hd), x.dtype))
        out = P.Dev(lib, np.zeros((sum(rows), heads * hd), x.dtype), behind=1024)
        assert c.batch.set(past, rows, c.tables) == 0, lib.tts_hip_last_error()
        at, size = dx.ptr, x.itemsize
        assert lib.tts_hip_rotary(turned.ptr, at, bf16, sum(rows), heads, hd, 0, width, c.batch.positions(), queries) == 0
        assert lib.tts_hip_paged_append(c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, at + heads * hd * size, at + (heads + kv) * hd * size, bf16, width, keys) == 0
        assert lib.tts_hip_paged_attention(out.ptr, turned.ptr, bf16, 0, c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, hd ** -0.5) == 0
        c.past, c.rows = list(past), list(rows)
        got, q, (k_bits, v_bits) = out.get(), turned.get(), c.download()
        if bf16:
            got, q, x = P.value16(got), P.value16(q), P.value16(x)
        pos = c.positions()
        pages = np.concatenate([c.tables[i][np.arange(p, p + r) // page] for i, (r, p) in enumerate(zip(rows, past))])
        k = x[:, heads * hd:(heads + kv) * hd].reshape(-1, kv, hd)
        for new, old, g in ((P.value16(np.ascontiguousarray(k_bits[pages, :, pos % page])), k, gain[1]),
                            (q.reshape(-1, heads, hd), x[:, :heads * hd].reshape(-1, heads, hd), gain[0])):
            want, both = P.turned(old, pos, t, 1, g, 1e-5)
            rel = 8 * 2.0 ** -23 + (hd / 8 + 8) * 2.0 ** -24
            rounded = bf16 or new.shape[1] == kv
            assert (np.abs(new - want) <= rel * both + (2.0 ** -8 * (np.abs(want) + rel * both) if rounded else 0)).all()
        v = x[:, (heads + kv) * hd:].reshape(-1, kv, hd)
        c.v[pages, :, pos % page] = P.bits16(v)
        c.k[pages, :, pos % page] = k_bits[pages, :, pos % page]
        assert np.array_equal(c.k, k_bits) and np.array_equal(c.v, v_bits)                          # and nothing else
        q = q.reshape(-1, heads, hd)
        assert P.check(c, got.reshape(q.shape), *c.attend(q, hd ** -0.5), bf16)
        past = [p + r for p, r in zip(past, rows)]
        for d in (dx, turned, out):
            d.free()
    for d in (dt, dq, dk):
        d.free()
    c.free()


def test_handles_side_by_side_and_a_new_context(hip):
    """Two handles in turn, described again while their calls are queued; a handle lives on through tts_hip_free and a new context."""
    a, b = (P.Cache(hip, s, 16, 8, 2, 64, seed=i) for i, s in enumerate(("200@30 1@700", "1@800 1@40")))
    q = [normal(np.random.default_rng(i), (sum(c.rows), 8, 64), 0) for i, c in enumerate((a, b))]
    for c in (a, b):
        c.fill()
        c.upload()
    lib = hip.lib
    bufs = [(P.Dev(lib, x), [P.Dev(lib, np.zeros(x.shape, np.float32)) for _ in range(6)]) for x in q]
    for i in range(6):
        for c, (dq, outs) in zip((a, b), bufs):
            assert c.batch.set(c.past, c.rows, c.tables) == 0
            assert lib.tts_hip_paged_attention(outs[i].ptr, dq.ptr, 0, 0, c.batch.ptr, c.dev["k"].ptr, c.dev["v"].ptr, 0.125) == 0
    for c, x, (dq, outs) in zip((a, b), q, bufs):
        want = c.attend(x, 0.125)
        first = outs[0].get()
        assert P.check(c, first, *want, 0)
        for o in outs[1:]:
            assert np.array_equal(o.get(), first)
    lib.tts_hip_free()
    assert lib.tts_hip_paged_set(a.batch.ptr, 0, None, None, None, 0) == -1
    assert lib.tts_hip_init(8) == 0
    assert a.batch.set(a.past, a.rows, a.tables) == 0
    assert np.array_equal(P.attention(a, q[0], 0, 0.125), bufs[0][1][0].get())
    for dq, outs in bufs:
        for d in (dq, *outs):
            d.free()
    a.free()
    b.free()
