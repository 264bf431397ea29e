"""Attention over the 4-bit cache where its kernel for many columns runs (queries times heads per kv head; vt_mx4_plans.h says from how many on),
against numpy in 64 bits: one part and several, groups of 1, 3, 4, 5 and 7 heads, tiles of columns and waves that are partly filled."""
import numpy as np
import pytest

import hipsupport as H
import mx4support as M
from test_gpu_kv4 import attend, oracle

pytestmark = pytest.mark.gpu

# heads, kv heads, head_dim, queries, rows in front -> workgroups that share a head's rows for a tile of columns at most, on 256 CUs (test_mx4_plans_cpu.py asserts
# these, and that the kernel for many columns is the one)
CASES = {(32, 8, 128, 333, 0): 1, (32, 8, 128, 333, 130): 1, (32, 8, 128, 600, 700): 3, (16, 16, 64, 530, 0): 3, (14, 2, 64, 601, 37): 3, (9, 3, 128, 911, 0): 4, (8, 8, 128, 1030, 5): 5,
         (20, 20, 128, 420, 999): 4, (15, 5, 64, 1100, 77): 4, (32, 8, 128, 1531, 0): 2}


@pytest.fixture(scope="module")
def hip():
    h = H.Hip(kv_max=8)
    yield h
    h.close()


def case(hip, heads, kv_heads, hd, rows, pos, spread=1.0, extra=37):
    c = M.Cache(hip, pos + rows + extra, kv_heads, hd)
    r = np.random.default_rng(heads + 31 * rows + pos)
    for a in c.host.values():
        a[:] = 255                                        # behind the last row: codes of -6, scales of NaN
    c.fill(*[(r.standard_normal((kv_heads, pos + rows, hd)) * spread).astype(np.float32) for _ in range(2)])
    return c, (r.standard_normal((rows, heads * hd)) * spread).astype(np.float32)


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", CASES)
def test_attention(hip, heads, kv_heads, hd, rows, pos):
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    scale = float(np.float32(1 / np.sqrt(hd)))
    cache = c.upload()
    got = attend(hip, cache, q, pos, heads, scale)
    want, tol = oracle(q, *c.values(pos + rows), pos, heads, scale)
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())
    for _ in range(3):
        assert np.array_equal(got, attend(hip, cache, q, pos, heads, scale))
    c.free()


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", [(32, 8, 128, 333, 130), (14, 2, 64, 601, 37), (9, 3, 128, 911, 0)])
@pytest.mark.parametrize("spread,scale", [(8.0, 1.0), (1e-3, 1.0), (1e15, 1e-31), (3.0, -0.5), (1.0, 0.0)])
def test_attention_scores_far_apart_and_equal(hip, heads, kv_heads, hd, rows, pos, spread, scale):
    c, q = case(hip, heads, kv_heads, hd, rows, pos, spread)
    got = attend(hip, c.upload(), q, pos, heads, scale)
    want, tol = oracle(q, *c.values(pos + rows), pos, heads, float(np.float32(scale)))
    c.free()
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", CASES)
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_attention_nan_reaches_who_sees_it(hip, heads, kv_heads, hd, rows, pos, which):
    """A NaN in one block of one key's or value's row of the last kv head, at four places of the rows: the queries that see the row answer NaN (all of it, or the block's
    values), the others what they answered without it, bit for bit."""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    group = heads // kv_heads
    clean = attend(hip, c.upload(), q, pos, heads, 0.1).reshape(rows, heads, hd)
    for bad in (pos + rows // 3, pos + rows - 1, (pos + rows) // 2, 63):
        held = c.host[which][-1, bad, 1]
        c.host[which][-1, bad, 1] = 255
        got = attend(hip, c.upload(), q, pos, heads, 0.1).reshape(rows, heads, hd)
        c.host[which][-1, bad, 1] = held
        hit = np.zeros(got.shape, bool)
        hit[pos + np.arange(rows) >= bad, heads - group:, :] = True
        if which == "vs":
            hit[..., :32] = False
            hit[..., 64:] = False
        assert np.array_equal(np.isnan(got), hit) and np.array_equal(got[~hit], clean[~hit])
    c.free()


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", [(32, 8, 128, 333, 130), (14, 2, 64, 601, 37), (9, 3, 128, 911, 0), (16, 16, 64, 530, 0)])
def test_attention_hidden_rows_change_nothing(hip, heads, kv_heads, hd, rows, pos):
    """Behind the last row, and so in front of the next head's first: zeros, the largest scales, NaN.  The same bits."""
    outs = []
    for fill in (0, 254, 255):
        c, q = case(hip, heads, kv_heads, hd, rows, pos, extra=1 + rows % 3)
        for a in c.host.values():
            a[:, pos + rows:] = fill
        outs.append(attend(hip, c.upload(), q, pos, heads, 0.1))
        c.free()
    assert np.isfinite(outs[0]).all() and np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


@pytest.mark.parametrize("heads,kv_heads,hd,rows,pos", [(32, 8, 128, 333, 130), (16, 16, 64, 530, 0), (9, 3, 128, 911, 0)])
def test_a_prompt_in_pieces_is_the_prompt(hip, heads, kv_heads, hd, rows, pos):
    """Its last queries alone, by the kernel for few columns, and all of them at once: each within the tolerance of the same results."""
    c, q = case(hip, heads, kv_heads, hd, rows, pos)
    cache = c.upload()
    whole = attend(hip, cache, q, pos, heads, 0.1)
    want, tol = oracle(q, *c.values(pos + rows), pos, heads, float(np.float32(0.1)))
    for n in (1, 5, 40):
        piece = attend(hip, cache, q[rows - n:], pos + rows - n, heads, 0.1)
        assert np.all(np.abs(piece - whole[rows - n:]) <= 2 * tol[rows - n:])
    c.free()
    assert np.all(np.abs(whole - want) <= tol)
