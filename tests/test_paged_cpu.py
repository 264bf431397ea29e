"""What the operators over a paged cache refuse, without a GPU: the arguments are looked at first.  Pointers here are numbers that nothing reads."""
import ctypes as C
import os

import numpy as np
import pytest

import hipsupport as H

pkg = H.load_package()
pytestmark = pytest.mark.skipif(not os.path.exists(pkg.LIB_PATH), reason="library not built (run __graft_entry__.build())")
P, Q, R, S = 1 << 20, 1 << 21, 1 << 22, 1 << 23
NAN, INF = float("nan"), float("inf")


def refused(name, *args, answer=-1):
    lib = pkg.lib()
    n = lib.tts_hip_error_count()
    assert getattr(lib, name)(*args) == answer
    assert lib.tts_hip_error_count() == n + 1
    text = lib.tts_hip_last_error().decode()
    assert text.startswith(name) and "not initialised" not in text, text
    return text


def shape(**other):
    s = pkg.PagedShape(10, 16, 32, 8, 128, 0)
    for k, v in other.items():
        setattr(s, k, v)
    return C.byref(s)


@pytest.fixture
def batch():
    b = pkg.lib().tts_hip_paged_create(shape(), 3, 64, 10)
    assert b
    yield b
    pkg.lib().tts_hip_paged_free(b)


@pytest.mark.parametrize("other", [{"n_pages": 0}, {"page_rows": 8}, {"page_rows": 48}, {"page_rows": 1 << 21}, {"page_rows": -16}, {"n_kv_heads": 0},
                                   {"n_heads": 33}, {"n_heads": 0}, {"n_heads": -32},
                                   {"head_dim": 32}, {"head_dim": 96}, {"head_dim": 320}, {"window": -1}, {"n_heads": 4097, "n_kv_heads": 1},
                                   {"n_heads": 1 << 17, "n_kv_heads": 1 << 17}])
def test_create_refuses_a_shape(other):
    refused("tts_hip_paged_create", shape(**other), 3, 64, 10, answer=None)


@pytest.mark.parametrize("seqs,rows,table", [(0, 64, 10), (3, 0, 10), (3, 64, 0), (-1, 64, 10), (3, (1 << 22) + 1, 10), ((1 << 22) + 1, 64, 10),
                                             (3, 64, (1 << 28) + 1)])
def test_create_refuses_sizes(seqs, rows, table):
    refused("tts_hip_paged_create", shape(), seqs, rows, table, answer=None)


def test_create_refuses_more_columns_than_are_counted():
    refused("tts_hip_paged_create", shape(n_heads=4096, n_kv_heads=1), 3, 1 << 20, 10, answer=None)
    refused("tts_hip_paged_create", None, 3, 64, 10, answer=None)


def ints(*v):
    return np.array(v, np.int32)


@pytest.mark.parametrize("n,past,rows,tables,stride,why", [
    (-1, (0,), (1,), (1,), 1, "sequences"), (4, (0,) * 4, (1,) * 4, (1, 2, 3, 4), 1, "sequences"), (1, (0,), (1,), (1,), -1, "sequences"),
    (1, (-1,), (1,), (1,), 1, "rows behind"), (1, (0,), (-1,), (1,), 1, "rows behind"), (1, (1 << 30,), (1,), (1,), 1, "rows behind"),
    (1, (0,), (65,), (1, 2, 3, 4, 5), 5, "new rows"), (1, (16,), (1,), (1,), 1, "pages"),
    (2, (95, 95), (1, 1), tuple(range(6)) + (0, 1, 2, 3, 4, 6), 6, "pages"), (1, (0,), (1,), (10,), 1, "page 0"), (1, (16,), (1,), (-1, 2), 2, "page 0"),
    (2, (3, 7), (1, 1), (4, 4), 1, "twice")])
def test_set_refuses(batch, n, past, rows, tables, stride, why):
    past, rows, tables = ints(*past), ints(*rows), ints(*tables)
    assert why in refused("tts_hip_paged_set", batch, n, past.ctypes.data, rows.ctypes.data, tables.ctypes.data, stride)


def test_set_refuses_pointers(batch):
    a = ints(1)
    refused("tts_hip_paged_set", None, 1, a.ctypes.data, a.ctypes.data, a.ctypes.data, 1)
    for i in range(3):
        refused("tts_hip_paged_set", batch, 1, *[None if i == j else a.ctypes.data for j in range(3)], 1)


@pytest.mark.skipif(H.gpu_present(), reason="only meaningful without a GPU")
def test_a_batch_needs_a_context(batch):
    lib, a = pkg.lib(), ints(1)
    assert lib.tts_hip_paged_set(batch, 1, a.ctypes.data, a.ctypes.data, a.ctypes.data, 1) == -1 and b"not initialised" in lib.tts_hip_last_error()
    assert lib.tts_hip_paged_positions(batch) is None
    assert lib.tts_hip_paged_attention(P, Q, 0, 0, batch, R, S, 1.0) == -1
    lib.tts_hip_paged_free(None)


@pytest.mark.parametrize("rot,theta,factor,original,low,high",
                         [(0, 1e6, 1, 0, 1, 32), (3, 1e6, 1, 0, 1, 32), (514, 1e6, 1, 0, 1, 32), (64, 0, 1, 0, 1, 32), (64, NAN, 1, 0, 1, 32),
                          (64, INF, 1, 0, 1, 32), (64, 1e6, 0, 0, 1, 32), (64, 1e6, -2, 0, 1, 32), (64, 1e6, 1, -1, 1, 32), (64, 1e6, 1, 0, 2, 2),
                          (64, 1e6, 1, 0, NAN, 2), (64, 1e6, 1, 0, 1, INF)])
def test_turns_refuses(rot, theta, factor, original, low, high):
    refused("tts_hip_rotary_turns", P, rot, theta, factor, original, low, high)


def test_turns_refuses_pointers():
    for p in (None, P + 4):
        refused("tts_hip_rotary_turns", p, 64, 1e6, 1.0, 0, 1.0, 32.0)


def how(**other):
    h = pkg.Rotary(P, None, 128, 0, 1.0, 1e-5)
    for k, v in other.items():
        setattr(h, k, v)
    return C.byref(h)


BAD_TURNS = [{"rot_dim": -2}, {"rot_dim": 3}, {"rot_dim": 130}, {"half": 2}, {"half": -1}, {"d_turns": None}, {"d_turns": P + 4}, {"magnitude": NAN},
             {"magnitude": INF}, {"d_gain": P + 2}, {"d_gain": P, "eps": -1.0}, {"d_gain": P, "eps": NAN}]


@pytest.mark.parametrize("other", BAD_TURNS)
def test_bad_turns_are_refused(batch, other):
    refused("tts_hip_rotary", P, Q, 0, 1, 32, 128, 0, 0, R, how(**other))
    refused("tts_hip_paged_append", batch, P, Q, R, S, 0, 0, how(**other))


@pytest.mark.parametrize("args", [(None, Q, 0, 1, 32, 128, 0, 0, R), (P, None, 0, 1, 32, 128, 0, 0, R), (P + 2, Q, 0, 1, 32, 128, 0, 0, R),
                                  (P, Q + 1, 1, 1, 32, 128, 0, 0, R), (P, Q, 0, -1, 32, 128, 0, 0, R), (P, Q, 0, 1, 0, 128, 0, 0, R),
                                  (P, Q, 0, 1, 32, 0, 0, 0, R), (P, Q, 0, 1, 32, 129, 0, 0, R), (P, Q, 0, 1, 32, 514, 0, 0, R),
                                  (P, Q, 0, 1, 32, 128, 4095, 0, R), (P, Q, 0, 1, 32, 128, 0, 4095, R), (P, Q, 0, 1, 32, 128, 0, -4096, R),
                                  (P, Q, 0, 1, 32, 128, 0, 0, None), (P, Q, 0, 1, 32, 128, 0, 0, R + 2), (P, Q, 0, (1 << 30) + 1, 32, 128, 0, 0, R),
                                  (P, Q, 0, 1, 1 << 23, 128, 0, 0, R)])
def test_rotary_refuses(args):
    refused("tts_hip_rotary", *args, how())
    refused("tts_hip_rotary", P, Q, 0, 1, 32, 128, 0, 0, R, None)


@pytest.mark.parametrize("args", [(None, Q, R, S, 0, 0), (P, None, R, S, 0, 0), (P, Q, None, S, 0, 0), (P, Q, R, None, 0, 0), (P + 8, Q, R, S, 0, 0),
                                  (P, Q + 2, R, S, 0, 0), (P, Q, R + 2, S, 0, 0), (P, Q, R, S + 1, 1, 0),
                                  (P, Q, R, S, 0, 1023), (P, Q, R, S, 0, -1024)])
def test_append_refuses(batch, args):
    refused("tts_hip_paged_append", batch, *args, None)
    refused("tts_hip_paged_append", None, P, Q, R, S, 0, 0, None)


@pytest.mark.parametrize("out,q,stride,k,v,scale", [(None, Q, 0, R, S, 1.0), (P, None, 0, R, S, 1.0), (P, Q, 0, None, S, 1.0), (P, Q, 0, R, None, 1.0),
                                                    (P + 8, Q, 0, R, S, 1.0), (P, Q + 4, 0, R, S, 1.0), (P, Q, 0, R + 8, S, 1.0),
                                                    (P, Q, 4095, R, S, 1.0), (P, Q, 4100, R, S, 1.0), (P, Q, 0, R, S, 0.0), (P, Q, 0, R, S, -1.0),
                                                    (P, Q, 0, R, S, NAN), (P, Q, 0, R, S, INF)])
def test_attention_refuses(batch, out, q, stride, k, v, scale):
    refused("tts_hip_paged_attention", out, q, 0, stride, batch, k, v, scale)
    refused("tts_hip_paged_attention", P, Q, 0, 0, None, R, S, 1.0)


def test_calls_without_a_batch_are_refused(batch):
    """A handle that no batch was described to yet."""
    assert "no batch" in refused("tts_hip_paged_attention", P, Q, 0, 0, batch, R, S, 1.0)
    assert "no batch" in refused("tts_hip_paged_append", batch, P, Q, R, S, 0, 0, None)
    assert "no batch" in refused("tts_hip_paged_positions", batch, answer=None)
