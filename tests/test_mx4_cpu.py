"""What the 4-bit operators refuse, without a GPU: the arguments are looked at first.  Pointers here are numbers that nothing reads."""
import ctypes as C
import os

import numpy as np
import pytest

import hipsupport as H
import mx4support as M

pkg = H.load_package()
pytestmark = pytest.mark.skipif(not os.path.exists(pkg.LIB_PATH), reason="library not built (run __graft_entry__.build())")
P, Q, R = 1 << 20, 1 << 21, 1 << 22


def refused(name, *args):
    lib = pkg.lib()
    n = lib.tts_hip_error_count()
    assert getattr(lib, name)(*args) == -1
    assert lib.tts_hip_error_count() == n + 1
    text = lib.tts_hip_last_error().decode()
    assert text.startswith(name) and "not initialised" not in text, text


@pytest.mark.parametrize("args", [(None, Q, R, 0, 4, 128, 0), (P, None, R, 0, 4, 128, 0), (P, Q, None, 0, 4, 128, 0), (P, Q, R, 0, 0, 128, 0), (P, Q, R, 0, 4, 0, 0),
                                  (P, Q, R, 0, -1, 128, 0), (P, Q, R, 0, 4, 128, 127), (P, Q, R, 0, 4, 128, -128), (P + 8, Q, R, 0, 4, 128, 0), (P, Q + 2, R, 0, 4, 128, 0),
                                  (P, Q, R + 2, 0, 4, 128, 0), (P, Q, R + 1, 1, 4, 128, 0), (P, Q, R, 0, 4, (1 << 27) + 1, 0), (P, Q, R, 0, (1 << 30) + 1, 1, 0)])
def test_quantize_refuses(args):
    refused("tts_hip_mx4_quantize", *args)
    codes, scales, x, bf16, rows, cols, stride = args
    if not bf16:
        refused("tts_hip_mx4_dequantize", x, codes, scales, rows, cols, stride)


@pytest.mark.parametrize("args", [(None, Q, P, R, 1, 8, 8), (P, None, Q, R, 1, 8, 8), (P, Q, None, R, 1, 8, 8), (P, Q, R, None, 1, 8, 8), (P, Q, R, P, 0, 8, 8),
                                  (P, Q, R, P, 1, 0, 8), (P, Q, R, P, 1, 8, 0), (P + 2, Q, R, P, 1, 8, 8), (P, Q + 1, R, P, 1, 8, 8), (P, Q, R + 4, P, 1, 8, 8), (P, Q, R, P + 1, 1, 8, 8), (P, Q, R, P, 1, (1 << 23) + 1, 8),
                                  (P, Q, R, P, (1 << 30) + 1, 8, 8), (P, Q, R, P, 1, 8, (1 << 30) + 1)])
def test_linear_refuses(args):
    refused("tts_hip_linear_mx4", *args)


def cache(**other):
    c = pkg.Kv4(P, P, P, P, 100, 8, 128)
    for k, v in other.items():
        setattr(c, k, v)
    return C.byref(c)


BAD = [{"k_codes": None}, {"v_scales": None}, {"k_codes": P + 8}, {"v_scales": P + 2}, {"max_rows": 0}, {"n_kv_heads": 0}, {"head_dim": 32}, {"head_dim": 96}, {"head_dim": 320}]


@pytest.mark.parametrize("other", BAD)
def test_every_call_refuses_a_bad_cache(other):
    c = cache(**other)
    refused("tts_hip_kv4_append", c, P, P, 1, 0, 0)
    refused("tts_hip_kv4_read", P, P, c, 1, 0, 0)
    refused("tts_hip_kv4_attention", P, P, c, 1, 0, 32, 0.1)


@pytest.mark.parametrize("n,pos", [(0, 0), (-1, 5), (1, -1), (1, 100), (101, 0), (50, 51), (1, 2 ** 31 - 1), (2 ** 31 - 1, 1)])
def test_rows_outside_the_cache(n, pos):
    refused("tts_hip_kv4_append", cache(), P, P, n, pos, 0)
    refused("tts_hip_kv4_read", P, P, cache(), n, pos, 0)
    refused("tts_hip_kv4_attention", P, P, cache(), n, pos, 32, 0.1)


def test_other_arguments():
    refused("tts_hip_kv4_append", None, P, P, 1, 0, 0)
    refused("tts_hip_kv4_append", cache(), None, P, 1, 0, 0)
    refused("tts_hip_kv4_append", cache(), P, P + 2, 1, 0, 0)
    refused("tts_hip_kv4_append", cache(), P, P, 1, 0, 1023)
    refused("tts_hip_kv4_read", P, None, cache(), 1, 0, 0)
    refused("tts_hip_kv4_attention", None, P, cache(), 1, 0, 32, 0.1)
    refused("tts_hip_kv4_attention", P, P + 4, cache(), 1, 0, 32, 0.1)
    refused("tts_hip_kv4_attention", P, P, cache(), 1, 0, 33, 0.1)
    refused("tts_hip_kv4_attention", P, P, cache(), 1, 0, 0, 0.1)
    refused("tts_hip_kv4_attention", P, P, cache(max_rows=2 ** 31 - 1), 1, 1 << 24, 32, 0.1)
    refused("tts_hip_kv4_attention", P, P, cache(n_kv_heads=65536), 1, 0, 65536, 0.1)
    refused("tts_hip_kv4_attention", P, P, cache(n_kv_heads=1), 1, 0, (1 << 19) + 1, 0.1)


def test_the_oracle_rounds_as_the_format_says():
    x = np.zeros((1, 32), np.float32)
    x[0, :10] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, 7]
    codes, scales = M.encode(x)
    assert scales[0, 0] == 127
    assert list(M.decode(codes, scales)[0, :10]) == [6, 0, 1, 1, 2, 2, 4, 4, 0, 6]
    near = np.random.default_rng(1).standard_normal((50, 64)).astype(np.float32)
    back = M.decode(*M.encode(near))
    top = M.block_max(near)
    assert np.all(np.abs(back - near) <= np.maximum(np.exp2(np.floor(np.log2(top))) / 4, top - 6 * np.exp2(np.floor(np.log2(top)) - 2)))
