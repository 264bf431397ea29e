"""Microscaled 4-bit floats in numpy, from their definition: blocks of 32 values of a row, a scale 2^(s - 127) each and codes
e2m1.  Plain and in 64 bits; the tests of the operators compare with it."""
import ctypes as C

import numpy as np

import hipsupport as H

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def panels(cols):
    return (cols + 127) // 128


def encode(x):
    """[..., 32 n] fp32 -> codes [..., 16 n], scales [..., n]."""
    b = np.asarray(x, np.float32).astype(np.float64).reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b)
    top = np.abs(b).max(-1)
    s = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127).clip(-127, None)
    q = np.abs(b) / np.exp2(s.astype(np.float64))[..., None]
    d = np.abs(q[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = np.arange(8) % 2 == 0
    code = np.where((near & even).any(-1), (near & even).argmax(-1), near.argmax(-1))      # a tie is between an even and an odd code
    code = np.where(q > 6, 7, code) + 8 * np.signbit(np.where(bad[..., None], 0.0, b))
    code = code.astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(bad, 255, s + 127).astype(np.uint8)


def decode(codes, scales):
    """-> float64 [..., 32 n]"""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (-1, 32))
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(codes.shape[:-1] + (-1,))


def encode_matrix(x):
    pad = 128 * panels(x.shape[1]) - x.shape[1]
    return encode(np.concatenate((x, np.zeros((x.shape[0], pad), np.float32)), 1))


def block_max(x):
    """Every value's block's largest magnitude, blocks of 32 from the row's start."""
    cols = x.shape[-1]
    p = np.concatenate((x, np.zeros(x.shape[:-1] + (-cols % 32,), x.dtype)), -1)
    b = np.abs(p.reshape(p.shape[:-1] + (-1, 32))).max(-1)
    return np.repeat(b, 32, -1)[..., :cols].astype(np.float64)


class Cache:
    """A 4-bit cache on the device, with its bytes on the host."""

    def __init__(self, hip, rows, kv_heads, head_dim):
        self.hip, self.shape = hip, (kv_heads, rows, head_dim)
        self.host = {n: np.zeros((kv_heads, rows, head_dim // (2 if n[1] == "c" else 32)), np.uint8) for n in ("kc", "ks", "vc", "vs")}
        self.buf = {}

    def fill(self, k, v, pos=0):
        """k, v [kv_heads, n, head_dim] -> rows from pos on"""
        for n, x in (("k", k), ("v", v)):
            self.host[n + "c"][:, pos:pos + x.shape[1]], self.host[n + "s"][:, pos:pos + x.shape[1]] = encode(x)

    def upload(self):
        self.free()
        self.buf = {n: H.DevBuf.from_numpy(self.hip.lib, a) for n, a in self.host.items()}
        h, r, d = self.shape
        self.c = self.hip.pkg.Kv4(*[self.buf[n].ptr for n in ("kc", "ks", "vc", "vs")], r, h, d)
        return C.byref(self.c)

    def download(self):
        return {n: b.to_numpy(np.uint8, self.host[n].shape) for n, b in self.buf.items()}

    def values(self, n):
        return decode(self.host["kc"][:, :n], self.host["ks"][:, :n]), decode(self.host["vc"][:, :n], self.host["vs"][:, :n])

    def free(self):
        for b in self.buf.values():
            b.free()
        self.buf = {}


def planes(x, n=5):
    """What n planes of e2m3 (0 .. 2 in steps of 1/8, 2 .. 4 of 1/4, 4 .. 7.5 of 1/2) hold of [rows, cols] fp32: each the nearest to what the ones before leave of
    its block of 32, with a scale of its own that puts the largest magnitude at 3.875 .. 7.75, the fifth's 2^-4 of the fourth's."""
    rows, cols = x.shape
    left = np.concatenate((x, np.zeros((rows, -cols % 32), np.float32)), 1).reshape(rows, -1, 32).astype(np.float32)
    held = np.zeros(left.shape)
    for i in range(n):
        top = np.abs(left).max(-1, keepdims=True).view(np.uint32).astype(np.int64)
        scale = np.maximum((top + 0x80000 >> 23) - 2 if i < 4 else scale - 4, 0)
        unit = np.exp2(scale.astype(np.float64) - 127)
        a = np.abs(left) / unit
        step = np.where(a < 2, 0.125, np.where(a < 4, 0.25, 0.5))
        q = np.copysign(np.minimum(np.round(a / step) * step, 7.5), left) * unit
        held += q
        left = (left - q).astype(np.float32)              # exact
    return held.reshape(rows, -1)[:, :cols]
