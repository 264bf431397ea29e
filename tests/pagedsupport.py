"""A paged cache, rotary positions and attention in numpy and 64 bits, from their definitions; the tests of the operators compare with it."""
import ctypes as C
import math

import numpy as np

import hipsupport as H
from voxtral_tts_c_amd.session import PagedBatch

NAN16 = 0x7FC1


def bits16(x):
    """fp32 -> bf16 bits, to nearest even; finite values"""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def value16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def seqs_of(batch):
    """"3@40 1@7" -> rows [3, 1], past [40, 7]"""
    pairs = [tuple(map(int, s.split("@"))) for s in batch.split()]
    return [r for r, _ in pairs], [p for _, p in pairs]


def turns(rot, theta, factor=1.0, original=0, low=1.0, high=32.0):
    f = theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot) / (2 * math.pi)
    keep = np.clip((f * original - low) / (high - low), 0, 1)
    return f if factor == 1 else f * (keep + (1 - keep) / factor)


def turned(x, positions, t, half, gain=None, eps=0.0, magnitude=1.0):
    """[rows, heads, head_dim] in 64 bits, and each value's |a| + |b| of its pair: what its rounding goes by"""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    rot = 2 * len(t)
    y, size = x.copy(), np.abs(x)
    a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if half else (x[..., 0:rot:2], x[..., 1:rot:2])
    angle = np.asarray(positions, np.float64)[:, None] * t[None, :]
    angle = ((angle - np.round(angle)) * 2 * math.pi)[:, None, :]
    c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
    both = (np.abs(a) + np.abs(b)) * magnitude
    for to, u, v in ((y, a * c - b * s, a * s + b * c), (size, both, both)):
        if half:
            to[..., :rot // 2], to[..., rot // 2:rot] = u, v
        else:
            to[..., 0:rot:2], to[..., 1:rot:2] = u, v
    return y, size


class Dev:
    """An array on the device, with what lies behind it."""

    def __init__(self, lib, a, behind=0):
        self.lib, self.dtype, self.shape, self.behind = lib, a.dtype, a.shape, behind
        self.buf = H.DevBuf(lib, max(16, a.nbytes + behind))
        if behind:
            lib.tts_hip_memset(self.buf.ptr, 0x5A, a.nbytes + behind)
        if a.nbytes:
            a = np.ascontiguousarray(a)
            lib.tts_hip_to_device(self.buf.ptr, a.ctypes.data, a.nbytes)
        self.ptr, self.nbytes = self.buf.ptr, a.nbytes

    def get(self):
        whole = np.empty(self.nbytes + self.behind, np.uint8)
        if whole.size:
            self.lib.tts_hip_to_host(whole.ctypes.data, self.ptr, whole.nbytes)
        assert (whole[self.nbytes:] == 0x5A).all(), "written behind the last row"
        return whole[:self.nbytes].view(self.dtype).reshape(self.shape)

    def free(self):
        self.buf.free()


class Cache:
    """Pools on the host and on the device, every row a NaN until a sequence's is there, and each sequence's pages in a random order."""

    def __init__(self, hip, batch, page_rows, heads, kv_heads, head_dim, window=0, seed=0, spare=2):
        self.hip, self.rows, self.past = hip, *seqs_of(batch)
        self.page_rows, self.heads, self.kv_heads, self.hd, self.window = page_rows, heads, kv_heads, head_dim, window
        self.rng = np.random.default_rng(seed)
        need = [-(-(r + p) // page_rows) for r, p in zip(self.rows, self.past)]
        self.n_pages = sum(need) + spare
        order = self.rng.permutation(self.n_pages).astype(np.int32)
        cut = np.cumsum([0] + need)
        self.tables = [order[cut[i]:cut[i + 1]] for i in range(len(need))]
        shape = (self.n_pages, kv_heads, page_rows, head_dim)
        self.k, self.v = np.full(shape, NAN16, np.uint16), np.full(shape, NAN16, np.uint16)
        self.batch = PagedBatch(self.n_pages, page_rows, heads, kv_heads, head_dim, window, max_seqs=max(1, len(need)), max_rows=max(1, sum(self.rows)),
                                max_table=max(1, sum(need)))
        assert self.batch.set(self.past, self.rows, self.tables) == 0, hip.lib.tts_hip_last_error()
        self.dev = {}

    def fill(self, upto=None, size=1.0):
        """Every sequence's rows (`upto`: the cached ones): k and v ~N(0, 1)"""
        for i, t in enumerate(self.tables):
            n = self.past[i] + (0 if upto == "past" else self.rows[i])
            for pool in (self.k, self.v):
                x = bits16(self.rng.standard_normal((n, self.kv_heads, self.hd), np.float32) * size)
                p = np.arange(n)
                pool[t[p // self.page_rows], :, p % self.page_rows] = x

    def upload(self):
        self.dev = {"k": Dev(self.hip.lib, self.k), "v": Dev(self.hip.lib, self.v)}

    def download(self):
        return self.dev["k"].get(), self.dev["v"].get()

    def sequence(self, i):
        """-> bits [kv_heads, rows, head_dim] of K and V"""
        n = self.past[i] + self.rows[i]
        p = np.arange(n)
        return [np.ascontiguousarray(pool[self.tables[i][p // self.page_rows], :, p % self.page_rows].transpose(1, 0, 2)) for pool in (self.k, self.v)]

    def positions(self):
        return np.concatenate([np.arange(p, p + r) for r, p in zip(self.rows, self.past)] or [np.zeros(0)]).astype(np.int32)

    def some(self):
        """Rows of the batch that are compared where it has many: of each sequence the first and last 20, those around its wave and workgroup borders, and
        some others."""
        keep, at = np.zeros(sum(self.rows), bool), 0
        for r in self.rows:
            for edge in (0, 32, 128, r // 2, r):
                keep[max(at, at + edge - 20):min(at + r, at + edge + 20)] = True
            keep[at + self.rng.integers(0, max(r, 1), min(r, 40))] = True
            at += r
        return keep

    def attend(self, q, scale, keep=None):
        """q [rows, heads, head_dim] -> results in 64 bits, the weighted sum of |v|, and the largest sum of |q k| scale that a query meets; NaN where it
        sees, in that value, a value that is not finite"""
        out, size, most = np.zeros(q.shape), np.zeros(q.shape), 0.0
        at, group = 0, self.heads // self.kv_heads
        for i, (r, p) in enumerate(zip(self.rows, self.past)):
            if r == 0:
                continue
            kb, vb = self.sequence(i)
            for h in range(self.kv_heads):
                k, v = value16(kb[h]).astype(np.float64), value16(vb[h]).astype(np.float64)
                clean, odd = np.where(np.isfinite(v), v, 0), ~np.isfinite(v)
                for r0 in range(0, r, 128):                                        # queries r0 .., of all heads on this one, over what they see
                    n = min(128, r - r0)
                    if keep is not None and not keep[at + r0:at + r0 + n].any():
                        continue
                    lo, hi = max(0, p + r0 - self.window + 1 if self.window else 0), p + r0 + n
                    age = np.arange(p + r0, hi)[:, None] - np.arange(lo, hi)[None, :]
                    hidden = (age < 0) | (age >= self.window if self.window else False)
                    to = (slice(at + r0, at + r0 + n), slice(h * group, (h + 1) * group))
                    x = q[to].astype(np.float64).transpose(1, 0, 2)
                    with np.errstate(invalid="ignore"):
                        w = np.where(hidden, -np.inf, x @ k[lo:hi].T * scale)
                        w = np.exp(w - w.max(-1, keepdims=True))
                        w = w / w.sum(-1, keepdims=True)
                        y = w @ clean[lo:hi]
                        out[to], size[to] = y.transpose(1, 0, 2), (w @ np.abs(clean[lo:hi])).transpose(1, 0, 2)
                        if odd[lo:hi].any():
                            out[to][((~hidden).astype(float) @ odd[lo:hi] > 0)[:, None, :].repeat(group, 1)] = np.nan
                    most = max(most, float((np.abs(x) @ np.where(np.isfinite(k[lo:hi]), np.abs(k[lo:hi]), 0).T * scale).max()))
            at += r
        return out, size, most

    def free(self):
        for d in self.dev.values():
            d.free()
        self.batch.free()


def attention(cache, q, bf16, scale, q_gap=0):
    """q [rows, heads, head_dim] fp32 (bf16 values where bf16) -> what the library answers, fp32"""
    lib, rows, width = cache.hip.lib, q.shape[0], q.shape[1] * q.shape[2]
    x = np.zeros((rows, width + q_gap), np.uint16 if bf16 else np.float32)
    x[:, :width] = bits16(q).reshape(rows, -1) if bf16 else q.reshape(rows, -1)
    dq, do = Dev(lib, x), Dev(lib, np.zeros((rows, width), x.dtype), behind=4096)
    try:
        assert lib.tts_hip_paged_attention(do.ptr, dq.ptr, int(bf16), width + q_gap if q_gap else 0, cache.batch.ptr, cache.dev["k"].ptr, cache.dev["v"].ptr,
                                           scale) == 0, lib.tts_hip_last_error()
        got = do.get()
    finally:
        dq.free()
        do.free()
    return (value16(got) if bf16 else got).reshape(q.shape)


def is_many(cache, i, bf16):
    """The kernel that rounds a bf16 batch's weights to bf16 (vt_paged_kinds_of)."""
    group = cache.heads // cache.kv_heads
    if cache.hd > 128 and not (cache.hd == 256 and bf16):
        return False
    all_of_them = sum(r * group * min(p + r / 2, cache.window or math.inf) * cache.kv_heads * cache.hd for r, p in zip(cache.rows, cache.past) if r * group > 64)
    return all_of_them >= (2.5e9 if cache.hd <= 128 else 1.3e9) and cache.rows[i] * group > 64


def check(cache, got, want, size, most, bf16, keep=None):
    """Elementwise by arithmetic, and fp32 by its norm too.  A score is the sum of 3 head_dim products (1: bf16) of bf16 values, exact, in fp32 that cuts:
    each of at most 3 head_dim / 8 additions is off by 2^-23 of what is summed so far, which `most` bounds; q times scale and its planes are off by 2^-24
    and 2^-25 of it, or a bf16 query's score times scale by 2^-24.  A weight is off by as much, relative to itself, by 2^-22 for the difference to the
    maximum and the exponential, and by the same again through the sum; sums of weights and results add 2^-23 of themselves for each of (row count / 8)
    steps at the worst, in practice a few.  bf16: a weight's rounding is 2^-8, at most, in the kernel for many columns, and 2^-16 in the other; a result's
    2^-8.  By norm: errors of single scores are independent, sqrt(3 head_dim / 16) 2^-24 times a few: 5e-7."""
    score = (3 * cache.hd / 8 + 3) * 2.0 ** -23 * most
    rel = np.full(got.shape[0], 2 * score + 64 * 2.0 ** -23)
    if bf16:
        at = 0
        for i, r in enumerate(cache.rows):
            rel[at:at + r] += 2.0 ** -8 if is_many(cache, i, bf16) else 2.0 ** -16
            at += r
    if keep is not None:
        got, want, size, rel = got[keep], want[keep], size[keep], rel[keep]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    tol = rel[:, None, None] * size + (2.0 ** -8 * (np.abs(want) + rel[:, None, None] * size) if bf16 else 0)
    d = np.abs(got - want)
    assert (d[ok] <= tol[ok]).all(), (float((d[ok] / np.maximum(tol[ok], 1e-300)).max()), np.argwhere(ok & (d > tol))[:5])
    if ok.any():
        off = float(np.linalg.norm(d[ok]) / max(np.linalg.norm(want[ok]), 1e-300))
        assert off < (4e-3 if bf16 else 1e-6), off
    return True


def how(hip, turns_dev, rot, half, gain_dev=None, eps=1e-5, magnitude=1.0):
    return C.byref(hip.pkg.Rotary(turns_dev, gain_dev, rot, half, magnitude, eps))
