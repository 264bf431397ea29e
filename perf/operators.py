"""The 4-bit operators that are timed: quantisation to microscaled e2m1 (MXFP4), linear layers with weights held that
way, and the key/value cache in 4 bits with the attention that reads it.

A block of 32 consecutive values of a row shares a scale 2^(s - 127), s = floor(log2 of its largest magnitude) - 2 + 127
as a byte; a value is one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times that scale and a sign: the nearest one, of two equally near
ones that with the even code.  A matrix [rows, cols] is codes [rows, 64 p] and scales [rows, 4 p] with p = cols / 128
rounded up: two codes a byte, the first in its low half, zeros behind the last column.  A cache is codes
[kv heads, max rows, head_dim / 2] and scales [kv heads, max rows, head_dim / 32], for K and for V.

What `prepare` makes is the same for the plain forms and for the library: the bytes that a program holds.  What is in
4 bits comes back as the values it stands for, through the calls that a program reads them with.
"""
import ctypes
import importlib.util
import math
import os
import sys

import torch

own = False

DIM, KV_DIM, FFN = 3072, 1024, 9216
HEADS, KV_HEADS, HEAD_DIM = 32, 8, 128
VOCAB, SEM_ROWS = 131072, 8320


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # a short prompt's activations with a width that ends inside a block: the smallest call
        {"name": "quantize_37x1000", "kind": "quantize", "rows": 37, "cols": 1000, "bf16": False, "gap": 24},
        # the gate projection of a layer at upload, from the checkpoint's bf16
        {"name": "quantize_gate_bf16", "kind": "quantize", "rows": FFN, "cols": DIM, "bf16": True, "gap": 0},
        # one token through the gate projection: the product of a decode step
        {"name": "linear_1row", "kind": "linear", "rows": 1, "n": FFN, "k": DIM},
        # one token against the output head over the vocabulary
        {"name": "linear_1row_vocab", "kind": "linear", "rows": 1, "n": VOCAB, "k": DIM},
        # a usual prompt (voice rows and a sentence) through the down projection
        {"name": "linear_226rows_down", "kind": "linear", "rows": 226, "n": DIM, "k": FFN},
        # a long prompt (long voice sample and a page of text) through the gate projection
        {"name": "linear_1531rows", "kind": "linear", "rows": 1531, "n": FFN, "k": DIM},
        # the row of one decode step
        {"name": "append_1row", "kind": "append", "rows": 1, "pos": 301, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
        # the rows of a long prompt
        {"name": "append_1531rows", "kind": "append", "rows": 1531, "pos": 0, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
        # a decode step near the end of the longest utterance
        {"name": "attend_1row_pos1999", "kind": "attend", "rows": 1, "pos": 1999, "heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
        # a decode step behind a book's worth of rows: what a cache of 4 bits is for
        {"name": "attend_1row_pos65535", "kind": "attend", "rows": 1, "pos": 65535, "heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
        # a sentence behind cached rows
        {"name": "attend_37rows_pos4000", "kind": "attend", "rows": 37, "pos": 4000, "heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
        # a long prompt from the start
        {"name": "attend_1531rows", "kind": "attend", "rows": 1531, "pos": 0, "heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM},
    ]


# (out, in) of the model's matrices: projections of a layer, the semantic head, the latent's, the vocabulary's
MATRICES = [(FFN, DIM), (DIM, FFN), (4096, DIM), (KV_DIM, DIM), (DIM, 4096), (SEM_ROWS, DIM), (DIM, 36), (36, DIM)]
# (heads, kv heads, head_dim): the model's, and others of the kinds that the attention takes
LAYOUTS = [(HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (16, 16, 64), (8, 1, 128), (12, 4, 256), (14, 2, 64), (6, 2, 192)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "append", "attend", "attend", "attend"])
    if kind == "quantize":
        rows, cols = _log(rng, 1, 8192), _log(rng, 1, 12288)
        return {"kind": kind, "rows": min(rows, FFN * DIM // cols), "cols": cols, "bf16": rng.random() < 0.5, "gap": rng.choice([0, 0, 5, 64])}
    if kind == "linear":
        n, k = rng.choice(MATRICES) if rng.random() < 0.6 else (_log(rng, 1, 20000), _log(rng, 1, 12288))
        return {"kind": kind, "rows": min(_log(rng, 1, 1500), 1500 * FFN * DIM // (n * k)), "n": n, "k": k}
    heads, kv_heads, head_dim = rng.choice(LAYOUTS)
    if kind == "append":
        return {"kind": kind, "rows": _log(rng, 1, 1500), "pos": rng.randrange(4000), "kv_heads": kv_heads, "head_dim": head_dim}
    rows = 1 if rng.random() < 0.4 else _log(rng, 2, 1400)
    most = min(60000, 1531 * 1531 * HEADS * HEAD_DIM // (2 * rows * heads * head_dim) - rows // 2)   # no more pairs than the longest prompt's
    return {"kind": kind, "rows": rows, "pos": 0 if most < 2 or rng.random() < 0.2 else _log(rng, 1, most), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim}


# ---- the plain forms ---------------------------------------------------------------------------

def _panels(cols):
    return (cols + 127) // 128


def _quantize(x):
    """[..., 32 n] -> codes [..., 16 n], scales [..., n]; finite values."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(top)[1] - 3                            # top = f 2^e', f in [0.5, 1)
    e = torch.where(top > 0, e.clamp(min=-127), -127)
    q = torch.ldexp(torch.ldexp(b, -(e // 2)), -(e - e // 2))   # in two steps: either factor is a normal number
    a = q.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)) + 8 * torch.signbit(b)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8).squeeze(-1)


def _dequantize(codes, scales):
    """codes [..., 16 n], scales [..., n] -> fp32 [..., 32 n]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2).unflatten(-1, (-1, 32))
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).flatten(-2)


def _quantize_matrix(x):
    return _quantize(torch.nn.functional.pad(x.float(), (0, 128 * _panels(x.shape[-1]) - x.shape[-1])))


def _visible(rows, pos, device):
    return torch.arange(pos + rows, device=device) <= torch.arange(pos, pos + rows, device=device).unsqueeze(1)


def _attend(s):
    rows, pos, group = s["rows"], s["pos"], s["heads"] // s["kv_heads"]
    n = pos + rows
    k = _dequantize(s["kc"][:, :n], s["ks"][:, :n])
    v = _dequantize(s["vc"][:, :n], s["vs"][:, :n])
    q = s["q"].view(rows, s["kv_heads"], group, s["head_dim"]).permute(1, 2, 0, 3).reshape(s["kv_heads"], group * rows, s["head_dim"])
    w = (q @ k.transpose(1, 2)) * s["scale"]
    w = w.view(s["kv_heads"], group, rows, n).masked_fill(~_visible(rows, pos, w.device), -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = w.view(s["kv_heads"], group * rows, n) @ v
    return o.view(s["kv_heads"], group, rows, s["head_dim"]).permute(2, 0, 1, 3).reshape(rows, -1)


# ---- what a program has in hand ----------------------------------------------------------------

_held = {}


def _package():
    """The library's Python mirror (its folder's name is no identifier)."""
    name = "voxtral_tts_c_amd"
    if name not in sys.modules:
        folder = os.path.abspath("voxtral-tts.c_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def _library():
    if "lib" not in _held:
        lib = _package().lib()
        if lib.tts_hip_init(64):
            raise RuntimeError(lib.tts_hip_last_error().decode())
        _held["lib"] = lib
    return _held["lib"]


def _ok(status):
    if status:
        raise RuntimeError(_library().tts_hip_last_error().decode())


def _normal(shape, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * std


def _cache(s, seed, held, max_rows):
    """A cache of `max_rows` rows, the first `held` of them filled: k and v ~N(0, 1)."""
    h, d = s["kv_heads"], s["head_dim"]
    for which in "kv":
        codes = torch.zeros((h, max_rows, d // 2), dtype=torch.uint8, device="cuda")
        scales = torch.zeros((h, max_rows, d // 32), dtype=torch.uint8, device="cuda")
        if held:
            codes[:, :held], scales[:, :held] = _quantize(_normal((h, held, d), 8 * seed + (3 if which == "k" else 4)))
        s[which + "c"], s[which + "s"] = codes, scales


def prepare(case, seed):
    s = dict(case)
    kind = s["kind"]
    rows = s["rows"]
    if kind == "quantize":
        wide = _normal((rows, s["cols"] + s["gap"]), seed, 0.02 if s["bf16"] else 1.0)
        s["wide"] = wide.bfloat16() if s["bf16"] else wide
        s["x"] = s["wide"][:, :s["cols"]]                  # columns of a wider matrix where there is a gap
        p = _panels(s["cols"])
        s["codes"] = torch.empty((rows, 64 * p), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty((rows, 4 * p), dtype=torch.uint8, device="cuda")
        s["y"] = torch.empty((rows, s["cols"]), device="cuda")
    elif kind == "linear":
        s["codes"], s["scales"] = _quantize_matrix(_normal((s["n"], s["k"]), 8 * seed + 1, 0.02))
        s["x"] = _normal((rows, s["k"]), 8 * seed + 2)
        s["y"] = torch.empty((rows, s["n"]), device="cuda")
    elif kind == "append":
        _cache(s, seed, s["pos"], s["pos"] + rows + 100)
        width = s["kv_heads"] * s["head_dim"]
        s["k"], s["v"] = _normal((rows, width), 8 * seed + 1), _normal((rows, width), 8 * seed + 2)
        s["k_out"], s["v_out"] = torch.empty((rows, width), device="cuda"), torch.empty((rows, width), device="cuda")
    else:
        _cache(s, seed, s["pos"] + rows, s["pos"] + rows + 100)
        s["q"] = _normal((rows, s["heads"] * s["head_dim"]), 8 * seed + 1)
        s["scale"] = 1.0 / math.sqrt(s["head_dim"])
        s["out"] = torch.empty((rows, s["heads"] * s["head_dim"]), device="cuda")
    if own:                                                # the handle: the library's context, the cache's description
        s["lib"] = _library()
        if "kc" in s:
            s["cache"] = _package().Kv4(s["kc"].data_ptr(), s["ks"].data_ptr(), s["vc"].data_ptr(), s["vs"].data_ptr(), s["kc"].shape[1], s["kv_heads"], s["head_dim"])
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    kind, lib = s["kind"], s["lib"]
    if kind == "quantize":
        codes, scales = s["codes"].data_ptr(), s["scales"].data_ptr()
        _ok(lib.tts_hip_mx4_quantize(codes, scales, s["x"].data_ptr(), int(s["bf16"]), s["rows"], s["cols"], s["cols"] + s["gap"]))
        _ok(lib.tts_hip_mx4_dequantize(s["y"].data_ptr(), codes, scales, s["rows"], s["cols"], s["cols"]))
        return s["y"]
    if kind == "linear":
        _ok(lib.tts_hip_linear_mx4(s["y"].data_ptr(), s["x"].data_ptr(), s["codes"].data_ptr(), s["scales"].data_ptr(), s["rows"], s["k"], s["n"]))
        return s["y"]
    cache = ctypes.byref(s["cache"])
    if kind == "append":
        _ok(lib.tts_hip_kv4_append(cache, s["k"].data_ptr(), s["v"].data_ptr(), s["rows"], s["pos"], 0))
        _ok(lib.tts_hip_kv4_read(s["k_out"].data_ptr(), s["v_out"].data_ptr(), cache, s["rows"], s["pos"], 0))
        return {"k": s["k_out"], "v": s["v_out"]}
    _ok(lib.tts_hip_kv4_attention(s["out"].data_ptr(), s["q"].data_ptr(), cache, s["rows"], s["pos"], s["heads"], s["scale"]))
    return s["out"]


def run(s):
    if own:
        return _run_own(s)
    kind = s["kind"]
    if kind == "quantize":
        return _dequantize(*_quantize_matrix(s["x"]))[:, :s["cols"]]
    if kind == "linear":
        return s["x"] @ _dequantize(s["codes"], s["scales"])[:, :s["k"]].T
    if kind == "append":
        to = slice(s["pos"], s["pos"] + s["rows"])
        out = {}
        for which in "kv":
            x = s[which].view(s["rows"], s["kv_heads"], s["head_dim"]).transpose(0, 1)
            s[which + "c"][:, to], s[which + "s"][:, to] = _quantize(x)
            out[which] = _dequantize(s[which + "c"][:, to], s[which + "s"][:, to]).transpose(0, 1).reshape(s["rows"], -1)
        return out
    return _attend(s)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    c, rows = case, case["rows"]
    if c["kind"] == "quantize":
        n = rows * c["cols"]                               # values in, codes and scales, values out
        return {"bytes": n * (2 if c["bf16"] else 4) + n * 17 // 32 + 4 * n, "flops": 4 * n}
    if c["kind"] == "linear":
        return {"bytes": c["n"] * c["k"] * 17 // 32 + 4 * rows * (c["n"] + c["k"]), "flops": 2 * rows * c["n"] * c["k"]}
    row = c["kv_heads"] * c["head_dim"]
    if c["kind"] == "append":
        return {"bytes": 2 * rows * (4 * row + row * 17 // 32 + 4 * row), "flops": 8 * rows * row}
    n = c["pos"] + rows
    wide = c["heads"] * c["head_dim"]
    return {"bytes": 8 * rows * wide + 2 * n * row * 17 // 32, "flops": 4 * wide * (rows * c["pos"] + rows * (rows + 1) // 2)}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _rounded(x):
    """What a row's 4-bit form stands for: blocks of 32, the last one as long as it is."""
    x = x.double()
    cols = x.shape[-1]
    x = torch.cat((x, x.new_zeros(x.shape[:-1] + (-cols % 32,))), -1)
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    largest = blocks.abs().max(-1, keepdim=True).values
    unit = torch.exp2(torch.floor(torch.log2(largest.clamp(min=2.0 ** -125))) - 2)
    m = blocks / unit
    step = torch.exp2(torch.floor(torch.log2(m.abs().clamp(min=1.0))) - 1)
    return ((torch.round(m / step) * step).clamp(-6, 6) * unit).reshape(x.shape)[..., :cols]


def _meaning(codes, scales):
    """What bytes stand for: sign, two bits of exponent and one of mantissa each."""
    c = torch.stack((codes.int() % 16, codes.int() // 16), -1).reshape(codes.shape[:-1] + (-1,))
    e, m = (c // 2) % 4, (c % 2).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1)) * (1 - 2 * (c // 8).double())
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "quantize":
        return _rounded(s["x"])
    if kind == "linear":
        return s["x"].double() @ _meaning(s["codes"], s["scales"])[:, :s["k"]].T
    if kind == "append":
        h, d = s["kv_heads"], s["head_dim"]
        return {which: _rounded(s[which].view(-1, h, d)).view(-1, h * d) for which in "kv"}
    rows, pos, group = s["rows"], s["pos"], s["heads"] // s["kv_heads"]
    q = s["q"].double().view(rows, s["heads"], s["head_dim"])
    out = torch.empty_like(q)
    here = torch.arange(pos, pos + rows, device=q.device)[:, None]
    hidden = torch.arange(pos + rows, device=q.device)[None, :] > here
    for h in range(s["heads"]):
        k = _meaning(s["kc"][h // group, :pos + rows], s["ks"][h // group, :pos + rows])
        v = _meaning(s["vc"][h // group, :pos + rows], s["vs"][h // group, :pos + rows])
        w = torch.softmax((q[:, h] @ k.T * s["scale"]).masked_fill(hidden, -math.inf), -1)
        out[:, h] = w @ v
    return out.view(rows, -1)
