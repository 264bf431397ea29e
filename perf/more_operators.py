"""The operators of a batch of sequences over a paged cache that are timed: position rotation with the norm of each head,
keys and values into pages, and the attention of the batch's new rows over them, in plain form.

A pool is [pages, kv heads, page rows, head_dim] bf16, one for K and one for V.  Row p of a sequence lies in row
p % page rows of the page that its table names at p / page rows.  A batch is its sequences' new rows one behind the other,
"3@40 1@7": three rows behind 40 cached ones, one behind 7.  Rows are columns of a wider matrix q|k|v, fp32 or bf16.

Pair i of a head's first `rot` values, (2 i, 2 i + 1) or with `half` (i, i + rot / 2), turns by the angle
position theta^(-2 i / rot), divided by `factor` where a pair makes fewer than 1 turn in `original` rows, as it is from 32 on
and in between by the line through both; a norm divides a head by its root mean square first and multiplies by a gain per value.
Query r of a sequence, at position p, sees its rows p - window + 1 .. p (all up to p without a window).
"""
import ctypes
import importlib.util
import math
import os
import sys

import torch

own = False

HEADS, KV_HEADS, HEAD_DIM = 32, 8, 128
THETA, EPS = 1e6, 1e-5
LOW_TURNS, HIGH_TURNS = 1.0, 32.0


# ---- the cases ---------------------------------------------------------------------------------

def _model(**more):
    return {"heads": HEADS, "kv_heads": KV_HEADS, "head_dim": HEAD_DIM, **more}


def listed():
    return [
        # the queries of one decode step, as this model turns them: the smallest call
        _model(name="rotary_1row", kind="rotary", rows=1, pos=301, rot=128, half=False, norm=False, bf16=False, factor=1.0, original=0),
        # a long prompt's queries, normed per head, halves turned against each other
        _model(name="rotary_1531rows_norm", kind="rotary", rows=1531, pos=0, rot=128, half=True, norm=True, bf16=True, factor=1.0, original=0),
        # a sentence far into a stretched context, half of each head turned
        _model(name="rotary_226rows_far", kind="rotary", rows=226, pos=1000000, rot=64, half=False, norm=False, bf16=False, factor=8.0, original=32768),
        # one decode step of eight utterances
        _model(name="append_8x1row", kind="append", batch=" ".join("1@%d" % p for p in (301, 37, 226, 64, 150, 16, 299, 0)), page=16, rot=128, half=False, norm=False, bf16=False),
        # a long prompt's rows
        _model(name="append_1531rows_norm", kind="append", batch="1531@0", page=64, rot=128, half=True, norm=True, bf16=True),
        # a decode step near the end of the longest utterance
        _model(name="attend_1row_pos1999", kind="attend", batch="1@1999", page=16, window=0, bf16=False),
        # a decode step behind a book's worth of rows
        _model(name="attend_1row_pos65535", kind="attend", batch="1@65535", page=64, window=0, bf16=False),
        # a decode step of 64 utterances of every age
        _model(name="attend_64x1row", kind="attend", batch=" ".join("1@%d" % round(100 * 80 ** (i / 63)) for i in range(64)), page=16, window=0, bf16=True),
        # a sentence behind cached rows
        _model(name="attend_37rows_pos4000", kind="attend", batch="37@4000", page=32, window=0, bf16=False),
        # a long prompt's chunk beside decode steps of 31 others
        _model(name="attend_512rows_31x1row", kind="attend", batch="512@1500 " + " ".join("1@%d" % (211 * (i + 1) % 2000) for i in range(31)), page=16, window=0, bf16=True),
        # a long prompt from the start
        _model(name="attend_1531rows", kind="attend", batch="1531@0", page=64, window=0, bf16=False),
        # prompts of four lengths at once, one of them behind cached rows, within a window: the largest call
        _model(name="attend_prompts_window", kind="attend", batch="1531@0 700@0 226@0 2000@3000", page=64, window=2048, bf16=True),
    ]


# (heads, kv heads, head_dim): the model's, and others of the kinds that the attention takes
LAYOUTS = [(HEADS, KV_HEADS, HEAD_DIM), (HEADS, KV_HEADS, HEAD_DIM), (16, 16, 64), (8, 1, 128), (12, 4, 256), (14, 2, 64), (6, 2, 192)]
PAIRS = 1531 * 1531 * HEADS * HEAD_DIM // 2                # of a long prompt, times heads and values


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _drawn_batch(rng, wide, most_rows):
    """Decode steps, one chunk, or both, of no more pairs than a long prompt has and no more than `most_rows` rows in all."""
    mode = rng.choice(["decode", "decode", "chunk", "chunk", "mixed"])
    seqs = []
    if mode != "decode":
        rows = min(_log(rng, 2, 1400), most_rows // 2)
        most = min(60000, PAIRS // (rows * wide) - rows // 2, most_rows - rows)
        seqs.append((rows, 0 if most < 2 or rng.random() < 0.2 else _log(rng, 1, most)))
    if mode != "chunk":
        n = _log(rng, 1, 64 if mode == "decode" else 16)
        longest = max(2, most_rows // (2 * n) if mode == "decode" else min(2000, most_rows // (2 * n)))
        seqs += [(1, _log(rng, 1, longest)) for _ in range(n)]
    rng.shuffle(seqs)
    return " ".join("%d@%d" % s for s in seqs)


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "append", "append", "attend", "attend", "attend", "attend"])
    heads, kv_heads, head_dim = rng.choice(LAYOUTS)
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "bf16": rng.random() < 0.5}
    if kind != "attend":
        case |= {"rot": rng.choice([head_dim, head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)]), "half": rng.random() < 0.5, "norm": rng.random() < 0.5}
    if kind == "rotary":
        far = rng.random() < 0.5
        return case | {"rows": _log(rng, 1, 2000), "pos": _log(rng, 1, 2000000) if far else rng.randrange(4000),
                       "factor": rng.choice([4.0, 8.0, 32.0]) if far else 1.0, "original": 0 if far and rng.random() < 0.3 else _log(rng, 2048, 32768)}
    case["page"] = rng.choice([16, 16, 32, 64, 64, 256])
    if kind == "append":
        return case | {"batch": _drawn_batch(rng, heads * head_dim, 2500000 // (kv_heads * head_dim))}
    return case | {"batch": _drawn_batch(rng, heads * head_dim, 120000), "window": 0 if rng.random() < 0.7 else _log(rng, 16, 4096)}


def _sequences(case):
    """[(new rows, cached rows)] of a batch."""
    return [tuple(map(int, s.split("@"))) for s in case["batch"].split()]


# ---- the plain forms ---------------------------------------------------------------------------

def _turns(s, device):
    """Turns per position of each pair, in 64 bits."""
    f = THETA ** (-2.0 * torch.arange(s["rot"] // 2, dtype=torch.float64, device=device) / s["rot"]) / (2 * math.pi)
    keep = ((f * s.get("original", 0) - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)).clamp(0, 1)
    return f * (keep + (1 - keep) / s.get("factor", 1.0))


def _turn(s, x, positions):
    """[rows, heads, head_dim] -> the same in fp32, normed and turned."""
    x = x.float()
    if s["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["gain"]
    rot = s["rot"]
    t = positions.double().unsqueeze(-1) * s["turns"]
    angle = (t - torch.round(t)) * (2 * math.pi)
    c, n = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    if s["half"]:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat((a * c - b * n, a * n + b * c, x[..., rot:]), -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat((torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2), x[..., rot:]), -1)


def _attend(s):
    past, rows, first, pr = s["past"], s["new"], s["first"], s["page"]
    most_rows, most = s["most_rows"], s["most"]
    heads, kv_heads, group = s["heads"], s["kv_heads"], s["heads"] // s["kv_heads"]
    j = torch.arange(most, device=past.device)
    pages = s["tables"][:, j // pr]
    k = s["kp"][pages, :, j % pr].float().permute(0, 2, 3, 1).contiguous()     # [sequences, kv heads, head_dim, rows]
    v = s["vp"][pages, :, j % pr].float().transpose(1, 2).contiguous()
    i = torch.arange(most_rows, device=past.device)
    q = s["q"].float()[(first.unsqueeze(1) + i).clamp(max=s["q"].shape[0] - 1)]
    q = q.view(len(past), most_rows, kv_heads, group, -1).permute(0, 2, 3, 1, 4).reshape(len(past), kv_heads, group * most_rows, -1)
    w = ((q @ k) * s["scale"]).view(len(past), kv_heads, group, most_rows, most)
    here = past.unsqueeze(1) + i
    hidden = (j > here.unsqueeze(-1)) | (j >= (past + rows).view(-1, 1, 1))
    if s["window"]:
        hidden = hidden | (j <= here.unsqueeze(-1) - s["window"])
    w = w.masked_fill_(hidden.view(len(past), 1, 1, most_rows, most), -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = (w.view(len(past), kv_heads, group * most_rows, most) @ v).view(len(past), heads, most_rows, -1).transpose(1, 2)
    return o[i < rows.unsqueeze(1)].flatten(1).to(s["q"].dtype)


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


class _Batch:
    """The library's handle of a batch, freed with the state."""

    def __init__(self, s, seqs, tables):
        self.lib = _library()
        shape = _package().PagedShape(s["kp"].shape[0], s["page"], s["heads"], s["kv_heads"], s["head_dim"], s.get("window", 0))
        self.ptr = self.lib.tts_hip_paged_create(ctypes.byref(shape), len(seqs), sum(r for r, _ in seqs), tables.numel())
        if not self.ptr:
            _ok(-1)
        past = (ctypes.c_int * len(seqs))(*[p for _, p in seqs])
        rows = (ctypes.c_int * len(seqs))(*[r for r, _ in seqs])
        _ok(self.lib.tts_hip_paged_set(self.ptr, len(seqs), past, rows, tables.data_ptr(), tables.shape[1]))

    def __del__(self):
        if self.ptr:
            self.lib.tts_hip_paged_free(self.ptr)


def _normal(shape, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def _pool(s, seed):
    """Pages in the order in which a program that serves comes by them, every row filled: k and v ~N(0, 1)."""
    seqs, pr = _sequences(s), s["page"]
    need = [-(-(r + p) // pr) for r, p in seqs]
    pages = sum(need) + 3
    g = torch.Generator()
    g.manual_seed(seed)
    order = torch.randperm(pages, generator=g, dtype=torch.int32)
    tables = torch.zeros((len(seqs), max(need)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    shape = (pages, s["kv_heads"], pr, s["head_dim"])
    s["kp"], s["vp"] = _normal(shape, 8 * seed + 3).bfloat16(), _normal(shape, 8 * seed + 4).bfloat16()
    rows, past = (torch.tensor(x, dtype=torch.int64) for x in zip(*seqs))
    s["new"], s["past"], s["tables"] = rows.cuda(), past.cuda(), tables.long().cuda()
    s["first"] = (rows.cumsum(0) - rows).cuda()
    s["most_rows"], s["most"] = int(rows.max()), int((rows + past).max())
    s["rows"] = int(rows.sum())
    s["positions"] = torch.cat([torch.arange(p, p + r, dtype=torch.int32) for r, p in seqs]).cuda()
    s["row_page"] = torch.cat([tables[i, torch.arange(p, p + r) // pr] for i, (r, p) in enumerate(seqs)]).long().cuda()
    s["row_at"] = s["positions"].long() % pr
    return seqs, tables.contiguous()


def prepare(case, seed):
    s = dict(case)
    if s["kind"] == "rotary":
        s["positions"] = torch.arange(s["pos"], s["pos"] + s["rows"], dtype=torch.int32, device="cuda")
    else:
        seqs, tables = _pool(s, seed)
    hd = s["head_dim"]
    wide = (s["heads"] + 2 * s["kv_heads"]) * hd
    x = _normal((s["rows"], wide), 8 * seed + 1)
    s["x"] = x.bfloat16() if s["bf16"] else x
    s["q"], s["k"], s["v"] = s["x"].split((s["heads"] * hd, s["kv_heads"] * hd, s["kv_heads"] * hd), 1)
    if s["kind"] != "append":
        s["out"] = torch.empty((s["rows"], s["heads"] * hd), dtype=s["x"].dtype, device="cuda")
    if s["kind"] == "attend":
        s["scale"] = 1.0 / math.sqrt(hd)
    else:
        s["turns"] = _turns(s, "cuda")
        s["gain"] = 1 + 0.1 * _normal((hd,), 8 * seed + 2)
    if own:                                                # the library's context and its handles
        s["lib"] = _library()
        if s["kind"] != "attend":
            s["how"] = _package().Rotary(s["turns"].data_ptr(), s["gain"].data_ptr() if s["norm"] else None, s["rot"], int(s["half"]), 1.0, EPS)
            _ok(s["lib"].tts_hip_rotary_turns(s["turns"].data_ptr(), s["rot"], THETA, s.get("factor", 1.0), s.get("original", 0), LOW_TURNS, HIGH_TURNS))
        if s["kind"] != "rotary":
            s["handle"] = _Batch(s, seqs, tables)
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    lib, bf16, apart = s["lib"], int(s["bf16"]), s["x"].shape[1]
    if s["kind"] == "rotary":
        _ok(lib.tts_hip_rotary(s["out"].data_ptr(), s["q"].data_ptr(), bf16, s["rows"], s["heads"], s["head_dim"], 0, apart, s["positions"].data_ptr(), ctypes.byref(s["how"])))
        return s["out"]
    kp, vp = s["kp"].data_ptr(), s["vp"].data_ptr()
    if s["kind"] == "append":
        _ok(lib.tts_hip_paged_append(s["handle"].ptr, kp, vp, s["k"].data_ptr(), s["v"].data_ptr(), bf16, apart, ctypes.byref(s["how"])))
        return {"k": s["kp"], "v": s["vp"]}
    _ok(lib.tts_hip_paged_attention(s["out"].data_ptr(), s["q"].data_ptr(), bf16, apart, s["handle"].ptr, kp, vp, s["scale"]))
    return s["out"]


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "rotary":
        return _turn(s, s["q"].unflatten(1, (s["heads"], -1)), s["positions"]).flatten(1).to(s["x"].dtype)
    if s["kind"] == "append":
        s["kp"][s["row_page"], :, s["row_at"]] = _turn(s, s["k"].unflatten(1, (s["kv_heads"], -1)), s["positions"]).bfloat16()
        s["vp"][s["row_page"], :, s["row_at"]] = s["v"].unflatten(1, (s["kv_heads"], -1)).bfloat16()
        return {"k": s["kp"], "v": s["vp"]}
    return _attend(s)


# ---- what a pass cannot do without -------------------------------------------------------------

def _seen(rows, past, window):
    """(rows of the cache that somebody sees, pairs of a query and a row that it sees)."""
    if not window:
        return rows + past, rows * past + rows * (rows + 1) // 2
    grows = max(0, min(rows, window - past))               # queries that see everything up to themselves
    return min(rows + past, rows + window - 1), grows * past + grows * (grows + 1) // 2 + (rows - grows) * window


def work(case):
    c, size = case, 2 if case["bf16"] else 4
    if c["kind"] == "rotary":
        n = c["rows"] * c["heads"] * c["head_dim"]
        return {"bytes": 2 * size * n, "flops": (3 + 4 * c["norm"]) * n}
    seqs = _sequences(c)
    rows, row = sum(r for r, _ in seqs), c["kv_heads"] * c["head_dim"]
    if c["kind"] == "append":
        return {"bytes": 2 * rows * row * (size + 2), "flops": (3 + 4 * c["norm"]) * rows * row}
    seen = [_seen(r, p, c["window"]) for r, p in seqs]
    wide = c["heads"] * c["head_dim"]
    return {"bytes": 2 * size * rows * wide + 4 * row * sum(n for n, _ in seen), "flops": 4 * wide * sum(p for _, p in seen)}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _turned(s, x):
    """[rows, heads, head_dim] as complex pairs times e^(i angle)."""
    x = x.double()
    if s["norm"]:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * s["gain"].double()
    rot = s["rot"]
    freq = torch.exp(torch.arange(0, rot, 2, dtype=torch.float64, device=x.device) * (-math.log(THETA) / rot))
    if s.get("factor", 1.0) != 1.0:
        share = (s["original"] * freq / (2 * math.pi) - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)
        share = torch.minimum(torch.maximum(share, torch.zeros_like(share)), torch.ones_like(share))
        freq = (1 - share) * freq / s["factor"] + share * freq
    angle = s["positions"].double()[:, None, None] * freq
    pairs = x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if s["half"] else x[..., :rot].unflatten(-1, (rot // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
    x[..., :rot] = (z.transpose(-1, -2) if s["half"] else z).flatten(-2)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    hd = s["head_dim"]
    if s["kind"] == "rotary":
        return _turned(s, s["q"].reshape(s["rows"], -1, hd)).view(s["rows"], -1)
    if s["kind"] == "append":
        k, v = s["kp"].double(), s["vp"].double()
        k[s["row_page"], :, s["row_at"]] = _turned(s, s["k"].reshape(s["rows"], -1, hd))
        v[s["row_page"], :, s["row_at"]] = s["v"].reshape(s["rows"], -1, hd).double()
        return {"k": k, "v": v}
    out = torch.empty((s["rows"], s["heads"], hd), dtype=torch.float64, device="cuda")
    q = s["q"].reshape(s["rows"], -1, hd)
    group, at = s["heads"] // s["kv_heads"], 0
    for i, (rows, past) in enumerate(_sequences(case)):
        pages = s["tables"][i, :-(-(rows + past) // s["page"])]
        age = torch.arange(past, past + rows, device="cuda")[:, None] - torch.arange(past + rows, device="cuda")[None, :]
        unseen = (age < 0) | (age >= s["window"]) if s["window"] else age < 0
        for h in range(s["kv_heads"]):
            k = s["kp"][pages, h].reshape(-1, hd)[:rows + past].double()
            v = s["vp"][pages, h].reshape(-1, hd)[:rows + past].double()
            for g in range(h * group, (h + 1) * group):
                scores = (q[at:at + rows, g].double() @ k.T * s["scale"]).masked_fill(unseen, -math.inf)
                out[at:at + rows, g] = torch.softmax(scores, -1) @ v
        at += rows
    return out.view(s["rows"], -1)
