"""Operators for serving from a paged cache: their cases, plain forms and 64-bit results.

A paged cache keeps keys as [pages][kv_heads][page][head_dim] and values transposed, as
[pages][kv_heads][head_dim][page], in bf16 or in e4m3 with one scale per kv head; a table
names the pages of every sequence in order.  The operators:

  append   projected rows to normalised and rotated queries and to keys and values in the pages:
           RMS norm with (weight + 1), rotary positions on one to three axes
  decode   attention of one new token a row over its sequence's pages, with an output gate or none
  prompt   causal attention of the last rows of packed sequences over their sequences' pages
  sample   tokens from logits: temperature, top-k, top-p, min-p and given uniform numbers

With `own` false run() computes them in elementary torch operations in 32 bits or more; with
`own` true it calls the library.  Sizes are the benchmark model's (16 query and 2 kv heads of 256,
rotary on 64 of them, gated outputs, vocabulary 151936) and generic ones.
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
F8 = torch.float8_e4m3fn
EPS = 1e-6
THETA = 1e7


def _package():
    """The package (its folder's name has a hyphen)."""
    if "rust_mlx_amd" not in sys.modules:
        path = os.path.join(_ROOT, "rust-mlx_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location("rust_mlx_amd", path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["rust_mlx_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["rust_mlx_amd"]


# ---- the cases ----------------------------------------------------------------------------
# heads, kv heads, head dim, gated: the benchmark model's and generic ones
_MODEL = {"heads": 16, "kv_heads": 2, "head_dim": 256, "gated": True}
_WIDE = {"heads": 32, "kv_heads": 8, "head_dim": 128, "gated": False}
_SEVEN = {"heads": 28, "kv_heads": 4, "head_dim": 128, "gated": False}
_SMALL = {"heads": 12, "kv_heads": 12, "head_dim": 64, "gated": False}
_GEOMETRIES = [_MODEL, _WIDE, _SEVEN, _SMALL, {"heads": 40, "kv_heads": 8, "head_dim": 128, "gated": True},
               {"heads": 64, "kv_heads": 4, "head_dim": 64, "gated": False}]


def listed():
    return [
        # eight users' next tokens enter the cache: the smallest call, launch and latency count
        dict(_MODEL, name="append_8_rows", kind="append", rows=8, context=300, rotary=64, axes=1, cache="bf16", page=16),
        # a prompt of text and pictures enters an 8-bit cache with time, height and width positions
        dict(_WIDE, name="append_4093_rows", kind="append", rows=4093, context=0, rotary=128, axes=3, cache="e4m3", page=64),
        # one user deep into a long document
        dict(_MODEL, name="decode_1_row", kind="decode", rows=1, context=60001, cache="bf16", page=64, lengths=1),
        # a full batch of the benchmark model, ragged contexts up to 4000
        dict(_MODEL, name="decode_8_rows", kind="decode", rows=8, context=4000, cache="bf16", page=16, lengths=2),
        # a large serving batch, ragged contexts up to 16384: the largest decode
        dict(_WIDE, name="decode_64_rows", kind="decode", rows=64, context=16384, cache="bf16", page=32, lengths=3),
        # an 8-bit cache and seven query heads to a kv head
        dict(_SEVEN, name="decode_40_rows_e4m3", kind="decode", rows=40, context=12001, cache="e4m3", page=128, lengths=4),
        # nine short prompts admitted together
        dict(_MODEL, name="prompt_9_short", kind="prompt", seqs=9, new=399, prior=0, cache="bf16", page=16, lengths=5),
        # a chunk of a long prompt: few queries on many cached keys
        dict(_MODEL, name="prompt_chunk", kind="prompt", seqs=1, new=512, prior=12001, cache="bf16", page=64, lengths=6),
        # packed prompts on cached prefixes of their own, 8-bit cache
        dict(_SEVEN, name="prompt_4_e4m3", kind="prompt", seqs=4, new=2047, prior=3001, cache="e4m3", page=32, lengths=7),
        # one long prompt from its start: the largest amount of matrix work
        dict(_WIDE, name="prompt_8192", kind="prompt", seqs=1, new=8192, prior=0, cache="bf16", page=64, lengths=8),
        # one user's next token with common settings
        dict(name="sample_1_row", kind="sample", rows=1, vocab=151936, settings="all"),
        # a batch where every request has its own settings
        dict(name="sample_64_rows", kind="sample", rows=64, vocab=151936, settings="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "prompt", "sample"])
    if kind == "sample":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 151936),
                "settings": rng.choice(["all", "mixed", "mixed", "none"])}
    case = dict(rng.choice(_GEOMETRIES), kind=kind, cache=rng.choice(["bf16", "bf16", "e4m3"]),
                page=rng.choice([16, 32, 64, 128]))
    if kind == "append":
        hd = case["head_dim"]
        return dict(case, rows=_log(rng, 1, 4093), context=_log(rng, 1, 1000), axes=rng.randint(1, 3),
                    rotary=rng.choice([hd, hd // 2, hd // 4]))
    case["lengths"] = rng.randrange(1000000)
    if kind == "decode":
        rows = _log(rng, 1, 64)
        most = min(60001, 64 * 16384 * 1024 // (rows * case["kv_heads"] * case["head_dim"]))
        return dict(case, rows=rows, context=_log(rng, 1, most))
    seqs, new = rng.randint(1, 9), _log(rng, 1, 4096)
    # queries x keys x heads stays below the largest listed prompt's
    room = 8192 * 8192 * 32 // 2 // (seqs * new * case["heads"])
    prior = rng.choice([0, _log(rng, 1, 30000)])
    return dict(case, seqs=seqs, new=min(new, room), prior=max(0, min(prior, room - new)))


def _new(case):
    """How many new rows each sequence of a prompt case has: the first the most, the others spread over the range."""
    rng = random.Random(case["lengths"])
    return [case["new"]] + [_log(rng, 1, case["new"]) for _ in range(case["seqs"] - 1)]


def _lengths(case):
    """Positions of each sequence in the cache, the new ones among them."""
    if case["kind"] == "append":
        return [case["context"] + case["rows"]] if case["rows"] > 64 else [case["context"] + 5 * r + 1 for r in range(case["rows"])]
    rng = random.Random(case["lengths"] + 1)
    if case["kind"] == "decode":
        return [case["context"]] + [rng.randint(1, case["context"]) for _ in range(case["rows"] - 1)]
    return [n + (case["prior"] if i == 0 else rng.randint(0, case["prior"])) for i, n in enumerate(_new(case))]


# ---- work ---------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (2 * case["vocab"] + 32), "flops": case["rows"] * case["vocab"]}
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    item = 2 if case["cache"] == "bf16" else 1
    if case["kind"] == "append":
        rows = case["rows"]
        read = rows * (h * (2 if case["gated"] else 1) * hd + 2 * kv * hd) * 2
        if case["gated"]:
            read -= rows * h * hd * 2  # the gate stays where it is
        return {"bytes": read + rows * h * hd * 2 + rows * 2 * kv * hd * item, "flops": rows * (h + kv) * hd * 8}
    lens = _lengths(case)
    new = _new(case) if case["kind"] == "prompt" else [1] * len(lens)
    q = sum(new) * h * hd * 2
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, lens))
    return {"bytes": q * (3 if case["gated"] else 2) + sum(lens) * 2 * kv * hd * item, "flops": 4 * pairs * h * hd}


# ---- inputs -------------------------------------------------------------------------------
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _normal(g, shape, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32 if dtype == F32 else BF16) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _pages(case, g):
    """The table of every sequence's pages, which lie scattered, and the number of pages of the cache."""
    page = case["page"]
    need = [-(-n // page) for n in _lengths(case)]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").to(I32)
    table = torch.full((len(need), max(need)), -1, dtype=I32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def _cache(case, g, pages):
    """Keys, values and their scales (none for bf16): what earlier steps have written."""
    kv, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    k, v = _normal(g, (pages, kv, page, hd)), _normal(g, (pages, kv, hd, page))
    if case["cache"] == "bf16":
        return k, v, None, None
    ks, vs = (torch.rand(kv, generator=g, device="cuda") * 0.01 + 0.01 for _ in range(2))
    shape = (1, kv, 1, 1)
    return (k / ks.view(shape)).clamp(-448, 448).to(F8), (v / vs.view(shape)).clamp(-448, 448).to(F8), ks, vs


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, g)
    h, kv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    table, pages = _pages(case, g)
    k, v, ks, vs = _cache(case, g, pages)
    s = {"case": case, "table": table, "k": k, "v": v, "k_scale": ks, "v_scale": vs, "page": case["page"], "pages": pages}
    if case["kind"] == "append":
        rows, axes, half = case["rows"], case["axes"], case["rotary"] // 2
        lens = _lengths(case)
        if rows > 64:  # one prompt: its rows in order
            s["seqs"] = _ints([0] * rows)
            pos = torch.arange(case["context"], case["context"] + rows, device="cuda", dtype=I32)
        else:  # the next token of `rows` users
            s["seqs"] = _ints(list(range(rows)))
            pos = _ints([n - 1 for n in lens])
        s["pos"] = pos
        # pictures: height and width run inside a picture while time stands
        side = torch.stack([pos, pos // 32 * 16 + pos // 8 % 4, pos // 32 * 16 + pos % 8])[:axes]
        s["rope_pos"] = side.contiguous()
        s["inv_freq"] = THETA ** (-torch.arange(half, device="cuda", dtype=F64) / half)
        s["pair_axis"] = [i % axes for i in range(half)]
        s["axis_index"] = torch.tensor(s["pair_axis"], device="cuda")
        s["qkv"] = _normal(g, (rows, (h * (2 if case["gated"] else 1) + 2 * kv) * hd), 1.7)
        s["q_norm"], s["k_norm"] = _normal(g, (hd,), 0.2), _normal(g, (hd,), 0.2)
        s["q_out"] = torch.empty((rows, h, hd), dtype=BF16, device="cuda")
        return s
    lens = _lengths(case)
    s["lens"] = _ints(lens)
    if case["kind"] == "prompt":
        new = _new(case)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        s["starts"], rows = _ints(starts), starts[-1]
        s["new"], s["longest"] = new, max(lens)
        # where a padded [sequences, longest new] layout has the packed rows
        s["at"] = torch.cat([torch.arange(n, device="cuda") + i * max(new) for i, n in enumerate(new)])
    else:
        rows = len(lens)
    s["q"] = _normal(g, (rows, h, hd), 1.2)
    if case["gated"]:
        s["qkv"] = _normal(g, (rows, (2 * h + 2 * kv) * hd))
    s["out"] = torch.zeros((rows, h, hd), dtype=BF16, device="cuda")
    return s


def _prepare_sample(case, g):
    rows, n = case["rows"], case["vocab"]
    logits = _normal(g, (rows, n), 2.5, F32)
    # the few likely tokens that a trained model has
    likely = torch.randint(0, n, (rows, 24), generator=g, device="cuda")
    logits.scatter_add_(1, likely, torch.rand((rows, 24), generator=g, device="cuda") * 14)
    pick = torch.rand((4, rows), generator=g, device="cuda")
    s = {"case": case, "logits": logits.to(BF16), "uniform": torch.rand(rows, generator=g, device="cuda")}
    if case["settings"] == "none":  # the whole distribution
        s["temperature"] = s["top_k"] = s["top_p"] = s["min_p"] = None
    elif case["settings"] == "all":
        s["temperature"] = torch.full((rows,), 0.7, device="cuda")
        s["top_k"] = torch.full((rows,), 20, dtype=I32, device="cuda")
        s["top_p"] = torch.full((rows,), 0.8, device="cuda")
        s["min_p"] = torch.full((rows,), 0.01, device="cuda")
    else:  # some rows without a filter, some greedy
        s["temperature"] = torch.where(pick[0] < 0.1, torch.zeros_like(pick[0]), 0.4 + pick[0])
        s["top_k"] = torch.where(pick[1] < 0.5, torch.zeros_like(pick[1]), pick[1] * 200).to(I32)
        s["top_p"] = torch.where(pick[2] < 0.3, torch.ones_like(pick[2]), 0.6 + 0.4 * pick[2])
        s["min_p"] = torch.where(pick[3] < 0.6, torch.zeros_like(pick[3]), 0.2 * pick[3])
    s["tokens"] = torch.empty(rows, dtype=I32, device="cuda")
    s["kept"] = torch.empty(rows, dtype=I32, device="cuda")
    s["logprob"] = torch.empty(rows, dtype=F32, device="cuda")
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt, "sample": _own_sample}[kind](state)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "sample": _plain_sample}[kind](state)


# ---- the library's calls --------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dims(s):
    """The description of the cache that a program keeps."""
    if "dims" not in s:
        mx, c = _package(), s["case"]
        page_elements = c["kv_heads"] * c["page"] * c["head_dim"]
        s["dims"] = mx.PageDimsC(c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["pages"], s["table"].shape[0],
                                 s["table"].shape[1], mx.MX_DT_BF16 if c["cache"] == "bf16" else mx.MX_DT_F8E4M3,
                                 int(c["gated"]), page_elements)
    return s["dims"]


def _own_append(s):
    mx, c = _package(), s["case"]
    if "rope" not in s:
        s["rope"] = mx.RopeAxesC(c["rotary"], c["axes"], s["inv_freq"].data_ptr())
        for i, a in enumerate(s["pair_axis"]):
            s["rope"].pair_axis[i] = a
    mx.check(mx.lib.mx_attn_paged_append(
        s["qkv"].data_ptr(), s["qkv"].shape[1], c["rows"], s["seqs"].data_ptr(), s["pos"].data_ptr(), s["rope_pos"].data_ptr(),
        ctypes.byref(s["rope"]), s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS, s["table"].data_ptr(),
        ctypes.byref(_dims(s)), _p(s["k_scale"]), _p(s["v_scale"]), s["q_out"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
        _stream()))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _workspace(s, size):
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(int(size), 1), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr()


def _gate(s):
    return (s["qkv"].data_ptr(), s["qkv"].shape[1]) if "qkv" in s else (None, 0)


def _own_decode(s):
    mx, c = _package(), s["case"]
    d = ctypes.byref(_dims(s))
    if "workspace" not in s:
        _workspace(s, mx.lib.mx_attn_paged_decode_workspace_bytes(c["rows"], d))
    mx.check(mx.lib.mx_attn_paged_decode(
        s["q"].data_ptr(), *_gate(s), c["rows"], None, s["lens"].data_ptr(), s["table"].data_ptr(), s["k"].data_ptr(),
        s["v"].data_ptr(), _p(s["k_scale"]), _p(s["v_scale"]), d, 0.0, s["workspace"].data_ptr(), s["out"].data_ptr(), _stream()))
    return {"out": s["out"]}


def _own_prompt(s):
    mx, rows = _package(), s["q"].shape[0]
    d = ctypes.byref(_dims(s))
    if "workspace" not in s:
        _workspace(s, mx.lib.mx_attn_paged_prefill_workspace_bytes(rows, d))
    mx.check(mx.lib.mx_attn_paged_prefill(
        s["q"].data_ptr(), *_gate(s), rows, s["starts"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(),
        s["k"].data_ptr(), s["v"].data_ptr(), _p(s["k_scale"]), _p(s["v_scale"]), d, 0.0, s["workspace"].data_ptr(),
        s["out"].data_ptr(), _stream()))
    return {"out": s["out"]}


def _own_sample(s):
    mx, c = _package(), s["case"]
    if "workspace" not in s:
        _workspace(s, mx.lib.mx_sample_workspace_bytes(c["rows"], c["vocab"]))
    mx.check(mx.lib.mx_sample_bf16(
        s["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"], _p(s["temperature"]), _p(s["top_k"]), _p(s["top_p"]),
        _p(s["min_p"]), s["uniform"].data_ptr(), s["tokens"].data_ptr(), s["logprob"].data_ptr(), s["kept"].data_ptr(),
        s["workspace"].data_ptr(), _stream()))
    return {"tokens": s["tokens"], "kept": s["kept"], "logprob": s["logprob"]}


# ---- the plain forms ------------------------------------------------------------------------
def _rotated(x, weight, cos, sin):
    """RMS norm with (weight + 1), then the first values' halves rotated: x [rows, heads, head_dim] in 32 bits."""
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (weight.float() + 1)
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_append(s):
    c = s["case"]
    rows, h, kv, hd = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float()
    wide = h * hd * (2 if c["gated"] else 1)
    q = x[:, :wide].reshape(rows, h, -1)[..., :hd]
    k = x[:, wide:wide + kv * hd].reshape(rows, kv, hd)
    v = x[:, wide + kv * hd:].reshape(rows, kv, hd)
    angle = s["rope_pos"][s["axis_index"]].t().double() * s["inv_freq"]  # far positions: in 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    s["q_out"].copy_(_rotated(q, s["q_norm"], cos, sin))
    k = _rotated(k, s["k_norm"], cos, sin)
    if s["k_scale"] is not None:
        k = (k / s["k_scale"][:, None]).clamp(-448, 448)
        v = (v / s["v_scale"][:, None]).clamp(-448, 448)
    pos = s["pos"].long()
    page, off = s["table"][s["seqs"].long(), pos // s["page"]].long(), pos % s["page"]
    raw = (lambda t: t.view(torch.uint8)) if s["k"].dtype == F8 else (lambda t: t)
    raw(s["k"])[page, :, off] = raw(k.to(s["k"].dtype))
    raw(s["v"])[page, :, :, off] = raw(v.to(s["v"].dtype))
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _rows_of(s):
    """Keys [sequences, kv, positions, head_dim] and values [sequences, kv, head_dim, positions] in 32 bits; the
    positions that a shorter sequence has no page for repeat the first page."""
    t = s["table"].clamp(min=0).long()
    raw = (lambda x: x.view(torch.uint8)[t].view(F8)) if s["k"].dtype == F8 else (lambda x: x[t])
    k, v = raw(s["k"]).float(), raw(s["v"]).float()
    n, p, kv, page, hd = k.shape
    k = k.permute(0, 2, 1, 3, 4).reshape(n, kv, p * page, hd)
    v = v.permute(0, 2, 3, 1, 4).reshape(n, kv, hd, p * page)
    if s["k_scale"] is not None:
        k *= s["k_scale"][:, None, None]
        v *= s["v_scale"][:, None, None]
    return k, v


def _gated(s, o):
    """o [rows, heads, head_dim] times the gate's logistic value, where there is one."""
    c = s["case"]
    if c["gated"]:
        h, hd = c["heads"], c["head_dim"]
        o = o * torch.sigmoid(s["qkv"][:, :2 * h * hd].reshape(-1, h, 2, hd)[:, :, 1].float())
    s["out"].copy_(o)
    return {"out": s["out"]}


def _softmax_(x):
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    return x


def _plain_decode(s):
    c = s["case"]
    rows, h, kv, hd = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    k, v = _rows_of(s)
    x = (s["q"].float() / math.sqrt(hd)).reshape(rows, kv, h // kv, hd) @ k.transpose(2, 3)
    past = torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None]
    x.masked_fill_(past[:, None, None], -math.inf)
    return _gated(s, (_softmax_(x) @ v.transpose(2, 3)).reshape(rows, h, hd))


def _plain_prompt(s):
    c = s["case"]
    n, h, kv, hd, m = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"], max(s["new"])
    k, v = _rows_of(s)
    q = torch.zeros((n * m, h, hd), device="cuda")
    q[s["at"]] = s["q"].float() / math.sqrt(hd)
    q = q.reshape(n, m, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, h // kv * m, hd)
    x = (q @ k.transpose(2, 3)).reshape(n, kv, h // kv, m, -1)
    new = s["starts"][1:] - s["starts"][:-1]
    limit = (s["lens"] - new)[:, None] + torch.arange(m, device="cuda")  # the last key that a row sees
    hidden = torch.arange(k.shape[2], device="cuda") > limit[..., None]
    x.masked_fill_(hidden[:, None, None], -math.inf)
    o = _softmax_(x).reshape(n, kv, h // kv * m, -1) @ v.transpose(2, 3)
    o = o.reshape(n, kv, h // kv, m, hd).permute(0, 3, 1, 2, 4).reshape(n * m, h, hd)
    return _gated(s, o[s["at"]])


def _plain_sample(s):
    rows, n = s["logits"].shape
    full = lambda t, v: torch.full((rows,), v, dtype=F64, device="cuda") if t is None else t.double()  # noqa: E731
    x, order = s["logits"].float().sort(dim=1, descending=True, stable=True)  # ties: the lowest index first
    t = full(s["temperature"], 1.0)
    greedy = t <= 0
    # long sums and values next to a border: in 64 bits
    w = ((x.double() - x[:, :1].double()) / torch.where(greedy, 1.0, t)[:, None]).exp()
    j = torch.arange(n, device="cuda")
    k = full(s["top_k"], 0.0)
    k = torch.where(k > 0, k, float(n))
    k = torch.where(greedy, 1.0, k)
    cum = w.cumsum(1)
    mass = cum.gather(1, k.clamp(max=n).long()[:, None] - 1)
    p = full(s["top_p"], 1.0)
    p = torch.where(p < 1, p, math.inf)  # from 1 on: no such filter
    keep = (j < k[:, None]) & ((cum - w < p[:, None] * mass) | (j == 0))
    keep &= (w >= full(s["min_p"], 0.0)[:, None]) & (w > 0) | (j == 0)
    kept = keep.long().cumprod(1).sum(1)
    mass = cum.gather(1, kept[:, None] - 1)
    u = s["uniform"].double()[:, None] * mass
    at = ((cum <= u) & (j < kept[:, None] - 1)).sum(1, keepdim=True)
    s["tokens"].copy_(order.gather(1, at)[:, 0])
    s["kept"].copy_(kept)
    s["logprob"].copy_((w.gather(1, at) / mass).log()[:, 0])
    return {"tokens": s["tokens"], "kept": s["kept"], "logprob": s["logprob"]}


# ---- the results in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_attention, "prompt": _exact_attention, "sample": _exact_sample}[case["kind"]](s)


def _stored(x, scale):
    """The value that the cache is to hold of x [kv, rows, head_dim], before it is rounded to the cache's type."""
    return x if scale is None else (x / scale.double()[:, None, None]).clamp(-448, 448)


def _exact_append(s):
    c = s["case"]
    h, kv, hd, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"]
    per = 2 * hd if c["gated"] else hd
    x = s["qkv"].double()
    # rotation of the pair (i, i + rot / 2) as a product of complex numbers
    turn = torch.polar(torch.ones((), dtype=F64, device="cuda"), s["rope_pos"].double()[s["axis_index"]].t() * s["inv_freq"])

    def head(first, weight):
        y = x[:, first:first + hd]
        y = y / (y.square().sum(1, keepdim=True) / hd + EPS).sqrt() * (1 + weight.double())
        z = torch.complex(y[:, :rot // 2].contiguous(), y[:, rot // 2:rot].contiguous()) * turn
        return torch.cat([z.real, z.imag, y[:, rot:]], 1)

    k_at, v_at = h * per, h * per + kv * hd
    q = torch.stack([head(i * per, s["q_norm"]) for i in range(h)], 1)
    k = torch.stack([head(k_at + i * hd, s["k_norm"]) for i in range(kv)])
    v = x[:, v_at:].reshape(-1, kv, hd).transpose(0, 1)
    page = s["page"]
    slot = s["table"].long()[s["seqs"].long(), (s["pos"] // page).long()] * page + s["pos"] % page
    flat = s["k"].double().transpose(1, 2).reshape(-1, kv, hd)
    flat[slot] = _stored(k, s["k_scale"]).transpose(0, 1)
    new_k = flat.reshape(-1, page, kv, hd).transpose(1, 2)
    flat = s["v"].double().permute(0, 3, 1, 2).reshape(-1, kv, hd)
    flat[slot] = _stored(v, s["v_scale"]).transpose(0, 1)
    return {"q": q, "k": new_k, "v": flat.reshape(-1, page, kv, hd).permute(0, 2, 3, 1)}


def _exact_attention(s):
    c = s["case"]
    h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lens = s["lens"].tolist()
    new = s.get("new") or [1] * len(lens)
    out, first = torch.zeros(s["q"].shape, dtype=F64, device="cuda"), 0
    for i, (n, total) in enumerate(zip(new, lens)):
        at = s["table"][i, :-(-total // page)].long()
        for g in range(kv):
            k = s["k"][at, g].double() if s["k"].dtype != F8 else s["k"].view(torch.uint8)[at, g].view(F8).double()
            v = s["v"][at, g].double() if s["v"].dtype != F8 else s["v"].view(torch.uint8)[at, g].view(F8).double()
            k, v = k.reshape(-1, hd)[:total], v.transpose(1, 2).reshape(-1, hd)[:total]
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
            for head in range(g * h // kv, (g + 1) * h // kv):
                x = s["q"][first:first + n, head].double() @ k.T * hd ** -0.5
                seen = torch.ones(x.shape, dtype=torch.bool, device="cuda").tril_(total - n)
                out[first:first + n, head] = torch.softmax(x.masked_fill_(~seen, -math.inf), 1) @ v
        first += n
    if c["gated"]:
        out *= 1 / (1 + torch.exp(-s["qkv"].double()[:, :2 * h * hd].reshape(-1, h, 2, hd)[:, :, 1]))
    return {"out": out}


def _exact_sample(s):
    """Row by row: tokens are whole numbers, so only the log-probability is compared in 64 bits."""
    value = lambda t, r, v: v if t is None else float(t[r])  # noqa: E731
    host = {n: None if s[n] is None else s[n].double().cpu() for n in ("temperature", "top_k", "top_p", "min_p", "uniform")}
    got = []
    for r in range(s["logits"].shape[0]):
        x = s["logits"][r].double()
        t, k = value(host["temperature"], r, 1.0), int(value(host["top_k"], r, 0))
        ids = torch.argsort(x, descending=True, stable=True)
        if t <= 0:
            got.append(0.0)
            continue
        p = torch.softmax(x / t, 0)[ids][:k if k > 0 else None]
        p = p / p.sum()
        before = torch.cat([p.new_zeros(1), p.cumsum(0)[:-1]])
        most = value(host["top_p"], r, 1.0)
        keep = (before < (most if most < 1 else math.inf)) & (p >= value(host["min_p"], r, 0.0) * p[0]) & (p > 0)
        keep[0] = True
        p = p[keep] / p[keep].sum()
        got.append(float(p[min(int((p.cumsum(0) <= float(host["uniform"][r])).sum()), len(p) - 1)].log()))
    return {"tokens": None, "kept": None, "logprob": torch.tensor(got, dtype=F64)}
