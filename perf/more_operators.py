"""Operators for serving from a latent cache and for steering what is sampled: their cases, plain forms and 64-bit results.

A latent cache keeps one vector a position for all heads, as [pages][page][latent + rope]: a latent
of 512 (or 256) values, from which every head's keys and values follow by products, and a rotary key
of 64 that the heads share.  It is bf16, or e4m3 with one scale a position, formed as it is written.
The operators:

  append    projected rows to latents and rotary keys in the pages, and rotated queries
  read      positions of sequences from the pages to packed rows in bf16
  decode    attention of one new token a row over the latents themselves: queries have each head's
            key product in them, and its value product follows the result
  prompt    causal attention of the last rows of packed sequences, whose keys and values have been
            formed from the latents for every head
  controls  penalties for repeated tokens, biases and masks on logits before sampling

With `own` false run() computes them in elementary torch operations in 32 bits or more; with
`own` true it calls the library.  Sizes are generic ones and the benchmark model's vocabulary of
151936.
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
THETA = 1e4
ROPE = 64
LEAST = 2.0 ** -100  # a position's largest value counts at least so much for its scale


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
_FULL = {"latent": 512, "nope": 128}
_HALF = {"latent": 256, "nope": 64}


def listed():
    return [
        # eight users' next tokens enter the cache: the smallest call, launch and latency count
        dict(_FULL, name="append_8_rows", kind="append", rows=8, context=300, heads=128, cache="bf16", page=64),
        # a prompt enters an 8-bit cache
        dict(_FULL, name="append_4093_rows_e4m3", kind="append", rows=4093, context=0, heads=20, cache="e4m3", page=64),
        # the cached prefixes of nine short prompts, whose keys and values are to be formed
        dict(_FULL, name="read_9_short", kind="read", seqs=9, context=399, cache="bf16", page=16, lengths=1),
        # a long document's prefix from an 8-bit cache
        dict(_FULL, name="read_60001_e4m3", kind="read", seqs=1, context=60001, cache="e4m3", page=64, lengths=2),
        # one user deep into a long document; an eighth of the heads, as one of eight devices has them
        dict(_FULL, name="decode_1_row", kind="decode", rows=1, context=60001, heads=16, cache="bf16", page=64, lengths=3),
        # a large serving batch with all heads, ragged contexts up to 8192: the largest decode
        dict(_FULL, name="decode_64_rows", kind="decode", rows=64, context=8192, heads=128, cache="bf16", page=64, lengths=4),
        # an 8-bit cache and an odd number of heads
        dict(_FULL, name="decode_40_rows_e4m3", kind="decode", rows=40, context=12001, heads=20, cache="e4m3", page=128, lengths=5),
        # nine short prompts admitted together
        dict(_FULL, name="prompt_9_short", kind="prompt", seqs=9, new=399, prior=0, heads=20, lengths=6),
        # a chunk of a long prompt: few queries on many keys
        dict(_FULL, name="prompt_chunk", kind="prompt", seqs=1, new=512, prior=12001, heads=20, lengths=7),
        # one long prompt from its start: the largest amount of matrix work
        dict(_FULL, name="prompt_8192", kind="prompt", seqs=1, new=8192, prior=0, heads=32, lengths=8),
        # one user's next token with the usual penalties
        dict(name="controls_1_row", kind="controls", rows=1, vocab=151936, history=1000, biases=0, masks=False, lengths=9),
        # a batch of long requests, some bound to a grammar, some with biases
        dict(name="controls_64_rows", kind="controls", rows=64, vocab=151936, history=8192, biases=300, masks=True, lengths=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt", "controls"])
    if kind == "controls":
        return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": _log(rng, 1000, 151936), "history": _log(rng, 1, 8192),
                "biases": rng.choice([0, _log(rng, 1, 300)]), "masks": rng.random() < 0.5, "lengths": rng.randrange(1000000)}
    case = dict(rng.choice([_FULL, _FULL, _FULL, _HALF]), kind=kind, lengths=rng.randrange(1000000))
    if kind == "prompt":
        heads = rng.choice([5, 8, 20, 32, 64, 128])
        seqs, new = rng.randint(1, 9), _log(rng, 1, 4096)
        # queries x keys x heads, and the keys and values of all heads, stay below the largest listed prompt's
        room = min(8192 * 8192 * 32 // 2 // (seqs * new * heads), 8192 * 32 // (seqs * heads))
        prior = rng.choice([0, _log(rng, 1, 12001)])
        new = max(1, min(new, room))
        return dict(case, heads=heads, seqs=seqs, new=new, prior=max(0, min(prior, room - new)))
    case.update(cache=rng.choice(["bf16", "bf16", "e4m3"]), page=rng.choice([16, 32, 64, 128]))
    if kind == "append":
        heads = rng.choice([5, 8, 20, 40, 128])
        return dict(case, heads=heads, rows=_log(rng, 1, 4093 * 20 // max(heads, 20)), context=_log(rng, 1, 1000))
    if kind == "read":
        seqs = rng.randint(1, 9)
        return dict(case, seqs=seqs, context=_log(rng, 1, 60001 // seqs))
    rows, heads = _log(rng, 1, 64), rng.choice([1, 8, 16, 20, 32, 40, 64, 100, 128])
    return dict(case, rows=rows, heads=heads, context=_log(rng, 1, min(60001, 64 * 8192 // rows)))


def _new(case):
    """How many new rows each sequence of a prompt case has: the first the most, the others spread over the range."""
    rng = random.Random(case["lengths"])
    return [case["new"]] + [_log(rng, 1, case["new"]) for _ in range(case["seqs"] - 1)]


def _lengths(case):
    """Positions of each sequence, the new ones among them; of controls the tokens of each row's history."""
    kind = case["kind"]
    if kind == "append":
        return [case["context"] + case["rows"]] if case["rows"] > 64 else [case["context"] + 5 * r + 1 for r in range(case["rows"])]
    rng = random.Random(case["lengths"] + 1)
    if kind == "prompt":
        return [n + (case["prior"] if i == 0 else rng.randint(0, case["prior"])) for i, n in enumerate(_new(case))]
    most = case["history"] if kind == "controls" else case["context"]
    return [most] + [rng.randint(1, most) for _ in range(case["seqs" if kind == "read" else "rows"] - 1)]


# ---- work ---------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "controls":
        rows, n = case["rows"], case["vocab"]
        masked = len(range(0, rows, 2)) if case["masks"] else 0
        return {"bytes": rows * (4 * n + 8 * case["biases"] + 16) + masked * n // 8 + 4 * sum(_lengths(case)),
                "flops": rows * n}
    wide, nope = case["latent"] + ROPE, case["nope"]
    if kind == "prompt":
        h, new, lens = case["heads"], _new(case), _lengths(case)
        pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, lens))
        return {"bytes": 2 * (sum(new) * h * (2 * nope + ROPE) + sum(lens) * (h * 2 * nope + ROPE)),
                "flops": 2 * pairs * h * (2 * nope + ROPE)}
    stored = 2 * wide if case["cache"] == "bf16" else wide + 4  # a position in the cache
    if kind == "append":
        rows, h = case["rows"], case["heads"]
        return {"bytes": rows * (2 * wide + stored + 4 * h * ROPE), "flops": rows * (8 * wide + 6 * h * ROPE)}
    if kind == "read":
        return {"bytes": sum(_lengths(case)) * (stored + 2 * wide), "flops": sum(_lengths(case)) * wide}
    rows, h, keys = case["rows"], case["heads"], sum(_lengths(case))
    return {"bytes": keys * stored + 2 * rows * h * (wide + case["latent"]), "flops": 2 * keys * h * (wide + case["latent"])}


# ---- inputs -------------------------------------------------------------------------------
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=BF16) * scale


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _cache(case, g):
    """The cache that earlier steps have written, and the table of every sequence's pages, which lie scattered."""
    page, wide = case["page"], case["latent"] + ROPE
    need = [-(-n // page) for n in _lengths(case)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(I32)
    table = torch.full((len(need), max(need)), -1, dtype=I32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    x = _normal(g, (pages, page, wide))
    s = {"case": case, "table": table, "pages": pages, "cache": x, "scale": None}
    if case["cache"] == "e4m3":
        s["scale"] = x.float().abs().amax(-1) / 448
        s["cache"] = (x.float() / s["scale"][..., None]).clamp(-448, 448).to(F8)
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "controls":
        return _prepare_controls(case, g)
    if kind == "prompt":
        return _prepare_prompt(case, g)
    s, lens = _cache(case, g), _lengths(case)
    latent, wide = case["latent"], case["latent"] + ROPE
    if kind == "append":
        rows, h = case["rows"], case["heads"]
        if rows > 64:  # one prompt: its rows in order
            s["seqs"] = _ints([0] * rows)
            pos = torch.arange(case["context"], case["context"] + rows, device="cuda", dtype=I32)
        else:  # the next token of `rows` users
            s["seqs"] = _ints(list(range(rows)))
            pos = _ints([n - 1 for n in lens])
        s["pos"], s["rope_pos"] = pos, pos[None].contiguous()
        s["inv_freq"] = THETA ** (-torch.arange(ROPE // 2, device="cuda", dtype=F64) / (ROPE // 2))
        s["x"] = _normal(g, (rows, wide), 1.7)
        s["q"] = _normal(g, (rows, h, case["nope"] + ROPE), 1.2)
        s["norm"] = _normal(g, (latent,), 0.2)
        s["q_rope"] = torch.empty((rows, h, ROPE), dtype=BF16, device="cuda")
        return s
    if kind == "read":
        starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
        s["starts"], s["rows"] = _ints(starts), starts[-1]
        s["latent"] = torch.empty((starts[-1], latent), dtype=BF16, device="cuda")
        s["rope"] = torch.empty((starts[-1], ROPE), dtype=BF16, device="cuda")
        return s
    rows, h = case["rows"], case["heads"]
    s["lens"], s["most"] = _ints(lens), max(lens)
    # the key product of unit keys spreads a query of `nope` values over the latent
    s["q_latent"] = _normal(g, (rows, h, latent), 1.2 * math.sqrt(case["nope"] / latent))
    s["q_rope"] = _normal(g, (rows, h, ROPE), 1.2)
    s["out"] = torch.zeros((rows, h, latent), dtype=BF16, device="cuda")
    s["factor"] = 1 / math.sqrt(case["nope"] + ROPE)
    return s


def _prepare_prompt(case, g):
    h, nope, new, lens = case["heads"], case["nope"], _new(case), _lengths(case)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    kv_starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    return {"case": case, "new": new, "lens": lens, "starts": _ints(starts), "kv_starts": _ints(kv_starts),
            "q": _normal(g, (starts[-1], h, nope + ROPE), 1.2), "q_rope": _normal(g, (starts[-1], h, ROPE), 1.2),
            "kv": _normal(g, (kv_starts[-1], h, 2 * nope)), "k_rope": _normal(g, (kv_starts[-1], ROPE)),
            "out": torch.zeros((starts[-1], h, nope), dtype=BF16, device="cuda"), "factor": 1 / math.sqrt(nope + ROPE)}


def _prepare_controls(case, g):
    rows, n, lens = case["rows"], case["vocab"], _lengths(case)
    logits = _normal(g, (rows, n), 2.5)
    # texts repeat their few frequent tokens
    rank = torch.rand((rows, case["history"]), generator=g, device="cuda", dtype=F64)
    s = {"case": case, "logits": logits, "tokens": (n ** rank).to(torch.int64).clamp(max=n).to(I32) - 1,
         "lens": _ints(lens), "out": torch.empty_like(logits)}
    pick = torch.rand((4, rows), generator=g, device="cuda")
    s["prompt_lens"] = (s["lens"] * pick[0]).to(I32)
    s["repetition"], s["frequency"], s["presence"] = 1 + 0.3 * pick[1], 0.5 * pick[2], pick[3] - 0.2
    s["bias_starts"] = s["bias_tokens"] = s["bias_values"] = s["masks"] = s["mask_rows"] = None
    if case["biases"]:
        k = min(case["biases"], n)
        s["bias_starts"] = _ints([k * r for r in range(rows + 1)])
        # different tokens within a row
        spread = torch.rand((rows, n), generator=g, device="cuda").argsort(1)[:, :k]
        s["bias_tokens"] = spread.reshape(-1).to(I32).contiguous()
        s["bias_values"] = torch.randn(rows * k, generator=g, device="cuda") * 5
    if case["masks"]:  # every second row, of 32 tokens a word
        words, states = (n + 31) // 32, (rows + 1) // 2
        s["masks"] = torch.randint(-2 ** 31, 2 ** 31, (states, words), generator=g, device="cuda").to(I32)
        s["mask_rows"] = _ints([r // 2 if r % 2 == 0 else -1 for r in range(rows)])
    return s


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "read": _own_read, "decode": _own_decode, "prompt": _own_prompt,
                "controls": _own_controls}[kind](state)
    return {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "prompt": _plain_prompt,
            "controls": _plain_controls}[kind](state)


# ---- the library's calls --------------------------------------------------------------------
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dims(s):
    """The description of the cache that a program keeps."""
    if "dims" not in s:
        mx, c = _package(), s["case"]
        s["dims"] = mx.LatentDimsC(c.get("heads", 1), c["nope"], c["nope"], c["latent"], ROPE, c["page"], s["pages"],
                                   s["table"].shape[0], s["table"].shape[1],
                                   mx.MX_DT_BF16 if c["cache"] == "bf16" else mx.MX_DT_F8E4M3,
                                   c["page"] * (c["latent"] + ROPE))
    return ctypes.byref(s["dims"])


def _own_append(s):
    mx, c = _package(), s["case"]
    if "axes" not in s:
        s["axes"] = mx.RopeAxesC(ROPE, 1, s["inv_freq"].data_ptr())
    mx.check(mx.lib.mx_attn_latent_append(
        s["x"].data_ptr(), s["x"].shape[1], s["q"].data_ptr(), c["heads"] * (c["nope"] + ROPE), c["rows"],
        s["seqs"].data_ptr(), s["pos"].data_ptr(), s["rope_pos"].data_ptr(), ctypes.byref(s["axes"]), s["norm"].data_ptr(),
        EPS, s["table"].data_ptr(), _dims(s), s["q_rope"].data_ptr(), s["cache"].data_ptr(), _p(s["scale"]), _stream()))
    return _appended(s)


def _own_read(s):
    mx = _package()
    mx.check(mx.lib.mx_attn_latent_read(
        s["cache"].data_ptr(), _p(s["scale"]), s["rows"], s["starts"].data_ptr(), None, s["table"].data_ptr(), _dims(s),
        s["latent"].data_ptr(), s["latent"].shape[1], s["rope"].data_ptr(), ROPE, _stream()))
    return {"latent": s["latent"], "rope": s["rope"]}


def _workspace(s, size):
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(int(size), 1), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr()


def _own_decode(s):
    mx, rows = _package(), s["case"]["rows"]
    d = _dims(s)
    if "workspace" not in s:
        _workspace(s, mx.lib.mx_attn_latent_decode_workspace_bytes(rows, d))
    mx.check(mx.lib.mx_attn_latent_decode(
        s["q_latent"].data_ptr(), s["q_rope"].data_ptr(), rows, None, s["lens"].data_ptr(), s["table"].data_ptr(),
        s["cache"].data_ptr(), _p(s["scale"]), d, s["factor"], s["workspace"].data_ptr(), s["out"].data_ptr(), _stream()))
    return {"out": s["out"]}


def _own_prompt(s):
    mx, c = _package(), s["case"]
    rows, kv_rows = s["q"].shape[0], s["kv"].shape[0]
    if "dims" not in s:
        s["dims"] = mx.LatentDimsC(c["heads"], c["nope"], c["nope"], c["latent"], ROPE, 16, 1, c["seqs"], 1, mx.MX_DT_BF16,
                                   16 * (c["latent"] + ROPE))
    d = ctypes.byref(s["dims"])
    if "workspace" not in s:
        _workspace(s, mx.lib.mx_attn_latent_prefill_workspace_bytes(rows, kv_rows, d))
    mx.check(mx.lib.mx_attn_latent_prefill(
        s["q"].data_ptr(), c["heads"] * (c["nope"] + ROPE), s["q_rope"].data_ptr(), rows, s["starts"].data_ptr(),
        s["kv"].data_ptr(), c["heads"] * 2 * c["nope"], s["k_rope"].data_ptr(), ROPE, kv_rows, s["kv_starts"].data_ptr(),
        d, s["factor"], s["workspace"].data_ptr(), s["out"].data_ptr(), _stream()))
    return {"out": s["out"]}


def _own_controls(s):
    mx, c = _package(), s["case"]
    if "controls" not in s:  # the description that a program keeps
        states, words = (0, 0) if s["masks"] is None else s["masks"].shape
        s["controls"] = mx.LogitsControlsC(
            tokens=s["tokens"].data_ptr(), tokens_stride=s["tokens"].shape[1], prompt_lens=s["prompt_lens"].data_ptr(),
            lens=s["lens"].data_ptr(), sequences=c["rows"], repetition=s["repetition"].data_ptr(),
            frequency=s["frequency"].data_ptr(), presence=s["presence"].data_ptr(), bias_starts=_p(s["bias_starts"]),
            bias_tokens=_p(s["bias_tokens"]), bias_values=_p(s["bias_values"]),
            bias_count=0 if s["bias_tokens"] is None else s["bias_tokens"].shape[0], masks=_p(s["masks"]),
            mask_rows=_p(s["mask_rows"]), mask_stride=words, mask_states=states)
    mx.check(mx.lib.mx_logits_control_bf16(s["logits"].data_ptr(), c["vocab"], c["rows"], c["vocab"],
                                           ctypes.byref(s["controls"]), s["out"].data_ptr(), c["vocab"], _stream()))
    return {"logits": s["out"]}


# ---- the plain forms ------------------------------------------------------------------------
def _appended(s):
    return {"q_rope": s["q_rope"], "cache": s["cache"], **({} if s["scale"] is None else {"scale": s["scale"]})}


def _turned(x, cos, sin):
    a, b = x[..., :ROPE // 2], x[..., ROPE // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _raw(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


def _plain_append(s):
    c = s["case"]
    x, latent = s["x"].float(), c["latent"]
    angle = s["rope_pos"][0].double()[:, None] * s["inv_freq"]  # far positions: in 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    s["q_rope"].copy_(_turned(s["q"][..., c["nope"]:].float(), cos[:, None], sin[:, None]))
    y = x[:, :latent]
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * (s["norm"].float() + 1)
    y = torch.cat([y, _turned(x[:, latent:], cos, sin)], -1)
    pos = s["pos"].long()
    page, off = s["table"][s["seqs"].long(), pos // c["page"]].long(), pos % c["page"]
    if s["scale"] is not None:
        scale = y.abs().amax(-1).clamp(min=LEAST) / 448
        s["scale"][page, off] = scale
        y = (y / scale[:, None]).clamp(-448, 448)
    _raw(s["cache"])[page, off] = _raw(y.to(s["cache"].dtype))
    return _appended(s)


def _positions(s, i, n):
    """The first n positions of sequence i in 32 bits."""
    at = s["table"][i, :-(-n // s["case"]["page"])].long()
    x = _raw(s["cache"])[at].view(s["cache"].dtype).float()
    if s["scale"] is not None:
        x = x * s["scale"][at][..., None]
    return x.flatten(0, 1)[:n]


def _plain_read(s):
    latent, at = s["case"]["latent"], 0
    for i, n in enumerate(_lengths(s["case"])):
        x = _positions(s, i, n)
        s["latent"][at:at + n] = x[:, :latent]
        s["rope"][at:at + n] = x[:, latent:]
        at += n
    return {"latent": s["latent"], "rope": s["rope"]}


def _softmax_(x):
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    x /= x.sum(-1, keepdim=True)
    return x


def _plain_decode(s):
    c, t = s["case"], s["table"].clamp(min=0).long()
    k = _raw(s["cache"])[t].view(s["cache"].dtype).float()  # a shorter sequence's missing pages repeat the first one
    if s["scale"] is not None:
        k *= s["scale"][t][..., None]
    k = k.flatten(1, 2)
    x = torch.cat([s["q_latent"], s["q_rope"]], -1).float() * s["factor"] @ k.transpose(1, 2)
    past = torch.arange(k.shape[1], device="cuda") >= s["lens"][:, None]
    s["out"].copy_(_softmax_(x.masked_fill_(past[:, None], -math.inf)) @ k[..., :c["latent"]])
    return {"out": s["out"]}


def _plain_prompt(s):
    nope, at, kv_at = s["case"]["nope"], 0, 0
    for n, t in zip(s["new"], s["lens"]):
        q = torch.cat([s["q"][at:at + n, :, :nope], s["q_rope"][at:at + n]], -1).float().transpose(0, 1) * s["factor"]
        kv = s["kv"][kv_at:kv_at + t].float().transpose(0, 1)
        k = torch.cat([kv[..., :nope], s["k_rope"][kv_at:kv_at + t].float().expand(kv.shape[0], t, ROPE)], -1)
        x = q @ k.transpose(1, 2)
        hidden = torch.arange(t, device="cuda") > torch.arange(t - n, t, device="cuda")[:, None]
        s["out"][at:at + n] = (_softmax_(x.masked_fill_(hidden, -math.inf)) @ kv[..., nope:]).transpose(0, 1)
        at, kv_at = at + n, kv_at + t
    return {"out": s["out"]}


def _plain_controls(s):
    c = s["case"]
    rows, n = c["rows"], c["vocab"]
    x = s["logits"].float()
    j = torch.arange(s["tokens"].shape[1], device="cuda")
    said = (j >= s["prompt_lens"][:, None]) & (j < s["lens"][:, None])  # the row's own output
    read = j < s["prompt_lens"][:, None]
    row = torch.arange(rows, device="cuda")[:, None]
    at = (row * n + s["tokens"])
    count = torch.bincount(at[said], minlength=rows * n).reshape(rows, n)
    seen = (torch.bincount(at[read], minlength=rows * n).reshape(rows, n) + count) > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x < 0, x * rep, x / rep), x)
    x = x - s["frequency"][:, None] * count
    x = x - s["presence"][:, None] * (count > 0)
    if s["bias_starts"] is not None:
        of = torch.repeat_interleave(torch.arange(rows, device="cuda"), s["bias_starts"].diff(),
                                     output_size=s["bias_tokens"].shape[0])
        x[of, s["bias_tokens"].long()] += s["bias_values"]
    if s["masks"] is not None:
        token = torch.arange(n, device="cuda")
        bits = (s["masks"][s["mask_rows"].clamp(min=0).long()][:, token // 32] >> (token % 32)) & 1
        x = x.masked_fill((bits == 0) & (s["mask_rows"] >= 0)[:, None], -math.inf)
    s["out"].copy_(x)
    return {"logits": s["out"]}


# ---- the results in 64 bits -------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "decode": _exact_decode, "prompt": _exact_prompt,
            "controls": _exact_controls}[case["kind"]](s)


def _values(s):
    """What the cache stands for, [pages, page, latent + rope]."""
    x = s["cache"].double()
    return x if s["scale"] is None else x * s["scale"].double()[..., None]


def _exact_append(s):
    c, latent, half = s["case"], s["case"]["latent"], ROPE // 2
    # rotation of the pair (i, i + half) as a product of complex numbers
    turn = torch.polar(torch.ones((), dtype=F64, device="cuda"), s["pos"].double()[:, None] * s["inv_freq"])

    def rotated(v):
        z = torch.complex(v[:, :half].contiguous(), v[:, half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], 1)

    x = s["x"].double()
    y = x[:, :latent]
    y = y / (y.square().sum(1, keepdim=True) / latent + EPS).sqrt() * (1 + s["norm"].double())
    y = torch.cat([y, rotated(x[:, latent:])], 1)
    slot = s["table"].long()[s["seqs"].long(), (s["pos"] // c["page"]).long()] * c["page"] + s["pos"] % c["page"]
    got = {"q_rope": torch.stack([rotated(s["q"][:, h, c["nope"]:].double()) for h in range(c["heads"])], 1)}
    flat = s["cache"].double().flatten(0, 1)
    if s["scale"] is not None:
        scale = y.abs().max(1).values.clamp(min=LEAST) / 448
        y = y / scale[:, None]
        scales = s["scale"].double().flatten()
        scales[slot] = scale
        got["scale"] = scales.reshape(s["scale"].shape)
    flat[slot] = y
    return dict(got, cache=flat.reshape(s["cache"].shape))


def _exact_read(s):
    c, x = s["case"], _values(s).flatten(0, 1)
    slots = [s["table"][i, p // c["page"]].long() * c["page"] + p % c["page"]
             for i, p in enumerate(torch.arange(n, device="cuda") for n in _lengths(c))]
    y = x[torch.cat(slots)]
    return {"latent": y[:, :c["latent"]], "rope": y[:, c["latent"]:]}


def _exact_decode(s):
    c, x, out = s["case"], _values(s).flatten(0, 1), torch.zeros(s["out"].shape, dtype=F64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        p = torch.arange(n, device="cuda")
        k = x[s["table"][r, p // c["page"]].long() * c["page"] + p % c["page"]]
        y = s["q_latent"][r].double() @ k[:, :c["latent"]].T + s["q_rope"][r].double() @ k[:, c["latent"]:].T
        out[r] = torch.softmax(y * s["factor"], 1) @ k[:, :c["latent"]]
    return {"out": out}


def _exact_prompt(s):
    nope, out = s["case"]["nope"], torch.zeros(s["out"].shape, dtype=F64, device="cuda")
    first, kv_first = s["starts"].tolist(), s["kv_starts"].tolist()
    for i, (n, t) in enumerate(zip(s["new"], s["lens"])):
        mine, keys = slice(first[i], first[i] + n), slice(kv_first[i], kv_first[i] + t)
        seen = torch.ones((n, t), dtype=torch.bool, device="cuda").tril_(t - n)
        for h in range(s["case"]["heads"]):
            x = s["q"][mine, h, :nope].double() @ s["kv"][keys, h, :nope].double().T
            x += s["q_rope"][mine, h].double() @ s["k_rope"][keys].double().T
            x = torch.softmax((x * s["factor"]).masked_fill_(~seen, -math.inf), 1)
            out[mine, h] = x @ s["kv"][keys, h, nope:].double()
    return {"out": out}


def _exact_controls(s):
    """Row by row, over the tokens that occur in it."""
    out = s["logits"].double()
    for r in range(out.shape[0]):
        mid, n = int(s["prompt_lens"][r]), int(s["lens"][r])
        rep, freq, pres = (float(s[k][r]) for k in ("repetition", "frequency", "presence"))
        every = s["tokens"][r, :n].unique().long()
        out[r, every] = torch.where(out[r, every] < 0, out[r, every] * rep, out[r, every] / rep)
        ids, counts = s["tokens"][r, mid:n].unique(return_counts=True)
        out[r, ids.long()] -= freq * counts.double() + pres
        if s["bias_starts"] is not None:
            mine = slice(int(s["bias_starts"][r]), int(s["bias_starts"][r + 1]))
            out[r, s["bias_tokens"][mine].long()] += s["bias_values"][mine].double()
        if s["masks"] is not None and int(s["mask_rows"][r]) >= 0:
            words = s["masks"][int(s["mask_rows"][r])]
            allowed = torch.stack([(words >> b) & 1 for b in range(32)], 1).flatten()[:out.shape[1]]
            out[r, allowed == 0] = -math.inf
    return {"logits": out}
