"""mx_logits_control_bf16 against the same steps in numpy's fp32, bit for bit: every step is one IEEE operation
(products are not fused), and the result is rounded once, to the nearest bf16 (ties to even)."""
import ctypes as C

import numpy as np
import pytest

from paged_ref import bf

pytestmark = pytest.mark.gpu

INF = np.float32(np.inf)


def say(*a):
    print(*a, flush=True)


def rounded(x):
    """fp32 -> bf16 bits with infinities; NaN as one pattern."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), 0x7FC0, r)


def reference(logits, n, tokens, prompt_lens, lens, seqs, rep, freq, pres, bias, masks, mask_rows, before):
    out = before.copy()
    f = np.float32
    with np.errstate(all="ignore"):
        for r in range(len(logits)):
            x = bf(logits[r, :n]).astype(f)
            if tokens is not None:
                s = r if seqs is None else seqs[r]
                if not 0 <= s < len(tokens):
                    continue
                length = min(max(lens[s], 0), tokens.shape[1])
                mid = min(max(prompt_lens[s], 0), length) if prompt_lens is not None else 0
                count = lambda t: np.bincount(t[(t >= 0) & (t < n)], minlength=n)  # noqa: E731
                said = count(tokens[s, mid:length])
                seen = said + count(tokens[s, :mid]) > 0
                if rep is not None and rep[r] > 0 and np.isfinite(rep[r]):
                    x = np.where(seen, np.where(x < 0, x * rep[r], x / rep[r]), x)
                if freq is not None and np.isfinite(freq[r]):
                    x = np.where(seen, x - freq[r] * said.astype(f), x)
                if pres is not None and np.isfinite(pres[r]):
                    x = np.where(said > 0, x - pres[r], x)
            if bias is not None:
                last = dict(zip(bias[1][bias[0][r]:bias[0][r + 1]], bias[2][bias[0][r]:bias[0][r + 1]]))
                for t, v in last.items():
                    if 0 <= t < n:
                        x[t] += v
            if masks is not None:
                state = r if mask_rows is None else mask_rows[r]
                if 0 <= state < len(masks):
                    j = np.arange(n)
                    x = np.where(masks[state][j // 32] >> (j % 32).astype(np.uint32) & 1, x, -INF)
            out[r, :n] = rounded(x)
    return out


def run(mx, logits, n, out, in_place=False, offset=0, **k):
    """k: the arrays by their names in the description (absent: NULL), and the sizes."""
    up = lambda a: None if a is None else mx.DeviceArray.from_numpy(np.ascontiguousarray(a))  # noqa: E731
    dev = {name: up(k.get(name)) for name in ("tokens", "prompt_lens", "lens", "seqs", "repetition", "frequency", "presence",
                                              "bias_starts", "bias_tokens", "bias_values", "masks", "mask_rows")}
    size = lambda name, axis: 0 if k.get(name) is None else k[name].shape[axis]  # noqa: E731
    c = mx.LogitsControlsC(tokens_stride=size("tokens", 1) if k.get("tokens") is not None else 0,
                           sequences=size("tokens", 0), bias_count=size("bias_tokens", 0),
                           mask_stride=size("masks", 1) if k.get("masks") is not None else 0, mask_states=size("masks", 0),
                           **{name: a.ptr if a is not None else None for name, a in dev.items()})
    dl = up(logits)
    do = dl if in_place else up(out)
    mx.check(mx.lib.mx_logits_control_bf16(dl.ptr + 2 * offset, logits.shape[1], len(logits), n, C.byref(c),
                                           do.ptr + 2 * offset, do.shape[1], None))
    mx.sync()
    return do.numpy()


def make(rng, rows, n, stride, history, sequences, biases, states):
    k = {}
    logits = rounded(3 * rng.standard_normal((rows, stride)).astype(np.float32)).astype(np.uint16)
    if history:
        k["tokens"] = np.minimum(n * rng.random((sequences, history)) ** 3, n - 1).astype(np.int32)
        k["tokens"][:, ::7] = rng.integers(-5, n + 5, k["tokens"][:, ::7].shape)  # some of no token
        k["lens"] = rng.integers(0, history + 1, sequences).astype(np.int32)
        k["prompt_lens"] = rng.integers(-3, history + 1, sequences).astype(np.int32)
        k["seqs"] = rng.integers(-1, sequences + 1, rows).astype(np.int32)
        k["repetition"] = rng.uniform(0.7, 1.6, rows).astype(np.float32)
        k["frequency"] = rng.uniform(-0.5, 1, rows).astype(np.float32)
        k["presence"] = rng.uniform(-1, 1, rows).astype(np.float32)
    if biases:
        counts = rng.integers(0, biases + 1, rows)
        k["bias_starts"] = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        k["bias_tokens"] = rng.integers(-2, n + 2, max(counts.sum(), 1)).astype(np.int32)
        k["bias_tokens"][1::5] = k["bias_tokens"][0::5][:len(k["bias_tokens"][1::5])]  # some twice
        k["bias_values"] = rng.normal(0, 4, len(k["bias_tokens"])).astype(np.float32)
        k["bias_values"][::11] = -np.inf
    if states:
        k["masks"] = rng.integers(0, 2 ** 32, (states, (n + 31) // 32 + 1)).astype(np.uint32)
        k["mask_rows"] = rng.integers(-1, states + 1, rows).astype(np.int32)
    return logits, k


def check(got, logits, n, before, k):
    bias = (k["bias_starts"], k["bias_tokens"], k["bias_values"]) if "bias_starts" in k else None
    want = reference(logits, n, k.get("tokens"), k.get("prompt_lens"), k.get("lens"), k.get("seqs"), k.get("repetition"),
                     k.get("frequency"), k.get("presence"), bias, k.get("masks"), k.get("mask_rows"), before)
    nan = np.isnan(bf(got)) & np.isnan(bf(want))
    assert ((got == want) | nan).all(), np.argwhere((got != want) & ~nan)[:5]


@pytest.mark.parametrize("rows,n,history,biases,states", [
    (1, 1, 1, 1, 1), (3, 7, 20, 3, 2), (2, 2047, 100, 0, 0), (5, 2048, 0, 40, 0), (4, 2049, 300, 9, 3), (1, 151936, 1000, 0, 0),
    (9, 32001, 5000, 300, 2), (64, 50257, 777, 20, 64), (130, 4097, 64, 5, 1), (300, 4096, 33, 0, 2), (6, 40000, 0, 0, 3)])
def test_against_the_same_steps(mx, rows, n, history, biases, states):
    say("controls", rows, n, history, biases, states)
    rng = np.random.default_rng(rows + n)
    for stride, offset in ((n, 0), (n + 3, 0), (n + 16, 1)):
        logits, k = make(rng, rows, n, stride, history, max(1, rows // 2 + 1), biases, states)
        if offset:  # rows that begin at no multiple of anything
            logits = np.concatenate([logits, logits[:1]])
            view = np.ascontiguousarray(logits.ravel()[offset:offset + rows * stride].reshape(rows, stride))
        else:
            view = logits
        before = np.full((rows + (offset > 0), stride), 0x1234, np.uint16)
        got = run(mx, logits[:rows + (offset > 0)] if not offset else logits, n, before, offset=offset, **k) \
            if not offset else None
        if offset:
            whole = run_offset(mx, logits, rows, n, before, offset, k)
            got = whole.ravel()[offset:offset + rows * stride].reshape(rows, stride)
            assert whole.ravel()[0] == 0x1234
        check(got, view, n, np.full((rows, stride), 0x1234, np.uint16), k)
        if not offset:
            check(run(mx, logits, n, None, in_place=True, **k), logits, n, logits, k)


def run_offset(mx, logits, rows, n, before, offset, k):
    """Rows of a buffer from element `offset` on."""
    up = lambda a: mx.DeviceArray.from_numpy(np.ascontiguousarray(a))  # noqa: E731
    dev = {name: up(a) for name, a in k.items()}
    size = lambda name, axis: k[name].shape[axis] if name in k else 0  # noqa: E731
    c = mx.LogitsControlsC(tokens_stride=size("tokens", 1), sequences=size("tokens", 0), bias_count=size("bias_tokens", 0),
                           mask_stride=size("masks", 1), mask_states=size("masks", 0),
                           **{name: a.ptr for name, a in dev.items()})
    dl, do = up(logits), up(before)
    mx.check(mx.lib.mx_logits_control_bf16(dl.ptr + 2 * offset, logits.shape[1], rows, n, C.byref(c), do.ptr + 2 * offset,
                                           before.shape[1], None))
    mx.sync()
    return do.numpy()


def test_values_that_switch_parts_off_and_special_logits(mx):
    say("special")
    n, rng = 300, np.random.default_rng(1)
    off = np.array([0, -1, np.nan, np.inf, 1, 1, 1, 1], np.float32)
    wild = np.array([0, 0.5, np.nan, np.inf, -np.inf, 0.5, -0.5, 0.25], np.float32)
    logits, k = make(rng, 8, n, n, 50, 8, 6, 1)
    k.update(seqs=None, repetition=off, frequency=wild, presence=wild[::-1].copy())
    del k["seqs"]
    logits[:, ::9], logits[:, 1::9], logits[:, 2::9] = 0x7F80, 0xFF80, 0x7FC0  # +inf, -inf, NaN
    logits[:, 3::9], logits[:, 4::9] = 0x8000, 0
    check(run(mx, logits, n, np.full_like(logits, 0x1234), **k), logits, n, np.full_like(logits, 0x1234), k)
    check(run(mx, logits, n, None, in_place=True, **k), logits, n, logits, k)


def test_a_row_without_an_allowed_token_and_the_sampler(mx):
    """Nothing allowed: all -inf, from which the sampler draws token 0 with nothing kept."""
    say("nothing allowed")
    n, up = 1000, mx.DeviceArray.from_numpy
    logits = rounded(np.random.default_rng(2).standard_normal((2, n)).astype(np.float32)).astype(np.uint16)
    masks = np.zeros((2, 32), np.uint32)
    masks[1, 20] = 1 << 5
    got = run(mx, logits, n, np.zeros_like(logits), masks=masks)
    assert (got[0] == 0xFF80).all() and (got[1] == 0xFF80).sum() == n - 1 and got[1, 645] == logits[1, 645]
    dl, u, tok, kept = up(got), up(np.array([0.5, 0.5], np.float32)), mx.DeviceArray((2,), np.uint32), \
        mx.DeviceArray((2,), np.int32)
    ws = mx.DeviceArray((mx.lib.mx_sample_workspace_bytes(2, n),), np.uint8)
    mx.check(mx.lib.mx_sample_bf16(dl.ptr, n, 2, n, None, None, None, None, u.ptr, tok.ptr, None, kept.ptr, ws.ptr, None))
    mx.sync()
    assert tok.numpy().tolist() == [0, 645] and kept.numpy().tolist() == [0, 1]


def test_the_same_bits_whatever_the_history_order(mx):
    """Counts are whole numbers: a shuffled history, and thousands of one token, change nothing."""
    say("order")
    n, rng = 20000, np.random.default_rng(3)
    logits, k = make(rng, 4, n, n, 6000, 4, 50, 0)
    k["tokens"][:, :3000] = 17
    k["seqs"], k["lens"][:], k["prompt_lens"][:] = np.arange(4, dtype=np.int32), 6000, 0
    first = run(mx, logits, n, np.zeros_like(logits), **k)
    k["tokens"] = k["tokens"][:, rng.permutation(6000)]
    assert (run(mx, logits, n, np.zeros_like(logits), **k) == first).all()
    check(first, logits, n, np.zeros_like(logits), k)


@pytest.mark.parametrize("rows,n", [(5, 3001), (40, 40000)])
def test_whole_histories_of_every_stride(mx, rows, n):
    """Histories that fill their row, reach past it (cut), end a token before it or are empty, of lengths around the
    reads of a workgroup, with more biases a row than it has threads."""
    rng = np.random.default_rng(33)
    for stride in (1, 2, 3, 4, 5, 1023, 1025, 2048, 2051, 4096, 4099, 8195, 20000):
        say("histories", rows, n, stride)
        logits, k = make(rng, rows, n, n, stride, rows, 900, 2)
        k["lens"] = np.array([stride, stride + 9, stride - 1, 0, -4], np.int32)[np.arange(rows) % 5]
        k["seqs"] = rng.permutation(rows).astype(np.int32)
        before = np.full((rows, n), 0x1234, np.uint16)
        check(run(mx, logits, n, before, **k), logits, n, before, k)
