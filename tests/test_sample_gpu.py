"""mx_sample_bf16 against the definition in 64 bits, tokens and counts equal: every
filter alone and together, ties, vocabularies of one to a million tokens at any
alignment, rows of one value (more equal tokens than a 16-bit counter holds),
masks of -inf and of the lowest value, infinities, NaN, greedy rows.

A token can only differ where u times the kept mass lies within the sums' 64-bit
rounding (2^-53 times their length, under 2^-33) of a prefix mass, or top-p's
target does: random inputs miss that, and where borders are meant to be hit, the
masses are exact.  logprob: an fp32 rounding (2^-24) of a 64-bit value."""
import ctypes as C

import numpy as np
import pytest

from paged_ref import Graph, bf, to_bf

pytestmark = pytest.mark.gpu


def reference(row, t, k, p, mp, u):
    """(token, kept, logprob) by sorting."""
    x = bf(row).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    x = x[order]
    if x[0] == -np.inf:
        return 0, 0, -np.inf
    if not t > 0:
        return int(order[0]), 1, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x[0], 1.0, np.exp((x - x[0]) / np.float64(t)))
    w = np.where(np.isnan(w) | (x == -np.inf), 0.0, w)
    n = int((w > 0).sum())
    if k > 0:
        n = min(n, int(k))
    cum = np.cumsum(w[:n])
    if p <= 0:
        n = 1
    elif p < 1:
        n = int((cum - w[:n] < np.float64(p) * cum[-1]).sum())
    if mp > 0:
        n = min(n, int((w >= np.float64(mp)).sum()))
    n = max(n, 1)
    u = np.float64(u) if u > 0 else 0.0
    j = min(int((cum[:n] <= min(u, 1.0) * cum[n - 1]).sum()), n - 1)
    return int(order[j]), n, float(np.log(w[j] / cum[n - 1]))


def sample(mx, logits, n=None, t=None, k=None, p=None, mp=None, u=None, offset=0, stream=None, want=("l", "k")):
    rows, stride = logits.shape
    n = n or stride
    flat = np.concatenate([np.zeros(offset, np.uint16), logits.ravel()])
    up = mx.DeviceArray.from_numpy
    dl = up(flat)
    par = [None if a is None else up(np.asarray(a, dt)) for a, dt in
           ((t, np.float32), (k, np.int32), (p, np.float32), (mp, np.float32))]
    du = up(np.asarray(u, np.float32))
    tok, lp, kept = mx.DeviceArray((rows,), np.uint32), mx.DeviceArray((rows,), np.float32), \
        mx.DeviceArray((rows,), np.int32)
    ws = mx.DeviceArray((max(1, mx.lib.mx_sample_workspace_bytes(rows, n)),), np.uint8)
    mx.check(mx.lib.mx_sample_bf16(dl.ptr + 2 * offset, stride, rows, n, *[a.ptr if a else None for a in par], du.ptr,
                                   tok.ptr, lp.ptr if "l" in want else None, kept.ptr if "k" in want else None, ws.ptr,
                                   stream))
    mx.sync()
    return tok.numpy(), kept.numpy(), lp.numpy()


def check(mx, logits, n=None, t=None, k=None, p=None, mp=None, u=None, **more):
    got = sample(mx, logits, n, t, k, p, mp, u, **more)
    at = lambda a, r, v: v if a is None else np.asarray(a)[r]  # noqa: E731
    for r in range(len(logits)):
        f = np.float32
        tok, kept, lp = reference(logits[r, :n], f(at(t, r, 1.0)), at(k, r, 0), f(at(p, r, 1.0)), f(at(mp, r, 0.0)),
                                  f(u[r]))
        assert (got[0][r], got[1][r]) == (tok, kept), (r, got[0][r], got[1][r], tok, kept)
        if np.isinf(lp):
            assert got[2][r] == lp
        else:
            assert abs(got[2][r] - lp) <= 2.0 ** -23 * abs(lp) + 1e-12, (r, got[2][r], lp)


@pytest.mark.parametrize("n", [1, 2, 7, 63, 64, 65, 511, 513, 1000, 8193, 50257, 151936])
def test_vocabularies_alignments_and_filters(mx, n):
    print("vocab", n, flush=True)
    rows = 12
    rng = np.random.default_rng(n)
    pad = n % 3  # odd strides: rows at every alignment
    logits = to_bf(3 * rng.standard_normal((rows, n + pad)))
    u = rng.random(rows).astype(np.float32)
    t = np.array([1, 0.7, 0, 2, 0.3, 1, 1.5, 0.01, 50, -1, 1, 0.8], np.float32)
    k = np.array([0, 20, 0, 1, 40, 0, n, 0, 3000, 5, n + 9, -3], np.int32)
    p = np.array([1, 0.8, 1, 0.5, 0.95, 0.9, 0.999, 1, 1.5, 0.5, 0.1, 0.7], np.float32)
    mp = np.array([0, 0.05, 0, 0, 0.001, 0, 0, 0.2, 0, 0, 0, 1.5], np.float32)
    check(mx, logits, n, t, k, p, mp, u, offset=n % 8)
    check(mx, logits, n, u=u)                       # the whole distribution
    for name, a in (("t", t), ("k", k), ("p", p), ("mp", mp)):
        check(mx, logits, n, u=u, **{name: a})


def test_borders_and_ties(mx):
    """Equal logits have equal weights of exactly 1: u and top-p meet borders exactly."""
    rows = 16
    logits = np.full((rows, 16), to_bf(np.float32(2.5)), np.uint16)
    u = (np.arange(rows) / 16).astype(np.float32)      # u * 16 is a whole number: the next token
    check(mx, logits, u=u)
    tok, kept, lp = sample(mx, logits, u=u)
    assert (tok == np.arange(16)).all() and (kept == 16).all()
    check(mx, logits, p=np.full(rows, 0.25), u=u)      # exactly four tokens reach a quarter
    assert (sample(mx, logits, p=np.full(rows, 0.25), u=u)[1] == 4).all()
    check(mx, logits, k=np.arange(rows), u=u)
    check(mx, logits, mp=np.full(rows, 1.0), u=u)      # weights of exactly min_p stay
    u = np.array([0, 1, 2, -1, np.nan, 0.999999] + [0.5] * 10, np.float32)
    tok = sample(mx, logits, u=u)[0]
    assert list(tok[:6]) == [0, 15, 15, 0, 0, 15]
    # -0 and 0 are one value: ids in order
    z = np.resize(np.array([0x8000, 0x0000, 0x8000], np.uint16), (8, 24))
    check(mx, z, k=np.arange(8) + 1, u=np.full(8, 0.99))


@pytest.mark.parametrize("n", [65535, 65537, 151936, 1 << 20])
def test_more_equal_tokens_than_a_counter_holds(mx, n):
    print("equal", n, flush=True)
    rng = np.random.default_rng(3)
    rows = 4
    logits = np.full((rows, n), to_bf(np.float32(-1.25)), np.uint16)
    logits[1, ::2] = to_bf(np.float32(-1.2421875))   # neighbouring bf16 values share a word of counters
    logits[2, rng.integers(0, n, 50)] = to_bf(np.float32(3))
    logits[3, : n // 2] = to_bf(np.float32(-200))
    u = np.array([0.123456, 0.87654, 0.99, 0.5], np.float32)
    check(mx, logits, u=u)
    check(mx, logits, u=u, k=[70000, n - 1, 0, 0], p=[0.5, 0.9, 0.7, 0.3])


def test_masked_and_special_logits(mx):
    n = 4096
    rng = np.random.default_rng(4)
    inf, ninf, nan, low = 0x7F80, 0xFF80, 0x7FC0, 0xFF7F
    logits = to_bf(2 * rng.standard_normal((10, n)))
    logits[0, 5:] = ninf                   # a mask leaves five tokens
    logits[1, 1:] = low                    # the lowest finite value as a mask
    logits[2] = low                        # everything masked with it: all equal
    logits[3] = ninf                       # nothing left
    logits[4] = nan
    logits[5, ::7] = nan                   # NaN never wins
    logits[6, [9, 100, 4000]] = inf        # +inf share the mass
    logits[7, ::2] = ninf
    logits[8] = to_bf(np.float32(3e38) * rng.standard_normal(n).clip(-1, 1))  # huge spreads
    logits[9] = to_bf((1e-38 * rng.standard_normal(n)).astype(np.float32))    # nearly equal
    u = rng.random(10).astype(np.float32)
    for t in (1.0, 0.5, 1e-30, 1e30, np.inf, np.nan, -2.0):
        check(mx, logits, t=np.full(10, t, np.float32), u=u)
    check(mx, logits, u=u, k=np.full(10, 7), p=np.full(10, 0.9), mp=np.full(10, 0.01))
    check(mx, logits, u=u, p=np.array([0, -1, np.nan, 0, 0, 0, 0.5, 1e-9, 1e-9, 1e-9]), mp=np.full(10, np.nan))


def test_many_rows_graph_and_optional_outputs(mx):
    """300 rows; without optional outputs; a captured call replayed with other numbers, between eager calls."""
    rng = np.random.default_rng(5)
    rows, n = 300, 3001
    logits = to_bf(3 * rng.standard_normal((rows, n)))
    u = rng.random(rows).astype(np.float32)
    check(mx, logits, p=np.full(rows, 0.9), u=u)
    whole = sample(mx, logits, u=u)[0]
    assert (sample(mx, logits, u=u, want=())[0] == whole).all()
    up = mx.DeviceArray.from_numpy
    dl, du, tok = up(logits), up(u), mx.DeviceArray((rows,), np.uint32)
    ws = mx.DeviceArray((max(1, mx.lib.mx_sample_workspace_bytes(rows, n)),), np.uint8)
    stream = C.c_void_p()
    mx.check(mx.lib.mx_stream_create(C.byref(stream)))
    call = lambda s: mx.check(mx.lib.mx_sample_bf16(dl.ptr, n, rows, n, None, None, None, None, du.ptr, tok.ptr, None,  # noqa: E731
                                                    None, ws.ptr, s))
    graph = Graph(mx, stream.value, lambda: call(stream.value))
    for i in range(3):
        v = rng.random(rows).astype(np.float32)
        du.upload(v)
        graph.launch()
        mx.check(mx.lib.mx_stream_sync(stream))
        assert (tok.numpy() == sample(mx, logits, u=v)[0]).all(), i
    graph.close()
    mx.check(mx.lib.mx_stream_destroy(stream))


def test_with_greedy_settings_it_is_the_argmax(mx):
    rng = np.random.default_rng(6)
    logits = to_bf(rng.standard_normal((8, 30001)))
    logits[:, 7] = logits.view(np.int16).max(1)  # the largest twice
    dl = mx.DeviceArray.from_numpy(logits)
    tok = mx.DeviceArray((8,), np.uint32)
    mx.check(mx.lib.mx_argmax_bf16(dl.ptr, 8, 30001, tok.ptr, None))
    got = sample(mx, logits, t=np.zeros(8), u=np.full(8, 0.9))
    assert (got[0] == tok.numpy()).all()
    assert (sample(mx, logits, k=np.ones(8), u=np.full(8, 0.9))[0] == tok.numpy()).all()
