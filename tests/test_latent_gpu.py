"""The latent cache (mx_attn_latent_append / _read / _decode / _prefill) against 64-bit evaluations of their
definitions: lengths 0, 1, around tiles and pages, padding and empty rows, unwritten positions that hold NaN,
pages that are gone, shared pages, strides, offsets past 32 bits, every number of heads' waves, both latents,
bf16 and e4m3.

Bounds.  bf16 rounds by at most 2^-8 relative (half a step).  An output has that rounding; every p (times its
position's scale) is rounded to bf16 too, which moves the output by at most 2^-8 sum p |v|.  The fp32 scores err by
at most (values of a key) 2^-24 sum |q k| scale: 576 * 2^-24 * 576 * 0.64 * 0.5 / 13.9 = 2^-11 for these inputs (q of
size 0.5, |q k| of 0.5 * 0.64 on average), which is the same relative error of p; sums in fp32 add less.  So:
2^-8 |out| + (2^-8 + 2^-10) mag."""
import ctypes as C

import numpy as np
import pytest

from latent_ref import ROPE, Latent, attend, attend_formed, softmax_rows
from paged_ref import E4M3, Graph, bf, to_bf

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8
F = lambda a: bf(a).astype(np.float64)  # noqa: E731


def say(*a):
    print(*a, flush=True)


def up(mx, a):
    return None if a is None else mx.DeviceArray.from_numpy(np.ascontiguousarray(a))


def ptr(a):
    return None if a is None else a.ptr


def close(got, ref, mag):
    g = F(got)
    bound = HALF * np.abs(ref) + (HALF + 2.0 ** -10) * mag + 1e-30
    off = np.abs(g - ref) / bound
    assert np.isfinite(g).all() and off.max(initial=0) <= 1, (off.max(initial=0), np.argwhere(off > 1)[:4])


def run_decode(mx, c, ql, qr, lens, seqs=None, scale=0.0, out=None):
    rows, d = len(ql), c.dims()
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_latent_decode_workspace_bytes(rows, C.byref(d))),), np.uint8)
    dl, dr, dn = up(mx, ql), up(mx, qr), up(mx, np.asarray(lens, np.int32))
    ds = up(mx, None if seqs is None else np.asarray(seqs, np.int32))
    o = up(mx, np.full(ql.shape, 0x1234, np.uint16) if out is None else out)
    mx.check(mx.lib.mx_attn_latent_decode(dl.ptr, dr.ptr, rows, ptr(ds), dn.ptr, c.dtable.ptr, c.dcache.ptr, c.pscales(),
                                          C.byref(d), scale, ws.ptr, o.ptr, None))
    mx.sync()
    return o.numpy()


def queries(rng, rows, heads, latent):
    return to_bf(0.5 * rng.standard_normal((rows, heads, latent))), to_bf(0.5 * rng.standard_normal((rows, heads, ROPE)))


def expected(c, ql, qr, lens, seqs=None, scale=None):
    scale = (c.nope + ROPE) ** -0.5 if scale is None else scale
    parts = [attend(c, i if seqs is None else seqs[i], F(ql[i]), F(qr[i]), int(n), scale) for i, n in enumerate(lens)]
    return [np.stack([p[j] for p in parts]) for j in (0, 1)]


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("latent", [256, 512])
@pytest.mark.parametrize("heads,page", [(1, 16), (5, 64), (32, 256), (33, 16), (64, 128), (65, 32), (100, 64), (128, 16)])
def test_decode_lengths_and_pages(mx, heads, page, latent, f8):
    lens = [0, 1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 97, 129, 255, 257, 600]
    say("decode", heads, page, latent, f8)
    c = Latent(mx, heads, latent, page, lens, f8, seed=heads + latent, stride_pad=16 * (page == 64))
    ql, qr = queries(np.random.default_rng(1), len(lens), heads, latent)
    got = run_decode(mx, c, ql, qr, lens)
    assert (got[0] == 0).all()  # nothing to attend to
    close(got, *expected(c, ql, qr, lens))
    assert (run_decode(mx, c, ql, qr, lens) == got).all()  # the same bits again


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads", [3, 40, 100])
def test_decode_long_rows_split_and_joined(mx, heads, f8):
    """One long row (many chunks), beside short ones, and 130 rows of one sequence at growing lengths."""
    for rows, context in ((1, 9000), (3, 5000), (130, 400)):
        say("split", heads, rows, context, f8)
        c = Latent(mx, heads, 512, 32, [context], f8, seed=rows)
        ql, qr = queries(np.random.default_rng(2), rows, heads, 512)
        lens = np.linspace(1, context, rows).astype(np.int32)[::-1]
        got = run_decode(mx, c, ql, qr, lens, seqs=np.zeros(rows))
        close(got, *expected(c, ql, qr, lens, [0] * rows))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads", [3, 40, 100])
def test_decode_shares_of_many_tiles(mx, heads, f8):
    """Workgroups that walk more tiles than they hold page ids of at once, of pages that a tile lies in and of pages
    of half a tile."""
    rows, context = 280, 2400
    for page in (16, 64):
        say("many tiles", heads, page, f8)
        c = Latent(mx, heads, 512, page, [context], f8, seed=22 + page)
        ql, qr = queries(np.random.default_rng(23), rows, heads, 512)
        lens = context - 3 * (np.arange(rows) % 7)
        got = run_decode(mx, c, ql, qr, lens, seqs=np.zeros(rows))
        x, _ = c.values(0, context)
        for r in range(0, rows, 1 if heads < 10 else 13):
            k = x[:lens[r]]
            p = softmax_rows(np.concatenate([F(ql[r]), F(qr[r])], 1) @ k.T * 192 ** -0.5)
            close(got[r], p @ k[:, :512], p @ np.abs(k[:, :512]))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,latent", [(20, 512), (50, 256), (128, 512)])
def test_decode_shares_of_many_rows(mx, heads, latent, f8):
    """Hundreds of short rows, several to a workgroup, with empty and padding rows between them and behind."""
    rows, contexts = 700, [70, 1, 33, 5, 64]
    say("many rows", heads, latent, f8)
    c = Latent(mx, heads, latent, 16, contexts, f8, seed=24)
    rng = np.random.default_rng(25)
    seqs = rng.integers(-1, len(contexts) + 1, rows)
    pad = (seqs < 0) | (seqs >= len(contexts))
    most = np.array(contexts + [9, 9])[seqs]
    lens = rng.integers(0, most + 1)
    lens[rows // 2:rows // 2 + 130] = 0                   # more than two rounds of 64 without any
    lens[5], seqs[-3:], pad[-3:] = -7, -1, True
    ql, qr = queries(rng, rows, heads, latent)
    before = rng.integers(0, 1 << 15, ql.shape).astype(np.uint16)
    got = run_decode(mx, c, ql, qr, lens, seqs, out=before)
    assert (got[pad] == before[pad]).all()
    x = [c.values(i, n)[0] for i, n in enumerate(contexts)]
    for r in np.flatnonzero(~pad):
        if lens[r] <= 0:
            assert (got[r] == 0).all()
            continue
        k = x[seqs[r]][:lens[r]]
        p = softmax_rows(np.concatenate([F(ql[r]), F(qr[r])], 1) @ k.T * 192 ** -0.5)
        close(got[r], p @ k[:, :latent], p @ np.abs(k[:, :latent]))


def test_decode_replayed_between_other_calls(mx):
    """Two captured calls that share one workspace, replayed in turn with eager calls of other rows between them: each
    gives its eager bits."""
    heads, f8 = 100, False
    say("replays")
    c = Latent(mx, heads, 512, 32, [900, 400], f8, seed=26)
    d, stream = c.dims(), C.c_void_p()
    mx.check(mx.lib.mx_stream_create(C.byref(stream)))
    s = stream.value
    ws = mx.DeviceArray((mx.lib.mx_attn_latent_decode_workspace_bytes(9, C.byref(d)),), np.uint8)
    calls = []
    for rows, lens in ((9, [900, 3, 0, 500, 64, 32, 31, 900, 17]), (2, [400, 900]), (5, [1, 33, 900, 900, 400])):
        ql, qr = queries(np.random.default_rng(27 + rows), rows, heads, 512)
        seqs = [0 if n > 400 else 1 for n in lens]
        dev = [up(mx, a) for a in (ql, qr, np.array(seqs, np.int32), np.array(lens, np.int32))]
        out = mx.DeviceArray(ql.shape, np.uint16)

        def call(dev=dev, out=out, rows=rows):
            mx.check(mx.lib.mx_attn_latent_decode(dev[0].ptr, dev[1].ptr, rows, dev[2].ptr, dev[3].ptr, c.dtable.ptr,
                                                  c.dcache.ptr, None, C.byref(d), 0.0, ws.ptr, out.ptr, s))
        call()
        mx.check(mx.lib.mx_stream_sync(s))
        want = out.numpy()
        close(want, *expected(c, ql, qr, lens, seqs))
        calls.append((call, out, want))
    graphs = [Graph(mx, s, call) for call, _, _ in calls[:2]]
    for _ in range(3):
        for g, (_, out, want) in zip(graphs, calls):
            out.upload(np.full(want.shape, 0x1234, np.uint16))
            g.launch()
            mx.check(mx.lib.mx_stream_sync(s))
            assert (out.numpy() == want).all()
            calls[2][0]()
            mx.check(mx.lib.mx_stream_sync(s))
            assert (calls[2][1].numpy() == calls[2][2]).all()
    for g in graphs:
        g.close()
    mx.check(mx.lib.mx_stream_destroy(stream))


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads", [20, 50, 128])
def test_decode_padding_shared_and_missing_pages(mx, heads, f8):
    say("padding", heads, f8)
    c = Latent(mx, heads, 512, 16, [100, 70, 50], f8, seed=3)
    c.table[1, :2] = c.table[0, :2]      # a common prefix
    c.table[2, 1] = -1                   # a page that is gone, in the middle
    c.table[2, 3] = c.pages              # and one past the cache
    c.upload()
    seqs = [1, -1, 0, 3, 2, 2, 0, 2]     # two of them padding
    lens = [70, 10, 100, 5, 50, 16, 1000, 10]
    ql, qr = queries(np.random.default_rng(4), len(seqs), heads, 512)
    before = np.random.default_rng(5).integers(0, 1 << 15, ql.shape).astype(np.uint16)
    got = run_decode(mx, c, ql, qr, lens, seqs, out=before)
    pad = np.array([not 0 <= s < 3 for s in seqs])
    assert (got[pad] == before[pad]).all()
    # a length past the table is cut to it; what lies there behind the contexts is NaN, so it is one that fits
    lens = [min(n, 16 * c.table.shape[1]) for n in lens]
    keep = ~pad & np.array([n != 16 * c.table.shape[1] for n in lens])
    at = np.flatnonzero(keep)
    close(got[at], *expected(c, ql[at], qr[at], np.array(lens)[at], [seqs[i] for i in at]))
    gone = Latent(mx, heads, 512, 16, [40], f8, seed=6)
    gone.table[:] = -1
    gone.upload()
    assert (run_decode(mx, gone, ql[:1], qr[:1], [40]) == 0).all()  # positions, but none in a page
    every = Latent(mx, heads, 512, 16, [48], f8, seed=7)
    got = run_decode(mx, every, ql[:1], qr[:1], [2 ** 31 - 1])
    close(got, *expected(every, ql[:1], qr[:1], [48]))


def test_decode_scale_and_large_scores(mx):
    """Scores that grow along the keys, so that the reference is moved on and on, and a scale of the caller's."""
    for heads, f8 in ((20, False), (128, False), (40, True)):
        say("scores", heads, f8)
        c = Latent(mx, heads, 512, 64, [700], f8, seed=8)
        ql, qr = queries(np.random.default_rng(9), 1, heads, 512)
        x = np.random.default_rng(10).standard_normal((700, 576))
        x[:, 512:] = 0
        x[:, 512] = np.linspace(-200, 200, 700)  # exact enough: its p differ by far more than a rounding of q k
        qr[:] = 0
        qr[..., 0] = to_bf(np.full(heads, 4.0))
        c.put(0, 0, x)
        c.upload()
        ref, mag = expected(c, ql, qr, [700], scale=0.125)
        # products of up to 800 in fp32: 2^-24 * 800 * 0.125 * 2 more than the usual bound
        close(run_decode(mx, c, ql, qr, [700], scale=0.125), ref, mag * 1.01)


def test_offsets_past_32_bits(mx):
    """Pages far apart: elements past 2^32 for append, read and attention."""
    heads, page, stride = 5, 16, 1 << 29
    say("far pages")
    pages = 10
    cache = mx.DeviceArray((pages * stride,), np.uint16)
    d = mx.LatentDimsC(heads, 128, 128, 512, ROPE, page, pages, 1, 2, mx.MX_DT_BF16, stride)
    table = up(mx, np.array([[9, 8]], np.int32))
    rng = np.random.default_rng(11)
    x, q = to_bf(rng.standard_normal((20, 576))), to_bf(rng.standard_normal((20, heads * 192)))
    inv = up(mx, 1e4 ** (-np.arange(32) / 32))
    rope = mx.RopeAxesC(ROPE, 1, inv.ptr)
    zero, pos = up(mx, np.zeros(20, np.int32)), up(mx, np.arange(20, dtype=np.int32))
    dx, dq, dr = up(mx, x), up(mx, q), mx.DeviceArray((20, heads, ROPE), np.uint16)
    mx.check(mx.lib.mx_attn_latent_append(dx.ptr, 576, dq.ptr, heads * 192, 20, zero.ptr, pos.ptr, zero.ptr, C.byref(rope),
                                          None, 0.0, table.ptr, C.byref(d), dr.ptr, cache.ptr, None, None))
    starts = up(mx, np.array([0, 20], np.int32))
    lat, rot = mx.DeviceArray((20, 512), np.uint16), mx.DeviceArray((20, 64), np.uint16)
    mx.check(mx.lib.mx_attn_latent_read(cache.ptr, None, 20, starts.ptr, None, table.ptr, C.byref(d), lat.ptr, 512, rot.ptr,
                                        64, None))
    mx.sync()
    assert (lat.numpy() == x[:, :512]).all() and (rot.numpy() == x[:, 512:]).all()  # turned by 0
    c = Latent(mx, heads, 512, page, [20], seed=0, fill=False)
    c.put(0, 0, F(x))
    ql, qr = queries(rng, 1, heads, 512)
    ws = mx.DeviceArray((mx.lib.mx_attn_latent_decode_workspace_bytes(1, C.byref(d)),), np.uint8)
    dl, dqr, n, out = up(mx, ql), up(mx, qr), up(mx, np.array([20], np.int32)), mx.DeviceArray((1, heads, 512), np.uint16)
    mx.check(mx.lib.mx_attn_latent_decode(dl.ptr, dqr.ptr, 1, None, n.ptr, table.ptr, cache.ptr, None, C.byref(d), 0.0,
                                          ws.ptr, out.ptr, None))
    mx.sync()
    close(out.numpy(), *expected(c, ql, qr, [20]))


@pytest.mark.parametrize("heads", [7, 60, 128])
def test_infinite_and_nan_values(mx, heads):
    """Past the end and in missing pages they are not seen; where a row sees one, softmax of its scores says what
    follows: NaN throughout, or with a score of -inf the weight 0, and NaN in that value's dim alone."""
    say("infinite", heads)
    c = Latent(mx, heads, 512, 16, [90, 90], seed=12)
    ql, qr = queries(np.random.default_rng(13), 2, heads, 512)
    lens = [77, 90]
    base = run_decode(mx, c, ql, qr, lens)
    v = c.view().copy()
    for p in range(77, 90):
        v[c.table[0, p // 16], p % 16] = 0x7F80 if p % 2 else 0xFFC0
    c.raw[:, :16 * 576] = v.reshape(c.pages, -1)
    c.upload()
    assert (run_decode(mx, c, ql, qr, lens)[0] == base[0]).all()
    pid, off = c.table[1, 2], 5
    c.view()[pid, off, 512 + 3] = 0x7F80   # in the rotary key: q's signs decide
    c.upload()
    got = F(run_decode(mx, c, ql, qr, lens))
    up_, down = F(qr[1, :, 3]) > 0, F(qr[1, :, 3]) < 0
    assert np.isnan(got[1][up_]).all()
    x, _ = c.values(1, 90)
    use = np.arange(90) != 2 * 16 + 5
    s = np.concatenate([F(ql[1]), F(qr[1])], 1)[down] @ x[use].T * 192 ** -0.5
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    close(to_bf(got[1][down].astype(np.float32)), p @ x[use, :512], p @ np.abs(x[use, :512]))
    c.view()[pid, off, 512 + 3] = 0
    c.view()[pid, off, 100] = 0xFF80       # in the latent
    c.upload()
    got = F(run_decode(mx, c, ql, qr, lens))
    assert np.isnan(got[1][:, 100]).all()
    assert (np.isnan(got[1]).all(1) | (F(ql[1, :, 100]) >= 0)).all()
    assert np.isfinite(got[1][F(ql[1, :, 100]) > 0][:, :100]).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("latent,nope,heads,axes,page,rows", [
    (512, 128, 128, 1, 64, 8), (512, 128, 20, 3, 16, 77), (256, 64, 5, 2, 32, 33), (512, 128, 1, 4, 128, 1),
    (256, 128, 17, 1, 256, 40), (512, 64, 100, 1, 16, 700)])
def test_append(mx, latent, nope, heads, axes, page, rows, f8):
    """fp32 arithmetic with one rounding: 2^-8 relative for bf16 (2^-4 for e4m3, half its smallest step 2^-10
    below), plus 2^-20 of the pair's size for the fp32 rotation (its sums of two products and the fp32
    sine and cosine, a few 2^-24 each).  A scale is the largest value's, so within 2^-20 of it."""
    say("append", latent, nope, heads, axes, page, rows, f8)
    seqs = np.arange(rows, dtype=np.int32) % 3
    pos = (np.arange(rows, dtype=np.int32) // 3) + np.array([0, 5, 1000 % (3 * page)], np.int32)[seqs]
    c = Latent(mx, heads, latent, page, [int(pos.max()) + 2] * 3, f8, nope, seed=rows, stride_pad=16, fill=False)
    rng = np.random.default_rng(14)
    x = to_bf(2 * rng.standard_normal((rows, c.wide + 8)))
    q = to_bf(rng.standard_normal((rows, heads * (nope + ROPE) + 16)))
    norm = None if rows == 1 else to_bf(0.3 * rng.standard_normal(latent))
    if rows > 3:
        x[3] = 0                                      # a position of zeros
        x[4, :c.wide] = to_bf(2.0 ** -105 * rng.standard_normal(c.wide))
    rope_pos = rng.integers(0, 2 ** 22, (axes, rows)).astype(np.int32)  # far positions
    inv = 1e4 ** (-np.arange(32) / 32)
    pair = rng.integers(0, axes, 32)
    dinv = up(mx, inv)
    rope = mx.RopeAxesC(ROPE, axes, dinv.ptr)
    for i in range(32):
        rope.pair_axis[i] = int(pair[i])
    seqs[-1] = -1 if rows > 1 else seqs[-1]           # a padding row
    pos_dev = pos.copy()
    if rows > 2:
        pos_dev[1] = page * c.table.shape[1]          # outside the table: only q
        pos_dev[2] = -1
    dx, dq, dseq, dpos, drp, dn = (up(mx, a) for a in (x, q, seqs, pos_dev, rope_pos, norm))
    dr, d = up(mx, np.full((rows, heads, ROPE), 0x1234, np.uint16)), c.dims()
    mx.check(mx.lib.mx_attn_latent_append(dx.ptr, x.shape[1], dq.ptr, q.shape[1], rows, dseq.ptr, dpos.ptr, drp.ptr,
                                          C.byref(rope), ptr(dn), 1e-6, c.dtable.ptr, C.byref(d), dr.ptr, c.dcache.ptr,
                                          c.pscales(), None))
    mx.sync()
    angle = rope_pos[pair].T * inv                    # [rows, 32]
    cos, sin = np.cos(angle), np.sin(angle)

    def turned(v, cos, sin):
        return np.concatenate([v[..., :32] * cos - v[..., 32:] * sin, v[..., 32:] * cos + v[..., :32] * sin], -1)

    xs = F(x)
    lat = xs[:, :latent]
    if norm is not None:
        lat = lat / np.sqrt((lat ** 2).mean(1, keepdims=True) + 1e-6) * (F(norm) + 1)
    want = np.concatenate([lat, turned(xs[:, latent:c.wide], cos, sin)], 1)
    want_q = turned(F(q)[:, :heads * (nope + ROPE)].reshape(rows, heads, -1)[..., nope:], cos[:, None], sin[:, None])
    got_q, before, before_s = dr.numpy(), c.view().copy(), None if c.scales is None else c.scales.copy()
    c.download()
    got = c.view()
    written = np.zeros(got.shape[:2], bool)
    for r in range(rows):
        if seqs[r] < 0:
            assert (got_q[r] == 0x1234).all()
            continue
        size = np.abs(want_q[r]).max()
        assert (np.abs(F(got_q[r]) - want_q[r]) <= HALF * np.abs(want_q[r]) + 2.0 ** -20 * size).all()
        if not 0 <= pos_dev[r] < page * c.table.shape[1]:
            continue
        pid, off = c.table[seqs[r], pos[r] // page], pos[r] % page
        written[pid, off] = True
        size = np.abs(want[r]).max()
        if f8:
            s = max(size, 2.0 ** -100) / 448
            assert abs(c.scales[pid, off] - s) <= 2.0 ** -20 * s
            ref = want[r] / s
            assert (np.abs(E4M3[got[pid, off]] - ref) <= 2.0 ** -4 * np.abs(ref) + 2.0 ** -10 + 2.0 ** -20 * 448).all()
        else:
            assert (np.abs(F(got[pid, off]) - want[r]) <= HALF * np.abs(want[r]) + 2.0 ** -20 * size).all()
    assert (got[~written] == before[~written]).all()  # everything else is as it was
    assert (c.raw[:, page * c.wide:] == (0x7F if f8 else 0x7FC1)).all()
    if f8:
        assert np.array_equal(c.scales[~written], before_s[~written], equal_nan=True)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("latent,page", [(512, 16), (512, 128), (256, 64)])
def test_read(mx, latent, page, f8):
    """bf16 comes back bit for bit; of e4m3 the product with the scale is rounded to fp32 and to bf16."""
    contexts = [70, 1, 33, 0, 129, 16]
    say("read", latent, page, f8)
    c = Latent(mx, 5, latent, page, contexts, f8, seed=15, stride_pad=32)
    c.table[2, 0] = -1 if page < 33 else c.table[2, 0]
    c.upload()
    first = np.array([3, 0, 0, 7, 100, 2 ** 31 - 5], np.int32)
    counts = [67, 1, 33, 0, 29, 9]            # the last sequence's are past the table
    starts = np.cumsum([2] + counts).astype(np.int32)  # two rows before the first sequence
    rows = starts[-1] + 3                     # three behind the last
    lat, rot = np.full((rows, latent + 8), 0x1234, np.uint16), np.full((rows, ROPE + 16), 0x1234, np.uint16)
    dl, dr, ds, df, d = up(mx, lat), up(mx, rot), up(mx, starts), up(mx, first), c.dims()
    mx.check(mx.lib.mx_attn_latent_read(c.dcache.ptr, c.pscales(), rows, ds.ptr, df.ptr, c.dtable.ptr, C.byref(d), dl.ptr,
                                        lat.shape[1], dr.ptr, rot.shape[1], None))
    mx.sync()
    got_l, got_r = dl.numpy(), dr.numpy()
    assert (got_l[:, latent:] == 0x1234).all() and (got_r[:, ROPE:] == 0x1234).all()
    inside = np.zeros(rows, bool)
    inside[2:starts[-1]] = True
    assert (got_l[~inside] == 0x1234).all() and (got_r[~inside] == 0x1234).all()
    for s, n in enumerate(counts[:5]):
        x, there = c.values(s, int(first[s]) + n) if n else (np.zeros((0, c.wide)), None)
        x = x[first[s]:]
        got = np.concatenate([F(got_l[starts[s]:starts[s + 1], :latent]), F(got_r[starts[s]:starts[s + 1], :ROPE])], 1)
        assert (np.abs(got - x) <= (HALF + 2.0 ** -22 if f8 else 0) * np.abs(x)).all()
    assert (got_l[starts[5]:starts[6], :latent] == 0).all() and (got_r[starts[5]:starts[6], :ROPE] == 0).all()


def run_prefill(mx, q, qr, kv, kr, starts, kv_starts, heads, nope, scale=0.0, sequences=None):
    """q [rows, stride], qr [rows, heads, 64], kv [kv rows, stride], kr [kv rows, stride]"""
    d = mx.LatentDimsC(heads, nope, nope, 512, ROPE, 16, 1, sequences or len(starts) - 1, 1, mx.MX_DT_BF16, 16 * 576)
    rows, kv_rows = len(q), len(kv)
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_latent_prefill_workspace_bytes(rows, kv_rows, C.byref(d))),), np.uint8)
    dev = [up(mx, a) for a in (q, qr, kv, kr, np.asarray(starts, np.int32), np.asarray(kv_starts, np.int32))]
    o = up(mx, np.full((rows, heads, nope), 0x1234, np.uint16))
    mx.check(mx.lib.mx_attn_latent_prefill(dev[0].ptr, q.shape[1], dev[1].ptr, rows, dev[4].ptr, dev[2].ptr, kv.shape[1],
                                           dev[3].ptr, kr.shape[1], kv_rows, dev[5].ptr, C.byref(d), scale, ws.ptr, o.ptr,
                                           None))
    mx.sync()
    return o.numpy()


def formed(rng, rows, kv_rows, heads, nope, pad=0):
    q = to_bf(0.5 * rng.standard_normal((rows, heads * (nope + ROPE) + pad)))
    q.reshape(rows, -1)[:, :heads * (nope + ROPE)].reshape(rows, heads, -1)[..., nope:] = 0x7FC1  # not read
    return (q, to_bf(0.5 * rng.standard_normal((rows, heads, ROPE))),
            to_bf(rng.standard_normal((kv_rows, heads * 2 * nope + pad))), to_bf(rng.standard_normal((kv_rows, ROPE + pad))))


def check_prefill(got, q, qr, kv, kr, starts, kv_starts, heads, nope, scale=None):
    scale = (nope + ROPE) ** -0.5 if scale is None else scale
    inside = np.zeros(len(q), bool)
    for s in range(len(starts) - 1):
        a, b, k0, k1 = starts[s], starts[s + 1], kv_starts[s], kv_starts[s + 1]
        inside[a:b] = True
        if a == b:
            continue
        ref, mag = attend_formed(F(q[a:b, :heads * (nope + ROPE)]).reshape(b - a, heads, nope + ROPE), F(qr[a:b]),
                                 F(kv[k0:k1, :heads * 2 * nope]).reshape(k1 - k0, heads, 2 * nope), F(kr[k0:k1, :ROPE]), scale)
        close(got[a:b], ref, mag)
    assert (got[~inside] == 0x1234).all()


@pytest.mark.parametrize("heads,nope", [(1, 128), (3, 64), (8, 128), (20, 64), (5, 128)])
def test_prefill_packed_sequences(mx, heads, nope):
    """Sequences of one row and of hundreds, with and without prefixes, none at all, and fewer positions than rows."""
    new = [1, 33, 0, 130, 128, 7, 300, 5, 40]
    total = [1, 33, 20, 131, 500, 9, 300, 3, 0]
    say("prompts", heads, nope)
    starts, kv_starts = np.cumsum([3] + new), np.cumsum([2] + total)  # rows before the first belong to none
    args = formed(np.random.default_rng(16), starts[-1] + 4, kv_starts[-1] + 5, heads, nope, pad=8)
    got = run_prefill(mx, *args, starts, kv_starts, heads, nope)
    check_prefill(got, *args, starts, kv_starts, heads, nope)
    assert (got[starts[8]:starts[9]] == 0).all()                  # no positions
    assert (got[starts[7]:starts[7] + 2] == 0).all()              # before position 0
    again = run_prefill(mx, *args, starts, kv_starts, heads, nope)
    assert (again == got).all()
    idle = run_prefill(mx, *args, list(starts) + [starts[-1]] * 200, list(kv_starts) + [kv_starts[-1]] * 200, heads, nope)
    assert (idle == got).all()                                    # sequences without rows change nothing


@pytest.mark.parametrize("heads,nope,count,total", [(2, 128, 1, 3000), (2, 64, 40, 2000), (3, 128, 128, 1500),
                                                    (8, 128, 200, 900), (1, 64, 700, 700), (2, 128, 1030, 1030)])
def test_prefill_few_rows_on_long_prefixes_and_whole_prompts(mx, heads, nope, count, total):
    say("split prompts", heads, nope, count, total)
    args = formed(np.random.default_rng(17), count, total, heads, nope)
    got = run_prefill(mx, *args, [0, count], [0, total], heads, nope, scale=0.11)
    check_prefill(got, *args, [0, count], [0, total], heads, nope, scale=0.11)


@pytest.mark.parametrize("heads,nope,count,total", [(2, 128, 150, 1200), (8, 64, 140, 140), (3, 128, 300, 300)])
def test_what_later_rows_hold_stays_unseen(mx, heads, nope, count, total):
    """Infinities and NaN in the keys and values of the last positions, past the last one, and between sequences:
    the rows before keep their bits, and an infinite value is infinite for the rows that see it."""
    say("unseen", heads, nope, count, total)
    rng = np.random.default_rng(18)
    q, qr, kv, kr = formed(rng, count, total + 40, heads, nope)
    base = run_prefill(mx, q, qr, kv, kr, [0, count], [0, total], heads, nope)
    kv2, kr2 = kv.copy(), kr.copy()
    kv2[total:], kr2[total:] = 0x7F80, 0x7FC1   # past the last position
    v = kv2.reshape(len(kv), heads, 2 * nope)
    at = total - 37
    v[at, :, nope + 3] = 0x7F80                 # an infinite value
    v[at + 10, :, nope + 3] = 0x7FC1            # and later NaN in the same dim
    v[at + 20, :, 5] = 0xFF80                   # a key
    kr2[at + 30, 1] = 0x7FC1
    got = run_prefill(mx, q, qr, kv2, kr2, [0, count], [0, total], heads, nope)
    row = at - (total - count)                  # the row of position `at`
    assert (got[:row] == base[:row]).all()
    inf = F(got[row:row + 10])[..., 3]
    assert (inf == np.inf).all()
    other = np.ones(nope, bool)
    other[3] = False
    a, b = F(got[row:row + 20])[..., other], F(base[row:row + 20])[..., other]
    assert (np.abs(a - b) <= 2 * HALF * np.abs(b) + 1e-6).all()
    assert np.isnan(F(got[row + 10:row + 20])[..., 3]).all()
    assert np.isnan(F(got[row + 30:])).all()


@pytest.mark.parametrize("heads,nope", [(3, 128), (2, 64)])
def test_infinite_values_in_one_sequence_of_many(mx, heads, nope):
    """An infinite value, NaN and one of each sign, early, late and in one head of a sequence among others, over
    several blocks of rows and with the keys split: what does not see them keeps its bits, what does has the formula's
    infinity or NaN in that dim and its other dims within the usual bounds."""
    new, total = [40, 600, 1, 300, 20], [300, 1900, 700, 300, 20]
    for count in (5, 2):  # the second: few rows, keys split
        say("infinite prompts", heads, nope, count)
        n, t = (new, total) if count == 5 else ([30, 100], [1500, 1300])
        starts, kv_starts = np.cumsum([0] + n), np.cumsum([0] + t)
        q, qr, kv, kr = formed(np.random.default_rng(31), starts[-1], kv_starts[-1], heads, nope)
        base = run_prefill(mx, q, qr, kv, kr, starts, kv_starts, heads, nope)
        check_prefill(base, q, qr, kv, kr, starts, kv_starts, heads, nope)
        kv2 = kv.copy()
        v = kv2.reshape(len(kv), heads, 2 * nope)
        at = [10, t[1] - 25, t[1] - 5]           # in sequence 1: what every row sees, and what its last rows see
        v[kv_starts[1] + at[0], 0, nope + 7] = 0xFF80
        v[kv_starts[1] + at[1], 1, nope + 9] = 0x7F80
        v[kv_starts[1] + at[2], 1, nope + 9] = 0xFF80
        got = run_prefill(mx, q, qr, kv2, kr, starts, kv_starts, heads, nope)
        a, b = starts[1], starts[2]
        seen = np.arange(t[1] - n[1], t[1])      # a row's own position
        same = np.ones(got.shape, bool)
        same[a:b, 0, 7] = False
        same[a:b, 1, 9] = seen < at[1]
        assert (F(got[a:b, 0, 7]) == -np.inf).all()
        late = F(got[a:b, 1, 9])
        assert (late[(seen >= at[1]) & (seen < at[2])] == np.inf).all() and np.isnan(late[seen >= at[2]]).all()
        assert (got[same] == base[same]).all()
        assert (run_prefill(mx, q, qr, kv2, kr, starts, kv_starts, heads, nope) == got).all()


@pytest.mark.parametrize("f8", [False, True])
def test_a_request_from_prompt_to_tokens(mx, f8):
    """The set as it is used, with a model's projections: two prompts enter the cache, the first in two parts (its
    prefix read back from the cache), keys and values are formed and attended to; then four steps of one token for
    both with the projections absorbed, whose results are those of the formed keys and values; the logits of the
    steps go through penalties, biases and masks to the sampler.  Steps run eagerly and as a captured graph
    replayed with the step's data copied in, bit for bit."""
    heads, latent, nope, page, vocab = 5, 512, 128, 16, 500
    counts, steps = [150, 40], 4
    say("request", f8)
    c = Latent(mx, heads, latent, page, [n + steps for n in counts], f8, nope, seed=19, fill=False)
    rng = np.random.default_rng(20)
    inv = 1e4 ** (-np.arange(32) / 32)
    dinv = up(mx, inv)
    rope, d = mx.RopeAxesC(ROPE, 1, dinv.ptr), c.dims()
    norm = up(mx, to_bf(0.2 * rng.standard_normal(latent)))
    w = rng.standard_normal((heads, 2 * nope, latent)) / np.sqrt(latent)  # of each head's keys and values
    wk, wv = w[:, :nope], w[:, nope:]
    qw = heads * (nope + ROPE)
    stream = C.c_void_p()
    mx.check(mx.lib.mx_stream_create(C.byref(stream)))
    s = stream.value

    def append(dx, dq, n, dseq, dpos, dr):
        mx.check(mx.lib.mx_attn_latent_append(dx.ptr, c.wide, dq.ptr, qw, n, dseq.ptr, dpos.ptr, dpos.ptr, C.byref(rope),
                                              norm.ptr, 1e-6, c.dtable.ptr, C.byref(d), dr.ptr, c.dcache.ptr, c.pscales(),
                                              s))

    def part(new):
        """Rows (sequence, first position, count) enter the cache and are attended to, over all positions so far."""
        rows = sum(n for _, _, n in new)
        x, q = to_bf(rng.standard_normal((rows, c.wide))), to_bf(0.5 * rng.standard_normal((rows, qw)))
        seqs = np.concatenate([np.full(n, i) for i, _, n in new]).astype(np.int32)
        pos = np.concatenate([np.arange(f, f + n) for _, f, n in new]).astype(np.int32)
        dx, dq, dseq, dpos, dr = up(mx, x), up(mx, q), up(mx, seqs), up(mx, pos), mx.DeviceArray((rows, heads, ROPE),
                                                                                                 np.uint16)
        append(dx, dq, rows, dseq, dpos, dr)
        count, total = np.zeros(2, int), np.zeros(2, int)
        for i, f, n in new:
            count[i], total[i] = n, f + n
        starts, kv_starts = np.cumsum([0, *count]).astype(np.int32), np.cumsum([0, *total]).astype(np.int32)
        ds, dk, t = up(mx, starts), up(mx, kv_starts), int(kv_starts[-1])
        lat, rot = mx.DeviceArray((t, latent), np.uint16), mx.DeviceArray((t, ROPE), np.uint16)
        mx.check(mx.lib.mx_attn_latent_read(c.dcache.ptr, c.pscales(), t, dk.ptr, None, c.dtable.ptr, C.byref(d), lat.ptr,
                                            latent, rot.ptr, ROPE, s))
        mx.check(mx.lib.mx_stream_sync(s))
        kv = to_bf(np.einsum("tl,hol->tho", F(lat.numpy()), w).reshape(t, -1))  # the caller's projection
        got = run_prefill(mx, q, dr.numpy(), kv, rot.numpy(), starts, kv_starts, heads, nope)
        check_prefill(got, q, dr.numpy(), kv, rot.numpy(), starts, kv_starts, heads, nope)

    part([(0, 0, 100)])
    part([(0, 100, 50), (1, 0, 40)])
    c.download()
    base, base_s = c.raw.copy(), None if c.scales is None else c.scales.copy()

    shape = lambda *n: mx.DeviceArray(n, np.uint16)  # noqa: E731
    dx, dq, dr, dl, out = shape(2, c.wide), shape(2, qw), shape(2, heads, ROPE), shape(2, heads, latent), \
        shape(2, heads, latent)
    dpos, dlen, dseq = mx.DeviceArray((2,), np.int32), mx.DeviceArray((2,), np.int32), up(mx, np.array([0, 1], np.int32))
    ws = mx.DeviceArray((mx.lib.mx_attn_latent_decode_workspace_bytes(2, C.byref(d)),), np.uint8)
    logits, controlled = shape(2, vocab), shape(2, vocab)
    history = up(mx, rng.integers(0, vocab, (2, 64)).astype(np.int32))
    f32 = lambda *v: up(mx, np.array(v, np.float32))  # noqa: E731
    i32 = lambda *v: up(mx, np.array(v, np.int32))  # noqa: E731
    keep = dict(prompt_lens=i32(30, 20), lens=i32(60, 50), repetition=f32(1.2, 1.0), frequency=f32(0.3, 0.1),
                presence=f32(0.2, 0.0), bias_starts=i32(0, 2, 2), bias_tokens=i32(7, 9), bias_values=f32(3.0, -np.inf),
                masks=up(mx, rng.integers(0, 2 ** 32, (1, 16)).astype(np.uint32)), mask_rows=i32(-1, 0))
    controls = mx.LogitsControlsC(tokens=history.ptr, tokens_stride=64, sequences=2, bias_count=2, mask_stride=16,
                                  mask_states=1, **{k: v.ptr for k, v in keep.items()})
    uniform, tokens = f32(0.3, 0.8), mx.DeviceArray((2,), np.uint32)
    sws = mx.DeviceArray((mx.lib.mx_sample_workspace_bytes(2, vocab),), np.uint8)

    def step():
        append(dx, dq, 2, dseq, dpos, dr)
        mx.check(mx.lib.mx_attn_latent_decode(dl.ptr, dr.ptr, 2, None, dlen.ptr, c.dtable.ptr, c.dcache.ptr, c.pscales(),
                                              C.byref(d), 0.0, ws.ptr, out.ptr, s))
        mx.check(mx.lib.mx_logits_control_bf16(logits.ptr, vocab, 2, vocab, C.byref(controls), controlled.ptr, vocab, s))
        mx.check(mx.lib.mx_sample_bf16(controlled.ptr, vocab, 2, vocab, None, None, None, None, uniform.ptr, tokens.ptr,
                                       None, None, sws.ptr, s))

    data = []
    for i in range(steps):
        q = to_bf(0.5 * rng.standard_normal((2, qw)))
        absorbed = to_bf(np.einsum("rho,hol->rhl", F(q).reshape(2, heads, -1)[..., :nope], wk))
        data.append((to_bf(rng.standard_normal((2, c.wide))), q, absorbed, to_bf(2 * rng.standard_normal((2, vocab)))))

    def feed(i):
        for dev, host in zip((dx, dq, dl, logits), data[i]):
            dev.upload(host)
        dpos.upload(np.array(counts) + i)
        dlen.upload(np.array(counts) + i + 1)

    eager = []
    for i in range(steps):
        feed(i)
        step()
        mx.check(mx.lib.mx_stream_sync(s))
        eager.append((out.numpy(), controlled.numpy(), tokens.numpy()))
        c.download()
        for r in (0, 1):
            n = counts[r] + i + 1
            got, qr = out.numpy()[r:r + 1], dr.numpy()[r]
            ref, mag = attend(c, r, F(data[i][2][r]), F(qr), n, 192 ** -0.5)
            close(got, ref[None], mag[None])
            # the values of the formed keys and values: the absorbed query's rounding moves scores by 2^-8 sum |q c|
            # scale, and so every p by as much; then the bounds of the result's own products
            x, _ = c.values(r, n)
            kv = np.einsum("tl,hol->tho", x[:, :latent], w)
            full, _ = attend_formed(F(data[i][1][r]).reshape(1, heads, -1), F(qr)[None], kv,
                                    x[:, latent:], 192 ** -0.5)
            via = np.einsum("hl,hol->ho", F(got[0]), wv)
            moved = HALF * np.abs(np.einsum("hl,tl->ht", np.abs(F(data[i][2][r])), np.abs(x[:, :latent]))).max(1) * 192 ** -0.5
            bound = np.einsum("hl,hol->ho", (3 * HALF + 2 * moved[:, None]) * mag, np.abs(wv))
            assert (np.abs(via - full[0]) <= bound).all()
        # masked and banned tokens are never drawn
        assert tokens.numpy()[0] != 9
        word = keep["masks"].numpy()[0]
        assert word[tokens.numpy()[1] // 32] >> (tokens.numpy()[1] % 32) & 1
    final = c.raw.copy()
    c.dcache.upload(base)
    if f8:
        c.dscales.upload(base_s)
    graph = Graph(mx, s, step)
    for i in range(steps):
        feed(i)
        graph.launch()
        mx.check(mx.lib.mx_stream_sync(s))
        for dev, want in zip((out, controlled, tokens), eager[i]):
            assert (dev.numpy() == want).all(), i
        mx.sync()
    assert (c.dcache.numpy() == final).all()
    graph.close()
    mx.check(mx.lib.mx_stream_destroy(s))
