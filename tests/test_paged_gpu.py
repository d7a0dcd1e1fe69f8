"""The paged cache (mx_attn_paged_append / _decode / _prefill) against 64-bit
evaluations of their definitions: lengths 0, 1, around tiles and pages, padding
and empty rows, unwritten positions that hold NaN, pages that are gone, shared
pages, page strides, offsets past 32 bits, every head width, group and page size,
bf16 and e4m3.

Bounds.  bf16 rounds by at most 2^-8 relative (half a step).  An output has that
rounding; the prompt kernel also rounds every p to bf16, which moves the output
by at most 2^-8 sum p |v|, where the one-token kernel keeps p in two bf16 parts
(2^-16).  The fp32 scores err by at most head_dim 2^-24 sum |q k| scale, under
2^-12 for these inputs (256 * 2^-24 * 256 * 0.8 / 16 = 2^-11.7 at worst, half of
that for the 0.5-scaled q), which is the same relative error of p; sums in fp32
add less.  So: 2^-8 |out| + (2^-8 or 0) mag + 2^-11 mag."""
import ctypes as C

import numpy as np
import pytest

from paged_ref import E4M3, Graph, Paged, attend, bf, gates, to_bf

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


def say(*a):
    print(*a, flush=True)


def run_decode(mx, c, q, lens, seqs=None, qkv=None, scale=0.0, out=None, stream=None, keep=None):
    rows = len(q)
    d = c.dims()
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_paged_decode_workspace_bytes(rows, C.byref(d))),), np.uint8)
    dev = [mx.DeviceArray.from_numpy(np.ascontiguousarray(a)) if a is not None else None
           for a in (q, qkv, np.asarray(lens, np.int32), None if seqs is None else np.asarray(seqs, np.int32))]
    o = mx.DeviceArray.from_numpy(np.full(q.shape, 0x1234, np.uint16) if out is None else out)
    args = (dev[0].ptr, dev[1].ptr if qkv is not None else None, 0 if qkv is None else qkv.shape[1], rows,
            dev[3].ptr if seqs is not None else None, dev[2].ptr, c.dtable.ptr, c.dk.ptr, c.dv.ptr, *c.scales(),
            C.byref(d), scale, ws.ptr, o.ptr)
    if keep is not None:
        keep.update(dev=dev, ws=ws, out=o, d=d, args=args)
    mx.check(mx.lib.mx_attn_paged_decode(*args, stream))
    mx.sync()
    return o.numpy()


def run_prefill(mx, c, q, starts, lens, qkv=None, scale=0.0):
    rows = len(q)
    d = c.dims()
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_paged_prefill_workspace_bytes(rows, C.byref(d))),), np.uint8)
    dq, ds, dl = (mx.DeviceArray.from_numpy(np.ascontiguousarray(a)) for a in
                  (q, np.asarray(starts, np.int32), np.asarray(lens, np.int32)))
    dg = mx.DeviceArray.from_numpy(qkv) if qkv is not None else None
    o = mx.DeviceArray.from_numpy(np.full(q.shape, 0x1234, np.uint16))
    mx.check(mx.lib.mx_attn_paged_prefill(
        dq.ptr, dg.ptr if dg else None, 0 if qkv is None else qkv.shape[1], rows, ds.ptr, dl.ptr, c.dtable.ptr,
        c.dk.ptr, c.dv.ptr, *c.scales(), C.byref(d), scale, ws.ptr, o.ptr, None))
    mx.sync()
    return o.numpy()


def close(got, ref, mag, p_bits16):
    g = bf(got).astype(np.float64)
    bound = HALF * np.abs(ref) + ((0 if p_bits16 else HALF) + 2.0 ** -11) * mag + 1e-30
    off = np.abs(g - ref) / bound
    assert np.isfinite(g).all() and off.max(initial=0) <= 1, (off.max(initial=0), np.argwhere(off > 1)[:4])


GEOMETRIES = [(16, 2, 256), (32, 8, 128), (7, 1, 128), (4, 4, 64), (32, 2, 64), (6, 2, 256), (5, 5, 128)]


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd", GEOMETRIES)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_lengths_and_pages(mx, heads, kv, hd, page, f8):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 63, 65, 127, 129, 255, 257, 600]
    gated = heads == 16
    say("decode", heads, kv, hd, page, f8)
    c = Paged(mx, heads, kv, hd, page, lens, f8, gated, seed=heads + hd + page, stride_pad=16 * (page == 64))
    rng = np.random.default_rng(1)
    q = to_bf(0.5 * rng.standard_normal((len(lens), heads, hd)))
    qkv = to_bf(rng.standard_normal((len(lens), 2 * heads * hd + 8))) if gated else None
    got = run_decode(mx, c, q, lens, qkv=qkv)
    parts = [attend(c, i, bf(q[i:i + 1]).astype(np.float64), [n]) for i, n in enumerate(lens)]
    ref, mag = (np.concatenate([p[j] for p in parts]) for j in (0, 1))
    if gated:
        ref, mag = ref * gates(qkv, heads, hd), mag * gates(qkv, heads, hd)
    assert (got[0] == 0).all()  # nothing to attend to
    close(got, ref, mag, True)
    assert (run_decode(mx, c, q, lens, qkv=qkv) == got).all()  # the same bits again


@pytest.mark.parametrize("f8", [False, True])
def test_decode_long_rows_split_and_joined(mx, f8):
    """One long row (many chunks), beside short ones, and 130 rows of one sequence at growing lengths."""
    for rows, context in ((3, 5000), (130, 700)):
        say("split", rows, context, f8)
        c = Paged(mx, 8, 2, 128, 32, [context], f8, seed=rows)
        rng = np.random.default_rng(2)
        q = to_bf(0.5 * rng.standard_normal((rows, 8, 128)))
        lens = np.linspace(1, context, rows).astype(np.int32)[::-1]
        got = run_decode(mx, c, q, lens, seqs=np.zeros(rows))
        ref, mag = attend(c, 0, bf(q).astype(np.float64), lens)
        close(got, ref, mag, True)


@pytest.mark.parametrize("f8", [False, True])
def test_decode_padding_shared_and_missing_pages(mx, f8):
    c = Paged(mx, 16, 2, 256, 16, [100, 70, 50], f8, seed=3)
    c.table[1, :2] = c.table[0, :2]      # a common prefix
    c.table[0, 3] = -1                   # an evicted page inside
    c.table[2, :] = [c.pages, -7, 2 ** 31 - 1, -2 ** 31] + [-1] * (c.table.shape[1] - 4)  # none left
    c.upload()
    rng = np.random.default_rng(4)
    seqs = [0, -1, 1, 2, 3, 0, 2 ** 31 - 1]
    lens = [100, 100, 70, 50, 10, 10 ** 9, 5]  # past the table: cut to it
    q = to_bf(0.5 * rng.standard_normal((len(seqs), 16, 256)))
    limit = [100, 0, 70, 50, 0, 16 * c.table.shape[1], 0]
    # the row whose length passes the table sees its last page to the end: positions 100 .. 111 get numbers
    rest = np.random.default_rng(5).standard_normal((2, 12, 2, 256))
    c.put(0, 100, *rest)
    c.upload()
    got = run_decode(mx, c, q, lens, seqs=seqs, scale=0.11)
    for i in (1, 4, 6):
        assert (got[i] == 0x1234).all()  # padding rows keep their output
    assert (got[3] == 0).all()           # no page left: zeros
    for i in (0, 2, 5):
        ref, mag = attend(c, seqs[i], bf(q[i:i + 1]).astype(np.float64), [limit[i]], scale=0.11)
        close(got[i:i + 1], ref, mag, True)


def test_offsets_past_32_bits(mx):
    """Pages 2^31 + 16 elements apart: two tokens appended and attended to, alone and as a prompt."""
    heads, kv, hd, page, stride = 4, 2, 64, 16, 2 ** 31 + 16
    nbytes = (2 * stride + kv * page * hd) * 2
    say("far pages", nbytes)
    dk, dv = mx.DeviceArray((nbytes,), np.uint8), mx.DeviceArray((nbytes,), np.uint8)
    d = mx.PageDimsC(heads, kv, hd, page, 3, 1, 3, mx.MX_DT_BF16, 0, stride)
    rng = np.random.default_rng(6)
    n = 40
    qkv = to_bf(rng.standard_normal((n, (heads + 2 * kv) * hd)))
    up = mx.DeviceArray.from_numpy
    dqkv, dtab, dseq, dpos = up(qkv), up(np.array([[2, 0, 1]], np.int32)), up(np.zeros(n, np.int32)), \
        up(np.arange(n, dtype=np.int32))
    dq = mx.DeviceArray((n, heads, hd), np.uint16)
    rope = mx.RopeAxesC(0, 1, None)
    mx.check(mx.lib.mx_attn_paged_append(dqkv.ptr, qkv.shape[1], n, dseq.ptr, dpos.ptr, None, C.byref(rope), None,
                                         None, 1e-6, dtab.ptr, C.byref(d), None, None, dq.ptr, dk.ptr, dv.ptr, None))
    x = bf(qkv).astype(np.float64).reshape(n, -1, hd)
    assert (dq.numpy() == qkv.reshape(n, -1, hd)[:, :heads]).all()  # no norm, no rotation: as it was

    class Flat:  # the reference's view: positions in order
        kv = 2

        @staticmethod
        def values(seq, m):
            return x[:m, heads:heads + kv], x[:m, heads + kv:], np.ones(m, bool)

    ws = mx.DeviceArray((max(mx.lib.mx_attn_paged_decode_workspace_bytes(1, C.byref(d)),
                             mx.lib.mx_attn_paged_prefill_workspace_bytes(n, C.byref(d)), 1),), np.uint8)
    out = mx.DeviceArray((n, heads, hd), np.uint16)
    dlen, dst = up(np.array([n], np.int32)), up(np.array([0, n], np.int32))
    mx.check(mx.lib.mx_attn_paged_prefill(dq.ptr, None, 0, n, dst.ptr, dlen.ptr, dtab.ptr, dk.ptr, dv.ptr, None, None,
                                          C.byref(d), 0.0, ws.ptr, out.ptr, None))
    ref, mag = attend(Flat, 0, x[:, :heads], np.arange(n) + 1)
    close(out.numpy(), ref, mag, False)
    mx.check(mx.lib.mx_attn_paged_decode(dq.ptr, None, 0, 1, None, dlen.ptr, dtab.ptr, dk.ptr, dv.ptr, None, None,
                                         C.byref(d), 0.0, ws.ptr, out.ptr, None))
    ref, mag = attend(Flat, 0, x[:1, :heads], [n])
    close(out.numpy()[:1], ref, mag, True)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd", GEOMETRIES)
@pytest.mark.parametrize("page", [16, 128])
def test_prefill_packed_sequences(mx, heads, kv, hd, page, f8):
    """Sequences of no, one and many rows, with and without a prefix, one with more rows than positions (its
    first rows see nothing), rows outside every sequence."""
    counts, lens = [5, 0, 1, 70, 33, 9, 40], [5, 30, 61, 70, 200, 4, 64]
    gated = heads == 16
    say("prefill", heads, kv, hd, page, f8)
    c = Paged(mx, heads, kv, hd, page, lens, f8, gated, seed=heads + page, stride_pad=32 * (page == 16))
    first = 3
    starts = first + np.concatenate([[0], np.cumsum(counts)])
    rows = starts[-1] + 4
    rng = np.random.default_rng(7)
    q = to_bf(0.5 * rng.standard_normal((rows, heads, hd)))
    qkv = to_bf(rng.standard_normal((rows, 2 * heads * hd + 16))) if gated else None
    got = run_prefill(mx, c, q, starts, lens, qkv)
    assert (got[:first] == 0x1234).all() and (got[starts[-1]:] == 0x1234).all()
    for s, (n, total) in enumerate(zip(counts, lens)):
        at = slice(starts[s], starts[s + 1])
        ref, mag = attend(c, s, bf(q[at]).astype(np.float64), total - n + np.arange(n) + 1)
        if gated:
            ref, mag = ref * gates(qkv[at], heads, hd), mag * gates(qkv[at], heads, hd)
        close(got[at], ref, mag, False)
    assert (got[starts[5]:starts[5] + 5] == 0).all()  # 9 rows, 4 positions
    assert (run_prefill(mx, c, q, starts, lens, qkv) == got).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,count,total", [
    (8, 1, 128, 20, 3000), (16, 2, 256, 64, 2100), (4, 4, 64, 3, 2500), (64, 4, 64, 300, 300), (14, 2, 256, 150, 151)])
def test_prefill_few_rows_on_long_prefixes_and_whole_prompts(mx, heads, kv, hd, count, total, f8):
    say("prefill long", heads, kv, hd, count, total, f8)
    c = Paged(mx, heads, kv, hd, 64, [total], f8, seed=total)
    rng = np.random.default_rng(8)
    q = to_bf(0.5 * rng.standard_normal((count, heads, hd)))
    got = run_prefill(mx, c, q, [0, count], [total])
    some = sorted({0, 1, count // 2, count - 1} & set(range(count)))
    ref, mag = attend(c, 0, bf(q[some]).astype(np.float64), [total - count + i + 1 for i in some])
    close(got[some], ref, mag, False)


@pytest.mark.parametrize("f8", [False, True])
def test_prefill_missing_pages(mx, f8):
    c = Paged(mx, 8, 2, 128, 16, [150, 90], f8, seed=9)
    c.table[0, 2] = -1
    c.table[0, 9] = c.pages + 5
    c.table[1, :] = -1
    c.upload()
    rng = np.random.default_rng(10)
    q = to_bf(0.5 * rng.standard_normal((100, 8, 128)))
    got = run_prefill(mx, c, q, [0, 60, 100], [150, 90])
    ref, mag = attend(c, 0, bf(q[:60]).astype(np.float64), 90 + np.arange(60) + 1)
    close(got[:60], ref, mag, False)
    assert (got[60:] == 0).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,total", [(8, 2, 128, 150), (16, 2, 256, 77), (4, 4, 64, 200)])
def test_what_later_rows_hold_stays_unseen(mx, heads, kv, hd, total, f8):
    """Infinite and NaN keys and values of a prompt's own later positions: earlier rows are as if they were
    other numbers; the rows that see one are not finite where they must not be."""
    c = Paged(mx, heads, kv, hd, 32, [total], f8, seed=20)
    rng = np.random.default_rng(21)
    q = to_bf(0.5 * rng.standard_normal((total, heads, hd)))
    ref, mag = attend(c, 0, bf(q).astype(np.float64), np.arange(total) + 1)
    at = total - 40  # inside the last blocks' tiles
    nan = 0x7F if f8 else 0x7FC0
    kc, vc = c.kview(), c.vview()
    for p, d, bits in ((at, 3, nan), (at + 7, hd - 1, nan if f8 else 0x7F80), (at + 20, 9, nan if f8 else 0xFF80)):
        vc[c.table[0, p // 32], 0, d, p % 32] = bits
    kc[c.table[0, (total - 1) // 32], 0, (total - 1) % 32, 5] = nan  # the last key
    c.k[:, :kc[0].size], c.v[:, :vc[0].size] = kc.reshape(c.pages, -1), vc.reshape(c.pages, -1)
    c.upload()
    got = run_prefill(mx, c, q, [0, total], [total])
    group = heads // kv
    seen = np.zeros(got.shape, bool)  # outputs that one of them reaches (kv head 0's)
    seen[at:, :group, 3] = seen[at + 7:, :group, hd - 1] = seen[at + 20:, :group, 9] = True
    seen[total - 1, :group] = True
    g = bf(got).astype(np.float64)
    assert not np.isfinite(g[seen]).any()
    if not f8:
        assert (g[at + 7:-1, :group, hd - 1] == np.inf).all() and (g[at + 20:-1, :group, 9] == -np.inf).all()
    close(np.where(seen, 0, got).astype(np.uint16), np.where(seen, 0, ref), np.where(seen, 0, mag), False)


@pytest.mark.parametrize("heads,kv,hd", [(12, 3, 64), (6, 3, 128), (6, 3, 256)])
def test_scales_of_either_sign_and_zero(mx, heads, kv, hd):
    """A kv head's scale may be negative, or 0 (then every position weighs the same).  At 64 dims scores
    reach over more than 128 octaves, past what fp32 would forgive a maximum of the wrong sign.  Their
    error, at worst hd 2^-24 sum |q k| / sqrt(hd) = hd^1.5 2^-24 0.64 |q| with |q| = 16 (64 / hd)^1.5, is
    under 2^-11.6: the bound of the other tests holds."""
    total = 170
    c = Paged(mx, heads, kv, hd, 16, [total], True, seed=22)
    c.ks *= np.array([-1, 0, 1], np.float32)
    c.vs *= np.array([1, -1, 0], np.float32)
    c.upload()
    rng = np.random.default_rng(23)
    q = to_bf(16 * (64 / hd) ** 1.5 * rng.standard_normal((total, heads, hd)))
    ref, mag = attend(c, 0, bf(q).astype(np.float64), np.arange(total) + 1)
    close(run_prefill(mx, c, q, [0, total], [total]), ref, mag, False)
    few = [0, 1, 33, total - 1]
    got = run_decode(mx, c, np.ascontiguousarray(q[few]), [i + 1 for i in few], seqs=[0] * len(few))
    close(got, ref[few], mag[few], True)


def reference_append(x, c, pos, rope_pos, inv_freq, pair_axis, rot, qn, kn, eps=1e-6):
    """Normalised and rotated q and k, and v, in 64 bits."""
    rows, hd, h, kv = len(x), c.hd, c.heads, c.kv
    per = 2 * hd if c.gated else hd
    q = x[:, :h * per].reshape(rows, h, per)[:, :, :hd]
    k, v = x[:, h * per:h * per + kv * hd].reshape(rows, kv, hd), \
        x[:, h * per + kv * hd:h * per + 2 * kv * hd].reshape(rows, kv, hd)
    half = rot // 2
    a = rope_pos[pair_axis[:half]].T.astype(np.float64) * inv_freq  # [rows, half]
    cos, sin = np.cos(a)[:, None], np.sin(a)[:, None]

    def turn(y, w):
        if w is not None:
            y = y / np.sqrt((y * y).mean(2, keepdims=True) + eps) * (w + 1)
        y1, y2 = y[..., :half], y[..., half:rot]
        return np.concatenate([y1 * cos - y2 * sin, y2 * cos + y1 * sin, y[..., rot:]], 2)

    return turn(q, qn), turn(k, kn), v


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rot,axes,page,rows", [
    (16, 2, 256, 64, 1, 16, 8), (32, 8, 128, 128, 3, 64, 77), (3, 3, 64, 20, 2, 32, 33), (7, 1, 128, 0, 1, 128, 1),
    (16, 2, 256, 256, 4, 256, 40)])
def test_append(mx, heads, kv, hd, rot, axes, page, rows, f8):
    """fp32 arithmetic with one rounding: 2^-8 relative for bf16 (2^-4 for e4m3, half its smallest step 2^-10
    below), plus 2^-20 of the pair's size for the fp32 rotation (its sums of two products and the fp32
    sine and cosine, a few 2^-24 each)."""
    gated = heads == 16
    say("append", heads, kv, hd, rot, axes, page, rows, f8)
    seqs = np.arange(rows, dtype=np.int32) % 3
    pos = (np.arange(rows, dtype=np.int32) // 3) + np.array([0, 5, 1000 % (3 * page)], np.int32)[seqs]
    c = Paged(mx, heads, kv, hd, page, [int(pos.max()) + 2] * 3, f8, gated, seed=rows, stride_pad=16, fill=False)
    rng = np.random.default_rng(11)
    x = to_bf(2 * rng.standard_normal((rows, (heads * (2 if gated else 1) + 2 * kv) * hd + 8)))
    qn, kn = (to_bf(0.3 * rng.standard_normal(hd)) for _ in range(2))
    if rows == 1:
        qn = kn = None  # no norm
    rope_pos = rng.integers(0, 2 ** 22, (axes, rows)).astype(np.int32)  # far positions
    half = rot // 2
    inv = 1e7 ** (-np.arange(half) / max(half, 1))
    pair = rng.integers(0, axes, 128)
    rope = mx.RopeAxesC(rot, axes, None)
    for i in range(half):
        rope.pair_axis[i] = int(pair[i])
    up = mx.DeviceArray.from_numpy
    seqs[-1] = -1 if rows > 1 else seqs[-1]          # a padding row
    pos_dev = pos.copy()
    if rows > 2:
        pos_dev[1] = page * c.table.shape[1]          # outside the table: only q
    dx, dseq, dpos, drp, dinv = up(x), up(seqs), up(pos_dev), up(rope_pos), up(inv if half else np.zeros(1))
    rope.inv_freq = dinv.ptr
    dn = [up(n) if n is not None else None for n in (qn, kn)]
    dq = up(np.full((rows, heads, hd), 0x1234, np.uint16))
    d = c.dims()
    mx.check(mx.lib.mx_attn_paged_append(
        dx.ptr, x.shape[1], rows, dseq.ptr, dpos.ptr, drp.ptr, C.byref(rope), *[n.ptr if n else None for n in dn], 1e-6,
        c.dtable.ptr, C.byref(d), *c.scales(), dq.ptr, c.dk.ptr, c.dv.ptr, None))
    mx.sync()
    f = lambda n: None if n is None else bf(n).astype(np.float64)  # noqa: E731
    q, k, v = reference_append(bf(x).astype(np.float64), c, pos, rope_pos, inv, pair, rot, f(qn), f(kn))
    got_q, got_k, got_v = dq.numpy(), c.dk.numpy(), c.dv.numpy()
    want_k, want_v = c.k.copy(), c.v.copy()
    kc, vc = c.kview(got_k), c.vview(got_v)

    def fits(got, ref, half_step, least):
        size = np.abs(ref).max()
        assert (np.abs(got - ref) <= half_step * np.abs(ref) + least + 2.0 ** -20 * size).all()

    wk, wv = np.zeros(c.kview().shape, bool), np.zeros(c.vview().shape, bool)
    for r in range(rows):
        if seqs[r] < 0:
            assert (got_q[r] == 0x1234).all()
            continue
        fits(bf(got_q[r]).astype(np.float64), q[r], HALF, 0)
        if pos_dev[r] // page >= c.table.shape[1]:
            continue
        pid, off = c.table[seqs[r], pos[r] // page], pos[r] % page
        wk[pid, :, off], wv[pid, :, :, off] = True, True
        if f8:
            lim = lambda t: np.clip(t, -448, 448)  # noqa: E731
            fits(E4M3[kc[pid, :, off]], lim(k[r] / c.ks[:, None]), 2.0 ** -4, 2.0 ** -10)
            fits(E4M3[vc[pid, :, :, off]], lim(v[r] / c.vs[:, None]), 2.0 ** -4, 2.0 ** -10)
        else:
            fits(bf(kc[pid, :, off]).astype(np.float64), k[r], HALF, 0)
            assert (bf(vc[pid, :, :, off]) == v[r]).all()
    # everything else is as it was
    assert (kc[~wk] == c.kview(want_k)[~wk]).all() and (vc[~wv] == c.vview(want_v)[~wv]).all()
    n = c.kv * page * hd
    assert (got_k[:, n:] == want_k[:, n:]).all() and (got_v[:, n:] == want_v[:, n:]).all()


def test_e4m3_rounds_to_nearest_and_saturates(mx):
    """Every tie and neighbour of the e4m3 values through the append's V: bit for bit."""
    from paged_ref import to_e4m3
    vals = np.unique(np.concatenate([E4M3[:127], (E4M3[:126] + E4M3[1:127]) / 2, [449, 464, 1000, 3e38, 2.0 ** -11]]))
    vals = bf(to_bf(np.concatenate([vals, -vals]).astype(np.float32)))  # exact in bf16
    vals = np.resize(vals, 64 * 8).reshape(8, 64)
    c = Paged(mx, 1, 1, 64, 16, [8], True, fill=False)
    c.vs[:] = 1
    c.upload()
    x = to_bf(np.concatenate([np.zeros((8, 128), np.float32), vals], 1))
    up = mx.DeviceArray.from_numpy
    dx, dseq, dpos, dq = up(x), up(np.zeros(8, np.int32)), up(np.arange(8, dtype=np.int32)), \
        mx.DeviceArray((8, 1, 64), np.uint16)
    rope, d = mx.RopeAxesC(0, 1, None), c.dims()
    mx.check(mx.lib.mx_attn_paged_append(dx.ptr, 192, 8, dseq.ptr, dpos.ptr, None, C.byref(rope), None, None, 0.0,
                                         c.dtable.ptr, C.byref(d), None, c.dvs.ptr, dq.ptr, c.dk.ptr, c.dv.ptr, None))
    mx.sync()
    got = c.vview(c.dv.numpy())[c.table[0, 0], 0, :, :8].T
    want = to_e4m3(vals)
    assert (got == want).all(), [(vals.ravel()[i], got.ravel()[i], want.ravel()[i]) for i in
                                 np.flatnonzero(got.ravel() != want.ravel())[:5]]


@pytest.mark.parametrize("f8", [False, True])
def test_a_request_from_prompt_to_tokens(mx, f8):
    """The set as it is used: two prompts enter the cache and are attended to, then four steps of one token for
    both, every output against 64 bits over what the cache holds; the steps once eagerly and once as a captured
    graph replayed with the step's data copied in, bit for bit."""
    heads, kv, hd, page, rot = 16, 2, 256, 16, 64
    counts, steps = [37, 21], 4
    c = Paged(mx, heads, kv, hd, page, [n + steps for n in counts], f8, True, seed=12, fill=False)
    rng = np.random.default_rng(13)
    width = (2 * heads + 2 * kv) * hd
    up = mx.DeviceArray.from_numpy
    inv = 1e7 ** (-np.arange(rot // 2) / (rot // 2))
    dinv = up(inv)
    rope = mx.RopeAxesC(rot, 1, dinv.ptr)
    qn, kn = (to_bf(0.2 * rng.standard_normal(hd)) for _ in range(2))
    dqn, dkn, d = up(qn), up(kn), c.dims()
    starts = np.array([0, 37, 58], np.int32)
    x = to_bf(rng.standard_normal((58, width)))
    seqs = np.repeat([0, 1], counts).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in counts]).astype(np.int32)
    stream = C.c_void_p()
    mx.check(mx.lib.mx_stream_create(C.byref(stream)))
    s = stream.value
    dx, dseq, dpos, dst, dlen = up(x), up(seqs), up(pos), up(starts), up(np.array(counts, np.int32))
    dq, out = mx.DeviceArray((58, heads, hd), np.uint16), mx.DeviceArray((58, heads, hd), np.uint16)
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_paged_prefill_workspace_bytes(58, C.byref(d)),
                             mx.lib.mx_attn_paged_decode_workspace_bytes(2, C.byref(d))),), np.uint8)

    def append(dx, n, dseq, dpos, dq):
        mx.check(mx.lib.mx_attn_paged_append(dx.ptr, width, n, dseq.ptr, dpos.ptr, dpos.ptr, C.byref(rope), dqn.ptr,
                                             dkn.ptr, 1e-6, c.dtable.ptr, C.byref(d), *c.scales(), dq.ptr, c.dk.ptr,
                                             c.dv.ptr, s))

    append(dx, 58, dseq, dpos, dq)
    mx.check(mx.lib.mx_attn_paged_prefill(dq.ptr, dx.ptr, width, 58, dst.ptr, dlen.ptr, c.dtable.ptr, c.dk.ptr,
                                          c.dv.ptr, *c.scales(), C.byref(d), 0.0, ws.ptr, out.ptr, s))
    mx.check(mx.lib.mx_stream_sync(s))

    def check_rows(got, q, x, which, limits, p16):
        c.k, c.v = c.dk.numpy(), c.dv.numpy()
        for seq in (0, 1):
            at = which == seq
            ref, mag = attend(c, seq, bf(q[at]).astype(np.float64), limits[at])
            g = gates(x[at], heads, hd)
            close(got[at], ref * g, mag * g, p16)

    check_rows(out.numpy(), dq.numpy(), x, seqs, pos + 1, False)
    base_k, base_v = c.dk.numpy(), c.dv.numpy()

    step_x = [to_bf(rng.standard_normal((2, width))) for _ in range(steps)]
    dx1, dq1, out1 = mx.DeviceArray((2, width), np.uint16), mx.DeviceArray((2, heads, hd), np.uint16), \
        mx.DeviceArray((2, heads, hd), np.uint16)
    dpos1, dlen1, dseq1 = mx.DeviceArray((2,), np.int32), mx.DeviceArray((2,), np.int32), up(np.array([0, 1], np.int32))

    def step():
        append(dx1, 2, dseq1, dpos1, dq1)
        mx.check(mx.lib.mx_attn_paged_decode(dq1.ptr, dx1.ptr, width, 2, None, dlen1.ptr, c.dtable.ptr, c.dk.ptr,
                                             c.dv.ptr, *c.scales(), C.byref(d), 0.0, ws.ptr, out1.ptr, s))

    def feed(i):
        dx1.upload(step_x[i])
        p = np.array(counts, np.int32) + i
        dpos1.upload(p)
        dlen1.upload(p + 1)

    eager = []
    for i in range(steps):
        feed(i)
        step()
        mx.check(mx.lib.mx_stream_sync(s))
        eager.append(out1.numpy())
        check_rows(eager[-1], dq1.numpy(), step_x[i], np.array([0, 1]), np.array(counts) + i + 1, True)
    final = c.dk.numpy(), c.dv.numpy()
    c.dk.upload(base_k)
    c.dv.upload(base_v)
    graph = Graph(mx, s, step)
    for i in range(steps):
        feed(i)
        graph.launch()
        mx.check(mx.lib.mx_stream_sync(s))
        assert (out1.numpy() == eager[i]).all(), i
        mx.sync()
    assert (c.dk.numpy() == final[0]).all() and (c.dv.numpy() == final[1]).all()
    graph.close()
    mx.check(mx.lib.mx_stream_destroy(s))
