"""The paged cache's other launch shapes against 64-bit evaluations, every row
compared: one-token rows of hundreds of chunks, joined by four and by sixteen
waves; batches whose chunks take two rounds of the device; appends whose waves take
several groups of heads.  Bounds as in test_paged_gpu.py."""
import ctypes as C

import numpy as np
import pytest

from paged_ref import E4M3, Paged, bf, to_bf
from test_paged_gpu import close, reference_append, run_decode
from test_paged_layouts_gpu import Filled, attend_rows

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8


def say(*a):
    print(*a, flush=True)


# q heads, kv heads, head dim, lengths: hundreds of chunks joined by sixteen waves and by four
LONG = [(16, 2, 256, [60001]), (16, 2, 256, [41, 30000, 9000]), (8, 2, 128, [20000, 5, 129, 800, 4099, 1, 600, 257, 90]),
        (16, 1, 64, [50000]), (16, 1, 64, [30011, 7, 900, 5000, 64])]


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("case", range(len(LONG)))
def test_one_token_rows_of_many_chunks(mx, case, f8):
    heads, kv, hd, lens = LONG[case]
    say("chunks", case, f8)
    c = Filled(mx, heads, kv, hd, 64, lens, f8, seed=70 + case)
    rng = np.random.default_rng(71)
    q = to_bf(0.5 * rng.standard_normal((len(lens), heads, hd)))
    got = run_decode(mx, c, q, lens)
    for r, n in enumerate(lens):
        close(got[r:r + 1], *attend_rows(c, r, bf(q[r:r + 1]).astype(np.float64), [n]), True)
    assert (run_decode(mx, c, q, lens) == got).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rows,context", [(8, 8, 128, 72, 3100), (12, 12, 64, 100, 2000), (4, 4, 256, 90, 3300)])
def test_one_token_batches_of_two_rounds(mx, heads, kv, hd, rows, context, f8):
    """At least sixteen units for every workgroup that runs at once: chunks of several units (one sequence's
    pages serve all rows).  e4m3 units are twice as long, so their rows are."""
    context *= 2 if f8 else 1
    say("rounds", heads, kv, hd, rows, context, f8)
    unit, at_once = (256 if f8 else 128), 256 * {64: 4, 128: 3, 256: 2}[hd]
    rng = np.random.default_rng(81)
    lens = np.concatenate([[context, context], rng.integers(context * 9 // 10, context + 1, rows - 2)])
    assert sum(-(-n // unit) for n in lens) * kv >= 16 * at_once
    c = Filled(mx, heads, kv, hd, 32, [context], f8, seed=80)
    q = to_bf(0.5 * rng.standard_normal((rows, heads, hd)))
    got = run_decode(mx, c, q, lens, seqs=np.zeros(rows))
    close(got, *attend_rows(c, 0, bf(q).astype(np.float64), lens), True)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,rot,rows", [(32, 8, 128, 128, 700), (32, 8, 128, 64, 1601), (16, 2, 256, 64, 4093),
                                                  (12, 12, 64, 20, 2049), (15, 1, 64, 64, 4000)])
def test_append_with_several_groups_of_heads_a_wave(mx, heads, kv, hd, rot, rows, f8):
    """Long prompts, whose waves take two to nine groups of a row's heads, four of them on their way.  Tolerances
    as in test_append."""
    say("append", heads, kv, hd, rot, rows, f8)
    page = 64
    c = Paged(mx, heads, kv, hd, page, [rows + 5], f8, seed=90, fill=False)
    rng = np.random.default_rng(91)
    width = (heads + 2 * kv) * hd
    x = to_bf(2 * rng.standard_normal((rows, width), np.float32))
    qn, kn = (to_bf(0.3 * rng.standard_normal(hd)) for _ in range(2))
    pos = (np.arange(rows) + 5).astype(np.int32)
    rope_pos = rng.integers(0, 2 ** 20, (2, rows)).astype(np.int32)
    half = rot // 2
    inv, pair = 1e6 ** (-np.arange(half) / half), rng.integers(0, 2, 128)
    up = mx.DeviceArray.from_numpy
    dx, dseq, dpos, drp, dinv, dqn, dkn = up(x), up(np.zeros(rows, np.int32)), up(pos), up(rope_pos), up(inv), up(qn), up(kn)
    rope = mx.RopeAxesC(rot, 2, dinv.ptr)
    for i in range(half):
        rope.pair_axis[i] = int(pair[i])
    dq, d = mx.DeviceArray((rows, heads, hd), np.uint16), c.dims()
    mx.check(mx.lib.mx_attn_paged_append(dx.ptr, width, rows, dseq.ptr, dpos.ptr, drp.ptr, C.byref(rope), dqn.ptr, dkn.ptr,
                                         1e-6, c.dtable.ptr, C.byref(d), *c.scales(), dq.ptr, c.dk.ptr, c.dv.ptr, None))
    mx.sync()
    f = lambda n: bf(n).astype(np.float64)  # noqa: E731
    q, k, v = reference_append(f(x), c, pos, rope_pos, inv, pair, rot, f(qn), f(kn))

    def fits(got, ref, half_step, least):
        size = np.abs(ref).max((1, 2), keepdims=True)
        assert (np.abs(got - ref) <= half_step * np.abs(ref) + least + 2.0 ** -20 * size).all()

    fits(f(dq.numpy()), q, HALF, 0)
    want = c.k.copy()
    got_k, got_v = c.kview(c.dk.numpy()), c.vview(c.dv.numpy())
    page_of, off = c.table[0, pos // page], pos % page
    if f8:
        fits(E4M3[got_k[page_of, :, off]], np.clip(k / c.ks[:, None], -448, 448), 2.0 ** -4, 2.0 ** -10)
        fits(E4M3[got_v[page_of, :, :, off]], np.clip(v / c.vs[:, None], -448, 448), 2.0 ** -4, 2.0 ** -10)
    else:
        fits(f(got_k[page_of, :, off]), k, HALF, 0)
        assert (f(got_v[page_of, :, :, off]) == v).all()
    rest = np.ones(c.kview().shape[0:1] + (page,), bool)
    rest[page_of, off] = False
    assert (got_k.transpose(0, 2, 1, 3)[rest] == c.kview(want).transpose(0, 2, 1, 3)[rest]).all()
    assert (got_v.transpose(0, 3, 1, 2)[rest] == c.vview(c.v).transpose(0, 3, 1, 2)[rest]).all()
