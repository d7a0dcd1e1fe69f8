"""Rows of the latent-cache calls and of controls on logits that lie far apart, past 2^32 bytes and elements: the
results are those of packed rows, bit for bit, and nothing is written between them."""
import ctypes as C

import numpy as np
import pytest

import test_latent_gpu as t
from latent_ref import ROPE, Latent
from paged_ref import to_bf

pytestmark = pytest.mark.gpu


class Far:
    """Rows [n, width] `stride` elements apart on the device."""

    def __init__(self, mx, rows, stride):
        self.mx, self.rows, self.stride = mx, rows, stride
        n, self.width = rows.shape
        self.buf = mx.DeviceArray(((n - 1) * stride + self.width + 8,), np.uint16)
        self.ptr = self.buf.ptr
        for i in range(n):
            row = np.concatenate([rows[i], np.full(8, 0x4321, np.uint16)])
            mx.check(mx.lib.mx_memcpy_htod(self.ptr + 2 * i * stride, row.ctypes.data, row.nbytes))

    def numpy(self):
        out = np.empty((len(self.rows), self.width + 8), np.uint16)
        for i in range(len(out)):
            self.mx.check(self.mx.lib.mx_memcpy_dtoh(out[i].ctypes.data, self.ptr + 2 * i * self.stride, out[i].nbytes))
        assert (out[:, self.width:] == 0x4321).all()
        return out[:, :self.width]


def test_prompts(mx):
    heads, nope = 2, 128
    t.say("far prompt rows")
    new, total = [1, 6], [1, 65]
    starts, kv_starts = np.cumsum([0, *new]), np.cumsum([0, *total])
    q, qr, kv, kr = t.formed(np.random.default_rng(70), 7, 66, heads, nope)
    want = t.run_prefill(mx, q, qr, kv, kr, starts, kv_starts, heads, nope)
    t.check_prefill(want, q, qr, kv, kr, starts, kv_starts, heads, nope)
    d = mx.LatentDimsC(heads, nope, nope, 512, ROPE, 16, 1, 2, 1, mx.MX_DT_BF16, 16 * 576)
    ws = mx.DeviceArray((max(1, mx.lib.mx_attn_latent_prefill_workspace_bytes(7, 66, C.byref(d))),), np.uint8)
    fq, fkv, fkr = Far(mx, q, 1 << 30), Far(mx, kv, (1 << 28) - 8), Far(mx, kr, 1 << 27)
    dr, ds, dk = t.up(mx, qr), t.up(mx, starts.astype(np.int32)), t.up(mx, kv_starts.astype(np.int32))
    out = t.up(mx, np.full(want.shape, 0x1234, np.uint16))
    mx.check(mx.lib.mx_attn_latent_prefill(fq.ptr, fq.stride, dr.ptr, 7, ds.ptr, fkv.ptr, fkv.stride, fkr.ptr, fkr.stride,
                                           66, dk.ptr, C.byref(d), 0.0, ws.ptr, out.ptr, None))
    mx.sync()
    assert (out.numpy() == want).all()


@pytest.mark.parametrize("f8", [False, True])
def test_append_and_read(mx, f8):
    heads, latent, nope, rows = 3, 512, 128, 5
    t.say("far appended rows", f8)
    rng = np.random.default_rng(71)
    x, q = to_bf(rng.standard_normal((rows, latent + ROPE))), to_bf(rng.standard_normal((rows, heads * (nope + ROPE))))
    inv, pos, zero = (t.up(mx, a) for a in (1e4 ** (-np.arange(32) / 32), np.arange(rows, dtype=np.int32),
                                            np.zeros(rows, np.int32)))
    rope, got = mx.RopeAxesC(ROPE, 1, inv.ptr), []
    for far in (1 << 30, None):
        c = Latent(mx, heads, latent, 16, [rows], f8, nope, seed=72, fill=False)
        fx, fq = Far(mx, x, far or latent + ROPE + 8), Far(mx, q, far or heads * (nope + ROPE) + 8)
        dr, d = mx.DeviceArray((rows, heads, ROPE), np.uint16), c.dims()
        mx.check(mx.lib.mx_attn_latent_append(fx.ptr, fx.stride, fq.ptr, fq.stride, rows, zero.ptr, pos.ptr, pos.ptr,
                                              C.byref(rope), None, 0.0, c.dtable.ptr, C.byref(d), dr.ptr, c.dcache.ptr,
                                              c.pscales(), None))
        lat, rot = (Far(mx, np.full((rows, w), 0x1234, np.uint16), far or w + 8) for w in (latent, ROPE))
        starts = t.up(mx, np.array([0, rows], np.int32))
        mx.check(mx.lib.mx_attn_latent_read(c.dcache.ptr, c.pscales(), rows, starts.ptr, None, c.dtable.ptr, C.byref(d),
                                            lat.ptr, lat.stride, rot.ptr, rot.stride, None))
        mx.sync()
        c.download()
        got.append([dr.numpy(), c.raw, lat.numpy(), rot.numpy()])
    for a, b in zip(*got):
        assert (a == b).all()
    assert (t.F(got[0][2]) != 0).any(1).all()


def test_controls(mx):
    n, rows = 2100, 4
    t.say("far logits")
    rng = np.random.default_rng(73)
    logits = to_bf(rng.standard_normal((rows, n)))
    tokens, lens = rng.integers(0, n, (rows, 300)).astype(np.int32), np.array([300, 7, 0, 299], np.int32)
    dt, dl, rep = t.up(mx, tokens), t.up(mx, lens), t.up(mx, np.full(rows, 1.3, np.float32))
    c = mx.LogitsControlsC(tokens=dt.ptr, tokens_stride=300, lens=dl.ptr, sequences=rows, repetition=rep.ptr)
    got = []
    for far, in_place in ((1 << 31, False), (1 << 31, True), (n + 8, False)):
        src = Far(mx, logits, far)
        out = src if in_place else Far(mx, np.full_like(logits, 0x1234), far)
        mx.check(mx.lib.mx_logits_control_bf16(src.ptr, far, rows, n, C.byref(c), out.ptr, far, None))
        mx.sync()
        got.append(out.numpy())
    assert (got[0] == got[2]).all() and (got[1] == got[2]).all()
    seen = np.zeros((rows, n), bool)
    for r in range(rows):
        seen[r, tokens[r, :lens[r]]] = True
    assert ((got[2] != logits) <= seen).all() and (got[2] != logits).any()
