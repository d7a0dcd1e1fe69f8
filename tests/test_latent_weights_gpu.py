"""Appended rows of models whose norm weights are plain and whose rotary pairs are interleaved."""
import ctypes as C

import numpy as np
import pytest

import test_latent_gpu as t
from latent_ref import ROPE, Latent
from paged_ref import to_bf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f8", [False, True])
def test_plain_norm_weights_and_interleaved_pairs(mx, f8):
    """A model with latents w x / rms(x) and rotary pairs (2 i, 2 i + 1): a norm of zeros normalises alone, w goes to
    the products that take the latents, and the rotary values of x and q are taken in the order 0, 2, .., 1, 3, ..
    What the cache stands for, times w, is the model's latent within the cache's own rounding, however small w."""
    rows, heads, nope, latent, page = 40, 5, 128, 512, 16
    t.say("plain weights", f8)
    rng = np.random.default_rng(64)
    c = Latent(mx, heads, latent, page, [rows], f8, nope, seed=65, fill=False)
    x = t.F(to_bf(2 * rng.standard_normal((rows, c.wide))))
    q = t.F(to_bf(rng.standard_normal((rows, heads, nope + ROPE))))
    w = np.exp(rng.uniform(np.log(1e-3), np.log(3), latent))
    order = np.concatenate([np.arange(0, ROPE, 2), np.arange(1, ROPE, 2)])
    inv, pos = 1e4 ** (-np.arange(32) / 32), np.arange(rows, dtype=np.int32)
    # as the model defines them
    norm = w * x[:, :latent] / np.sqrt((x[:, :latent] ** 2).mean(1, keepdims=True) + 1e-6)
    angle = pos[:, None] * inv

    def turned(v, angle):
        out = np.empty_like(v)
        out[..., ::2] = v[..., ::2] * np.cos(angle) - v[..., 1::2] * np.sin(angle)
        out[..., 1::2] = v[..., 1::2] * np.cos(angle) + v[..., ::2] * np.sin(angle)
        return out

    k_rot, q_rot = turned(x[:, latent:], angle), turned(q[..., nope:], angle[:, None])
    xp, qp = x.copy(), q.copy()
    xp[:, latent:], qp[..., nope:] = x[:, latent:][:, order], q[..., nope:][..., order]
    dx, dq, dp, dn, di = (t.up(mx, a) for a in (to_bf(xp), to_bf(qp), pos, np.zeros(latent, np.uint16), inv))
    rope, d, dr = mx.RopeAxesC(ROPE, 1, di.ptr), c.dims(), mx.DeviceArray((rows, heads, ROPE), np.uint16)
    zero = t.up(mx, np.zeros(rows, np.int32))
    mx.check(mx.lib.mx_attn_latent_append(dx.ptr, c.wide, dq.ptr, heads * (nope + ROPE), rows, zero.ptr, dp.ptr, dp.ptr,
                                          C.byref(rope), dn.ptr, 1e-6, c.dtable.ptr, C.byref(d), dr.ptr, c.dcache.ptr,
                                          c.pscales(), None))
    mx.sync()
    c.download()
    got, _ = c.values(0, rows)
    size = np.abs(np.concatenate([norm / w, k_rot], 1)).max(1, keepdims=True)
    # a rounding of e4m3 (2^-4, and half its smallest step, 2^-10, in units of the scale) or of bf16, and 2^-20 of the
    # largest value for the fp32 steps
    least = 2.0 ** -10 / 448 * 1.001 if f8 else 0
    rel = 2.0 ** -4 if f8 else t.HALF
    for mine, model, by in ((got[:, :latent] * w, norm, w), (got[:, latent:], k_rot[:, order], 1)):
        assert (np.abs(mine - model) <= rel * np.abs(model) + (least + 2.0 ** -20) * size * by).all()
    q_rot = q_rot[..., order]
    assert (np.abs(t.F(dr.numpy()) - q_rot) <= t.HALF * np.abs(q_rot) + 2.0 ** -20 * np.abs(q_rot).max()).all()
