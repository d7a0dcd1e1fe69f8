"""Argument checks of the latent-cache entry points, and how their workspaces grow (no device: a refused
call launches nothing, and pointers are never followed)."""
import ctypes as C

import pytest

P = 4096  # stands for any aligned pointer


def dims(mx, **over):
    d = dict(heads=20, nope_dim=128, v_dim=128, latent_dim=512, rope_dim=64, page_size=16, pages=10, sequences=3,
             table_width=5, dtype=mx.MX_DT_F8E4M3, page_stride=16 * 576)
    d.update(over)
    return mx.LatentDimsC(**d)


BAD = [
    (dict(heads=0), "EINVAL"), (dict(heads=-1), "EINVAL"), (dict(heads=129), "EUNSUPPORTED"),
    (dict(latent_dim=128), "EUNSUPPORTED"), (dict(latent_dim=0), "EUNSUPPORTED"), (dict(rope_dim=32), "EUNSUPPORTED"),
    (dict(nope_dim=64), "EUNSUPPORTED"), (dict(nope_dim=96, v_dim=96), "EUNSUPPORTED"), (dict(v_dim=64), "EUNSUPPORTED"),
    (dict(page_size=8), "EUNSUPPORTED"), (dict(page_size=48), "EUNSUPPORTED"), (dict(page_size=512), "EUNSUPPORTED"),
    (dict(pages=0), "EINVAL"), (dict(sequences=0), "EINVAL"), (dict(table_width=0), "EINVAL"),
    (dict(dtype=2), "EUNSUPPORTED"), (dict(page_stride=16 * 576 - 16), "EINVAL"),
    (dict(page_stride=16 * 576 + 8), "EINVAL"), (dict(page_stride=1 << 59), "EINVAL"),
    (dict(table_width=1 << 28), "EUNSUPPORTED"),
]


def calls(mx, d, rows=2, **over):
    """The entry points with good arguments but for `over`."""
    a = dict(x=P, x_stride=576, q=P, q_stride=20 * 192, seqs=P, pos=P, rp=P, rope=mx.RopeAxesC(64, 3, P), norm=P, eps=1e-6,
             table=P, q_rope=P, cache=P, scales=P, starts=P, first=P, latent=P, latent_stride=512, rot=P, rot_stride=64,
             q_latent=P, lens=P, scale=0.0, ws=P, out=P, kv=P, kv_stride=20 * 256, kv_rows=9, kv_starts=P)
    a.update(over)
    dd = C.byref(d) if d is not None else None
    rope = C.byref(a["rope"]) if a["rope"] is not None else None
    lib = mx.lib
    return {
        "append": lambda: lib.mx_attn_latent_append(a["x"], a["x_stride"], a["q"], a["q_stride"], rows, a["seqs"], a["pos"],
                                                    a["rp"], rope, a["norm"], a["eps"], a["table"], dd, a["q_rope"],
                                                    a["cache"], a["scales"], None),
        "read": lambda: lib.mx_attn_latent_read(a["cache"], a["scales"], rows, a["starts"], a["first"], a["table"], dd,
                                                a["latent"], a["latent_stride"], a["rot"], a["rot_stride"], None),
        "decode": lambda: lib.mx_attn_latent_decode(a["q_latent"], a["q_rope"], rows, a["seqs"], a["lens"], a["table"],
                                                    a["cache"], a["scales"], dd, a["scale"], a["ws"], a["out"], None),
        "prefill": lambda: lib.mx_attn_latent_prefill(a["q"], a["q_stride"], a["q_rope"], rows, a["starts"], a["kv"],
                                                      a["kv_stride"], a["rot"], a["rot_stride"], a["kv_rows"],
                                                      a["kv_starts"], dd, a["scale"], a["ws"], a["out"], None),
    }


@pytest.mark.parametrize("over,status", BAD)
def test_bad_caches_are_refused(mx, over, status):
    want = getattr(mx, "MX_" + status)
    d = dims(mx, **over)
    for name, call in calls(mx, d).items():
        assert call() == want, (name, mx.lib.mx_last_error())
        assert f"mx_attn_latent_{name}: ".encode() in mx.lib.mx_last_error()
    assert mx.lib.mx_attn_latent_decode_workspace_bytes(4, C.byref(d)) == 0
    assert mx.lib.mx_attn_latent_prefill_workspace_bytes(4, 4, C.byref(d)) == 0


def test_null_pointers_and_rows(mx):
    d = dims(mx)
    for name, missing in (("append", "x q pos rp rope table q_rope cache scales"),
                          ("read", "cache scales starts table latent rot"),
                          ("decode", "q_latent q_rope lens table cache scales ws out"),
                          ("prefill", "q q_rope starts kv rot kv_starts out")):
        for m in missing.split():
            assert calls(mx, d, **{m: None})[name]() == mx.MX_EINVAL, (name, m)
        assert calls(mx, None)[name]() == mx.MX_EINVAL
        assert calls(mx, d, rows=-1)[name]() == mx.MX_EINVAL
        assert calls(mx, d, rows=0)[name]() == mx.MX_OK
    assert calls(mx, d, kv_rows=-1)["prefill"]() == mx.MX_EINVAL
    assert mx.lib.mx_attn_latent_prefill_workspace_bytes(2, 4000, C.byref(d)) > 0
    assert calls(mx, d, kv_rows=4000, ws=None)["prefill"]() == mx.MX_EINVAL  # keys split, with partials


def test_strides_alignment_and_numbers(mx):
    d = dims(mx)
    for name, over in (("append", dict(x_stride=568)), ("append", dict(q_stride=20 * 192 - 8)),
                       ("append", dict(eps=-1.0)), ("append", dict(eps=float("nan"))),
                       ("append", dict(rope=mx.RopeAxesC(32, 1, P))), ("append", dict(rope=mx.RopeAxesC(64, 5, P))),
                       ("append", dict(rope=mx.RopeAxesC(64, 0, P))), ("append", dict(rope=mx.RopeAxesC(64, 1, None))),
                       ("read", dict(latent_stride=504)), ("read", dict(rot_stride=56)),
                       ("decode", dict(scale=-1.0)), ("decode", dict(scale=float("nan"))),
                       ("decode", dict(scale=float("inf"))), ("prefill", dict(scale=-1.0)),
                       ("prefill", dict(q_stride=20 * 192 - 8)), ("prefill", dict(kv_stride=20 * 256 - 8)),
                       ("prefill", dict(rot_stride=56))):
        assert calls(mx, d, **over)[name]() == mx.MX_EINVAL, (name, over)
    axis = mx.RopeAxesC(64, 2, P)
    axis.pair_axis[31] = 2
    assert calls(mx, d, rope=axis)["append"]() == mx.MX_EINVAL
    for name, over in (("append", "x q norm q_rope cache"), ("read", "cache latent rot"),
                       ("decode", "q_latent q_rope cache ws out"), ("prefill", "q q_rope kv rot ws out")):
        for m in over.split():
            assert calls(mx, d, **{m: P + 8})[name]() == mx.MX_EUNSUPPORTED, (name, m)
    for name, over in (("append", dict(x_stride=580)), ("append", dict(q_stride=20 * 192 + 4)),
                       ("read", dict(latent_stride=516)), ("read", dict(rot_stride=68)),
                       ("prefill", dict(q_stride=20 * 192 + 4)), ("prefill", dict(kv_stride=20 * 256 + 4)),
                       ("prefill", dict(rot_stride=68)), ("prefill", dict(kv_stride=1 << 29)),
                       ("prefill", dict(rows=1 << 30))):
        rows = over.pop("rows", 2)
        assert calls(mx, d, rows=rows, **over)[name]() == mx.MX_EUNSUPPORTED, (name, over)


@pytest.mark.parametrize("heads", [1, 32, 33, 64, 65, 128])
@pytest.mark.parametrize("latent", [256, 512])
def test_one_token_workspace_grows_with_rows(mx, heads, latent):
    d = dims(mx, heads=heads, latent_dim=latent, table_width=4000)
    f = mx.lib.mx_attn_latent_decode_workspace_bytes
    sizes = [f(r, C.byref(d)) for r in range(1, 300)]
    assert 0 < sizes[0] and all(a < b for a, b in zip(sizes, sizes[1:]))


@pytest.mark.parametrize("heads,nope", [(1, 128), (5, 64), (20, 128), (32, 128), (128, 128)])
def test_prompt_workspace_never_falls(mx, heads, nope):
    d = dims(mx, heads=heads, nope_dim=nope, v_dim=nope)
    f = mx.lib.mx_attn_latent_prefill_workspace_bytes
    for kv in (1, 300, 2000, 100000):
        sizes = [f(r, kv, C.byref(d)) for r in list(range(1, 900)) + list(range(900, 30000, 97))]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), kv
    for rows in (1, 100, 512):
        sizes = [f(rows, kv, C.byref(d)) for kv in range(1, 20000, 111)]
        assert all(a <= b for a, b in zip(sizes, sizes[1:])), rows
    # bounded: a split call has fewer than 1024 workgroups, of 128 rows each
    assert f(1 << 20, 1 << 20, C.byref(d)) <= 1024 * 128 * (nope + 2) * 4
    idle = dims(mx, heads=heads, nope_dim=nope, v_dim=nope, sequences=5000)  # sequences without rows
    assert f(40, 3000, C.byref(d)) == f(40, 3000, C.byref(idle))


def test_more_tiles_than_are_counted_are_refused(mx):
    """Rows times the tiles that the table allows each, of 32 positions and 8 more a row, must not pass 2^30."""
    wide = dims(mx, table_width=1 << 26)                  # 2^30 positions a row: 2^25 tiles
    for rows in (32, 33, 1 << 20):
        assert calls(mx, wide, rows=rows)["decode"]() == mx.MX_EUNSUPPORTED, rows
        assert b"mx_attn_latent_decode: " in mx.lib.mx_last_error()
    narrow = dims(mx, table_width=2)                      # one tile
    assert calls(mx, narrow, rows=(1 << 30) // 9 + 1)["decode"]() == mx.MX_EUNSUPPORTED
