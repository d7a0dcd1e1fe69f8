"""Argument checks of the paged-cache and sampling entry points (no device: a
refused call launches nothing, and pointers are never followed)."""
import ctypes as C

import pytest

P = 4096  # stands for any aligned pointer


def dims(mx, **over):
    d = dict(heads=16, kv_heads=2, head_dim=128, page_size=16, pages=10, sequences=3, table_width=5,
             dtype=mx.MX_DT_BF16, gated=0, page_stride=2 * 16 * 128)
    d.update(over)
    return mx.PageDimsC(**d)


BAD = [
    (dict(heads=0), "EINVAL"), (dict(kv_heads=0), "EINVAL"), (dict(heads=15), "EINVAL"),
    (dict(heads=34), "EUNSUPPORTED"), (dict(head_dim=96), "EUNSUPPORTED"), (dict(page_size=8), "EUNSUPPORTED"),
    (dict(page_size=48), "EUNSUPPORTED"), (dict(page_size=512), "EUNSUPPORTED"), (dict(pages=0), "EINVAL"),
    (dict(sequences=0), "EINVAL"), (dict(table_width=0), "EINVAL"), (dict(dtype=2), "EUNSUPPORTED"),
    (dict(gated=2), "EINVAL"), (dict(page_stride=4000), "EINVAL"), (dict(page_stride=4096 + 8), "EINVAL"),
    (dict(page_stride=1 << 59), "EINVAL"), (dict(table_width=1 << 28), "EUNSUPPORTED"),
    (dict(kv_heads=-2), "EINVAL"), (dict(heads=1 << 20, kv_heads=1 << 20, page_stride=1 << 31), "EUNSUPPORTED"),
]


def calls(mx, d, rows=2, **over):
    """The three entry points with good arguments but for `over`."""
    a = dict(q=P, qkv=P, stride=4096 + 1024, seqs=P, pos=P, rp=P, qn=P, kn=P, eps=1e-6, table=P, ks=None, vs=None, out=P,
             k=P, v=P, ws=P, scale=0.0, starts=P, lens=P, rope=mx.RopeAxesC(64, 3, P))
    a.update(over)
    dd = C.byref(d) if d is not None else None
    rope = C.byref(a["rope"]) if a["rope"] is not None else None
    return {
        "append": lambda: mx.lib.mx_attn_paged_append(a["qkv"], a["stride"], rows, a["seqs"], a["pos"], a["rp"], rope,
                                                      a["qn"], a["kn"], a["eps"], a["table"], dd, a["ks"], a["vs"],
                                                      a["out"], a["k"], a["v"], None),
        "decode": lambda: mx.lib.mx_attn_paged_decode(a["q"], a["qkv"], a["stride"], rows, a["seqs"], a["lens"],
                                                      a["table"], a["k"], a["v"], a["ks"], a["vs"], dd, a["scale"],
                                                      a["ws"], a["out"], None),
        "prefill": lambda: mx.lib.mx_attn_paged_prefill(a["q"], a["qkv"], a["stride"], rows, a["starts"], a["lens"],
                                                        a["table"], a["k"], a["v"], a["ks"], a["vs"], dd, a["scale"],
                                                        a["ws"], a["out"], None),
    }


@pytest.mark.parametrize("over,status", BAD)
def test_bad_caches_are_refused(mx, over, status):
    want = getattr(mx, "MX_" + status)
    for name, call in calls(mx, dims(mx, **over)).items():
        assert call() == want, (name, mx.lib.mx_last_error())
        assert f"mx_attn_paged_{name}: ".encode() in mx.lib.mx_last_error()
    d = dims(mx, **over)
    assert mx.lib.mx_attn_paged_decode_workspace_bytes(4, C.byref(d)) == 0
    assert mx.lib.mx_attn_paged_prefill_workspace_bytes(4, C.byref(d)) == 0


def test_null_pointers_and_rows(mx):
    d = dims(mx)
    for name, missing in (("append", "qkv pos table out k v rp"), ("decode", "q lens table k v ws out"),
                          ("prefill", "q starts lens table k v out")):
        for m in missing.split():
            assert calls(mx, d, **{m: None})[name]() == mx.MX_EINVAL, (name, m)
    wide = dims(mx, table_width=1000)  # few rows that may see many keys: split, with partials
    assert mx.lib.mx_attn_paged_prefill_workspace_bytes(2, C.byref(wide)) > 0
    assert calls(mx, wide, ws=None)["prefill"]() == mx.MX_EINVAL
    for call in calls(mx, None).values():
        assert call() == mx.MX_EINVAL
    for call in calls(mx, d, rows=-1).values():
        assert call() == mx.MX_EINVAL
    for call in calls(mx, d, rows=0).values():
        assert call() == mx.MX_OK  # nothing to do
    for name in ("decode", "prefill"):  # gated outputs need the rows with the gates
        assert calls(mx, dims(mx, gated=1), qkv=None)[name]() == mx.MX_EINVAL
        assert calls(mx, dims(mx, gated=1), stride=2 * 16 * 128 - 8)[name]() == mx.MX_EINVAL


def test_alignment_strides_and_scales(mx):
    d = dims(mx)
    for name, what in (("append", "qkv out k v qn kn"), ("decode", "q k v ws"), ("prefill", "q k v ws out")):
        for m in what.split():
            assert calls(mx, d, **{m: P + 8})[name]() == mx.MX_EUNSUPPORTED, (name, m)
    assert calls(mx, d, stride=20 * 128 - 8)["append"]() == mx.MX_EINVAL
    assert calls(mx, d, stride=20 * 128 + 4)["append"]() == mx.MX_EUNSUPPORTED
    for name in ("decode", "prefill"):
        assert calls(mx, dims(mx, gated=1), qkv=P + 2)[name]() == mx.MX_EUNSUPPORTED
        for s in (-1.0, float("nan"), float("inf")):
            assert calls(mx, d, scale=s)[name]() == mx.MX_EINVAL
    assert calls(mx, d, eps=-1.0)["append"]() == mx.MX_EINVAL
    assert calls(mx, d, eps=float("nan"))["append"]() == mx.MX_EINVAL


def test_rotary_descriptions(mx):
    d = dims(mx)
    for rot, axes in ((63, 1), (130, 1), (-2, 1), (64, 0), (64, 5)):
        assert calls(mx, d, rope=mx.RopeAxesC(rot, axes, P))["append"]() == mx.MX_EINVAL
    assert calls(mx, d, rope=mx.RopeAxesC(64, 1, None))["append"]() == mx.MX_EINVAL
    assert calls(mx, d, rope=None)["append"]() == mx.MX_EINVAL
    r = mx.RopeAxesC(64, 2, P)
    r.pair_axis[31] = 2
    assert calls(mx, d, rope=r)["append"]() == mx.MX_EINVAL
    assert b"pair_axis" in mx.lib.mx_last_error()


def test_workspaces_cover_any_lengths(mx):
    """The one-token workspace holds a partial for every chunk that any lengths give, and stops growing with the
    context once the target number of chunks is reached."""
    small = mx.lib.mx_attn_paged_decode_workspace_bytes(1, C.byref(dims(mx, table_width=1)))
    assert small >= 2 * 8 * 130 * 4
    a = mx.lib.mx_attn_paged_decode_workspace_bytes(8, C.byref(dims(mx, table_width=1 << 20)))
    b = mx.lib.mx_attn_paged_decode_workspace_bytes(8, C.byref(dims(mx, table_width=1 << 24)))
    assert a == b < 1 << 28
    assert mx.lib.mx_attn_paged_decode_workspace_bytes(0, C.byref(dims(mx))) == 0
    # prompts that fill the device need none
    assert mx.lib.mx_attn_paged_prefill_workspace_bytes(100000, C.byref(dims(mx))) == 0


def test_sampling_arguments(mx):
    f = lambda **o: (lambda a: mx.lib.mx_sample_bf16(a["l"], a["stride"], a["rows"], a["n"], None, None, None, None, a["u"],  # noqa: E731
                                                     a["t"], None, None, a["ws"], None))(
        dict(dict(l=P, stride=1000, rows=2, n=1000, u=P, t=P, ws=P), **o))
    assert f(rows=0) == mx.MX_OK
    for o in (dict(rows=-1), dict(n=0), dict(n=-5), dict(stride=999), dict(l=None), dict(u=None), dict(t=None)):
        assert f(**o) == mx.MX_EINVAL, o
    assert f(n=(1 << 20) + 1, stride=1 << 21) == mx.MX_EUNSUPPORTED
    assert f(ws=P + 4) == mx.MX_EUNSUPPORTED
    assert mx.lib.mx_sample_workspace_bytes(-1, 10) == 0
