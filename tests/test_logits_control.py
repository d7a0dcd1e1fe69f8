"""Argument checks of mx_logits_control_bf16 (no device: a refused call launches nothing, and pointers are
never followed)."""
import ctypes as C

P = 4096


def call(mx, rows=2, n=1000, stride=1000, out_stride=1000, logits=P, out=2 * P, null=False, **over):
    a = dict(tokens=P, tokens_stride=50, prompt_lens=P, lens=P, seqs=P, sequences=4, repetition=P, frequency=P, presence=P,
             bias_starts=P, bias_tokens=P, bias_values=P, bias_count=3, masks=P, mask_rows=P, mask_stride=32, mask_states=1)
    a.update(over)
    c = mx.LogitsControlsC(**a)
    return mx.lib.mx_logits_control_bf16(logits, stride, rows, n, None if null else C.byref(c), out, out_stride, None)


def test_refusals(mx):
    for over in (dict(rows=-1), dict(n=0), dict(n=-5), dict(stride=999), dict(out_stride=999), dict(null=True),
                 dict(logits=None), dict(out=None), dict(lens=None), dict(tokens_stride=-1), dict(sequences=0),
                 dict(bias_tokens=None), dict(bias_values=None), dict(bias_count=-1), dict(mask_states=0),
                 dict(mask_stride=31), dict(logits=P, out=P, out_stride=1004)):
        assert call(mx, **over) == mx.MX_EINVAL, over
        assert b"mx_logits_control_bf16: " in mx.lib.mx_last_error()
    assert call(mx, rows=1 << 26, n=1 << 20, stride=1 << 20, out_stride=1 << 20, mask_stride=1 << 15) == mx.MX_EUNSUPPORTED
    assert call(mx, rows=0) == mx.MX_OK


def test_what_is_absent_is_not_asked_for(mx):
    none = dict(tokens=None, lens=None, sequences=0, masks=None, mask_states=0, mask_stride=0, bias_starts=None,
                bias_tokens=None, bias_values=None, bias_count=0, rows=0)
    assert call(mx, **none) == mx.MX_OK
    assert call(mx, rows=0, bias_count=0, bias_tokens=None, bias_values=None) == mx.MX_OK


def test_more_workgroups_than_a_launch_has_are_refused(mx):
    """The largest vocabulary too: its segments are counted in 64 bits."""
    n = (1 << 31) - 1
    assert call(mx, rows=1 << 20, n=n, stride=n, out_stride=n, mask_stride=1 << 26) == mx.MX_EUNSUPPORTED
