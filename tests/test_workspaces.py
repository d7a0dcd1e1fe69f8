"""Workspace sizes of the operators for serving: a workspace for a program's largest
batch serves every smaller one, so the sizes never fall as a call grows (no device:
the entry points cannot see how large a workspace is)."""
import ctypes as C

import pytest


@pytest.mark.parametrize("n", [1, 1000, 32000, 50257, 151936, 1 << 20])
def test_sampling_workspace_never_falls_with_rows(mx, n):
    sizes = [mx.lib.mx_sample_workspace_bytes(r, n) for r in range(1, 700)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])), [r + 2 for r, (a, b) in enumerate(zip(sizes, sizes[1:])) if a > b]
    assert 0 < sizes[0] and sizes[-1] == mx.lib.mx_sample_workspace_bytes(100000, n) < 1 << 27


@pytest.mark.parametrize("rows", [1, 8, 31, 32, 33, 64, 100, 255, 256, 300])
def test_sampling_workspace_never_falls_with_the_vocabulary(mx, rows):
    sizes = [mx.lib.mx_sample_workspace_bytes(rows, n) for n in range(1, 1 << 20, 511)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def dims(mx, heads, kv, hd, page=64, sequences=1, width=196):
    return mx.PageDimsC(heads, kv, hd, page, 1000, sequences, width, mx.MX_DT_BF16, 0, kv * page * hd)


@pytest.mark.parametrize("sequences", [1, 5, 64, 300])
@pytest.mark.parametrize("heads,kv,hd", [(16, 2, 256), (32, 8, 128), (28, 4, 128), (7, 1, 64), (5, 5, 128), (9, 9, 64)])
@pytest.mark.parametrize("width", [3, 196, 4000])
def test_prompt_workspace_never_falls_with_rows(mx, heads, kv, hd, sequences, width):
    d = dims(mx, heads, kv, hd, sequences=sequences, width=width)
    at = list(range(1, 1200)) + list(range(1200, 40000, 97))
    sizes = [mx.lib.mx_attn_paged_prefill_workspace_bytes(r, C.byref(d)) for r in at]
    assert all(a <= b for a, b in zip(sizes, sizes[1:])), [r for r, a, b in zip(at[1:], sizes, sizes[1:]) if a > b][:9]
    assert (sizes[0] > 0) == (width > 3)  # few rows that may see many keys are split
    # bounded: a split call has fewer than 1024 workgroups, of 128 pairs each
    assert mx.lib.mx_attn_paged_prefill_workspace_bytes(1 << 20, C.byref(d)) <= 1024 * 128 * (hd + 2) * 4


@pytest.mark.parametrize("rows", [1, 8, 64, 130, 1000])
def test_one_token_workspace_never_falls_with_rows(mx, rows):
    d = dims(mx, 16, 2, 256)
    f = mx.lib.mx_attn_paged_decode_workspace_bytes
    assert f(rows, C.byref(d)) < f(rows + 1, C.byref(d))


@pytest.mark.parametrize("rows", [1, 40, 512, 1500])
def test_idle_rows_of_the_table_do_not_change_a_prompts_shape(mx, rows):
    """How many workgroups share a prompt's keys follows from its rows, not from the sequences that have none."""
    f = mx.lib.mx_attn_paged_prefill_workspace_bytes
    sizes = {f(rows, C.byref(dims(mx, 16, 2, 256, sequences=s))) for s in (1, 2, 64, 300, 5000)}
    assert len(sizes) == 1 and sizes.pop() > 0
