"""Workspace sizes of the operators for serving: a workspace for a program's largest
batch serves every smaller one, so the sizes never fall as a call grows (no device:
the entry points cannot see how large a workspace is)."""
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
