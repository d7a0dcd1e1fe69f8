"""mx_attn_paged_decode over values that are infinite or NaN where a row sees them:
such a value has a positive weight, so its output is infinite like it, NaN beside
one of the other sign or a NaN, and every other output stays as it was.  Bounds of
the finite ones as in test_paged_gpu.py."""
import numpy as np
import pytest

from paged_ref import Paged, attend, bf, gates, to_bf
from test_paged_gpu import close, run_decode

pytestmark = pytest.mark.gpu

INF, NINF, NAN = 0x7F80, 0xFF80, 0x7FC0


def say(*a):
    print(*a, flush=True)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("heads,kv,hd,page,total", [
    (16, 2, 256, 16, 200), (16, 2, 256, 64, 5000), (8, 2, 128, 32, 130), (32, 8, 128, 64, 3000), (6, 1, 64, 128, 1500),
    (4, 4, 64, 16, 90)])
def test_infinite_values_that_a_row_sees(mx, heads, kv, hd, page, total, gated):
    say("infinite", heads, kv, hd, page, total, gated)
    c = Paged(mx, heads, kv, hd, page, [total], False, gated, seed=30)
    rng = np.random.default_rng(31)
    lens = [total, total - 1, total // 2, 40, 3, 1]
    rows = len(lens)
    q = to_bf(0.5 * rng.standard_normal((rows, heads, hd)))
    qkv = to_bf(rng.standard_normal((rows, 2 * heads * hd))) if gated else None
    ref, mag = attend(c, 0, bf(q).astype(np.float64), lens)
    if gated:
        ref, mag = ref * gates(qkv, heads, hd), mag * gates(qkv, heads, hd)
    # (position, dim, bits) of kv head 0: alone at the first and last key and at places between, two of one
    # sign, two of either, beside a NaN
    odd = [(0, 0, INF), (total - 1, 1, NINF), (total // 3, 2, INF), (37, 3, NINF), (5, 4, INF), (total - 2, 4, INF),
           (6, 5, INF), (total // 2 + 1, 5, NINF), (7, 6, NAN), (8, hd - 1, NINF), (9, hd - 1, NAN), (2, 7, NINF)]
    vc = c.vview()
    for p, d, bits in odd:
        vc[c.table[0, p // page], 0, d, p % page] = bits
    c.v[:, :vc[0].size] = vc.reshape(c.pages, -1)
    c.upload()
    got = run_decode(mx, c, q, lens, seqs=[0] * rows, qkv=qkv)
    group, seen = heads // kv, np.zeros(got.shape, bool)
    g = bf(got).astype(np.float64)
    with np.errstate(invalid="ignore"):
        for r, n in enumerate(lens):
            for dim in {d for _, d, _ in odd}:
                some = [float(bf([b])[0]) for p, d, b in odd if d == dim and p < n]
                if not some:
                    continue
                seen[r, :group, dim] = True
                want = sum(some)  # inf, -inf or NaN
                np.testing.assert_array_equal(g[r, :group, dim], want, err_msg=f"row {r} dim {dim}")
    assert seen.any() and not seen.all()
    close(np.where(seen, 0, got).astype(np.uint16), np.where(seen, 0, ref), np.where(seen, 0, mag), True)
    assert (run_decode(mx, c, q, lens, seqs=[0] * rows, qkv=qkv) == got).all()


def test_infinite_values_of_missing_pages_and_past_the_end(mx):
    """What a row does not see stays unseen beside an infinite value that it does see."""
    heads, kv, hd, page, total = 8, 2, 128, 16, 100
    c = Paged(mx, heads, kv, hd, page, [total], seed=32)
    rng = np.random.default_rng(33)
    q = to_bf(0.5 * rng.standard_normal((2, heads, hd)))
    c.table[0, 2] = -1
    lens = [total - 3, 60]
    ref, mag = attend(c, 0, bf(q).astype(np.float64), lens)
    vc = c.vview()
    for p, d, bits in ((total - 2, 3, INF), (50, 4, INF), (61, 5, NINF)):
        vc[c.table[0, p // page], 1, d, p % page] = bits
    vc[sorted(set(range(c.pages)) - set(c.table[0].tolist()))] = NINF  # pages that no entry names
    c.v[:, :vc[0].size] = vc.reshape(c.pages, -1)
    c.upload()
    got = run_decode(mx, c, q, lens, seqs=[0, 0])
    g = bf(got)
    seen = np.zeros(got.shape, bool)
    seen[:, 4:, 4] = seen[0, 4:, 5] = True
    assert (g[:, 4:, 4] == np.inf).all() and (g[0, 4:, 5] == -np.inf).all()
    close(np.where(seen, 0, got).astype(np.uint16), np.where(seen, 0, ref), np.where(seen, 0, mag), True)
