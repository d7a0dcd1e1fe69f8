"""mx_attn_paged_prefill's launch shapes against 64-bit evaluations, every row
compared: few and many workgroups, with the keys split and whole, in tables with
idle rows.  Bounds as in test_paged_gpu.py."""
import numpy as np
import pytest

from paged_ref import E4M3, Paged, bf, to_bf, to_e4m3
from test_paged_gpu import close, run_prefill

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


class Filled(Paged):
    """A cache whose pages are filled at once (positions past a length are numbers too)."""

    def __init__(self, mx, heads, kv, hd, page, contexts, f8=False, seed=0, **more):
        super().__init__(mx, heads, kv, hd, page, contexts, f8, False, seed=seed, fill=False, **more)
        rng = np.random.default_rng(seed + 1)
        some = rng.standard_normal(1 << 16)  # rounded once, and drawn from
        for to, scale in ((self.k, self.ks), (self.v, self.vs)):
            for h in range(kv):
                x = to_e4m3(some / scale[h]) if f8 else to_bf(some)
                to[:, h * page * hd:(h + 1) * page * hd] = x[rng.integers(0, 1 << 16, (self.pages, page * hd), np.uint16)]
        self.upload()

    def sequence(self, seq, n):
        """K and V [kv, n, hd] of a sequence whose pages are all there, in 64 bits."""
        at = self.table[seq, :-(-n // self.page)]
        k = self.kview()[at].transpose(1, 0, 2, 3).reshape(self.kv, -1, self.hd)[:, :n]
        v = self.vview()[at].transpose(1, 0, 3, 2).reshape(self.kv, -1, self.hd)[:, :n]
        if self.f8:
            return E4M3[k] * self.ks[:, None, None], E4M3[v] * self.vs[:, None, None]
        return bf(k).astype(np.float64), bf(v).astype(np.float64)


def attend_rows(c, seq, q, limits):
    """softmax(q k^T / sqrt(hd)) v of rows q [n, heads, hd] that see positions below limits[i], and sum p |v|."""
    n, heads, hd = q.shape
    k, v = c.sequence(seq, int(max(limits)))
    out, mag = np.empty((n, heads, hd)), np.empty((n, heads, hd))
    hidden = np.arange(k.shape[1]) >= np.asarray(limits)[:, None]
    for h in range(heads):
        g = h // (heads // c.kv)
        s = q[:, h] @ k[g].T * hd ** -0.5
        s[hidden] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h], mag[:, h] = p @ v[g], p @ np.abs(v[g])
    return out, mag


# q heads, kv heads, head dim, page, (rows, positions) of every sequence, workgroups: below 257, up to 512 (where
# the second 256 take the blocks from the last on) and above; kv heads times splits below 8 and in whole XCDs
PROMPTS = [
    (16, 1, 64, 16, [(n, n + 7 * i) for i, n in enumerate((150, 3, 200, 90, 170, 1, 240, 210, 130, 88, 160, 230, 190, 37, 210, 240))]),
    (16, 8, 128, 32, [(500, 500), (131, 400), (1, 290), (700, 700), (260, 300), (333, 480)]),
    (8, 2, 128, 64, [(500, 4200)]),
    (16, 1, 64, 32, [(300, 1300), (20, 40), (410, 900), (60, 1250)]),
    (16, 8, 64, 128, [(1000, 1100), (64, 65), (1500, 1500), (900, 1000), (128, 300), (77, 77), (831, 901)]),
    (4, 2, 256, 16, [(90, 2000), (7, 7), (200, 700)]),
]


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts_of_many_workgroups(mx, case, f8):
    heads, kv, hd, page, seqs = PROMPTS[case]
    say("prompts", case, f8)
    c = Filled(mx, heads, kv, hd, page, [n for _, n in seqs], f8, seed=40 + case)
    starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
    rng = np.random.default_rng(41)
    q = to_bf(0.5 * rng.standard_normal((starts[-1], heads, hd)))
    got = run_prefill(mx, c, q, starts, [n for _, n in seqs])
    for s, (n, total) in enumerate(seqs):
        at = slice(starts[s], starts[s + 1])
        close(got[at], *attend_rows(c, s, bf(q[at]).astype(np.float64), total - n + np.arange(n) + 1), False)
    assert (run_prefill(mx, c, q, starts, [n for _, n in seqs]) == got).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,kv,hd,count,total", [(16, 2, 256, 64, 2100), (8, 1, 128, 200, 3000), (8, 8, 64, 1, 4000)])
def test_idle_rows_of_the_table_change_nothing(mx, heads, kv, hd, count, total, f8):
    """A prompt of one sequence among 300 is shared out, and rounded, as it is alone; packed rows that no
    sequence has keep their outputs."""
    say("idle", heads, kv, hd, count, total, f8)
    c = Filled(mx, heads, kv, hd, 64, [total], f8, seed=50)
    rng = np.random.default_rng(51)
    q = to_bf(0.5 * rng.standard_normal((count, heads, hd)))
    alone = run_prefill(mx, c, q, [0, count], [total])
    close(alone, *attend_rows(c, 0, bf(q).astype(np.float64), total - count + np.arange(count) + 1), False)
    row = c.table[0].copy()
    for rows, mine in ((64, 63), (300, 0), (300, 64), (300, 150), (300, 299)):
        c.table = np.full((rows, len(row)), -1, np.int32)
        c.table[mine] = row
        c.upload()
        lens = np.full(rows, 77, np.int32)  # of sequences without rows in this call
        lens[mine] = total
        starts = np.where(np.arange(rows + 1) > mine, count, 0)
        assert (run_prefill(mx, c, q, starts, lens) == alone).all(), (rows, mine)
    more = np.concatenate([q, q[:5]])
    got = run_prefill(mx, c, more, starts, lens)
    close(got[:count], *attend_rows(c, 299, bf(q).astype(np.float64), total - count + np.arange(count) + 1), False)
    assert (got[count:] == 0x1234).all()


@pytest.mark.parametrize("heads,kv,hd,count,total", [(16, 2, 256, 64, 2100), (8, 2, 128, 40, 3000), (4, 4, 64, 90, 2500)])
def test_infinite_values_of_later_rows_with_the_keys_split(mx, heads, kv, hd, count, total):
    say("split infinities", heads, kv, hd)
    c = Filled(mx, heads, kv, hd, 32, [total], seed=60)
    rng = np.random.default_rng(61)
    q = to_bf(0.5 * rng.standard_normal((count, heads, hd)))
    limits = total - count + np.arange(count) + 1
    ref, mag = attend_rows(c, 0, bf(q).astype(np.float64), limits)
    vc, seen = c.vview(), np.zeros(q.shape, bool)
    group = heads // kv
    # among the prompt's own rows, and one in an early split that every row sees
    for p, d, bits in ((total - 30, 3, 0x7F80), (total - 7, 9, 0xFF80), (total - 20, hd - 1, 0x7FC0), (100, 5, 0x7F80)):
        vc[c.table[0, p // 32], 0, d, p % 32] = bits
        seen[limits > p, :group, d] = True
    c.v[:, :vc[0].size] = vc.reshape(c.pages, -1)
    c.upload()
    got = run_prefill(mx, c, q, [0, count], [total])
    g = bf(got)
    assert not np.isfinite(g[seen]).any() and (g[:, :group, 5] == np.inf).all()
    assert (g[limits > total - 30, :group, 3] == np.inf).all() and (g[limits > total - 7, :group, 9] == -np.inf).all()
    close(np.where(seen, 0, got).astype(np.uint16), np.where(seen, 0, ref), np.where(seen, 0, mag), False)
