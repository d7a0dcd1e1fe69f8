"""The latent cache's attentions where a score is -inf: the position has the weight 0, which leaves what the other
positions give but for NaN (0 times infinity) in the dims where its value is infinite; rows whose scores are all -inf
give zeros.  Bounds of finite results are those of test_latent_gpu.py."""
import numpy as np
import pytest

from latent_ref import Latent, softmax_rows
from paged_ref import to_bf
from test_latent_gpu import F, close, formed, queries, run_decode, run_prefill, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,nope,count,total", [
    (3, 128, 300, 300), (2, 64, 130, 130), (5, 128, 513, 700), (2, 128, 40, 1500), (3, 64, 150, 1200)])
def test_prompts(mx, heads, nope, count, total):
    """Keys whose score is -inf or +inf by the sign of a row's query, with infinite values: before all rows, in tiles
    that some rows see and some do not, and the first of all; whole and with the keys split."""
    say("scores of -inf", heads, nope, count, total)
    rng = np.random.default_rng(40 + count)
    q, qr, kv, kr = formed(rng, count, total, heads, nope)
    sign = np.where(rng.random((count, heads)) < 0.1, 1, -1)  # of the query against the infinite keys
    sign[:2] = -1
    qr[..., 1] = to_bf(0.3 * sign)
    v = kv.reshape(total, heads, 2 * nope)
    odd = {0: 7, (total - count) // 2 + 1: 3, total - count // 2: 5, total - 70: 6, total - 2: 9}  # positions, dims
    for at, dim in odd.items():
        kr[at, 1] = 0x7F80
        v[at, at % heads, nope + dim] = 0x7F80 if dim % 2 else 0xFF80
    got = F(run_prefill(mx, q, qr, kv, kr, [0, count], [0, total], heads, nope))
    places = np.array(sorted(odd))
    use = np.ones(total, bool)
    use[places] = False
    own = np.arange(total - count, total)
    seen = (np.arange(total) <= own[:, None]) & use
    some = seen.any(1)
    clean = np.where(np.isfinite(F(kv)), F(kv), 0).reshape(total, heads, 2 * nope)
    ks = np.where(np.isfinite(F(kr)), F(kr), 0)
    for h in range(heads):
        qn = F(q).reshape(count, heads, -1)[:, h, :nope]
        s = (qn @ clean[:, h, :nope].T + F(qr[:, h]) @ ks.T) * (nope + 64) ** -0.5
        p = np.zeros((count, total))
        p[some] = softmax_rows(np.where(seen, s, -np.inf)[some])
        ref, mag = p @ clean[:, h, nope:], p @ np.abs(clean[:, h, nope:])
        nan = np.zeros((count, nope), bool)
        for at in places:
            if at % heads == h:
                nan[own >= at, odd[at]] = True
        nan[~some] = False                                  # all scores -inf: zeros
        nan[(sign[:, h] > 0) & (own >= places[0])] = True   # a score of +inf: NaN throughout
        assert (np.isnan(got[:, h]) == nan).all(), (h, np.argwhere(np.isnan(got[:, h]) != nan)[:4])
        assert (got[:, h][~some] == 0).all()
        close(to_bf(np.where(nan, 0, got[:, h]).astype(np.float32)), np.where(nan, 0, ref), np.where(nan, 0, mag))


@pytest.mark.parametrize("count", [7, 40, 64, 200])
def test_an_infinite_value_in_the_first_tile(mx, count):
    """With finite scores it is infinite for the rows that see it, also where the softmax reference is first set."""
    heads, nope, at = 3, 128, 5
    say("first tile", count)
    q, qr, kv, kr = formed(np.random.default_rng(43), count, count, heads, nope)
    base = run_prefill(mx, q, qr, kv, kr, [0, count], [0, count], heads, nope)
    kv.reshape(count, heads, 2 * nope)[at, :, nope + 8] = 0x7F80
    got = run_prefill(mx, q, qr, kv, kr, [0, count], [0, count], heads, nope)
    assert (F(got)[at:, :, 8] == np.inf).all()
    same = np.ones(got.shape, bool)
    same[at:, :, 8] = False
    assert (got[same] == base[same]).all()


@pytest.mark.parametrize("heads", [7, 60, 128])
def test_one_token_rows_whose_scores_are_all_minus_infinity(mx, heads):
    say("all -inf", heads)
    lens = [1, 40, 700]
    c = Latent(mx, heads, 512, 16, lens, seed=41)
    for i, n in enumerate(lens):
        for p in range(n):
            c.view()[c.table[i, p // 16], p % 16, 512 + 2] = 0x7F80
    c.upload()
    ql, qr = queries(np.random.default_rng(42), 3, heads, 512)
    qr[..., 2] = to_bf(np.full(qr.shape[:2], -0.5))
    assert (F(run_decode(mx, c, ql, qr, lens)) == 0).all()
