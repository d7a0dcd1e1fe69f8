"""How many bits of P the one-token attention over latents takes to its second product: 16 with up to 64 heads (two
bf16 parts), 8 with more.

Scores come from one rotary value alone, q k with q = 1 and a factor of 1, so that they are exact but for the
roundings below, and every p errs by:
  2^-16           the rounding of its second part, at most 2^-8 of a part that is at most 2^-8 of p
  16 * 2^-22      its exponent, of up to 16 in size, after three roundings of 2^-24 (the factor in log2 units, the
                  position's scale, the difference from the maximum)
  2^-22           the exponential, the product with the scale
and sums of up to 129 positions in fp32, of P V and of p, by 2 * 129 * 2^-24 < 2^-15.9.  Together less than 2^-14 of
sum p |v|, beside the output's own rounding 2^-8 |out|."""
import numpy as np
import pytest

from latent_ref import Latent, softmax_rows
from paged_ref import bf, to_bf
from test_latent_gpu import F, HALF, close, run_decode, say

pytestmark = pytest.mark.gpu

LENS = [1, 2, 9, 31, 32, 47, 64, 129]


def case(mx, heads, latent, f8):
    c = Latent(mx, heads, latent, 16, LENS, f8, seed=50 + heads, fill=False)
    rng = np.random.default_rng(51)
    for i, n in enumerate(LENS):
        x = rng.standard_normal((n, c.wide))
        x[:, latent:] = 0
        x[:, latent + 5] = rng.uniform(0, 3, n)
        c.put(i, 0, x)
    c.upload()
    ql = np.zeros((len(LENS), heads, latent), np.uint16)
    qr = np.zeros((len(LENS), heads, 64), np.uint16)
    qr[..., 5] = to_bf(rng.choice([0.25, 1, 1.5, 2], qr.shape[:2]))
    want = []
    for i, n in enumerate(LENS):
        x, _ = c.values(i, n)
        want.append((softmax_rows(F(qr[i, :, 5])[:, None] * x[:, latent + 5]), x[:, :latent]))
    return c, ql, qr, want


def off(got, p, v):
    """The largest error in units of the bound."""
    ref = p @ v
    return (np.abs(got - ref) / (HALF * np.abs(ref) + 2.0 ** -14 * (p @ np.abs(v)))).max()


def rounded(x):
    return bf(to_bf(x.astype(np.float32))).astype(np.float64)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,latent", [(1, 512), (20, 512), (32, 256), (33, 512), (64, 512), (64, 256)])
def test_sixteen_bits_with_up_to_64_heads(mx, heads, latent, f8):
    say("two parts", heads, latent, f8)
    c, ql, qr, want = case(mx, heads, latent, f8)
    got = F(run_decode(mx, c, ql, qr, LENS, scale=1.0))
    for i, (p, v) in enumerate(want):
        assert off(got[i], p, v) <= 1, LENS[i]
        if LENS[i] < 9:
            continue
        # the bound tells them from one part, of every p or of every second one
        w = p / p.max(1, keepdims=True)
        second = np.arange(LENS[i]) % 2 == 0
        for one in (rounded(w), np.where(second, rounded(w), w), np.where(second, w, rounded(w))):
            assert off(rounded(one @ v / w.sum(1, keepdims=True)), p, v) > 2, LENS[i]


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("heads,latent", [(65, 512), (128, 512), (100, 256)])
def test_eight_bits_with_more(mx, heads, latent, f8):
    say("one part", heads, latent, f8)
    c, ql, qr, want = case(mx, heads, latent, f8)
    got = run_decode(mx, c, ql, qr, LENS, scale=1.0)
    for i, (p, v) in enumerate(want):
        close(got[i], p @ v, p @ np.abs(v))
