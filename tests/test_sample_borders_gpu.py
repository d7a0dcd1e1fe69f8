"""mx_sample_bf16 where the sampled mass meets the kept mass or a border between
two values: every row with a token above -inf is given one of its kept tokens,
also where the prefix sums' rounding decides.  Outputs start as a value that no
call writes.

Prefix masses are 64-bit sums of at most 1024 + 64 terms, each rounded by at most
2^-53 of the sum, and u times the mass rounds once more: together under 2^-42 of
the mass.  Within that of a border either neighbour is right."""
import numpy as np
import pytest

from paged_ref import bf, to_bf
from test_sample_gpu import reference

pytestmark = pytest.mark.gpu

UNWRITTEN = 0xDEADBEEF


def sample(mx, logits, t=None, k=None, p=None, mp=None, u=None):
    rows, n = logits.shape
    up = mx.DeviceArray.from_numpy
    dl, du = up(logits), up(np.asarray(u, np.float32))
    par = [None if a is None else up(np.asarray(a, dt)) for a, dt in
           ((t, np.float32), (k, np.int32), (p, np.float32), (mp, np.float32))]
    tok, lp, kept = up(np.full(rows, UNWRITTEN, np.uint32)), up(np.full(rows, 7.0, np.float32)), \
        up(np.full(rows, -7, np.int32))
    ws = mx.DeviceArray((max(1, mx.lib.mx_sample_workspace_bytes(rows, n)),), np.uint8)
    mx.check(mx.lib.mx_sample_bf16(dl.ptr, n, rows, n, *[a.ptr if a else None for a in par], du.ptr, tok.ptr, lp.ptr,
                                   kept.ptr, ws.ptr, None))
    mx.sync()
    return tok.numpy(), kept.numpy(), lp.numpy()


def allowed(row, t, kept, u):
    """Tokens whose stretch of the kept mass u times that mass falls into, within the sums' rounding."""
    x = bf(row).astype(np.longdouble)
    order = np.argsort(-bf(row), kind="stable")[:kept]
    cum = np.cumsum(np.exp((x[order] - x[order[0]]) / np.longdouble(np.float32(t))))
    at, d = np.longdouble(np.float32(u)) * cum[-1], cum[-1] * 2.0 ** -42
    before = np.concatenate([[0], cum[:-1]])
    return set(order[(before <= at + d) & (cum >= at - d)].tolist())


# 40 logits with temperature 1.69165277, top-k 19 and uniform 0.797730803: the sampled mass lies between the
# prefix of the last value before a run of values that do not occur and the same prefix summed in another order
GAP = """3e4c 400c c070 be3d 408b 3f01 be82 c0a5 3fe5 3db7 3f4b c0a2 3dad 3e86 3e4b 3cca c017 c032 3d82 4040 3f66 bd8a c011 bfa9
 bd6a be4d be01 be03 3e62 bff1 3e3d bf7d be9c bd5b 3fbc 4010 bdaa 3ffa 3e92 3cd7"""


def test_a_border_before_values_that_do_not_occur(mx):
    row = np.array([int(h, 16) for h in GAP.split()], np.uint16)
    t, u = np.float32(1.69165277), np.float32(0.797730803)
    for rows in (1, 40):
        tok, kept, lp = sample(mx, np.tile(row, (rows, 1)), t=np.full(rows, t), k=np.full(rows, 19), u=np.full(rows, u))
        assert (kept == 19).all() and np.isfinite(lp).all() and (tok == tok[0]).all()
        assert int(tok[0]) in allowed(row, t, 19, u)


@pytest.mark.parametrize("n", [16, 30, 45, 70, 100, 150, 200, 300, 3001])
def test_the_whole_kept_mass_is_the_last_kept_token(mx, n):
    print("whole mass", n, flush=True)
    rows = 512
    rng = np.random.default_rng(n)
    logits = to_bf(2 * rng.standard_normal((rows, n)))
    logits[rows // 2:] = to_bf(40 * rng.standard_normal((rows // 2, n)))  # weights far below the sums' rounding too
    f = np.float32
    for k, p, mp in ((None, None, None), (rng.integers(1, n + 1, rows), None, None),
                     (None, f(0.5) + f(0.5) * rng.random(rows).astype(f), None), (None, None, rng.random(rows).astype(f)),
                     (rng.integers(1, n + 1, rows), f(0.5) + f(0.5) * rng.random(rows).astype(f), None)):
        at = lambda a, r, v: v if a is None else a[r]  # noqa: E731
        tok, kept, lp = sample(mx, logits, k=k, p=p, mp=mp, u=np.ones(rows))
        for r in range(rows):
            want = reference(logits[r], f(1), at(k, r, 0), at(p, r, f(1)), at(mp, r, f(0)), f(1))
            assert (int(tok[r]), int(kept[r])) == want[:2], (r, tok[r], kept[r], want)
            assert abs(lp[r] - want[2]) <= 2.0 ** -23 * abs(want[2]) + 1e-12, (r, lp[r], want)


@pytest.mark.parametrize("n", [40, 130, 1000])
def test_uniforms_next_to_borders(mx, n):
    """Uniform numbers that are the nearest fp32 to a border between two tokens, and their neighbours."""
    print("borders", n, flush=True)
    rows = 600
    rng = np.random.default_rng(n + 1)
    logits = to_bf(2 * rng.standard_normal((rows, n)))
    t = (0.5 + rng.random(rows)).astype(np.float32)
    u = np.empty(rows, np.float32)
    for r in range(rows):
        x = np.sort(bf(logits[r]).astype(np.float64))[::-1]
        cum = np.cumsum(np.exp((x - x[0]) / np.float64(t[r])))
        u[r] = np.float32(cum[rng.integers(0, n)] / cum[-1])
    u[1::3] = np.nextafter(u[1::3], np.float32(0))
    u[2::3] = np.nextafter(u[2::3], np.float32(1))
    tok, kept, lp = sample(mx, logits, t=t, u=u)
    assert (kept == n).all() and np.isfinite(lp).all()
    for r in range(rows):
        assert int(tok[r]) in allowed(logits[r], t[r], n, u[r]), (r, tok[r])
