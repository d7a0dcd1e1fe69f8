"""What the latent-cache tests share: a host copy of a latent cache, and its attention in 64 bits from
the definitions."""
import numpy as np

from paged_ref import E4M3, bf, to_bf, to_e4m3

ROPE = 64


class Latent:
    """A latent cache and its table on the device, with what its pages stand for on the host.

    contexts: positions each sequence holds; they are normal numbers in a random order of pages,
    and every position that no context covers is NaN (of e4m3 its scale too)."""

    def __init__(self, mx, heads, latent, page, contexts, f8=False, nope=128, seed=0, spare=2, stride_pad=0,
                 fill=True):
        self.mx, self.heads, self.latent, self.page, self.f8, self.nope = mx, heads, latent, page, f8, nope
        self.wide = latent + ROPE
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in contexts]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(contexts), max(max(need), 1)), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.stride = page * self.wide + stride_pad
        self.raw = np.full((self.pages, self.stride), 0x7F if f8 else 0x7FC1, np.uint8 if f8 else np.uint16)
        self.scales = np.full((self.pages, page), np.nan, np.float32) if f8 else None
        if fill:
            for i, n in enumerate(contexts):
                self.put(i, 0, rng.standard_normal((n, self.wide)))
        self.upload()

    def view(self, a=None):
        return (self.raw if a is None else a)[:, :self.page * self.wide].reshape(-1, self.page, self.wide)

    def put(self, seq, first, x):
        """Rounds x [n, latent + rope] into positions first .. of a sequence."""
        v = self.view().copy()
        for j, row in enumerate(x):
            pid, off = self.table[seq, (first + j) // self.page], (first + j) % self.page
            if self.f8:
                self.scales[pid, off] = np.float32(np.abs(row).max() / 448)
                v[pid, off] = to_e4m3(row / self.scales[pid, off])
            else:
                v[pid, off] = to_bf(row)
        self.raw[:, :self.page * self.wide] = v.reshape(self.pages, -1)

    def upload(self):
        up = self.mx.DeviceArray.from_numpy
        self.dcache, self.dtable = up(self.raw), up(self.table)
        self.dscales = up(self.scales) if self.f8 else None

    def download(self):
        self.raw = self.dcache.numpy()
        if self.f8:
            self.scales = self.dscales.numpy()

    def dims(self):
        mx = self.mx
        return mx.LatentDimsC(self.heads, self.nope, self.nope, self.latent, ROPE, self.page, self.pages, len(self.table),
                              self.table.shape[1], mx.MX_DT_F8E4M3 if self.f8 else mx.MX_DT_BF16, self.stride)

    def pscales(self):
        return self.dscales.ptr if self.f8 else None

    def values(self, seq, n):
        """Positions 0 .. n - 1 of a sequence [n, latent + rope] in 64 bits, and which of them lie in a page."""
        x, there = np.zeros((n, self.wide)), np.zeros(n, bool)
        v = self.view()
        for p in range(n):
            pid = self.table[seq, p // self.page]
            if 0 <= pid < self.pages:
                there[p] = True
                row = v[pid, p % self.page]
                x[p] = E4M3[row] * np.float64(self.scales[pid, p % self.page]) if self.f8 else bf(row)
        return x, there


def softmax_rows(s):
    p = np.exp(s - s.max(-1, keepdims=True))
    return p / p.sum(-1, keepdims=True)


def attend(c, seq, q_latent, q_rope, n, scale):
    """softmax(q x^T scale) c of one row (q [heads, ..]) that sees n positions, in 64 bits; also sum p |c|, which
    rounding errors of p scale with."""
    x, there = c.values(seq, n)
    x = x[there]
    if not len(x):
        z = np.zeros((c.heads, c.latent))
        return z, z
    p = softmax_rows(np.concatenate([q_latent, q_rope], 1) @ x.T * scale)
    return p @ x[:, :c.latent], p @ np.abs(x[:, :c.latent])


def attend_formed(q, q_rope, kv, k_rope, scale):
    """Causal attention of n last rows (q [n, heads, nope + rope]) over t positions kv [t, heads, 2 nope], in 64 bits."""
    n, heads = q.shape[:2]
    t, nope = kv.shape[0], kv.shape[2] // 2
    out, mag = np.zeros((n, heads, nope)), np.zeros((n, heads, nope))
    seen = np.arange(t) <= np.arange(t - n, t)[:, None]
    rows = seen.any(1)
    for h in range(heads):
        s = (q[:, h, :nope] @ kv[:, h, :nope].T + q_rope[:, h] @ k_rope.T) * scale
        p = np.zeros((n, t))
        if rows.any():
            p[rows] = softmax_rows(np.where(seen, s, -np.inf)[rows])
        out[:, h], mag[:, h] = p @ kv[:, h, nope:], p @ np.abs(kv[:, h, nope:])
    return out, mag
