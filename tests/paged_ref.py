"""What the paged-cache tests share: numpy conversions, a host copy of a paged
cache, and the operators in 64 bits from their definitions."""
import ctypes as C

import numpy as np


def bf(h):
    return (np.asarray(h, np.uint16).astype(np.uint32) << 16).view(np.float32)


def to_bf(x):
    """fp32 -> bf16 bits, to the nearest, ties to even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


# every e4m3 value by its byte: 4 exponent bits (bias 7), 3 of mantissa, no infinity
_b = np.arange(256)
_e, _m = (_b >> 3) & 15, _b & 7
E4M3 = np.where(_e > 0, (1 + _m / 8) * 2.0 ** (_e - 7), _m / 8 * 2.0 ** -6)
E4M3[(_b & 127) == 127] = np.nan
E4M3 = np.where(_b >= 128, -E4M3, E4M3)
_order = np.argsort(E4M3[:127], kind="stable")  # the non-negative ones ascend already
assert (_order == np.arange(127)).all()


def to_e4m3(x):
    """Bytes of the nearest e4m3 value (ties to the even byte), 448 beyond the largest."""
    a = np.minimum(np.abs(np.asarray(x, np.float64)), 448.0)
    hi = np.clip(np.searchsorted(E4M3[:127], a), 1, 126)
    lo = hi - 1
    dl, dh = a - E4M3[lo], E4M3[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return (pick | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


class Paged:
    """A paged cache and its table on the device, with what its pages stand for on the host.

    contexts: positions each sequence holds; K and V are normal numbers in a
    random order of pages, and every position that no context covers is NaN."""

    def __init__(self, mx, heads, kv_heads, hd, page, contexts, f8=False, gated=False, seed=0,
                 spare=2, stride_pad=0, table_width=None, fill=True):
        self.mx, self.heads, self.kv, self.hd, self.page = mx, heads, kv_heads, hd, page
        self.f8, self.gated, self.contexts = f8, gated, list(contexts)
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in contexts]
        self.pages = sum(need) + spare
        width = table_width or max(max(need), 1)
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(contexts), width), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.stride = kv_heads * page * hd + stride_pad
        item = np.uint8 if f8 else np.uint16
        nan = 0x7F if f8 else 0x7FC1
        self.k = np.full((self.pages, self.stride), nan, item)
        self.v = np.full((self.pages, self.stride), nan, item)
        self.ks = rng.uniform(0.01, 0.03, kv_heads).astype(np.float32) if f8 else None
        self.vs = rng.uniform(0.01, 0.03, kv_heads).astype(np.float32) if f8 else None
        if fill:
            for i, n in enumerate(contexts):
                self.put(i, 0, rng.standard_normal((n, kv_heads, hd)),
                         rng.standard_normal((n, kv_heads, hd)))
        self.upload()

    # views of a page array: K [pages, kv, page, hd], V [pages, kv, hd, page]
    def kview(self, a=None):
        n = self.kv * self.page * self.hd
        return (self.k if a is None else a)[:, :n].reshape(-1, self.kv, self.page, self.hd)

    def vview(self, a=None):
        n = self.kv * self.page * self.hd
        return (self.v if a is None else a)[:, :n].reshape(-1, self.kv, self.hd, self.page)

    def put(self, seq, first, k, v):
        """Rounds k, v [n, kv, hd] into positions first .. of a sequence."""
        kc, vc = self.kview(), self.vview()
        for j in range(len(k)):
            p = first + j
            pid, off = self.table[seq, p // self.page], p % self.page
            if self.f8:
                kc[pid, :, off] = to_e4m3(k[j] / self.ks[:, None])
                vc[pid, :, :, off] = to_e4m3(v[j] / self.vs[:, None])
            else:
                kc[pid, :, off] = to_bf(k[j])
                vc[pid, :, :, off] = to_bf(v[j])
        self.k[:, :kc[0].size] = kc.reshape(self.pages, -1)
        self.v[:, :vc[0].size] = vc.reshape(self.pages, -1)

    def upload(self):
        d = self.mx.DeviceArray.from_numpy
        self.dk, self.dv, self.dtable = d(self.k), d(self.v), d(self.table)
        self.dks, self.dvs = (d(self.ks), d(self.vs)) if self.f8 else (None, None)

    def dims(self):
        mx = self.mx
        return mx.PageDimsC(self.heads, self.kv, self.hd, self.page, self.pages, len(self.table),
                            self.table.shape[1], mx.MX_DT_F8E4M3 if self.f8 else mx.MX_DT_BF16,
                            int(self.gated), self.stride)

    def scales(self):
        return (self.dks.ptr, self.dvs.ptr) if self.f8 else (None, None)

    def values(self, seq, n):
        """K and V [n, kv, hd] in 64 bits and which positions lie in a page."""
        k, v = np.zeros((n, self.kv, self.hd)), np.zeros((n, self.kv, self.hd))
        there = np.zeros(n, bool)
        kc, vc = self.kview(), self.vview()
        for p in range(n):
            pid = self.table[seq, p // self.page]
            if not 0 <= pid < self.pages:
                continue
            there[p] = True
            a, b = kc[pid, :, p % self.page], vc[pid, :, :, p % self.page]
            if self.f8:
                k[p], v[p] = E4M3[a] * self.ks[:, None], E4M3[b] * self.vs[:, None]
            else:
                k[p], v[p] = bf(a), bf(b)
        return k, v, there


def attend(cache, seq, q, limits, scale=None):
    """softmax(q k^T scale) v in 64 bits for rows q [n, heads, hd] of one sequence that see positions
    below limits[i]; also sum p |v|, which rounding errors of p scale with."""
    n, heads, hd = q.shape
    group = heads // cache.kv
    most = max([0] + [int(x) for x in limits])
    k, v, there = cache.values(seq, most)
    out, mag = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    scale = hd ** -0.5 if scale is None else scale
    for i in range(n):
        use = there & (np.arange(most) < limits[i])
        if not use.any():
            continue
        for h in range(heads):
            kk, vv = k[use, h // group], v[use, h // group]
            s = kk @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mag[i, h] = p @ vv, p @ np.abs(vv)
    return out, mag


def gates(qkv, heads, hd):
    g = bf(qkv)[:, :2 * heads * hd].reshape(-1, heads, 2, hd)[:, :, 1].astype(np.float64)
    return 1 / (1 + np.exp(-g))


class Graph:
    """Work captured from a stream into a HIP graph, to be launched again."""

    def __init__(self, mx, stream, record):
        self.hip, self.stream = C.CDLL("libamdhip64.so"), C.c_void_p(stream)
        self._do("hipStreamBeginCapture", self.stream, 2)
        record()
        graph = C.c_void_p()
        self._do("hipStreamEndCapture", self.stream, C.byref(graph))
        self.exe = C.c_void_p()
        self._do("hipGraphInstantiate", C.byref(self.exe), graph, None, None, C.c_size_t(0))
        self._do("hipGraphDestroy", graph)

    def _do(self, name, *args):
        rc = getattr(self.hip, name)(*args)
        assert rc == 0, (name, rc)

    def launch(self):
        self._do("hipGraphLaunch", self.exe, self.stream)

    def close(self):
        self._do("hipGraphExecDestroy", self.exe)
