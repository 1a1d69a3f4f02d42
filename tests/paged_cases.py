"""Plain 64-bit forms of the paged-cache operators and the types' encodings, for
the tests of moe_paged_*_dev."""
import ctypes

import numpy as np

F32, F16, BF16, E4M3 = 0, 1, 4, 5
TYPES = {"f32": F32, "f16": F16, "bf16": BF16, "e4m3": E4M3}
RAW = {F32: np.float32, F16: np.uint16, BF16: np.uint16, E4M3: np.uint8}
NAN_BITS = {F32: 0x7fc00000, F16: 0x7e00, BF16: 0x7fc0, E4M3: 0x7f}
INF_BITS = {F32: 0xff800000, F16: 0x7c00, BF16: 0xff80, E4M3: 0xff}   # (e4m3 has no infinity: its other NaN)
# half a step relative to the value, and half the smallest step of all
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8, E4M3: 2.0 ** -4}
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134, E4M3: 2.0 ** -10}
U = 2.0 ** -24   # half a step of fp32


def _e4m3_values():
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(b & 127) == 127] = np.nan
    return np.where(b >> 7, -v, v)


E4M3_VALUES = _e4m3_values()


def decode(raw, dtype):
    if dtype == F32:
        return raw.astype(np.float64)
    if dtype == F16:
        return raw.view(np.float16).astype(np.float64)
    if dtype == BF16:
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return E4M3_VALUES[raw]


def encode(x, dtype):
    """fp32 -> raw, to nearest even (e4m3 saturated)"""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == F32:
        return x
    if dtype == F16:
        return x.astype(np.float16).view(np.uint16)
    if dtype == BF16:
        u = x.view(np.uint32).astype(np.uint64)
        return ((u + 0x7fff + (u >> 16 & 1)) >> 16).astype(np.uint16)
    a = np.minimum(np.abs(x).astype(np.float64), 448.0)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 1e-30))), -6)
    n = np.rint(a / 2.0 ** (e - 3))   # steps of 2^(e-3), 8..16
    code = np.where(n >= 16, (e + 8) * 8, np.where(n >= 8, (e + 7) * 8 + n - 8, n)).astype(np.int64)
    return (code | (np.signbit(x).astype(np.int64) << 7)).astype(np.uint8)


def nan_fill(shape, dtype):
    """a pool that holds NaNs and infinities wherever nothing was written"""
    a = np.empty(shape, RAW[dtype])
    bits = a.view(np.uint32) if dtype == F32 else a
    bits[...] = NAN_BITS[dtype]
    bits.reshape(-1)[::3] = INF_BITS[dtype]
    return a


def attend(q, k, v, scale):
    """One row: q [nq, hd], k and v [len, nkv, hd] in 64 bits -> (out [nq, hd], bound on an fp32 evaluation's error).

    The bound: a score's products and sums lose (hd + 8) half steps of the sum of its products' sizes; an exponential's
    argument 4 of its size; a weight's relative error is that twice (its own and the largest score's) and the sums over
    the positions lose len + 32 half steps more, all of it against sum p |v|."""
    nq, hd = q.shape
    n, nkv = k.shape[:2]
    if n == 0:
        return np.zeros((nq, hd)), np.zeros((nq, hd))
    g = nq // nkv
    out, tol = np.empty((nq, hd)), np.empty((nq, hd))
    for h in range(nq):
        kh, vh = k[:, h // g], v[:, h // g]
        s = scale * (kh @ q[h])
        size = abs(scale) * np.max(np.abs(kh) @ np.abs(q[h]))
        p = np.exp(s - s.max())
        out[h] = p @ vh / p.sum()
        delta = 2 * (hd + 8) * U * size + 4 * U * (s.max() - s.min()) + 8 * U
        tol[h] = (2 * delta + (n + 32) * U) * (p @ np.abs(vh)) / p.sum() + 1e-30
    return out, tol


def rope_tables(n, dim, theta=1e4):
    a = np.arange(n)[:, None] * theta ** (-np.arange(0, dim, 2) / max(dim, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def turn_head(x, w, eps, cos, sin, rope_dim):
    """[.., hd] rows in 64 bits -> (normed and turned, bound on an fp32 evaluation's error)"""
    hd = x.shape[-1]
    y = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    tol = np.abs(y) * ((hd / 2 + 8) * U if w is not None else 0.0)
    h = rope_dim // 2
    if not h:
        return y, tol
    a, b = y[..., :h], y[..., h:rope_dim]
    size = np.abs(a) + np.abs(b)
    both = size * (hd / 2 + 12) * U
    return (np.concatenate([a * cos - b * sin, b * cos + a * sin, y[..., rope_dim:]], -1),
            np.concatenate([both, both, tol[..., rope_dim:]], -1))


class Pool:
    """Host image of one layer's pages and its device copy.  order: "slot", "head" or "shared" (K and V in one pool)."""

    def __init__(self, M, dtype, n_pages, page_size, n_kv, hd, order="slot", k_scale=None, v_scale=None):
        self.M, self.dtype, self.n_pages, self.ps, self.n_kv, self.hd = M, dtype, n_pages, page_size, n_kv, hd
        lanes = 2 if order == "shared" else 1
        slot, head = (n_kv * hd, hd) if order != "head" else (hd, page_size * hd)
        page = page_size * n_kv * hd
        self.strides = (page * lanes, head, slot)
        raw = nan_fill((n_pages, lanes, page), dtype) if order == "shared" else nan_fill((2, n_pages, page), dtype)
        self.raw = raw
        sides = (raw[:, 0], raw[:, 1]) if order == "shared" else (raw[0], raw[1])
        shape = (n_pages, page_size, n_kv, hd) if order != "head" else (n_pages, n_kv, page_size, hd)
        self.k, self.v = (np.lib.stride_tricks.as_strided(s, shape, [self.strides[0] * raw.itemsize] + [
            i * raw.itemsize for i in ((slot, head, 1) if order != "head" else (head, slot, 1))]) for s in sides)
        if order == "head":
            self.k, self.v = self.k.transpose(0, 2, 1, 3), self.v.transpose(0, 2, 1, 3)   # [page, offset, head, dim]
        self.scales = [None if s is None else np.asarray(s, np.float32) for s in (k_scale, v_scale)]
        self.buf = M.DeviceBuffer.from_array(raw)
        self.sbuf = [None if s is None else M.DeviceBuffer.from_array(s) for s in self.scales]
        gap = page if order == "shared" else page * n_pages
        self.pages = M.Pages(self.buf.ptr, self.buf.ptr + gap * raw.itemsize, dtype, n_pages, page_size, n_kv, hd, *self.strides,
                             *[None if s is None else s.ptr for s in self.sbuf])

    def factor(self, side):
        s = self.scales[side]
        return np.ones((self.n_kv, 1)) if s is None else s.astype(np.float64)[:, None]

    def put(self, page, off, k, v):
        """fp32 rows [n_kv, hd] into a slot of the host image"""
        for side, (pool, x) in enumerate(((self.k, k), (self.v, v))):
            pool[page, off] = encode((x / self.factor(side)).astype(np.float32), self.dtype)

    def upload(self):
        self.buf.upload(self.raw)

    def download(self):
        self.raw[...] = self.buf.download(self.raw.shape, self.raw.dtype)

    def rows(self, table, n):
        """keys and values of positions 0 .. n - 1 in 64 bits"""
        p = np.arange(n)
        at = np.asarray(table, np.int64)[p // self.ps], p % self.ps
        return (decode(np.ascontiguousarray(self.k[at]), self.dtype) * self.factor(0),
                decode(np.ascontiguousarray(self.v[at]), self.dtype) * self.factor(1))


def ref(a):
    return ctypes.byref(a)
