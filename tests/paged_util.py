"""A paged cache in host memory, and append and attention over it computed row by row in 64 bits."""
import numpy as np

NAN_BF16 = 0x7FC0


def to_bf16(x):
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(NAN_BF16), r)


def from_bf16(b):
    return (np.ascontiguousarray(b, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


class HostCache:
    """Pools [pages, page_size, kv, D] (or head-major [pages, kv, page_size, D]) of bf16 bits, NaN wherever no sequence owns a row."""

    def __init__(self, rng, lens, page_size, kv, D, head_major=False, spare=2, room=0):
        self.lens, self.ps, self.kv, self.D, self.head_major = list(lens), page_size, kv, D, head_major
        need = [(n + room + page_size - 1) // page_size for n in lens]
        self.pages = sum(need) + spare
        self.table_stride = max(need + [1])
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.table_stride), -7, dtype=np.int32)   # entries nobody needs are no pages
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv, page_size, D) if head_major else (self.pages, page_size, kv, D)
        self.k = np.full(shape, NAN_BF16, dtype=np.uint16)
        self.v = np.full(shape, NAN_BF16, dtype=np.uint16)
        for s, n in enumerate(lens):
            self.put(s, np.arange(n), rng.standard_normal((n, kv, D)), rng.standard_normal((n, kv, D)) + 0.25)

    def rows(self, pool):
        return pool.transpose(0, 2, 1, 3) if self.head_major else pool

    def put(self, s, pos, k, v):
        page, off = self.table[s, pos // self.ps], pos % self.ps
        self.rows(self.k)[page, off] = to_bf16(k)
        self.rows(self.v)[page, off] = to_bf16(v)

    def get(self, s, n):
        pos = np.arange(n)
        page, off = self.table[s, pos // self.ps], pos % self.ps
        return (from_bf16(self.rows(p)[page, off]).astype(np.float64) for p in (self.k, self.v))

    def device(self, lthn):
        strides = dict(row_stride=self.D, head_stride=self.ps * self.D, page_stride=self.kv * self.ps * self.D) if self.head_major else {}
        return lthn.PagedKV(lthn.Buf.from_array(self.k), lthn.Buf.from_array(self.v), lthn.Buf.from_array(self.table), pages=self.pages,
                            page_size=self.ps, kv_heads=self.kv, head_dim=self.D, seqs=len(self.lens), table_stride=self.table_stride, **strides)


def attention(cache, s, q, pos0, length, *, scale=None, softcap=0.0, slopes=None, window=0, prefix=0):
    """q [n, Hq, D] at positions pos0.. of sequence s. Returns out, lse and sum_j weight_j |v_j| (what a relative error of the
    weights is multiplied with), all f64."""
    n, Hq, D = q.shape
    G = Hq // cache.kv
    scale = scale or 1.0 / np.sqrt(D)
    out, mag = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    lse = np.full((n, Hq), -np.inf)
    if length <= 0:
        return out, lse, mag
    k, v = cache.get(s, length)
    i, j = pos0 + np.arange(n)[:, None], np.arange(length)[None]
    seen = (j <= i) & ((window == 0) | (j > i - window)) | (j < prefix)
    some = seen.any(1)
    for h in range(Hq):
        x = q[:, h].astype(np.float64) @ k[:, h // G].T * scale
        if softcap:
            x = softcap * np.tanh(x / softcap)
        if slopes is not None:
            x = x - np.float64(slopes[h]) * np.abs(i - j)
        x = np.where(seen, x, -np.inf)
        m = np.where(some, x.max(1), 0.0)[:, None]
        w = np.exp(x - m)
        t = w.sum(1)
        w = w / np.where(some, t, 1.0)[:, None]
        out[:, h], mag[:, h] = w @ v[:, h // G], w @ np.abs(v[:, h // G])
        lse[some, h] = (m[:, 0] + np.log(np.where(some, t, 1.0)))[some]
    return out, lse, mag


def turn(x, pos, inv_freq, interleaved=False, w=None, eps=1e-6):
    """x [rows, heads, D] f64 through the norm and the rotation."""
    x = x.astype(np.float64).copy()
    D = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    if inv_freq is not None:
        h = len(inv_freq)
        t = np.asarray(pos, dtype=np.float64)[:, None] * inv_freq[None]
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        lo = 2 * np.arange(h) if interleaved else np.arange(h)
        hi = lo + 1 if interleaved else lo + D // 2
        a, b = x[..., lo].copy(), x[..., hi].copy()
        x[..., lo], x[..., hi] = a * c - b * s, a * s + b * c
    return x
