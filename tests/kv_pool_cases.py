"""Pools of key/value pages for the tests: the stored form worked out with numpy, page tables in no order, and attention in 64 bits."""

import numpy as np

from bobcat_b200 import F16, I8, KvPool, KvRows

NAN_HALF, NAN_BYTE = 0x7E00, 0xFF


def stored(x: np.ndarray, fmt: int):
    """What a page holds of rows x [..., hd] (f32): halves, or (bytes, scales)."""
    if fmt == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16), None
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = np.abs(x).max(axis=-1)
        scale = (top.astype(np.float64) / 127.0).astype(np.float32)
        scale = np.where(scale < np.float32(2.0) ** -126, np.float32(0), scale)
        whole = np.rint(x.astype(np.float64) / scale[..., None].astype(np.float64))
        whole = np.clip(np.where(scale[..., None] > 0, whole, 0.0), -127, 127)
        bad = ~np.isfinite(x).all(axis=-1)
        whole = np.where(bad[..., None], 0.0, whole)
        return (whole + 128).astype(np.uint8), np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def values(held, scales, dtype=np.float64) -> np.ndarray:
    if scales is None:
        return held.astype(dtype)
    return (held.astype(dtype) - dtype(128)) * scales[..., None].astype(dtype)


class Pool:
    """Keys and values of several sequences in pages handed out in no order. Whatever is not written is NaN."""

    def __init__(self, cuda, fmt, page_size, kv, hd, lens, rng, spare_pages=3, spare_columns=2):
        self.cuda, self.fmt, self.page_size, self.kv, self.hd = cuda, fmt, page_size, kv, hd
        self.lens = list(lens)
        per_seq = [-(-n // page_size) for n in self.lens]
        self.n_pages, self.max_pages = sum(per_seq) + spare_pages, max(per_seq + [0]) + spare_columns
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(self.lens), self.max_pages), 0xFFFFFFFF, dtype=np.uint32)
        at = 0
        for s, n in enumerate(per_seq):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.row_bytes = 2 * hd if fmt == F16 else hd
        self.page_bytes = kv * page_size * (self.row_bytes + (4 if fmt == I8 else 0))
        self.bytes = cuda.kv_pool_bytes(fmt, self.n_pages, page_size, kv, hd)
        assert self.bytes == self.n_pages * self.page_bytes
        if fmt == F16:
            self.k_raw = np.full(self.bytes // 2, NAN_HALF, dtype=np.uint16).view(np.uint8).reshape(self.n_pages, -1)
        else:
            self.k_raw = np.full((self.n_pages, self.page_bytes), NAN_BYTE, dtype=np.uint8)
        self.v_raw = self.k_raw.copy()

    def put(self, which: np.ndarray, seq: int, pos: int, x: np.ndarray) -> None:
        """Stores x [kv][hd] of one position."""
        held, scales = stored(x, self.fmt)
        page, slot = int(self.table[seq, pos // self.page_size]), pos % self.page_size
        n = self.kv * self.page_size * self.row_bytes
        which[page, :n].reshape(self.kv, self.page_size, self.row_bytes)[:, slot] = held.view(np.uint8).reshape(self.kv, -1)
        if scales is not None:
            which[page, n:].reshape(self.kv, self.page_size, 4)[:, slot] = scales.reshape(self.kv, 1).view(np.uint8).reshape(self.kv, 4)

    def get(self, which: np.ndarray, seq: int, pos: int, dtype=np.float64) -> np.ndarray:
        page, slot = int(self.table[seq, pos // self.page_size]), pos % self.page_size
        n = self.kv * self.page_size * self.row_bytes
        held = np.ascontiguousarray(which[page, :n].reshape(self.kv, self.page_size, self.row_bytes)[:, slot])
        if self.fmt == F16:
            return held.view(np.float16).astype(dtype)
        scales = np.ascontiguousarray(which[page, n:].reshape(self.kv, self.page_size, 4)[:, slot]).view(np.float32).reshape(self.kv)
        return values(held, scales, dtype)

    def fill(self, rng, amplitude=1.0):
        for s, n in enumerate(self.lens):
            for pos in range(n):
                self.put(self.k_raw, s, pos, (rng.standard_normal((self.kv, self.hd)) * amplitude).astype(np.float32))
                self.put(self.v_raw, s, pos, (rng.standard_normal((self.kv, self.hd)) * amplitude).astype(np.float32))

    def fill_at_once(self, rng, amplitude=1.0):
        """The same for long contexts: every position of a sequence in one go."""
        for s, n in enumerate(self.lens):
            pos = np.arange(n)
            page, slot = self.table[s, pos // self.page_size], pos % self.page_size
            for which in (self.k_raw, self.v_raw):
                held, scales = stored((rng.standard_normal((n, self.kv, self.hd)) * amplitude).astype(np.float32), self.fmt)
                m = self.kv * self.page_size * self.row_bytes
                view = np.lib.stride_tricks.as_strided(which, (self.n_pages, self.kv, self.page_size, self.row_bytes),
                                                       (self.page_bytes, self.page_size * self.row_bytes, self.row_bytes, 1))
                view[page, :, slot] = held.view(np.uint8).reshape(n, self.kv, self.row_bytes)
                if scales is not None:
                    view = np.lib.stride_tricks.as_strided(which[:, m:], (self.n_pages, self.kv, self.page_size, 4), (self.page_bytes, self.page_size * 4, 4, 1))
                    view[page, :, slot] = scales.astype(np.float32).reshape(n, self.kv, 1).view(np.uint8).reshape(n, self.kv, 4)

    def context(self, which, seq, length) -> np.ndarray:
        """[length][kv][hd] in 64 bits."""
        if length == 0:
            return np.zeros((0, self.kv, self.hd))
        pos = np.arange(length)
        page, slot = self.table[seq, pos // self.page_size], pos % self.page_size
        m = self.kv * self.page_size * self.row_bytes
        held = np.ascontiguousarray(which[:, :m].reshape(self.n_pages, self.kv, self.page_size, self.row_bytes)[page, :, slot])
        if self.fmt == F16:
            return held.view(np.float16).astype(np.float64)
        scales = np.ascontiguousarray(which[:, m:].reshape(self.n_pages, self.kv, self.page_size, 4)[page, :, slot]).view(np.float32).reshape(length, self.kv)
        return values(held, scales)

    def upload(self):
        self.k, self.v = self.cuda.buffer_from(self.k_raw), self.cuda.buffer_from(self.v_raw)
        self.pool = KvPool(self.fmt, self.n_pages, self.page_size, self.kv, self.hd, self.k, self.v)
        return self.pool

    def rows(self, news, n_rows=None, lens=None, max_queries=None) -> KvRows:
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.uint32)
        c = self.cuda
        return KvRows(len(news), int(starts[-1]) if n_rows is None else n_rows, max(list(news) + [1]) if max_queries is None else max_queries, self.max_pages,
                      c.buffer_from(self.table), c.buffer_from(starts), c.buffer_from(np.asarray(self.lens if lens is None else lens, dtype=np.uint32)))

    def download(self):
        return (self.cuda.read(self.k, np.zeros_like(self.k_raw)), self.cuda.read(self.v, np.zeros_like(self.v_raw)))


def attention(q, k, v, first):
    """Rows q [n][heads][hd] at positions first .. over k, v [length][kv][hd], in 64 bits, and how far an answer may lie from it.

    The bound. A score is a sum of hd products of exact halves (or whole numbers) with a query element of two halves: 22 bits, and 2^-25 of
    the row's largest element where the lower half is below the normal halves; its f32 sums, hd / 8 multiplies of 16, lose at most the last
    place each, the factors behind it four more. A probability is off by its score's error and that of the maximum, and by
    the exponential's two last places; its products with values are sums over at most n / 64 + 64 steps, each off by
    the last place, relative to the sum of magnitudes."""
    n, heads, hd = q.shape
    kv, group = k.shape[1], heads // k.shape[1]
    q = q.astype(np.float64)
    out, bound = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    see = np.clip(first + np.arange(n) + 1, 0, len(k))
    rows = np.flatnonzero(see > 0)
    if rows.size == 0:
        return out, bound
    unseen = np.arange(len(k)) >= see[rows, None]
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        x = q[rows, h]
        magnitude = np.where(unseen, 0.0, np.abs(x) @ np.abs(kk).T) / np.sqrt(hd)
        floor = np.abs(x).max(axis=1, keepdims=True) * np.where(unseen, 0.0, np.abs(kk).sum(axis=1)) / np.sqrt(hd)
        ds = (magnitude * (2.0 ** -22 + (hd / 8 + 8) * 2.0 ** -23) + 2.0 ** -25 * floor).max(axis=1, keepdims=True)
        s = np.where(unseen, -np.inf, x @ kk.T / np.sqrt(hd))
        p = np.exp(s - s.max(axis=1, keepdims=True))
        total = p.sum(axis=1, keepdims=True)
        out[rows, h] = p @ vv / total
        bound[rows, h] = (2 * ds + 2.0 ** -20 + (see[rows, None] / 64 + 64) * 2.0 ** -23) * (p @ np.abs(vv)) / total
    return out, bound
