"""Ragged batches over a paged pool and their results in 64 bits (numpy), for the tests."""
import numpy as np


class Batch:
    """Sequences of ctx[b] cached and new[b] new tokens, their pages a random draw from a pool that has
    `spare` pages more; pool rows that no sequence holds are NaN. pool: the pages come from a pool of this many
    instead, any of them as often as it is drawn."""

    def __init__(self, seed, ctx, new, hq, hkv, d, page=16, spare=3, behind=0, q_f16=False, std=1.0, pool=0):
        g = self.g = np.random.default_rng([seed, len(ctx), sum(ctx), sum(new)])
        self.ctx, self.new, self.hq, self.hkv, self.d, self.page = list(ctx), list(new), hq, hkv, d, page
        self.lens = [a + b for a, b in zip(ctx, new)]
        self.T, self.rows = sum(new), sum(new) + behind
        pages = [-(-n // page) for n in self.lens]
        self.n_pages, self.max_pages = sum(pages) + spare if not pool else pool, max(max(pages), 1) + 1
        perm, at = g.permutation(self.n_pages), 0
        self.table = np.full((len(ctx), self.max_pages), -7, np.int32)  # out of range: never used
        self.kp, self.vp = (np.full((hkv, self.n_pages * page, d), np.nan, np.float16) for _ in range(2))
        if pool:
            self.kp, self.vp = ((g.standard_normal((hkv, pool * page, d)) * std).astype(np.float16) for _ in range(2))
            for b, n in enumerate(pages):
                self.table[b, :n] = g.integers(0, pool, n)
        for b, n in enumerate(pages if not pool else ()):
            self.table[b, :n] = perm[at:at + n]
            at += n
            s = self.slots(b, self.lens[b])
            for pool in (self.kp, self.vp):
                pool[:, s] = g.standard_normal((hkv, self.lens[b], d)) * std
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.seq_lens = np.array(self.lens, np.int32)
        self.max_len = max(max(self.lens), 1)
        self.q = (g.standard_normal((self.rows, hq, d)) * std).astype(np.float16 if q_f16 else np.float32)
        self.scale = float(np.float32(1.0) / np.sqrt(np.float32(d)))

    def slots(self, b, n):
        p = np.arange(n)
        return self.table[b, p // self.page].astype(np.int64) * self.page + p % self.page

    def shape(self, hip, q_f16):
        return (hip.DTYPE_F16 if q_f16 else hip.DTYPE_F32, self.rows, len(self.ctx), self.hq, self.hkv, self.d, self.page, self.n_pages,
                self.max_pages, self.max_len)

    def attention(self):
        """[rows, hq, d] f64 (NaN behind the last sequence), and the error bound of every element: the scores
        are off by their operands' 22 bits and the sums' f32 roundings, the output by twice that (weights and
        their sum) and the same for its own sum, times the largest |v| of the row."""
        self.largest = 0.0  # score, as the sum of its terms' sizes
        out = np.full((self.rows, self.hq, self.d), np.nan)
        tol = np.zeros((self.rows, self.hq, 1))
        G = self.hq // self.hkv
        for b, (c, n) in enumerate(zip(self.ctx, self.new)):
            if n == 0:
                continue
            s, r0 = self.slots(b, c + n), self.starts[b]
            hidden = np.arange(c + n)[None] > c + np.arange(n)[:, None]
            for h in range(self.hq):
                k, v = self.kp[h // G, s].astype(np.float64), self.vp[h // G, s].astype(np.float64)
                q = self.q[r0:r0 + n, h].astype(np.float64)
                x = q @ k.T * self.scale
                x[hidden] = -np.inf
                w = np.exp(x - x.max(1, keepdims=True))
                out[r0:r0 + n, h] = w @ v / w.sum(1, keepdims=True)
                size = (np.abs(q) @ np.abs(k).T).max(1) * abs(self.scale)
                self.largest = max(self.largest, size.max())
                eps = 2.0 ** -24
                delta = size * (4 * eps + (self.d / 16 + 4) * eps)
                tol[r0:r0 + n, h, 0] = np.abs(v).max() * (2 * delta + 4 * eps + ((c + n) / 16 + 64) * eps)
        return out, tol


def turned(x, w, pos, theta, eps, freq_scale=1.0):
    """RMSNorm (w None: none) and NeoX rotation of [rows, heads, d] at positions pos, in 64 bits."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    a = np.asarray(pos, np.float64)[:, None] * float(np.float32(freq_scale)) * float(np.float32(theta)) ** (-2.0 * np.arange(d // 2) / d)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    u, v = x[..., :d // 2], x[..., d // 2:]
    return np.concatenate([u * c - v * s, u * s + v * c], -1)
