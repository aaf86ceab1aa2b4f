"""Plain 64-bit forms of the operators on device memory, over numpy arrays,
and the batches their tests run."""
import numpy as np


class Batch:
    """Host tables of a batch: groups of (prefix length, [(past, new), ...])."""

    def __init__(self, groups, page, rng, spare=2, grouped=True):
        self.page = page
        self.q_start, self.lens, self.group_start, self.prefix_lens = [0], [], [0], []
        own, pre = [], []
        for plen, seqs in groups:
            self.prefix_lens.append(plen)
            pre.append(-(-plen // page))
            for past, new in seqs:
                self.lens.append(past + new)
                self.q_start.append(self.q_start[-1] + new)
                own.append(-(-(past + new) // page))
            self.group_start.append(len(self.lens))
        self.n_pages = sum(own) + sum(pre) + spare
        order = rng.permutation(self.n_pages)
        self.spare = order[-spare:] if spare else order[:0]
        self.pages = np.full((len(own), max(own + [1]) + 1), -7, np.int32)
        self.prefix_pages = np.full((len(pre), max(pre + [1]) + 1), self.n_pages + 3, np.int32)
        at = 0
        for table, counts in ((self.pages, own), (self.prefix_pages, pre)):
            for i, n in enumerate(counts):
                table[i, :n] = order[at:at + n]
                at += n
        self.grouped = grouped
        self.tokens = self.q_start[-1]

    def device(self, ops, torch, dev, **override):
        t = {"q_start": self.q_start, "lens": self.lens, "pages": self.pages}
        if self.grouped:
            t.update(group_start=self.group_start, prefix_lens=self.prefix_lens,
                     prefix_pages=self.prefix_pages)
        t.update(override)
        return ops.PagedBatch(**{k: torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)
                                 for k, v in t.items()})

    def sequences(self):
        """(sequence, prefix length, group, its query rows, own index of the first)."""
        for g, plen in enumerate(self.prefix_lens):
            for s in range(self.group_start[g], self.group_start[g + 1]):
                rows = range(self.q_start[s], self.q_start[s + 1])
                yield s, plen if self.grouped else 0, g, rows, self.lens[s] - len(rows)

    def rows(self, table, n):
        i = np.arange(n)
        return table[i // self.page].astype(np.int64) * self.page + i % self.page

    def used_rows(self):
        """Every cache row that holds a token."""
        r = [self.rows(self.prefix_pages[g], n) for g, n in enumerate(self.prefix_lens)]
        r += [self.rows(self.pages[s], n) for s, n in enumerate(self.lens)]
        return np.concatenate(r + [np.zeros(0, np.int64)])


def attention(q, cache, b, scale, window):
    """out [tokens, heads, hd] f64 and sum_k p |v| (for error bounds); rows of
    padding are NaN in both. Only visible keys enter, so what masked rows hold
    does not matter."""
    heads, hd = q.shape[1:]
    kvh = cache.shape[3]
    flat = cache.reshape(-1, 2, kvh, hd).astype(np.float64)
    out = np.full(q.shape, np.nan)
    mag = np.full(q.shape, np.nan)
    for s, plen, g, rows, i0 in b.sequences():
        pre = b.rows(b.prefix_pages[g], plen) if plen else np.zeros(0, np.int64)
        kv = flat[np.concatenate([pre, b.rows(b.pages[s], max(b.lens[s], 0))])]
        for j, t in enumerate(rows):
            pos = plen + i0 + j
            lo = max(0, pos - window + 1) if window else 0
            vis = kv[lo:max(pos + 1, 0)]
            for h in range(heads):
                k = h // (heads // kvh)
                if not len(vis):
                    out[t, h] = mag[t, h] = 0
                    continue
                z = vis[:, 0, k] @ q[t, h].astype(np.float64) * scale
                p = np.exp(z - z.max())
                p /= p.sum()
                out[t, h] = p @ vis[:, 1, k]
                mag[t, h] = p @ np.abs(vis[:, 1, k])
    return out, mag


def append(qkv, cache, b, heads, qn, kn, offset, eps, v_norm, freq, q_scale):
    """(q, cache) in f64; the cache's other rows as they were."""
    kvh, hd = cache.shape[3:]
    n = b.tokens
    x = qkv[:n].astype(np.float64).reshape(n, -1, hd)
    has_kv = x.shape[1] > heads
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]

    def rms(y):
        return y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)

    if qn is not None:
        q = rms(q) * (offset + qn.astype(np.float64))
    if kn is not None:
        k = rms(k) * (offset + kn.astype(np.float64))
    if v_norm:
        v = rms(v)
    flat = cache.astype(np.float64).reshape(-1, 2, kvh, hd)
    out = np.empty((n, heads, hd))
    for s, plen, g, rows, i0 in b.sequences():
        for j, t in enumerate(rows):
            a = np.float64(plen + i0 + j) * freq
            c, sn = np.cos(a), np.sin(a)

            def rot(y):
                y = y.copy()
                m = len(freq)
                lo, hi = y[:, :m].copy(), y[:, hd // 2:hd // 2 + m].copy()
                y[:, :m], y[:, hd // 2:hd // 2 + m] = lo * c - hi * sn, hi * c + lo * sn
                return y

            out[t] = rot(q[t]) * q_scale
            if has_kv:
                i = i0 + j
                row = int(b.pages[s][i // b.page]) * b.page + i % b.page
                flat[row, 0], flat[row, 1] = rot(k[t]), v[t]
    return out, flat.reshape(cache.shape)


def sample(x, u, temperature, top_k, top_p, min_p):
    """(token, probability) of one row in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    best = x[order[0]]
    if best == -np.inf:
        return -1, 0.0
    if not temperature > 0 or top_p <= 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == best, 1.0, np.exp((x - best) / np.float64(temperature)))
    w = np.nan_to_num(w)
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        cum = np.cumsum(w[order])
        order = order[:np.searchsorted(cum, np.float64(top_p) * cum[-1], side="left") + 1]
    order = order[w[order] >= min(float(min_p), 1.0)]
    kept = np.sort(order)
    cum = np.cumsum(w[kept])
    at = min(int(np.searchsorted(cum, np.float64(u) * cum[-1], side="right")), len(kept) - 1)
    return int(kept[at]), w[kept[at]] / cum[-1]
