"""The key/value cache and the attention over it in numpy, by their definitions: appending in the fp32 operations that the interface
states (codes and scales come out bit for bit), attention in fp64."""
import numpy as np

F = np.float32
SMALLEST = F(np.finfo(np.float32).tiny)


def rope_rows(positions, rotary_dim, base=10000.0):
    angle = np.arange(positions, dtype=np.float64)[:, None] * base ** (-np.arange(0, rotary_dim, 2) / rotary_dim)
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(F)


def rotate(x, row, interleaved):
    """x [heads, dim] fp32, row [rotary_dim]: cosines, then sines."""
    r = row.size
    c, s = row[:r // 2], row[r // 2:]
    out = x.copy()
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[:, first], x[:, second]
    out[:, first], out[:, second] = a * c - b * s, b * c + a * s
    return out


class Cache:
    def __init__(self, k, v, k_scale, v_scale):
        self.codes = [k.copy(), v.copy()]  # [pages, heads, page, dim]
        self.scales = [k_scale.copy(), v_scale.copy()]
        self.page = k.shape[2]

    def append(self, k, v, table, lengths, starts, rope=None, interleaved=False, q=None):
        """k, v [tokens, heads, dim] fp32. Returns the rotated q (rows of no sequence as they were)."""
        q = None if q is None else q.copy()
        pages = self.codes[0].shape[0]
        for b, length in enumerate(lengths):
            first, n = starts[b], starts[b + 1] - starts[b]
            if length <= 0 or length < n or length > table.shape[1] * self.page:
                continue
            turned = [k[first:first + n].copy(), v[first:first + n]]
            if rope is not None:
                for i in range(n):
                    row = rope[min(length - n + i, len(rope) - 1)]
                    turned[0][i] = rotate(k[first + i], row, interleaved)
                    if q is not None:
                        q[first + i] = rotate(q[first + i], row, interleaved)
            at = length - n
            while at < length:
                end = min(length, (at // self.page + 1) * self.page)
                page = table[b, at // self.page]
                if 0 <= page < pages:
                    for which in range(2):
                        self._fill(which, page, at % self.page, turned[which][at - (length - n):end - (length - n)])
                at = end
        return q

    def _fill(self, which, page, slot, x):
        for h in range(x.shape[1]):
            codes, rows = self.codes[which][page, h], x[:, h]
            before = self.scales[which][page, h] if slot else F(0)
            with np.errstate(all="ignore"):
                scale = np.abs(rows).max() * (F(1) / F(127)) if np.isfinite(rows).all() else F(np.nan)
                if scale < SMALLEST:
                    scale = F(0)
                if before > scale or np.isnan(before):
                    scale = before
                self.scales[which][page, h] = scale
                if scale > before:
                    codes[:slot] = np.rint(codes[:slot].astype(F) * F(before / scale))
                if scale > 0:
                    codes[slot:slot + len(rows)] = np.clip(np.rint(rows * F(F(1) / scale)), -127, 127)
                else:
                    codes[slot:slot + len(rows)] = 0

    def values(self, which, table_row, length):
        """fp64 [length, heads, dim], and which tokens lie on pages of the cache."""
        pages = -(-length // self.page)
        ids = np.asarray(table_row[:pages])
        good = (ids >= 0) & (ids < self.codes[0].shape[0])
        ids = np.where(good, ids, 0)
        x = self.codes[which][ids].astype(np.float64) * self.scales[which][ids].astype(np.float64)[:, :, None, None]
        return x.transpose(0, 2, 1, 3).reshape(pages * self.page, *x.shape[1:2], x.shape[3])[:length], np.repeat(good, self.page)[:length]


def attention(cache, q, table, lengths, starts, scale, out, bias=0):
    """q fp64 [tokens, q_heads, dim]. Returns (o, lse, magnitude = sum p |v|, largest sum of |q k| a row meets, keys seen times the
    largest value a code of theirs can stand for); rows of no sequence keep ``out``. ``bias``: what the sums carry with every code."""
    o, lse = out.copy(), np.full(q.shape[:2], np.nan)
    magnitude, products, reach = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    group = q.shape[1] // cache.codes[0].shape[1]
    for b, length in enumerate(lengths):
        first, n = starts[b], starts[b + 1] - starts[b]
        if length <= 0 or length < n or length > table.shape[1] * cache.page:
            o[first:first + n], lse[first:first + n] = 0, -np.inf
            continue
        (k, good), (v, _) = (cache.values(w, table[b], length) for w in range(2))
        for i in range(n):
            seen = np.arange(length) <= length - n + i
            seen &= good
            for h in range(q.shape[1]):
                row = q[first + i, h]
                if not seen.any():
                    o[first + i, h], lse[first + i, h] = 0, -np.inf
                    continue
                kk, vv = k[seen, h // group], v[seen, h // group]
                z = kk @ row * scale
                m = z.max()
                w = np.exp(z - m)
                o[first + i, h] = w @ vv / w.sum()
                lse[first + i, h] = m + np.log(w.sum())
                magnitude[first + i, h] = w @ np.abs(vv) / w.sum()
                on = table[b, np.flatnonzero(seen) // cache.page]
                products[first + i, h] = ((np.abs(kk) + bias * cache.scales[0][on, h // group][:, None]) @ np.abs(row)).max()
                reach[first + i, h] = seen.sum() * 127 * cache.scales[1][on, h // group].max()
    return o, lse, magnitude, products, reach
