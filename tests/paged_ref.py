"""Plain NumPy statements of the paged 4-bit cache's operators: integers and stored values exactly, attention in 64 bits."""
import numpy as np

F = np.float32


def bf16_nearest(x):
    u = np.asarray(x, F).view(np.uint32).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)).view(F)


def bf16_up(x):
    u = np.asarray(x, F).view(np.uint32).astype(np.uint64)
    return (((u + 0xFFFF) & 0xFFFF0000).astype(np.uint32)).view(F)


def quantise(x):
    """x [..., head_dim] f32 -> (codes, z, d), every operation in f32; a row that is not finite has z = d = NaN, codes 0."""
    x = np.asarray(x, F)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(x).all(-1)
        x0 = np.where(bad[..., None], F(0), x)
        lo, hi = x0.min(-1), x0.max(-1)
        z = bf16_nearest(F(0.5) * lo + F(0.5) * hi)
        h = np.maximum(hi - z, z - lo)
        bad |= ~np.isfinite(h)
        d = np.where(h == 0, F(0), np.maximum(bf16_up(np.where(bad, F(0), h) * (F(1) / F(7.5))), F(2.0 ** -120)))
        r = np.where(h == 0, F(0), F(1) / d)
        n = np.clip(np.rint((x0 - z[..., None]) * r[..., None] + F(7.5)), 0, 15)
    nan = F(np.nan)
    return (np.where(bad[..., None], 0, n).astype(np.uint8), np.where(bad, nan, z).astype(F), np.where(bad, nan, d).astype(F))


def values(n, z, d):
    """f32, as the cache's read-back computes them."""
    return (d[..., None] * (n.astype(F) - F(7.5)) + z[..., None]).astype(F)


class Cache:
    """Rows by slot: values of keys and values, [slots, heads, head_dim]; rows never written are 0."""

    def __init__(self, num_blocks, block_size, heads, hd):
        self.bs, self.nb = block_size, num_blocks
        shape = (num_blocks * block_size, heads)
        self.n = [np.zeros(shape + (hd,), np.uint8) for _ in range(2)]
        self.z = [np.zeros(shape, F) for _ in range(2)]
        self.d = [np.zeros(shape, F) for _ in range(2)]

    def append(self, k, v, slots):
        live = (slots >= 0) & (slots < self.nb * self.bs)
        for side, x in enumerate((k, v)):
            n, z, d = quantise(x[live])
            self.n[side][slots[live]], self.z[side][slots[live]], self.d[side][slots[live]] = n, z, d

    def f32(self, side, slots):
        return values(self.n[side][slots], self.z[side][slots], self.d[side][slots])

    def f64(self, side, slots):
        """The exact values that codes, centre and step stand for."""
        return self.z[side][slots][..., None].astype(np.float64) + self.d[side][slots][..., None].astype(np.float64) * (self.n[side][slots] - 7.5)


def slots_of(table, positions, bs):
    return table[positions // bs].astype(np.int64) * bs + positions % bs


def summary(keys):
    """keys [tokens, heads, hd] f32 -> (lo, hi) int, scale [heads] f32; scale inf for a block with a NaN row."""
    lo, hi = keys.min(0), keys.max(0)
    bad = np.isnan(keys).any((0, 2))
    most = np.where(bad, F(0), np.maximum(np.abs(np.nan_to_num(lo)), np.abs(np.nan_to_num(hi))).max(-1)).astype(F)
    with np.errstate(all="ignore"):
        r = np.where(most < F(2.0 ** -100), F(0), F(1) / most * F(127)).astype(F)
    lo8, hi8 = (np.rint(np.where(bad[:, None], F(0), x) * r[:, None]).astype(np.int64) for x in (np.nan_to_num(lo), np.nan_to_num(hi)))
    return lo8, hi8, np.where(bad, F(np.inf), most * (F(1) / F(127))).astype(F)


def select(q, cache, table, pos, top, first, recent):
    """q [heads, group, hd] of one row -> selected [heads, top]."""
    heads = q.shape[0]
    blocks = pos // cache.bs + 1 if pos >= 0 else 0
    out = np.full((heads, top), -1, np.int32)
    if blocks <= top:
        out[:, :blocks] = np.arange(blocks)
        return out
    for h in range(heads):
        with np.errstate(all="ignore"):
            a = np.abs(q[h]).max(-1, keepdims=True).astype(F)
            bad = ~np.isfinite(q[h]).all(-1, keepdims=True)
            r = np.where(bad | (a < F(2.0 ** -100)), F(0), F(1) / a * F(127)).astype(F)
            x = np.where(bad, 0, np.rint(np.nan_to_num(q[h]) * r)).astype(np.int64)
            unit = np.where(bad, F(0), a * (F(1) / F(127))).astype(F)[:, 0]
        score = np.zeros(blocks, F)
        for j in range(blocks):
            count = min(cache.bs, cache.lens_now - j * cache.bs)
            lo8, hi8, sb = (s[h] for s in summary(cache.f32(0, slots_of(table, np.arange(j * cache.bs, j * cache.bs + count), cache.bs))))
            whole = (np.maximum(x, 0) * hi8 + np.minimum(x, 0) * lo8).sum(-1)
            with np.errstate(all="ignore"):
                score[j] = np.inf if np.isinf(sb) else (whole.astype(F) * unit * sb).max()
        key = score.astype(np.float64)
        forced = (np.arange(blocks) < first) | (np.arange(blocks) >= blocks - recent)
        order = np.lexsort((np.arange(blocks), -key, ~forced))
        out[h] = np.sort(order[:top])
    return out


def attend(q, k, v, scale, seen, cap=0.0):
    """One row and head in 64 bits: q [hd], k, v [keys, hd], seen [keys] -> ([hd], the largest |error| that f32 roundings
    can make of it by the bound below).

    A score is d A + w S with A = sum q (n - 8), w = z + d / 2, S = sum q.  q is within half a unit u = max|q| / (127 * 2^16) of
    its fixed point; A's and S's conversions, the products and sums are 8 roundings of 2^-24 of |d A| + |w S|, the sum with
    the maximum one of |s| + |m|, a cap's tanh 4 of the cap; exp2 and the products into p d three more.  p d is two f16: 2^-21 of it
    (and 2^-35 of the row's largest, where f16 ends).  The output's sums over N keys are N + 64 roundings of their
    largest partial sum, and numerator and sum share a row's common error, which counts twice at most."""
    if not seen.any():
        return np.zeros(k.shape[-1]), np.zeros(k.shape[-1])
    k, v, q = k[seen], v[seen], q.astype(np.float64)
    s = k @ q * scale
    u = np.abs(q).max() / (127 * 65536)
    size = np.abs(scale) * (np.abs(k) @ np.abs(q) + 2 * np.abs(k).max(1) * np.abs(q).sum())
    if cap:
        s = cap * np.tanh(s / cap)
    m = s.max()
    err = np.abs(scale) * u * np.abs(k).sum(1) + 2.0 ** -24 * (8 * size + 2 * (np.abs(s) + abs(m)) / np.log(2) + 4 * cap) + 2.0 ** -22
    p = np.exp(s - m)
    p /= p.sum()
    out = p @ v
    most = np.abs(v).max(1) if len(v) else np.zeros(0)
    bound = 2 * (p * (err + 2.0 ** -21 + (len(p) + 64) * 2.0 ** -24) * most).sum() + 2.0 ** -35 * len(p) * p.max() * most.max()
    return out, np.full(v.shape[-1], bound)
