"""Plain 64-bit restatement of the paged 8-bit KV cache (vxc_kv8_*,
include/veltrix_cuda.h) on numpy arrays: test infrastructure only."""
import numpy as np

INT8, E4M3 = 1, 2
QMAX = {INT8: 127.0, E4M3: 448.0}


def e4m3_value(b):
    b = np.asarray(b, np.int64)
    e, m = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7.0), m / 8 * 2.0 ** -6)
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >> 7, -v, v)


_E4M3 = e4m3_value(np.arange(127))   # the non-negative codes, ascending


def value(code, kind):
    """Codes (uint8) as float64."""
    return code.view(np.int8).astype(np.float64) if kind == INT8 else e4m3_value(code)


def encode(y, kind):
    """Nearest code (uint8) of y, ties to even."""
    y = np.asarray(y, np.float64)
    if kind == INT8:
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    hi = np.minimum(np.searchsorted(_E4M3, a), 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _E4M3[lo], _E4M3[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (c | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def pow2_scale(amax, kind):
    """Smallest power of two s >= 2^-126 with amax <= qmax s; 0 for 0."""
    if amax == 0:
        return 0.0
    e = -126
    while amax > QMAX[kind] * 2.0 ** e:
        e += 1
    return 2.0 ** e


class Cache:
    """[n_blocks][kh][bs][hd] codes and [n_blocks][kh] scales of K and V."""

    def __init__(self, kind, nb, bs, kh, hd):
        self.kind, self.nb, self.bs, self.kh, self.hd = kind, nb, bs, kh, hd
        self.code = [np.zeros((nb, kh, bs, hd), np.uint8) for _ in range(2)]
        self.scale = [np.zeros((nb, kh), np.float32) for _ in range(2)]

    def append(self, k, v, slot):
        """k, v [n][kh][hd] fp32 (non-finite elements count as 0)."""
        slot = np.asarray(slot)
        ok = (slot >= 0) & (slot < self.nb * self.bs)
        for c, x in ((0, k), (1, v)):
            x = np.where(np.isfinite(x), x, 0).astype(np.float64)
            for b in np.unique(slot[ok] // self.bs):
                rows = np.nonzero(ok & (slot // self.bs == b))[0]
                off = slot[rows] % self.bs
                stay = np.setdiff1d(np.arange(self.bs), off)
                for h in range(self.kh):
                    old = 0.0 if 0 in off else float(self.scale[c][b, h])
                    s = max(old, pow2_scale(np.abs(x[rows, h]).max(), self.kind))
                    if s > old > 0:
                        q = value(self.code[c][b, h, stay], self.kind)
                        self.code[c][b, h, stay] = encode(q * (old / s), self.kind)
                    for r, o in zip(rows, off):   # in order: the later row stays
                        self.code[c][b, h, o] = encode(x[r, h] / s if s > 0 else x[r, h] * 0.0, self.kind)
                    self.scale[c][b, h] = s

    def rows(self, blocks, n):
        """K and V [kh][n][hd] of the first n tokens in `blocks`, float64."""
        out = []
        for c in range(2):
            x = value(self.code[c][blocks], self.kind) * self.scale[c][blocks].astype(np.float64)[:, :, None, None]
            out.append(x.transpose(1, 0, 2, 3).reshape(self.kh, -1, self.hd)[:, :n])
        return out


def tables(length, new, bs, nb, table, held, ring, state, n_rows):
    """vxc_kv8_tables in place on numpy arrays; returns (row0, slot)."""
    n, max_blocks = table.shape
    row0, slot = np.zeros(n + 1, np.int32), np.full(n_rows, -1, np.int32)
    want = [-(-(int(a) + int(b)) // bs) for a, b in zip(length, new)]
    status = 0
    if sum(max(0, w - int(h)) for w, h in zip(want, held)) > state[1]:
        status = 1
    if max(want) > max_blocks:
        status = 2
    if min(length) < 0 or min(new) < 0 or sum(map(int, new)) > n_rows or held.sum() + state[1] > nb or not 0 <= state[0] < nb:
        status = 3
    state[2] = status
    if status:
        return row0, slot
    front, count = int(state[0]), int(state[1])
    back = (front + count) % nb
    for r in range(n):
        for j in range(int(held[r]), want[r]):
            table[r, j] = ring[front]
            front, count = (front + 1) % nb, count - 1
    for r in range(n):
        for j in range(want[r], int(held[r])):
            ring[back] = table[r, j]
            table[r, j] = -1
            back, count = (back + 1) % nb, count + 1
        held[r] = want[r]
    state[0], state[1] = front, count
    i = 0
    for r in range(n):
        for t in range(int(new[r])):
            p = int(length[r]) + t
            slot[i] = table[r, p // bs] * bs + p % bs
            i += 1
        row0[r + 1] = i
    return row0, slot


def attention(cache, q, scale, table, row0, pos):
    """(out, bound) of the new rows, float64: bound is what an fp32 evaluation
    with exact codes and products split into two fp16 parts may be off by,
    element by element:
      score: the split 2^-22 of |q||k|, head_dim / 16 + 20 sequential sums of
        at most 2^-23 each (a tensor core's sums may truncate), scaled sums
        and the exponent's argument 4 roundings of 2^-23 |s|;
      weights: exp 2^-21; their sums over n tokens, at most n / 16 + 64 in
        sequence, 2^-23 each; the split of the weights 2^-22; the quotient.
    """
    rows, H, hd = q.shape
    G = H // cache.kh
    out, bound = np.zeros((rows, H, hd)), np.zeros((rows, H, hd))
    for r in range(len(pos)):
        total = int(pos[r]) + int(row0[r + 1] - row0[r])
        if total <= 0:
            continue
        nblk = -(-total // cache.bs)
        blocks = np.asarray(table[r, :nblk])
        k, v = cache.rows(np.clip(blocks, 0, cache.nb - 1), total)
        good = np.repeat((blocks >= 0) & (blocks < cache.nb), cache.bs)[:total]
        for i in range(int(row0[r]), int(row0[r + 1])):
            p = int(pos[r]) + i - int(row0[r])
            seen = good[:p + 1].nonzero()[0] if p >= 0 else np.zeros(0, int)
            if not seen.size:
                continue
            for h in range(H):
                kk, vv, qq = k[h // G][seen], v[h // G][seen], q[i, h].astype(np.float64)
                s = kk @ qq * scale
                size = np.abs(kk) @ np.abs(qq) * abs(scale)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, h] = w @ vv
                d = (2.0 ** -22 + (hd / 16 + 20) * 2.0 ** -23) * size.max() + 4 * 2.0 ** -23 * np.abs(s).max()
                rel = 2 * d + 2.0 ** -20 + 2 * (seen.size / 16 + 64) * 2.0 ** -23
                bound[i, h] = rel * (w @ np.abs(vv)) + 1e-30
    return out, bound
