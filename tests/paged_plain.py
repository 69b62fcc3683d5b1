"""Plain forms of the paged cache for its tests: the codec as it is defined (IEEE fp32, one operation at a time), attention in 64 bits, and
a host model of rows, pages and counts.  Nothing here uses the package."""
import math

import numpy as np

PAGE = 64


def books():
    """levels [128, 16] and the code of the level nearest r [128, 128], ties to the lower code."""
    book = np.zeros((128, 16), dtype=np.int64)
    for z in range(128):
        zc = round(15 * z / 127)
        for e in range(16):
            if e >= zc:
                book[z, e] = z + round((127 - z) * math.expm1(math.log(3.0) * (e - zc) / max(15 - zc, 1)) / 2)
            else:
                book[z, e] = z - round(z * math.expm1(math.log(3.0) * (zc - e) / zc) / 2)
    nearest = np.abs(book[:, None, :] - np.arange(128)[None, :, None]).argmin(-1)
    return book, nearest


BOOK, NEAREST = books()


def quantize(x):
    """rows [..., 64] of fp32 -> codes [..., 64], words [...] (uint32)."""
    f = np.float32
    with np.errstate(all="ignore"):
        x = np.clip(np.where(np.isnan(x), f(0), x.astype(f)), f(-65504), f(65504))
        lo, hi = x.min(-1), x.max(-1)
        a16 = np.where(lo > 0, lo, np.where(hi < 0, hi, f(0))).astype(np.float16)
        bits = a16.view(np.uint16).astype(np.uint32)
        off = (bits & 0x7FFF) >= 128
        a = np.where(off, a16.astype(f), f(0))
        dn = np.where(a > 0, f(0), np.maximum(a - lo, f(0)))
        up = np.where(a < 0, f(0), np.maximum(hi - a, f(0)))
        extent = dn + up
        z = np.where(extent > 0, np.rint((f(127) * dn) / np.where(extent > 0, extent, f(1))), f(0))
        z = np.where(a < 0, f(127), z)
        t = (extent * f(32.0 / 127.0)).astype(np.float16)
        inv = np.where(t > 0, f(32) / np.where(t > 0, t, np.float16(1)).astype(f), f(0))
        y = ((x - a[..., None]) * inv[..., None]).astype(f) + z[..., None]
        r = np.clip(np.rint(y), 0, 127).astype(np.int64)
    codes = NEAREST[z.astype(np.int64)[..., None], r]
    return codes, t.view(np.uint16).astype(np.uint32) | (np.where(off, bits, z.astype(np.uint32)) << 16)


def dequantize(codes, words):
    """inverse, in 64 bits"""
    t = (words & 0xFFFF).astype(np.uint16).view(np.float16).astype(np.float64)
    field = words >> 16
    off = (field & 0x7FFF) >= 128
    a = np.where(off, field.astype(np.uint16).view(np.float16).astype(np.float64), 0.0)
    z = np.where(off, np.where(a < 0, 127, 0), field).astype(np.int64)
    return a[..., None] + t[..., None] * (BOOK[z[..., None], codes] - z[..., None]) / 32.0


def pack_page(k, v):
    """one kv head's 64 tokens of keys and values [64, D] -> the page's bytes"""
    d = k.shape[1]
    parts = []
    for codes, words in (quantize(k.T), quantize(v.reshape(PAGE * (d // 64), 64))):
        parts.append((codes[:, 0::2] | codes[:, 1::2] << 4).astype(np.uint8).reshape(-1))
        parts.append(words.astype("<u4").view(np.uint8).reshape(-1))
    return np.concatenate(parts)


def unpack_page(raw, d):
    out = []
    for codes, words, rows in ((raw[:32 * d], raw[32 * d:36 * d], d), (raw[36 * d:68 * d], raw[68 * d:], PAGE * (d // 64))):
        c = codes.reshape(rows, 32)
        e = np.empty((rows, 64), dtype=np.int64)
        e[:, 0::2], e[:, 1::2] = c & 15, c >> 4
        out.append(dequantize(e, words.copy().view("<u4").astype(np.uint32)))
    return out[0].T, out[1].reshape(PAGE, d)


def packed(length, residual):
    return max(0, (length - residual) // PAGE) * PAGE


def held(k, v, residual):
    """what a cache holds of a row's tokens [n, kvh, D]: pages through the codec, the newest as they are; in 64 bits"""
    n, h, d = k.shape
    kk, vv = k.astype(np.float64).copy(), v.astype(np.float64).copy()
    for p in range(packed(n, residual) // PAGE):
        s = slice(p * PAGE, (p + 1) * PAGE)
        for j in range(h):
            kk[s, j], vv[s, j] = unpack_page(pack_page(k[s, j], v[s, j]), d)
    return kk, vv


def attention(q, k, v, scaling):
    """q [l, H, D]: the newest l of k's, v's n tokens [n, kvh, D] -> [l, H, D] in 64 bits"""
    lq, hq, d = q.shape
    n, kvh = k.shape[:2]
    out = np.zeros((lq, hq, d))
    with np.errstate(all="ignore"):
        for j in range(lq):
            m = n - lq + j + 1
            if m <= 0:
                continue
            for h in range(hq):
                s = k[:m, h // (hq // kvh)] @ q[j, h].astype(np.float64) * scaling
                w = np.exp(s - s.max())
                out[j, h] = (w / w.sum()) @ v[:m, h // (hq // kvh)]
    return out


class Model:
    """rows, pages and counts on the host"""

    def __init__(self, rows, pages, width, residual):
        self.table = [[-1] * width for _ in range(rows)]
        self.length, self.refs, self.residual, self.width = [0] * rows, [0] * pages, residual, width

    def extend(self, rows, counts):
        need = [packed(self.length[r] + n, self.residual) // PAGE - packed(self.length[r], self.residual) // PAGE for r, n in zip(rows, counts)]
        if any(packed(self.length[r] + n, self.residual) // PAGE > self.width for r, n in zip(rows, counts)):
            return 2
        free = [p for p, c in enumerate(self.refs) if c == 0]
        if sum(need) > len(free):
            return 1
        for r, n, m in zip(rows, counts, need):
            at = packed(self.length[r], self.residual) // PAGE
            for i in range(m):
                self.table[r][at + i] = free[0]
                self.refs[free.pop(0)] = 1
            self.length[r] += n
        return 0

    def free(self, rows):
        for r in rows:
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r] = [-1] * self.width
            self.length[r] = 0

    def fork(self, source, target):
        for s, t in zip(source, target):
            self.free([t])
            self.table[t] = list(self.table[s])
            self.length[t] = self.length[s]
            for p in self.table[t]:
                if p >= 0:
                    self.refs[p] += 1

    def compact(self):
        n = sum(c > 0 for c in self.refs)
        src = [p for p, c in enumerate(self.refs) if c > 0 and p >= n]
        dst = [p for p, c in enumerate(self.refs) if c == 0 and p < n]
        moved = dict(zip(src, dst))
        for a, b in moved.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[moved.get(p, p) for p in row] for row in self.table]
        return src, dst
