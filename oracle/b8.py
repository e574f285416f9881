"""The 8-bit block-scaled K/V cache restated in numpy (float64): scales, codes, append, read, attention, the accounts of
attention weight and eviction, from their definitions (include/dspark.h)."""
import numpy as np

PAGE = 32
E4M3 = np.full(256, np.nan)  # the value of each byte: sign, 4 exponent bits (bias 7), 3 mantissa bits; all ones is NaN
for _b in range(256):
    _e, _m = (_b >> 3) & 15, _b & 7
    if _b & 127 != 127:
        E4M3[_b] = (-1.0 if _b & 128 else 1.0) * ((8 + _m) * 2.0 ** (_e - 10) if _e else _m * 2.0 ** -9)
_E4M3_POS = E4M3[:127]  # ascending: the codes' order is the values'


def scale_of(code, amax):
    """The scale of blocks whose largest finite magnitudes are amax."""
    amax = np.asarray(amax, np.float64)
    if code == "int8":
        q = (amax / 127).astype(np.float32)
        return ((q.view(np.uint32) + np.uint32(255)) & np.uint32(0xFFFFFF00)).view(np.float32)
    out = np.zeros(amax.shape, np.float32)
    for i, a in np.ndenumerate(amax):
        if a > 0:
            e = -60
            while 448 * 2.0 ** e < a:
                e += 1
            out[i] = 2.0 ** e
    return out


def codes_of(code, x, scale):
    """Bytes of x / scale rounded once to nearest, ties to even; NaN -> 0, past the codes -> the largest one."""
    x, scale = np.asarray(x, np.float64), np.broadcast_to(np.asarray(scale, np.float64), np.shape(x))
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(scale > 0, x / scale, 0.0)
    y = np.where(np.isnan(y), 0.0, y)
    if code == "int8":
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    m = np.minimum(np.abs(y), 448.0)
    hi = np.clip(np.searchsorted(_E4M3_POS, m), 1, 126)  # m lies in (value[hi - 1], value[hi]], or is 0
    up = m - _E4M3_POS[hi - 1], _E4M3_POS[hi] - m
    low = (up[0] < up[1]) | ((up[0] == up[1]) & ((hi - 1) % 2 == 0))
    return (np.where(low, hi - 1, hi) | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def values(code, raw):
    return raw.view(np.int8).astype(np.float64) if code == "int8" else E4M3[raw]


class Cache:
    """Codes (bytes) k, v [pages][KVH][32][D], scales fp32 [pages][KVH], table (logical -> physical; None = identity)."""

    def __init__(self, code, pages, KVH, D, table=None):
        self.code, self.KVH, self.D, self.pages, self.table = code, KVH, D, pages, table
        self.raw = {x: np.zeros((pages, KVH, PAGE, D), np.uint8) for x in "kv"}
        self.scale = {x: np.zeros((pages, KVH), np.float32) for x in "kv"}

    def page(self, lp):
        pg = lp if self.table is None else int(self.table[lp])
        return pg if 0 <= pg < self.pages else -1

    def write(self, k, v, pos0):
        """Rows fp16 [n][KVH][D]."""
        n = len(k)
        for lp in range(pos0 // PAGE, (pos0 + n - 1) // PAGE + 1 if n else 0):
            pg = self.page(lp)
            if pg < 0:
                continue
            s0, s1 = max(pos0 - lp * PAGE, 0), min(pos0 + n - lp * PAGE, PAGE)
            for x, rows in (("k", k), ("v", v)):
                new = rows[lp * PAGE + s0 - pos0:lp * PAGE + s1 - pos0].astype(np.float64).transpose(1, 0, 2)
                need = scale_of(self.code, np.where(np.isfinite(new), np.abs(new), 0).max((1, 2)))
                was = self.scale[x][pg].copy()
                s = np.maximum(was, need) if s0 else need
                raw = self.raw[x][pg]
                if s0:
                    held = values(self.code, raw[:, :s0]) * was[:, None, None]
                    raw[:, :s0] = np.where((s == was)[:, None, None], raw[:, :s0], codes_of(self.code, held, s[:, None, None]))
                raw[:, s0:s1] = codes_of(self.code, new, s[:, None, None])
                raw[:, s1:] = 0
                self.scale[x][pg] = s

    def read(self, pos0, n):
        """Values of positions as float64 [n][KVH][D], and which positions are present."""
        out = {x: np.zeros((n, self.KVH, self.D)) for x in "kv"}
        here = np.zeros(n, bool)
        for i in range(n):
            pg = self.page((pos0 + i) // PAGE)
            if pg >= 0:
                here[i] = True
                for x in "kv":
                    out[x][i] = values(self.code, self.raw[x][pg][:, (pos0 + i) % PAGE]) * self.scale[x][pg].astype(np.float64)[:, None]
        return out["k"], out["v"], here


def visible(M, a, start, window, causal, here):
    """Which of positions 0 .. a + M - 1 each token sees."""
    p, t = np.arange(a + M), np.arange(M)[:, None]
    see = (p < a) & (p >= start) & ((window == 0) | (p > a + t - window))
    return (see | ((p >= a) & (not causal or p - a <= t))) & here


def attention(q, k, v, see, gate=None):
    """o, lse and the attention with |v| (the size that rounding errors of the probabilities scale with)."""
    M, QH, D = q.shape
    G = QH // k.shape[1]
    o, lse, mag = np.zeros((M, QH, D)), np.full((M, QH), -np.inf), np.zeros((M, QH, D))
    for t in range(M):
        w = np.flatnonzero(see[t])
        if not len(w):
            continue
        for h in range(k.shape[1]):
            x = q[t, h * G:(h + 1) * G].astype(np.float64) @ k[w, h].T / np.sqrt(D)
            m = x.max(1, keepdims=True)
            e = np.exp(x - m)
            l = e.sum(1, keepdims=True)
            r = slice(h * G, (h + 1) * G)
            o[t, r], mag[t, r] = e @ v[w, h] / l, e @ np.abs(v[w, h]) / l
            lse[t, r] = (np.log(l) + m)[:, 0]
    if gate is not None:
        s = 1 / (1 + np.exp(-gate.astype(np.float64)))[..., None]
        o, mag = o * s, mag * s
    return o, lse, mag


def mass(q, k, see, lse, rows, a, mass_in):
    """The accounts of positions 0 .. a + rows - 1."""
    M, QH, D = q.shape
    KVH = k.shape[1]
    G = QH // KVH
    out = np.zeros((KVH, a + M)) if mass_in is None else mass_in[:, :a + M].astype(np.float64).copy()
    out[:, a:] = 0
    for t in range(rows):
        w = np.flatnonzero(see[t])
        for h in range(KVH):
            for g in range(h * G, (h + 1) * G):
                if len(w) and lse[t, g] > -np.inf:
                    out[h, w] += np.exp(k[w, h] @ q[t, g].astype(np.float64) / np.sqrt(D) - float(lse[t, g]))
    return out[:, :a + rows]


def kept(mass_row, length, keep, sinks, recent):
    mid = np.arange(sinks, length - recent)
    m = mass_row[mid].astype(np.float64) + 0.0
    order = np.lexsort((mid, -np.where(np.isnan(m), -np.inf, m), np.isnan(m)))  # numbers first, largest first, lowest position
    top = mid[order[:keep - sinks - recent]]
    return np.sort(np.concatenate([np.arange(sinks), top, np.arange(length - recent, length)])).astype(np.int32)


def evict(src, dst, length, keep, mass_in, sinks, recent):
    """kept [KVH][keep] and their accounts; dst receives the rows."""
    ks = np.stack([kept(mass_in[h], length, keep, sinks, recent) for h in range(src.KVH)])
    for h in range(src.KVH):
        pg = np.array([src.page(p // PAGE) for p in ks[h]])
        for lp in range((keep + PAGE - 1) // PAGE):
            to = dst.page(lp)
            if to < 0:
                continue
            rows = np.arange(lp * PAGE, min(keep, (lp + 1) * PAGE))
            for x in "kv":
                s = np.where(pg[rows] >= 0, src.scale[x][pg[rows], h], 0).astype(np.float32)
                raw = np.where((pg[rows] >= 0)[:, None], src.raw[x][pg[rows], h, ks[h][rows] % PAGE], 0).astype(np.uint8)
                new = codes_of(src.code, values(src.code, raw) * s.astype(np.float64)[:, None], np.float64(s.max()))
                dst.raw[x][to, h, :len(rows)] = np.where((s == s.max())[:, None], raw, new)
                dst.raw[x][to, h, len(rows):] = 0
                dst.scale[x][to, h] = s.max()
    return ks, np.take_along_axis(mass_in[:, :length], ks, 1)
