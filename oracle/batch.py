"""The operators for a batch of sequences restated in numpy (float64) from their definitions (include/dspark.h): rotary positions,
attention behind a shared prefix, sampling."""
import math

import numpy as np

PAGE = 32


# ---------------------------------------------------------------- rotary positions
def rope_freqs(rot, base, scaling=None, factor=1.0, trained=0.0, low=1.0, high=32.0):
    """(frequencies [rot / 2], scale)."""
    if scaling == "base" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    if scaling == "linear":
        f = f / factor
    if scaling != "ramp":
        return f, 1.0
    keep = np.clip((trained * f / (2 * math.pi) - low) / (high - low), 0, 1)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1


def rope(x, positions, freqs, interleaved=False, inverse=False, scale=1.0):
    """x [n][heads][D] -> float64."""
    x = np.asarray(x, np.float64)
    P, rot = len(freqs), 2 * len(freqs)
    i, j = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(P), np.arange(P, rot))
    a = np.asarray(positions, np.float64)[:, None, None] * freqs * (-1 if inverse else 1)
    y = x.copy()
    y[..., i] = scale * (x[..., i] * np.cos(a) - x[..., j] * np.sin(a))
    y[..., j] = scale * (x[..., j] * np.cos(a) + x[..., i] * np.sin(a))
    return y


# ---------------------------------------------------------------- attention behind a shared prefix
def shared_attention(q, pk, pv, prefix_there, q_start, own, max_tokens, window=0, causal=True, gate=None):
    """q [tokens][QH][D]; pk, pv [prefix][KVH][D]; prefix_there [prefix] (False: on an absent page); own: for each sequence
    (k, v [len][KVH][D], there [len]). Returns out, lse (float64; NaN for rows in no sequence) and the largest |v| a row sees."""
    q = np.asarray(q, np.float64)
    T, QH, D = q.shape
    KVH = pk.shape[1]
    G, prefix = QH // KVH, len(pk)
    out, lse, size = np.full((T, QH, D), np.nan), np.full((T, QH), np.nan), np.zeros((T, QH))
    for r, (k, v, there) in enumerate(own):
        t0, m, n = int(q_start[r]), int(q_start[r + 1] - q_start[r]), len(k)
        a = prefix + n - m
        keys, vals = (np.concatenate([x, y]).astype(np.float64) for x, y in ((pk, k), (pv, v)))
        p, ok = np.arange(prefix + n), np.concatenate([prefix_there, there]).astype(bool)
        for i in range(min(m, max_tokens)):
            see = ok & ((p < a) | ((p <= a + i) if causal else True))
            if window:
                see &= (p >= a) | (p > a + i - window)
            for h in range(KVH):
                g = slice(h * G, (h + 1) * G)
                if not see.any():
                    out[t0 + i, g], lse[t0 + i, g] = 0.0, -np.inf
                    continue
                s = q[t0 + i, g] @ keys[see, h].T / math.sqrt(D)
                top = s.max(1, keepdims=True)
                w = np.exp(s - top)
                out[t0 + i, g] = (w / w.sum(1, keepdims=True)) @ vals[see, h]
                lse[t0 + i, g] = top[:, 0] + np.log(w.sum(1))
                size[t0 + i, g] = np.abs(vals[see, h]).max()
    if gate is not None:
        out = out / (1 + np.exp(-np.asarray(gate, np.float64)))[..., None]
    return out, lse, size


# ---------------------------------------------------------------- sampling
def sample_row(z, u, t, k=0, p=1.0, low=0.0):
    """(token, kept, logprob) of one row."""
    z = np.asarray(z, np.float64)
    z = np.where(np.isnan(z), -np.inf, z) + 0.0
    live = np.flatnonzero(z > -np.inf)
    if not len(live):
        return -1, 0, -math.inf
    first = int(live[np.argmax(z[live])])
    if not t > 0:
        return first, 1, 0.0
    top = z[first]
    with np.errstate(invalid="ignore"):
        x = np.where(z == top, 0.0, (z - top) * (1.0 / float(t)))
    x = np.where(np.isnan(x), -np.inf, x)
    order = live[np.lexsort((live, -z[live]))]
    if 0 < k < len(z):
        order = order[:k]
    w = np.exp(x[order])
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        stay = before < max(float(p), 0.0) * w.sum()
        stay[0] = True
        order = order[stay]
    if low > 0:
        order = order[x[order] >= math.log(min(low, 1.0))]
    order = np.sort(order)
    w = np.exp(x[order])
    sums = np.cumsum(w)
    u = min(float(u), 1 - 2.0 ** -24) if u > 0 else 0.0  # (the largest fp32 number below 1)
    at = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(order) - 1)
    return int(order[at]), len(order), math.log(w[at] / sums[-1]) if w[at] > 0 else -math.inf
