"""Plain float64 numpy restatement of the transformer-layer operators, from their formulas (test infrastructure)."""
import numpy as np


def layer_norm(x, gamma, beta, eps=1e-5):
    x = np.asarray(x, np.float64)
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = 1.0 / np.sqrt((d * d).mean(-1) + eps)
    return d * rstd[..., None] * gamma + beta, mean, rstd


def layer_norm_pullback(x, gamma, gy, eps=1e-5):
    x, gamma, gy = (np.asarray(a, np.float64) for a in (x, gamma, gy))
    _, mean, rstd = layer_norm(x, gamma, 0.0, eps)
    xhat = (x - mean[..., None]) * rstd[..., None]
    g = gy * gamma
    gx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - xhat * (g * xhat).mean(-1, keepdims=True))
    rows = tuple(range(x.ndim - 1))
    return gx, (gy * xhat).sum(rows), gy.sum(rows)


def random16(groups, seed, step, channel):
    """[len(groups), 8]: the 16-bit numbers of each generator group (Philox4x32, 7 rounds; key = the seed, counter =
    group low, group high, channel, step low)."""
    m = 0xFFFFFFFF
    out = np.empty((len(groups), 8), np.int64)
    for n, g in enumerate(groups):
        c, k = [g & m, (g >> 32) & m, channel, step & m], [seed & m, (seed >> 32) & m]
        for _ in range(7):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
            k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
        out[n] = [v for w in c for v in (w & 0xFFFF, w >> 16)]
    return out


def threshold(p):
    return int(np.floor(p * 65536.0 + 0.5))


def keep_factors(shape, p, seed, step=0, channel=0):
    """keep / share kept for an array: element e takes number e % 8 of group e // 8."""
    n, t = int(np.prod(shape, dtype=np.int64)), threshold(p)
    u = random16(range((n + 7) // 8), seed, step, channel).reshape(-1)[:n]
    return ((u >= t) * (65536.0 / (65536 - t))).reshape(shape)


def attention_keep(B, H, Tq, Tk, p, seed, step=0, channel=0):
    """Keep factors [B,H,Tq,Tk]: row r = (b * H + h) * Tq + i has two groups for each block of 16 keys; key j takes
    number (j & 3) + 4 * (j >> 3 & 1) of group 2 * (r * blocks + j // 16) + (j >> 2 & 1)."""
    blocks, t = (Tk + 15) // 16, threshold(p)
    u = random16(range(B * H * Tq * blocks * 2), seed, step, channel).reshape(B * H * Tq, blocks * 2, 8)
    j = np.arange(Tk)
    u = u[:, 2 * (j // 16) + (j >> 2 & 1), (j & 3) + 4 * (j >> 3 & 1)]
    return ((u >= t) * (65536.0 / (65536 - t))).reshape(B, H, Tq, Tk)


def bucket(rel, buckets, max_distance, bidirectional):
    """Bucket of a relative position (key minus query), by whole numbers."""
    side = buckets // 2 if bidirectional else buckets
    first = side // 2
    n = abs(rel) if bidirectional else max(0, -rel)
    b = n
    if n >= first:
        e, n = 0, min(n, max_distance)
        while e + 1 < side - first and n ** (side - first) * first ** (e + 1) >= max_distance ** (e + 1) * first ** (side - first):
            e += 1
        b = first + e
    return b + (side if bidirectional and rel > 0 else 0)


class Attention(object):
    """softmax(scale * q k^T + table[bucket(j - i - offset)]) (with dropout) v and its gradients, for q, k, v [B,H,T,D]."""

    def __init__(self, q, k, v, table=None, scale=None, causal=False, bidirectional=None, max_distance=128, q_offset=0,
                 q_lengths=None, k_lengths=None, keep=None):
        self.q, self.k, self.v = (np.asarray(a, np.float64) for a in (q, k, v))
        B, H, Tq, D = self.q.shape
        Tk = self.k.shape[2]
        self.scale = D ** -0.5 if scale is None else scale
        i, j = np.arange(Tq)[:, None], np.arange(Tk)[None, :]
        s = self.scale * np.einsum("bhid,bhjd->bhij", self.q, self.k)
        self.bucket = self.buckets = None
        if table is not None:
            self.buckets = table.shape[0]
            bidirectional = not causal if bidirectional is None else bidirectional
            by_rel = {r: bucket(r, self.buckets, max_distance, bidirectional) for r in range(-q_offset - Tq, Tk - q_offset + 1)}
            self.bucket = np.array([[by_rel[int(jj - ii - q_offset)] for jj in range(Tk)] for ii in range(Tq)], np.int64).reshape(Tq, Tk)
            s = s + np.asarray(table, np.float64)[self.bucket].transpose(2, 0, 1)
        seen = np.ones((B, 1, Tq, Tk), bool)
        if causal:
            seen &= j <= i + q_offset
        if k_lengths is not None:
            seen &= j < np.clip(k_lengths, 0, Tk)[:, None, None, None]
        self.q_seen = np.ones((B, 1, Tq, 1), bool)
        if q_lengths is not None:
            self.q_seen = i < np.clip(q_lengths, 0, Tq)[:, None, None, None]
            seen &= self.q_seen
        s = np.where(seen, s, -np.inf)
        top = s.max(-1, initial=-np.inf, keepdims=True)
        top = np.where(top == -np.inf, 0.0, top)
        e = np.exp(s - top)
        total = e.sum(-1, keepdims=True)
        self.prob = e / np.where(total == 0, 1.0, total)
        self.keep = 1.0 if keep is None else keep
        # masked values do not reach a sum, whatever they hold
        self.vm = self.v if k_lengths is None else np.where(
            np.arange(Tk)[None, None, :, None] < np.clip(k_lengths, 0, Tk)[:, None, None, None], self.v, 0.0)
        self.o = np.einsum("bhij,bhjd->bhid", self.prob * self.keep, self.vm)
        with np.errstate(divide="ignore"):
            self.lse = (top + np.log(total))[..., 0]

    def pullback(self, go):
        go = np.where(self.q_seen, np.asarray(go, np.float64), 0.0)
        gp = np.einsum("bhid,bhjd->bhij", go, self.vm) * self.keep
        gv = np.einsum("bhij,bhid->bhjd", self.prob * self.keep, go)
        gs = self.prob * (gp - (go * self.o).sum(-1, keepdims=True))
        gq = self.scale * np.einsum("bhij,bhjd->bhid", gs, self.k)
        gk = self.scale * np.einsum("bhij,bhid->bhjd", gs, self.q)
        gtable = None
        if self.bucket is not None:
            total = gs.sum(0)
            gtable = np.stack([(total * (self.bucket == b)).sum((1, 2)) for b in range(self.buckets)])
        return gq, gk, gv, gtable
