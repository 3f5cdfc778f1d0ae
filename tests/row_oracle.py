"""Plain 64-bit forms of the row operators (layer norm, counter-based dropout, the tail of a hidden layer), with the error
that a 32-bit evaluation may have, for the tests of artifact_amd.row_ops.  numpy only."""
import numpy as np

U = 2.0 ** -24          # half a step of float32, relative to the value
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8}


def philox(counter, key, rounds=7):
    """Philox4x32 (Salmon, Moraes, Dror, Shaw 2011).  counter: [..., 4], key: [2], whole numbers below 2^32."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    mask = np.uint64(0xFFFFFFFF)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1)


def threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def kept(rows, f, p, seed, offset):
    """bool [len(rows), f]: the elements that dropout keeps in the rows of these numbers."""
    groups = (f + 7) // 8
    i = (np.asarray(rows, dtype=np.uint64)[:, None] * np.uint64(groups) + np.arange(groups, dtype=np.uint64)).ravel()
    seed, offset = int(seed) % 2 ** 64, int(offset) % 2 ** 64
    c = np.zeros((len(i), 4), dtype=np.uint64)
    c[:, 0], c[:, 1] = i & np.uint64(0xFFFFFFFF), i >> np.uint64(32)
    c[:, 2], c[:, 3] = offset & 0xFFFFFFFF, offset >> 32
    w = philox(c, (seed & 0xFFFFFFFF, seed >> 32))
    u = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(len(rows), groups * 8)[:, :f]
    return u >= np.uint64(threshold(p))


def scale(p):
    return 65536.0 / (65536 - threshold(p)) if threshold(p) < 65536 else 0.0


class Norm:
    """Forward and backward of dropout(relu(layer_norm(x))) in 64 bits, and what 32 bits may be off by.

    A lane adds at most 32 numbers of a row, the cross-lane sum at most 22 more (54 additions), each off by u of the sum of
    the magnitudes; the mean is then off by 55 u mean|x| <= 55 u (|m| + 1/r), h = (x - m) r by that times r, by as much
    again through r, and by the roundings of its own operations: below a = 128 u (r (|x| + |m|) + 1) for |m| r up to 2^10."""

    def __init__(self, x, weight=None, bias=None, eps=1e-5, relu=False, keep=None, p=0.0):
        x = np.asarray(x, dtype=np.float64)
        f = x.shape[1]
        self.w = np.ones(f) if weight is None else np.asarray(weight, dtype=np.float64)
        self.b = np.zeros(f) if bias is None else np.asarray(bias, dtype=np.float64)
        m = x.mean(1, keepdims=True)
        self.r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + eps)
        self.h = (x - m) * self.r
        self.a = 128 * U * (self.r * (np.abs(x) + np.abs(m)) + 1)
        self.pre = self.h * self.w + self.b
        self.pre_tol = self.a * np.abs(self.w) + 128 * U * np.abs(self.b)
        self.factor = np.ones_like(x) if keep is None else keep * scale(p)
        self.gate = self.pre > 0 if relu else np.ones_like(x, dtype=bool)
        self.y = np.where(self.factor != 0, (np.maximum(self.pre, 0) if relu else self.pre) * self.factor, 0.0)
        self.y_tol = np.abs(self.factor) * self.pre_tol + 4 * U * np.abs(self.y)

    def backward(self, dy):
        """(dx, dw, db) and their tolerances.  The sums over a row are off by 60 u of the magnitudes added; the sums over rows
        by ceil(n / 1024) + 100 additions (the rows of one lane, then a fixed tree of at most 100)."""
        d = np.where((self.factor != 0) & self.gate, np.asarray(dy, dtype=np.float64) * self.factor, 0.0)
        n = len(d)
        g = d * self.w
        s1, s2 = g.mean(1, keepdims=True), (g * self.h).mean(1, keepdims=True)
        dx = self.r * (g - s1 - self.h * s2)
        e1 = 60 * U * np.abs(g).mean(1, keepdims=True)
        e2 = 60 * U * np.abs(g * self.h).mean(1, keepdims=True) + (np.abs(g) * self.a).mean(1, keepdims=True)
        dx_tol = self.r * (e1 + np.abs(self.h) * e2 + self.a * np.abs(s2) + 8 * U * (np.abs(g) + np.abs(s1) + np.abs(self.h * s2)))
        dx_tol = dx_tol + 128 * U * np.abs(dx)      # of r: 30 u from its sum, (55 u (|m| r + 1))^2 / 2 < 94 u from the mean
        adds = -(-n // 1024) + 100
        dw, db = (d * self.h).sum(0), d.sum(0)
        dw_tol = (np.abs(d) * self.a).sum(0) + (adds + 4) * U * np.abs(d * self.h).sum(0)
        db_tol = (adds + 4) * U * np.abs(d).sum(0)
        return (dx, dw, db), (dx_tol, dw_tol, db_tol)
