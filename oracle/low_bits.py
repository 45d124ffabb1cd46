"""Plain float64 restatements of the operators that hold a decoder's cache in 8 bits and its weights in 4: the cache of
pages with their unrounded tail, attention over it, and microscaled 4-bit rows.  CPU tensors, loops where they are
clearest."""
import math

import torch

GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pow2(e):
    """2^e in float64, exactly (e an integer tensor)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


# ----------------------------------------------------------------------------------------------- e4m3 pages
def scale8(x):
    """The scale of a block of float64 values: the smallest power of two that brings the largest finite magnitude to 448
    or less, within [2^-126, 2^127]; 1 when nothing but zeros (or nothing finite) is there."""
    fin = x[torch.isfinite(x)].abs()
    amax = float(fin.max()) if fin.numel() else 0.0
    if amax == 0.0:
        return 1.0
    e = -126
    while e < 127 and amax > 448.0 * math.ldexp(1.0, e):
        e += 1
    return math.ldexp(1.0, e)


def round8(y):
    """Nearest e4m3 number, halves to even; NaN for what is not finite.  |y| <= 448."""
    ex = torch.frexp(y)[1].clamp(min=-5) - 1
    step = pow2(ex - 3)
    return torch.where(torch.isfinite(y), torch.round(y / step) * step, float('nan'))


class Cache:
    """(B, H) caches of at most tcap positions: blocks[b][h][j] = (codes (2, leaf, D) float64, scales (2,)) of the blocks
    that are whole, tail (B, H, 2, leaf, D) float64 and held[b][h], the block the tail holds (-1: none).  pages: bool
    (B, H, blocks), whether a block has a page."""

    def __init__(self, B, H, D, leaf, tcap, pages=None):
        self.B, self.H, self.D, self.leaf, self.tcap = B, H, D, leaf, tcap
        self.blocks = [[{} for _ in range(H)] for _ in range(B)]
        self.tail = torch.zeros(B, H, 2, leaf, D, dtype=torch.float64)
        self.held = [[-1] * H for _ in range(B)]
        self.pages = pages if pages is not None else torch.ones(B, H, (tcap + leaf - 1) // leaf, dtype=torch.bool)

    def close(self, b, h, j, rows):
        sc = [scale8(rows[i]) for i in (0, 1)]
        self.blocks[b][h][j] = (torch.stack([round8(rows[i] / sc[i]) for i in (0, 1)]), sc)

    def page_rows(self, b, h, j):
        if j not in self.blocks[b][h]:
            return torch.zeros(2, self.leaf, self.D, dtype=torch.float64)
        codes, sc = self.blocks[b][h][j]
        return codes * torch.tensor(sc, dtype=torch.float64).view(2, 1, 1)

    def append(self, b, h, t, k, v):
        if not 0 <= t < self.tcap or not self.pages[b, h, t // self.leaf]:
            return
        j, r = divmod(t, self.leaf)
        if self.held[b][h] != j and r:
            self.tail[b, h, :, :r] = self.page_rows(b, h, j)[:, :r]
        self.tail[b, h, 0, r], self.tail[b, h, 1, r] = k.double(), v.double()
        self.held[b][h] = j
        if r == self.leaf - 1:
            self.close(b, h, j, self.tail[b, h])

    def key(self, b, h, pos):
        """(k, v) of a position, or None when its block has no page and is not in the tail."""
        j, r = divmod(pos, self.leaf)
        if j == self.held[b][h]:
            return self.tail[b, h, :, r]
        if not self.pages[b, h, j]:
            return None
        return self.page_rows(b, h, j)[:, r]


def attend8(cache, q, b, h, t, leaves, neighbours, local, scale):
    """Attention of one query q (D,) float64 at position t over `leaves` (blocks, as far as its budget goes), the matched
    `neighbours` (each once, before the own block), the own block up to t and the static keys 0, t, t-1, ...: (out, lse,
    number of keys); zeros and -1e30 without a key."""
    leaf = cache.leaf
    zero = torch.zeros(cache.D, dtype=torch.float64)
    if not 0 <= t < cache.tcap:
        return zero, -1e30, 0
    own = t // leaf
    used = list(leaves)
    for j in neighbours:
        if 0 <= j < own and j not in used:
            used.append(j)
    pos = [p for j in used for p in range(j * leaf, (j + 1) * leaf)]
    pos += list(range(own * leaf, t + 1))
    n = len(pos)
    for p in [0] + [t - i for i in range(max(local, 3))]:
        if p >= 0 and p < own * leaf and p // leaf not in used and p not in pos:
            pos.append(p)
            n += 1
    kv = [cache.key(b, h, p) for p in pos if 0 <= p // leaf < cache.pages.shape[2]]
    kv = [x for x in kv if x is not None]
    if not kv:
        return zero, -1e30, n
    kv = torch.stack(kv)
    s = kv[:, 0] @ q * scale
    return torch.softmax(s, 0) @ kv[:, 1], float(torch.logsumexp(s, 0)), n


# ----------------------------------------------------------------------------------------------- 4-bit rows
def quant4(x):
    """x (rows, K) float64 -> (codes (rows, Kp) int, scale bytes (rows, Kp / 32) int, values (rows, K) float64)."""
    rows, K = x.shape
    Kp = (K + 127) // 128 * 128
    pad = torch.zeros(rows, Kp, dtype=torch.float64)
    pad[:, :K] = x
    blk = pad.view(rows, Kp // 32, 32)
    bad = ~torch.isfinite(blk).all(-1)
    blk = torch.where(bad.unsqueeze(-1), 0.0, blk)
    amax = blk.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(min=-127)
    a = blk.abs() / pow2(e).unsqueeze(-1)
    code = torch.zeros_like(a, dtype=torch.long)
    for i in range(1, 8):
        border = (GRID4[i - 1] + GRID4[i]) / 2
        code[(a >= border) if i % 2 == 0 else (a > border)] = i
    val = torch.tensor(GRID4, dtype=torch.float64)[code] * pow2(e).unsqueeze(-1)
    neg = torch.signbit(blk)
    val = torch.where(bad.unsqueeze(-1), float('nan'), torch.where(neg, -val, val))
    code = code + 8 * neg.long()
    byte = torch.where(bad, 255, e.long() + 127)
    return code.view(rows, Kp), byte, val.view(rows, Kp)[:, :K]


def layernorm_product(x, w, g, eps):
    """LN(x) @ w.T of x (M, K), w (N, K), g (K,) in float64, and how far an evaluation may be from it that takes mean and
    deviation in float32 and holds every normalised value n to 2^-16 of it:
    - the mean is off by d * 2^-24 of the mean magnitude and the deviation by d * 2^-24 of itself (d roundings one after
      another: eight values a vector, a vector for every 4096 of a row, and the joins); both are common to a row, so the first
      moves a result by that times |sum of g w| / deviation, the second by that times the result;
    - the values' own errors, 2^-16 and three float32 roundings, are independent: six times their root sum of squares;
    - so are the 2 K roundings of the float32 sums (2^-23 each of a partial sum, which stays within six times the root sum
      of squares of the products)."""
    x, w, g = x.double(), w.double(), g.double()
    K = x.shape[1]
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    dev = torch.sqrt(var + eps)
    n = (x - mean) / dev * g
    y = n @ w.T
    d = (30 + K / 4096) * 2.0 ** -24
    rss = torch.sqrt((n * n) @ (w * w).T)
    tol = (d * y.abs() + d * x.abs().mean(-1, keepdim=True) / dev * (w @ g).abs()
           + 6 * (2.0 ** -16 + 3 * 2.0 ** -24) * rss + 6 * 2.0 ** -23 * math.sqrt(2 * K) * 6 * rss)
    return y, tol
