"""The 4-bit cache bank in plain numpy, 64 bits throughout: what tests/test_cache_bank*.py compare the kernels with."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """float64 [..., dim] -> (element values on the grid [..., blocks, 32], exponents [..., blocks]); finite input."""
    dim = x.shape[-1]
    x = np.concatenate([x, np.zeros(x.shape[:-1] + ((-dim) % 32,))], -1).reshape(x.shape[:-1] + (-1, 32))
    top = np.abs(x).max(-1)
    e = np.full(top.shape, -126)
    for k in range(-126, 125):                          # the smallest exponent whose 7 * 2^e covers the block
        e = np.where(top > 7.0 * 2.0 ** k, k + 1, e)
    y = x / 2.0 ** e[..., None]
    a = np.minimum(np.abs(y), 6.0)
    near = np.abs(a[..., None] - GRID)
    best = near.min(-1, keepdims=True)
    tie = near == best                                   # one candidate, or two neighbours: then the even code
    code = np.where(tie & (np.arange(8) % 2 == 0), np.arange(8), -1).max(-1)
    code = np.where(tie.sum(-1) == 1, tie.argmax(-1), code)
    return GRID[code] * np.where(np.signbit(y), -1.0, 1.0), e


def held_pair(key, value):
    """The float64 values that the bank holds for rows [..., dim] of one head; a row with a non-finite entry on either side is NaN on both."""
    out = []
    bad = ~(np.isfinite(key).all(-1) & np.isfinite(value).all(-1))
    for x in (key, value):
        x = np.where(bad[..., None], 0.0, x).astype(np.float64)
        v, e = quantise(x)
        v = (v * 2.0 ** e[..., None]).reshape(x.shape[:-1] + (-1,))[..., :x.shape[-1]]
        out.append(np.where(bad[..., None], np.nan, v))
    return out


class RefBank:
    """Lists of rows for each (sequence, head): (key, value, weight, position)."""

    def __init__(self, batch, heads, dim, k):
        self.batch, self.heads, self.dim, self.k = batch, heads, dim, k
        self.key = [[np.zeros((0, dim)) for _ in range(heads)] for _ in range(batch)]
        self.value = [[np.zeros((0, dim)) for _ in range(heads)] for _ in range(batch)]
        self.weight = [[np.zeros(0) for _ in range(heads)] for _ in range(batch)]
        self.position = [[np.zeros(0, int) for _ in range(heads)] for _ in range(batch)]
        self.seen = [0] * batch

    def length(self, b):
        return len(self.weight[b][0])

    def push(self, key, value, counts=None):
        T = key.shape[2]
        held = held_pair(key, value)
        for b in range(self.batch):
            n = T if counts is None else int(counts[b])
            for h in range(self.heads):
                self.key[b][h] = np.concatenate([self.key[b][h], held[0][b, h, :n]])
                self.value[b][h] = np.concatenate([self.value[b][h], held[1][b, h, :n]])
                self.weight[b][h] = np.concatenate([self.weight[b][h], np.zeros(n)])
                self.position[b][h] = np.concatenate([self.position[b][h], self.seen[b] + np.arange(n)])
            for side in held:
                side[b, :, n:] = 0.0
            self.seen[b] += n
        return held

    def trim(self, lengths):
        for b in range(self.batch):
            n = int(lengths[b] if np.ndim(lengths) else lengths)
            self.seen[b] -= max(0, self.length(b) - n)
            for part in (self.key, self.value, self.weight, self.position):
                part[b] = [x[:n] for x in part[b]]

    def attend(self, query, counts=None, scale=None, causal=True, accumulate=False):
        """(out, bound): float64 results and how far float32 arithmetic with outputs rounded elsewhere may be off.

        The bound counts: scores are float32 sums of dim exact products (dim roundings of 2^-24 relative to the sum of magnitudes, and as
        many again for an order that is not sequential), times the scale, less the maximum, through exp2 (a few more); their error
        enters p relatively, twice (numerator and denominator).  Sums over n rows are float32 in at least 16 partial sums.  What is
        below 2^-126 in float32 and bfloat16 may be taken as zero: exp's result (at most 1, the denominator at least 1) and each of its
        up to three pieces, so every p is off by up to 4 * 2^-126 besides, and a result by that times the sum of |value|."""
        scale = self.dim ** -0.5 if scale is None else scale
        group, T = query.shape[1] // self.heads, query.shape[2]
        out, bound = np.zeros(query.shape), np.zeros(query.shape)
        weigh_bound = [[np.zeros(len(w)) for w in row] for row in self.weight]
        for b in range(self.batch):
            n = T if counts is None else int(counts[b])
            for h in range(self.heads):
                K, V = self.key[b][h], self.value[b][h]
                got = np.zeros(len(K))
                for g in range(group):
                    for t in range(n):
                        see = len(K) - n + t + 1 if causal else len(K)
                        if see <= 0:
                            continue
                        q = query[b, h * group + g, t]
                        s = K[:see] @ q * scale
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        out[b, h * group + g, t] = p @ V[:see]
                        mag = (np.abs(K[:see]) @ np.abs(q)).max() * scale
                        rel = 2.0 ** -24 * (4 * (self.dim + 16) * mag + see / 16 + 64)
                        bound[b, h * group + g, t] = rel * (p @ np.abs(V[:see])) + 4 * 2.0 ** -126 * np.abs(V[:see]).sum(0)
                        got[:see] += p
                        weigh_bound[b][h][:see] += rel * p
                if accumulate:
                    self.weight[b][h] = self.weight[b][h] + got
                    weigh_bound[b][h] += 2.0 ** -24 * 64 * np.abs(self.weight[b][h])
        return (out, bound, weigh_bound) if accumulate else (out, bound)

    def evict(self, keep, recent=0):
        for b in range(self.batch):
            for h in range(self.heads):
                w, pos = self.weight[b][h], self.position[b][h]
                if len(w) <= keep:
                    continue
                fresh = pos >= self.seen[b] - recent

                def rank(i):
                    if fresh[i]:
                        return (0, 0.0, i)
                    return (1, 0.0, i) if np.isnan(w[i]) else (2, -w[i], i)

                stay = set(sorted(range(len(w)), key=rank)[:keep])
                above = iter(sorted(i for i in stay if i >= keep))
                source = [i if i in stay else next(above) for i in range(keep)]
                for part in (self.key, self.value, self.weight, self.position):
                    part[b][h] = part[b][h][source]
