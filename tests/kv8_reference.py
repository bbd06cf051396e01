"""Plain 64-bit restatement of the 8-bit KV cache's operators (tests only), token by token, on the CPU."""
import math

import torch

MIN_EXP, MAX_EXP = -110, 120


def exponent(top):
    """Least e with top <= 448 * 2^e, clamped."""
    if not top > 0:
        return MIN_EXP
    e = math.frexp(top)[1] - 9
    if top > 448 * 2.0 ** e:
        e += 1
    return min(max(e, MIN_EXP), MAX_EXP)


def to_e4m3(x):
    """Nearest e4m3 value of each element, ties to even, infinities to +-448; x float64."""
    y = torch.where(torch.isinf(x), torch.sign(x) * 448.0, x)
    assert not (y.abs() > 448).any()
    e = torch.frexp(torch.where(y == 0, torch.ones_like(y), y))[1].to(torch.float64) - 1
    step = torch.exp2(torch.clamp(e, min=-6) - 3)          # three mantissa bits; below 2^-6 the step stays 2^-9
    y = torch.round(y / step) * step                       # torch.round: half to even
    return torch.where(torch.isnan(x), x, y)


class Cache:
    """The cache as numbers: values [2, blocks, heads, size, dim] and exponents [2, blocks, heads]."""

    def __init__(self, cache):
        self.values = cache.values.cpu().double()
        self.scales = cache.scales.cpu().double()
        self.size = cache.block_size

    def rows(self, kv, table, head, n):
        """[n, dim]: what the first n tokens of a block table hold."""
        out = [self.values[kv, int(table[j // self.size]), head, j % self.size] * self.scales[kv, int(table[j // self.size]), head]
               for j in range(n)]
        return torch.stack(out) if out else torch.zeros((0, self.values.shape[-1]), dtype=torch.float64)

    def store(self, kv, block, head, rows):
        """{row: numbers} go into one tile whose other rows do not count: a scale of their own."""
        finite = [r[torch.isfinite(r)].abs().max().item() if torch.isfinite(r).any() else 0.0 for r in rows.values()]
        scale = 2.0 ** exponent(max(finite))
        self.scales[kv, block, head] = scale
        for row, x in rows.items():
            self.values[kv, block, head, row] = to_e4m3(x / scale)

    def append(self, x, kv, table, old, head):
        """x [n, dim] float64 becomes tokens old, old + 1, ...; all new rows of a block are written together."""
        n, i = x.shape[0], 0
        while i < n:
            pos = old + i
            block, row = int(table[pos // self.size]), pos % self.size
            m = min(self.size - row, n - i)
            new = x[i:i + m]
            fin = new[torch.isfinite(new)]
            scale = 2.0 ** exponent(fin.abs().max().item() if fin.numel() else 0.0)
            if row:
                was = float(self.scales[kv, block, head])
                was = 2.0 ** min(max(math.frexp(was)[1] - 1, MIN_EXP), MAX_EXP) if was > 0 else 2.0 ** MIN_EXP
                if scale > was:
                    self.values[kv, block, head, :row] = to_e4m3(self.values[kv, block, head, :row] * (was / scale))
                scale = max(scale, was)
            self.scales[kv, block, head] = scale
            self.values[kv, block, head, row:row + m] = to_e4m3(new / scale)
            i += m


def attention(q, cache, tables, lens, starts, scale, causal):
    """(out, lse, magnitude, weights): magnitude = sum p |v|, weights[s][head] = each token's summed probability;
    spread = scale * sum |q| |k|, the size that a score's rounding goes by."""
    rows, q_heads, dim = q.shape
    heads = cache.values.shape[2]
    group = q_heads // heads
    out = torch.zeros((rows, q_heads, dim), dtype=torch.float64)
    size_of = torch.zeros_like(out)
    lse = torch.full((rows, q_heads), -math.inf, dtype=torch.float64)
    spread = torch.zeros((rows, q_heads), dtype=torch.float64)
    weights = [[torch.zeros(int(n), dtype=torch.float64) for _ in range(heads)] for n in lens]
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        for head in range(heads):
            k, v = cache.rows(0, tables[s], head, n), cache.rows(1, tables[s], head, n)
            for i in range(a, b):
                see = min(max(n - (b - a) + (i - a) + 1, 0), n) if causal else n
                if not see:
                    continue
                for g in range(head * group, (head + 1) * group):
                    x = q[i, g].double()
                    sc = (k[:see] @ x) * scale
                    lse[i, g] = torch.logsumexp(sc, 0)
                    p = torch.exp(sc - lse[i, g])
                    out[i, g] = p @ v[:see]
                    size_of[i, g] = p @ v[:see].abs()
                    spread[i, g] = (k[:see].abs() @ x.abs()).max() * abs(scale)
                    weights[s][head][:see] += p
    return out, lse, size_of, spread, weights


def choose(w, n, keep, recent):
    """Indices that eviction keeps of one sequence and head; w: list of floats."""
    r = min(recent, n)
    key = [(-math.inf, 1) if math.isnan(w[j]) else (w[j], 0) for j in range(n - r)]
    order = sorted(range(n - r), key=lambda j: (key[j][1], -key[j][0], j))
    return sorted(order[: min(n, keep) - r]) + list(range(n - r, n))
