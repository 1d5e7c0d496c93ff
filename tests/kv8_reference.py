"""The operators around the 8-bit cache in 64 bits, from their definition: what the tests compare with."""
import math

import torch

D, BLOCK, RECORD, LARGEST = 128, 16, 4112, 448.0


def grid():
    """The 256 values of e4m3 in 64 bits; 0x7F and 0xFF are NaN."""
    out = []
    for c in range(256):
        e, m = c // 8 % 16, c % 8
        size = math.nan if c % 128 == 127 else m / 512 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out.append(-size if c >= 128 else size)
    return torch.tensor(out, dtype=torch.float64)


def codes_of(y):
    """Values in 64 bits to the nearest codes, ties to even, cut at 448; the sign of zero stays. NaN (codes that no append has written) to 0x7F."""
    sizes = grid()[:127]
    a = y.abs().clamp(max=LARGEST)
    high = torch.searchsorted(sizes, a).clamp(max=126)          # the first size >= a
    low = (high - 1).clamp(min=0)
    d_low, d_high = a - sizes[low], sizes[high] - a
    code = torch.where((d_low < d_high) | ((d_low == d_high) & (low % 2 == 0)), low, high)
    return torch.where(torch.isnan(y), 127, code + 128 * torch.signbit(y).long()).to(torch.uint8)


def scale_of(largest):
    """The smallest power of two with largest <= 448 times it, from 2^-90 to 2^119."""
    s = 2.0 ** -90
    while largest > LARGEST * s and s < 2.0 ** 119:
        s *= 2
    return s


def places():
    """Byte of each token's elements in a block's K part and V part, int64 [16, 128] each."""
    k, v = torch.zeros(BLOCK, D, dtype=torch.int64), torch.zeros(BLOCK, D, dtype=torch.int64)
    for t in range(BLOCK):
        for d in range(D):
            j = t // 2
            k[t, d] = 128 * t + 16 * ((d // 16) ^ (t % 8)) + d % 16
            v[t, d] = 2048 + 256 * j + 16 * ((d // 8) ^ (j % 2 + 4 * (j // 2 % 2))) + 2 * (d % 8) + t % 2
    return k, v


PLACES = places()


class Block:
    """Views of one block: a page, a head, a number within the page."""

    def __init__(self, pool, page, head, number):
        self.bytes = pool[page, head, RECORD * number:RECORD * (number + 1)]

    def codes(self, part):
        return self.bytes[PLACES[part]]

    def set_codes(self, part, at, codes):
        self.bytes[PLACES[part][at]] = codes

    def scale(self, part):
        return self.bytes[4096 + 4 * part:4100 + 4 * part].clone().view(torch.float32).double().item()

    def mask(self, part):
        return int(self.bytes[4104 + 2 * part]) | int(self.bytes[4105 + 2 * part]) << 8

    def set_meta(self, part, scale, mask):
        self.bytes[4096 + 4 * part:4100 + 4 * part] = torch.tensor([scale], dtype=torch.float32).view(torch.uint8)
        self.bytes[4104 + 2 * part], self.bytes[4105 + 2 * part] = mask & 255, mask >> 8

    def values(self, part):
        v = grid()[self.codes(part).long()] * self.scale(part)
        v[torch.tensor([self.mask(part) >> t & 1 for t in range(BLOCK)], dtype=torch.bool)] = math.nan
        return v


def page_tokens(pool):
    return pool.shape[2] // 257


def block_at(pool, table, b, head, t):
    """The block of token t, None where the table names no page of the pool."""
    page = page_tokens(pool)
    number = int(table[b, t // page])
    return Block(pool, number, head, t % page // BLOCK) if 0 <= number < pool.shape[0] else None


def new_tokens(lengths, counts, S):
    out = []
    for b, L in enumerate(lengths):
        n = min(S, L)
        out.append(n if counts is None else max(0, min(n, int(counts[b]))))
    return out


def append(pool, table, lengths, counts, k, v):
    """Changes pool (on the CPU) as an append does."""
    HK, S = pool.shape[1], k.shape[1]
    for b, (L, n) in enumerate(zip(lengths, new_tokens(lengths, counts, S))):
        first = L - n
        for start in range(first // BLOCK * BLOCK, L if n else 0, BLOCK):
            at = torch.arange(start, min(start + BLOCK, L))
            new = at[at >= first]
            old = int((at < first).sum())
            for h in range(HK):
                block = block_at(pool, table, b, h, start)
                if block is None:
                    continue
                for part, x in ((0, k), (1, v)):
                    rows = x[b, new - first, h].double()
                    broken = ~torch.isfinite(rows).all(-1)
                    rows = torch.where(broken[:, None], 0.0, rows)
                    scale, mask = scale_of(rows.abs().max().item()), 0
                    if old:
                        before = block.scale(part)
                        scale, mask = max(scale, before), block.mask(part) & ((1 << old) - 1)
                        if scale > before:
                            was = torch.arange(old)
                            block.set_codes(part, was, codes_of(grid()[block.codes(part)[was].long()] * (before / scale)))
                    block.set_codes(part, new - start, codes_of(rows / scale))
                    for t, bad in zip((new - start).tolist(), broken.tolist()):
                        mask |= int(bad) << t
                    block.set_meta(part, scale, mask)


def tokens(pool, table, b, head, n):
    """K, V f64 [n, 128] and V's scales [n] of the first n tokens of a sequence."""
    k, v, scale = (torch.full((n, D), math.nan, dtype=torch.float64) for _ in range(2)), None, torch.ones(n, dtype=torch.float64)
    k, v = k
    for start in range(0, n, BLOCK):
        block, m = block_at(pool, table, b, head, start), min(BLOCK, n - start)
        if block is not None:
            k[start:start + m], v[start:start + m], scale[start:start + m] = block.values(0)[:m], block.values(1)[:m], block.scale(1)
    return k, v, scale


def attend(q, pool, table, lengths, causal, counts=None, scale=None):
    """out, lse in 64 bits, and what the tolerances are made of: per output element sum p |v|, per row the largest p times V's scale of a token and the largest sum |q k| scale."""
    B, S, H, _ = q.shape
    HK = pool.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, spread = torch.zeros(B, S, H, D, dtype=torch.float64), torch.zeros(B, S, H, D, dtype=torch.float64)
    lse, peak, size = torch.full((B, H, S), -math.inf, dtype=torch.float64), torch.zeros(B, H, S, dtype=torch.float64), torch.zeros(B, H, S, dtype=torch.float64)
    cap = table.shape[1] * page_tokens(pool)
    lengths = [max(0, min(int(n), cap)) for n in lengths]
    for b, (L, n) in enumerate(zip(lengths, new_tokens(lengths, counts, S))):
        if n == 0 or L == 0:
            continue
        hidden = torch.arange(L) > (L - n + torch.arange(n))[:, None] if causal else torch.zeros(n, L, dtype=torch.bool)
        for hk in range(HK):
            k, v, vs = tokens(pool, table, b, hk, L)
            for h in range(hk * (H // HK), (hk + 1) * (H // HK)):
                rows = q[b, :n, h].double()
                x = (rows @ k.T * scale).masked_fill(hidden, -math.inf)
                lse[b, h, :n] = torch.logsumexp(x, 1)
                p = torch.exp(x - lse[b, h, :n, None]).masked_fill(hidden, 0.0)
                seen = torch.where(hidden[..., None], 0.0, v) if torch.isnan(v).any() else v
                out[b, :n, h] = torch.einsum("st,std->sd", p, seen) if seen.dim() == 3 else p @ seen
                spread[b, :n, h] = p @ v.abs().nan_to_num()
                peak[b, h, :n] = (p * vs).nan_to_num().amax(1)
                size[b, h, :n] = (rows.abs() @ k.abs().nan_to_num().T * scale).masked_fill(hidden, 0.0).amax(1)
    return out, lse, spread, peak, size
