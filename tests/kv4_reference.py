"""The operators around the 4-bit cache in 64 bits, from their definition, on whatever device the tensors are: what the tests compare with."""
import math

import torch

D, BLOCK, TOKEN = 128, 32, 136
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def element_of_nibble():
    """The element of a head in each of a token's 128 nibbles: byte 8 g + 2 b + r holds 32 b + 4 g + 2 r (low) and the next."""
    at = []
    for byte in range(64):
        g, b, r = byte // 8, byte // 2 % 4, byte % 2
        at += [32 * b + 4 * g + 2 * r, 32 * b + 4 * g + 2 * r + 1]
    return torch.tensor(at)


def power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def encode(x):
    """bf16 [n, 128] to (codes [n, 64], scales [n, 4], values f64 [n, 128])."""
    x = x.double()
    n = x.shape[0]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    blocks = x.view(n, 4, BLOCK)
    broken = ~torch.isfinite(blocks).all(-1)
    blocks = torch.where(broken[..., None], torch.zeros_like(blocks), blocks)
    top = blocks.abs().amax(-1)
    e = torch.where(top == 0, 1, torch.frexp(top).exponent - 1 - 2 + 127).clamp(1, 252)
    y = blocks * power(127 - e).unsqueeze(-1)
    a = y.abs().clamp(max=6.0)
    low = (a[..., None] >= grid).sum(-1) - 1
    high = (low + 1).clamp(max=7)
    d_low, d_high = a - grid[low], grid[high] - a
    code = torch.where((d_high < d_low) | ((d_high == d_low) & (low % 2 == 1)), high, low)
    value = torch.copysign(grid[code], y) * power(e - 127).unsqueeze(-1)
    value = torch.where(broken[..., None], torch.full_like(value, math.nan), value).view(n, D)
    nibble = (code + 8 * torch.signbit(y).long()).masked_fill(broken[..., None], 0).view(n, D)[:, element_of_nibble().to(x.device)]
    return (nibble[:, 0::2] + 16 * nibble[:, 1::2]).to(torch.uint8), torch.where(broken, 255, e).to(torch.uint8), value


def decode(codes, scales):
    """codes [n, 64], scales [n, 4] to values f64 [n, 128]."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device=codes.device)
    nibble = torch.stack([codes & 15, codes >> 4], -1).view(-1, D).long()
    value = torch.zeros(codes.shape[0], D, dtype=torch.float64, device=codes.device)
    value[:, element_of_nibble().to(codes.device)] = grid[nibble]
    s = power(scales.long() - 127)
    s = torch.where(scales == 0, 0.0, torch.where(scales == 255, math.nan, s)).repeat_interleave(BLOCK, 1)
    return value * s


def record(pool, page, head, part):
    """Views of the codes [page, 64] and scales [page, 4] of one page and head; part 0: K, 1: V."""
    p = pool.shape[2] // TOKEN
    r = pool[page, head]
    return r[64 * p * part:64 * p * (part + 1)].view(p, 64), r[(128 + 4 * part) * p:(132 + 4 * part) * p].view(p, 4)


def tokens(pool, table_row, head, n):
    """K and V, f64 [n, 128], of the first n tokens of a sequence."""
    p = pool.shape[2] // TOKEN
    out = []
    for part in (0, 1):
        got = [decode(*record(pool, int(page), head, part)) for page in table_row[:-(-n // p)]]
        out.append(torch.cat(got)[:n] if got else torch.zeros(0, D, dtype=torch.float64, device=pool.device))
    return out


def attend(q, pool, table, lengths, causal, counts=None, scale=None, weights_in=None):
    """out, lse, weights in 64 bits, and what the tolerances are made of: per output element sum p |v|, per row the
    largest p |v| of a token and the largest sum |q k| scale, per weight sum p times that."""
    B, S, H, _ = q.shape
    HK, width = pool.shape[1], table.shape[1] * (pool.shape[2] // TOKEN)
    scale = 1 / math.sqrt(D) if scale is None else scale
    f64 = dict(dtype=torch.float64, device=q.device)
    out, spread, peak, size = torch.zeros(B, S, H, D, **f64), torch.zeros(B, S, H, D, **f64), torch.zeros(B, S, H, **f64), torch.zeros(B, H, S, **f64)
    lse = torch.full((B, H, S), -math.inf, **f64)
    weights, doubt = torch.zeros(B, HK, width, **f64), torch.zeros(B, HK, width, **f64)
    for b in range(B):
        L = int(lengths[b])
        n = min(S, L) if counts is None else max(0, min(S, L, int(counts[b])))
        for hk in range(HK):
            k, v = tokens(pool, table[b].tolist(), hk, L)
            for h in range(hk * (H // HK), (hk + 1) * (H // HK)):
                for i in range(n):
                    see = L - n + i + 1 if causal else L
                    if see <= 0:
                        continue
                    row = q[b, i, h].double()
                    x = k[:see] @ row * scale
                    lse[b, h, i] = torch.logsumexp(x, 0)
                    p = torch.exp(x - lse[b, h, i])
                    out[b, i, h] = p @ v[:see]
                    spread[b, i, h] = p @ v[:see].abs()
                    peak[b, i, h] = (p * v[:see].abs().amax(1)).max()
                    each = k[:see].abs() @ row.abs() * scale
                    size[b, h, i] = each.max()
                    weights[b, hk, :see] += p
                    doubt[b, hk, :see] += p * size[b, h, i]
            if weights_in is not None:
                old = L - n if causal else L
                weights[b, hk, :old] += weights_in[b, hk, :old].double()
    return out, lse, weights, spread, peak, size, doubt


def evict(weights, lengths, keep, recent, first):
    """Positions that stay, [B][HK] lists."""
    B, HK, _ = weights.shape
    stay = [[] for _ in range(B)]
    for b in range(B):
        L = int(lengths[b])
        for hk in range(HK):
            if L <= keep:
                stay[b].append(list(range(L)))
                continue
            must = [t for t in range(L) if t < first or t >= L - recent]
            w = weights[b, hk].tolist()
            rank = sorted(range(first, L - recent), key=lambda t: (0 if math.isnan(w[t]) else 1, 0.0 if math.isnan(w[t]) else -w[t], t))
            stay[b].append(sorted(must + rank[:keep - len(must)]))
    return stay
