"""Performance cases of the operators around a key/value cache held in 4 bits: what a server of a language model does with it, layer by layer.

  append  `kv4_append` rounds new bf16 keys and values to MXFP4 (e2m1, one E8M0 per 32 elements of a head) into the pages of the cache;
          `kv4_read` gives back the values that the cache now holds for them
  attend  `fmha_fwd_kv4`: attention of bf16 queries over the cache, from one token per sequence to whole prompts; with `weights` the attention
          weight that every cached token received is accumulated too
  evict   `kv4_evict` keeps the first and the last tokens of a sequence and, per KV head, those with the most accumulated weight, packed into other
          pages; `kv4_read` gives back what they hold

Keys of a case: B, H, HK (sequences, query heads, KV heads), page (tokens of a page), L (tokens of the longest sequence, the new ones among them),
ragged (the sequences have lengths of their own, one of them none), S (new tokens or query rows of a sequence: the newest of its tokens; a shorter
sequence has fewer, the last rows); causal, lse, weights of attend; keep, recent, first of evict (tokens kept per head, the last and the first that
always are).

A page holds for each KV head, one behind the other: 64 bytes of K codes for each of its tokens, 64 bytes of V codes, 4 E8M0 bytes of K, 4 of V.
Byte 8 g + 2 b + r of a token's 64 holds its elements 32 b + 4 g + 2 r (low nibble) and 32 b + 4 g + 2 r + 1.
"""
import math

import torch

own = False

D, BLOCK, TOKEN = 128, 32, 136   # head size, elements of a scale, bytes of a token and KV head (K and V)
SCALE = 1.0 / math.sqrt(D)
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _append(name, B, H, HK, S, L, page=64, ragged=False):
    return {"name": name, "kind": "append", "B": B, "H": H, "HK": HK, "S": S, "L": L, "page": page, "ragged": ragged}


def _attend(name, B, H, HK, S, L, page=64, ragged=False, causal=True, lse=False, weights=False):
    return {"name": name, "kind": "attend", "B": B, "H": H, "HK": HK, "S": S, "L": L, "page": page, "ragged": ragged, "causal": causal, "lse": lse, "weights": weights}


def _evict(name, B, HK, L, keep, recent, first, page=64, ragged=False):
    return {"name": name, "kind": "evict", "B": B, "HK": HK, "L": L, "keep": keep, "recent": recent, "first": first, "page": page, "ragged": ragged}


def listed():
    return [
        # a decode step's new token of 16 sequences: the smallest append, launches and host time
        _append("append_decode_b16", 16, 32, 8, 1, 4096),
        # prompts of odd lengths of a batch go into small pages
        _append("append_prompts_s1337", 8, 32, 8, 1337, 1337, page=16, ragged=True),
        # the smallest attention call: one token of one sequence on two heads
        _attend("decode_tiny", 1, 2, 2, 1, 256),
        # a decode step of 16 sequences with 4096 tokens each that also keeps account of which tokens are looked at
        _attend("decode_weights_b16_sk4096", 16, 32, 8, 1, 4096, weights=True),
        # a decode step late in a large batch's life: the largest cache
        _attend("decode_b64_sk16384", 64, 32, 8, 1, 16384),
        # continuous batching: sequences from nothing to 32768 tokens in small pages, eight query heads to a KV head
        _attend("decode_ragged_b24", 24, 64, 8, 1, 32768, page=16, ragged=True),
        # a draft of five tokens is verified over one long context
        _attend("draft_s5_sk65536", 1, 16, 4, 5, 65536, lse=True),
        # a 512-token chunk of a long prompt against the cache of what came before
        _attend("chunk_s512_sk16384", 1, 16, 4, 512, 16384),
        # the last tokens of ragged prompts, with the weights that an eviction after the prompt goes by
        _attend("chunk_weights_s100", 4, 32, 8, 100, 4001, page=32, ragged=True, lse=True, weights=True),
        # the second half of an 8192-token prompt: the largest product
        _attend("prompt_s4096_sk8192", 1, 32, 8, 4096, 8192),
        # the caches of 16 sequences cut to a quarter
        _evict("evict_b16_sk4096", 16, 8, 4096, 1024, 128, 4),
        # long contexts of odd lengths cut to an eighth
        _evict("evict_b3_sk50001", 3, 8, 50001, 6250, 500, 16, page=128, ragged=True),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """A case of the same ranges: 1 to 64 sequences, 1 to 8 KV heads with 1 to 16 query heads each, 1 to 65536 cached tokens, 1 to 4096 new ones, any
    page size and option; no more work than the largest listed cases."""
    while True:
        kind = rng.choice(["append", "attend", "attend", "attend", "evict"])
        B, HK, g = _log_uniform(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 16])
        L, page, ragged = _log_uniform(rng, 16, 65536), rng.choice([16, 32, 64, 128]), rng.random() < 0.5
        if rng.random() < 0.3:    # round lengths are common too
            L = -(-L // 64) * 64
        if B * L * HK > 64 * 16384 * 8:
            continue
        if kind == "evict":
            if L < 64 or B * HK * L > 16 * 8 * 8192:
                continue
            keep = _log_uniform(rng, 16, L)
            recent = rng.randint(0, keep)
            return _case(_evict("", B, HK, L, keep, recent, rng.randint(0, min(16, keep - recent)), page, ragged))
        if kind == "append":
            S = min(L, rng.choice([1, _log_uniform(rng, 1, 4096)]))
            if B * S * HK <= 8 * 4096 * 8:
                return _case(_append("", B, HK * g, HK, S, L, page, ragged))
            continue
        use = rng.choice(["decode", "decode", "draft", "chunk"])
        S = min(L, 1 if use == "decode" else rng.randint(2, 8) if use == "draft" else _log_uniform(rng, 9, 4096))
        case = _attend("", B, HK * g, HK, S, L, page, ragged, rng.random() < 0.8, rng.random() < 0.4, rng.random() < 0.3)
        if B * HK * g * S * L <= 32 * 4096 * 8192:
            return _case(case)


def _case(case):
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths: all L, or spread over the logarithm below it in an order of no meaning, the second one empty."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    spread = [max(1, int(round(L ** (1.0 - 0.4 * ((b * 0.6180339887498949) % 1.0))))) for b in range(B)]
    return [0 if b == 1 else n for b, n in enumerate(spread)]


def _new(case):
    """New tokens of each sequence."""
    return [min(case["S"], n) for n in _lengths(case)]


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------------------------------------- the format, in torch
def _order(device):
    """Element of a head that each nibble of a token's 64 bytes holds."""
    n = torch.arange(D, device=device)
    g, b, r, low = n // 16, n // 4 % 4, n // 2 % 2, n % 2
    return 32 * b + 4 * g + 2 * r + low


def _power(e):
    """2^e in f32 for -127 < e < 128, by its bits: the exponential's last bit would decide ties."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _round(x):
    """bf16 [..., 128] to 64 code bytes and 4 scale bytes: E8M0 = floor(log2 of the block's largest) - 2, codes rounded to nearest, ties to even."""
    x = x.float().unflatten(-1, (4, BLOCK))
    e = (torch.frexp(x.abs().amax(-1)).exponent - 1 - 2 + 127).clamp(1, 252)
    y = x * _power(127 - e).unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)) | (torch.signbit(y).to(torch.uint8) << 3)
    code = code.flatten(-2)[..., _order(x.device)]
    return code[..., 0::2] | (code[..., 1::2] << 4), e.to(torch.uint8)


def _values(codes, scales):
    """Code bytes [..., 64] and scale bytes [..., 4] to the f32 values [..., 128] they stand for."""
    one = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    two = torch.stack([one.repeat(16), one.repeat_interleave(16)], dim=-1)
    v = two[codes.int()].unflatten(-2, (8, 4, 2)).transpose(-4, -3).flatten(-3)                # [..., 4 blocks, 32]
    return (v * _power(scales.int() - 127).unsqueeze(-1)).flatten(-2)


def _parts(pool, page):
    """Views of a pool [pages, HK, 136 page]: codes [pages, HK, page, 64] and scales [pages, HK, page, 4], of K and of V."""
    k, v = pool[..., :64 * page].unflatten(-1, (page, 64)), pool[..., 64 * page:128 * page].unflatten(-1, (page, 64))
    ks, vs = pool[..., 128 * page:132 * page].unflatten(-1, (page, 4)), pool[..., 132 * page:].unflatten(-1, (page, 4))
    return (k, ks), (v, vs)


def _cached(part, table):
    """f32 [B, HK, table width x page, 128] of one part of a pool."""
    codes, scales = (x[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3) for x in part)
    return _values(codes, scales)


def _store(part, table, page, at, live, x):
    """Rounds x bf16 [B, T, HK, 128] to tokens at [B, T] of the sequences where live; gives the values that are then held, 0 elsewhere."""
    codes, scales = _round(x)
    b, t = live.nonzero(as_tuple=True)
    p = at[b, t]
    where = (table[b, p // page].long(), slice(None), p % page)
    part[0][where], part[1][where] = codes[b, t], scales[b, t]
    return (_values(codes, scales) * live[..., None, None]).bfloat16()


# ------------------------------------------------------------------------------------------------- inputs
def _activations(g, shape, spread):
    """bf16 normal samples whose 128 channels differ in size, as the keys' of a trained model do; rows are made a slice at a time."""
    gain = torch.exp2(torch.randn(shape[-1], generator=g, device="cuda") * spread)
    x = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    for i in range(shape[0]):
        x[i] = torch.randn(shape[1:], generator=g, device="cuda") * gain
    return x


def _table(g, lengths, page, from_page):
    """A page table over pages in a shuffled order, -1 where a sequence has none."""
    counts = [_pages(n, page) for n in lengths]
    width, total = max(1, max(counts)), sum(counts)
    mine = torch.arange(width, device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    table[mine] = (torch.randperm(total, generator=g, device="cuda") + from_page).int()
    return table, total


def prepare(case, seed):
    B, HK, page, lengths = case["B"], case["HK"], case["page"], _lengths(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    table, pages = _table(g, lengths, page, 0)
    kept = [min(case["keep"], n) for n in lengths] if case["kind"] == "evict" else []
    into, more = _table(g, kept, page, pages) if kept else (None, 0)
    s = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "pool": torch.zeros((max(1, pages + more), HK, TOKEN * page), dtype=torch.uint8, device="cuda")}
    if case["kind"] != "evict" and case["ragged"]:
        s["counts"] = torch.tensor(_new(case), dtype=torch.int32, device="cuda")
    else:
        s["counts"] = None
    if case["kind"] != "append":   # what the cache holds: whole pages, a few million elements at a time
        step = max(1, (1 << 22) // (HK * page * D))
        for i, (codes, scales) in enumerate(_parts(s["pool"], page)):
            gain = torch.exp2(torch.randn(HK, 1, D, generator=g, device="cuda") * (0.7 if i == 0 else 0.2))
            for p in range(0, pages, step):
                n = min(step, pages - p)
                codes[p:p + n], scales[p:p + n] = _round((torch.randn((n, HK, page, D), generator=g, device="cuda") * gain).bfloat16())
    if case["kind"] == "append":
        # K and V as a projection leaves them, between the queries and the end of a token's row
        qkv = _activations(g, (B, case["S"], (case["H"] + 2 * HK) * D), 0.5).view(B, case["S"], case["H"] + 2 * HK, D)
        s["k"], s["v"] = qkv[:, :, case["H"]:case["H"] + HK], qkv[:, :, case["H"] + HK:]
        s["k_held"], s["v_held"] = (torch.empty((B, case["S"], HK, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    elif case["kind"] == "attend":
        H, S = case["H"], case["S"]
        # rows from flat to peaked, as the heads of a trained model are
        gain = torch.exp2(torch.rand(H, 1, generator=g, device="cuda") * 2.6 - 1.0)
        s["q"] = (torch.randn((B, S, H, D), generator=g, device="cuda") * gain).bfloat16()
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((B, H, S), device="cuda") if case["lse"] else None
        s["weights_in"] = s["weights"] = None
        if case["weights"]:
            s["weights_in"] = torch.rand((B, HK, table.shape[1] * page), generator=g, device="cuda")
            s["weights"] = torch.zeros_like(s["weights_in"])
    else:
        # accumulated weights have a long tail, and tokens that nothing looked at have none
        w = torch.exp2(torch.randn((B, HK, table.shape[1] * page), generator=g, device="cuda") * 3.0)
        s["weights"] = w * (torch.rand(w.shape, generator=g, device="cuda") > 0.1)
        s["into_table"], s["into_lengths"] = into, torch.zeros(B, dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty((B, HK, case["keep"]), dtype=torch.int32, device="cuda")
        s["weights_out"] = torch.zeros((B, HK, into.shape[1] * page), device="cuda")
        s["k_held"], s["v_held"] = (torch.empty((B, case["keep"], HK, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if own:
        from amdgpu_rustdsl_b200 import Kv4Cache
        s["cache"] = Kv4Cache(s["pool"], s["table"], s["lengths"])
        if into is not None:
            s["into"] = Kv4Cache(s["pool"], into, s["into_lengths"])
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["kind"]](s)


def _own_append(s):
    from amdgpu_rustdsl_b200 import kv4_append, kv4_read
    kv4_append(s["cache"], s["k"], s["v"], counts=s["counts"])
    kv4_read(s["cache"], s["k_held"], s["v_held"], last=True, counts=s["counts"])
    return {"k": s["k_held"], "v": s["v_held"]}


def _own_attend(s):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv4
    fmha_fwd_kv4(s["q"], s["cache"], s["out"], causal=s["case"]["causal"], counts=s["counts"], lse=s["lse"], weights=s["weights"], weights_in=s["weights_in"])
    return {"out": s["out"], "lse": s["lse"], "weights": s["weights"]}


def _own_evict(s):
    from amdgpu_rustdsl_b200 import kv4_evict, kv4_read
    case = s["case"]
    kv4_evict(s["cache"], s["weights"], s["into"], keep=case["keep"], recent=case["recent"], first=case["first"], kept=s["kept"], weights_out=s["weights_out"])
    kv4_read(s["into"], s["k_held"], s["v_held"])
    return {"kept": s["kept"], "lengths": s["into_lengths"], "weights": s["weights_out"], "k": s["k_held"], "v": s["v_held"]}


def _rows(s):
    """Position of each of the S rows in its sequence [B, S] and whether the sequence has that row: the new tokens are the last ones."""
    S, lengths = s["case"]["S"], s["lengths"][:, None]
    counts = lengths.clamp(max=S) if s["counts"] is None else s["counts"][:, None]
    row = torch.arange(S, device=lengths.device)[None, :]
    return lengths - counts + row, row < counts


def _plain_append(s):
    at, live = _rows(s)
    k, v = _parts(s["pool"], s["case"]["page"])
    return {"k": _store(k, s["table"], s["case"]["page"], at, live, s["k"]), "v": _store(v, s["table"], s["case"]["page"], at, live, s["v"])}


def _plain_attend(s):
    case = s["case"]
    B, H, HK, S, page = (case[x] for x in ("B", "H", "HK", "S", "page"))
    at, live = _rows(s)
    part_k, part_v = _parts(s["pool"], page)
    k = _cached(part_k, s["table"])
    T = k.shape[2]
    q = s["q"].float().view(B, S, HK, H // HK, D).permute(0, 2, 3, 1, 4).flatten(2, 3)           # [B, HK, heads x rows, D]
    x = (q @ k.transpose(-1, -2)).mul_(SCALE).view(B, HK, H // HK, S, T)
    del k
    t = torch.arange(T, device=x.device)
    seen = (t < s["lengths"][:, None])[:, None, :] & live[..., None]                             # [B, S, T]
    if case["causal"]:
        seen = seen & (t <= at[..., None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total == 0, 1.0, total))
    out = x.flatten(2, 3) @ _cached(part_v, s["table"])
    out = out.view(B, HK, H // HK, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, H, D).bfloat16()
    lse = (top + total.log()).view(B, H, S) if case["lse"] else None
    weights = None
    if case["weights"]:
        # new tokens (where the rows are the new tokens) bring no weight along
        fresh = s["lengths"] - live.sum(-1) if case["causal"] else s["lengths"]
        before = torch.where(t < fresh[:, None, None], s["weights_in"], 0.0)
        weights = torch.where(t < s["lengths"][:, None, None], before + x.sum((2, 3)), 0.0)
    return {"out": out, "lse": lse, "weights": weights}


def _plain_evict(s):
    case = s["case"]
    B, HK, page, keep = (case[x] for x in ("B", "HK", "page", "keep"))
    w, lengths = s["weights"], s["lengths"][:, None, None]
    t = torch.arange(w.shape[-1], device=w.device)
    w_or = torch.where((t < case["first"]) | (t >= lengths - case["recent"]), math.inf, w)
    order = torch.where(t < lengths, w_or, -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=w.shape[-1])
    kept = torch.where(order < lengths, order, 1 << 30).sort(dim=-1).values                      # [B, HK, keep]
    live = kept < (1 << 30)
    b, h, j = live.nonzero(as_tuple=True)
    src, dst = kept[b, h, j], j
    held = []
    for codes, scales in _parts(s["pool"], page):
        where = (s["table"][b, src // page].long(), h, src % page)
        to = (s["into_table"][b, dst // page].long(), h, dst % page)
        codes[to], scales[to] = codes[where], scales[where]
        x = torch.zeros((B, keep, HK, D), dtype=torch.bfloat16, device=w.device)
        x[b, j, h] = _values(codes[to], scales[to]).bfloat16()
        held.append(x)
    weights = torch.zeros_like(s["weights_out"])
    weights[b, h, j] = w[b, h, src]
    return {"kept": torch.where(live, kept, -1).int(), "lengths": s["lengths"].clamp(max=keep), "weights": weights, "k": held[0], "v": held[1]}


_run_own = {"append": _own_append, "attend": _own_attend, "evict": _own_evict}
_run_plain = {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    HK, lengths, new = case["HK"], _lengths(case), _new(case) if case["kind"] != "evict" else []
    tokens, pages = sum(lengths), sum(_pages(n, case["page"]) for n in lengths)
    if case["kind"] == "append":
        # bf16 in, codes and scales out, the values that are held out in bf16
        rows = case["B"] * case["S"] * HK
        return {"bytes": sum(new) * HK * (4 * D + TOKEN) + rows * 4 * D + 4 * len(lengths), "flops": 6 * sum(new) * HK * D}
    if case["kind"] == "evict":
        kept = sum(min(case["keep"], n) for n in lengths)
        moved = kept * HK * (2 * TOKEN + 4 + 4) + case["B"] * case["keep"] * HK * (4 * D + 4)
        return {"bytes": tokens * HK * 4 + moved + 4 * pages, "flops": 2 * tokens * HK}
    H, rows = case["H"], case["B"] * case["S"] * case["H"]
    n_bytes = tokens * HK * TOKEN + 4 * pages + rows * 4 * D + (rows * 4 if case["lse"] else 0) + (8 * tokens * HK if case["weights"] else 0)
    pairs = sum(n * (L - n) + n * (n + 1) // 2 if case["causal"] else n * L for n, L in zip(new, lengths))
    return {"bytes": n_bytes, "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------------- from the definition, in 64 bits
def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(codes, scales):
    """Values of code bytes [n, 64] and scale bytes [n, 4] in 64 bits, from the format's definition: sign, two exponent bits, one mantissa bit."""
    nibble = torch.stack([codes % 16, codes // 16], dim=-1).reshape(codes.shape[0], D).to(torch.int64)
    exponent, mantissa = nibble // 2 % 4, nibble % 2
    size = torch.where(exponent == 0, mantissa * 0.5, (1.0 + 0.5 * mantissa.double()) * torch.pow(2.0, exponent.double() - 1.0))
    value = torch.empty(codes.shape[0], D, dtype=torch.float64, device=codes.device)
    value[:, _order(codes.device)] = torch.where(nibble >= 8, -size, size).double()
    return value * _power64(scales.long() - 127).repeat_interleave(BLOCK, dim=1)


def _encode64(x):
    """The values [n, 128] that rows [n, 128] are rounded to, in 64 bits."""
    out = torch.zeros_like(x)
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    even = torch.arange(8, device=x.device) % 2 == 0
    for b in range(0, D, BLOCK):
        y = x[:, b:b + BLOCK]
        top = y.abs().amax(1, keepdim=True)
        scale = _power64(torch.where(top > 0, torch.frexp(top).exponent - 3, 0))
        far = ((y / scale).abs().clamp(max=6.0)[..., None] - grid).abs()
        near = far == far.amin(-1, keepdim=True)
        pick = torch.where((near & even).any(-1), (near & even).int().argmax(-1), near.int().argmax(-1))
        out[:, b:b + BLOCK] = torch.sign(y) * grid[pick] * scale
    return out


def _tokens64(pool, part, page, table_row, head, tokens):
    """Values [n, 128] in 64 bits of the given tokens of one sequence and head; part 0: K, 1: V."""
    record = pool[table_row[tokens // page].long(), head]
    lane = torch.arange(64, device=pool.device)
    codes = torch.gather(record, 1, (part * 64 * page + 64 * (tokens % page))[:, None] + lane)
    scales = torch.gather(record, 1, ((128 + 4 * part) * page + 4 * (tokens % page))[:, None] + lane[:4])
    return _decode64(codes, scales)


def exact(case, seed):
    s = prepare(case, seed)
    lengths, HK, page = _lengths(case), case["HK"], case["page"]
    if case["kind"] == "append":
        new, held = _new(case), {}
        for name in ("k", "v"):
            held[name] = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
            for b, n in enumerate(new):
                held[name][b, :n] = _encode64(s[name][b, :n].double().reshape(-1, D)).view(n, HK, D)
        return held
    if case["kind"] == "evict":
        out = {name: torch.zeros(s[name + "_held"].shape, dtype=torch.float64, device="cuda") for name in ("k", "v")}
        out["weights"] = torch.zeros(s["weights_out"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            for h in range(HK):
                some = min(n, case["keep"])
                must = [t for t in range(n) if t < case["first"] or t >= n - case["recent"]] if n > some else list(range(n))
                weight = s["weights"][b, h, :n].double().cpu()
                if n > some:
                    rest = torch.arange(case["first"], n - case["recent"])
                    more = rest[torch.argsort(-weight[rest], stable=True)[:some - len(must)]]
                    must = sorted(must + more.tolist())
                at = torch.tensor(must, dtype=torch.int64, device="cuda")
                out["weights"][b, h, :some] = weight.cuda()[at]
                for part, name in enumerate(("k", "v")):
                    out[name][b, :some, h] = _tokens64(s["pool"], part, page, s["table"][b], h, at)
        return {"kept": None, "lengths": None, **out}
    H, S, new = case["H"], case["S"], _new(case)
    group = H // HK
    out = torch.zeros((case["B"], S, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((case["B"], H, S), -math.inf, dtype=torch.float64, device="cuda")
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda") if case["weights"] else None
    for b, (n, L) in enumerate(zip(new, lengths)):
        if not L:
            continue
        tokens = torch.arange(L, device="cuda")
        hidden = tokens[None, :] > (L - n + torch.arange(n, device="cuda"))[:, None] if case["causal"] else None
        for h in range(HK):
            k, v = (_tokens64(s["pool"], part, page, s["table"][b], h, tokens) for part in (0, 1))
            mass = torch.zeros(L, dtype=torch.float64, device="cuda")
            for head in range(h * group, (h + 1) * group):
                x = (s["q"][b, :n, head].double() @ k.T) / math.sqrt(D)
                if hidden is not None:
                    x.masked_fill_(hidden, -math.inf)
                lse[b, head, :n] = torch.logsumexp(x, 1)
                p = torch.exp(x - lse[b, head, :n][:, None])
                out[b, :n, head] = p @ v
                mass += p.sum(0)
            if weights is not None:
                old = L - n if case["causal"] else L
                mass[:old] += s["weights_in"][b, h, :old].double()
                weights[b, h, :L] = mass
    return {"out": out, "lse": lse if case["lse"] else None, "weights": weights}
