"""Performance cases of the operators around a paged key/value cache held in 8 bits: what a server of a language model does for every new token, layer by layer.

  rope    `rope_rotate` turns queries and keys by their positions (pairs of halves or neighbours, all of a head or its first part, frequencies scaled for
          long contexts); backward: the gradient of that
  pages   `pages_take` hands pages of a stack of free ones to the sequences that need them for their new tokens, raises the lengths and gives positions and a
          slot map; `pages_cut` takes the tokens back (a draft that was not accepted, a batch that is put off), so that a pass ends as it began
  append  `kv8_append` rounds new bf16 keys and values to e4m3 with one power of two for a block of 16 tokens of a head, into the pages of the cache;
          `kv8_read` gives back the values that the cache now holds for them
  attend  `fmha_fwd_kv8`: attention of bf16 queries over that cache, from one token per sequence to whole prompts

Keys of a case: B, H, HK (sequences, query heads, KV heads), S (new tokens or rows of a sequence), page (tokens of a page), L (tokens of the longest
sequence, the new ones among them; of pages: without them), ragged (the sequences have lengths of their own, one of them none; of pages and append: new tokens
of their own number too). rope: D, rotary (elements of a head, of its rotated part), type, interleaved, scaling, backward, far (positions lie below it).
pages: spare (free pages, as a part of what is asked for). attend: causal, lse.

A block of 16 tokens and a head is 4112 bytes: 2048 of K codes, 2048 of V codes, the two scales in f32, a word with a bit for each token whose K (lower half) or V
holds no numbers, and a word that is not used. K's byte of token t and element d lies at 128 t + 16 ((d / 16) ^ (t % 8)) + d % 16. V's tokens lie in pairs j = t / 2:
256 j + 16 ((d / 8) ^ s) + 2 (d % 8) + t % 2, with s = j % 2 + 4 (j / 2 % 2). A page has one such block behind the other for each KV head, head after head.
"""
import math

import torch

own = False

D, BLOCK, RECORD = 128, 16, 4112   # head size, tokens of a scale, bytes of a block
SCALE = 1.0 / math.sqrt(D)
LARGEST = 448.0                    # of e4m3
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# scalings for contexts longer than the one trained on: (kind, factor, original context)
BASE = 10000.0


def _rope(name, B, S, H, HK, head, rotary, type, interleaved=False, scaling="none", backward=False, far=32768):
    return {"name": name, "kind": "rope", "B": B, "S": S, "H": H, "HK": HK, "D": head, "rotary": rotary, "type": type, "interleaved": interleaved, "scaling": scaling,
            "backward": backward, "far": far}


def _pages_case(name, B, S, L, page, ragged, spare):
    return {"name": name, "kind": "pages", "B": B, "S": S, "L": L, "page": page, "ragged": ragged, "spare": spare}


def _append(name, B, H, HK, S, L, page=64, ragged=False):
    return {"name": name, "kind": "append", "B": B, "H": H, "HK": HK, "S": S, "L": L, "page": page, "ragged": ragged}


def _attend(name, B, H, HK, S, L, page=64, ragged=False, causal=True, lse=False):
    return {"name": name, "kind": "attend", "B": B, "H": H, "HK": HK, "S": S, "L": L, "page": page, "ragged": ragged, "causal": causal, "lse": lse}


def listed():
    return [
        # a decode step's new token of 64 sequences: launches and host time
        _rope("rope_decode_b64", 64, 1, 32, 8, 128, 128, "bf16"),
        # prompts of a batch, queries and keys as slices of one projection, context four times the trained one
        _rope("rope_prompt_b4_s4096", 4, 4096, 32, 8, 128, 128, "bf16", scaling="yarn", far=16384),
        # the gradient in a training step in 32 bits: neighbours as pairs, part of a head of 96
        _rope("rope_backward_part_s1337", 3, 1337, 20, 4, 96, 40, "f32", interleaved=True, scaling="linear", backward=True, far=8192),
        # a decode step of 256 sequences: one token each, now and then a new page
        _pages_case("pages_decode_b256", 256, 1, 8192, 16, True, 1.5),
        # prompts of a batch are let in, as far as the free pages go
        _pages_case("pages_prompts_b64_s2048", 64, 2048, 4096, 16, True, 0.8),
        # a decode step's new token of 64 sequences goes into blocks that have tokens already
        _append("append_decode_b64", 64, 32, 8, 1, 4090),
        # chunks of prompts of odd lengths go into small pages behind what is there
        _append("append_prompts_s1337", 8, 32, 8, 1337, 2001, page=16, ragged=True),
        # the smallest attention call: one token of one sequence on two heads
        _attend("decode_tiny", 1, 2, 2, 1, 256),
        # a decode step late in a large batch's life: the largest cache
        _attend("decode_b64_sk16384", 64, 32, 8, 1, 16384),
        # drafts of five tokens are verified, sequences from nothing to 32768 tokens in small pages
        _attend("draft_ragged_b24_s5", 24, 16, 4, 5, 32768, page=16, ragged=True, lse=True),
        # the last tokens of ragged prompts, three query heads to a KV head
        _attend("chunk_ragged_s333", 4, 24, 8, 333, 4001, page=32, ragged=True, lse=True),
        # the second half of an 8192-token prompt: the largest product
        _attend("prompt_s4096_sk8192", 1, 32, 8, 4096, 8192),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    """A case of the same ranges: 1 to 64 sequences (512 of pages), 1 to 8 KV heads with 1 to 16 query heads each, 1 to 65536 cached tokens, 1 to 4096 new ones, any page
    size and option, heads of up to 256 elements for rope; no more work than the largest listed cases."""
    while True:
        kind = rng.choice(["rope", "pages", "append", "attend", "attend"])
        B, HK, g = _log_uniform(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 16])
        L, page, ragged = _log_uniform(rng, 16, 65536), rng.choice([16, 32, 64, 128]), rng.random() < 0.5
        if rng.random() < 0.3:    # round lengths are common too
            L = -(-L // 64) * 64
        S = rng.choice([1, _log_uniform(rng, 1, 4096)])
        if kind == "rope":
            head = 2 * rng.randint(8, 128) if rng.random() < 0.4 else rng.choice([64, 96, 128, 128, 128, 192, 256])
            rotary = head if rng.random() < 0.5 else 2 * rng.randint(1, head // 2)
            type = rng.choice(["bf16", "bf16", "f16", "f32"])
            if B * S * (g + 1) * HK * head * (2 if type == "f32" else 1) <= 4 * 4096 * 40 * 128:
                return _case(_rope("", B, S, g * HK, HK, head, rotary, type, rng.random() < 0.4, rng.choice(["none", "none", "linear", "ntk", "yarn", "bands"]), rng.random() < 0.3,
                                   _log_uniform(rng, 1024, 1 << 20)))
            continue
        if kind == "pages":
            B = _log_uniform(rng, 1, 512)
            if B * S <= 256 * 2048 and B * L <= 256 * 8192:
                return _case(_pages_case("", B, S, L, page, ragged, rng.choice([0.0, 0.5, 0.8, 1.0, 1.5])))
            continue
        if B * L * HK > 64 * 16384 * 8:
            continue
        if kind == "append":
            S = min(L, S)
            if B * S * HK <= 8 * 4096 * 8:
                return _case(_append("", B, HK * g, HK, S, L, page, ragged))
            continue
        use = rng.choice(["decode", "decode", "draft", "chunk"])
        S = min(L, 1 if use == "decode" else rng.randint(2, 8) if use == "draft" else _log_uniform(rng, 9, 4096))
        if B * HK * g * S * L <= 32 * 4096 * 8192:
            return _case(_attend("", B, HK * g, HK, S, L, page, ragged, rng.random() < 0.8, rng.random() < 0.4))


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
    """New tokens of each sequence: of append and attend no more than there are, of pages of their own number too."""
    S, lengths = case["S"], _lengths(case)
    if case["kind"] == "pages":
        return [S - (b * 7919) % S if case["ragged"] else S for b in range(case["B"])]
    if case["kind"] == "append" and case["ragged"]:
        return [min(S - (b * 7919) % S, n) for b, n in enumerate(lengths)]
    return [min(S, n) for n in lengths]


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------------------------------------- rope: frequencies
def _frequencies(case):
    """Radians per position of each pair, in 64 bits, and what the results are multiplied by."""
    n, kind = case["rotary"] // 2, case["scaling"]
    i = torch.arange(n, dtype=torch.float64)
    f = BASE ** (-i / n)
    if kind == "linear":      # positions are divided
        return f / 2.5, 1.0
    if kind == "ntk":         # the base grows, so that the slowest pair turns as if positions were divided (one pair alone turns as it did)
        return (BASE * 4.0 ** (n / (n - 1.0))) ** (-i / n) if n > 1 else f, 1.0
    if kind == "yarn":        # fast pairs stay, slow ones are divided, a ramp between those that turn 32 times and once in the original context
        at = [2 * n * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), 2 * n - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        return f / 4.0 * ramp + f * (1.0 - ramp), 0.1 * math.log(4.0) + 1.0
    if kind == "bands":       # by wavelength: below an original context / 4 as they are, above the context divided by 8, blended between
        smooth = ((8192 * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return (1.0 - smooth) * f / 8.0 + smooth * f, 1.0
    return f, 1.0


def _scaling(case):
    """The same as the framework's option."""
    return {"none": None, "linear": {"kind": "linear", "factor": 2.5}, "ntk": {"kind": "ntk", "factor": 4.0}, "yarn": {"kind": "yarn", "factor": 4.0, "original": 4096},
            "bands": {"kind": "bands", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}[case["scaling"]]


# ------------------------------------------------------------------------------------------------- the cache's format, in torch
def _places(device):
    """Byte of a block's K part and of its V part for each token and element: int64 [16, 128] each."""
    t, d = torch.arange(BLOCK, device=device)[:, None], torch.arange(D, device=device)[None, :]
    j = t // 2
    return 128 * t + 16 * ((d // 16) ^ (t % 8)) + d % 16, 256 * j + 16 * ((d // 8) ^ (j % 2 + 4 * (j // 2 % 2))) + 2 * (d % 8) + t % 2


def _blocks(pool, page):
    """A pool [pages, HK, 257 page] as blocks: K codes and V codes [pages, HK, page / 16, 2048] and scales f32 [pages, HK, page / 16, 2] (views)."""
    r = pool.view(*pool.shape[:2], page // BLOCK, RECORD)
    return r[..., :2048], r[..., 2048:4096], r[..., 4096:4104].view(torch.float32)


def _scale_of(largest):
    """The smallest power of two that brings `largest` to 448 or less, from 2^-90 to 2^119."""
    mantissa, exponent = torch.frexp(largest)
    e = torch.where(largest == 0, -90, exponent - 9 + (mantissa > LARGEST / 512).int())
    return torch.ldexp(torch.ones_like(largest), e.clamp(-90, 119).int())


def _round(x, scale):
    """f32 to e4m3 codes as bytes, nearest, ties to even."""
    return (x / scale).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn).view(torch.uint8)


def _value(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _cached(codes, scales, places, table):
    """f32 [B, HK, table width x page, 128] of one part of a pool."""
    at = table.clamp(min=0).long()
    v = _value(codes[at][..., places.flatten()]).unflatten(-1, (BLOCK, D)) * scales[at][..., None, None]     # [B, width, HK, blocks, 16, 128]
    return v.transpose(1, 2).flatten(2, 4)


# ------------------------------------------------------------------------------------------------- inputs
def _activations(g, shape, spread, dtype=torch.bfloat16):
    """Normal samples whose channels differ in size, as the keys' of a trained model do; rows are made a slice at a time."""
    gain = torch.exp2(torch.randn(shape[-1], generator=g, device="cuda") * spread)
    x = torch.empty(shape, dtype=dtype, device="cuda")
    for i in range(shape[0]):
        x[i] = torch.randn(shape[1:], generator=g, device="cuda") * gain
    return x


def _table(g, counts, width):
    """A page table over pages in a shuffled order, -1 where a sequence has none."""
    total = sum(counts)
    mine = torch.arange(width, device="cuda")[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[mine] = torch.randperm(total, generator=g, device="cuda").int()
    return table, total


def _prepare_rope(case, g):
    B, S, H, HK, head, dtype = case["B"], case["S"], case["H"], case["HK"], case["D"], TYPES[case["type"]]
    # queries and keys as a projection leaves them, values behind
    qkv = _activations(g, (B, S, (H + 2 * HK) * head), 0.5, dtype).view(B, S, H + 2 * HK, head)
    start = torch.randint(0, max(1, case["far"] - S), (B, 1), generator=g, device="cuda")
    s = {"case": case, "q": qkv[:, :, :H], "k": qkv[:, :, H:H + HK], "positions": (start + torch.arange(S, device="cuda")).int(),
         "q_out": torch.empty((B, S, H, head), dtype=dtype, device="cuda"), "k_out": torch.empty((B, S, HK, head), dtype=dtype, device="cuda")}
    if own:
        from amdgpu_rustdsl_b200 import Rope
        s["rope"] = Rope(case["rotary"], base=BASE, interleaved=case["interleaved"], scaling=_scaling(case), device="cuda")
    else:
        f, s["factor"] = _frequencies(case)
        s["frequencies"] = f.cuda()
    return s


def _prepare_pages(case, g):
    B, S, page, lengths = case["B"], case["S"], case["page"], _lengths(case)
    width = _pages(case["L"] + S, page)
    table, used = _table(g, [_pages(n, page) for n in lengths], width)
    asked = sum(_pages(n + m, page) - _pages(n, page) for n, m in zip(lengths, _new(case)))
    free = int(case["spare"] * asked)
    pool = torch.zeros(4 + used + max(1, free), dtype=torch.int32, device="cuda")
    pool[0] = free
    pool[4:4 + free] = used + torch.randperm(free, generator=g, device="cuda").int()
    s = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "counts": torch.tensor(_new(case), dtype=torch.int32, device="cuda"),
         "free": pool, "granted": torch.empty(B, dtype=torch.int32, device="cuda"), "starts": torch.empty(B + 1, dtype=torch.int32, device="cuda"),
         "positions": torch.empty((B, S), dtype=torch.int32, device="cuda"), "slots": torch.empty((B, S), dtype=torch.int64, device="cuda")}
    s["keep"] = s["lengths"].clone()
    if own:
        from amdgpu_rustdsl_b200 import Kv8Cache
        # (the cache's own memory is not looked at: one KV head, as small as it can be)
        s["cache"] = Kv8Cache(torch.zeros((used + max(1, free), 1, 257 * page), dtype=torch.uint8, device="cuda"), table, s["lengths"])
        s["positions"] = torch.empty_like(s["slots"])   # (64 bits, which the plain form's sums come out in)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["kind"] == "rope":
        return _prepare_rope(case, g)
    if case["kind"] == "pages":
        return _prepare_pages(case, g)
    B, HK, page, lengths = case["B"], case["HK"], case["page"], _lengths(case)
    counts = [_pages(n, page) for n in lengths]
    table, pages = _table(g, counts, max(1, max(counts)))
    s = {"case": case, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "pool": torch.zeros((max(1, pages), HK, 257 * page), dtype=torch.uint8, device="cuda"),
         "counts": torch.tensor(_new(case), dtype=torch.int32, device="cuda") if case["ragged"] else None, "places": _places("cuda")}
    # what the cache holds: whole pages, a few million elements at a time
    step = max(1, (1 << 22) // (HK * page * D))
    k_codes, v_codes, scales = _blocks(s["pool"], page)
    for i, codes in enumerate((k_codes, v_codes)):
        gain = torch.exp2(torch.randn(HK, 1, 1, D, generator=g, device="cuda") * (0.7 if i == 0 else 0.2))
        back = torch.argsort(s["places"][i].flatten())
        for p in range(0, pages, step):
            n = min(step, pages - p)
            x = torch.randn((n, HK, page // BLOCK, BLOCK, D), generator=g, device="cuda") * gain
            scale = _scale_of(x.abs().amax((-1, -2)))
            scales[p:p + n, ..., i] = scale
            codes[p:p + n] = _round(x, scale[..., None, None]).flatten(-2)[..., back]
    if case["kind"] == "append":
        # K and V as a projection leaves them, between the queries and the end of a token's row
        qkv = _activations(g, (B, case["S"], (case["H"] + 2 * HK) * D), 0.5).view(B, case["S"], case["H"] + 2 * HK, D)
        s["k"], s["v"] = qkv[:, :, case["H"]:case["H"] + HK], qkv[:, :, case["H"] + HK:]
        s["k_held"], s["v_held"] = (torch.empty((B, case["S"], HK, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    else:
        H, S = case["H"], case["S"]
        # rows from flat to peaked, as the heads of a trained model are
        gain = torch.exp2(torch.rand(H, 1, generator=g, device="cuda") * 2.6 - 1.0)
        s["q"] = (torch.randn((B, S, H, D), generator=g, device="cuda") * gain).bfloat16()
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((B, H, S), device="cuda") if case["lse"] else None
    if own:
        from amdgpu_rustdsl_b200 import Kv8Cache
        s["cache"] = Kv8Cache(s["pool"], s["table"], s["lengths"])
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["kind"]](s)


def _own_rope(s):
    from amdgpu_rustdsl_b200 import rope_rotate
    rope_rotate(s["rope"], s["q"], s["positions"], s["q_out"], y=s["k"], y_out=s["k_out"], backward=s["case"]["backward"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_pages(s):
    from amdgpu_rustdsl_b200 import pages_cut, pages_take
    pages_take(s["free"], s["cache"], s["counts"], s["granted"], positions=s["positions"], slots=s["slots"], starts=s["starts"])
    pages_cut(s["free"], s["cache"], s["keep"])
    return {name: s[name] for name in ("granted", "starts", "positions", "slots", "lengths", "table", "free")}


def _own_append(s):
    from amdgpu_rustdsl_b200 import kv8_append, kv8_read
    kv8_append(s["cache"], s["k"], s["v"], counts=s["counts"])
    kv8_read(s["cache"], s["k_held"], s["v_held"], last=True, counts=s["counts"])
    return {"k": s["k_held"], "v": s["v_held"]}


def _own_attend(s):
    from amdgpu_rustdsl_b200 import fmha_fwd_kv8
    fmha_fwd_kv8(s["q"], s["cache"], s["out"], causal=s["case"]["causal"], counts=s["counts"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_rope(s):
    case = s["case"]
    n = case["rotary"] // 2
    # angles of far positions need 64 bits; what they multiply does not
    angle = s["positions"].double()[..., None] * s["frequencies"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, :, None] for f in (torch.cos, torch.sin))
    if case["backward"]:
        sin = -sin
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        part = x[..., :2 * n]
        a, b = (part[..., 0::2], part[..., 1::2]) if case["interleaved"] else (part[..., :n], part[..., n:])
        a, b = a * cos - b * sin, a * sin + b * cos
        part = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
        out[name] = torch.cat([part, x[..., 2 * n:]], -1).to(s[name].dtype)
    return out


def _plain_pages(s):
    page, S = s["case"]["page"], s["case"]["S"]
    free, table, lengths, counts = s["free"], s["table"], s["lengths"].clone(), s["counts"]
    width, n_free = table.shape[1], s["free"][0].long()
    had, fits = (lengths.long() + page - 1) // page, lengths.long() + counts <= width * page
    need = torch.where(fits, (lengths.long() + counts + page - 1) // page - had, 0)
    upto = need.cumsum(0)
    ok = fits & ((upto <= n_free) | (need == 0))
    granted = torch.where(ok, counts, 0)
    # the pages that are handed out, in order, from the top of the stack
    column = torch.arange(width, device=table.device)[None, :]
    taken = (column >= had[:, None]) & (column < (had + need)[:, None]) & ok[:, None]
    rank = (upto - need)[:, None] + column - had[:, None]
    table[taken] = free[4 + (n_free - 1 - rank)[taken]]
    lengths += granted
    row = torch.arange(S, device=table.device)[None, :]
    position = (lengths - granted)[:, None] + row
    live = row < granted[:, None]
    at = table.gather(1, (position // page).clamp(max=width - 1).long())
    positions = torch.where(live, position, -1)
    slots = torch.where(live, at.long() * page + position % page, -1)
    starts = torch.cat([torch.zeros_like(granted[:1]), granted.cumsum(0).int()])
    # and back: what was handed out last goes onto the stack first (it has not been written over)
    table[taken] = -1
    lengths = torch.minimum(lengths, s["keep"])
    return {"granted": granted, "starts": starts, "positions": positions, "slots": slots, "lengths": lengths, "table": table, "free": free}


def _rows(s):
    """Position of each of the S rows in its sequence [B, S] and whether the sequence has that row: the new tokens are the last ones."""
    S, lengths = s["case"]["S"], s["lengths"][:, None]
    counts = lengths.clamp(max=S) if s["counts"] is None else s["counts"][:, None]
    row = torch.arange(S, device=lengths.device)[None, :]
    return lengths - counts + row, row < counts


def _plain_append(s):
    """(The inputs are finite: the words for tokens that hold no numbers stay 0.)"""
    page, S, table, lengths = s["case"]["page"], s["case"]["S"], s["table"], s["lengths"].long()
    counts = lengths.clamp(max=S) if s["counts"] is None else s["counts"].long()
    first = lengths - counts
    k_codes, v_codes, scales = _blocks(s["pool"], page)
    # the blocks that new tokens fall into: [B, N]; their tokens: [B, N, 16]
    N = (S + 2 * BLOCK - 2) // BLOCK
    block = (first // BLOCK)[:, None] + torch.arange(N, device=table.device)
    token = block[..., None] * BLOCK + torch.arange(BLOCK, device=table.device)
    new, old = (token >= first[:, None, None]) & (token < lengths[:, None, None]), token < first[:, None, None]
    b, n = new.any(-1).nonzero(as_tuple=True)
    block, token, new, old = block[b, n], token[b, n], new[b, n], old[b, n]
    where = (table[b, block * BLOCK // page].long(), slice(None), block % (page // BLOCK))
    row = (token - first[b][:, None]).clamp(0, S - 1)
    at, live = _rows(s)
    held = {}
    for i, (name, codes) in enumerate((("k", k_codes), ("v", v_codes))):
        x = s[name][b[:, None], row].float().transpose(1, 2)                                         # [blocks, HK, 16, 128]
        had = _value(codes[where][..., s["places"][i].flatten()]).unflatten(-1, (BLOCK, D))
        scale = _scale_of((x * new[:, None, :, None]).abs().amax((-1, -2)))
        before = scales[(*where, i)]
        scale = torch.where(old.any(-1)[:, None], torch.maximum(scale, before), scale)[..., None, None]
        code = torch.where(new[:, None, :, None], _round(x, scale), _round(had * torch.where(old[:, None, :, None], before[..., None, None] / scale, 1.0), 1.0))
        codes[where] = code.flatten(-2)[..., torch.argsort(s["places"][i].flatten())]
        scales[(*where, i)] = scale[..., 0, 0]
        value = (_value(code) * scale).transpose(1, 2).bfloat16()                                    # [blocks, 16, HK, 128]
        out = torch.zeros_like(s[name + "_held"])
        out[b[:, None].expand_as(row)[new], row[new]] = value[new]
        held[name] = out
    return held


def _plain_attend(s):
    case = s["case"]
    B, H, HK, S, page = (case[x] for x in ("B", "H", "HK", "S", "page"))
    at, live = _rows(s)
    k_codes, v_codes, scales = _blocks(s["pool"], page)
    k = _cached(k_codes, scales[..., 0], s["places"][0], s["table"])
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
    out = x.flatten(2, 3) @ _cached(v_codes, scales[..., 1], s["places"][1], s["table"])
    out = out.view(B, HK, H // HK, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, H, D).bfloat16()
    return {"out": out, "lse": (top + total.log()).view(B, H, S) if case["lse"] else None}


_run_own = {"rope": _own_rope, "pages": _own_pages, "append": _own_append, "attend": _own_attend}
_run_plain = {"rope": _plain_rope, "pages": _plain_pages, "append": _plain_append, "attend": _plain_attend}


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    B, S = case["B"], case["S"]
    if case["kind"] == "rope":
        rows, size = B * S * (case["H"] + case["HK"]), TYPES[case["type"]].itemsize
        return {"bytes": 2 * rows * case["D"] * size + 4 * B * S, "flops": 3 * rows * case["rotary"]}
    lengths, new, page = _lengths(case), _new(case), case["page"]
    if case["kind"] == "pages":
        pages = sum(_pages(n + m, page) - _pages(n, page) for n, m in zip(lengths, new))
        # counts, lengths there and back, granted and starts; positions and slots; pages from the stack to the table and back
        return {"bytes": B * (4 + 8 + 8 + 4 + 4 + 4) + 12 * B * S + 16 * pages, "flops": 8 * B * S}
    HK = case["HK"]
    if case["kind"] == "append":
        # bf16 in, codes and scales out (a block that has older tokens: its scales in too), the values that are held out in bf16
        rows, tokens = B * S * HK, sum(new)
        blocks = sum(_pages(n, BLOCK) - (n - m) // BLOCK for n, m in zip(lengths, new))
        return {"bytes": tokens * HK * (4 * D + 2 * D) + blocks * HK * 32 + rows * 4 * D + 4 * len(lengths), "flops": 6 * tokens * HK * D}
    H, rows, tokens = case["H"], B * S * case["H"], sum(lengths)
    n_bytes = tokens * HK * 257 + 4 * sum(_pages(n, page) for n in lengths) + rows * 4 * D + (rows * 4 if case["lse"] else 0)
    pairs = sum(n * (L - n) + n * (n + 1) // 2 if case["causal"] else n * L for n, L in zip(new, lengths))
    return {"bytes": n_bytes, "flops": 4 * H * D * pairs}


# ------------------------------------------------------------------------------------------------- from the definition, in 64 bits
def _e4m3_64(codes):
    """Bytes to the values they stand for: sign, four exponent bits, three mantissa bits."""
    c = codes.long()
    exponent, mantissa = c // 8 % 16, c % 8
    size = torch.where(exponent == 0, mantissa.double() / 512, (1 + mantissa.double() / 8) * torch.pow(2.0, (exponent - 7).double()))
    return torch.where(c >= 128, -size, size)


def _nearest_64(y):
    """The values of e4m3 nearest to y, ties to even."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.pow(2.0, e) > y.abs().clamp(min=2.0 ** -6), e - 1, e)
    step = torch.pow(2.0, e - 3)
    return (torch.round(y / step) * step).clamp(-LARGEST, LARGEST)


def _tokens_64(s, head, b, tokens):
    """K and V codes' values [n, 128], and the blocks' scales [n] of each, in 64 bits, of the given tokens of one sequence and head."""
    page = s["case"]["page"]
    start = tokens % page // BLOCK * RECORD
    record = s["pool"][s["table"][b][tokens // page].long(), head]
    t, d = (tokens % BLOCK)[:, None], torch.arange(D, device=tokens.device)[None, :]
    pair = t // 2
    k = torch.gather(record, 1, start[:, None] + t * 128 + ((d // 16) ^ (t & 7)) * 16 + (d & 15))
    v = torch.gather(record, 1, start[:, None] + 2048 + pair * 256 + ((d // 8) ^ ((pair & 1) + 2 * (pair & 2))) * 16 + (d & 7) * 2 + (t & 1))
    words = torch.gather(record, 1, start[:, None] + 4096 + torch.arange(8, device=tokens.device)).contiguous().view(torch.float32).double()
    return _e4m3_64(k), _e4m3_64(v), words[:, 0], words[:, 1]


def _exact_rope(case, s):
    n = case["rotary"] // 2
    f, factor = _frequencies(case)
    angle = s["positions"].double()[..., None] * f.cuda()
    # a pair as a complex number
    turn = torch.polar(torch.full_like(angle, factor), -angle if case["backward"] else angle)[:, :, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        pair = x[..., :2 * n].unflatten(-1, (n, 2) if case["interleaved"] else (2, n))
        pair = pair if case["interleaved"] else pair.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        x[..., :2 * n] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        out[name] = x
    return out


def _exact_append(case, s):
    """Sequence by sequence, the new tokens' blocks filled up with what they held and with zeros."""
    lengths, new = _lengths(case), _new(case)
    out = {name: torch.zeros(s[name].shape, dtype=torch.float64, device="cuda") for name in ("k", "v")}
    for b, (L, n) in enumerate(zip(lengths, new)):
        if n == 0:
            continue
        first = L - n
        old = first % BLOCK
        fill = (-L) % BLOCK
        for h in range(case["HK"]):
            held = _tokens_64(s, h, b, torch.arange(first - old, first, device="cuda"))
            for i, name in enumerate(("k", "v")):
                x = s[name][b, :n, h].double()
                blocks = torch.cat([torch.zeros(old, D, device="cuda", dtype=torch.float64), x, torch.zeros(fill, D, device="cuda", dtype=torch.float64)]).view(-1, BLOCK * D)
                scale = torch.pow(2.0, torch.ceil(torch.log2(blocks.abs().amax(1).clamp(min=LARGEST * 2.0 ** -90) / LARGEST)))
                if old:
                    scale[0] = torch.maximum(scale[0], held[2 + i][0])
                out[name][b, :n, h] = (_nearest_64(blocks / scale[:, None]) * scale[:, None]).view(-1, D)[old:old + n]
    return out


def exact(case, seed):
    if case["kind"] == "pages":
        return None   # whole numbers throughout
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(case, s)
    if case["kind"] == "append":
        return _exact_append(case, s)
    lengths, HK, H, S, new = _lengths(case), case["HK"], case["H"], case["S"], _new(case)
    group = H // HK
    out = torch.zeros((case["B"], S, H, D), dtype=torch.float64, device="cuda")
    lse = torch.full((case["B"], H, S), -math.inf, dtype=torch.float64, device="cuda")
    for b, (n, L) in enumerate(zip(new, lengths)):
        if not L:
            continue
        tokens = torch.arange(L, device="cuda")
        hidden = tokens[None, :] > (L - n + torch.arange(n, device="cuda"))[:, None] if case["causal"] else None
        for h in range(HK):
            k, v, k_scale, v_scale = _tokens_64(s, h, b, tokens)
            k, v = k * k_scale[:, None], v * v_scale[:, None]
            for head in range(h * group, (h + 1) * group):
                x = (s["q"][b, :n, head].double() @ k.T) / math.sqrt(D)
                if hidden is not None:
                    x.masked_fill_(hidden, -math.inf)
                lse[b, head, :n] = torch.logsumexp(x, 1)
                out[b, :n, head] = torch.exp(x - lse[b, head, :n][:, None]) @ v
    return {"out": out, "lse": lse if case["lse"] else None}
