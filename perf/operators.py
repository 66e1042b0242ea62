"""Serving from a cache of 4-bit keys and values, and drawing the next token: what is measured, with its plain forms.

Three kinds of case.  ``append``: a step's projected queries, keys and values are rotated by their positions, the queries
narrowed, the keys and values brought to 4 bits and put into their blocks of the cache; the answer is the queries and what the blocks that
the step wrote now stand for.  ``attend``: the step's queries attend over the cache.  ``sample``: the next token of every row of
logits from a given random number, with the row's own temperature, top-k, top-p and min-p.

The cache.  Tokens lie in blocks of 64, which a table names per sequence.  A head of D numbers is cut into G = D / 32 groups of 32
neighbouring numbers.  A group of a token is 32 codes n of 4 bits with a scale s and a least value m, both bfloat16, and stands
for m + s n: m is the least of the 32 numbers rounded down, s the fifteenth part of (greatest - m) rounded up, n the
nearest whole number to (x - m) / s.  Where a number is not finite, or its group's scale or least value would not be, s is NaN, m and n are zero.

A block of one head, as bytes.  Keys: codes as 32-bit words [64 tokens][4][G], then [64 tokens][G] pairs (s, m).  Word [t][c][g] holds
numbers 32 g + 8 c + 2 i + h of token t at bits 4 i + 16 h (i = 0..3, h = 0, 1).  Values: codes as 32-bit words [4][G][8][4][2], then
s as [64 tokens][G], then m as [G][64 tokens].  Word [a][g][r][c][j] holds, at bits 4 (2 p + e) + 16 h, number 32 g + 16 j + 8 e + r of
token 16 a + 4 c + 2 p + h.  (These are the orders in which tensor-core fragments take them.)
"""
import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 64


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # A chat server's decode step: eight sequences bring a token each; their products come in four k-slices.
        {"name": "append_decode_8", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 64, "rotary": 64, "interleaved": False, "slices": 4,
         "batch": 8, "context": 900, "new": 1},
        # A prompt of the headline benchmark's length, heads of the 8B shape.
        {"name": "append_prompt_2048", "kind": "append", "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "slices": 1,
         "batch": 1, "context": 0, "new": 2048},
        # Pieces of several conversations that start and end anywhere in a block; half of a head rotated, neighbours paired, far positions.
        {"name": "append_ragged_5", "kind": "append", "heads": 20, "kv_heads": 4, "dim": 96, "rotary": 48, "interleaved": True, "slices": 2,
         "batch": 5, "context": 70001, "new": 157},
        # One user's chat, a token at a time: the smallest call, whose latency is felt.
        {"name": "attend_decode_1", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 64, "batch": 1, "context": 2048, "new": 1, "window": 0},
        # A busy server's decode step: 64 conversations of up to 4,096 tokens, heads of the 8B shape.
        {"name": "attend_decode_64", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 64, "context": 4096, "new": 1, "window": 0},
        # Two readers of long documents.
        {"name": "attend_decode_long_2", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 2, "context": 40001, "new": 1, "window": 0},
        # Layers that see the last 1,000 tokens, sixteen query heads to a key head, heads of 96.
        {"name": "attend_decode_window_31", "kind": "attend", "heads": 32, "kv_heads": 2, "dim": 96, "batch": 31, "context": 2500, "new": 1, "window": 1000},
        # Drafted tokens that a large model checks: five more for each of 16 conversations.
        {"name": "attend_draft_16", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 16, "context": 2011, "new": 5, "window": 0},
        # The second piece of a long prompt.
        {"name": "attend_prompt_2048", "kind": "attend", "heads": 32, "kv_heads": 8, "dim": 128, "batch": 1, "context": 1000, "new": 2048, "window": 0},
        # One user's next token: nucleus and min-p.
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 128256, "temperature": 0.8, "top_k": 0, "top_p": 0.95, "min_p": 0.02, "mixed": False},
        # A server's batch whose requests ask for different things.
        {"name": "sample_mixed_64", "kind": "sample", "rows": 64, "vocab": 128256, "temperature": 1.0, "top_k": 50, "top_p": 0.9, "min_p": 0.05, "mixed": True},
        # A smaller, odd vocabulary and many rows, temperature and top-k alone.
        {"name": "sample_topk_200", "kind": "sample", "rows": 200, "vocab": 32003, "temperature": 0.7, "top_k": 40, "top_p": 1.0, "min_p": 0.0, "mixed": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "sample"))
    if kind == "sample":
        vocab = _spread(rng, 300, 152000)
        return {"kind": kind, "rows": _spread(rng, 1, max(1, min(256, 64 * 128256 // vocab))), "vocab": vocab, "temperature": rng.choice((0.6, 0.8, 1.0, 1.3)),
                "top_k": rng.choice((0, 1, 20, 64, 500)), "top_p": rng.choice((1.0, 0.95, 0.8, 0.3)), "min_p": rng.choice((0.0, 0.02, 0.1)),
                "mixed": rng.random() < 0.5}
    dim = rng.choice((64, 128, 64, 128, 32, 96))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 3, 4, 7, 8, 12, 16) if kv_heads < 4 else (1, 2, 4, 5))
    if kind == "append":
        new = 1 if rng.random() < 0.5 else _spread(rng, 2, 1500)
        return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice((dim, dim, dim // 2, 0)),
                "interleaved": rng.random() < 0.3, "slices": rng.choice((1, 1, 2, 3)), "batch": _spread(rng, 1, min(64, max(1, 3000 // new))),
                "context": _spread(rng, 1, 2000 if new == 1 else 100000), "new": new}
    what = rng.random()
    if what < 0.55:                                             # decoding
        batch = _spread(rng, 1, 64)
        context, new = _spread(rng, 5, min(40000, 64 * 4096 // batch)), 1
    elif what < 0.8:                                            # a few tokens each
        batch, new = _spread(rng, 1, 24), rng.randint(2, 12)
        context = _spread(rng, 1, 4000)
    else:
        batch, new, context = rng.randint(1, 3), _spread(rng, 20, 1400), _spread(rng, 1, 2500)
    return {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "batch": batch, "context": context, "new": new,
            "window": rng.choice((0, 0, 0, 100, 777))}


def lengths(case):
    """Per sequence: the tokens that the cache holds already and those that the step brings.  The first sequence has the case's numbers,
    the others fewer; decoding sequences bring one token each."""
    rng = random.Random(case["context"] * 131 + case["batch"] * 7 + case["new"])
    before, new = [case["context"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        before.append(max(0, int(case["context"] * (0.55 + 0.45 * rng.random()))))
        new.append(case["new"] if case["new"] <= 5 else max(1, int(case["new"] * (0.4 + 0.6 * rng.random()))))
    return before, new


def _first_key(position, window):
    return max(0, position - window + 1) if window else 0


# --------------------------------------------------------------------------------------------------- the cache's format

def quantise(x):
    """Float32 [..., D] -> codes int32 [..., D], scales and least values bfloat16 [..., G]."""
    x = x.float().unflatten(-1, (-1, 32))
    least = x.amin(-1)
    bits = least.view(torch.int32)
    up = torch.where((bits < 0) & ((bits & 0xFFFF) != 0), bits + 0x10000, bits) & -0x10000          # towards minus infinity
    m = up.view(torch.float32)
    s = (x.amax(-1) - m) * torch.tensor(1.0 / 15.0, dtype=torch.float32, device=x.device)
    bits = s.view(torch.int32)
    s = (torch.where((bits & 0xFFFF) != 0, bits + 0x10000, bits) & -0x10000).view(torch.float32)    # upwards
    bad = ~(torch.isfinite(x).all(-1) & torch.isfinite(m) & torch.isfinite(s))
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    inverse = torch.where(s > 0, 1.0 / s, 0.0)
    n = torch.round((x - m[..., None]) * inverse[..., None]).clamp(0.0, 15.0)
    n = torch.where(bad[..., None], 0.0, n).to(torch.int32)
    return n.flatten(-2), torch.where(bad, math.nan, s).to(torch.bfloat16), torch.where(bad, 0.0, m).to(torch.bfloat16)


def _bytes(t, lead):
    """The bytes of what stands behind the first ``lead`` axes."""
    return t.flatten(lead).contiguous().view(torch.uint8)


def pack_keys(n, s, m):
    """Codes [..., 64, D], scales and least values [..., 64, G] -> bytes [..., 64 * 20 * G]."""
    lead, groups = n.shape[:-2], s.shape[-1]
    n = n.reshape(*lead, 64, groups, 4, 4, 2)                                                        # token, g, c, i, h
    shifts = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], dtype=torch.int32, device=n.device)
    words = (n << shifts).sum((-1, -2), dtype=torch.int64).to(torch.int32).transpose(-1, -2)         # token, c, g
    return torch.cat((_bytes(words, len(lead)), _bytes(torch.stack((s, m), dim=-1), len(lead))), dim=-1)


def unpack_keys(pool, dim):
    """The inverse: bytes [..., 64 * 20 * G] -> codes, scales, least values."""
    lead, groups = pool.shape[:-1], dim // 32
    words = pool[..., :32 * dim].contiguous().view(torch.int32).reshape(*lead, 64, 4, groups)
    shifts = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], dtype=torch.int32, device=pool.device)
    n = ((words.transpose(-1, -2)[..., None, None] >> shifts) & 15).reshape(*lead, 64, dim)
    pairs = pool[..., 32 * dim:].contiguous().view(torch.bfloat16).reshape(*lead, 64, groups, 2)
    return n, pairs[..., 0], pairs[..., 1]


_VALUE_SHIFTS = [[[0, 16], [4, 20]], [[8, 24], [12, 28]]]                                            # p, e, h


def pack_values(n, s, m):
    lead, groups = n.shape[:-2], s.shape[-1]
    k = len(lead)
    n = n.reshape(*lead, 4, 4, 2, 2, groups, 2, 2, 8)                                                # a, c, p, h, g, j, e, r
    n = n.permute(*range(k), k, k + 4, k + 7, k + 1, k + 5, k + 2, k + 6, k + 3)                     # a, g, r, c, j, p, e, h
    shifts = torch.tensor(_VALUE_SHIFTS, dtype=torch.int32, device=n.device)
    words = (n << shifts).sum((-1, -2, -3), dtype=torch.int64).to(torch.int32)
    return torch.cat((_bytes(words, k), _bytes(s, k), _bytes(m.transpose(-1, -2), k)), dim=-1)


def unpack_values(pool, dim):
    lead, groups = pool.shape[:-1], dim // 32
    k = len(lead)
    words = pool[..., :32 * dim].contiguous().view(torch.int32).reshape(*lead, 4, groups, 8, 4, 2)
    shifts = torch.tensor(_VALUE_SHIFTS, dtype=torch.int32, device=pool.device)
    n = (words[..., None, None, None] >> shifts) & 15                                                # a, g, r, c, j, p, e, h
    n = n.permute(*range(k), k, k + 3, k + 5, k + 7, k + 1, k + 4, k + 6, k + 2).reshape(*lead, 64, dim)
    rest = pool[..., 32 * dim:].contiguous().view(torch.bfloat16)
    s = rest[..., :64 * groups].reshape(*lead, 64, groups)
    m = rest[..., 64 * groups:].reshape(*lead, groups, 64).transpose(-1, -2)
    return n, s, m


def stands_for(n, s, m):
    """Float32 numbers: m + s n, group by group."""
    n = n.unflatten(-1, (-1, 32))
    return (m.float()[..., None] + s.float()[..., None] * n.float()).flatten(-2)


# --------------------------------------------------------------------------------------------------------------- inputs

def _vectors(shape, generator, keys):
    """What heads look like: channels of different sizes, and for keys a few large ones and offsets that all tokens share."""
    dim = shape[-1]
    size = torch.exp(0.4 * torch.randn(dim, generator=generator, device=DEVICE))
    x = torch.randn(shape, generator=generator, device=DEVICE) * size
    if keys:
        x += torch.randn(dim, generator=generator, device=DEVICE)
    return x


def _pools(blocks, case, generator):
    """What earlier steps left: every block full (behind a sequence's end lie an older sequence's tokens)."""
    kv, dim = case["kv_heads"], case["dim"]
    k_pool = torch.empty((blocks, kv, 40 * dim), dtype=torch.uint8, device=DEVICE)
    v_pool = torch.empty_like(k_pool)
    for at in range(0, blocks, 512):                            # bounds the memory that the making takes
        count = min(512, blocks - at)
        k_pool[at:at + count] = pack_keys(*quantise(_vectors((count, kv, BLOCK, dim), generator, True)))
        v_pool[at:at + count] = pack_values(*quantise(_vectors((count, kv, BLOCK, dim), generator, False)))
    return k_pool, v_pool


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE)
    generator.manual_seed(seed)
    if case["kind"] == "sample":
        return _prepare_rows(case, seed, generator)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    before, new = lengths(case)
    cu = [0]
    for count in new:
        cu.append(cu[-1] + count)
    totals = [b + c for b, c in zip(before, new)]
    window = case.get("window", 0)
    # append: the blocks that the step writes; attend: those that it sees.  Blocks before them were given back (-1).
    firsts = [b // BLOCK if case["kind"] == "append" else _first_key(b, window) // BLOCK for b in before]
    ends = [-(-t // BLOCK) for t in totals]
    blocks = sum(e - f for f, e in zip(firsts, ends))
    names = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(ends) + 1
    table = [[-1] * f + [names.pop() for _ in range(e - f)] + [-1] * (width - e) for f, e in zip(firsts, ends)]
    s = {"case": case, "n_tokens": cu[-1], "sequences": len(new), "width": width, "longest": max(totals), "most_new": max(new),
         "cu": _ints(cu), "len_before": _ints(before), "table": _ints(table), "status": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    s["k_pool"], s["v_pool"] = _pools(blocks, case, generator)
    # where each packed token stands, for the plain forms: its sequence, its place in it, its position
    s["sequence"] = torch.cat([torch.full((c,), i, dtype=torch.int64) for i, c in enumerate(new)]).to(DEVICE)
    s["place"] = torch.cat([torch.arange(c) for c in new]).to(DEVICE)
    s["position"] = torch.cat([torch.arange(c) + b for b, c in zip(before, new)]).to(DEVICE)
    if case["kind"] == "attend":
        # queries lean towards some keys, so that the softmax is neither flat nor one key
        q = 0.7 * _vectors((cu[-1], heads, dim), generator, True)
        s["q"] = q.to(torch.bfloat16).reshape(cu[-1], heads * dim)
        s["out"] = torch.zeros((cu[-1], heads * dim), dtype=torch.bfloat16, device=DEVICE)
        return s
    slices = case["slices"]
    keys = _vectors((cu[-1], kv, dim), generator, True).flatten(1)
    rows = torch.cat((_vectors((cu[-1], heads * dim), generator, False), keys, _vectors((cu[-1], kv * dim), generator, False)), dim=1)
    parts = torch.randn((slices, *rows.shape), generator=generator, device=DEVICE)                   # partial sums of k-slices
    parts[0] += rows - parts.sum(0)
    s["qkv"] = parts
    s["inv_freq"] = (500000.0 ** (-torch.arange(0, max(case["rotary"], 2), 2, dtype=torch.float64) / max(case["rotary"], 2))).float().to(DEVICE)
    s["q_out"] = torch.empty((cu[-1], heads * dim), dtype=torch.bfloat16, device=DEVICE)
    # the read-back: for each sequence as many blocks as any of them touches; what a sequence does not touch stays zero
    span = max(e - f for f, e in zip(firsts, ends))
    s["keys"] = torch.zeros((len(new) * span, kv, BLOCK, dim), dtype=torch.bfloat16, device=DEVICE)
    s["values"] = torch.zeros((len(new) * span, kv, dim, BLOCK), dtype=torch.bfloat16, device=DEVICE)
    s["table_tmp"] = torch.zeros_like(s["table"])
    touched = [(i, w) for i, (f, e) in enumerate(zip(firsts, ends)) for w in range(f, e)]
    index = {pair: k for k, pair in enumerate(touched)}
    s["touched"] = torch.tensor([i * span + w - firsts[i] for i, w in touched], device=DEVICE)
    s["touched_pool"] = torch.tensor([table[i][w] for i, w in touched], device=DEVICE)
    s["touched_left"] = torch.tensor([totals[i] - w * BLOCK for i, w in touched], device=DEVICE)     # tokens in the block
    s["token_block"] = torch.tensor([index[(i, (b + j) // BLOCK)] for i, (b, c) in enumerate(zip(before, new)) for j in range(c)], device=DEVICE)
    return s


def _prepare_rows(case, seed, generator):
    rows, vocab = case["rows"], case["vocab"]
    rng = random.Random(seed)
    logits = 2.5 * torch.randn((rows, vocab), generator=generator, device=DEVICE)
    favoured = torch.randint(0, vocab, (rows, 30), generator=generator, device=DEVICE)               # a next token is rarely anybody's guess
    logits.scatter_add_(1, favoured, 6.0 + 4.0 * torch.rand((rows, 30), generator=generator, device=DEVICE))
    settings = [(case["temperature"], case["top_k"], case["top_p"], case["min_p"])] * rows
    if case["mixed"]:                                           # each request asks for its own filters, some for none, some for the likeliest token
        settings = [(rng.choice((0.0, t, t, 1.2 * t, 0.8 * t)), rng.choice((0, k)), rng.choice((1.0, p)), rng.choice((0.0, m))) for t, k, p, m in settings]
    column = lambda i, dtype: torch.tensor([row[i] for row in settings], dtype=dtype, device=DEVICE)  # noqa: E731
    return {"case": case, "logits": logits, "uniform": torch.rand(rows, generator=generator, device=DEVICE), "temperature": column(0, torch.float32),
            "top_k": column(1, torch.int32), "top_p": column(2, torch.float32), "min_p": column(3, torch.float32),
            "out": torch.zeros(rows, dtype=torch.int32, device=DEVICE)}


# ---------------------------------------------------------------------------------------------------------- plain forms

def _rotate(x, position, inv_freq, rotary, interleaved):
    """Float32 [tokens, heads, D]; the angles are formed in 64 bits."""
    if not rotary:
        return x
    angle = position[:, None].double() * inv_freq[:rotary // 2].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    turned, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _put(s, pool, new, unpack, pack):
    """The step's vectors into their places, and what the blocks then stand for."""
    n, scale, least = unpack(pool[s["touched_pool"]], new.shape[-1])
    block, at = s["token_block"], s["position"] % BLOCK
    n[block, :, at], scale[block, :, at], least[block, :, at] = quantise(new)
    pool[s["touched_pool"]] = pack(n, scale, least)
    kept = torch.arange(BLOCK, device=DEVICE) < s["touched_left"][:, None]
    return torch.where(kept[:, None, :, None], stands_for(n, scale, least), 0.0).to(torch.bfloat16)


def _plain_append(s):
    case = s["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    rows = s["qkv"].sum(0).unflatten(1, (-1, dim))
    turned = _rotate(rows[:, :heads + kv], s["position"], s["inv_freq"], case["rotary"], case["interleaved"])
    q = turned[:, :heads].flatten(1).to(torch.bfloat16)
    keys = _put(s, s["k_pool"], turned[:, heads:], unpack_keys, pack_keys)
    values = _put(s, s["v_pool"], rows[:, heads + kv:], unpack_values, pack_values)
    s["keys"][s["touched"]] = keys
    s["values"][s["touched"]] = values.transpose(-1, -2)
    return {"q": q, "keys": s["keys"], "values": s["values"]}


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    seqs, most, longest = s["sequences"], s["most_new"], s["longest"]
    blocks = s["table"][:, :-(-longest // BLOCK)].long().clamp_min(0)
    k = stands_for(*unpack_keys(s["k_pool"][blocks], dim)).permute(0, 2, 1, 3, 4).flatten(2, 3)      # [sequences, kv, keys, D]
    v = stands_for(*unpack_values(s["v_pool"][blocks], dim)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    q = torch.zeros((seqs, most, heads, dim), device=DEVICE)
    q[s["sequence"], s["place"]] = s["q"].float().unflatten(1, (heads, dim))
    at = s["len_before"].long()[:, None] + torch.arange(most, device=DEVICE)
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if window:
        seen &= key > at[..., None] - window
    q = q.view(seqs, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim)
    scores = (q @ k.transpose(-1, -2)).view(seqs, kv, heads // kv, most, -1) * dim ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p.flatten(2, 3) @ v).view(seqs, kv, heads // kv, most, dim) / p.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * dim)
    return out[s["sequence"], s["place"]].to(torch.bfloat16)


def _plain_sample(s):
    x = torch.where(torch.isnan(s["logits"]), -math.inf, s["logits"]).double()
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    temperature = s["temperature"].double()[:, None]
    greedy = temperature == 0
    w = torch.exp(torch.where(x == top, 0.0, (x - top) / torch.where(greedy, 1.0, temperature)))
    ordered, order = x.sort(1, descending=True)
    k = s["top_k"].long()[:, None]
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    least = ordered.gather(1, k - 1)
    mass = torch.where(ordered >= least, w.gather(1, order), 0.0)
    above = mass.cumsum(1) - mass
    starts = torch.cat((torch.ones_like(ordered[:, :1], dtype=torch.bool), ordered[:, 1:] != ordered[:, :-1]), dim=1)
    above = torch.where(starts, above, 0.0).cummax(1).values                                         # of the strictly larger ones
    p = s["top_p"].double()[:, None]
    stays = (ordered >= least) & ((p >= 1.0) | (above <= p * mass.sum(1, keepdim=True)))
    edge = torch.where(stays, ordered, math.inf).amin(1, keepdim=True)
    kept = torch.where((x >= edge) & (w >= s["min_p"].double()[:, None]), w, 0.0).cumsum(1)
    drawn = (kept <= s["uniform"].double()[:, None] * kept[:, -1:]).sum(1, keepdim=True)
    likeliest = torch.where(x == top, torch.arange(vocab, device=x.device), vocab).amin(1, keepdim=True)
    drawn = torch.where(greedy, likeliest, drawn)
    return torch.where(top == -math.inf, 0, drawn)[:, 0].to(torch.int32)


# ------------------------------------------------------------------------------------------------------------------ run

def _layer(s):
    """What a program that runs an attention layer keeps: the layer, its step's description and scratch memory."""
    from thintensor_b200.cache.cache import RunCache
    from thintensor_b200.engine.context import StepContext, Workspace
    from thintensor_b200.parts import MIXERS

    case = s["case"]
    mixer = MIXERS.build("attention", {"hidden": case["heads"] * case["dim"], "heads": case["heads"], "kv_heads": case["kv_heads"],
                                       "head_dim": case["dim"], "window": case["window"] or None})
    ctx = StepContext(n_tokens=s["n_tokens"], sequences=s["sequences"], decode=s["most_new"] == 1, max_new=s["most_new"],
                      max_total=s["width"] * BLOCK, tokens=s["cu"], cu=s["cu"], len_before=s["len_before"], slots=s["cu"], tables=[s["table"]],
                      act_dtype=torch.bfloat16, workspace=Workspace(torch.device(DEVICE, torch.cuda.current_device())), status=s["status"])
    return mixer, ctx, RunCache(0, s["k_pool"], s["v_pool"], True, case["window"] or None)


def run(s):
    case = s["case"]
    if case["kind"] == "append":
        if not own:
            return _plain_append(s)
        from thintensor_b200.kernels import api

        api.rope_append_4bit(s["qkv"], s["inv_freq"], case["rotary"], 1.0, s["q_out"], s["k_pool"], s["v_pool"], s["table"], s["cu"],
                             s["len_before"], s["sequences"], s["n_tokens"], case["heads"], case["kv_heads"], case["dim"], s["status"],
                             interleaved=case["interleaved"])
        api.expand_4bit(s["k_pool"], s["v_pool"], s["table"], s["cu"], s["len_before"], s["sequences"], 1, s["keys"], s["values"],
                        s["table_tmp"], s["status"])
        return {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}
    if case["kind"] == "attend":
        if not own:
            return _plain_attend(s)
        if "layer" not in s:
            s["layer"] = _layer(s)
        mixer, ctx, cache = s["layer"]
        mixer.attend(ctx, s["q"], cache, s["table"], s["out"])
        return s["out"]
    if not own:
        return _plain_sample(s)
    from thintensor_b200.kernels import api

    api.sample_filtered(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["out"], uniform=s["uniform"])
    return s["out"]


def work(case):
    if case["kind"] == "sample":
        numbers = case["rows"] * case["vocab"]
        return {"bytes": 4 * numbers + 24 * case["rows"], "flops": 4 * numbers}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    before, new = lengths(case)
    token = 2 * kv * (dim * 5 // 8)                             # bytes of a token's keys and values: 4 bits, and 32 bits for each 32
    if case["kind"] == "append":
        row = (heads + 2 * kv) * dim
        # partial sums in, queries out, codes out, and the written tokens' values out again
        return {"bytes": sum(new) * (4 * case["slices"] * row + 2 * heads * dim + 2 * token + 4 * kv * dim), "flops": sum(new) * row * 6}
    seen = sum(b + c - _first_key(b, case["window"]) for b, c in zip(before, new))
    pairs = sum(b + j + 1 - _first_key(b + j, case["window"]) for b, c in zip(before, new) for j in range(c))
    return {"bytes": seen * token + sum(new) * heads * dim * 4, "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------------------------------------------------------ in 64 bits

def _bit_places(dim):
    """Word and shift of each (token, number) of a block, for keys and for values."""
    groups = dim // 32
    token, d = np.meshgrid(np.arange(64), np.arange(dim), indexing="ij")
    g, u = d // 32, d % 32
    key_word, key_shift = (token * 4 + u // 8) * groups + g, 4 * (u % 8 // 2) + 16 * (u % 2)
    value_word = (((token // 16 * groups + g) * 8 + u % 8) * 4 + token % 16 // 4) * 2 + u // 16
    value_shift = 4 * (2 * (token % 4 // 2) + u % 16 // 8) + 16 * (token % 2)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)  # noqa: E731
    return to(key_word), to(key_shift), to(value_word), to(value_shift)


def _numbers(pool, places, dim, values):
    """Blocks of one head or more, bytes [..., 40 D] -> float64 [..., 64, D]."""
    word, shift = places[2:] if values else places[:2]
    whole = pool.contiguous().view(torch.int32).long()
    n = (whole[..., word] >> shift) & 15
    token = torch.arange(64, device=DEVICE)[:, None]
    group = torch.arange(dim, device=DEVICE) // 32
    groups = dim // 32
    halves = pool.contiguous().view(torch.bfloat16).double()
    base = 16 * dim
    if values:
        scale, least = halves[..., base + token * groups + group], halves[..., base + 64 * groups + group * 64 + token]
    else:
        scale, least = halves[..., base + 2 * (token * groups + group)], halves[..., base + 2 * (token * groups + group) + 1]
    return least + scale * n


def _to_eight_bits(x, up):
    """Float64 to 8 significant bits, down (towards minus infinity) or up."""
    mantissa, exponent = torch.frexp(x)
    steps = mantissa * 256.0
    return torch.ldexp(steps.ceil() if up else steps.floor(), exponent - 8)


def _nearest_values(x):
    """What 4 bits leave of float64 [..., D]."""
    x = x.unflatten(-1, (-1, 32))
    m = _to_eight_bits(x.amin(-1, keepdim=True), False)
    s = _to_eight_bits((x.amax(-1, keepdim=True) - m) / 15.0, True)
    n = torch.where(s > 0, (x - m) / s, 0.0).round().clamp(0, 15)
    return (m + s * n).flatten(-2)


def exact(case, seed):
    if case["kind"] == "sample":
        return None
    s = prepare(case, seed)
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    before, new = lengths(case)
    places = _bit_places(dim)
    if case["kind"] == "attend":
        out = torch.empty((sum(new), heads * dim), dtype=torch.float64, device=DEVICE)
        at = 0
        for i, (b, c) in enumerate(zip(before, new)):
            first = _first_key(b, case["window"]) // BLOCK
            names = s["table"][i, first:-(-(b + c) // BLOCK)].long()
            position = torch.arange(b, b + c, device=DEVICE)[:, None]
            key = torch.arange(first * BLOCK, first * BLOCK + len(names) * BLOCK, device=DEVICE)
            hidden = (key > position) | ((key <= position - case["window"]) if case["window"] else False)
            for h in range(kv):
                k = _numbers(s["k_pool"][names, h], places, dim, False).flatten(0, 1)
                v = _numbers(s["v_pool"][names, h], places, dim, True).flatten(0, 1)
                for j in range(h * (heads // kv), (h + 1) * (heads // kv)):
                    z = s["q"][at:at + c, j * dim:(j + 1) * dim].double() @ k.T / math.sqrt(dim)
                    z[hidden] = -math.inf
                    out[at:at + c, j * dim:(j + 1) * dim] = torch.softmax(z, dim=1) @ v
            at += c
        return out
    rows = s["qkv"].double().sum(0)
    angle = s["position"].double()[:, None] * s["inv_freq"].double()[None, :case["rotary"] // 2]
    turn = torch.polar(torch.ones_like(angle), angle)
    for h in range(heads + kv if case["rotary"] else 0):
        part = rows[:, h * dim:h * dim + case["rotary"]]
        pairs = part.reshape(len(part), -1, 2) if case["interleaved"] else part.reshape(len(part), 2, -1).transpose(1, 2)
        done = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        rows[:, h * dim:h * dim + case["rotary"]] = done.reshape(len(part), -1) if case["interleaved"] else done.transpose(1, 2).reshape(len(part), -1)
    keys = torch.zeros((s["keys"].shape[0], kv, BLOCK, dim), dtype=torch.float64, device=DEVICE)
    values = torch.zeros_like(keys)
    keys[s["touched"]] = _numbers(s["k_pool"][s["touched_pool"]], places, dim, False)
    values[s["touched"]] = _numbers(s["v_pool"][s["touched_pool"]], places, dim, True)
    where, at = s["touched"][s["token_block"]], s["position"] % BLOCK
    keys[where, :, at] = _nearest_values(rows[:, heads * dim:(heads + kv) * dim].reshape(-1, kv, dim))
    values[where, :, at] = _nearest_values(rows[:, (heads + kv) * dim:].reshape(-1, kv, dim))
    gone = torch.arange(BLOCK, device=DEVICE) >= s["touched_left"][:, None]
    for t in (keys, values):
        t[s["touched"]] = t[s["touched"]].masked_fill(gone[:, None, :, None], 0.0)
    return {"q": rows[:, :heads * dim], "keys": keys, "values": values.transpose(-1, -2).contiguous()}
