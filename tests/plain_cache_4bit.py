"""The 4-bit cache and the attention over it, stated plainly: codes, scales and least values by their definition, bytes by their places, softmax
attention in float64; and the token that a row of logits gives at a random number."""
from __future__ import annotations

import math

import torch

BLOCK = 64


def _up(x: torch.Tensor) -> torch.Tensor:
    """Float32 to the next bfloat16 upwards, as float32."""
    bits = x.view(torch.int32)
    away = (bits & 0xFFFF) != 0
    return torch.where((bits >= 0) & away, (bits & -0x10000) + 0x10000, bits & -0x10000).view(torch.float32)


def quantise(x: torch.Tensor):
    """Float32 [..., D] on the CPU -> codes int64 [..., D], s and m float32 [..., D / 32], by the operations that the definition names."""
    x = x.float().cpu().reshape(*x.shape[:-1], -1, 32)
    m = -_up(-x.amin(-1))
    s = _up((x.amax(-1) - m) * torch.tensor(1.0 / 15.0, dtype=torch.float32))
    bad = ~(torch.isfinite(x).all(-1) & torch.isfinite(m) & torch.isfinite(s))
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    n = torch.round((x - m[..., None]) * inverse[..., None]).clamp(0, 15)
    n = torch.where(bad[..., None], torch.zeros_like(n), n).to(torch.int64)
    return n.reshape(*n.shape[:-2], -1), torch.where(bad, torch.full_like(s, math.nan), s), torch.where(bad, torch.zeros_like(m), m)


def places(dim: int):
    """For token t and number d of a block of one head: (word, shift) of its code among the keys and among the values."""
    groups = dim // 32
    keys, values = {}, {}
    for t in range(BLOCK):
        for d in range(dim):
            g, u = divmod(d, 32)
            c, (i, h) = u // 8, divmod(u % 8, 2)
            keys[t, d] = ((t * 4 + c) * groups + g, 4 * i + 16 * h)
            j, e, r = u // 16, u % 16 // 8, u % 8
            a, cc, (p, hh) = t // 16, t % 16 // 4, divmod(t % 4, 2)
            values[t, d] = ((((a * groups + g) * 8 + r) * 4 + cc) * 2 + j, 4 * (2 * p + e) + 16 * hh)
    return keys, values


_maps: dict = {}


def _index(dim: int, values: bool):
    if (dim, values) not in _maps:
        table = places(dim)[1 if values else 0]
        word = torch.tensor([[table[t, d][0] for d in range(dim)] for t in range(BLOCK)])
        shift = torch.tensor([[table[t, d][1] for d in range(dim)] for t in range(BLOCK)])
        _maps[dim, values] = word, shift
    return _maps[dim, values]


def read_block(raw: torch.Tensor, dim: int, values: bool):
    """Bytes [40 * dim] of one head's keys (values) of one block -> codes int64 [64, dim], s, m float32 [64, dim / 32]."""
    raw, groups = raw.cpu().contiguous(), dim // 32
    word, shift = _index(dim, values)
    n = (raw[:32 * dim].view(torch.int32).long()[word] >> shift) & 15
    rest = raw[32 * dim:].view(torch.bfloat16).float()
    if values:
        return n, rest[:64 * groups].view(64, groups), rest[64 * groups:].view(groups, 64).T
    pairs = rest.view(64, groups, 2)
    return n, pairs[..., 0], pairs[..., 1]


def write_block(n: torch.Tensor, s: torch.Tensor, m: torch.Tensor, values: bool) -> torch.Tensor:
    """The inverse: bytes [40 * dim]."""
    dim = n.shape[1]
    word, shift = _index(dim, values)
    words = torch.zeros(8 * dim, dtype=torch.int64)
    words.index_add_(0, word.flatten(), (n << shift).flatten())
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    rest = torch.cat((s.flatten(), m.T.flatten())) if values else torch.stack((s, m), dim=-1).flatten()
    return torch.cat((words.view(torch.uint8), rest.to(torch.bfloat16).view(torch.uint8)))


def numbers(n, s, m) -> torch.Tensor:
    """Float64 [..., D]: m + s n."""
    wide = lambda t: t.double().repeat_interleave(32, dim=-1)  # noqa: E731
    return wide(m) + wide(s) * n.double()


class Cache:
    """Pools on the device and what they stand for on the host, for sequences of given lengths; blocks in any order, everything behind a sequence's
    end left over from an older one."""

    def __init__(self, totals, kv_heads: int, dim: int, seed: int = 0, spare: int = 2, key_scale: float = 1.0, value_scale: float = 1.0, extra_width: int = 1):
        g = torch.Generator().manual_seed(seed)
        self.kv_heads, self.dim, self.totals = kv_heads, dim, list(totals)
        self.width = max(-(-t // BLOCK) for t in totals) + extra_width
        count = sum(-(-t // BLOCK) for t in totals) + spare
        order = torch.randperm(count, generator=g).tolist()
        self.table = torch.full((len(totals), self.width), -1, dtype=torch.int32)
        for b, t in enumerate(totals):
            for w in range(-(-t // BLOCK)):
                self.table[b, w] = order.pop()
        self.codes = {"k": [], "v": []}
        for name, scale, offset in (("k", key_scale, 1.0), ("v", value_scale, 0.0)):
            x = scale * (torch.randn(count, kv_heads, BLOCK, dim, generator=g) + offset * torch.randn(dim, generator=g))
            n, s, m = quantise(x)
            setattr(self, name + "_parts", (n, s, m))
            self.__dict__[name + "_host"] = torch.stack([torch.stack([write_block(n[i, h], s[i, h], m[i, h], name == "v") for h in range(kv_heads)])
                                                         for i in range(count)])

    def pools(self, device="cuda"):
        return self.k_host.to(device), self.v_host.to(device)

    def poison(self, name: str, b: int, token: int, head: int, group: int) -> None:
        """One group of one token becomes NaN."""
        block, at = int(self.table[b, token // BLOCK]), token % BLOCK
        n, s, m = getattr(self, name + "_parts")
        s[block, head, at, group], m[block, head, at, group] = math.nan, 0.0
        n[block, head, at, 32 * group:32 * group + 32] = 0
        getattr(self, name + "_host")[block, head] = write_block(n[block, head], s[block, head], m[block, head], name == "v")

    def rows(self, name: str, b: int, head: int, upto: int):
        """(numbers [upto, dim], codes, s, m) of a sequence's tokens."""
        n, s, m = getattr(self, name + "_parts")
        blocks = self.table[b, :-(-upto // BLOCK)].long()
        cut = lambda t: t[blocks, head].flatten(0, 1)[:upto]  # noqa: E731
        return numbers(cut(n), cut(s), cut(m)), cut(n), cut(s), cut(m)


def first_key(pos: int, window: int) -> int:
    return pos - pos % -window if window < 0 else max(0, pos - window + 1) if window > 0 else 0


def attend(cache: Cache, q: torch.Tensor, before, new, heads: int, scale: float, window: int = 0, sinks=None):
    """Float64 [tokens, heads, dim], and for each number what the tolerances are made of: the sum of p (s n + |m|), and the largest sum of the magnitudes that a
    visible key's score is added up from."""
    q = q.double().cpu().view(-1, heads, cache.dim)
    out, weight, reach = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[:2], dtype=torch.float64)
    at = 0
    for b, (have, count) in enumerate(zip(before, new)):
        for h in range(heads):
            kh = h // (heads // cache.kv_heads)
            k, kn, ks, km = cache.rows("k", b, kh, have + count)
            v, vn, vs, vm = cache.rows("v", b, kh, have + count)
            wide = lambda t: t.double().repeat_interleave(32, dim=-1)  # noqa: E731
            size_k, size_v = wide(ks) * kn + wide(km).abs(), wide(vs) * vn + wide(vm).abs()
            for j in range(count):
                pos, row = have + j, at + j
                lo = first_key(pos, window)
                z = (k[lo:pos + 1] @ q[row, h]) * scale
                if sinks is not None:
                    z = torch.cat((z, sinks[h].double().cpu()[None]))
                p = torch.softmax(z, 0)[:pos + 1 - lo]
                out[row, h] = p @ v[lo:pos + 1]
                weight[row, h] = p @ size_v[lo:pos + 1]
                reach[row, h] = (size_k[lo:pos + 1] @ q[row, h].abs()).max() * scale
        at += count
    return out, weight, reach


def choose(logits: torch.Tensor, u: float, temperature: float, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> int:
    """The token of one row, in float64, by sorting; exact sums by math.fsum."""
    x = [(-math.inf if v != v else v) for v in logits.double().tolist()]
    top = max(x)
    if top == -math.inf:
        return 0
    if temperature == 0:
        return x.index(top)
    w = [1.0 if v == top else math.exp((v - top) / temperature) for v in x]
    keep = [j for j in range(len(x)) if x[j] > -math.inf]
    if 0 < top_k < len(x):
        least = sorted(x, reverse=True)[top_k - 1]
        keep = [j for j in keep if x[j] >= least]
    if top_p < 1.0:
        whole = math.fsum(w[j] for j in keep)
        by_value: dict = {}
        for j in keep:
            by_value.setdefault(x[j], []).append(w[j])
        above, edge = 0.0, math.inf
        for value in sorted(by_value, reverse=True):
            if above <= top_p * whole:
                edge = value
            above = math.fsum([above, *by_value[value]])
        keep = [j for j in keep if x[j] >= edge]
    keep = [j for j in keep if w[j] >= min_p]
    target = u * math.fsum(w[j] for j in keep)
    running = 0.0
    for j in keep:
        running = math.fsum((running, w[j]))
        if running > target:
            return j
    return keep[-1]
