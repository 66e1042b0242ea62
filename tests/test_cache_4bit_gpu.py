"""The 4-bit cache on the GPU: appending, reading back and attention against the plain forms in tests/plain_cache_4bit.py, and whole models that keep it.

Tolerances, derived from the kernels' roundings (a rounding is off by at most eps / 2 of its value: bf16 2^-8, fp16 2^-11, float32 2^-24).  Attention over 4 bits:
the output 2^-8 of itself; the weights 2^-11 each, so 2^-11 of the sum of p (s n + |m|) (the second term's 16 bits are less); scores are float32 sums of at
most 4 x (32 + 4) terms, so within 2^-24 * 160 of the terms' magnitudes, of which the exponentials and their sum take twice that and 2^-20 of their own.
Through copies of the blocks in 16 bits, to bfloat16's precision: keys 2^-8, which moves a score by 2^-8 of its terms' magnitudes and the output by twice that
of its own; weights and values 2^-8 each (float16 blocks have bounds of their own, below)."""
from __future__ import annotations

import math

import pytest
import torch

import plain_cache_4bit as plain
from conftest import TINY

pytestmark = pytest.mark.gpu

DEV = "cuda"


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def offsets(new):
    out = [0]
    for count in new:
        out.append(out[-1] + count)
    return out


class Step:
    """A cache that holds `before` tokens of every sequence, and room for the `new` ones."""

    def __init__(self, before, new, kv_heads, dim, seed=0, **cache):
        self.before, self.new, self.kv, self.dim = before, new, kv_heads, dim
        self.totals = [b + c for b, c in zip(before, new)]
        self.cache = plain.Cache([max(1, t) for t in self.totals], kv_heads, dim, seed, **cache)
        self.cu, self.len_before, self.table = ints(offsets(new)), ints(before), self.cache.table.to(DEV)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.n = sum(new)
        self.k_pool, self.v_pool = self.cache.pools()

    def common(self):
        return dict(table=self.table, cu=self.cu, len_before=self.len_before, sequences=len(self.new), status=self.status)


def part_scratch(dim):
    from thintensor_b200.kernels import api

    rows = api.attention_4bit_part_rows()
    return dict(part_acc=torch.full((rows * dim,), math.nan, device=DEV), part_ml=torch.full((rows * 2,), math.nan, device=DEV),
                tickets=torch.zeros(4 * api.sm_count(), dtype=torch.int32, device=DEV))


def run_attention(step, q, heads, window=0, splits=1, one=False, sinks=None, scale=None, out=None, scratch=None):
    from thintensor_b200.kernels import api

    out = torch.full((step.n, heads * step.dim), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
    more = (scratch or part_scratch(step.dim)) if splits == 0 else dict(part_acc=None, part_ml=None)
    api.attention_4bit(q, step.k_pool, step.v_pool, n_tokens=step.n, heads=heads, kv_heads=step.kv, head_dim=step.dim, scale=scale or step.dim ** -0.5, window=window,
                       splits=splits, out=out, one_token_each=one, sinks=sinks, **more, **step.common())
    return out


def queries(step, heads, seed=1, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(step.n, heads * step.dim, generator=g)).bfloat16().to(DEV)


def close_to(got, step, q, heads, window=0, sinks=None, scale=None, expanded=False):
    scale = scale or step.dim ** -0.5
    want, weight, reach = plain.attend(step.cache, q, step.before, step.new, heads, scale, window, sinks)
    if expanded:
        moved = (2.0 ** -8 + 2.0 ** -16) * reach[..., None]
        allowed = 2.0 ** -8 * want.abs() + (torch.expm1(2 * moved) + 3 * 2.0 ** -8) * weight
    else:
        moved = 160 * 2.0 ** -24 * reach[..., None] + 2.0 ** -20
        allowed = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 4 * moved) * weight
    off = (got.double().cpu().view_as(want) - want).abs()
    assert bool((off <= allowed + 1e-30).all()), float((off / (allowed + 1e-30)).max())
    assert int(step.status.item()) == 0


# --------------------------------------------------------------------------------------------------------- appending
def append(step, qkv, heads, rotary, interleaved=False, inv_freq=None, scaling=1.0, n=None, pools=True, q_out=None):
    from thintensor_b200.kernels import api

    n = step.n if n is None else n
    q_out = torch.full((n, heads * step.dim), 7.0, dtype=torch.bfloat16, device=DEV) if q_out is None else q_out
    inv_freq = torch.zeros(64, device=DEV) if inv_freq is None else inv_freq
    api.rope_append_4bit(qkv, inv_freq, rotary, scaling, q_out, step.k_pool if pools else None, step.v_pool if pools else None, n_tokens=n, heads=heads,
                         kv_heads=step.kv, head_dim=step.dim, interleaved=interleaved, **step.common())
    return q_out


SHAPES = [(32, 2, 6), (64, 8, 32), (64, 1, 16), (96, 3, 3), (128, 2, 10), (32, 5, 5), (64, 3, 9)]
RAGGED = [([0], [1]), ([63, 0, 64, 129], [1, 1, 1, 1]), ([0, 61, 5, 127, 200], [3, 7, 1, 2, 130]), ([2, 66, 0], [1, 1, 1]), ([1, 0, 3], [2, 65, 4])]


@pytest.mark.parametrize("dim,kv,heads", SHAPES)
@pytest.mark.parametrize("before,new", RAGGED)
def test_appending_unrotated_vectors_writes_the_defined_bytes(dim, kv, heads, before, new):
    step = Step(before, new, kv, dim, seed=dim + len(new))
    k_old, v_old = step.k_pool.cpu(), step.v_pool.cpu()
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, step.n, (heads + 2 * kv) * dim, generator=g)
    x[0, :, 3::7] *= 40.0
    q = append(step, x.to(DEV), heads, 0)
    assert torch.equal(q.cpu(), x[0, :, :heads * dim].bfloat16())
    k_want, v_want = k_old.clone(), v_old.clone()
    at = 0
    for b, (have, count) in enumerate(zip(before, new)):
        for h in range(kv):
            for name, want, lo in (("k", k_want, heads), ("v", v_want, heads + kv)):
                n, s, m = plain.quantise(x[0, at:at + count, (lo + h) * dim:(lo + h + 1) * dim])
                for w in range(have // 64, -(-(have + count) // 64)):
                    block = int(step.cache.table[b, w])
                    have_n, have_s, have_m = plain.read_block(want[block, h], dim, name == "v")
                    for j in range(count):
                        if (have + j) // 64 == w:
                            t = (have + j) % 64
                            have_n[t], have_s[t], have_m[t] = n[j], s[j], m[j]
                    want[block, h] = plain.write_block(have_n, have_s, have_m, name == "v")
        at += count
    # codes that stood behind a sequence's end, in words that the step began, may be cleared: what a sequence holds is compared
    for name, got, want in (("k", step.k_pool.cpu(), k_want), ("v", step.v_pool.cpu(), v_want)):
        touched = set()
        for b, total in enumerate(step.totals):
            for w in range(-(-total // 64)):
                block = int(step.cache.table[b, w])
                touched.add(block)
                upto = min(64, total - 64 * w)
                for h in range(kv):
                    for a, c in zip(plain.read_block(got[block, h], dim, name == "v"), plain.read_block(want[block, h], dim, name == "v")):
                        assert torch.equal(a[:upto], c[:upto])
        rest = [i for i in range(got.shape[0]) if i not in touched]
        assert torch.equal(got[rest], want[rest])
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("dim,rotary,interleaved", [(64, 64, False), (64, 32, True), (128, 128, False), (128, 128, True), (96, 48, False), (96, 34, False), (32, 30, True),
                                                    (128, 6, False)])
@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("far", [0, 131000])
def test_appending_rotates_by_exact_angles(dim, rotary, interleaved, slices, far):
    heads, kv, before, new = 4, 2, [far, far + 70], [5, 1]
    step = Step([b % 64 for b in before], new, kv, dim)
    width = max(before) // 64 + 2
    table = torch.full((2, width), -1, dtype=torch.int32)
    for b in range(2):
        table[b, before[b] // 64] = step.cache.table[b, 0]
        table[b, before[b] // 64 + 1] = step.cache.table[b, 1] if step.cache.table[b, 1] >= 0 else 0
    step.table, step.len_before = table.to(DEV), ints(before)
    g = torch.Generator().manual_seed(rotary)
    x = torch.randn(slices, step.n, (heads + 2 * kv) * dim, generator=g)
    inv_freq = (10000.0 ** (-torch.arange(0, rotary, 2).double() / rotary)).float()
    q = append(step, x.to(DEV), heads, rotary, interleaved, inv_freq.to(DEV), scaling=1.25)
    rows = x.double().sum(0).view(step.n, -1, dim)
    size = x.double().abs().sum(0).view(step.n, -1, dim)
    position = torch.tensor([b + j for b, c in zip(before, new) for j in range(c)]).double()
    angle = position[:, None, None] * inv_freq.double()
    pairs = lambda t: (t[..., 0:rotary:2], t[..., 1:rotary:2]) if interleaved else (t[..., :rotary // 2], t[..., rotary // 2:rotary])  # noqa: E731
    a, b = pairs(rows)
    ra, rb = 1.25 * (a * angle.cos() - b * angle.sin()), 1.25 * (b * angle.cos() + a * angle.sin())
    turned = rows.clone()
    for part, value in zip(pairs(turned), (ra, rb)):
        part.copy_(value)
    # float32: the slices' sums, sine and cosine (2 ulp and the reduced angle's rounding, 2^-22), two products and their sum
    sa, sb = pairs(size)
    slack = 2.0 ** -24 * (slices + 1) * size
    for part in pairs(slack):
        part.copy_(1.25 * (sa + sb) * 2.0 ** -21)
    want_q, slack_q = turned[:, :heads].flatten(1), slack[:, :heads].flatten(1)
    assert bool(((q.double().cpu() - want_q).abs() <= 2.0 ** -8 * (want_q.abs() + slack_q) + slack_q).all())
    at = 0
    for b, count in enumerate(new):
        for j in range(count):
            pos = before[b] + j
            block, t = int(table[b, pos // 64]), pos % 64
            for h in range(kv):
                for name, pool, lo in (("k", step.k_pool, heads), ("v", step.v_pool, heads + kv)):
                    n, s, m = plain.read_block(pool[block, h], dim, name == "v")
                    got = plain.numbers(n, s, m)[t]
                    exact, soft = (turned if name == "k" else rows)[at + j, lo + h], slack[at + j, lo + h]
                    half = s[t].double().repeat_interleave(32) * (0.5 + 15 * 2.0 ** -22)
                    assert bool(((got - exact).abs() <= half + 2 * soft + 2.0 ** -23 * exact.abs()).all())
        at += count
    assert int(step.status.item()) == 0


def test_appending_queries_alone_and_rows_behind_the_last_sequence():
    step = Step([3, 70], [2, 1], 2, 64)
    x = torch.randn(1, 5, 4 * 64, device=DEV)
    old = step.k_pool.clone(), step.v_pool.clone()
    q = append(step, x, 4, 0, n=5, pools=False)
    assert torch.equal(q[:3], x[0, :3].bfloat16()) and bool((q[3:] == 7.0).all())
    y = torch.randn(1, 5, 8 * 64, device=DEV)
    append(step, y, 4, 0, n=5)
    append_again = step.k_pool.clone()
    step.k_pool.copy_(old[0])
    step.v_pool.copy_(old[1])
    append(step, y[:, :3].contiguous(), 4, 0)
    assert torch.equal(append_again, step.k_pool) and int(step.status.item()) == 0


def test_appending_in_pieces_gives_the_same_cache():
    """Any cut of the tokens: value words are shared by four neighbouring tokens, and whoever comes later keeps what is there."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 150, 8 * 64, generator=g).to(DEV)
    whole = Step([0], [150], 2, 64)
    append(whole, x, 4, 0)
    for cuts in ([1] * 150, [2, 3, 5, 7, 11, 122], [63, 2, 85], [149, 1]):
        step = Step([0], [150], 2, 64)
        done = 0
        for count in cuts:
            step.cu, step.len_before, step.n = ints([0, count]), ints([done]), count
            append(step, x[:, done:done + count].contiguous(), 4, 0)
            done += count
        for b in range(3):
            block = int(step.cache.table[0, b])
            for got, want, values in ((step.k_pool, whole.k_pool, False), (step.v_pool, whole.v_pool, True)):
                for h in range(2):
                    for a, c in zip(plain.read_block(got[block, h], 64, values), plain.read_block(want[block, h], 64, values)):
                        assert torch.equal(a[:150 - 64 * b], c[:150 - 64 * b])


@pytest.mark.parametrize("entry", [-1, 99, 1 << 30])
def test_a_table_entry_outside_the_pool_is_flagged_and_nothing_is_written(entry):
    from thintensor_b200.kernels import api

    step = Step([64, 3], [2, 1], 2, 64)
    step.table[0, 1] = entry
    k_old, v_old = step.k_pool.clone(), step.v_pool.clone()
    x = torch.randn(1, 3, 8 * 64, device=DEV)
    q = append(step, x, 4, 0)
    assert torch.equal(q, x[0, :, :256].bfloat16()) and int(step.status.item()) == api.STATUS_BAD_BLOCK
    mine = int(step.cache.table[1, 0])
    changed = (step.k_pool != k_old).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [mine] and (step.v_pool != v_old).flatten(1).any(1).nonzero().flatten().tolist() == [mine]
    # a position that the table has no entry for
    step.status.zero_()
    step.len_before = ints([64 * step.table.shape[1], 3])
    append(step, x, 4, 0)
    assert int(step.status.item()) == api.STATUS_BAD_BLOCK


# ------------------------------------------------------------------------------------------------------- reading back
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("before,new,window", [([0, 130, 64], [1, 70, 1], 0), ([200, 64, 0], [1, 9, 3], 70), ([129, 300], [60, 1], -64), ([191], [1], 1)])
def test_reading_back(dim, before, new, window):
    from thintensor_b200.kernels import api

    step = Step(before, new, 3, dim, seed=7)
    firsts = [plain.first_key(b, window) // 64 for b in before]
    span = max(-(-t // 64) - f for t, f in zip(step.totals, firsts))
    keys = torch.full((len(new) * span, 3, 64, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    values, named = torch.full((len(new) * span, 3, dim, 64), 7.0, dtype=torch.bfloat16, device=DEV), torch.full_like(step.table, 5)
    for b, f in enumerate(firsts):                                     # given back: never looked at
        step.table[b, :f] = -1
    api.expand_4bit(step.k_pool, step.v_pool, window=window, keys=keys, values=values, table_tmp=named, **step.common())
    for b, total in enumerate(step.totals):
        last = (total - 1) // 64
        for w in range(step.table.shape[1]):
            place = int(named[b, w])
            if not firsts[b] <= w <= last:
                assert place == -1
                continue
            assert place == b * span + w - firsts[b]
            for h in range(3):
                block, upto = int(step.cache.table[b, w]), min(64, total - 64 * w)
                for name, got in (("k", keys[place, h]), ("v", values[place, h].T)):
                    n, s, m = (t[block, h] for t in getattr(step.cache, name + "_parts"))
                    want = plain.numbers(n, s, m).float().bfloat16()
                    want[upto:] = 0
                    assert torch.equal(got.cpu(), want)
        used = last - firsts[b] + 1
        assert bool((keys[b * span + used:(b + 1) * span] == 7.0).all())
    assert int(step.status.item()) == 0
    if span > 1:                                                       # too few places: flagged, and what fits is there
        small = len(new) * (span - 1)
        api.expand_4bit(step.k_pool, step.v_pool, window=window, keys=keys[:small], values=values[:small], table_tmp=named, **step.common())
        assert int(step.status.item()) == api.STATUS_BAD_SHAPE


# ----------------------------------------------------------------------------------------------------------- attention
LENGTHS = [[0], [62, 63, 64, 0, 1], [200, 5, 700, 129], [1500, 90]]


@pytest.mark.parametrize("dim,kv,heads", [(32, 2, 2), (64, 2, 8), (64, 1, 16), (96, 2, 6), (128, 2, 8), (128, 1, 12), (64, 3, 15), (128, 2, 14)])
@pytest.mark.parametrize("before", LENGTHS)
@pytest.mark.parametrize("splits", [1, 3, 8, 0])
def test_decoding(dim, kv, heads, before, splits):
    step = Step(before, [1] * len(before), kv, dim, seed=dim + heads)
    q = queries(step, heads)
    close_to(run_attention(step, q, heads, splits=splits, one=True), step, q, heads)


@pytest.mark.parametrize("window", [1, 63, 64, 65, 300, -1, -64, -100])
@pytest.mark.parametrize("splits", [1, 4, 0])
def test_decoding_with_windows_and_chunks(window, splits):
    step = Step([500, 63, 64, 0, 299], [1] * 5, 2, 64, seed=3)
    for b, have in enumerate(step.before):                             # blocks before the window have been given back
        step.table[b, :plain.first_key(have, window) // 64] = -1
    q = queries(step, 8)
    close_to(run_attention(step, q, 8, window=window, splits=splits, one=True), step, q, 8, window=window)


@pytest.mark.parametrize("dim,kv,heads", [(32, 1, 3), (64, 2, 8), (96, 1, 8), (128, 2, 10), (64, 1, 16), (128, 1, 7)])
@pytest.mark.parametrize("before,new", [([100, 0, 63], [5, 1, 3]), ([0], [70]), ([64, 127, 130, 1], [2, 12, 1, 9])])
@pytest.mark.parametrize("window", [0, 50, -64])
@pytest.mark.parametrize("splits", [1, 2, 0])
def test_several_tokens_a_sequence(dim, kv, heads, before, new, window, splits):
    step = Step(before, new, kv, dim, seed=dim)
    q = queries(step, heads)
    close_to(run_attention(step, q, heads, window=window, splits=splits), step, q, heads, window=window)


@pytest.mark.parametrize("splits", [1, 5, 0])
def test_sequences_without_a_token_and_rows_behind_the_last(splits):
    step = Step([100, 70, 5, 9], [0, 3, 0, 2], 2, 64)
    q = queries(step, 8)
    out = run_attention(step, q, 8, splits=splits)
    close_to(out, step, q, 8)
    more = torch.cat((q, q[:2]))
    step.n = 7
    wide = run_attention(step, more, 8, splits=splits)
    assert torch.equal(wide[:5], out) and bool((wide[5:] == 7.0).all())


@pytest.mark.parametrize("splits", [1, 4, 0])
def test_sinks(splits):
    step = Step([300, 2, 64], [1, 1, 1], 2, 64)
    sinks = torch.tensor([0.0, 5.0, -3.0, 40.0, -40.0, 1.0, 2.0, 0.5], device=DEV)
    q = queries(step, 8)
    close_to(run_attention(step, q, 8, splits=splits, one=True, sinks=sinks), step, q, 8, sinks=sinks)


@pytest.mark.parametrize("q_scale,key_scale,value_scale", [(0.0, 1.0, 1.0), (1e-20, 1.0, 1.0), (30.0, 1.0, 1.0), (1e-3, 1e3, 1.0), (1e10, 1e-10, 1.0), (1.0, 1.0, 1e-15),
                                                           (1.0, 1.0, 1e15), (1.0, 1.0, 1e-6), (1.0, 0.0, 0.0), (1e4, 1e3, 1.0), (1e6, 1e6, 1.0)])
@pytest.mark.parametrize("splits", [1, 0])
def test_numbers_of_any_size(q_scale, key_scale, value_scale, splits):
    step = Step([400, 70], [1, 1], 2, 128, key_scale=key_scale, value_scale=value_scale)
    q = queries(step, 8, scale=q_scale)
    close_to(run_attention(step, q, 8, splits=splits, one=True), step, q, 8)


def test_values_whose_scales_differ_by_many_binades():
    """A group with scales of 2^20 beside one of 2^-10, and blocks whose scales grow along the sequence."""
    step = Step([500], [1], 1, 64)
    n, s, m = step.cache.v_parts
    s[..., 0] *= 2.0 ** 20
    m[..., 0] *= 2.0 ** 20
    for w in range(8):
        block = int(step.cache.table[0, w])
        s[block], m[block] = s[block] * 2.0 ** (3 * w - 10), m[block] * 2.0 ** (3 * w - 10)
    step.cache.v_host = torch.stack([plain.write_block(n[i, 0], s[i, 0], m[i, 0], True)[None] for i in range(n.shape[0])])
    step.k_pool, step.v_pool = step.cache.pools()
    q = queries(step, 4)
    got = run_attention(step, q, 4, one=True)
    want, weight, reach = plain.attend(step.cache, q, step.before, step.new, 4, 64 ** -0.5)
    # weights are float16 down to 2^-29 of the largest weight times the largest scale: that much of the largest is what a small group may be off by as well
    largest = float((s[step.cache.table[0, :8].long()]).max()) * 15
    allowed = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 640 * 2.0 ** -24 * reach[..., None] + 2.0 ** -18) * weight + 2.0 ** -37 * largest
    assert bool(((got.double().cpu().view_as(want) - want).abs() <= allowed).all())


@pytest.mark.parametrize("splits", [1, 8, 0])
def test_what_is_not_a_number_shows_where_it_is_seen_and_nowhere_else(splits):
    step = Step([300, 300, 300, 300], [1] * 4, 2, 64)
    q = queries(step, 8)
    window = 100
    clean = run_attention(step, q, 8, window=window, splits=splits, one=True).clone()
    for name in "kv":
        step.cache.poison(name, 0, 300 - window, 0, 1)                 # the last token before the window, in its first block
        step.cache.poison(name, 0, 10, 1, 0)
    for name in "kv":                                                  # behind the sequence's end, in its last block
        block = int(step.cache.table[0, 4])
        parts = getattr(step.cache, name + "_parts")
        parts[1][block, :, 301 % 64:] = math.nan
        parts[2][block, :, 301 % 64:] = math.inf
        host = getattr(step.cache, name + "_host")
        for h in range(2):
            host[block, h] = plain.write_block(*(t[block, h] for t in parts), name == "v")
    step.k_pool, step.v_pool = step.cache.pools()
    assert torch.equal(run_attention(step, q, 8, window=window, splits=splits, one=True), clean)
    step.cache.poison("k", 1, 250, 0, 1)                               # a key: all numbers of the heads that see it
    step.cache.poison("v", 2, 299, 1, 0)                               # a value: its group of those
    step.k_pool, step.v_pool = step.cache.pools()
    got = run_attention(step, q, 8, window=window, splits=splits, one=True).view(4, 8, 64)
    bad = torch.zeros(4, 8, 64, dtype=torch.bool, device=DEV)
    bad[1, :4] = True
    bad[2, 4:, :32] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean.view(4, 8, 64)[~bad])


@pytest.mark.parametrize("splits", [1, 0])
def test_a_token_that_later_ones_alone_see_is_no_number(splits):
    step = Step([10], [4], 1, 64)
    step.cache.poison("k", 0, 12, 0, 0)
    step.cache.poison("v", 0, 12, 0, 1)
    step.k_pool, step.v_pool = step.cache.pools()
    got = run_attention(step, queries(step, 4), 4, splits=splits).view(4, -1)
    assert torch.isnan(got).all(1).tolist() == [False, False, True, True] and not torch.isnan(got[:2]).any()


def test_one_key_that_is_no_number_and_queries_that_are_none():
    step = Step([0], [1], 1, 64)
    step.cache.poison("k", 0, 0, 0, 0)
    step.k_pool, step.v_pool = step.cache.pools()
    for splits in (1, 2, 0):
        assert torch.isnan(run_attention(step, queries(step, 4), 4, splits=splits, one=True)).all()
    step = Step([100], [1], 1, 64)
    q = queries(step, 4)
    clean = run_attention(step, q, 4, one=True).view(4, 64).clone()
    for value in (math.nan, math.inf):
        poisoned = q.clone()
        poisoned[0, 70] = value
        got = run_attention(step, poisoned, 4, one=True).view(4, 64)
        assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2, 3]], clean[[0, 2, 3]])


@pytest.mark.parametrize("splits", [1, 3, 0])
def test_blocks_outside_the_pool_are_flagged_and_left_out(splits):
    from thintensor_b200.kernels import api

    step = Step([500, 100], [1, 1], 2, 64)
    q = queries(step, 8)
    clean = run_attention(step, q, 8, splits=splits, one=True).clone()
    step.table[0, 3], step.table[0, 5] = -1, 1 << 20
    got = run_attention(step, q, 8, splits=splits, one=True)
    assert int(step.status.item()) == api.STATUS_BAD_BLOCK and torch.isfinite(got).all() and torch.equal(got[1], clean[1])
    step.table[0] = -1
    got = run_attention(step, q, 8, splits=splits, one=True)
    assert not got[0].any() and torch.equal(got[1], clean[1])


def test_even_runs_leave_their_tickets_as_they_found_them():
    scratch = part_scratch(64)
    for before in ([5000], [3000, 9, 2000], [64] * 40, [700] * 3):
        step = Step(before, [1] * len(before), 2, 64)
        q = queries(step, 8)
        first = run_attention(step, q, 8, splits=0, one=True, scratch=scratch).clone()
        assert not scratch["tickets"].any()
        for _ in range(3):                                             # the parts are joined in their order: the same bits
            assert torch.equal(run_attention(step, q, 8, splits=0, one=True, scratch=scratch), first)
        close_to(first, step, q, 8)


def test_offsets_beyond_32_bits():
    """A pool of more than 2^32 bytes whose last blocks are the ones in use."""
    from thintensor_b200.kernels import api

    blocks, kv, dim = 105_000, 8, 128                                  # 40 KB a block of keys: 4.3 GB, and as much for values
    k_pool, v_pool = (torch.zeros((blocks, kv, 40 * dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    step = Step([150], [3], kv, dim)
    names = [blocks - 1, blocks - 2, 0]
    for w, name in enumerate(names):
        k_pool[name], v_pool[name] = step.k_pool[int(step.cache.table[0, w])], step.v_pool[int(step.cache.table[0, w])]
    small = run_attention(step, queries(step, 32), 32).clone()
    x = torch.randn(1, 3, 48 * dim, device=DEV)
    append(step, x, 32, 0)
    after = run_attention(step, queries(step, 32), 32).clone()
    step.k_pool, step.v_pool = k_pool, v_pool
    step.table[0, :3] = ints(names)
    for splits in (1, 0):
        assert torch.equal(run_attention(step, queries(step, 32), 32), small)
    append(step, x, 32, 0)
    assert torch.equal(run_attention(step, queries(step, 32), 32), after)
    keys = torch.zeros((3, kv, 64, dim), dtype=torch.bfloat16, device=DEV)
    values, named = torch.zeros((3, kv, dim, 64), dtype=torch.bfloat16, device=DEV), torch.zeros_like(step.table)
    api.expand_4bit(k_pool, v_pool, window=0, keys=keys, values=values, table_tmp=named, **step.common())
    n, s, m = plain.read_block(k_pool[blocks - 1, 5], dim, False)
    assert torch.equal(keys[0, 5].cpu(), plain.numbers(n, s, m).float().bfloat16())


# -------------------------------------------------------------------------------------------------- the layer's choice
def layer(step, heads, decode, **options):
    from thintensor_b200.cache.cache import RunCache
    from thintensor_b200.engine.context import StepContext, Workspace
    from thintensor_b200.parts import MIXERS

    mixer = MIXERS.build("attention", dict(hidden=heads * step.dim, heads=heads, kv_heads=step.kv, head_dim=step.dim, **options))
    ctx = StepContext(n_tokens=step.n, sequences=len(step.new), decode=decode, max_new=max(step.new), max_total=step.table.shape[1] * 64, tokens=step.cu, cu=step.cu,
                      len_before=step.len_before, slots=step.cu, tables=[step.table], act_dtype=torch.bfloat16,
                      workspace=Workspace(torch.device("cuda", torch.cuda.current_device())), status=step.status)
    return mixer, ctx, RunCache(0, step.k_pool, step.v_pool, True, None)


@pytest.mark.parametrize("dim,kv,heads", [(32, 2, 8), (64, 2, 8), (96, 1, 3), (128, 2, 8)])
@pytest.mark.parametrize("before,new", [([0], [200]), ([70, 0, 129], [90, 33, 64])])
@pytest.mark.parametrize("options", [dict(), dict(window=100), dict(chunk=64)])
def test_prompts_through_expanded_blocks(dim, kv, heads, before, new, options):
    step = Step(before, new, kv, dim)
    mixer, ctx, cache = layer(step, heads, False, **options)
    reach = mixer.reach
    for b, have in enumerate(before):
        step.table[b, :plain.first_key(have, reach) // 64] = -1
    q = queries(step, heads)
    for copies in (True, False):                                       # both ways that a prompt of this size could go
        mixer.expands_4bit = lambda ctx, width: copies  # noqa: B023
        out = torch.full_like(q, 7.0)
        mixer.attend(ctx, q, cache, step.table, out)
        close_to(out, step, q, heads, window=reach, expanded=copies)


def expanded(step, window=0, fill=7.0):
    """The step's blocks as float16 numbers with scales and marks, and the table that names them."""
    from thintensor_b200.kernels import api

    places = len(step.new) * step.table.shape[1]
    keys = torch.full((places, step.kv, 64, step.dim), fill, dtype=torch.float16, device=DEV)
    values, named = torch.full((places, step.kv, step.dim, 64), fill, dtype=torch.float16, device=DEV), torch.full_like(step.table, 5)
    scales, marks = torch.full((2, places, step.kv), 1.0, device=DEV), torch.zeros((places, step.kv, 64), dtype=torch.uint8, device=DEV)
    api.expand_4bit(step.k_pool, step.v_pool, window=window, keys=keys, values=values, table_tmp=named, scales=scales, marks=marks, **step.common())
    return keys, values, scales, marks, named


def run_half(step, q, heads, window=0, sinks=None, out=None, n=None, fill=7.0):
    from thintensor_b200.kernels import api

    keys, values, scales, marks, named = expanded(step, window, fill)
    out = torch.full_like(q, 7.0) if out is None else out
    api.attention_half(q, keys, values, scales, marks, n_tokens=n or q.shape[0], heads=heads, kv_heads=step.kv, head_dim=step.dim, scale=step.dim ** -0.5, window=window,
                       out=out, sinks=sinks, **(step.common() | dict(table=named)))
    return out


def close_to_half(got, step, q, heads, window=0, sinks=None):
    """Output 2^-8; keys 2^-11, which moves a score by that much of its terms' magnitudes and the output by twice that of its own, with the float32 sums'
    2^-16 beside it; weights, values and their sum 2^-11 each; a weight, kept
    2^7 times as large, under float16's 2^-14 by 2^-25, which beside a value scaled by 2^8k less (at least 2^7 in size) is 2^-24 of the largest value."""
    want, weight, reach = plain.attend(step.cache, q, step.before, step.new, heads, step.dim ** -0.5, window, sinks)
    moved = (2.0 ** -11 + 2.0 ** -16) * reach[..., None]
    largest = max(float((s.double() * 15).nan_to_num(0.0).abs().max() + m.double().nan_to_num(0.0).abs().max()) for _, s, m in [step.cache.v_parts])
    allowed = 2.0 ** -8 * want.abs() + (torch.expm1(2 * moved) + 3 * 2.0 ** -11) * weight + max(step.totals) * 2.0 ** -24 * largest
    off = (got.double().cpu().view_as(want) - want).abs()
    assert bool((off <= allowed + 1e-30).all()), float((off / (allowed + 1e-30)).max())
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("before,new,window", [([0, 130, 64], [1, 70, 1], 0), ([200, 64, 0], [1, 9, 3], 70), ([129, 300], [60, 1], -64)])
@pytest.mark.parametrize("key_scale,value_scale", [(1.0, 1.0), (1e30, 1e-30), (0.0, 3e4)])
def test_reading_back_float16_and_scales(dim, before, new, window, key_scale, value_scale):
    step = Step(before, new, 3, dim, seed=7, key_scale=key_scale, value_scale=value_scale)
    step.cache.poison("v", 0, step.totals[0] - 1, 1, 0)
    step.k_pool, step.v_pool = step.cache.pools()
    keys, values, scales, marks, named = expanded(step, window)
    assert bool((scales[0] > 0).all()) and bool((torch.frexp(scales).mantissa.abs() == 0.5).all())
    for b, total in enumerate(step.totals):
        for w in range(plain.first_key(before[b], window) // 64, (total - 1) // 64 + 1):
            place, block, upto = int(named[b, w]), int(step.cache.table[b, w]), min(64, total - 64 * w)
            for h in range(3):
                for i, (name, got) in enumerate((("k", keys[place, h]), ("v", values[place, h].T))):
                    n, s, m = (t[block, h] for t in getattr(step.cache, name + "_parts"))
                    want = plain.numbers(n, s, m)
                    bad = torch.isnan(want)
                    want[bad] = 0
                    want[upto:] = 0
                    scale = float(scales[i, place, h])
                    off = (got.double().cpu() * abs(scale) - want).abs()
                    # 11 bits, after a float32 multiply-add; under 2^-14 half of float16's last place
                    assert bool((off <= (2.0 ** -11 + 2.0 ** -23) * want.abs() + 2.0 ** -25 * abs(scale)).all())
                    if name == "v":
                        mark = torch.stack([bad[:, 32 * g] for g in range(dim // 32)], 1)
                        mark[upto:] = False
                        assert (scale < 0) == bool(mark.any())
                        if scale < 0:
                            assert torch.equal(marks[place, h].cpu().long(), (mark.long() << torch.arange(dim // 32)).sum(1))
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("dim,kv,heads", [(32, 2, 2), (64, 2, 8), (64, 3, 15), (96, 2, 6), (96, 1, 16), (128, 2, 8), (128, 1, 12), (128, 2, 14), (32, 1, 16)])
@pytest.mark.parametrize("before,new", [([0], [1]), ([62, 0, 64, 5], [3, 130, 1, 0]), ([200, 0, 700], [17, 0, 33]), ([63], [300])])
@pytest.mark.parametrize("window", [0, 1, 70, -64])
def test_attention_over_float16_blocks(dim, kv, heads, before, new, window):
    step = Step(before, new, kv, dim, seed=dim + heads)
    for b, have in enumerate(before):
        step.table[b, :plain.first_key(have, window) // 64] = -1
    q = queries(step, heads)
    more = torch.cat((q, q[:1]))                                       # a row behind the last sequence
    got = run_half(step, more, heads, window=window)
    close_to_half(got[:step.n], step, q, heads, window=window)
    assert bool((got[step.n:] == 7.0).all())
    # what stands in places that no block fills is never part of an output
    assert torch.equal(run_half(step, q, heads, window=window, fill=math.nan), got[:step.n])


@pytest.mark.parametrize("dim", [64, 96])
@pytest.mark.parametrize("q_scale,key_scale,value_scale", [(0.0, 1.0, 1.0), (1e-20, 1.0, 1.0), (30.0, 1.0, 1.0), (1e-3, 1e3, 1.0), (1e10, 1e-10, 1.0), (1.0, 1.0, 1e-15),
                                                           (1.0, 1.0, 1e15), (1.0, 1.0, 1e-6), (1.0, 0.0, 0.0), (1e30, 1e-30, 1e5), (1e-30, 1e30, 1e30), (1e-35, 1e-3, 1e-30), (1e4, 1e3, 1.0),
                                                           (1e6, 1e6, 1.0)])
def test_float16_blocks_of_any_size(dim, q_scale, key_scale, value_scale):
    step = Step([300, 70], [40, 3], 2, dim, key_scale=key_scale, value_scale=value_scale)
    q = queries(step, 8, scale=q_scale)
    close_to_half(run_half(step, q, 8), step, q, 8)


def test_float16_blocks_whose_scales_differ():
    """Keys and values that grow by 2^3 from block to block, and rows of queries by 2^5 from token to token."""
    for names, ways in (("k", (1, -1)), ("v", (1, -1)), ("kv", (1,))):
        for way in ways:
            step = Step([500], [20], 1, 64)
            for name in names:
                n, s, m = getattr(step.cache, name + "_parts")
                for w in range(9):
                    block, factor = int(step.cache.table[0, w]), 2.0 ** (way * (3 * w - 18))
                    s[block], m[block] = s[block] * factor, m[block] * factor
                setattr(step.cache, name + "_host", torch.stack([plain.write_block(n[i, 0], s[i, 0], m[i, 0], name == "v")[None] for i in range(n.shape[0])]))
            step.k_pool, step.v_pool = step.cache.pools()
            q = queries(step, 4) * (2.0 ** (5.0 * torch.arange(20, device=DEV) - 80))[:, None].bfloat16()
            close_to_half(run_half(step, q, 4), step, q, 4)


def test_float16_blocks_with_sinks():
    step = Step([300, 2, 64], [10, 30, 1], 2, 64)
    sinks = torch.tensor([0.0, 5.0, -3.0, 40.0, -40.0, 1.0, 2.0, 0.5], device=DEV)
    q = queries(step, 8)
    close_to_half(run_half(step, q, 8, sinks=sinks), step, q, 8, sinks=sinks)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_what_is_not_a_number_in_a_prompt(dim):
    step = Step([300, 20, 0], [30, 100, 5], 2, dim)
    q = queries(step, 8)
    window = 100
    clean = run_half(step, q, 8, window=window).clone()
    step.cache.poison("v", 0, 300 - window, 0, 0)                      # before the first row's window, in its first block
    step.cache.poison("k", 0, 300 - window, 1, 0)
    step.cache.poison("v", 1, 60, 1, dim // 32 - 1)                    # seen by its own token and the 99 after it
    step.cache.poison("k", 1, 90, 0, 0)
    step.k_pool, step.v_pool = step.cache.pools()
    q[132] = q[132].clone()
    q[132, 3 * dim + 5] = math.inf                                     # the third sequence's third token, its fourth head
    got = run_half(step, q, 8, window=window).view(-1, 8, dim)
    bad = torch.zeros_like(got, dtype=torch.bool)
    position = torch.arange(20, 120, device=DEV)
    bad[30:130, 4:, dim - 32:] = ((position >= 60) & (position < 160))[:, None, None]
    bad[30:130, :4] |= (position >= 90)[:, None, None]
    bad[132, 3] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean.view_as(got)[~bad])
    assert int(step.status.item()) == 0


def test_float16_blocks_outside_the_places_are_flagged():
    from thintensor_b200.kernels import api

    step = Step([100], [50], 2, 64)
    step.table[0, 1] = 1 << 20
    run_half(step, queries(step, 8), 8)
    assert int(step.status.item()) == api.STATUS_BAD_BLOCK


def test_a_table_too_narrow_for_the_lengths_is_flagged():
    from thintensor_b200.kernels import api

    step = Step([10], [300], 2, 64)
    q = queries(step, 8)
    keys, values, scales, marks, named = expanded(step)
    padded = torch.full((4, 2), 1 << 20, dtype=torch.int32, device=DEV)      # what lies behind the row is never taken for a block
    padded[0] = named[0, :2]
    api.attention_half(q, keys, values, scales, marks, n_tokens=step.n, heads=8, kv_heads=2, head_dim=64, scale=0.125, window=0, out=torch.empty_like(q),
                       **(step.common() | dict(table=padded[:1])))
    assert int(step.status.item()) == api.STATUS_BAD_BLOCK


def test_tensors_of_another_device_are_refused(monkeypatch):
    from thintensor_b200.kernels import api

    step = Step([10], [20], 2, 64)
    q, blocks = queries(step, 8), expanded(step)
    logits = torch.randn(2, 100, device=DEV)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    calls = [lambda: append(step, torch.empty(1, 20, 12 * 64, device=DEV), 8, 0), lambda: run_attention(step, q, 8), lambda: expanded(step),
             lambda: api.attention_half(q, *blocks[:4], n_tokens=20, heads=8, kv_heads=2, head_dim=64, scale=0.125, window=0, out=torch.empty_like(q),
                                        **(step.common() | dict(table=blocks[4]))),
             lambda: api.sample_filtered(logits, 1.0, 0, 1.0, 0.0, torch.empty(2, dtype=torch.int32, device=DEV), uniform=torch.zeros(2, device=DEV))]
    for call in calls:
        with pytest.raises(api.KernelError, match="the current device is cuda:1"):
            call()


def test_prompts_captured_and_replayed_for_other_lengths():
    step = Step([170, 90], [40, 60], 2, 96)
    mixer, ctx, cache = layer(step, 8, False)
    mixer.expands_4bit = lambda ctx, width: True
    q = queries(step, 8)
    out = torch.full_like(q, 7.0)
    mixer.attend(ctx, q, cache, step.table, out)
    close_to_half(out, step, q, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mixer.attend(ctx, q, cache, step.table, out)
    for before in ([1, 70], [0, 0], [170, 90]):
        step.before, step.totals = before, [before[0] + 40, before[1] + 60]
        step.len_before.copy_(ints(before))
        out.fill_(7.0)
        graph.replay()
        close_to_half(out, step, q, 8)


def test_which_way_a_step_goes():
    step = Step([0], [100], 2, 64)
    mixer, ctx, cache = layer(step, 8, False)
    ctx.n_tokens = 4096
    assert mixer.expands_4bit(ctx, 4) and mixer.span_4bit(ctx, 4) == 4
    assert not mixer.expands_4bit(ctx, 1 << 24)                        # copies that would not fit their scratch memory
    ctx.n_tokens = 15
    assert not mixer.expands_4bit(ctx, 4)
    windowed, ctx, _ = layer(step, 8, False, window=100)
    assert windowed.span_4bit(ctx, 1000) == (100 + 100 - 1 + 62) // 64 + 1
    ctx.n_tokens, ctx.decode = 4096, True
    assert not windowed.expands_4bit(ctx, 4)


@pytest.mark.parametrize("before", [[30000], [9000] * 4, [100] * 3])
def test_decoding_through_the_layer(before):
    step = Step(before, [1] * len(before), 2, 64)
    mixer, ctx, cache = layer(step, 8, True)
    q = queries(step, 8)
    out = torch.full_like(q, 7.0)
    mixer.attend(ctx, q, cache, step.table, out)
    close_to(out, step, q, 8)
    # captured once, replayed for other lengths
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mixer.attend(ctx, q, cache, step.table, out)
    for cut in (0, 1, 65):
        step.before = [max(0, b - cut) for b in before]
        step.len_before.copy_(ints(step.before))
        out.fill_(7.0)
        graph.replay()
        close_to(out, step, q, 8)


def test_a_stream_of_its_own():
    step = Step([700, 64], [1, 1], 2, 64)
    q = queries(step, 8)
    want = run_attention(step, q, 8, splits=0, one=True).clone()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = [run_attention(step, q, 8, splits=s, one=True) for s in (0, 1, 4)]
    stream.synchronize()
    assert torch.equal(got[0], want)
    close_to(got[1], step, q, 8)
    close_to(got[2], step, q, 8)


# --------------------------------------------------------------------------------------------------------- whole models
def cosines(a, b):
    return torch.nn.functional.cosine_similarity(a.double(), b.double(), dim=-1)


@pytest.mark.parametrize("name", ["b", "d", "e"])
def test_models_that_keep_4_bits(tmp_path, name):
    """Prompts, drafts and single tokens of one sequence, and batches, see one and the same cache; it takes 5 / 16 of the plain one's memory; and what comes
    out is what the plain cache gives but for 4 bits' error: keys and values off by at most s / 2 = 1/30 of their group's range, 0.02 of a unit normal
    vector's length in the mean (1 / (sqrt(12) 15) of 4.1 standard deviations: 0.08 of each number), which leaves the attention's part of a residual stream, and
    so the logits, at a cosine of 0.99 and more."""
    import thintensor_b200
    from thintensor_b200 import Entry

    thintensor_b200.save_random_model(tmp_path, TINY[name], seed=1)
    four, full = thintensor_b200.load_model(tmp_path, cache="4bit"), thintensor_b200.load_model(tmp_path)
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, TINY[name]["vocab_size"], (150,), generator=g).tolist()

    def run(runtime, cuts):
        engine = runtime.new_engine(max_tokens=512, max_sequences=2)
        slot, out, done = engine.open(), [], 0
        for count in cuts:
            out.append(engine.step([Entry(slot, tokens[done:done + count], list(range(count)))]).clone())
            done += count
        engine.check_status()
        return torch.cat(out), engine

    whole, engine = run(four, [150])
    plain_logits, plain_engine = run(full, [150])
    assert engine.cache.bytes() * 16 == plain_engine.cache.bytes() * 5
    assert float(cosines(whole, plain_logits).min()) > 0.99
    for cuts in ([100, 5, 5, 40], [70, *[1] * 80], [7, 143]):
        assert float(cosines(run(four, cuts)[0], whole).min()) > 0.999
    prompts = [tokens[:90], tokens[:3], tokens[20:81]]
    alone = [four.generate([p], max_new_tokens=12, stop_ids=(), temperature=0.7, min_p=0.05, seed=3)[0] for p in prompts[:1]]
    for graph in (True, False):
        got = four.generate(prompts, max_new_tokens=12, stop_ids=(), temperature=0.7, min_p=0.05, seed=3, use_graph=graph)
        assert [len(x) for x in got] == [12, 12, 12] and all(0 <= t < TINY[name]["vocab_size"] for x in got for t in x)
    assert len(alone[0]) == 12


def test_the_command_line_keeps_4_bits(tmp_path, capsys):
    import json

    import thintensor_b200
    from thintensor_b200 import cli

    thintensor_b200.save_random_model(tmp_path, TINY["d"], seed=1)
    assert cli.main(["run", str(tmp_path), "--prompt-token-ids", "1,2,3", "--max-new-tokens", "5", "--cache", "4bit", "--temperature", "0.8", "--min-p", "0.1", "--ignore-eos",
                     "--json"]) == 0
    report = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert report["cache"] == "4bit" and report["min_p"] == 0.1 and len(report["generated_token_ids"][0]) == 5
    assert cli.main(["bench", str(tmp_path), "--cache", "4bit", "--steps", "4", "--warmup", "2", "--prompt-len", "80", "--json"]) == 0
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["cache"] == "4bit"
    assert cli.main(["validate", str(tmp_path), "--cache", "4bit", "--length", "40", "--json"]) in (0, 1)
    assert json.loads(capsys.readouterr().out.strip().splitlines()[-1])["modes"]["whole"]["cosine_similarity"] > 0.99
    assert cli.main(["run", str(tmp_path), "--prompt-token-ids", "1,2", "--cache", "4bit", "--dtype", "fp32"]) == 2
    assert "4 bits" in capsys.readouterr().err


def test_even_runs_on_two_streams_at_once_with_scratch_of_their_own():
    steps = [Step([9000], [1], 2, 64, seed=1), Step([3000, 7000], [1, 1], 2, 64, seed=2)]
    inputs = [queries(step, 8) for step in steps]
    scratch = [part_scratch(64) for _ in steps]
    want = [run_attention(step, q, 8, splits=0, one=True).clone() for step, q in zip(steps, inputs)]
    outs = [torch.full_like(w, 7.0) for w in want]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                run_attention(steps[i], inputs[i], 8, splits=0, one=True, scratch=scratch[i], out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and not any(s["tickets"].any() for s in scratch)


def test_the_same_scratch_for_steps_of_other_shapes():
    """A layer's workspace serves prompts and decoding in turn, captured steps among them."""
    mixers = []
    for before, new in (([170, 90], [40, 60]), ([9000], [1]), ([64] * 3, [30, 2, 1])):
        step = Step(before, new, 2, 64)
        mixer, ctx, cache = layer(step, 8, all(n == 1 for n in new))
        mixers.append((step, mixer, ctx, cache, queries(step, 8)))
    shared = mixers[0][2].workspace
    graphs = []
    for copies in (True, False):
        for step, mixer, ctx, cache, q in mixers:
            ctx.workspace = shared
            if not ctx.decode:
                mixer.expands_4bit = lambda ctx, width: copies  # noqa: B023
            out = torch.full_like(q, 7.0)
            mixer.attend(ctx, q, cache, step.table, out)
    for copies in (True, False):
        for step, mixer, ctx, cache, q in mixers:
            if not ctx.decode:
                mixer.expands_4bit = lambda ctx, width: copies  # noqa: B023
            out, graph = torch.full_like(q, 7.0), torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                mixer.attend(ctx, q, cache, step.table, out)
            graphs.append((graph, out, step, q, copies and not ctx.decode))
    for graph, out, step, q, copies in graphs + graphs[::-1]:
        out.fill_(7.0)
        graph.replay()
        (close_to_half if copies else close_to)(out, step, q, 8)
