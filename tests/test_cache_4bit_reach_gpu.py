"""What a query does not see, or hardly weighs, leaves its output alone: sizes of other tokens' keys and values in the same block, in other blocks and in the same
tile of query rows.

The tolerances are those of test_cache_4bit_gpu.py, made of what the row itself sees."""
from __future__ import annotations

import math

import pytest
import torch

import plain_cache_4bit as plain
from test_cache_4bit_gpu import Step, close_to, layer, queries, run_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"


def rewrite(step, name):
    """The pool's bytes from the codes, scales and least values as they now are."""
    n, s, m = getattr(step.cache, name + "_parts")
    setattr(step.cache, name + "_host", torch.stack([torch.stack([plain.write_block(n[i, h], s[i, h], m[i, h], name == "v") for h in range(step.kv)])
                                                     for i in range(n.shape[0])]))
    step.k_pool, step.v_pool = step.cache.pools()


def enlarge(step, name, b, token, factor):
    """All heads' numbers of one token times a power of two."""
    _, s, m = getattr(step.cache, name + "_parts")
    block, at = int(step.cache.table[b, token // 64]), token % 64
    s[block, :, at] *= factor
    m[block, :, at] *= factor
    rewrite(step, name)


def turn_away(step, b, token, size):
    """The token's keys are -size in every number: queries of positive numbers hardly weigh it."""
    n, s, m = step.cache.k_parts
    block, at = int(step.cache.table[b, token // 64]), token % 64
    n[block, :, at], s[block, :, at], m[block, :, at] = 0, 1.0, -size
    rewrite(step, "k")


def close_to_own(got, step, q, heads, window=0, copied=False, sinks=None):
    """Every row by what it sees itself.  A score is off by `moved` of the magnitudes that it is added up from, its weight by twice that of itself (the maximum moves
    as well), and so every key counts by its own weight in the output's sum and in the sum of weights.

    Over 4 bits: scores within 160 float32 roundings and 2^-20; weights 2^-11, and a weight under float16's 2^-14 by 2^-25, 2^-39 of the row's largest weight
    times scale.  Over copies: keys 2^-11 of themselves and 2^-24 of their token's largest number (float16's smallest step beside a largest number of at least 2^-1),
    float32 sums 2^-16; weights, values and the sum 2^-11 each; a weight under 2^-14 by 2^-25 times a value of at most 2^15, where the row's largest weight is at least 2^7 and
    that token's largest number at least 2^-1: 2^-16 of the largest product.  The output 2^-8."""
    rows, scale = q.double().cpu().view(-1, heads, step.dim), step.dim ** -0.5
    got, at = got.double().cpu().view_as(rows), 0
    for b, (have, count) in enumerate(zip(step.before, step.new)):
        for h in range(heads):
            kh = h // (heads // step.kv)
            wide = lambda t: t.double().repeat_interleave(32, dim=-1)  # noqa: E731
            k, kn, ks, km = step.cache.rows("k", b, kh, have + count)
            v, vn, vs, vm = step.cache.rows("v", b, kh, have + count)
            k_size, v_size = wide(ks) * kn + wide(km).abs(), wide(vs) * vn + wide(vm).abs()
            for j in range(count):
                seen, row = slice(plain.first_key(have + j, window), have + j + 1), rows[at + j, h]
                z = (k[seen] @ row) * scale
                if sinks is not None:
                    z = torch.cat((z, sinks[h].double().cpu()[None]))
                p = torch.softmax(z, 0)[:z.numel() - (sinks is not None)]
                want, weight = p @ v[seen], p @ v_size[seen]
                reach = (k_size[seen] @ row.abs()) * scale
                if copied:
                    moved = (2.0 ** -11 + 2.0 ** -16) * reach + 2.0 ** -24 * k[seen].abs().amax(1) * row.abs().sum() * scale
                    least, fixed = 2.0 ** -16 * (p * v[seen].abs().amax(1)).max(), 3 * 2.0 ** -11
                else:
                    moved = 160 * 2.0 ** -24 * reach + 2.0 ** -20
                    least, fixed = 2.0 ** -39 * 16 * (p * vs[seen].amax(1)).max(), 2.0 ** -11
                off = p * torch.expm1((2 * moved).clamp_max(500.0))
                allowed = 2.0 ** -8 * want.abs() + fixed * weight + off @ v_size[seen] + off.sum() * weight + len(p) * least
                found = (got[at + j, h] - want).abs()
                assert bool((found <= allowed + 1e-30).all()), (b, h, j, float((found / (allowed + 1e-30)).max()))
        at += count
    assert int(step.status.item()) == 0


# -------------------------------------------------------------------------------------------- attention over 4 bits
@pytest.mark.parametrize("dim,kv,heads", [(32, 2, 2), (64, 2, 8), (96, 1, 8), (128, 2, 10), (128, 1, 16)])
@pytest.mark.parametrize("token", [62, 66, 70])                         # in the block of what the rows before it see, and in the next one
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 34, 2.0 ** 100])
@pytest.mark.parametrize("splits", [1, 2, 0])
def test_a_value_that_later_tokens_alone_see(dim, kv, heads, token, factor, splits):
    step = Step([60, 5], [12, 3], kv, dim, seed=dim + heads)
    enlarge(step, "v", 0, token, factor)
    q = queries(step, heads)
    close_to_own(run_attention(step, q, heads, splits=splits), step, q, heads)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("group", [1, 4, 16])
@pytest.mark.parametrize("token", [3, 199, 140])
@pytest.mark.parametrize("factor", [2.0 ** 40, 2.0 ** 70, 2.0 ** 110])
@pytest.mark.parametrize("splits", [1, 3, 0])
def test_a_value_of_little_weight(dim, group, token, factor, splits):
    """Weights of e^-100 to e^-400 beside values of 2^40 to 2^110."""
    step = Step([200, 90], [1, 1], 2, dim, seed=dim)
    turn_away(step, 0, token, 32.0)
    enlarge(step, "v", 0, token, factor)
    q = queries(step, 2 * group).abs()
    close_to_own(run_attention(step, q, 2 * group, splits=splits, one=True), step, q, 2 * group)


@pytest.mark.parametrize("splits", [1, 0])
def test_a_value_that_is_no_number_counts_however_little_it_weighs(splits):
    """A weight that is zero in float32 times NaN is NaN wherever the row sees the value: in its last block as in those before it."""
    for token in (130, 20):
        step = Step([140], [1], 2, 64)
        turn_away(step, 0, token, 32.0)
        step.cache.poison("v", 0, token, 1, 0)
        step.k_pool, step.v_pool = step.cache.pools()
        got = run_attention(step, queries(step, 8).abs(), 8, splits=splits, one=True).view(8, 64)
        bad = torch.zeros_like(got, dtype=torch.bool)
        bad[4:, :32] = True
        assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("splits", [1, 4, 0])
def test_sinks_of_minus_infinity_are_none(splits):
    """Also for rows that see no key in a slice: of several tokens with a window the last ones start behind the first slice."""
    step = Step([895, 70], [8, 2], 2, 64)
    q = queries(step, 8)
    sinks = torch.tensor([-math.inf, 1.0, -math.inf, 0.0, -math.inf, 2.0, -math.inf, -math.inf], device=DEV)
    for window in (0, 60, 2):
        close_to(run_attention(step, q, 8, window=window, splits=splits, sinks=sinks), step, q, 8, window=window, sinks=sinks)


# ----------------------------------------------------------------------------------------------- prompts over copies
def copies(step, window=0):
    """The step's blocks as float16 numbers with scales and marks, and the table that names them."""
    from thintensor_b200.kernels import api

    places = len(step.new) * step.table.shape[1]
    keys = torch.full((places, step.kv, 64, step.dim), math.nan, dtype=torch.float16, device=DEV)
    values, named = torch.full((places, step.kv, step.dim, 64), math.nan, dtype=torch.float16, device=DEV), torch.full_like(step.table, 5)
    scales, marks = torch.full((2, places, step.kv), 1.0, device=DEV), torch.full((places, step.kv, 64), 255, dtype=torch.uint8, device=DEV)
    api.expand_4bit(step.k_pool, step.v_pool, window=window, keys=keys, values=values, table_tmp=named, scales=scales, marks=marks, **step.common())
    return keys, values, scales, marks, named


def run_prompt(step, q, heads, window=0, sinks=None):
    from thintensor_b200.kernels import api

    keys, values, scales, marks, named = copies(step, window)
    out = torch.full_like(q, 7.0)
    api.attention_half(q, keys, values, scales, marks, n_tokens=q.shape[0], heads=heads, kv_heads=step.kv, head_dim=step.dim, scale=step.dim ** -0.5, window=window,
                       out=out, sinks=sinks, **(step.common() | dict(table=named)))
    return out


@pytest.mark.parametrize("dim,kv,heads", [(32, 2, 2), (64, 2, 8), (96, 1, 8), (128, 2, 10), (128, 1, 16)])
@pytest.mark.parametrize("token", [62, 66, 85])
@pytest.mark.parametrize("factor", [2.0 ** 12, 2.0 ** 20, 2.0 ** 34, 2.0 ** 100])
@pytest.mark.parametrize("names", ["v", "k", "kv"])
def test_prompts_and_what_later_tokens_alone_see(dim, kv, heads, token, factor, names):
    step = Step([60, 5], [30, 20], kv, dim, seed=dim + heads)
    for name in names:
        enlarge(step, name, 0, token, factor)
    q = queries(step, heads)
    close_to_own(run_prompt(step, q, heads), step, q, heads, copied=True)


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("group", [1, 6])
@pytest.mark.parametrize("token", [3, 140, 199])
@pytest.mark.parametrize("factor", [2.0 ** 40, 2.0 ** 70, 2.0 ** 110])
def test_prompts_and_a_value_of_little_weight(dim, group, token, factor):
    step = Step([200, 90], [24, 3], 2, dim, seed=dim)
    turn_away(step, 0, token, 32.0)
    enlarge(step, "v", 0, token, factor)
    q = queries(step, 2 * group).abs()
    close_to_own(run_prompt(step, q, 2 * group), step, q, 2 * group, copied=True)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("names", ["v", "k", "kv"])
@pytest.mark.parametrize("shrunk", [1.0, 2.0 ** -30])
def test_prompts_with_a_large_token_beside_one_that_is_no_number(dim, names, shrunk):
    """The block's tokens have powers of two of their own and groups that are not numbers at once; where the token that is none is itself small, too."""
    step = Step([60], [30], 2, dim, seed=dim)
    for name in names:
        enlarge(step, name, 0, 85, 2.0 ** 34)
        if shrunk != 1.0:
            enlarge(step, name, 0, 75, shrunk)
    step.cache.poison("v", 0, 75, 1, 0)
    step.k_pool, step.v_pool = step.cache.pools()
    heads = 8
    q = queries(step, heads)
    got = run_prompt(step, q, heads).view(30, heads, dim)
    small = dim > 32 and "k" in names                                  # a small token then is not a number as a whole
    for j in range(30):
        seen = 60 + j >= 75
        bad = torch.isnan(got[j])
        assert bool(bad[4:, :32].all()) == seen and not bool(bad[:4].any())
        assert bool(bad[4:].any()) == seen
        assert bool(bad[4:, 32:].all()) == seen if small else not bool(bad[4:, 32:].any())
    clean = Step([60], [15], 2, dim, seed=dim)
    clean.cache = step.cache
    close_to_own(got[:15].reshape(15, -1), clean, q[:15], heads, copied=True)


@pytest.mark.parametrize("dim", [32, 96, 128])
@pytest.mark.parametrize("factors", [dict(k=2.0 ** 9), dict(v=2.0 ** 9), dict(k=2.0 ** 40, v=2.0 ** 12), dict(k=2.0 ** -30), dict(v=2.0 ** -120), dict(k=2.0 ** 60, v=2.0 ** 60)])
@pytest.mark.parametrize("bad", [False, True])
def test_reading_back_blocks_of_unlike_tokens(dim, factors, bad):
    """float16 times the block's power of two and 2^-8 for each step of the token; the marks' two readings as documented."""
    step = Step([100], [3], 2, dim, seed=3)
    for name, factor in factors.items():
        enlarge(step, name, 0, 70, factor)
        enlarge(step, name, 0, 102, 0.0)
    if bad:
        step.cache.poison("v", 0, 80, 1, dim // 32 - 1)
        step.k_pool, step.v_pool = step.cache.pools()
    keys, values, scales, marks, named = copies(step)
    for w in (0, 1):
        place, block, upto = int(named[0, w]), int(step.cache.table[0, w]), min(64, 103 - 64 * w)
        for h in range(2):
            k_scale, v_scale, byte = float(scales[0, place, h]), float(scales[1, place, h]), marks[place, h].cpu().long()
            low, high = (byte & 15, byte >> 4) if k_scale < 0 or v_scale < 0 else (torch.zeros(64, dtype=torch.long),) * 2
            if k_scale < 0:
                none = high == 15
                mask, k_step, v_step = torch.where(none, low, 0), torch.where(none, 0, low), torch.where(none, 0, high)
            else:
                mask, k_step, v_step = low, torch.zeros_like(low), high
            for name, got, scale, steps in (("k", keys[place, h], k_scale, k_step), ("v", values[place, h].T, v_scale, v_step)):
                n, s, m = (t[block, h] for t in getattr(step.cache, name + "_parts"))
                want = plain.numbers(n, s, m)[:upto]
                gone = torch.isnan(want)
                whole = (k_scale < 0) & (mask[:upto] == 15)            # a small token with a group that is no number
                if name == "v":
                    assert bool((gone.any(1) | ~whole).all())
                    marked = torch.stack([(mask[:upto] >> g & 1).bool() for g in range(dim // 32)], 1)
                    assert torch.equal(marked, gone[:, ::32] | whole[:, None])
                gone = gone | whole[:, None]
                off = (got.double().cpu()[:upto] * (abs(scale) * 2.0 ** (-8.0 * steps[:upto].double()))[:, None] - want).abs()
                largest = want.nan_to_num(0.0).abs().amax(1, keepdim=True)
                assert bool(((off <= (2.0 ** -11 + 2.0 ** -23) * want.abs() + 2.0 ** -24 * largest + 1e-45) | gone).all())
                assert bool((got.cpu()[upto:] == 0).all())
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_prompts_give_the_same_bits_every_time(dim):
    """More tiles than the GPU holds at once, two of them on an SM, whose warps store weights over each other's scores."""
    step = Step([700, 3], [1500, 400], 8, dim)
    q = queries(step, 32)
    first = run_prompt(step, q, 32)
    for _ in range(20):
        assert torch.equal(run_prompt(step, q, 32), first)
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 40, 2.0 ** 80, 2.0 ** 110])
@pytest.mark.parametrize("empty", [(0, 64), (64, 128), (30, 50), (128, 199)])
@pytest.mark.parametrize("copied", [True, False])
def test_values_of_zero_beside_large_ones(factor, empty, copied):
    """What weighs as much as anything and adds nothing counts among the weights, before the large values and after them."""
    step = Step([200], [6], 2, 64, value_scale=factor)
    _, s, m = step.cache.v_parts
    for token in range(*empty):
        block, at = int(step.cache.table[0, token // 64]), token % 64
        s[block, :, at], m[block, :, at] = 0.0, 0.0
    rewrite(step, "v")
    q = queries(step, 8)
    for splits in (None,) if copied else (1, 3, 0):
        close_to_own(run_prompt(step, q, 8) if copied else run_attention(step, q, 8, splits=splits), step, q, 8, copied=copied)


@pytest.mark.parametrize("size", [1.0, 2.0 ** 90, 2.0 ** -90])
@pytest.mark.parametrize("copied", [True, False])
def test_values_that_are_all_alike(size, copied):
    """Groups whose scale is zero: their least values are all there is."""
    step = Step([200], [6], 2, 64)
    n, s, m = step.cache.v_parts
    n.zero_(), s.zero_(), m.fill_(size)
    m[..., 1] = -size
    rewrite(step, "v")
    q = queries(step, 8)
    for splits in (None,) if copied else (1, 3, 0):
        close_to_own(run_prompt(step, q, 8) if copied else run_attention(step, q, 8, splits=splits), step, q, 8, copied=copied)


@pytest.mark.parametrize("window", [40, 100, -64])
@pytest.mark.parametrize("token", [130, 150, 170, 185])                 # before the windows of some rows or of all, and behind some
@pytest.mark.parametrize("names", ["v", "k", "kv"])
@pytest.mark.parametrize("copied", [True, False])
def test_windows_and_what_lies_before_them(window, token, names, copied):
    step = Step([170, 30], [40, 9], 2, 64, seed=token)
    for name in names:
        enlarge(step, name, 0, token, 2.0 ** 34)
    q = queries(step, 8)
    for splits in (None,) if copied else (1, 2, 0):
        got = run_prompt(step, q, 8, window=window) if copied else run_attention(step, q, 8, window=window, splits=splits)
        close_to_own(got, step, q, 8, window=window, copied=copied)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("factor", [2.0 ** 20, 2.0 ** 90])
@pytest.mark.parametrize("copied", [True, False])
def test_sinks_beside_values_of_unlike_sizes(dim, factor, copied):
    """The sink joins the weights in their own units: in tiles of unlike blocks, of unlike tokens, and where no key weighs anything beside it."""
    step = Step([150, 30], [30, 9], 2, dim)
    for token in (20, 65, 175):
        enlarge(step, "v", 0, token, factor)
    sinks = torch.tensor([0.0, 5.0, -3.0, 40.0, -40.0, 1.0, -math.inf, 0.5], device=DEV)
    q = queries(step, 8)
    for splits in (None,) if copied else (1, 2, 0):
        got = run_prompt(step, q, 8, sinks=sinks) if copied else run_attention(step, q, 8, splits=splits, sinks=sinks)
        close_to_own(got, step, q, 8, copied=copied, sinks=sinks)


# ----------------------------------------------------------------------------------------------- the layer's copies
@pytest.mark.parametrize("options", [dict(), dict(window=100), dict(chunk=64)])
def test_prompts_of_one_sequence_among_many_without_a_token(options):
    """A step whose tokens are nearly all one sequence's: the copies have places for all that it sees."""
    before, new = [700] + [3] * 199, [300] + [0] * 198 + [1]
    step = Step(before, new, 2, 64)
    mixer, ctx, cache = layer(step, 8, False, **options)
    mixer.expands_4bit = lambda ctx, width: True
    q = queries(step, 8)
    out = torch.full_like(q, 7.0)
    mixer.attend(ctx, q, cache, step.table, out)
    close_to_own(out, step, q, 8, window=mixer.reach, copied=True)
