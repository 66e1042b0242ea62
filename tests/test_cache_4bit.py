"""The 4-bit cache without a GPU: its format, what the entry points and models refuse, the cache's storage, and the sampler's settings."""
import math

import pytest
import torch

import plain_cache_4bit as plain
from conftest import TINY
from thintensor_b200.cache.cache import SequenceCache
from thintensor_b200.config.registry import load_config
from thintensor_b200.engine.model import DecoderModel
from thintensor_b200.kernels import api
from thintensor_b200.parts import MIXERS
from thintensor_b200.parts.base import KVNeed
from thintensor_b200.runtime import parse_cache
from thintensor_b200.sampling.sampler import SamplingParams


@pytest.mark.parametrize("dim", [32, 64, 96, 128])
@pytest.mark.parametrize("values", [False, True])
def test_every_code_has_a_place_of_its_own(dim, values):
    table = plain.places(dim)[1 if values else 0]
    assert len(set(table.values())) == 64 * dim and {w for w, _ in table.values()} == set(range(8 * dim)) and {s for _, s in table.values()} == set(range(0, 32, 4))
    n = torch.randint(0, 16, (64, dim))
    s, m = torch.rand(64, dim // 32).bfloat16().float(), torch.randn(64, dim // 32).bfloat16().float()
    raw = plain.write_block(n, s, m, values)
    assert raw.numel() == api.cache_4bit_bytes(dim) == 40 * dim
    for got, want in zip(plain.read_block(raw, dim, values), (n, s, m)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("scale,offset", [(1.0, 0.0), (1e-3, 5.0), (1e3, -1e4), (1e-30, 0.0), (1e30, 1e31)])
def test_codes_meet_every_number_within_half_a_scale(scale, offset):
    x = scale * torch.randn(500, 128) + offset
    n, s, m = plain.quantise(x)
    off = (plain.numbers(n, s, m) - x.double()).abs().view(500, 4, 32)
    # half a step, and the float32 roundings of (x - m) and of its product with 1 / s: 2^-23 of 15 steps each, and 2^-24 of x where it is taken from m
    assert bool((off <= s.double()[..., None] * (0.5 + 15 * 2.0 ** -22) + 2.0 ** -24 * x.abs().view(500, 4, 32).double()).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3.4e38])
def test_what_is_not_finite_is_not_a_number_in_its_group_alone(bad):
    x = torch.randn(3, 64)
    x[1, 40] = bad
    if bad == 3.4e38:
        x[1, 41] = -bad                                      # finite numbers whose range is not
    n, s, m = plain.quantise(x)
    assert torch.isnan(s[1, 1]) and m[1, 1] == 0 and not n[1, 32:].any()
    s[1, 1] = 0
    assert torch.isfinite(s).all() and torch.isfinite(m).all()


def step(sequences=1, width=3):
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    return dict(table=z(sequences, width), cu=z(sequences + 1), len_before=z(sequences), sequences=sequences, status=z(1))


def append_args(**change):
    s = step()
    args = dict(qkv=torch.zeros(1, 2, 4 * 64 + 4 * 64), inv_freq=torch.zeros(32), rotary_dim=64, attention_scaling=1.0, q_out=torch.zeros(2, 256, dtype=torch.bfloat16),
                k_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), v_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), n_tokens=2, heads=4, kv_heads=2, head_dim=64, **s)
    args.update(change)
    return args


@pytest.mark.parametrize("change,match", [
    (dict(head_dim=48), "head sizes"), (dict(heads=3), "head sizes|expected"), (dict(kv_heads=0), "head sizes"), (dict(heads=34, kv_heads=2), "16 query heads"),
    (dict(qkv=torch.zeros(1, 2, 511)), "expected"), (dict(qkv=torch.zeros(1, 3, 512)), "expected"), (dict(qkv=torch.zeros(1, 2, 512, dtype=torch.bfloat16)), "float32"),
    (dict(q_out=torch.zeros(2, 256)), "bfloat16"), (dict(q_out=torch.zeros(3, 256, dtype=torch.bfloat16)), "fit"), (dict(rotary_dim=63), "even"),
    (dict(rotary_dim=66), "even"), (dict(inv_freq=torch.zeros(31)), "frequencies"), (dict(k_pool=None), "both"),
    (dict(k_pool=torch.zeros(3, 2, 2559, dtype=torch.uint8)), "2560"), (dict(v_pool=torch.zeros(3, 2, 2560)), "uint8"),
    (dict(v_pool=torch.zeros(4, 2, 2560, dtype=torch.uint8)), "as many blocks"), (dict(table=torch.zeros(1, 3)), "int32"),
    (dict(cu=torch.zeros(1, dtype=torch.int32)), "offset"), (dict(sequences=2), "row and a length"),
    (dict(k_pool=torch.zeros(3 * 2 * 2560 + 8, dtype=torch.uint8)[8:].view(3, 2, 2560)), "16-byte"),
])
def test_appending_refuses(change, match):
    with pytest.raises(api.KernelError, match=match):
        api.rope_append_4bit(**append_args(**change))


def attend_args(**change):
    args = dict(q=torch.zeros(2, 256, dtype=torch.bfloat16), k_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), v_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8),
                n_tokens=2, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=0, splits=1, out=torch.zeros(2, 256, dtype=torch.bfloat16), part_acc=None,
                part_ml=None, **step())
    args.update(change)
    return args


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 256)), "bfloat16"), (dict(out=torch.zeros(2, 256)), "bfloat16"), (dict(out=torch.zeros(1, 256, dtype=torch.bfloat16)), "fit"),
    (dict(n_tokens=3), "fit"), (dict(scale=0.0), "positive"), (dict(scale=float("nan")), "positive"), (dict(scale=-1.0), "positive"), (dict(splits=9), "slices"),
    (dict(splits=-1), "slices"), (dict(one_token_each=True), "one token"), (dict(sinks=torch.zeros(3)), "sinks"), (dict(head_dim=80), "head sizes"),
    (dict(k_pool=torch.zeros(3, 2, 64, 64, dtype=torch.uint8)), "2560"), (dict(len_before=torch.zeros(1)), "int32"),
    (dict(q=torch.zeros(520, dtype=torch.bfloat16)[4:516].view(2, 256)), "16-byte"),
])
def test_attending_refuses(change, match):
    with pytest.raises(api.KernelError, match=match):
        api.attention_4bit(**attend_args(**change))


@pytest.mark.parametrize("change,match", [
    (dict(keys=torch.zeros(4, 2, 64, 64)), "bfloat16"), (dict(keys=torch.zeros(4, 2, 64, 48, dtype=torch.bfloat16)), "head size"),
    (dict(values=torch.zeros(4, 2, 64, 32, dtype=torch.bfloat16)), "fit"), (dict(table_tmp=torch.zeros(1, 2, dtype=torch.int32)), "fit"),
    (dict(**{**step(2), "table_tmp": torch.zeros(2, 3, dtype=torch.int32)}, keys=torch.zeros(5, 2, 64, 64, dtype=torch.bfloat16),
          values=torch.zeros(5, 2, 64, 64, dtype=torch.bfloat16)), "places"),
])
def test_reading_back_refuses(change, match):
    args = dict(k_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), v_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), window=0,
                keys=torch.zeros(4, 2, 64, 64, dtype=torch.bfloat16), values=torch.zeros(4, 2, 64, 64, dtype=torch.bfloat16),
                table_tmp=torch.zeros(1, 3, dtype=torch.int32), **step())
    args.update(change)
    with pytest.raises(api.KernelError, match=match):
        api.expand_4bit(**args)


HALF = dict(keys=torch.zeros(4, 2, 64, 64, dtype=torch.float16), values=torch.zeros(4, 2, 64, 64, dtype=torch.float16), scales=torch.zeros(2, 4, 2),
            marks=torch.zeros(4, 2, 64, dtype=torch.uint8))


@pytest.mark.parametrize("change,match", [
    (dict(keys=torch.zeros(4, 2, 64, 64, dtype=torch.bfloat16)), "float16"), (dict(scales=torch.zeros(2, 3, 2)), "scales"), (dict(scales=None), "bfloat16"),
    (dict(marks=None), "marks"), (dict(marks=torch.zeros(4, 2, 32, dtype=torch.uint8)), "marks"), (dict(scales=torch.zeros(2, 4, 2, dtype=torch.float64)), "float32"),
    (dict(keys=torch.zeros(4, 2, 64, 64, dtype=torch.bfloat16), values=torch.zeros(4, 2, 64, 64, dtype=torch.bfloat16), scales=None), "marks"),
])
def test_reading_back_float16_refuses(change, match):
    args = dict(k_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), v_pool=torch.zeros(3, 2, 2560, dtype=torch.uint8), window=0,
                table_tmp=torch.zeros(1, 3, dtype=torch.int32), **HALF, **step())
    args.update(change)
    with pytest.raises(api.KernelError, match=match):
        api.expand_4bit(**args)


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(2, 256)), "does not take"), (dict(out=torch.zeros(2, 256)), "bfloat16"), (dict(out=torch.zeros(1, 256, dtype=torch.bfloat16)), "fit"),
    (dict(n_tokens=3), "fit"), (dict(head_dim=80), "head"), (dict(heads=34, kv_heads=2), "does not take"), (dict(sinks=torch.zeros(3)), "sinks"),
    (dict(scale=0.0), "positive"), (dict(scale=float("nan")), "positive"), (dict(scales=torch.zeros(4, 2)), "fit"), (dict(marks=torch.zeros(4, 2, 64)), "uint8"),
    (dict(values=torch.zeros(3, 2, 64, 64, dtype=torch.float16)), "fit"), (dict(len_before=torch.zeros(1)), "int32"),
    (dict(q=torch.zeros(520, dtype=torch.bfloat16)[4:516].view(2, 256)), "16-byte"), (dict(table=torch.zeros(2, 2, 2, dtype=torch.int32)), "row"),
])
def test_attention_over_float16_blocks_refuses(change, match):
    args = dict(q=torch.zeros(2, 256, dtype=torch.bfloat16), n_tokens=2, heads=4, kv_heads=2, head_dim=64, scale=0.125, window=0,
                out=torch.zeros(2, 256, dtype=torch.bfloat16), **HALF, **step())
    args.update(change)
    with pytest.raises(api.KernelError, match=match):
        api.attention_half(**args)


def test_what_a_4bit_call_would_do_on_the_cpu_is_an_error():
    with pytest.raises(api.KernelError):
        api.rope_append_4bit(**append_args())
    with pytest.raises(api.KernelError):
        api.attention_4bit(**attend_args())


@pytest.mark.parametrize("change,match", [
    (dict(logits=torch.zeros(3, 8, dtype=torch.bfloat16)), "float32"), (dict(logits=torch.zeros(8, 3).T), "side by side"), (dict(logits=torch.zeros(8)), "rows"),
    (dict(logits=torch.zeros(3, 0)), "vocabularies"), (dict(logits=torch.zeros(1, 1).expand(3, api.SAMPLE_FILTERED_VOCAB + 1)), "side by side|vocabularies"),
    (dict(out=torch.zeros(2, dtype=torch.int32)), "tokens"), (dict(out=torch.zeros(3)), "int32"), (dict(uniform=torch.zeros(2)), "random numbers"),
    (dict(uniform=torch.zeros(3, dtype=torch.float64)), "float32"), (dict(uniform=None), "request"), (dict(temperature=-0.5), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=1.5), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"),
    (dict(temperature=torch.zeros(2)), "temperature"), (dict(top_k=torch.zeros(3)), "int32"), (dict(top_p=torch.zeros(3, dtype=torch.float64)), "float32"),
])
def test_sampling_refuses(change, match):
    args = dict(logits=torch.zeros(3, 8), temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=torch.zeros(3, dtype=torch.int32), uniform=torch.zeros(3))
    args.update(change)
    with pytest.raises(api.KernelError, match=match):
        api.sample_filtered(**args)


@pytest.mark.parametrize("min_p", [-0.1, 1.01, float("nan")])
def test_min_p_is_a_fraction(min_p):
    with pytest.raises(ValueError, match="min_p"):
        SamplingParams(temperature=1.0, min_p=min_p)
    assert SamplingParams(1.0, 5, 0.9, 3) == SamplingParams(temperature=1.0, top_k=5, top_p=0.9, seed=3, min_p=0.0)


# ------------------------------------------------------------------------------------------------------------- models
def spec_of(name):
    arch, config = load_config(TINY[name])
    return arch.describe(config)


@pytest.mark.parametrize("name,fits", [("a", False), ("b", True), ("c", False), ("d", True), ("e", True), ("f", False)])
def test_which_models_keep_4_bits(name, fits):
    if fits:
        model = DecoderModel(spec_of(name), torch.bfloat16, None, 4)
        assert {need.bits for need in model.cache_needs()[0]} == {4}
    else:
        with pytest.raises(ValueError, match="4 bits.*head sizes"):
            DecoderModel(spec_of(name), torch.bfloat16, None, 4)
    with pytest.raises(ValueError, match="float32"):
        DecoderModel(spec_of(name), torch.float32, None, 4)
    assert {need.bits for need in DecoderModel(spec_of(name), torch.bfloat16, None).cache_needs()[0]} == {None}


@pytest.mark.parametrize("options,word", [(dict(value_dim=32), "another size"), (dict(qk_norm_eps=1e-6), "normed"), (dict(conv=4), "convolution"),
                                          (dict(softcap=30.0), "capped"), (dict(slope_exponent=8.0), "bias"), (dict(gate="head"), "gate")])
def test_layers_with_options_that_no_4bit_kernel_has(options, word):
    make = lambda **more: MIXERS.build("attention", dict(hidden=128, heads=4, kv_heads=2, head_dim=64, **more))  # noqa: E731
    assert word in make(**options).no_4bit_cache(torch.bfloat16)
    for plain_form in (dict(), dict(window=100), dict(chunk=128), dict(sink=True), dict(null_score=0.0), dict(bias=True)):
        assert make(**plain_form).no_4bit_cache(torch.bfloat16) is None


def test_other_designs_say_why_they_cannot():
    from famalorn_models import CONFIGS

    arch, config = load_config(next(iter(CONFIGS.values())))
    with pytest.raises(ValueError, match="cannot keep its cache in 4 bits"):
        DecoderModel(arch.describe(config), torch.bfloat16, None, 4)


@pytest.mark.parametrize("cache", ["4", "int4", 4, True, "bf16"])
def test_cache_names(cache):
    with pytest.raises(ValueError, match="4bit"):
        parse_cache(cache)
    assert parse_cache("4bit") == 4 and parse_cache(None) is None


def test_storage_of_a_4bit_group():
    need = KVNeed(2, 64, bits=4)
    cache = SequenceCache([need, need, KVNeed(2, 64)], [None] * 3, [None, None, None], 5, 2, torch.bfloat16, "cpu")
    assert len(cache.kv_groups) == 2
    for run in (0, 1):
        view = cache.run_cache(run)
        assert view.k_pool.dtype == torch.uint8 and tuple(view.k_pool.shape) == tuple(view.v_pool.shape) == (5, 2, 2560)
        assert view.k_pool.is_contiguous() and view.v_pool.is_contiguous() and view.k_pool.data_ptr() % 16 == view.v_pool.data_ptr() % 16
    view.k_pool.fill_(1)
    view.v_pool.fill_(2)
    assert not cache.run_cache(0).k_pool.any() and not cache.run_cache(0).v_pool.any()
    plain_bytes = SequenceCache([KVNeed(2, 64)] * 2, [None] * 2, [None, None], 5, 2, torch.bfloat16, "cpu").bytes()
    assert cache.kv_groups[0].bytes() * 16 == plain_bytes * 5 and need.token_bytes(torch.bfloat16) * 64 * 5 * 2 == cache.kv_groups[0].bytes()
    with pytest.raises(RuntimeError, match="shape differs"):
        SequenceCache([need, KVNeed(2, 64)], [None] * 2, [None, 0], 5, 2, torch.bfloat16, None)


@pytest.mark.parametrize("logits,u,settings,want", [
    ([0.0, 1.0, 1.0], 0.9, dict(temperature=0.0), 1), ([0.0, 0.0, 0.0, 0.0], 0.5, dict(temperature=1.0), 2), ([0.0, 0.0, 0.0, 0.0], 0.49999, dict(temperature=1.0), 1),
    ([3.0, 1.0, 3.0, 2.0], 0.99, dict(temperature=1.0, top_k=1), 2), ([math.nan, -math.inf], 0.3, dict(temperature=1.0), 0),
    ([0.0, math.log(3.0)], 0.0, dict(temperature=1.0, min_p=0.34), 1), ([0.0, 5.0, 4.0], 0.999, dict(temperature=1.0, top_p=0.5), 1),
])
def test_the_plain_choice(logits, u, settings, want):
    assert plain.choose(torch.tensor(logits), u, **settings) == want


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (32, 8), (16, 2), (32, 2)])
def test_slices_of_a_step(heads, kv_heads):
    """Slices are taken while their clusters are resident together and have 256 keys each; even runs for long caches alone."""
    for sequences in (1, 2, 7, 40, 300):
        for new in (1, 3, 24):
            for longest in (1, 255, 511, 512, 3000, 8191, 8192, 40000):
                splits = api.attention_4bit_splits(sequences, sequences * new, heads, kv_heads, longest, 148)
                assert splits in (0, 1, 2, 4, 8)
                if splits == 0:
                    assert longest >= 8192 and sequences * kv_heads <= 4 * 148
                else:
                    assert splits == 1 or (longest >= 256 * splits and sequences * kv_heads * splits <= 4 * 148)
    assert api.attention_4bit_splits(1, 1, heads, kv_heads, 2048, 148) == 8
    assert api.attention_4bit_splits(1, 1, heads, kv_heads, 100, 148) == 1
    assert api.attention_4bit_splits(2000, 2000, heads, kv_heads, 100000, 148) == 1
