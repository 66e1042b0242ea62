"""Sampling from given random numbers, with settings of a row's own: token by token the plain choice of tests/plain_cache_4bit.py (float64, exact sums)."""
from __future__ import annotations

import math

import pytest
import torch

import plain_cache_4bit as plain

pytestmark = pytest.mark.gpu

DEV = "cuda"


def draw(logits, uniform, **settings):
    from thintensor_b200.sampling.sampler import sample_given

    out = torch.full((logits.shape[0],), -5, dtype=torch.int32, device=DEV)
    sample_given(logits.to(DEV), uniform.to(DEV), out, **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
    return out.cpu().tolist()


def compare(logits, uniform, **settings):
    got = draw(logits, uniform, **settings)
    for i, token in enumerate(got):
        mine = {k: (v[i].item() if isinstance(v, torch.Tensor) else v) for k, v in settings.items()}
        # settings are float32 on the device
        mine = {k: (torch.tensor(v, dtype=torch.float32).item() if k != "top_k" else v) for k, v in mine.items()}
        assert token == plain.choose(logits[i], uniform[i].item(), **mine), (i, mine)


def logits_of(rows, vocab, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(rows, vocab, generator=g)
    if vocab > 40:
        x.scatter_add_(1, torch.randint(0, vocab, (rows, 10), generator=g), 6.0 * torch.rand(rows, 10, generator=g))
    return x, torch.rand(rows, generator=g)


SETTINGS = [dict(temperature=1.0), dict(temperature=0.0), dict(temperature=0.7, top_k=5), dict(temperature=1.0, top_k=1), dict(temperature=1.3, top_p=0.9),
            dict(temperature=0.6, min_p=0.1), dict(temperature=1.0, top_k=50, top_p=0.8), dict(temperature=1.0, top_k=300, top_p=0.95, min_p=0.01),
            dict(temperature=3.0, top_p=0.999), dict(temperature=1.0, top_p=0.05, min_p=0.5), dict(temperature=2.0, top_k=1000), dict(temperature=1.0, min_p=1.0),
            dict(temperature=0.9, top_p=0.0), dict(temperature=50.0, min_p=0.9)]


@pytest.mark.parametrize("settings", SETTINGS, ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()))
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 127, 511, 1025, 4099, 20000])
def test_every_filter(settings, vocab):
    compare(*logits_of(9, vocab, seed=vocab), **settings)


@pytest.mark.parametrize("vocab,rows", [(128256, 3), (151937, 2), (262144, 2), (300001, 2)])
@pytest.mark.parametrize("settings", [dict(temperature=0.8, top_p=0.95, min_p=0.02), dict(temperature=0.8, top_k=40), dict(temperature=1.0), dict(temperature=1.0, top_k=700, top_p=0.9)])
def test_large_vocabularies(vocab, rows, settings):
    compare(*logits_of(rows, vocab, seed=1), **settings)


def test_settings_of_every_rows_own():
    rows = 60
    x, u = logits_of(rows, 5003)
    g = torch.Generator().manual_seed(2)
    pick = lambda values, dtype: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=g)].to(dtype)  # noqa: E731
    compare(x, u, temperature=pick([0.0, 0.5, 1.0, 1.7], torch.float32), top_k=pick([0, 1, 7, 400, 6000], torch.int32), top_p=pick([1.0, 0.9, 0.4], torch.float32),
            min_p=pick([0.0, 0.03, 0.3], torch.float32))


@pytest.mark.parametrize("vocab", [5, 700, 6001])
@pytest.mark.parametrize("temperature", [1e-3, 0.4, 1.6])
def test_a_nucleus_of_few_tokens(vocab, temperature):
    """Weights that stand out of what is left, whose sums come close to the share: within the error of a float32 sum of all weights, and further off."""
    g = torch.Generator().manual_seed(vocab)
    rows = 9
    weights = torch.tensor([8.0, 4.0, 2.0, 1.0, 1.0], dtype=torch.float64)          # their running sums are 1/2, 3/4, 7/8 of the whole
    x = torch.full((rows, vocab), -math.inf)
    for i in range(rows):
        x[i, torch.randperm(vocab, generator=g)[:5]] = (temperature * weights.log()).float()
    if vocab > 5:
        x[::3] = torch.maximum(x[::3], temperature * (-17.0 + 0.5 * torch.randn(rows // 3, vocab, generator=g)))      # a little weight beside them
    u = torch.rand(rows, generator=g)
    for top_p in (0.3, 0.4999, 0.5001, 0.749, 0.7499, 0.7501, 0.8749, 0.8751, 0.9999):
        for min_p in (0.0, 0.07, 0.2, 0.3, 0.7):
            compare(x, u, temperature=temperature, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("min_p", [0.0, 1e-6, 0.001, 0.05, 0.4])
@pytest.mark.parametrize("top_p", [0.05, 0.6, 0.97, 1.0])
def test_min_p_and_a_nucleus(top_p, min_p):
    """From rows whose nucleus is a handful to rows where half the vocabulary is above min-p (more than are compared with each other)."""
    for spread, temperature in ((0.1, 1.0), (1.0, 0.5), (2.5, 0.8), (6.0, 1.0)):
        compare(*logits_of(2, 30011, seed=int(10 * spread), spread=spread), temperature=temperature, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("settings", [dict(temperature=1.0, top_k=3), dict(temperature=1.0, top_p=0.5), dict(temperature=1.0, min_p=0.5), dict(temperature=0.0),
                                      dict(temperature=1.0, top_k=300), dict(temperature=1.0)])
@pytest.mark.parametrize("vocab", [64, 3000, 40000])
def test_equal_logits(settings, vocab):
    """All equal; a few values over and over (more than a bin or a list holds); bfloat16's steps; zeros of both signs."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.stack([torch.full((vocab,), 2.0), torch.randint(0, 3, (vocab,), generator=g).float(), torch.randn(vocab, generator=g).bfloat16().float(),
                     torch.where(torch.rand(vocab, generator=g) < 0.5, 0.0, -0.0), torch.where(torch.arange(vocab) % 7 == 0, 5.0, 4.999999)])
    compare(x, torch.rand(5, generator=g), **settings)


@pytest.mark.parametrize("settings", SETTINGS[:8], ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()))
@pytest.mark.parametrize("vocab", [50, 9001])
def test_masked_logits(settings, vocab):
    x, u = logits_of(8, vocab)
    lowest = torch.finfo(torch.float32).min
    x[0, 5:] = -math.inf                                               # a handful left
    x[1, :] = -math.inf
    x[1, 33] = -3.0                                                    # one left
    x[2, :] = -math.inf                                                # none left: token 0
    x[3, :] = math.nan
    x[4, ::3] = math.nan
    x[5, 7:] = lowest                                                  # masked by the type's lowest number
    x[6, :] = lowest
    x[7, ::2] = -math.inf
    compare(x, u, **settings)


def test_infinite_logits():
    x = torch.randn(3, 700)
    x[0, 600] = math.inf
    x[1, 3] = x[1, 650] = math.inf
    x[2, 5], x[2, 6] = math.inf, -math.inf
    u = torch.tensor([0.5, 0.75, 0.1])
    for settings in (dict(temperature=1.0), dict(temperature=0.0), dict(temperature=1.0, top_k=4), dict(temperature=1.0, top_p=0.9), dict(temperature=1.0, min_p=0.1)):
        assert draw(x, u, **settings)[0] == 600 and draw(x, u, **settings)[1] in (3, 650) and draw(x, u, **settings)[2] == 5
    assert draw(x, u, temperature=1.0)[1] == 650 and draw(x, u * 0.5, temperature=1.0)[1] == 3


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 1.0 - 2.0 ** -24, 1.0, 3.0, -1.0])
def test_random_numbers_at_and_beyond_their_ends(u):
    x, _ = logits_of(4, 3001)
    for settings in (dict(temperature=1.0), dict(temperature=1.0, top_k=20), dict(temperature=1.0, top_p=0.9)):
        got = draw(x, torch.full((4,), u), **settings)
        mine = {k: (torch.tensor(v, dtype=torch.float32).item() if k != "top_k" else v) for k, v in settings.items()}
        assert got == [plain.choose(x[i], min(max(u, 0.0), 1.0), **mine) for i in range(4)]


def test_extreme_temperatures_and_spreads():
    x, u = logits_of(6, 2000, spread=30.0)
    for t in (1e-30, 1e-3, 1e4, 1e30):
        compare(x, u, temperature=t)
        compare(x, u, temperature=t, top_p=0.7)
        compare(x, u, temperature=t, min_p=0.2)
    compare(1e30 * x, u, temperature=1.0, top_p=0.9)
    compare(1e-30 * x, u, temperature=1.0, top_k=9, top_p=0.9)


def test_rows_that_do_not_lie_side_by_side():
    x, u = logits_of(5, 1003)
    wide = torch.full((5, 1500), 99.0)
    wide[:, 3:1006] = x
    want = draw(x, u, temperature=1.0, top_k=30, top_p=0.9)
    from thintensor_b200.kernels import api

    out = torch.zeros(5, dtype=torch.int32, device=DEV)
    api.sample_filtered(wide.to(DEV)[:, 3:1006], 1.0, 30, 0.9, 0.0, out, uniform=u.to(DEV))
    assert out.tolist() == want


def test_no_rows():
    from thintensor_b200.kernels import api

    api.sample_filtered(torch.zeros((0, 9), device=DEV), 1.0, 0, 1.0, 0.0, torch.zeros(0, dtype=torch.int32, device=DEV), uniform=torch.zeros(0, device=DEV))


def test_the_counters_random_numbers_are_the_samplers():
    """Without min-p the two samplers draw the same token but where a random number lies within float32's error of a border; 200 rows of 50 tokens do not meet one."""
    from thintensor_b200.kernels import api

    x, _ = logits_of(200, 50, seed=4)
    request, steps = torch.arange(200, dtype=torch.int32, device=DEV), torch.arange(7, 207, dtype=torch.int32, device=DEV)
    a, b = torch.zeros(200, dtype=torch.int32, device=DEV), torch.zeros(200, dtype=torch.int32, device=DEV)
    api.sample_rows(x.to(DEV), 0.9, 20, 0.95, 1234567890123, request, steps, a)
    api.sample_filtered(x.to(DEV), 0.9, 20, 0.95, 0.0, b, seed=1234567890123, request=request, step=steps)
    assert torch.equal(a, b)


def test_frequencies():
    """What is drawn follows the kept distribution: 20,000 even random numbers land on every token as often as its probability says, to one."""
    n = 20000
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 1.5, -3.0])
    u = (torch.arange(n) + 0.5) / n
    got = torch.bincount(torch.tensor(draw(x.repeat(n, 1), u.float(), temperature=1.0, top_p=0.95, min_p=0.1)), minlength=6)
    w = torch.where((x - 2.0).exp() >= 0.1, (x.double() - 2.0).exp(), 0.0)
    assert bool(((got - n * w / w.sum()).abs() <= 2.0).all())


def test_captured_and_on_a_stream_of_its_own():
    from thintensor_b200.kernels import api

    x, u = logits_of(6, 30000)
    logits, uniform, out = x.to(DEV), u.to(DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    run = lambda: api.sample_filtered(logits, 0.9, 0, 0.9, 0.01, out, uniform=uniform)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(3):
        y, v = logits_of(6, 30000, seed=seed)
        logits.copy_(y)
        uniform.copy_(v)
        graph.replay()
        mine = dict(temperature=torch.tensor(0.9).item(), top_p=torch.tensor(0.9).item(), min_p=torch.tensor(0.01).item())
        assert out.tolist() == [plain.choose(y[i], v[i].item(), **mine) for i in range(6)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        run()
    stream.synchronize()
    assert out.tolist() == [plain.choose(y[i], v[i].item(), **mine) for i in range(6)]


def test_generation_keeps_to_min_p(tmp_path):
    """Every token of a greedy-fed sequence drawn with min-p is one whose probability reaches that fraction of the largest."""
    import thintensor_b200
    from conftest import TINY
    from thintensor_b200 import Entry

    thintensor_b200.save_random_model(tmp_path, TINY["d"], seed=2)
    runtime = thintensor_b200.load_model(tmp_path)
    prompt = [5, 9, 200, 7]
    for graph in (False, True):
        new = runtime.generate([prompt], max_new_tokens=20, stop_ids=(), temperature=1.5, min_p=0.5, seed=11, use_graph=graph)[0]
        engine = runtime.new_engine(max_tokens=64, max_sequences=1)
        slot = engine.open()
        logits = engine.step([Entry(slot, prompt + new[:-1], list(range(len(prompt) - 1, len(prompt) + len(new) - 1)))])
        ratio = ((logits - logits.amax(1, keepdim=True)) / 1.5).exp().gather(1, torch.tensor(new, device=DEV)[:, None])
        # the prompt in one step and token by token differ by bfloat16's rounding of the logits' inputs, a hundredth of a logit here
        assert float(ratio.min()) >= 0.5 * math.exp(-0.05)
