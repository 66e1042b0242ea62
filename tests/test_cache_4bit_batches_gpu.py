"""Decoding steps of a batch whose model keeps its cache in 4 bits, captured and not, against each sequence by itself."""
from __future__ import annotations

import pytest
import torch

from conftest import TINY

pytestmark = pytest.mark.gpu


def cosines(a, b):
    return torch.nn.functional.cosine_similarity(a.double(), b.double(), dim=-1)


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("name", ["b", "d", "e"])
def test_a_batch_reads_every_sequences_own_cache(tmp_path, name, graph):
    """Each step's logits are those of the sequence alone in one piece, but for codes that move where bfloat16 rounds a key or value otherwise (the bound that
    pieces of one sequence are held to); with another sequence's prompt before them they are not.  What is drawn reaches min-p of its step's largest probability."""
    import thintensor_b200
    from thintensor_b200 import Entry, SamplingParams
    from thintensor_b200.engine.generate import EngineBackend

    thintensor_b200.save_random_model(tmp_path, TINY[name], seed=1)
    runtime = thintensor_b200.load_model(tmp_path, cache="4bit")
    g = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, TINY[name]["vocab_size"], (400,), generator=g).tolist()
    prompts, steps = [tokens[:90], tokens[100:103], tokens[200:261], tokens[270:398]], 20        # the third and fourth come to a block's end
    backend = EngineBackend(runtime.new_engine(max_tokens=1024, max_sequences=4), SamplingParams(0.9, 0, 1.0, 3, 0.02), graph)
    new = [[t] for t in backend.start_batch(range(4), prompts, [len(p) + steps for p in prompts])]
    logits = []
    for _ in range(steps - 1):
        for mine, token in zip(new, backend.decode_step(range(4))):
            mine.append(token)
        logits.append(backend._state.logits[:4].clone())
    for position in range(4):
        backend.finish(position)
    for i in range(4):
        got = torch.stack([step[i] for step in logits])
        for other in (i, (i + 1) % 4):
            engine = runtime.new_engine(max_tokens=1024, max_sequences=1)
            fed = prompts[other] + new[i][:-1]
            alone = engine.step([Entry(engine.open(), fed, list(range(len(prompts[other]), len(fed))))])
            engine.check_status()
            assert (float(cosines(got, alone).min()) > 0.999) == (other == i)
        drawn = torch.tensor(new[i][1:], device=got.device)
        ratio = ((got - got.amax(1, keepdim=True)).double() / 0.9).exp().gather(1, drawn[:, None])
        assert float(ratio.min()) >= 0.02 * (1 - 2.0 ** -20)
