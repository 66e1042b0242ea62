"""The memory that a prompt's copies of a 4-bit cache take in a layer's workspace, without a GPU."""
import pytest
import torch

from thintensor_b200.engine.context import StepContext, Workspace
from thintensor_b200.kernels import api
from thintensor_b200.parts import MIXERS


def test_a_buffer_grows_no_further_than_it_may():
    workspace = Workspace(torch.device("cpu"))
    workspace.get("copies", (10_000,), torch.uint8, most=16_384)
    assert workspace.bytes() == 10_240
    view = workspace.get("copies", (11_000,), torch.uint8, most=16_384)
    assert view.shape == (11_000,) and workspace.bytes() == 16_384 and workspace.generation == 2
    workspace.get("copies", (16_000,), torch.uint8, most=16_384)
    assert workspace.generation == 2
    workspace.get("copies", (20_000,), torch.uint8, most=16_384)       # what is asked for is given all the same
    assert workspace.bytes() == 20_224
    workspace.get("others", (1_000,), torch.uint8)
    workspace.get("others", (1_100,), torch.uint8)
    assert workspace.bytes() == 20_224 + 2_048                         # without a limit: twice what it was


@pytest.mark.parametrize("widths", [(10, 11, 12, 16), (9, 13, 14, 15, 16), (16,)])
def test_copies_keep_to_their_limit(monkeypatch, widths):
    """Prompts over longer and longer tables: keys and values together stay within the limit that the layer's rule names, whatever came before."""
    calls = []
    monkeypatch.setattr(api, "sm_count", lambda device=None: 148)
    monkeypatch.setattr(api, "expand_4bit", lambda *args, **named: calls.append(args[7].shape[0]))
    monkeypatch.setattr(api, "attention_half", lambda *args, **named: None)
    monkeypatch.setattr(api, "attention_4bit", lambda *args, **named: calls.append(None))
    mixer = MIXERS.build("attention", dict(hidden=512, heads=8, kv_heads=2, head_dim=64))
    mixer.EXPAND_4BIT_BYTES = 16 * 2 * 64 * 64 * 4                     # sixteen blocks of keys and values
    workspace, status = Workspace(torch.device("cpu")), torch.zeros(1, dtype=torch.int32)
    q = torch.zeros(4096, 512, dtype=torch.bfloat16)
    ints = torch.zeros(2, dtype=torch.int32)
    for width in (*widths, 17):
        ctx = StepContext(n_tokens=4096, sequences=1, decode=False, max_new=4096, max_total=width * 64, tokens=ints, cu=ints, len_before=ints, slots=ints, tables=[],
                          act_dtype=torch.bfloat16, workspace=workspace, status=status)
        cache = type("Cache", (), dict(k_pool=None, v_pool=None))
        mixer.attend_4bit(ctx, q, cache, torch.zeros((1, width), dtype=torch.int32), torch.empty_like(q))
        assert calls.pop() == (width if width <= 16 else None)
        copies = sum(workspace._buffers[name].numel() for name in ("attention.keys", "attention.values"))
        assert width * 2 * 64 * 64 * 4 <= copies <= mixer.EXPAND_4BIT_BYTES or width > 16
        assert copies <= mixer.EXPAND_4BIT_BYTES
