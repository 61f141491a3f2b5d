"""SharedPromptDecoder's bookkeeping without a GPU."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch


def decoder(streams=2, blocks=10, max_ctx=160):
    """A decoder whose model, pool and graphs are stand-ins: only what the host decides is real."""
    from flint_b200.shared_prompt import SharedPromptDecoder
    dec = object.__new__(SharedPromptDecoder)
    dec.M, dec.graphs, dec.replays = streams, {}, 0
    dec.m = SimpleNamespace(dev="cpu", blocks_per_stream=blocks, cos_sin=torch.zeros(max_ctx, 128), embed=torch.zeros(64, 8))
    dec.bt = torch.arange(streams * blocks, dtype=torch.int32).view(streams, blocks)
    dec.tokens, dec.seq_lens = torch.zeros(streams, dtype=torch.int32), torch.zeros(streams, dtype=torch.int32)
    dec.positions, dec.slots = torch.zeros(streams, dtype=torch.int64), torch.zeros(streams, dtype=torch.int64)
    dec.history = torch.zeros((streams, 40), dtype=torch.int32)
    return dec


def test_positions_behind_the_table_have_no_slot(fb):
    dec = decoder()
    dec.bt[1, 3:] = -1
    for at, slots in (([5, 47], [5, 207]), ([159, 48], [159, -1]), ([160, 170], [-1, -1])):
        dec.positions.copy_(torch.tensor(at))
        dec._follow_tables()
        assert dec.slots.tolist() == slots and dec.seq_lens.tolist() == [at[0] + 1, at[1] + 1]


class Untouchable:
    def __getattr__(self, name):
        raise AssertionError(f"went on to {name}")


def test_prompts_end_with_the_rotary_table(fb):
    """Pages are whole, so they may hold more tokens than the model has positions for."""
    dec = decoder(blocks=10, max_ctx=150)
    dec.c, dec.graphs, dec.pool = None, {"step": None}, Untouchable()
    for length, room in ((145, 6), (151, 0), (1, 150)):
        with pytest.raises(ValueError, match="do not fit 150"):
            dec.read_prompt(np.zeros(length, np.int64), room)
    dec.all_streams = torch.arange(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="went on to free"):
        dec.read_prompt(np.zeros(145, np.int64), 5)


@pytest.mark.parametrize("prompt", [[1, 64, 2], [-1, 3], [3, 4, 64], [10 ** 12]])
def test_prompt_tokens_are_in_the_vocabulary(fb, prompt):
    dec = decoder()
    dec.c, dec.graphs, dec.pool = None, {"step": None}, Untouchable()
    dec.all_streams = torch.arange(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="token ids"):
        dec.read_prompt(prompt, 3)
