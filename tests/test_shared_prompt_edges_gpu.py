"""SharedPromptDecoder at its edges: the end of its room, decoding in parts, the prompt's router."""
import numpy as np
import pytest
import torch

from test_shared_prompt_gpu import VOCAB, build

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def test_steps_end_with_the_room(fb):
    """Behind the pages that read_prompt reserved a step has nowhere to write and no keys to read: it is refused, through
    decode() and through the graph, and the state stays as it was."""
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = build(fb)
    dec = SharedPromptDecoder(model, 2)
    dec.reserve_history(30)
    dec.capture()
    with pytest.raises(ValueError, match="room"):
        dec.decode(1)                                             # no prompt yet
    with pytest.raises(ValueError, match="read_prompt"):
        dec.branch([1], [0])
    with pytest.raises(ValueError):
        dec.read_prompt(np.zeros(20, np.int64), room=-1)
    for length, room in ((20, 4), (33, 0), (3, 17)):
        dec.read_prompt(np.random.default_rng(room).integers(0, VOCAB, size=length), room=room)
        with pytest.raises(ValueError, match="room"):
            dec.decode(room + 2)
        dec.decode(room)
        dec.branch([1], [0])
        dec.graphs["step"].replay()                               # reads the last of the room, draws one more token
        assert dec.positions.tolist() == [length + room] * 2
        for call in (lambda: dec.decode(1), dec.graphs["step"].replay):
            with pytest.raises(ValueError, match="room"):
                call()
        assert dec.positions.tolist() == [length + room] * 2
        dec.check_status()
    dec.capture()
    with pytest.raises(ValueError, match="room"):
        dec.decode(1)                                             # capturing runs a step of its own: the prompt is gone
    dec.close()


def test_decode_gives_the_tokens_of_its_own_steps(fb):
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = build(fb)
    dec = SharedPromptDecoder(model, 3, sampling=dict(temperature=1.0, top_k=20, top_p=1.0, seeds=[1, 2, 3]))
    dec.reserve_history(10)
    dec.capture()
    prompt, runs = np.random.default_rng(6).integers(0, VOCAB, size=30), []
    for parts in ((10,), (4, 5, 1)):
        dec.read_prompt(prompt, room=20)
        runs.append([dec.decode(n).cpu().numpy() for n in parts])
        assert [t.shape for t in runs[-1]] == [(3, n) for n in parts]
        with pytest.raises(ValueError, match="history"):
            dec.decode(1)                                         # ten are recorded
    np.testing.assert_array_equal(runs[0][0], np.concatenate(runs[1], axis=1))
    dec.close()
