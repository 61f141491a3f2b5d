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


@pytest.mark.parametrize("flint", [False, True])
def test_prompt_router_is_the_decode_router(fb, flint):
    """The prompt's routing on the rows and logits of the decode route op (softmax and sigmoid, tied logits among them).
    Logits: sums of the same 32-bit products in another order, rounded to bf16 (one step of 2^-7 of them, or 2^-11 of the
    largest where they cancel).  On equal logits the experts are equal; weights are a few 32-bit roundings and two
    exponentials of 2^-21: 2^-18."""
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = build(fb, flint)
    dec = SharedPromptDecoder(model, 2)
    L, c, T = model.layers[0], model.cfg, 8
    gate, ew = L["gate"], L["experts"]
    gate[3], gate[17], gate[30] = gate[9], gate[9], gate[9]
    g = torch.Generator(device="cuda").manual_seed(3)
    e = lambda *s, dt=torch.bfloat16: torch.empty(s, dtype=dt, device="cuda")
    seen = set()
    for _ in range(40):
        a, res = (torch.randn((T, c.hidden), generator=g, device="cuda").bfloat16() for _ in range(2))
        a += gate[9] * float(torch.randint(0, 3, (1,), generator=g, device="cuda")) / c.weight_std
        lg, ti, tw = e(T, c.num_experts, dt=torch.float32), e(T, c.topk, dt=torch.int32), e(T, c.topk, dt=torch.float32)
        xn = e(T, c.hidden)
        torch.ops.flint_b200.moe_route(a, res, L["ln2"], c.rms_eps, gate, c.topk, ew.score_fn, lg, ti, tw, xn,
                                       torch.empty_like(xn), True, True)
        logits = dec._router_logits(xn, gate)
        assert ((logits - lg).abs() <= lg.abs() * 2 ** -7 + lg.abs().amax(-1, keepdim=True) * 2 ** -11).all()
        ids, weight = dec._choose(lg, ew)
        assert ids.dtype == torch.int32 and torch.equal(ids, ti)
        torch.testing.assert_close(weight, tw, rtol=2 ** -18, atol=0)
        seen |= {int(i) for i in ids.flatten()}
    assert {3, 9} <= seen
    dec.close()
