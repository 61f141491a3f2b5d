"""The path that runs the prompt attention, the page operations and the shared-prefix attention together, against the
Decoder that feeds the same prompt token by token into pages of each stream's own."""
import numpy as np
import pytest
import torch

from helpers import assert_bf16_close

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
VOCAB = 4096


def build(fb, flint=False):
    from flint_b200.model import FlintConfig, FlintModel
    if flint:
        cfg = FlintConfig.flint(layers=3, vocab=VOCAB, num_experts=32, layer_types=("sliding_attention", "full_attention",
                                                                                    "sliding_attention"),
                                sliding_window=20, no_rope_layers=(1,), mlp_only_layers=(2,), dense_inter=512)
    else:
        cfg = FlintConfig(layers=2, vocab=VOCAB)
    return FlintModel(cfg, torch.device("cuda", 0), seed=5, max_ctx=160, max_batch=4)


def after_prompt(model, prompt, shared):
    """(hidden state of each stream after the prompt's last token, K/V of the prompt's tokens in stream 0's pages)"""
    from flint_b200.model import Decoder
    from flint_b200.shared_prompt import SharedPromptDecoder
    if shared:
        dec = SharedPromptDecoder(model, 3)
        dec.capture()
        dec.read_prompt(prompt, room=20)
    else:
        dec = Decoder(model, batch=3, moe="fused", attn="chain")
        dec.capture()
        dec.prefill(np.tile(prompt, (3, 1)))
    dec.graphs["layers"].replay()
    torch.cuda.synchronize()
    n = len(prompt)
    pos = torch.arange(n, device=model.dev)
    kv = [kv[dec.bt[0, pos // 16].long(), :, pos % 16].float().cpu().numpy() for kv in model.kv]
    h = dec.h.float().cpu().numpy().copy()
    dec.check_status()
    dec.close()
    return h, kv


@pytest.mark.parametrize("flint", [False, True])
@pytest.mark.parametrize("length", [1, 2, 17, 70])
def test_prompt_matches_token_by_token(fb, flint, length):
    """Same tolerance as between the decode paths of test_model_gpu: rounding to bf16 at other places of the sums.  The
    routers are set to zero (equal logits: the lowest experts, equal weights), since a choice of experts is not
    continuous: a token whose last two candidates nearly tie may go to another expert for the last bit of a norm."""
    model = build(fb, flint)
    for L in model.layers:
        if L["gate"] is not None:
            L["gate"].zero_()
    prompt = np.random.default_rng(length).integers(0, VOCAB, size=length)
    h0, kv0 = after_prompt(model, prompt, False)
    h1, kv1 = after_prompt(model, prompt, True)
    for l, (a, b) in enumerate(zip(kv1, kv0)):
        assert_bf16_close(a, b, rel=2 ** -5, abs_frac=2e-2, what=f"cache of layer {l}")
    assert_bf16_close(h1, h0, rel=2 ** -5, abs_frac=2e-2, what="hidden state")


def test_streams_share_pages_branch_and_compact(fb):
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = build(fb)
    dec = SharedPromptDecoder(model, 4, sampling=dict(temperature=1.0, top_k=20, top_p=1.0, seeds=[3, 3, 4, 5]))
    dec.reserve_history(12)
    dec.capture()
    prompt = np.random.default_rng(1).integers(0, VOCAB, size=50)
    dec.read_prompt(prompt, room=12)
    table = dec.bt.cpu().numpy()
    assert (table[:, :3] == table[0, :3]).all() and len(set(table[:, 3])) == 4        # 48 of 49 tokens are shared
    assert dec.pool.ref[:3].tolist() == [4, 4, 4] and int(dec.pool.ref.sum()) == 4 * 4
    step = dec.graphs["step"].replay
    for _ in range(6):
        step()
    dec.branch([1, 3], [0, 2])
    hist = dec.history.cpu().numpy()
    assert (hist[1, :6] == hist[0, :6]).all() and (hist[3, :6] == hist[2, :6]).all() and (hist[2] != hist[0]).any()
    before = {b: cached(dec, model, b) for b in range(4)}
    for a, b in ((1, 0), (3, 2)):
        np.testing.assert_array_equal(before[a], before[b])
    assert dec.compact() == 3 + 4
    assert dec.bt.max().item() == 6
    for b in range(4):
        np.testing.assert_array_equal(cached(dec, model, b), before[b])
    for _ in range(6):
        step()
    torch.cuda.synchronize()
    dec.check_status()
    assert dec.positions.tolist() == [49 + 12] * 4
    dec.close()


def cached(dec, model, b):
    pos = torch.arange(int(dec.positions[b]), device=model.dev)
    return model.kv_all[:, dec.bt[b, pos // 16].long(), :, pos % 16].float().cpu().numpy()


def test_a_compacted_and_branched_cache_decodes_as_before(fb):
    """Moving the pages changes no token: the same run with and without compaction in the middle."""
    from flint_b200.shared_prompt import SharedPromptDecoder
    prompt, runs = np.random.default_rng(2).integers(0, VOCAB, size=37), []
    for moves in (False, True):
        model = build(fb)
        dec = SharedPromptDecoder(model, 3, sampling=dict(temperature=1.0, top_k=20, top_p=1.0, seeds=[1, 2, 3]))
        dec.reserve_history(10)
        dec.capture()
        dec.read_prompt(prompt, room=10)
        for i in range(10):
            if i == 4:
                dec.branch([0], [2])
            if moves and i in (3, 5):
                dec.compact()
            dec.graphs["step"].replay()
        torch.cuda.synchronize()
        runs.append(dec.history.cpu().numpy().copy())
        dec.close()
    np.testing.assert_array_equal(runs[0], runs[1])


def test_refusals(fb):
    from flint_b200.shared_prompt import SharedPromptDecoder
    model = build(fb)
    dec = SharedPromptDecoder(model, 2)
    dec.capture()
    with pytest.raises(ValueError):
        dec.read_prompt(np.zeros(150, np.int64), room=40)
    with pytest.raises(ValueError):
        dec.read_prompt(np.zeros(0, np.int64), room=4)
    dec.read_prompt(np.zeros(20, np.int64), room=4)
    for dst, src in (([1], [1]), ([0, 1], [1, 0]), ([2], [0]), ([0], []), ([1, 1], [0, 0])):
        with pytest.raises(ValueError):
            dec.branch(dst, src)
    dec.branch([], [])
    for call in (lambda: dec.prefill(np.zeros((2, 4), np.int64)), lambda: dec.fill_kv_random(np.zeros((2, 4))),
                 lambda: dec.generate_host_driven(1, {})):
        with pytest.raises(NotImplementedError):
            call()
    dec.close()
