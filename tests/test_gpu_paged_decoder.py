"""The decoder assembled from the operators on a paged cache, against the CPU oracle's logits (the bounds of
the other decoder tests: 2e-2 max-abs, cosine 0.9999), and what pages and forks have to keep."""

import numpy as np
import pytest
import torch

from qwenscriber_b200 import paged, quant, synthetic
from qwenscriber_b200 import runtime as rt
from qwenscriber_b200.paged_decoder import PagedDecoder

from .parity import cosine, oracle_model, small_config

pytestmark = pytest.mark.gpu


def close(got, want):
    assert float(np.max(np.abs(got - want))) <= 2e-2 and cosine(got, want) >= 0.9999


@pytest.mark.parametrize("page_size", [16, 24])
def test_logits_match_the_oracle(gpu, cuda_lib, oracle_lib, page_size):
    c = small_config(quant.Q8)
    model = synthetic.make_model(c, quant.Q8, seed=11)
    prompt = synthetic.make_prompt(c, 80, 9, seed=11)
    om = oracle_model(model)
    nxt = om.prefill(prompt.tokens, prompt.audio, prompt.audio.shape[0])
    d = PagedDecoder(model, pages=40, page_size=page_size, device=gpu)
    a, b, other = d.start(), d.start(), d.start()
    # One step holds a whole prompt, the first part of the same prompt, and another prompt's tokens.
    cut = 53
    logits = d.step([(a, prompt.tokens, prompt.audio), (b, prompt.tokens[:cut], prompt.audio[:cut]),
                     (other, np.arange(7), None)]).cpu().numpy()
    close(logits[0], om.logits(c.vocab_size))
    logits = d.step([(b, prompt.tokens[cut:], prompt.audio[cut:])]).cpu().numpy()
    close(logits[0], om.logits(c.vocab_size))
    for _ in range(6):
        following = om.step(nxt)
        logits = d.step([(a, [nxt], None), (other, [5, 6], None), (b, [nxt], None)]).cpu().numpy()
        close(logits[0], om.logits(c.vocab_size))
        close(logits[2], om.logits(c.vocab_size))
        nxt = following
    om.close()


def test_forks_share_full_pages_and_diverge(gpu, cuda_lib):
    c = small_config(quant.Q4)
    model = synthetic.make_model(c, quant.Q4, seed=2)
    prompt = synthetic.make_prompt(c, 40, 5, seed=2)
    d = PagedDecoder(model, pages=20, page_size=16, device=gpu)
    a = d.start()
    d.step([(a, prompt.tokens, prompt.audio)])
    b = d.fork(a)
    assert a.pages[:2] == b.pages[:2] and a.pages[2] != b.pages[2] and d.holders[a.pages[0]] == 2
    one = d.step([(a, [7], None), (b, [9], None)])
    fresh = d.start()
    d.step([(fresh, prompt.tokens, prompt.audio)])
    two = d.step([(fresh, [9], None)])
    assert torch.allclose(one[1], two[0], atol=1e-4, rtol=1e-4) and not torch.allclose(one[0], one[1], atol=1e-2)
    for s in (a, b, fresh):
        d.release(s)
    assert not any(d.holders)
    with pytest.raises(rt.QwcError) as e:
        d.step([(d.start(), np.zeros(16 * 21, np.int64), None)])
    assert e.value.name == "limit_exceeded"


def test_transcripts(gpu, cuda_lib):
    c = small_config(quant.Q8)
    model = synthetic.make_model(c, quant.Q8, seed=4)
    prompt = synthetic.make_prompt(c, 30, 5, seed=4)
    d = PagedDecoder(model, pages=30, page_size=16, device=gpu)
    run = lambda seed, **s: d.transcripts(prompt, 3, 8, torch.Generator().manual_seed(seed), **s)  # noqa: E731
    greedy = run(1, temperature=0.0)
    assert greedy[0][0] == greedy[1][0] == greedy[2][0]
    sampled = run(1, temperature=1.5, top_k=200)
    assert sampled == run(1, temperature=1.5, top_k=200)
    assert len({tuple(t) for t, _ in sampled}) > 1 and all(s < 0 for _, s in sampled)
    assert not any(d.holders)


def test_a_step_after_a_refused_one_is_as_if_there_had_been_none(gpu, cuda_lib):
    c = small_config(quant.Q8)
    model = synthetic.make_model(c, quant.Q8, seed=6)
    prompt = synthetic.make_prompt(c, 20, 6, seed=6)
    d = PagedDecoder(model, pages=5, page_size=16, device="cuda")  # the current device
    want = d.start()
    d.step([(want, prompt.tokens, prompt.audio)])
    want_logits = d.step([(want, [7, 8], None)])
    d.release(want)
    a, filler = d.start(), d.start()
    d.step([(a, prompt.tokens, prompt.audio), (filler, np.arange(40), None)])
    for work in ([(a, [7, 8], None), (filler, np.arange(30), None)], [(a, np.arange(40), None)]):
        with pytest.raises(rt.QwcError) as e:
            d.step(work)
        assert e.value.name == "limit_exceeded" and a.length == 26 and filler.length == 40 and d.holders.count(0) == 0
    d.release(filler)
    # 28 positions in the same pages: the refused tokens have left nothing behind.
    assert torch.equal(d.step([(a, [7, 8], None)]), want_logits)
    # A wait that ran out in a step's attention is told of by the step.
    stream = paged.current_stream(d.device)
    paged._workspaces[d.device.index, stream][2][0] = 1
    with pytest.raises(rt.QwcError) as e:
        d.step([(a, [9], None)])
    assert e.value.name == "invalid_state" and a.length == 28
    d.step([(a, [9], None)])
    assert a.length == 29
