"""What PagedDecoder keeps of its sequences and pages when a step or a fork is refused or fails: no GPU is needed,
the layers are left out."""

import numpy as np
import pytest
import torch

from qwenscriber_b200 import paged, quant
from qwenscriber_b200 import runtime as rt
from qwenscriber_b200.paged_decoder import PagedDecoder

from .parity import small_config

PAGE = 16


@pytest.fixture
def decoder(monkeypatch):
    d = object.__new__(PagedDecoder)
    d.config, d.page_size, d.holders, d.pools = small_config(quant.Q8), PAGE, [0] * 6, []
    d.device = torch.device("cpu")
    d.stepped = []
    d._forward = lambda work: d.stepped.append([(s.length, list(s.pages)) for s, _, _ in work]) or torch.zeros(len(work), 4)
    monkeypatch.setattr(paged, "check_waits", lambda *a, **k: None)
    return d


def state(d, *seqs):
    return [(s.length, list(s.pages)) for s in seqs], list(d.holders)


def refused(name, f, *a):
    with pytest.raises(rt.QwcError) as e:
        f(*a)
    assert e.value.name == name


def tokens(n):
    return np.arange(n) % 5


def test_a_refused_step_changes_nothing(decoder):
    d = decoder
    a, b = d.start(), d.start()
    d.step([(a, tokens(20), None), (b, tokens(17), None)])
    before = state(d, a, b)
    c, pad = d.config, d.config.token_audio_pad
    rows = lambda n: np.zeros((n, c.text_hidden_size), np.float32)  # noqa: E731
    for name, work in (
        ("limit_exceeded", [(a, tokens(1), None), (b, tokens(16 * 5), None)]),           # the pool is too small
        ("limit_exceeded", [(a, tokens(30), None), (b, tokens(30), None)]),              # for both together
        ("limit_exceeded", [(a, tokens(1), None), (b, tokens(0), None)]),                # nothing to run
        ("limit_exceeded", [(a, tokens(1), None), (b, tokens(c.max_positions), None)]),  # too long
        ("invalid_argument", [(a, tokens(1), None), (a, tokens(1), None)]),              # twice the same sequence
        ("invalid_argument", [(a, tokens(1), None), (b, [c.vocab_size], None)]),         # rows that the embedding lacks
        ("invalid_argument", [(a, tokens(1), None), (b, [3, -1], None)]),
        ("invalid_argument", [(a, tokens(1), None), (b, [0.5], None)]),
        ("shape_mismatch", [(a, tokens(1), None), (b, np.zeros((1, 2), np.int64), None)]),
        ("shape_mismatch", [(a, [pad, 1], rows(2)), (b, [pad, pad], rows(1))]),          # another sequence's rows would be taken
        ("shape_mismatch", [(a, tokens(1), None), (b, [pad], np.zeros((1, 3), np.float32))]),
    ):
        refused(name, d.step, work)
        assert state(d, a, b) == before, work
    assert len(d.stepped) == 1
    d.step([(a, [pad, 1, pad], rows(2)), (b, tokens(3), None)])
    assert d.stepped[1] == [(23, a.pages), (20, b.pages)]
    assert d.step([]).shape == (0, c.vocab_size)


@pytest.mark.parametrize("where", ["layers", "waits"])
def test_a_step_that_fails_changes_nothing(decoder, monkeypatch, where):
    d = decoder
    a, b = d.start(), d.start()
    d.step([(a, tokens(20), None)])
    before = state(d, a, b)
    forward = d._forward

    def fail(*args, **kw):
        raise rt.QwcError(rt.STATUS_CODE["invalid_state"], "test")

    if where == "layers":
        d._forward = fail
    else:
        monkeypatch.setattr(paged, "check_waits", fail)
    refused("invalid_state", d.step, [(a, tokens(20), None), (b, tokens(5), None)])
    assert state(d, a, b) == before
    d._forward = forward
    monkeypatch.setattr(paged, "check_waits", lambda *args, **kw: None)
    d.step([(a, tokens(20), None), (b, tokens(5), None)])
    assert a.length == 40 and len(a.pages) == 3 and len(b.pages) == 1


def test_a_refused_fork_changes_nothing(decoder):
    d = decoder
    a, b = d.start(), d.start()
    d.step([(a, tokens(40), None), (b, tokens(48), None)])  # all six pages
    before = state(d, a, b)
    refused("limit_exceeded", d.fork, a)
    assert state(d, a, b) == before
    c = d.fork(b)  # full pages only: none is copied
    assert c.pages == b.pages and [d.holders[p] for p in b.pages] == [2, 2, 2]
    for s in (a, b, c):
        d.release(s)
    assert not any(d.holders)


def test_transcripts_that_fail_hold_no_pages(decoder):
    d = decoder

    class Prompt:
        tokens, audio = np.arange(17) % 5, None

    refused("limit_exceeded", lambda: d.transcripts(Prompt, 7, 4, torch.Generator()))  # two pages, then one for each fork
    assert not any(d.holders)
