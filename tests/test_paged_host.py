"""PagedModel's bookkeeping on the host, with stand-ins for its device passes: what a step that cannot give its tokens leaves
behind."""
import contextlib

import pytest
import torch

from agxforge.inference import paged
from agxforge.kernels import kv4


class Shape:
    VOCAB, EPS = 100, 1e-6


@pytest.fixture
def model(monkeypatch):
    """A model of two sequences whose passes count rows and whose sampler gives `model.tokens`."""
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda d=None: None)
    m = paged.PagedModel.__new__(paged.PagedModel)
    m.device, m.shape, m.seqs, m._next, m.spare, m.page_size = 0, Shape, {}, 0, list(range(8)), 16
    m.head = m.final_gain = None
    m.passes, m.tokens = [], None

    def rows(ids, n):
        m.passes.append([(s, m.seqs[s]["held"], m.seqs[s]["tokens"][m.seqs[s]["held"]:m.seqs[s]["held"] + n]) for s in ids])
        for s in ids:
            m._reserve(s, m.seqs[s]["held"] + n)
            m.seqs[s]["held"] += n
        return torch.zeros(len(ids), 4)

    def sample(lg, u, *options):
        if u.numel() != lg.shape[0]:
            raise ValueError("sample: u is contiguous float32 [batch] on the logits' device")
        return torch.tensor(m.tokens[:lg.shape[0]], dtype=torch.int32), torch.full((lg.shape[0],), 0.5)

    monkeypatch.setattr(kv4, "check_errors", lambda device=0: None)
    monkeypatch.setattr(paged.sampling, "sample", sample)
    m._rows = rows
    m._gemv = lambda pack, x, **kw: torch.zeros(x.shape[0], 100)
    m.add([1, 2, 3])
    m.add([4])
    return m


def state(m):
    return {s: (q["held"], list(q["tokens"])) for s, q in m.seqs.items()}


def test_a_refused_step_can_be_asked_for_again(model):
    before = state(model)
    with pytest.raises(ValueError, match="u is"):
        model.step([0.5])                                 # one number for two sequences
    assert state(model) == before
    model.tokens = [7, 8]
    assert model.step([0.5, 0.5]) == {0: (7, 0.5), 1: (8, 0.5)}
    assert model.passes[-1] == model.passes[-2]           # the same rows at the same places
    assert state(model) == {0: (3, [1, 2, 3, 7]), 1: (1, [4, 8])}


def test_a_row_without_a_token_is_no_token(model):
    """Token -1 (no finite logit, or a min_p above 1) is no index of the embedding."""
    before = state(model)
    model.tokens = [7, -1]
    with pytest.raises(RuntimeError, match=r"no token for sequence 1\b"):
        model.step([0.5, 0.5], min_p=2.0)
    assert state(model) == before
    model.tokens = [7, 8]
    assert model.step([0.5, 0.5])[1] == (8, 0.5)


def test_a_pass_that_went_wrong_on_the_device_raises(model, monkeypatch):
    """A wait that gave up, a page out of range: nothing is returned, nothing counts as held."""
    before = state(model)
    model.tokens = [7, 8]
    bad = []

    def check(device=0):
        if bad:
            raise TimeoutError(bad.pop())

    monkeypatch.setattr(kv4, "check_errors", check)
    for call in (lambda: model.step([0.5, 0.5]), lambda: model.logits()):
        bad.append("a bounded device wait gave up")
        with pytest.raises(TimeoutError, match="gave up"):
            call()
        assert state(model) == before and not bad
    spare = list(model.spare)
    bad.append("a bounded device wait gave up")
    with pytest.raises(TimeoutError):
        model.add([5, 6, 7])
    assert state(model) == before and model.spare == spare
    assert model.step([0.5, 0.5]) == {0: (7, 0.5), 1: (8, 0.5)}


def test_a_sequence_named_twice_is_refused(model):
    """Its one new token would be two rows at two places, the second past its end."""
    before = state(model)
    model.tokens = [7, 8]
    for call in (lambda: model.logits([0, 0]), lambda: model.step([0.5, 0.5, 0.5], [1, 0, 1])):
        with pytest.raises(ValueError, match="twice"):
            call()
    assert state(model) == before
    assert model.step([0.5, 0.5], [1, 0]) == {1: (7, 0.5), 0: (8, 0.5)}
