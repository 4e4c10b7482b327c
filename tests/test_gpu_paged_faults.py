"""What PagedModel does where a step cannot give its tokens, on the B200: the sequences stay as they were, and the step asked
for again gives what a model that never failed gives."""
import numpy as np
import pytest

from tests.test_gpu_paged import _weights

pytestmark = pytest.mark.gpu

SHAPE = dict(NAME="paged", D_MODEL=256, LAYERS=1, HEADS=4, KV_HEADS=2, HEAD_DIM=64, FFN=512, VOCAB=1024, ROPE_THETA=1e6,
             EPS=1e-6)


@pytest.fixture
def twins():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from agxforge.inference import paged
    packs, _ = _weights(SHAPE, 3)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 1024, n).tolist() for n in (5, 33)]
    a, b = (paged.PagedModel(dict(model=SHAPE, bits=4), packs, pages=16, page_size=32) for _ in range(2))
    for m in (a, b):
        for p in prompts:
            m.add(p)
    return a, b


def test_refused_options_lose_nothing(twins):
    a, b = twins
    u = np.array([0.3, 0.6], np.float32)
    for bad in (dict(u=u[:1]), dict(u=u, temperature=-1.0)):
        with pytest.raises(ValueError):
            a.step(**bad)
    for _ in range(3):
        assert a.step(u, top_k=20) == b.step(u, top_k=20)


def test_no_token(twins):
    """A row that keeps nothing (min_p above 1) and rows of NaN logits raise; no sequence goes on from token -1."""
    a, b = twins
    u = [0.3, 0.6]
    with pytest.raises(RuntimeError, match="no token"):
        a.step(u, min_p=2.0)
    gain = a.final_gain.clone()
    a.final_gain.fill_(float("nan"))
    with pytest.raises(RuntimeError, match="no token"):
        a.step(u)
    a.final_gain.copy_(gain)
    for _ in range(3):
        got = a.step(u, temperature=0.8)
        assert got == b.step(u, temperature=0.8) and min(t for t, _ in got.values()) >= 0


def test_the_error_word_is_read(twins):
    """A page outside the cache in a sequence's table: its keys would be missing without a word."""
    a, b = twins
    pages = a.seqs[0]["pages"]
    good = pages[0]
    for call in (lambda: a.step([0.3, 0.6]), a.logits):
        pages[0] = 1000
        with pytest.raises(RuntimeError, match="out of range"):
            call()
        pages[0] = good
    assert a.step([0.3, 0.6]) == b.step([0.3, 0.6])
