"""Options at the ends of their ranges, on the B200: temperatures below fp32's normal numbers, values that are no temperature,
and a top_k past 32 bits."""
import numpy as np
import pytest

from tests.test_gpu_sampling import _logits, check_row

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T", [1e-30, 1e-37, 1.1754944e-38, 1e-38, 3e-39, 1e-40, 1.4e-45])
def test_the_smallest_temperatures(torch, T, dtype):
    """All the weight on the maximum: at these temperatures any other logit is further below than 2^-40 reaches."""
    from agxforge.kernels import sampling
    rng = np.random.default_rng(3)
    x = torch.from_numpy(_logits(rng, 5, 5003)).to(getattr(torch, dtype)).cuda()
    x[torch.arange(5), torch.tensor([0, 17, 4000, 5002, 333])] = 40.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    array = torch.full((5,), T, device="cuda")
    assert bool((array > 0).all())
    for t in (T, array):
        for k, p, least in [(0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (7, 0.9, 0.05)]:
            token, prob = sampling.sample(x, u, t, k, p, least)
            assert token.tolist() == [0, 17, 4000, 5002, 333] and prob.tolist() == [1.0] * 5, (k, p, least)


def test_values_that_are_no_temperature(torch):
    """Below zero or NaN in a device array: no token, the error word set, the other rows as they are."""
    from agxforge.kernels import kv4, sampling
    rng = np.random.default_rng(4)
    B, V = 9, 50257
    x = torch.from_numpy(_logits(rng, B, V)).cuda()
    x[4] = 0.5
    u = torch.from_numpy(rng.random(B, np.float32)).cuda()
    T = torch.tensor([1.0, -1.0, 0.0, float("nan"), -0.5, 0.7, -float("inf"), -1e-40, float("inf")], device="cuda")
    bad = [1, 3, 4, 6, 7]
    kv4.check_errors()
    for k, p in [(0, 1.0), (50, 0.9), (0, 0.95)]:
        token, prob = sampling.sample(x, u, T, k, p)
        with pytest.raises(RuntimeError, match="option"):
            kv4.check_errors()
        assert token[bad].tolist() == [-1] * 5 and prob[bad].tolist() == [0.0] * 5
        for r in (0, 2, 5):
            check_row(x[r].cpu().numpy(), float(u[r]), float(T[r]), k, p, 0.0, int(token[r]), float(prob[r]))
        assert int(token[8]) >= 0
    T[T < 0] = -0.0                                                   # a zero of either sign is greedy
    token, _ = sampling.sample(x, u, torch.nan_to_num(T, 0.0), 0, 1.0)
    kv4.check_errors()
    assert token[[1, 2, 3, 6, 7]].tolist() == x[[1, 2, 3, 6, 7]].argmax(-1).tolist()
    for t in (-1.0, float("nan"), -1e-40):
        with pytest.raises(ValueError, match="temperature"):
            sampling.sample(x, u, t)


def test_top_k_past_32_bits(torch):
    from agxforge.kernels import sampling
    rng = np.random.default_rng(5)
    x = torch.from_numpy(_logits(rng, 3, 1000)).cuda()
    u = torch.tensor([0.1, 0.5, 0.9], device="cuda")
    want = sampling.sample(x, u, 2.0)
    for k in (1000, (1 << 31) - 1, 1 << 31, (1 << 32) + 1, 1 << 40, -(1 << 31) - 1, -(1 << 32) + 1):
        got = sampling.sample(x, u, 2.0, k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), k
