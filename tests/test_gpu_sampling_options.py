"""Options at the ends of their ranges, on the B200: values that are no temperature."""
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
