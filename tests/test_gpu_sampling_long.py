"""Sampling over vocabularies that a cluster's shared memory does not hold in fp32 (the rest is read again from global memory), on
the B200, within test_gpu_sampling's bound."""
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


@pytest.mark.parametrize("V", [1 << 20, (1 << 20) - 1, 1000003])
def test_options(torch, V):
    from agxforge.kernels import sampling
    rng = np.random.default_rng(V)
    B = 4
    x = _logits(rng, B, V)
    x[1, ::5] = np.nan
    x[1, 7::11] = -np.inf
    x[2, V - 3] = x[2].max() + 1                          # the largest among what is read again
    wide = torch.zeros((B, V + 5), device="cuda")
    wide[:, 3:3 + V] = torch.from_numpy(x).cuda()
    for T, k, p, least in [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 30000, 0.95, 0.0),
                           (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0), (5.0, 0, 0.99, 0.0)]:
        u = rng.random(B, np.float32)
        token, prob = sampling.sample(wide[:, 3:3 + V], torch.from_numpy(u).cuda(), T, k, p, least)
        for r in range(B):
            check_row(x[r], u[r], T, k, p, least, int(token[r]), float(prob[r]))


def test_structured_rows(torch):
    """Infinities, one value all over, nothing at all: exact answers, on both sides of what shared memory holds."""
    from agxforge.kernels import sampling
    V, n = 1 << 20, 16
    x = torch.full((7, V), -float("inf"), device="cuda")
    x[1] = 1.5
    at = torch.arange(0, V, V // n, device="cuda") + V // n - 1           # the last of each CTA's range
    x[2, at] = float("inf")
    x[3, at] = 2.0
    x[4] = float("nan")
    x[4, V - 1] = -3.0
    x[5] = -1.0
    x[5, at] = float("nan")
    x[5, at[1:3]] = float("inf")
    x[6, at[-1]] = 0.0
    for u in (0.0, 0.3, 0.5, 1 - 2.0 ** -24):
        for k, p in [(0, 1.0), (5, 1.0), (0, 0.5), (V - 1, 0.75)]:
            token, prob = sampling.sample(x, torch.full((7,), u, device="cuda"), 0.9, k, p)
            token, prob = token.tolist(), prob.tolist()
            assert token[0] == -1 and prob[0] == 0
            for r, where in ((1, None), (2, at), (3, at), (5, at[1:3])):
                m = V if where is None else where.numel()
                m = k if 0 < k < m else m
                m = max(1, -(-int(np.ceil(p * m * 2.0 ** 40)) // 2 ** 40)) if p < 1 else m
                i = int(np.float64(np.float32(u)) * (m * 2.0 ** 40)) >> 40
                assert token[r] == (i if where is None else int(where[i])), (u, k, p, r)
                assert prob[r] == np.float32(1.0 / m)
            assert (token[4], prob[4]) == (V - 1, 1.0) and (token[6], prob[6]) == (int(at[-1]), 1.0)
