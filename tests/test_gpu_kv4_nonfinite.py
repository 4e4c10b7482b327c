"""NaN and infinities through the 4-bit cache on the B200: a value that is not finite makes its group of 64 dims NaN or
infinite in the cache."""
import numpy as np
import pytest

from tests import kv4_ref as R
from tests.test_gpu_kv4 import _poisoned, _rope, _rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_append(torch, hd, dtype):
    """The groups that hold a NaN or an infinity read back as the definition gives them, the others as ever."""
    from agxforge.kernels import kv4
    T, H, KVH, page = 40, 4, 2, 16
    rng = np.random.default_rng(hd)
    x = rng.standard_normal((T, H + 2 * KVH, hd)).astype(np.float32)
    for t, bad in enumerate([np.nan, np.inf, -np.inf, np.nan, np.nan]):
        x[3 * t, H + t % KVH, (37 * t + 5) % hd] = bad               # a key's: both dims of its RoPE pair
        x[3 * t + 1, H + KVH + t % KVH, (29 * t + 2) % hd] = bad     # a value's
    x[20, H + KVH] = np.nan
    x[21, H + KVH, :64] = -np.nan
    rows = torch.from_numpy(x.reshape(T, -1)).cuda().to(getattr(torch, dtype))
    x = rows.float().cpu().numpy().reshape(x.shape)
    cos, sin = _rope(rng, T, hd)
    cache = _poisoned(torch, -(-T // page), KVH, hd, page)
    slots = torch.arange(T, device="cuda")
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    kv4.append(cache, rows, dev(np.arange(T, dtype=np.int32)), slots, dev(cos), dev(sin), H)
    got = [a.cpu().numpy().astype(np.float64) for a in cache.rows(slots)]
    kv4.check_errors()
    with np.errstate(all="ignore"):
        rot = _rotate(x[:, :H + KVH], cos, sin)
        for g, src in zip(got, (rot[:, H:], x[:, H + KVH:])):
            want = R.values(*R.quantise(src)).astype(np.float32).astype(np.float16).astype(np.float64)
            assert np.array_equal(g, want, equal_nan=True)
            broken = ~np.isfinite(src.reshape(T, KVH, -1, 64)).all(-1)
            assert broken.sum() >= 5
            assert not np.isfinite(g.reshape(T, KVH, -1, 64)[broken]).any()
            assert np.isfinite(g.reshape(T, KVH, -1, 64)[~broken]).all()
