"""The 4-bit cache's host side: sizes, the byte order's description, and the native refusals that need no GPU."""
import ctypes as C

import numpy as np
import pytest

from agxforge_b200 import _native as N
from tests import kv4_ref as R


@pytest.fixture(scope="module")
def lib():
    from agxforge_b200 import build
    build.build()
    return N.lib()


@pytest.mark.parametrize("hd", [64, 128])
def test_tile_bytes_are_used_once(hd):
    k, v = R.offsets(hd)
    every = np.concatenate([np.unique(k), np.unique(v)])
    assert np.array_equal(np.sort(every), np.arange(16 * hd))           # two dims a byte, no byte twice
    assert R.tile_bytes(hd) == 16 * hd + 16 * 2 * 4 * (hd // 64)


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_pack_and_values(hd):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 16, hd)).astype(np.float32)
    codes, pairs = R.quantise(x)
    step = pairs[..., 0].astype(np.float64).repeat(64, -1)
    assert np.all(np.abs(R.values(codes, pairs) - x) <= 0.51 * step + 1e-3)
    tiles = R.pack_tiles(codes, codes[:, ::-1], pairs, pairs)
    k, v = R.offsets(hd)
    for d in range(hd):
        assert np.array_equal(tiles[:, k[:, d]] >> (4 * (d & 1)) & 15, codes[..., d])
        assert np.array_equal(tiles[:, v[:, d]] >> (4 * (d & 1)) & 15, codes[:, ::-1, d])


def test_bytes(lib):
    from agxforge.kernels import kv4
    for pages, kvh, hd, page in [(1, 1, 64, 16), (7, 8, 128, 64), (3, 2, 64, 48)]:
        c = N.Kv4Cache(None, pages, kvh, hd, page)
        assert lib.agxc_kv4_bytes(C.byref(c)) == pages * kvh * page * kv4.token_bytes(hd)
    for bad in [(1, 1, 96, 16), (1, 1, 64, 8), (1, 1, 64, 0), (0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 64, 24)]:
        assert lib.agxc_kv4_bytes(C.byref(N.Kv4Cache(None, *bad))) == -1
    assert lib.agxc_kv4_bytes(None) == -1
    with pytest.raises(ValueError, match="head_dim"):
        kv4.token_bytes(96)


def test_null_arguments(lib):
    assert lib.agxc_kv4_append_dev(None, None, None) == N.EINVAL
    assert lib.agxc_kv4_attention_dev(None, None, None) == N.EINVAL
    assert lib.agxc_kv4_attention_workspace(None, None) == N.EINVAL
    assert lib.agxc_kv4_rows_dev(None, None, None, 1, None, None, None) == N.EINVAL
    assert lib.agxc_sample_dev(None, None, None) == N.EINVAL
    with pytest.raises(ValueError, match="null"):
        N.check(N.EINVAL, "sample")


def test_host_tensors_are_refused():
    import torch

    from agxforge.kernels import kv4, sampling
    with pytest.raises(ValueError, match="on the GPU"):
        sampling.sample(torch.zeros(1, 4), torch.zeros(1))
    with pytest.raises(ValueError, match="on the GPU"):
        kv4.KV4Cache.of(torch.zeros((1, 1, 16 * kv4.token_bytes(64)), dtype=torch.uint8), 64, 16)
