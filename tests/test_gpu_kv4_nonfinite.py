"""NaN and infinities through the 4-bit cache on the B200: a value that is not finite makes its group of 64 dims NaN in the
cache, a query row that is not finite or sees such a key is not finite, and no other row is touched, whatever lies in the same
block of keys (the attention's tolerance is test_gpu_kv4's)."""
import numpy as np
import pytest

from tests import kv4_ref as R
from tests.test_gpu_kv4 import _case, _check, _poisoned, _rope, _rotate

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


FEW = [([300, 211], 5, 14, 2, 64, 16, "fp16"), ([17, 5, 0, 40], 16, 16, 8, 128, 64, "bf16"), ([700, 90], 1, 24, 3, 128, 48, "fp16"),
       ([190, 77], 30, 4, 2, 64, 32, "fp16")]
LINE = [([700, 3, 450, 90] * 16, 1, 32, 8, 128, 64, "fp16"), ([300, 17, 211, 64] * 16, 5, 32, 8, 64, 16, "bf16"),
        ([300, 17, 211, 64] * 8, 12, 32, 8, 128, 64, "fp16")]
MANY = [([333], 100, 14, 2, 64, 48, "bf16"), ([260, 130], 128, 32, 8, 128, 64, "fp16"), ([64, 65, 200] * 3, 64, 8, 8, 128, 64, "fp16")]


def _entry(torch, cache, table, b, t, which):
    """The fp16 {scale, bias} pairs [kv_heads, groups, 2] of token t of sequence b, as a view of the cache."""
    hd, P = cache.head_dim, cache.page_size
    tiles = cache.data.view(cache.pages, cache.kv_heads, P // 16, -1)
    page = tiles[int(table[b, t // P]), :, t % P // 16]
    return page[:, 16 * hd:].view(torch.float16).view(cache.kv_heads, 16, 2, hd // 64, 2)[:, t % 16, which]


@pytest.mark.parametrize("lens,n,H,KVH,hd,page,dtype", FEW + LINE + MANY)
@pytest.mark.parametrize("which,part,bad", [(0, 0, "nan"), (0, 1, "nan"), (1, 0, "nan"), (1, 1, "nan"), (1, 0, "inf"),
                                            (1, 1, "-inf")])
def test_attention_keys(torch, lens, n, H, KVH, hd, page, dtype, which, part, bad):
    """One scale or bias of K (which = 0) or V of some keys is not finite, in one KV head and one group of dims."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(n + hd + 10 * which + part)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    cache, table, q, seqs = _case(torch, rng, lens, n, H, KVH, hd, page, dt)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    host = table.cpu().numpy()
    G, per = hd // 64, H // KVH
    hit = []                                              # (sequence, key, KV head, group)
    for b, L in list(enumerate(lens))[:4]:
        if L:
            t = [L - 1, max(0, L - 1 - n // 2), max(0, L - n + 1)][b % 3]
            j, g = int(rng.integers(KVH)), int(rng.integers(G))
            _entry(torch, cache, host, b, t, which)[j, g, part] = float(bad)
            hit.append((b, t, j, g))
    out = kv4.attention(q, cache, table, lt)
    kv4.check_errors()
    got = out.float().cpu().numpy().reshape(len(lens), n, H, hd)
    clean = out.clone().view(len(lens), n, H, hd)
    for b, t, j, g in hit:
        first = max(0, t - (lens[b] - n))                 # the first row that sees key t
        dims = slice(0, hd) if which == 0 else slice(64 * g, 64 * g + 64)
        heads = slice(j * per, (j + 1) * per)
        assert not np.isfinite(got[b, first:, heads, dims]).any(), (b, t, j, g)
        if which:                                         # the other group of those rows
            rest = np.delete(got[b, first:, heads], np.r_[dims], -1)
            assert np.isfinite(rest).all()
        # rows that see it are left out of the comparison below
        K, V, pairs = seqs[b]
        want = torch.from_numpy(R.attention(q[b].float().cpu().numpy(), K, V, lens[b])).to(out.dtype).cuda()
        clean[b, first:, heads] = want[first:, heads]
    _check(torch, clean.view(q.shape), q, seqs, lens)
    again = kv4.attention(q, cache, table, lt)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("lens,n,H,KVH,hd,page,dtype", FEW + LINE + MANY)
def test_attention_queries(torch, lens, n, H, KVH, hd, page, dtype):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(n + hd)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    cache, table, q, seqs = _case(torch, rng, lens, n, H, KVH, hd, page, dt)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    bad = q.clone()
    hit = []
    for b, L in list(enumerate(lens))[:4]:
        i, h = n - 1 if b % 2 else n - 1 - n // 3, int(rng.integers(H))
        if L - n + i >= 0:
            bad[b, i, h, int(rng.integers(hd))] = [float("nan"), float("inf"), float("-inf")][b % 3]
            hit.append((b, i, h))
    assert hit
    out = kv4.attention(bad, cache, table, lt)
    kv4.check_errors()
    for b, i, h in hit:
        assert bool(out[b, i, h].isnan().all()), (b, i, h)
        out[b, i, h] = torch.from_numpy(R.attention(q[b].float().cpu().numpy(), *seqs[b][:2], lens[b])[i, h]).cuda()
    _check(torch, out, q, seqs, lens)
