"""The 4-bit attention's path of many sequences on the B200: the blocks of all items on one line, equal shares a CTA, pieces in the
workspace joined by a second kernel. Every case asserts that it takes this path (it is the one that needs a workspace), on
poisoned caches, against 64 bits within test_gpu_kv4's bound."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_kv4 import _case, _check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def _ragged(seed, B, most):
    lens = np.random.default_rng(seed).integers(0, most + 1, B)
    lens[[0, 3, B - 1]] = 0
    lens[[1, 5]] = [most, 1]
    return lens.tolist()


def _on_the_line(cache):
    return all(v > 0 for v in cache._workspace.values()) and len(cache._workspace) > 0


CASES = [
    (_ragged(1, 128, 1792), 1, 14, 2, 64, 16, "fp16", "normal"),
    (_ragged(2, 40, 700), 1, 32, 8, 128, 64, "fp16", "normal"),
    (_ragged(3, 40, 700), 5, 32, 8, 128, 48, "bf16", "normal"),         # twenty columns a KV head, in two blocks
    (_ragged(4, 90, 500), 5, 14, 2, 64, 32, "fp16", "normal"),          # thirty-five columns, the last block of them short
    (_ragged(5, 64, 400), 3, 8, 8, 64, 16, "bf16", "normal"),
    (_ragged(6, 300, 260), 1, 12, 1, 128, 128, "fp16", "normal"),       # twelve heads on one KV head
    ([8192] + [1] * 63, 1, 32, 8, 128, 64, "fp16", "normal"),           # an item of many pieces
    ([1, 0] * 20 + [6000] + [130] * 23, 4, 16, 8, 64, 64, "bf16", "normal"),
    ([129] * 64, 1, 32, 8, 128, 16, "fp16", "normal"),                  # two blocks each, the second of one key
    (_ragged(7, 60, 600), 1, 32, 8, 128, 64, "fp16", "spread"),
    (_ragged(8, 60, 600), 1, 32, 8, 64, 64, "bf16", "peaks"),
    (_ragged(9, 40, 600), 6, 16, 8, 128, 64, "fp16", "peaks"),
]


@pytest.mark.parametrize("lens,n,H,KVH,hd,page,dtype,kind", CASES)
def test_values(torch, lens, n, H, KVH, hd, page, dtype, kind):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(len(lens) * 100 + n + hd)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    cache, table, q, seqs = _case(torch, rng, lens, n, H, KVH, hd, page, dt, kind)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = kv4.attention(q, cache, table, lt)
    assert _on_the_line(cache)
    kv4.check_errors()
    _check(torch, out, q, seqs, lens)
    for b, L in enumerate(lens):
        if L == 0:
            assert bool((out[b] == 0).all())
    for _ in range(3):                                                   # in whatever memory the pieces lie
        assert torch.equal(out, kv4.attention(q, cache, table, lt))


def test_no_tokens_at_all(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(1)
    lens = [0] * 64
    cache, table, q, seqs = _case(torch, rng, [700] + [0] * 63, 1, 32, 8, 128, 64, torch.float16)
    out = torch.full_like(q, float("nan"))
    kv4.attention(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out=out)
    assert _on_the_line(cache)
    kv4.check_errors()
    assert bool((out == 0).all())


def test_bad_lengths_and_pages(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(9)
    lens = [192] * 64
    cache, table, q, seqs = _case(torch, rng, lens, 1, 32, 8, 128, 64, torch.float16)
    table = table[:, :3].contiguous()
    length = lambda at, L: torch.tensor(lens[:at] + [L] + lens[at + 1:], dtype=torch.int32, device="cuda")  # noqa: E731
    for L in (1 << 30, 193):                                            # clamped to what the table can hold
        out = kv4.attention(q, cache, table, length(7, L))
        assert _on_the_line(cache)
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        _check(torch, out, q, seqs, lens)
    out = kv4.attention(q, cache, table, length(7, -5))
    with pytest.raises(RuntimeError, match="out of range"):
        kv4.check_errors()
    assert bool((out[7] == 0).all())
    keep = [b for b in range(64) if b != 7]
    rest = lambda o: _check(torch, o[keep], q[keep], [seqs[b] for b in keep], [192] * 63)  # noqa: E731
    rest(out)
    for page in (-1, cache.pages):                                      # pages outside the cache: no keys from them
        t2 = table.clone()
        t2[7] = page
        out = kv4.attention(q, cache, t2, length(7, 192))
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        assert bool((out[7] == 0).all())
        rest(out)
        t2 = table.clone()
        t2[7, 1] = page                                                 # one of three: the others' keys
        out = kv4.attention(q, cache, t2, length(7, 192))
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        K, V, pairs = seqs[7]
        left = np.r_[0:64, 128:192]
        # the same keys as a sequence of 128 tokens
        _check(torch, out[7:8], q[7:8], [(K[left], V[left], [p[left] for p in pairs])], [128])
        rest(out)


@pytest.mark.parametrize("n", [1, 5])
def test_in_a_graph(torch, n):
    """Captured once, replayed with other lengths: the shares, the pieces and the join follow them."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(4 + n)
    lens = _ragged(11, 60, 400)
    cache, table, q, seqs = _case(torch, rng, lens, n, 32, 8, 128, 64, torch.float16)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv4.attention(q, cache, table, lt)
    assert _on_the_line(cache)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kv4.attention(q, cache, table, lt)
    cuts = [lens, [min(L, 17) for L in lens], [0] * 59 + [lens[59]], [L if b == 1 else 0 for b, L in enumerate(lens)],
            [max(0, L - 129) for L in lens]]
    for cut in cuts:
        lt.copy_(torch.tensor(cut, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        _check(torch, out, q, [(K[:L], V[:L], [p[:L] for p in pr]) for (K, V, pr), L in zip(seqs, cut)], cut)
    kv4.check_errors()


def test_side_stream(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(3)
    lens = _ragged(12, 64, 300)
    cache, table, q, seqs = _case(torch, rng, lens, 1, 32, 8, 128, 64, torch.float16)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late, lengths = torch.zeros_like(q), torch.zeros_like(lt)
        torch.cuda._sleep(2_000_000)
        late.copy_(q)
        lengths.copy_(lt)
        out = kv4.attention(late, cache, table, lengths)
    side.synchronize()
    assert _on_the_line(cache)
    _check(torch, out, q, seqs, lens)


def test_the_workspace_is_refused_where_it_does_not_do(torch):
    from agxforge.kernels import kv4
    from agxforge_b200 import _native as N
    L, ctx = N.lib(), N.context(0)
    c = kv4.KV4Cache(64, 8, 128, 64)
    q = torch.zeros((64, 32, 128), dtype=torch.float16, device="cuda")
    table = torch.zeros((64, 40), dtype=torch.int32, device="cuda")
    lens = torch.ones(64, dtype=torch.int32, device="cuda")
    a = N.Kv4AttentionArgs(c._c, q.data_ptr(), q.data_ptr(), N.F16, 64, 1, 32, table.data_ptr(), 40, 40, lens.data_ptr(), None, 0)
    need = L.agxc_kv4_attention_workspace(ctx, C.byref(a))
    assert need > 0
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    for at, size in [(0, 0), (None, need), (0, need - 1), (8, need)]:
        a.workspace_dev, a.workspace_bytes = (None if at is None else ws.data_ptr() + at), size
        assert L.agxc_kv4_attention_dev(ctx, C.byref(a), 1) == N.EINVAL
    a.workspace_dev, a.workspace_bytes = ws.data_ptr(), need
    assert L.agxc_kv4_attention_dev(ctx, C.byref(a), 1) == 0
    kv4.check_errors()
