"""The paged 4-bit KV cache on the B200: the append against its fp32 restatement bit for bit and against 64 bits within
half a code, the attention against the 64-bit softmax over the cache's exact values, and the refusals of both.

Every cache is filled with NaN scales and biases first and only the places in use are written, unused page-table entries
are out of range, and pages are handed out in a shuffled order: a read of any of it shows."""
import math

import numpy as np
import pytest

from tests import kv4_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def _rope(rng, n, hd):
    ang = rng.uniform(0, 2 * np.pi, (n, hd // 2))
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def _rotate(x, cos, sin):
    """fp32, each product and sum rounded: x [T, heads, hd], cos and sin [T, hd / 2]."""
    h = x.shape[-1] // 2
    x1, x2, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return np.concatenate([x1 * c - x2 * s, x2 * c + x1 * s], -1)


def _poisoned(torch, pages, kvh, hd, page):
    from agxforge.kernels import kv4
    data = torch.zeros((pages, kvh, page // 16, R.tile_bytes(hd)), dtype=torch.uint8, device="cuda")
    data[..., 16 * hd:].view(torch.float16).fill_(float("nan"))
    return kv4.KV4Cache.of(data.view(pages, kvh, -1), hd, page)


TYPES = {"fp32": np.float32, "fp16": np.float16, "bf16": None}


@pytest.mark.parametrize("T,H,KVH,hd,page,dtype,bias,norm", [
    (1, 16, 8, 128, 64, "fp32", False, False),
    (1, 14, 2, 64, 16, "fp16", True, False),
    (5, 3, 3, 64, 32, "bf16", False, True),
    (33, 32, 8, 128, 16, "fp32", True, True),
    (130, 7, 1, 128, 48, "bf16", True, False),
    (257, 14, 2, 64, 128, "fp32", True, False),
    (1000, 6, 2, 128, 64, "fp16", False, False),
])
def test_append(torch, T, H, KVH, hd, page, dtype, bias, norm):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(T * 7 + hd)
    W = (H + 2 * KVH) * hd
    x = rng.standard_normal((T, W)).astype(np.float32)
    x[0, H * hd:H * hd + 64] = 0.25                     # a constant group (before the rotation, K) and one of V
    x[0, (H + KVH) * hd:(H + KVH) * hd + 64] = -3.0
    x[T // 2, -hd:] *= 1e-9                             # a group whose scale rounds to zero in 16 bits
    t = torch.from_numpy(x).cuda()
    t = t.to({"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}[dtype])
    wide = torch.zeros((T, W + 24), dtype=t.dtype, device="cuda")
    wide[:, 8:8 + W] = t                                # strided rows, off their 16-byte boundary
    rows = wide[:, 8:8 + W]
    x = t.float().cpu().numpy()
    cos, sin = _rope(rng, 50, hd)
    pos = rng.integers(0, 50, T).astype(np.int32)
    pages = -(-T // page) + 2
    cache = _poisoned(torch, pages, KVH, hd, page)
    before = cache.data.clone()
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    if T > 4:
        slots[rng.integers(0, T, T // 5)] = -1
    b = rng.standard_normal(W).astype(np.float16) if bias else None
    gains = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2)] if norm else [None, None]
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
    q = kv4.append(cache, rows, dev(pos), dev(slots), dev(cos), dev(sin), H, bias=dev(b), q_norm=dev(gains[0]),
                   k_norm=dev(gains[1]), eps=1e-5)
    k, v = cache.rows(dev(slots))
    kv4.check_errors()
    assert q.dtype == (torch.bfloat16 if dtype == "bf16" else torch.float16) and q.shape == (T, H, hd)

    x = x + b.astype(np.float32) if bias else x
    x = x.reshape(T, H + 2 * KVH, hd)
    if norm:
        for part, g in ((slice(0, H), gains[0]), (slice(H, H + KVH), gains[1])):
            y = x[:, part].astype(np.float64)
            x[:, part] = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-5) * g.astype(np.float64)
    rot = _rotate(x[:, :H + KVH], cos[pos], sin[pos])
    scaled = rot[:, :H] * np.float32(R.LOG2E / math.sqrt(hd))
    got_q = q.float().cpu().numpy()
    got = [k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)]
    used = slots >= 0
    for i, src in enumerate((rot[:, H:], x[:, H + KVH:])):
        codes, pairs = R.quantise(src)
        want = R.values(codes, pairs)
        assert np.all(got[i][~used] == 0)
        if norm and i == 0:        # the norm's sum of squares in another order: a code may move by one at a tie
            step = pairs[..., 0].astype(np.float64).repeat(64, -1)
            off = np.abs(got[i] - want)[used]
            assert np.all(off <= (1.001 * step + 2.0 ** -10 * np.abs(want) + 1e-6)[used])
            assert np.mean(off > 2.0 ** -9 * (1 + np.abs(want[used]))) < 1e-3
        else:
            assert np.array_equal(got[i][used], want[used].astype(np.float32).astype(np.float16).astype(np.float64))
        # against 64 bits: half a code, the 16-bit rounding of scale (15 codes of it) and bias, and of the read-back
        g = src.astype(np.float64).reshape(T, KVH, -1, 64)
        s = np.where(np.ptp(g, -1) > 0, np.ptp(g, -1) / 15, 1.0)
        tol = (0.5 * s + 15 * s * 2.0 ** -11 + 15 * 2.0 ** -25 + 2.0 ** -11 * np.abs(g).max(-1) + 2.0 ** -24).repeat(64, -1)
        tol = tol.reshape(got[i].shape) + 2.0 ** -11 * np.abs(got[i])
        if norm and i == 0:
            tol = tol + 1e-5
        assert np.all(np.abs(got[i] - src)[used] <= tol[used])
    if norm:
        assert np.all(np.abs(got_q - scaled) <= (2.0 ** -7 if dtype == "bf16" else 2.0 ** -10) * np.abs(scaled) + 1e-6)
    else:
        want = torch.from_numpy(scaled).to(q.dtype).float().numpy()
        assert np.array_equal(got_q, want)
    # nothing else of the cache changed
    same = (cache.data.view(pages, KVH, page // 16, -1) == before.view(pages, KVH, page // 16, -1)).all(-1).cpu().numpy()
    touched = np.zeros((pages, page // 16), bool)
    for s in slots[used]:
        touched[s // page, s % page // 16] = True
    assert np.all(same[~touched.repeat(1).reshape(pages, -1)[:, None].repeat(KVH, 1)])
    free = torch.from_numpy(np.setdiff1d(np.arange(pages * page), slots[used])).cuda()
    kf, vf = cache.rows(free)
    assert bool(kf.isnan().all()) and bool(vf.isnan().all())


def test_append_order_and_stream(torch):
    """One call of T tokens and T calls of one token leave the same bytes; a call on a side stream is ordered there."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(5)
    T, H, KVH, hd, page = 40, 4, 2, 128, 16
    x = torch.from_numpy(rng.standard_normal((T, (H + 2 * KVH) * hd)).astype(np.float32)).cuda()
    cos, sin = (torch.from_numpy(a).cuda() for a in _rope(rng, T, hd))
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    slots = torch.from_numpy(rng.permutation(4 * page)[:T].astype(np.int64)).cuda()
    a, b = (kv4.KV4Cache(4, KVH, hd, page) for _ in range(2))
    qa = kv4.append(a, x, pos, slots, cos, sin, H)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.empty_like(x)
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        parts = [kv4.append(b, late[i:i + 1], pos[i:i + 1], slots[i:i + 1], cos, sin, H) for i in range(T)]
    side.synchronize()
    assert torch.equal(a.data, b.data) and torch.equal(qa, torch.cat(parts))


def test_append_refuses(torch):
    from agxforge.kernels import kv4
    c = kv4.KV4Cache(2, 2, 64, 16)
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    i32, i64 = torch.int32, torch.int64
    ok = dict(qkv=z(3, 8 * 64), positions=z(3, dtype=i32), slots=torch.arange(3, device="cuda"), cos=z(4, 32), sin=z(4, 32),
              heads=4)
    kv4.append(c, **ok)
    for bad, text in [(dict(heads=3), "multiple of kv_heads"), (dict(qkv=z(3, 100)), "qkv is"),
                      (dict(qkv=z(3, 8 * 64, dtype=i32)), "fp32, fp16 or bf16"), (dict(positions=z(3, dtype=i64)), "positions"),
                      (dict(slots=z(2, dtype=i64)), "one position and one slot"), (dict(cos=z(4, 16)), "cos and sin"),
                      (dict(bias=z(8 * 64)), "bias"), (dict(q_norm=z(64, dtype=torch.float16)), "neither"),
                      (dict(out=z(3, 4, 32, dtype=torch.float16)), "out is"), (dict(q_dtype=torch.float32), "q fp16 or bf16")]:
        with pytest.raises(ValueError, match=text):
            kv4.append(c, **dict(ok, **bad))
    for args, text in [((2, 2, 96), "head_dim"), ((2, 2, 64, 24), "page_size"), ((0, 2, 64), "one page")]:
        with pytest.raises(ValueError, match=text):
            kv4.KV4Cache(*args)
    with pytest.raises(ValueError, match="data is"):
        kv4.KV4Cache.of(z(2, 2, 100, dtype=torch.uint8), 64, 16)
    assert kv4.append(c, z(0, 8 * 64), z(0, dtype=i32), z(0, dtype=i64), z(4, 32), z(4, 32), 4).shape == (0, 4, 64)
    kv4.check_errors()


def test_append_out_of_range(torch):
    """A position past the tables or a slot past the cache leaves that token out, is reported, and harms no other."""
    from agxforge.kernels import kv4
    c = kv4.KV4Cache(2, 1, 64, 16)
    x = torch.randn(4, 3 * 64, device="cuda")
    cos, sin = torch.ones(8, 32, device="cuda"), torch.zeros(8, 32, device="cuda")
    for pos, slot in [([0, 8, 2, 3], [0, 1, 2, 3]), ([0, -1, 2, 3], [0, 1, 2, 3]), ([0, 1, 2, 3], [0, 32, 2, 3])]:
        c.data.zero_()
        kv4.append(c, x, torch.tensor(pos, dtype=torch.int32, device="cuda"), torch.tensor(slot, device="cuda"), cos, sin, 1)
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        k, _ = c.rows(torch.arange(4, device="cuda"))
        assert bool((k[1] == 0).all()) and bool((k[[0, 2, 3]] != 0).any(-1).all())
        kv4.check_errors()
    c.rows(torch.tensor([40], device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        kv4.check_errors()


def _case(torch, rng, lens, n, H, KVH, hd, page, dtype, kind="normal", spare=3):
    """A poisoned cache with sequences of `lens`, q, and the exact values: (cache, table, q, per sequence (K, V, pairs))."""
    B = len(lens)
    per = [-(-L // page) for L in lens]
    mp = max(1, max(per)) + 1
    pages = sum(per) + spare
    order = rng.permutation(pages)
    table = np.full((B, mp), 1 << 30, np.int32)                     # unused entries are out of range
    cache = _poisoned(torch, pages, KVH, hd, page)
    G, m = hd // 64, page // 16
    blocks = cache.data.view(pages, KVH, m, -1)
    seqs, at = [], 0
    for b, L in enumerate(lens):
        codes = [rng.integers(0, 16, (L, KVH, hd)).astype(np.uint8) for _ in range(2)]
        s = [rng.uniform(0.2, 0.4, (L, KVH, G)) for _ in range(2)]
        if kind == "spread":                                         # scales over five orders of magnitude in V
            s[1] = 10.0 ** rng.uniform(-4.5, 0.5, (L, KVH, G))
        if kind == "tiny":
            s[1] = np.full((L, KVH, G), 3e-7)
        pairs = [np.stack([x, -7.5 * x], -1).astype(np.float16) for x in s]
        if kind == "peaks":                                          # a few keys far above the rest, late ones highest
            hot = rng.integers(0, max(L, 1), 5)
            for r, t in enumerate(sorted(hot[:min(5, L)])):
                pairs[0][t, ..., 0] *= 4 + 4 * r
                pairs[0][t, ..., 1] *= 4 + 4 * r
        if kind == "flat":                                           # every scale zero: keys and values are their biases
            for x in pairs:
                x[..., 0] = 0
        K, V = (R.values(c, p) for c, p in zip(codes, pairs))
        full = per[b] * page
        pad = lambda a, v=0: np.concatenate([a, np.full((full - L,) + a.shape[1:], v, a.dtype)])  # noqa: E731
        shape = lambda a: a.reshape((per[b], m, 16) + a.shape[1:]).transpose(  # noqa: E731
            (0, 3, 1, 2) + tuple(range(4, a.ndim + 2)))
        if L:
            tiles = R.pack_tiles(shape(pad(codes[0])), shape(pad(codes[1])), shape(pad(pairs[0], np.nan)),
                                 shape(pad(pairs[1], np.nan)))
            mine = order[at:at + per[b]]
            blocks[torch.from_numpy(mine).cuda()] = torch.from_numpy(tiles).cuda()
            table[b, :per[b]] = mine
            at += per[b]
        seqs.append((K, V, pairs))
    q = (rng.standard_normal((B, n, H, hd)) * 1.5 * R.LOG2E / math.sqrt(hd)).astype(np.float32)
    if kind == "small q":
        q *= 1e-4
    q = torch.from_numpy(q).cuda().to(dtype)
    return cache, torch.from_numpy(table).cuda(), q, seqs


def _check(torch, got, q, seqs, lens):
    ulp = 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    got, qn = got.double().cpu().numpy().reshape(q.shape), q.float().cpu().numpy()
    for b, L in enumerate(lens):
        K, V, pairs = seqs[b]
        want = R.attention(qn[b], K, V, L)
        tol = R.attention_bound(qn[b], K, V, want, *pairs, ulp) + ulp * np.abs(want) + 2.0 ** -25
        off = np.abs(got[b] - want)
        assert np.all(off <= tol), (b, L, float(off.max()), float(tol.min()), float((off / tol).max()))


@pytest.mark.parametrize("lens,n,H,KVH,hd,page,dtype,kind", [
    ([1], 1, 16, 8, 128, 64, "fp16", "normal"),
    ([0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65], 1, 16, 8, 128, 64, "fp16", "normal"),
    ([0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 129, 300], 1, 14, 2, 64, 16, "fp16", "normal"),
    ([1000, 0, 3, 517], 1, 32, 8, 128, 16, "bf16", "normal"),
    ([2049], 1, 4, 4, 64, 128, "fp16", "normal"),
    ([700, 90], 1, 24, 3, 128, 48, "fp16", "normal"),
    ([333], 1, 12, 1, 128, 32, "fp16", "normal"),          # twelve heads on one KV head
    ([250, 129], 1, 40, 1, 64, 16, "bf16", "normal"),
    ([17, 5, 0, 40], 16, 16, 8, 128, 64, "fp16", "normal"),  # rows before the sequence begins
    ([300, 211], 5, 14, 2, 64, 16, "bf16", "normal"),
    ([64, 65, 200], 64, 4, 2, 128, 64, "fp16", "normal"),
    ([260], 256, 8, 2, 128, 64, "fp16", "normal"),
    ([190, 77], 77, 7, 1, 64, 32, "fp16", "normal"),
    ([600, 40], 1, 16, 8, 128, 64, "fp16", "spread"),
    ([600, 40], 1, 16, 8, 128, 64, "fp16", "tiny"),
    ([900, 40], 1, 16, 8, 128, 64, "fp16", "peaks"),
    ([900, 40], 3, 14, 2, 64, 64, "bf16", "peaks"),
    ([200], 1, 16, 8, 128, 64, "fp16", "flat"),
    ([200], 1, 16, 8, 128, 64, "bf16", "small q"),
])
def test_attention(torch, lens, n, H, KVH, hd, page, dtype, kind):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(len(lens) * 100 + n + hd)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    cache, table, q, seqs = _case(torch, rng, lens, n, H, KVH, hd, page, dt, kind)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    wide = torch.full((table.shape[0], table.shape[1] + 3), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out = kv4.attention(q, cache, wide[:, :table.shape[1]], lt)
    assert out.shape == q.shape and out.dtype == q.dtype
    kv4.check_errors()
    _check(torch, out, q, seqs, lens)
    again = kv4.attention(q, cache, table, lt)
    assert torch.equal(out, again)                                    # no order of addition left to chance
    if n == 1:
        flat = kv4.attention(q[:, 0], cache, table, lt)
        assert flat.shape == (len(lens), H, hd) and torch.equal(flat, out[:, 0])
    else:
        last = kv4.attention(q[:, -1:].contiguous(), cache, table, lt)
        _check(torch, last, q[:, -1:], seqs, lens)


@pytest.mark.parametrize("lens,n,H,KVH,hd,page,dtype,kind", [
    ([0, 1, 130, 64, 257], 96, 16, 8, 128, 64, "fp16", "normal"),   # rows before the sequence begins, one key
    ([2049], 80, 16, 8, 128, 16, "fp16", "normal"),                  # an item's keys over a cluster, a second block of columns
    ([333], 100, 14, 2, 64, 48, "bf16", "normal"),                   # pages that end inside a block of keys
    ([512], 512, 16, 8, 64, 16, "fp16", "normal"),                   # a prompt from its first token
    ([70, 3, 71, 200, 64, 128, 1, 90] * 3, 70, 8, 8, 128, 32, "fp16", "normal"),
    ([300, 90], 65, 40, 1, 64, 16, "bf16", "normal"),                # forty heads on one KV head
    ([1, 6, 0, 16] * 20, 10, 32, 8, 128, 16, "fp16", "normal"),      # many sequences of a block at most
    ([1, 6, 0, 16] * 20, 5, 32, 8, 128, 16, "bf16", "normal"),
    ([2, 30, 0, 17] * 20, 1, 32, 8, 64, 16, "fp16", "normal"),
    ([900, 40], 77, 32, 8, 128, 64, "fp16", "peaks"),
    ([900, 140], 150, 14, 2, 64, 64, "bf16", "peaks"),
    ([600, 40], 64, 32, 8, 128, 64, "fp16", "spread"),
    ([600, 40], 64, 32, 8, 64, 64, "fp16", "spread"),
    ([600], 64, 32, 8, 128, 64, "bf16", "tiny"),
    ([200], 64, 32, 8, 128, 64, "fp16", "flat"),
    ([200], 64, 32, 8, 128, 64, "bf16", "small q"),
])
def test_attention_many_rows(torch, lens, n, H, KVH, hd, page, dtype, kind):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(len(lens) * 100 + n + hd)
    dt = torch.float16 if dtype == "fp16" else torch.bfloat16
    cache, table, q, seqs = _case(torch, rng, lens, n, H, KVH, hd, page, dt, kind)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = kv4.attention(q, cache, table, lt)
    kv4.check_errors()
    _check(torch, out, q, seqs, lens)
    assert torch.equal(out, kv4.attention(q, cache, table, lt))
    # the rows of a chunk one by one, as single tokens see them
    last = kv4.attention(q[:, -1], cache, table, lt)
    _check(torch, last[:, None], q[:, -1:], seqs, lens)


def test_attention_many_rows_bad_lengths_and_pages(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(19)
    lens = [128, 128]
    cache, table, q, seqs = _case(torch, rng, lens, 100, 32, 8, 128, 64, torch.float16)
    table = table[:, :2].contiguous()
    out = kv4.attention(q, cache, table, torch.tensor([128, 1 << 30], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        kv4.check_errors()
    _check(torch, out, q, seqs, lens)
    out = kv4.attention(q, cache, table, torch.tensor([128, -5], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        kv4.check_errors()
    assert bool((out[1] == 0).all())
    _check(torch, out[:1], q[:1], seqs[:1], lens[:1])
    for page in (-1, cache.pages):                                    # pages outside the cache: no keys from them
        t2 = table.clone()
        t2[1] = page
        out = kv4.attention(q, cache, t2, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        _check(torch, out[:1], q[:1], seqs[:1], lens[:1])
        assert bool((out[1] == 0).all())


def test_attention_many_rows_in_a_graph(torch):
    """Captured once, replayed with other lengths."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(14)
    lens = [400, 190]
    cache, table, q, seqs = _case(torch, rng, lens, 64, 32, 8, 128, 64, torch.float16)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv4.attention(q, cache, table, lt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kv4.attention(q, cache, table, lt)
    for cut in ([400, 190], [17, 64]):
        lt.copy_(torch.tensor(cut, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        _check(torch, out, q, [(K[:L], V[:L], [p[:L] for p in pr]) for (K, V, pr), L in zip(seqs, cut)], cut)


def test_attention_far_pages(torch):
    """Pages past 4 GiB of a cache: byte offsets beyond 32 bits."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(11)
    KVH, hd, page, L = 8, 128, 64, 300
    near, table, q, seqs = _case(torch, rng, [L], 1, 16, KVH, hd, page, torch.float16)
    bytes_page = KVH * page * kv4.token_bytes(hd)
    pages = (5 << 30) // bytes_page
    data = torch.empty((pages, KVH, page * kv4.token_bytes(hd)), dtype=torch.uint8, device="cuda")
    far = torch.arange(pages - near.pages, pages, device="cuda")
    data[far] = near.data
    cache = kv4.KV4Cache.of(data, hd, page)
    used = -(-L // page)
    moved = table.clone()
    moved[:, :used] += pages - near.pages
    lt = torch.tensor([L], dtype=torch.int32, device="cuda")
    out = kv4.attention(q, cache, moved, lt)
    _check(torch, out, q, seqs, [L])
    assert torch.equal(out, kv4.attention(q, near, table, lt))
    # and the append writes there
    x = torch.randn(1, (16 + 2 * KVH) * hd, device="cuda")
    one, zero = torch.ones(1, hd // 2, device="cuda"), torch.zeros(1, hd // 2, device="cuda")
    slot = torch.tensor([pages * page - 1], device="cuda")
    kv4.append(cache, x, torch.zeros(1, dtype=torch.int32, device="cuda"), slot, one, zero, 16)
    k, v = cache.rows(slot)
    kv4.check_errors()
    want = x.view(16 + 2 * KVH, hd)
    assert float((k[0].float() - want[16:16 + KVH]).abs().max()) < 0.4
    assert float((v[0].float() - want[16 + KVH:]).abs().max()) < 0.4


def test_attention_side_stream_and_out(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(3)
    lens = [513, 77]
    cache, table, q, seqs = _case(torch, rng, lens, 1, 16, 8, 128, 64, torch.float16)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        torch.cuda._sleep(2_000_000)
        late.copy_(q)
        out = torch.full_like(q, float("nan"))
        got = kv4.attention(late, cache, table, lt, out=out)
    side.synchronize()
    assert got is out
    _check(torch, out, q, seqs, lens)


def test_attention_in_a_graph(torch):
    """Captured once, replayed with other lengths and queries."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(4)
    lens = [400, 90, 33]
    cache, table, q, seqs = _case(torch, rng, lens, 1, 16, 8, 128, 64, torch.float16)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    kv4.attention(q, cache, table, lt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kv4.attention(q, cache, table, lt)
    for cut in ([400, 90, 33], [17, 0, 1]):
        lt.copy_(torch.tensor(cut, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        _check(torch, out, q, [(K[:L], V[:L], [p[:L] for p in pr]) for (K, V, pr), L in zip(seqs, cut)], cut)


def test_attention_bad_lengths_and_pages(torch):
    from agxforge.kernels import kv4
    rng = np.random.default_rng(9)
    lens = [64, 64]
    cache, table, q, seqs = _case(torch, rng, lens, 1, 16, 8, 128, 64, torch.float16)
    table = table[:, :1].contiguous()
    for bad in ([64, 1 << 30], [64, 65]):                             # clamped to what the table can hold
        out = kv4.attention(q, cache, table, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        _check(torch, out, q, seqs, lens)
    out = kv4.attention(q, cache, table, torch.tensor([64, -5], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="out of range"):
        kv4.check_errors()
    assert bool((out[1] == 0).all())
    for page in (-1, cache.pages):                                    # a page outside the cache: no keys from it
        t2 = table.clone()
        t2[1, 0] = page
        out = kv4.attention(q, cache, t2, torch.tensor(lens, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError, match="out of range"):
            kv4.check_errors()
        _check(torch, out[:1], q[:1], seqs[:1], lens[:1])
        assert bool((out[1] == 0).all())


def test_attention_refuses(torch):
    from agxforge.kernels import kv4
    c = kv4.KV4Cache(2, 2, 64, 16)
    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    i32 = torch.int32
    ok = dict(q=z(1, 4, 64), page_table=z(1, 2, dtype=i32), lengths=z(1, dtype=i32))
    kv4.attention(cache=c, **ok)
    for bad, text in [(dict(q=z(1, 4, 128)), "head_dim"), (dict(q=z(1, 3, 64)), "multiple of kv_heads"),
                      (dict(q=z(1, 4, 64, dtype=torch.float32)), "fp16 or bf16"), (dict(lengths=z(2, dtype=i32)), "one length"),
                      (dict(lengths=z(1, dtype=torch.int64)), "lengths"), (dict(page_table=z(2, 2, dtype=i32)), "page_table"),
                      (dict(out=z(1, 4, 64, dtype=torch.bfloat16)), "out")]:
        with pytest.raises(ValueError, match=text):
            kv4.attention(cache=c, **dict(ok, **bad))
    assert kv4.attention(z(0, 4, 64), c, z(0, 2, dtype=i32), z(0, dtype=i32)).shape == (0, 4, 64)
    assert kv4.attention(z(2, 0, 4, 64), c, z(2, 2, dtype=i32), z(2, dtype=i32)).shape == (2, 0, 4, 64)
    empty = kv4.attention(z(1, 4, 64) + 1, c, z(1, 0, dtype=i32), z(1, dtype=i32))
    assert bool((empty == 0).all())
    kv4.check_errors()
