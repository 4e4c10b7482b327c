"""The append from rows, tables and vectors off their 16-byte boundaries, with odd strides, and inside a CUDA graph, on the B200."""
import numpy as np
import pytest

from tests.test_gpu_kv4 import _case, _check, _rope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def _off(torch, t, by):
    """t's values in memory that starts `by` elements past a 256-byte boundary."""
    buf = torch.full((t.numel() + by,), float("nan"), dtype=t.dtype, device=t.device)
    buf[by:] = t.reshape(-1)
    out = buf[by:].view(t.shape)
    assert out.is_contiguous() and out.data_ptr() % 16 == by * t.element_size() % 16
    return out


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,H,KVH,hd", [(1, 16, 8, 128), (33, 14, 2, 64), (70, 6, 2, 128)])
def test_append_off_its_boundaries(torch, T, H, KVH, hd, dtype):
    """Each of the rows, the row stride, the tables and the bias alone, and all together: the bits of the aligned call."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(T)
    dt, W = getattr(torch, dtype), (H + 2 * KVH) * hd
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    x = dev(rng.standard_normal((T, W)).astype(np.float32)).to(dt)
    cos, sin = (dev(a) for a in _rope(rng, 50, hd))
    pos, slots = dev(rng.integers(0, 50, T).astype(np.int32)), dev(rng.permutation(128)[:T].astype(np.int64))
    bias = dev(rng.standard_normal(W).astype(np.float16))
    gains = [dev((1 + 0.1 * rng.standard_normal(hd)).astype(np.float16)) for _ in range(2)]

    def run(x, cos, sin, bias, gains=(None, None)):
        c = kv4.KV4Cache(4, KVH, hd, 32)
        q = kv4.append(c, x, pos, slots, cos, sin, H, bias=bias, q_norm=gains[0], k_norm=gains[1])
        return q, c.data

    def strided(by, extra):
        wide = torch.full((T, W + extra), float("nan"), dtype=dt, device="cuda")
        wide[:, by:by + W] = x
        return wide[:, by:by + W]

    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))  # noqa: E731
    for b in (None, bias):
        want = run(x, cos, sin, b)
        kinds = [dict(x=_off(torch, x, by)) for by in (1, 2, 3, 5)] + [dict(x=strided(by, e)) for by, e in ((1, 1), (0, 1), (3, 7), (4, 6))]
        kinds += [dict(cos=_off(torch, cos, 1)), dict(sin=_off(torch, sin, 3))]
        if b is not None:
            kinds += [dict(bias=_off(torch, bias, 1)), dict(bias=_off(torch, bias, 2))]
        kinds += [dict(x=strided(1, 2), cos=_off(torch, cos, 2), sin=_off(torch, sin, 1), bias=b if b is None else _off(torch, b, 3))]
        for kind in kinds:
            assert same(run(**dict(dict(x=x, cos=cos, sin=sin, bias=b), **kind)), want), list(kind)
    want = run(x, cos, sin, bias, gains)
    assert same(run(strided(1, 2), cos, sin, bias, [_off(torch, g, 1) for g in gains]), want)
    kv4.check_errors()


def test_a_decode_step_in_a_graph(torch):
    """Append, read-back and attention captured once and replayed for later tokens."""
    from agxforge.kernels import kv4
    rng = np.random.default_rng(14)
    lens, H, KVH, hd, page, dt = [100, 30, 0], 16, 8, 128, 64, torch.float16
    cache, table, q, seqs = _case(torch, rng, [L + 3 for L in lens], 1, H, KVH, hd, page, dt)
    cos, sin = (torch.from_numpy(a).cuda() for a in _rope(rng, 256, hd))
    pos, lt = torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda") + 1
    host = table.cpu().numpy()
    place = lambda step: torch.tensor([int(host[b, (L + step) // page]) * page + (L + step) % page  # noqa: E731
                                       for b, L in enumerate(lens)], device="cuda")
    slots = place(0)
    x = torch.zeros((3, (H + 2 * KVH) * hd), device="cuda")
    other = kv4.KV4Cache.of(cache.data.clone(), hd, page)

    def step(c):
        q = kv4.append(c, x, pos, slots, cos, sin, H)
        return q, c.rows(slots), kv4.attention(q, c, table, lt)

    step(cache)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(cache)
    for i in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)))
        pos.copy_(torch.tensor(lens, dtype=torch.int32) + i)
        lt.copy_(torch.tensor(lens, dtype=torch.int32) + i + 1)
        slots.copy_(place(i))
        g.replay()
        want = step(other)
        torch.cuda.synchronize()
        flat = lambda r: [r[0], *r[1], r[2]]  # noqa: E731
        assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))
        K, V = (a.double().cpu().numpy() for a in got[1])
        for b, L in enumerate(lens):                                     # the appended key is the last one seen
            k, v, pairs = seqs[b]
            k[L + i], v[L + i] = K[b], V[b]
        cut = [L + i + 1 for L in lens]
        _check(torch, got[2][:, None], got[0][:, None], [(k[:L], v[:L], [p[:L] for p in pr])
                                                         for (k, v, pr), L in zip(seqs, cut)], cut)
    kv4.check_errors()
