"""Sampling on the B200 against its definition in 64 bits.

A weight of the kernel is floor(2^40 e) with e an fp32 exp of a rounded argument: relative error at most
|z| 2^-23 + 2^-22 plus 2^-40 absolute, and a weight with |z| > 4 is under 2 % of the largest, so any sum of a row's
weights is within TOL = 4e-6 of the total (V 2^-40 is below 3e-7 for every vocabulary here). The token's cumulative
interval must hold u within that, and the cut at top-p may fall one rank apart only where the sum before it is within
that of the bar; min-p's likewise. Structured rows (equal logits, masks) have exact weights and exact answers."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 4e-6


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def kept_sets(x, T, k, p, least):
    """(e, the ranks certainly kept, the ranks possibly kept) of one row in 64 bits; e is relative to the maximum."""
    x = np.where(np.isnan(x), -np.inf, x)
    best = x.max()
    with np.errstate(invalid="ignore"):
        d = np.where(x == best, 0.0, x - best)
    e = (d == 0).astype(np.float64) if T == 0 else np.exp(d / T)
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    w = e[order]
    before, total = np.cumsum(w) - w, w.sum()
    bar = p * total if p < 1 else np.inf
    sets = []
    for sign in (-1, 1):
        ok = (before < bar + sign * TOL * total) & (w >= least * (1 - sign * TOL)) & (w > 0)
        ok[0] = w[0] >= least
        sets.append(order[ok])
    return e, sets[0], sets[1]


def check_row(x, u, T, k, p, least, token, prob):
    x, u, p, least = x.astype(np.float64), float(np.float32(u)), float(np.float32(p)), float(np.float32(least))
    T = float(np.float32(T))
    if not (x > -np.inf).any():
        assert token == -1 and prob == 0
        return
    if T == 0:
        assert token == int(np.argmax(np.where(np.isnan(x), -np.inf, x))) and prob == 1
        return
    e, sure, maybe = kept_sets(x, T, k, p, least)
    if len(maybe) == 0:
        assert token == -1 and prob == 0
        return
    assert token in maybe
    good = False
    for ids in {tuple(np.sort(sure)), tuple(np.sort(maybe))}:
        ids = np.array(ids, np.int64)
        if token not in ids:
            continue
        up, total = np.cumsum(e[ids]), e[ids].sum()
        i = int(np.searchsorted(ids, token))
        lo, hi = (up[i - 1] if i else 0.0), up[i]
        good |= lo - TOL * total <= u * total <= hi + TOL * total and abs(prob - e[token] / total) <= 2 * TOL
    assert good


def _logits(rng, B, V, spread=2.0):
    x = rng.standard_normal((B, V)).astype(np.float32) * spread
    for r in range(B):
        x[r, rng.integers(0, V, 40)] += rng.uniform(0, 10, 40).astype(np.float32)
    return x


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 31), (5, 1000), (4, 4097), (3, 50257), (2, 92544), (2, 151936), (1, 300001)])
def test_options(torch, B, V, dtype):
    from agxforge.kernels import sampling
    rng = np.random.default_rng(V + B)
    x = torch.from_numpy(_logits(rng, B, V)).to(getattr(torch, dtype)).cuda()
    ref = x.float().cpu().numpy()
    for T, k, p, least in [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 1000, 0.95, 0.0), (1.0, 0, 1.0, 0.05),
                           (0.8, 50, 0.9, 0.02), (1.0, 1, 1.0, 0.0), (2.0, 0, 0.5, 0.001), (0.0, 7, 0.3, 0.5), (5.0, 0, 0.99, 0.0),
                           (1.0, V + 9, 1.5, 0.0), (1.0, -1, 0.0, 0.0), (0.02, 0, 0.999, 0.0), (30.0, 20000, 1.0, 0.0)]:
        u = rng.random(B, np.float32)
        token, prob = sampling.sample(x, torch.from_numpy(u).cuda(), T, k, p, least)
        assert token.dtype == torch.int32 and prob.dtype == torch.float32
        for r in range(B):
            check_row(ref[r], u[r], T, k, p, least, int(token[r]), float(prob[r]))


def test_every_row_its_own_options(torch):
    """Rows with options of their own give what they give alone, in any batch, from strided rows."""
    from agxforge.kernels import sampling
    rng = np.random.default_rng(2)
    B, V = 70, 20011
    x = _logits(rng, B, V)
    x[3] = -np.inf
    x[4, 1:] = -np.inf
    x[5, ::3] = np.nan
    x[6, 77] = np.inf
    x[7] = 1.5
    T = rng.choice([0.0, 0.5, 1.0, 1.7], B).astype(np.float32)
    k = rng.choice([0, 1, 5, 50, 3000], B).astype(np.int32)
    p = rng.choice([1.0, 0.9, 0.5], B).astype(np.float32)
    m = rng.choice([0.0, 0.05], B).astype(np.float32)
    u = rng.random(B, np.float32)
    wide = torch.zeros((B, V + 5), device="cuda")
    wide[:, 3:3 + V] = torch.from_numpy(x).cuda()
    dev = [torch.from_numpy(a).cuda() for a in (T, k, p, m)]
    token, prob = sampling.sample(wide[:, 3:3 + V], torch.from_numpy(u).cuda(), *dev)
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    for r in range(B):
        check_row(x[r], u[r], float(T[r]), int(k[r]), float(p[r]), float(m[r]), int(token[r]), float(prob[r]))
    for r in list(range(8)) + [20, 69]:
        t1, p1 = sampling.sample(torch.from_numpy(x[r:r + 1]).cuda(), torch.from_numpy(u[r:r + 1]).cuda(), float(T[r]),
                                 int(k[r]), float(p[r]), float(m[r]))
        assert int(t1[0]) == token[r] and float(p1[0]) == prob[r]


@pytest.mark.parametrize("V", [5, 1024, 5000, 92544, 151936])
def test_equal_logits(torch, V):
    """All weights are 2^40: ranks are indices, and every answer is exact."""
    from agxforge.kernels import sampling
    B = 12
    x = torch.full((B, V), -0.75, device="cuda")
    x[:, V // 2] = -0.75
    u = (torch.arange(B, device="cuda").float() + 0.5) / B
    un = u.double().cpu().numpy()
    for k, p in [(0, 1.0), (5, 1.0), (V - 1, 1.0), (0, 0.5), (0, 0.25), (4, 0.75), (V // 2 + 1, 0.5)]:
        n = V if not 0 < k < V else k
        if p < 1:
            n = max(1, -(-int(np.ceil(p * n * 2.0 ** 40)) // 2 ** 40))
        token, prob = sampling.sample(x, u, 0.9, k, p)
        want = np.floor(np.floor(un * (n * 2.0 ** 40)) / 2.0 ** 40).astype(np.int64)
        assert np.array_equal(token.cpu().numpy(), want), (k, p)
        assert np.array_equal(prob.cpu().numpy(), np.full(B, 1.0 / n, np.float32))


def test_two_values_and_ties_at_the_cut(torch):
    """Zeros of both signs rank by index; a cut inside a run of equal values keeps the lowest indices."""
    from agxforge.kernels import sampling
    V = 30000
    x = torch.full((1, V), -50.0, device="cuda")
    at = torch.arange(100, V, 7, device="cuda")
    x[0, at] = 0.0
    x[0, at[::2]] = -0.0
    n = at.numel()
    for k in (1, 2, 100, 2049, n):
        for u in (0.0, 0.25, 0.5, 1 - 2.0 ** -24):
            token, prob = sampling.sample(x, torch.tensor([u], device="cuda"), 1.0, k)
            want = min(int(u * k), k - 1)          # e^-50 is far below a weight's unit
            assert int(token[0]) == int(at[want]) and abs(float(prob[0]) - 1 / k) <= 2.0 ** -23 / k


def test_u_at_its_ends(torch):
    from agxforge.kernels import sampling
    rng = np.random.default_rng(8)
    x = torch.from_numpy(_logits(rng, 1, 5000)).cuda()
    x[0, :10] = -float("inf")
    x[0, -10:] = -float("inf")
    lo, _ = sampling.sample(x, torch.zeros(1, device="cuda"))
    hi, _ = sampling.sample(x, torch.full((1,), 1 - 2.0 ** -24, device="cuda"))
    over, _ = sampling.sample(x, torch.ones(1, device="cuda"))          # past the end: the last kept index
    assert int(lo[0]) == 10
    assert 4900 < int(hi[0]) <= 4989 and int(over[0]) == 4989


def test_frequencies(torch):
    """Evenly spaced u give each token as often as its weight says, to one draw at each end."""
    from agxforge.kernels import sampling
    B, V = 4096, 300
    rng = np.random.default_rng(1)
    row = rng.standard_normal(V).astype(np.float32)
    x = torch.from_numpy(row).cuda().expand(B, V)
    x = x.contiguous()
    u = (torch.arange(B, device="cuda").float() + 0.5) / B
    token, _ = sampling.sample(x, u, 1.0, 40)
    e, keep, _ = kept_sets(row.astype(np.float64), 1.0, 40, 1.0, 0.0)
    want = np.zeros(V)
    want[keep] = e[keep] / e[keep].sum() * B
    assert np.all(np.abs(np.bincount(token.cpu().numpy(), minlength=V) - want) <= 1 + 1e-3)


def test_side_stream_and_graph(torch):
    from agxforge.kernels import sampling
    rng = np.random.default_rng(6)
    x = torch.from_numpy(_logits(rng, 4, 30011)).cuda()
    u = torch.from_numpy(rng.random(4, np.float32)).cuda()
    want, _ = sampling.sample(x, u, 0.9, 50, 0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(2_000_000)
        late.copy_(x)
        got, _ = sampling.sample(late, u, 0.9, 50, 0.9)
    side.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = sampling.sample(x, u, 0.9, 50, 0.9)
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want.flip(0))


def test_refuses(torch):
    from agxforge.kernels import sampling
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    sampling.sample(x, u)
    for args, text in [((x.double(), u), "fp32, fp16 or bf16"), ((x[0], u), "batch, vocab"), ((x.t(), u), "contiguous"),
                       ((x, u[:1]), "u is"), ((x, u.double()), "u is"), ((x, u, -1.0), "temperature"),
                       ((x, u, torch.zeros(3, device="cuda")), "temperature is"), ((x, u, 1.0, u), "top_k is"),
                       ((x, u, 1.0, 0, u.half()), "top_p is"), ((x[:, :0], u), "batch, vocab")]:
        with pytest.raises(ValueError, match=text):
            sampling.sample(*args)
    token, prob = sampling.sample(x[:0], u[:0])
    assert token.shape == (0,) and prob.shape == (0,)


def test_refuses_a_vocabulary_past_the_limit(torch):
    from agxforge.kernels.sampling import sample
    u = torch.zeros(1, device="cuda")
    with pytest.raises(ValueError, match="1,048,576"):
        sample(torch.zeros(1, (1 << 20) + 1, device="cuda"), u)
    x = torch.zeros(1, 1 << 20, dtype=torch.float16, device="cuda")
    x[0, (1 << 20) - 1] = 40.0                                        # all the weight on the last index
    token, prob = sample(x, u + 0.5)
    assert int(token) == (1 << 20) - 1 and abs(float(prob) - 1.0) <= 2.0 ** -18
