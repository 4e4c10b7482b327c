"""Serving with the paged 4-bit cache (agxforge.inference.paged) against a 64-bit pass of the same packs that attends to
the K and V the cache holds (quantising the pass's own would differ by whole codes wherever the two chains fall on two
sides of a rounding): the logits within the framework's model-level bound (0.05 + 0.003 |ref|), what is held within half
a code of the pass's own K and V and a fiftieth of the group's largest for the fp16 chain's distance, the sampled token as sampling's definition gives it from the device's own logits, pages handed back and used again."""
import numpy as np
import pytest

from tests import kv4_ref as R
from tests.test_gpu_sampling import check_row

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    if not t.cuda.is_available():
        pytest.skip("no GPU")
    return t


def _weights(shape, seed):
    from agxforge.inference import assemble
    m = assemble.build(dict(model=shape, bits=4, batch=1, cap=64, seed=seed), keep_packs=True)
    packs, S = m.packs, m.shape
    m.close()
    return packs, S


def _held(m, s, n):
    """Per layer, the (K, V) of sequence s's first n tokens as the cache holds them."""
    import torch
    P, pages = m.page_size, m.seqs[s]["pages"]
    slots = torch.tensor([pages[i // P] * P + i % P for i in range(n)], device="cuda")
    return [[a.double().cpu().numpy() for a in d["cache"].rows(slots)] for d in m.layers]


def _forward64(k, S, tokens, held):
    """Logits [len(tokens), vocab] in 64 bits, attending to `held`'s K and V."""
    from oracle import pack as P
    W = lambda key, n, kk: P.dequant64(P.unpack(k[key][0], 4, n, kk), k[key][1], k[key][2], "fp16")  # noqa: E731
    norm = lambda v, g: v / np.sqrt((v * v).mean(-1, keepdims=True) + S.EPS) * g  # noqa: E731
    T, H, KVH, hd = len(tokens), S.HEADS, S.KV_HEADS, S.HEAD_DIM
    ang = np.arange(T)[:, None] / S.ROPE_THETA ** (np.arange(0, hd, 2) / hd)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    rope = lambda v: np.concatenate([v[..., :hd // 2] * c - v[..., hd // 2:] * s, v[..., hd // 2:] * c + v[..., :hd // 2] * s], -1)  # noqa: E731
    x = k["embed"][tokens].astype(np.float64)
    for l in range(S.LAYERS):
        w = {r: W((l, r), n, kk) for r, n, kk in S.matrices()}
        qkv = norm(x, k[(l, "attn_gain")].astype(np.float64)) @ w["qkv"].T
        if S.QKV_BIAS:
            qkv = qkv + k[(l, "qkv_bias")].astype(np.float64)
        qkv = qkv.reshape(T, H + 2 * KVH, hd)
        q, kk, v = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
        if S.QK_NORM:
            q, kk = norm(q, k[(l, "q_norm")].astype(np.float64)), norm(kk, k[(l, "k_norm")].astype(np.float64))
        q = rope(q) * R.LOG2E / np.sqrt(hd)
        K, V = held[l]
        for own, has in ((rope(kk), K), (v, V)):
            g = own.reshape(T, KVH, -1, 64)
            tol = np.ptp(g, -1) / 30 + np.abs(g).max(-1) / 50
            assert np.all(np.abs(own - has) <= tol.repeat(64, -1).reshape(own.shape))
        a = R.attention(q, K, V, T).reshape(T, -1)
        h = x + a @ w["wo"].T
        y = norm(h, k[(l, "ffn_gain")].astype(np.float64))
        g, u = y @ w["gate"].T, y @ w["up"].T
        x = h + (g / (1 + np.exp(-g)) * u) @ w["down"].T
    return norm(x, k["final_gain"].astype(np.float64)) @ W((None, "head"), S.VOCAB, S.D_MODEL).T


@pytest.mark.parametrize("extra", [dict(HEAD_DIM=64, QKV_BIAS=True), dict(HEAD_DIM=128, QK_NORM=True), dict(HEAD_DIM=128)])
def test_paged_serving(torch, extra):
    from agxforge.inference import paged
    shape = dict(dict(NAME="paged", D_MODEL=256, LAYERS=2, HEADS=4, KV_HEADS=2, FFN=512, VOCAB=1024, ROPE_THETA=1e6,
                      EPS=1e-6), **extra)
    packs, S = _weights(shape, 11)
    rng = np.random.default_rng(4)
    m = paged.PagedModel(dict(model=shape, bits=4), packs, pages=24, page_size=16)
    prompts = [rng.integers(0, 1024, n).tolist() for n in (1, 17, 40, 9, 2, 31, 5, 12, 16, 3)]     # ten: two groups of rows
    ids = [m.add(p) for p in prompts]
    got = {s: [] for s in ids}
    for _ in range(3):
        lg, order = m.logits()
        for s, row in zip(order, lg.cpu().numpy()):
            got[s].append(row)
        for s in order:                                              # forced, then sampled below
            m.seqs[s]["tokens"].append(int(rng.integers(0, 1024)))
    for s in ids:
        toks = m.seqs[s]["tokens"]
        n = len(prompts[ids.index(s)])
        want = _forward64(packs, S, np.asarray(toks[:n + 2]), _held(m, s, n + 2))[n - 1:n + 2]
        off = np.abs(np.stack(got[s]) - want)
        assert np.all(off <= 0.05 + 0.003 * np.abs(want)), (s, float(off.max()))
    spare = len(m.spare)
    m.free(ids[2])
    assert len(m.spare) == spare + 3
    with pytest.raises(MemoryError):
        m.add(rng.integers(0, 1024, 16 * len(m.spare) + 2).tolist())
    assert len(m.spare) == spare + 3                                 # a sequence that did not fit left nothing behind
    again = m.add(prompts[2])                                        # into pages that others have used
    lg, _ = m.logits([again])
    want = _forward64(packs, S, np.asarray(prompts[2]), _held(m, again, len(prompts[2])))[-1]
    assert np.all(np.abs(lg[0].cpu().numpy() - want) <= 0.05 + 0.003 * np.abs(want))


def test_paged_sampling(torch):
    from agxforge.inference import paged
    shape = dict(NAME="paged", D_MODEL=256, LAYERS=1, HEADS=4, KV_HEADS=2, HEAD_DIM=64, FFN=512, VOCAB=1024,
                 ROPE_THETA=1e6, EPS=1e-6)
    packs, _ = _weights(shape, 3)
    a, b = (paged.PagedModel(dict(model=shape, bits=4), packs, pages=16, page_size=32) for _ in range(2))
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 1024, n).tolist() for n in (5, 33)]
    ia, ib = [a.add(p) for p in prompts], [b.add(p) for p in prompts]
    for _ in range(4):
        u = rng.random(2, np.float32)
        lg, order = a.logits()                                       # the logits that b's step samples from
        tok = b.step(u, temperature=0.7, top_k=20, top_p=0.9)
        for i, s in enumerate(order):
            t, p = tok[ib[ia.index(s)]]
            check_row(lg[i].cpu().numpy(), u[i], 0.7, 20, 0.9, 0.0, t, p)
            a.seqs[s]["tokens"].append(t)
    greedy = b.step([0.3, 0.9], temperature=0.0)
    assert all(p == 1.0 for _, p in greedy.values())
    with pytest.raises(ValueError, match="no new token"):
        b.seqs[ib[0]]["tokens"].pop()
        b.logits()
    with pytest.raises(ValueError, match="at least one token"):
        b.add([])
    with pytest.raises(ValueError, match="at least one token"):
        b.add([1024])
