"""What the serving operators cost: the append to a 4-bit paged KV cache, the attention that reads it, and sampling.

Each case is one pass through one operator at sizes of this repository's decoder shapes (16/8 and 32/8 heads of 128,
14/2 heads of 64, vocabularies 92,544 and 151,936) or generic ones. `run` makes the framework's call where `own` is
true and computes the plain form (elementary torch operations in fp32) where it is false.

The cache holds, per page and KV head, tiles of 16 tokens: K codes, V codes (4 bits, low nibble first), then each
token's fp16 scale and bias of every 64 dims of K and of V; a value is code * scale + bias.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
LOG2E = 1.4426950408889634
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
W_ONE = 2.0 ** 40          # a weight of 1 in the sampler's fixed point


def listed():
    A = dict(op="attention", page=64, dtype="fp16")
    P = dict(op="append", page=64, bias=False, skip=False)
    S = dict(op="sample", mixed=False, masked=0.0)
    return [
        # one sequence of the 16/8-head decoder, the repository's headline history: the smallest call of a decode step
        dict(A, name="attn-1x1792", batch=1, rows=1, heads=16, kv_heads=8, hd=128, longest=1792, ragged=False),
        # 64 sequences of the 32/8-head decoder at 8,192 tokens: the largest serving batch of the benchmark
        dict(A, name="attn-64x8192", batch=64, rows=1, heads=32, kv_heads=8, hd=128, longest=8192, ragged=False),
        # a busy server of the 14/2-head model: 128 sequences of every length from none to 1,792, 16-token pages
        dict(A, name="attn-128-ragged", batch=128, rows=1, heads=14, kv_heads=2, hd=64, longest=1792, ragged=True,
             page=16),
        # speculative verification: the current token and 15 drafts of each of 8 sequences, in bf16
        dict(A, name="attn-verify", batch=8, rows=16, heads=16, kv_heads=8, hd=128, longest=1807, ragged=True,
             dtype="bf16"),
        # a 256-row prompt chunk at the end of a 2,048-token history
        dict(A, name="attn-chunk", batch=1, rows=256, heads=32, kv_heads=8, hd=128, longest=2304, ragged=False),
        # the append of one decode step of one sequence (fp32 rows, as the GEMV leaves them)
        dict(P, name="append-1", tokens=1, heads=16, kv_heads=8, hd=128, dtype="fp32"),
        # the append of a 64-sequence decode step, a few of the batch's places unused
        dict(P, name="append-64", tokens=64, heads=32, kv_heads=8, hd=128, dtype="fp32", skip=True),
        # a prompt of 3,585 tokens written at once (odd, fp16 rows, qkv bias, heads of 64, 16-token pages)
        dict(P, name="append-prompt", tokens=3585, heads=14, kv_heads=2, hd=64, dtype="fp16", bias=True, page=16),
        # the token choice of one sequence: nucleus sampling over the large vocabulary
        dict(S, name="sample-1", batch=1, vocab=151936, dtype="fp32", top_k=50, top_p=0.9, min_p=0.0, temp=0.8),
        # 64 sequences at temperature with min-p, no sorting options
        dict(S, name="sample-64-minp", batch=64, vocab=92544, dtype="fp32", top_k=0, top_p=1.0, min_p=0.05, temp=1.0),
        # 256 sequences, each with its own options (greedy rows among them), some under a grammar's mask
        dict(S, name="sample-256-mixed", batch=256, vocab=151936, dtype="fp32", top_k=0, top_p=0.95, min_p=0.0,
             temp=1.0, mixed=True, masked=0.5),
        # 16-bit logits with many equal values, an odd vocabulary and an odd batch
        dict(S, name="sample-33-bf16", batch=33, vocab=50257, dtype="bf16", top_k=1000, top_p=0.95, min_p=0.0,
             temp=1.3),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "sample"])
    heads, kv_heads, hd = rng.choice([(16, 8, 128), (32, 8, 128), (14, 2, 64), (8, 8, 64), (24, 3, 128), (12, 1, 128)])
    page = rng.choice([16, 32, 64, 128])
    if op == "attention":
        rows = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 256)])
        longest = _log(rng, 1, 16384) if rows == 1 else rows + _log(rng, 1, 4096)
        # at most the listed 64 x 8,192 tokens of 8 heads of 128, and that many multiplications of a 256-row chunk
        most = 64 * 8192 * 8 * 128 // (longest * kv_heads * hd)
        if rows > 1:
            most = min(most, 2 * 256 * 32 * 128 * 2304 // (rows * heads * hd * longest))
        batch = _log(rng, 1, max(1, min(256, most)))
        return dict(op=op, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, hd=hd, longest=longest,
                    ragged=rng.random() < 0.6, page=page, dtype=rng.choice(["fp16", "bf16"]))
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 4096), heads=heads, kv_heads=kv_heads, hd=hd, page=page,
                    dtype=rng.choice(["fp32", "fp16", "bf16"]), bias=rng.random() < 0.5, skip=rng.random() < 0.3)
    return dict(op=op, batch=_log(rng, 1, 256), vocab=_log(rng, 1000, 151936), dtype=rng.choice(["fp32", "fp16", "bf16"]),
                top_k=rng.choice([0, 0, 1, 5, 50, 1000]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                min_p=rng.choice([0.0, 0.0, 0.05]), temp=rng.choice([0.5, 0.8, 1.0, 1.5]), mixed=rng.random() < 0.3,
                masked=rng.choice([0.0, 0.0, 0.5]))


def work(c):
    if c["op"] == "attention":
        n, group = c["rows"], c["hd"] // 64
        lens = _lengths(c, np.random.RandomState(1)).astype(np.int64)
        q = 2 * 2 * c["batch"] * n * c["heads"] * c["hd"]
        kv = int(lens.sum()) * c["kv_heads"] * 2 * (c["hd"] // 2 + 4 * group)
        seen = sum(int(np.maximum(lens - n + 1 + i, 0).sum()) for i in range(n))
        return {"bytes": kv + q, "flops": 4 * seen * c["heads"] * c["hd"]}
    if c["op"] == "append":
        size = {"fp32": 4, "fp16": 2, "bf16": 2}[c["dtype"]]
        T, H, KVH, hd = c["tokens"], c["heads"], c["kv_heads"], c["hd"]
        held = T * KVH * 2 * (hd // 2 + hd // 16)
        # rows and tables in, q out, the codes written and read back, the rows they stand for out
        b = T * (H + 2 * KVH) * hd * size + T * hd * 4 + T * H * hd * 2 + 2 * held + T * KVH * 2 * hd * 2
        return {"bytes": b, "flops": T * (H + 2 * KVH) * hd * 4}
    size = {"fp32": 4, "fp16": 2, "bf16": 2}[c["dtype"]]
    return {"bytes": c["batch"] * (c["vocab"] * size + 24), "flops": c["batch"] * c["vocab"] * 4}


# ---------------------------------------------------------------------------------------------------- the inputs
def _lengths(c, rs):
    if not c["ragged"]:
        return np.full(c["batch"], c["longest"], np.int32)
    lens = rs.randint(0, c["longest"] + 1, c["batch"]).astype(np.int32)
    lens[rs.randint(c["batch"])] = c["longest"]
    return lens


def _blank(pages, c):
    """The pages of a cache: [pages, kv_heads, 16-token tiles, bytes of a tile]."""
    g = c["hd"] // 64
    return torch.zeros((pages, c["kv_heads"], c["page"] // 16, 16 * c["hd"] + 128 * g), dtype=torch.uint8, device=DEV)


def _parts(data, hd):
    """The K codes, V codes and scale/bias pairs of a cache's pages, as views in the order of their storage."""
    P, KVH, m, _ = data.shape
    g = hd // 64
    k = data[..., :8 * hd].unflatten(-1, (16, 4, g, 8))                       # token, 16-dim chunk, group, byte
    v = data[..., 8 * hd:16 * hd].unflatten(-1, (2, 8, 4, 2, g, 4))           # t/8, 8-dim chunk, t/2%4, t%2, group, byte
    sb = data[..., 16 * hd:].view(torch.float16).unflatten(-1, (16, 2, g, 2))  # token, K or V, group, scale or bias
    return k, v, sb


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 32))
    if c["op"] == "attention":
        B, n, KVH, hd, page = c["batch"], c["rows"], c["kv_heads"], c["hd"], c["page"]
        lens = _lengths(c, np.random.RandomState((seed + 1) % (1 << 32)))
        per = -(-c["longest"] // page)
        pages = B * per
        data = _blank(pages, c)
        k, v, sb = _parts(data, hd)
        # keys and values of unit size, in the codes that quantising them gives; the scales are those of 64 normal values
        spread = torch.randn((1 << 16, 2), generator=gen, device=DEV)
        table = ((spread * 2.9 + 7.5).round().clamp(0, 15).to(torch.uint8) * torch.tensor([1, 16], dtype=torch.uint8, device=DEV)).sum(-1).to(torch.uint8)
        normal = table[torch.randint(0, 1 << 16, (1 << 16,), generator=gen, device=DEV)]
        flat = data.view(-1)
        for at in range(0, flat.numel(), 1 << 28):
            part = flat[at:at + (1 << 28)]
            part.copy_(normal[torch.randint(0, 1 << 16, part.shape, generator=gen, device=DEV, dtype=torch.int32)])
        scale = (torch.rand(sb.shape[:-1], generator=gen, device=DEV) * 0.12 + 0.28)
        sb[..., 0] = scale.half()
        sb[..., 1] = (-scale * (7.0 + torch.rand(scale.shape, generator=gen, device=DEV))).half()
        order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32).view(B, per)
        q = torch.randn((B, n, c["heads"], hd), generator=gen, device=DEV) * (1.5 * LOG2E / math.sqrt(hd))
        st = dict(q=q.to(DTYPES[c["dtype"]]), data=data, table=order, lens=torch.from_numpy(lens).to(DEV))
        if n == 1:
            st["q"] = st["q"][:, 0]
    elif c["op"] == "append":
        T, H, KVH, hd, page = c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
        pages = -(-T // page) + 3
        qkv = torch.randn((T, (H + 2 * KVH) * hd), generator=gen, device=DEV)
        pos = torch.randint(0, 8192, (T,), generator=gen, device=DEV, dtype=torch.int32)
        slots = torch.randperm(pages * page, generator=gen, device=DEV)[:T].contiguous()
        if T > 100 and not c["skip"]:      # a prompt: consecutive positions and places of shuffled pages
            pos = torch.arange(T, device=DEV, dtype=torch.int32)
            order = torch.randperm(pages, generator=gen, device=DEV)
            at = torch.arange(T, device=DEV)
            slots = order[at // page] * page + at % page
        if c["skip"]:
            slots[torch.rand(T, generator=gen, device=DEV) < 0.1] = -1
        angle = torch.arange(8192, device=DEV, dtype=torch.float64)[:, None] * \
            (1e6 ** (-torch.arange(hd // 2, device=DEV, dtype=torch.float64) * 2 / hd))
        st = dict(qkv=qkv.to(DTYPES[c["dtype"]]), pos=pos, slots=slots, cos=angle.cos().float(), sin=angle.sin().float(),
                  bias=torch.randn((H + 2 * KVH) * hd, generator=gen, device=DEV).half() if c["bias"] else None,
                  data=_blank(pages + 1, c))      # the last page is no cache's: the plain form's place for skipped tokens
    else:
        B, V = c["batch"], c["vocab"]
        x = torch.randn((B, V), generator=gen, device=DEV) * 2.0
        # a few likely tokens above the bulk, as a language model's logits have them
        top = torch.randint(0, V, (B, 64), generator=gen, device=DEV)
        x.scatter_add_(1, top, torch.rand((B, 64), generator=gen, device=DEV) * 10.0)
        if c["masked"]:
            bar = torch.rand((B, V), generator=gen, device=DEV) < 0.7
            x.masked_fill_(bar & (torch.rand((B, 1), generator=gen, device=DEV) < c["masked"]), -math.inf)
        opts = {k: c[k] for k in ("temp", "top_k", "top_p", "min_p")}
        if c["mixed"]:
            pick = lambda v, d: torch.tensor(v, dtype=d)[torch.from_numpy(rs.randint(0, len(v), B))].to(DEV)  # noqa: E731
            opts = dict(temp=pick([0.0, 0.5, c["temp"], 1.0, 1.5], torch.float32),
                        top_k=pick([0, 1, c["top_k"], 50, 2000], torch.int32),
                        top_p=pick([1.0, c["top_p"], 0.9, 0.5], torch.float32),
                        min_p=pick([0.0, 0.0, c["min_p"], 0.02], torch.float32))
        st = dict(logits=x.to(DTYPES[c["dtype"]]), u=torch.rand(B, generator=gen, device=DEV), **opts)
    st["case"] = c
    if own and c["op"] != "sample":
        from agxforge.kernels import kv4
        st["cache"] = kv4.KV4Cache.of(st["data"][:pages].view(pages, c["kv_heads"], -1), c["hd"], c["page"])
    return st


# ------------------------------------------------------------------------------------------------- the two forms
def run(st):
    c = st["case"]
    if own:
        from agxforge.kernels import kv4, sampling
        if c["op"] == "attention":
            return kv4.attention(st["q"], st["cache"], st["table"], st["lens"])
        if c["op"] == "append":
            q = kv4.append(st["cache"], st["qkv"], st["pos"], st["slots"], st["cos"], st["sin"], c["heads"],
                           bias=st["bias"])
            k, v = st["cache"].rows(st["slots"])
            return {"q": q, "k": k, "v": v}
        token, prob = sampling.sample(st["logits"], st["u"], temperature=st["temp"], top_k=st["top_k"],
                                      top_p=st["top_p"], min_p=st["min_p"])
        return {"token": token, "prob": prob}
    if c["op"] == "attention":
        return _plain_attention(st, c)
    return _plain_append(st, c) if c["op"] == "append" else _plain_sample(st, c)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1)


def _plain_attention(st, c):
    q, lens = st["q"], st["lens"].long()
    B, hd, KVH, H, n = c["batch"], c["hd"], c["kv_heads"], c["heads"], c["rows"]
    k, v, sb = _parts(st["data"][st["table"].long()].flatten(0, 1), hd)     # [B * pages, heads, tiles, ...]
    g = hd // 64

    def whole(codes, which):
        """Codes [B * pages, heads, tiles, 16 tokens, groups, 64] as values [B, heads, tokens, hd]."""
        sc = sb[:, :, :, :, which].float()
        x = codes.float() * sc[..., 0:1] + sc[..., 1:2]
        return x.unflatten(0, (B, -1)).transpose(1, 2).reshape(B, KVH, -1, hd)

    K = whole(_nibbles(k.transpose(-2, -3).reshape(*k.shape[:4], g, 32)).flatten(-2), 0)
    V = whole(_nibbles(v.permute(0, 1, 2, 3, 5, 6, 7, 4, 8).reshape(*k.shape[:4], g, 32)).flatten(-2), 1)
    L = K.shape[2]
    qf = q.float().view(B, n, KVH, H // KVH, hd).transpose(1, 2).reshape(B, KVH, n * (H // KVH), hd)
    S = torch.matmul(qf, K.transpose(-1, -2)).view(B, KVH, n, H // KVH, L)
    last = lens[:, None] - n + torch.arange(n, device=DEV)                   # the last key of each row
    bar = torch.arange(L, device=DEV) > last[..., None]
    S = S.masked_fill(bar[:, None, :, None, :], -math.inf)
    m = S.amax(-1, keepdim=True)
    p = torch.exp2(S - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    # values past a sequence's end may hold anything: they count as nothing
    V = V.masked_fill((torch.arange(L, device=DEV) >= lens[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(p.view(B, KVH, -1, L), V).view(B, KVH, n, H // KVH, hd)
    o = o / torch.where(total == 0, 1.0, total)
    return o.transpose(1, 2).reshape(q.shape).to(q.dtype)


def _quantised(x):
    """Codes, scales and biases of [T, heads, groups, 64]: scale = (max - min) / 15 and bias = min, in 16 bits."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = torch.where(hi > lo, (hi - lo) / 15.0, 1.0).half()
    b = lo.half()
    code = ((x - b.float()) / s.float()).round()
    code = torch.where(code.isfinite(), code, 0.0).clamp(0, 15).to(torch.uint8)
    return code, torch.cat([s, b], -1)


def _bytes(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _plain_append(st, c):
    T, H, KVH, hd, page = c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    g = hd // 64
    x = st["qkv"].float()
    if st["bias"] is not None:
        x = x + st["bias"].float()
    x = x.view(T, H + 2 * KVH, hd)
    pos = st["pos"].long()
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    x1, x2 = x[:, :H + KVH, :hd // 2], x[:, :H + KVH, hd // 2:]
    rot = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    q = (rot[:, :H] * float(np.float32(LOG2E / math.sqrt(hd))))
    kc, ksb = _quantised(rot[:, H:].reshape(T, KVH, g, 64))
    vc, vsb = _quantised(x[:, H + KVH:].reshape(T, KVH, g, 64))
    k, v, sb = _parts(st["data"], hd)
    spare = (st["data"].shape[0] - 1) * page
    slot = torch.where(st["slots"] < 0, spare, st["slots"])
    at, tile, t = slot // page, slot % page // 16, slot % 16
    k[at, :, tile, t] = _bytes(kc).view(T, KVH, g, 4, 8).transpose(2, 3)
    v[at, :, tile, t // 8, :, t // 2 % 4, t % 2] = _bytes(vc).view(T, KVH, g, 8, 4).transpose(2, 3)
    sb[at, :, tile, t] = torch.stack([ksb, vsb], 2)
    # what the cache holds at these places
    kh = _nibbles(k[at, :, tile, t].transpose(2, 3).reshape(T, KVH, g, 32)).flatten(-2)
    vh = _nibbles(v[at, :, tile, t // 8, :, t // 2 % 4, t % 2].transpose(2, 3).reshape(T, KVH, g, 32)).flatten(-2)
    pair = sb[at, :, tile, t].float()
    none = (st["slots"] < 0)[:, None, None]
    rows = [torch.where(none, 0.0, (h.float() * pair[:, :, i, :, 0:1] + pair[:, :, i, :, 1:2]).view(T, KVH, hd)).half()
            for i, h in ((0, kh), (1, vh))]
    return {"q": q.to(torch.bfloat16 if c["dtype"] == "bf16" else torch.float16), "k": rows[0], "v": rows[1]}


def _per_row(v, B, dtype):
    return v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((B,), v, dtype=dtype, device=DEV)


def _plain_sample(st, c):
    B, V = st["logits"].shape
    T, k = _per_row(st["temp"], B, torch.float32), _per_row(st["top_k"], B, torch.int64)
    p, least = _per_row(st["top_p"], B, torch.float32), _per_row(st["min_p"], B, torch.float32)
    x = st["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    best = x.amax(-1, keepdim=True)
    greedy = (T == 0)[:, None]
    d = torch.where(x == best, 0.0, x - best)
    e = torch.where(greedy, (d == 0).float(), torch.exp(d * (1.0 / torch.where(T == 0, 1.0, T))[:, None]))
    e = torch.where(x == -math.inf, 0.0, e)
    w = (e * W_ONE).to(torch.int64)          # whole units of 2^-40: their sums do not depend on the order
    rank = torch.sort(x, dim=-1, descending=True, stable=True).indices       # equal values: the lower index first
    ws = w.gather(-1, rank)
    ks = torch.where((k <= 0) | (k >= V), V, k)[:, None]
    ws = torch.where(torch.arange(V, device=DEV) < ks, ws, 0)
    before = ws.cumsum(-1) - ws
    total = ws.sum(-1)
    bar = torch.where(p >= 1, total.double(), (p.double() * total.double()).ceil()).to(torch.int64).clamp(min=1)
    ws = torch.where((before < bar[:, None]) | (p >= 1)[:, None], ws, 0)
    ws = torch.where(e.gather(-1, rank) >= least[:, None], ws, 0)
    kept = torch.zeros_like(w).scatter_(-1, rank, ws)
    up = kept.cumsum(-1)
    total = up[:, -1]
    u = torch.where(T == 0, 0.0, st["u"])
    r = torch.minimum((u.double() * total.double()).floor().to(torch.int64), total - 1)
    token = (up <= r[:, None]).sum(-1)
    own_w = kept.gather(-1, token.clamp(max=V - 1)[:, None])[:, 0]
    token = torch.where(total == 0, -1, token)
    prob = torch.where(total == 0, 0.0, torch.where(T == 0, 1.0, own_w.double() / total.double().clamp(min=1)))
    return {"token": token.to(torch.int32), "prob": prob.float()}


# ---------------------------------------------------------------------------------------------- in 64 bits, apart
def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["op"] == "attention":
        return _exact_attention(st, c)
    if c["op"] == "append":
        return _exact_append(st, c)
    return _exact_sample(st, c)


def _unpack(page_bytes, hd, tokens, which):
    """Values [tokens, hd] in 64 bits of one KV head's tiles, byte by byte from the layout's description."""
    tiles = page_bytes.reshape(-1, page_bytes.shape[-1])
    t = torch.arange(16, device=DEV)[:, None]
    dim = torch.arange(hd, device=DEV)[None]
    grp, in_g, G = dim // 64, dim % 64, hd // 64
    if which == 0:
        at = t * (hd // 2) + (in_g // 16) * (8 * G) + grp * 8 + in_g % 16 // 2
    else:
        at = 8 * hd + (t // 8) * 4 * hd + ((in_g // 8) * 4 + t % 8 // 2) * (8 * G) + (t % 2) * (4 * G) + grp * 4 + in_g % 8 // 2
    code = (tiles[:, at] >> (dim % 2 * 4).to(torch.uint8)) & 15
    pair = tiles[:, 16 * hd:].contiguous().view(torch.float16).view(-1, 16, 2, G, 2)[:, :, which].double()
    val = code.double() * pair[..., 0].repeat_interleave(64, -1) + pair[..., 1].repeat_interleave(64, -1)
    return val.view(-1, hd)[:tokens]


def _exact_attention(st, c):
    B, n, H, KVH, hd = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    q = st["q"].view(B, n, H, hd)
    out = torch.zeros((B, n, H, hd), dtype=torch.float64, device=DEV)
    for b, L in enumerate(st["lens"].tolist()):
        if L == 0:
            continue
        pages = st["data"][st["table"][b].long()]
        for j in range(KVH):
            K, V = (_unpack(pages[:, j], hd, L, i) for i in (0, 1))
            heads = slice(j * (H // KVH), (j + 1) * (H // KVH))
            S = torch.einsum("nhd,ld->nhl", q[b, :, heads].double(), K)
            ok = torch.arange(L, device=DEV)[None] <= (L - n + torch.arange(n, device=DEV))[:, None]
            S = torch.where(ok[:, None], S, -math.inf)
            P = torch.softmax(S * math.log(2.0), -1).nan_to_num(0.0)
            out[b, :, heads] = torch.einsum("nhl,ld->nhd", P, V)
    return out.view(st["q"].shape)


def _exact_append(st, c):
    T, H, KVH, hd = c["tokens"], c["heads"], c["kv_heads"], c["hd"]
    x = st["qkv"].double().cpu().numpy()
    if st["bias"] is not None:
        x = x + st["bias"].double().cpu().numpy()
    x = x.reshape(T, H + 2 * KVH, hd)
    pos, slots = st["pos"].cpu().numpy(), st["slots"].cpu().numpy()
    co = st["cos"].double().cpu().numpy()[pos][:, None]
    si = st["sin"].double().cpu().numpy()[pos][:, None]
    h = hd // 2
    z = (x[:, :H + KVH, :h] + 1j * x[:, :H + KVH, h:]) * (co + 1j * si)
    rot = np.concatenate([z.real, z.imag], -1)

    def held(y):
        y = y.reshape(T, KVH, hd // 64, 64)
        lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
        s = np.where(hi > lo, (hi - lo) / 15, 1.0).astype(np.float16).astype(np.float64)
        b = lo.astype(np.float16).astype(np.float64)
        v = np.clip(np.rint((y - b) / s), 0, 15) * s + b
        v[slots < 0] = 0
        return torch.from_numpy(v.reshape(T, KVH, hd))

    return {"q": torch.from_numpy(rot[:, :H] * (LOG2E / math.sqrt(hd))), "k": held(rot[:, H:]), "v": held(x[:, H + KVH:])}


def _exact_sample(st, c):
    B, V = st["logits"].shape
    probs = np.zeros(B)
    host = lambda v: v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(B, v)  # noqa: E731
    T, ks, ps, least, us = (host(st[n]) for n in ("temp", "top_k", "top_p", "min_p", "u"))
    logits = st["logits"].double().cpu().numpy()
    for i in range(B):
        x = logits[i]
        best = x.max()
        if best == -np.inf:
            continue
        if T[i] == 0:
            probs[i] = 1.0
            continue
        e = np.exp((x - best) / np.float64(T[i]))
        order = np.argsort(-x, kind="stable")
        if 0 < ks[i] < V:
            order = order[:ks[i]]
        if ps[i] < 1:
            up = np.cumsum(e[order])
            order = order[:max(1, int(np.searchsorted(up - e[order], np.float64(np.float32(ps[i])) * up[-1], "left")))]
        order = np.sort(order[e[order] >= np.float32(least[i])])
        up = np.cumsum(e[order])
        probs[i] = e[order][min(np.searchsorted(up, np.float64(us[i]) * up[-1], "right"), len(order) - 1)] / up[-1]
    return {"token": None, "prob": torch.from_numpy(probs)}
