"""Serving with a paged 4-bit KV cache and sampling (no counterpart in the reference): the decoder's packs through the
GEMV family, K/V in kernels.kv4 pages shared by all sequences, tokens by kernels.sampling.

    m = PagedModel(config, weights, pages=512)      weights: reference-format packs and fp16 vectors, as assemble.build
                                                    takes and keeps them ({(layer, role): (packed, scales, biases)})
    s = m.add(prompt)                               a sequence: its prompt in chunks of up to 256 rows, all but the last
                                                    token, whose row the next step runs
    m.step(u, temperature=0.8, top_k=50)            one token for every sequence, {sequence: (token, probability)}
    m.free(s)                                       its pages go back

A step is, per layer: RMSNorm + qkv GEMV; append (bias, QK-norm, RoPE, 4-bit K/V); attention over the pages; o_proj +
residual; RMSNorm + gate/up + SiLU mul; down + residual; then the final norm, the head and the sampler. Rows go through
the GEMVs eight at a time; the append, the attention and the sampler take all of them at once.
"""
from __future__ import annotations

import contextlib
import functools

import numpy as np
import torch

from agxforge.inference import assemble
from agxforge.kernels import kv4, sampling
from agxforge.kernels import qmv as Q

CHUNK = 256          # prompt rows a pass


def _on_device(method):
    """The model's device is current while a method runs: the GEMV calls take the current device's stream."""
    @functools.wraps(method)
    def run(self, *args, **kwargs):
        with torch.cuda.device(self.device):
            return method(self, *args, **kwargs)
    return run


def _device(a, device):
    if isinstance(a, np.ndarray):
        a = np.ascontiguousarray(a)
        a = torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a.view(np.int16) if a.dtype == np.uint16 else a)
    return a.to("cuda:%d" % device).contiguous()


class PagedModel:
    """The weights on the device, a cache of `pages` pages a layer, and the sequences that hold them."""

    def __init__(self, config, weights, pages, page_size=64, device=0):
        cfg = assemble.configure(config)
        self.shape = S = cfg["shape"]
        if S.HEAD_DIM not in (64, 128) or S.HEADS % S.KV_HEADS:
            raise ValueError("PagedModel: head_dim 64 or 128 and heads a multiple of kv_heads")
        self.device, self.page_size = device, page_size
        with torch.cuda.device(device):
            self._load(cfg, weights, pages)

    def _load(self, cfg, weights, pages):
        S, device, page_size = self.shape, self.device, self.page_size
        bits, sdt = cfg["bits"], cfg["scale_dtype"]
        dev = lambda key: _device(weights[key], device).to(torch.float16)  # noqa: E731
        pack = lambda l, role, n, k: Q.Pack(*weights[(l, role)], n, k, bits, sdt, device)  # noqa: E731
        self.layers = []
        for l in range(S.LAYERS):
            d = {r: pack(l, r, n, k) for r, n, k in S.matrices() if r not in ("gate", "up")}
            d["gateup"] = Q.Pack.gateup(weights[(l, "gate")], weights[(l, "up")], S.FFN, S.D_MODEL, bits, sdt, device)
            for v in ("attn_gain", "ffn_gain"):
                d[v] = dev((l, v))
            d["bias"] = dev((l, "qkv_bias")) if S.QKV_BIAS else None
            d["q_norm"], d["k_norm"] = (dev((l, v)) if S.QK_NORM else None for v in ("q_norm", "k_norm"))
            d["cache"] = kv4.KV4Cache(pages, S.KV_HEADS, S.HEAD_DIM, page_size, device)
            self.layers.append(d)
        self.head = pack(None, "head", S.VOCAB, S.D_MODEL)
        self.embed, self.final_gain = dev("embed"), dev("final_gain")
        self.spare = list(range(pages))[::-1]        # pages nobody holds
        self.seqs = {}                               # id -> {pages, tokens, held}
        self._next = 0
        self._tables(1024)

    def _tables(self, n):
        hd = self.shape.HEAD_DIM
        inv = 1.0 / self.shape.ROPE_THETA ** (np.arange(0, hd, 2, dtype=np.float64) / hd)
        ang = np.arange(n, dtype=np.float64)[:, None] * inv
        self.cos, self.sin = (_device(f(ang).astype(np.float32), self.device) for f in (np.cos, np.sin))

    # ---------------------------------------------------------------- sequences
    @_on_device
    def add(self, prompt):
        """A sequence with its prompt (at least one token); returns its id. MemoryError where the pages do not reach; what
        raises leaves no sequence behind."""
        toks = [int(t) for t in prompt]
        if not toks or min(toks) < 0 or max(toks) >= self.shape.VOCAB:
            raise ValueError("add: a prompt of at least one token of the vocabulary")
        s, self._next = self._next, self._next + 1
        self.seqs[s] = dict(pages=[], tokens=toks, held=0)
        try:
            while self.seqs[s]["held"] < len(toks) - 1:
                n = min(CHUNK, len(toks) - 1 - self.seqs[s]["held"])
                self._rows([s], n)
            kv4.check_errors(self.device)
        except BaseException:
            self.free(s)
            raise
        return s

    def free(self, s):
        self.spare.extend(self.seqs.pop(s)["pages"][::-1])

    def _reserve(self, s, length):
        q = self.seqs[s]
        need = -(-length // self.page_size) - len(q["pages"])
        if need > len(self.spare):
            raise MemoryError("PagedModel: %d pages wanted, %d spare" % (need, len(self.spare)))
        for _ in range(need):
            q["pages"].append(self.spare.pop())

    # ---------------------------------------------------------------- the pass
    def _gemv(self, pack, x, **kw):
        res = kw.pop("res", None)
        out = [Q.qmv(pack, x[i:i + 8], res=None if res is None else res[i:i + 8], **kw) for i in range(0, x.shape[0], 8)]
        return out[0] if len(out) == 1 else torch.cat(out)

    def _rows(self, ids, n):
        """The next n tokens of each sequence through every layer; their K/V are held afterwards. Returns the rows that
        come out of the last layer, fp16 [sequences * n, d_model]."""
        S, P = self.shape, self.page_size
        for s in ids:
            self._reserve(s, self.seqs[s]["held"] + n)
        at = [self.seqs[s]["held"] for s in ids]
        if max(at) + n > self.cos.shape[0]:
            self._tables(2 * (max(at) + n))
        pos = np.asarray(at)[:, None] + np.arange(n)
        pages = np.zeros((len(ids), max(len(self.seqs[s]["pages"]) for s in ids)), np.int32)
        for i, s in enumerate(ids):
            pages[i, :len(self.seqs[s]["pages"])] = self.seqs[s]["pages"]
        slots = np.take_along_axis(pages, pos // P, 1).astype(np.int64) * P + pos % P
        toks = np.asarray([self.seqs[s]["tokens"][a:a + n] for s, a in zip(ids, at)])
        dev = lambda a, t: _device(np.ascontiguousarray(a.astype(t)), self.device)  # noqa: E731
        x = self.embed[dev(toks.reshape(-1), np.int64)]
        pos, slots, table = dev(pos.reshape(-1), np.int32), dev(slots.reshape(-1), np.int64), dev(pages, np.int32)
        lengths = dev(np.asarray(at) + n, np.int32)
        for d in self.layers:
            qkv = self._gemv(d["qkv"], x, norm_gain=d["attn_gain"], eps=S.EPS)
            q = kv4.append(d["cache"], qkv, pos, slots, self.cos, self.sin, S.HEADS, bias=d["bias"], q_norm=d["q_norm"],
                           k_norm=d["k_norm"], eps=S.EPS)
            a = kv4.attention(q.view(len(ids), n, S.HEADS, S.HEAD_DIM), d["cache"], table, lengths)
            h = self._gemv(d["wo"], a.view(len(ids) * n, -1), epi="add16", res=x)
            act = self._gemv(d["gateup"], h, norm_gain=d["ffn_gain"], eps=S.EPS, epi="swiglu")
            x = self._gemv(d["down"], act, epi="add32_to16", res=h)
        for s in ids:
            self.seqs[s]["held"] += n
        return x

    @contextlib.contextmanager
    def _or_as_before(self, ids):
        """What fails leaves the sequences as they were: asked for again, the pass writes the same K and V once more."""
        held = {s: self.seqs[s]["held"] for s in ids}
        try:
            yield
        except BaseException:
            for s, n in held.items():
                self.seqs[s]["held"] = n
            raise

    def _ids(self, ids):
        ids = sorted(self.seqs) if ids is None else list(ids)
        if not ids:
            raise ValueError("logits: no sequence")
        if len(set(ids)) != len(ids):
            raise ValueError("logits: a sequence named twice")
        for s in ids:
            if self.seqs[s]["held"] != len(self.seqs[s]["tokens"]) - 1:
                raise ValueError("logits: sequence %d has no new token" % s)
        return ids

    def _logits(self, ids):
        return self._gemv(self.head, self._rows(ids, 1), norm_gain=self.final_gain, eps=self.shape.EPS)

    @_on_device
    def logits(self, ids=None):
        """Run the last token of each sequence (all of them by default, in the order of their ids): logits fp32
        [sequences, vocab] of the next one, and the ids."""
        ids = self._ids(ids)
        with self._or_as_before(ids):
            lg = self._logits(ids)
            kv4.check_errors(self.device)
        return lg, ids

    @_on_device
    def step(self, u, ids=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """One token for each sequence, chosen at the uniform numbers u (one a sequence, in the order of the ids); the
        options are sampling.sample's. Returns {id: (token, probability)}; a step that raises leaves the sequences as
        they were."""
        ids = self._ids(ids)
        with self._or_as_before(ids):
            lg = self._logits(ids)
            ut = torch.as_tensor(np.asarray(u, np.float32)).to(lg.device).reshape(-1)
            tok, prob = sampling.sample(lg, ut, temperature, top_k, top_p, min_p)
            out = dict(zip(ids, zip(tok.tolist(), prob.tolist())))
            kv4.check_errors(self.device)
            none = [s for s, (t, _) in out.items() if t < 0]
            if none:
                raise RuntimeError("step: no token for sequence %s (no finite logit, or a min_p above 1)"
                                   % ", ".join(map(str, none)))
        for s, (t, _) in out.items():
            self.seqs[s]["tokens"].append(t)
        return out
