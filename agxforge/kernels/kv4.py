"""A paged KV cache held in 4 bits, the append that fills it and the attention that reads it, on the B200 (the reference
keeps one contiguous fp16 cache and has no counterpart).

A cache has `pages` pages of `page_size` tokens; a sequence is a row of page numbers and a length. A place in the cache
is a slot, page * page_size + offset. Keys (after RoPE) and values are kept as scale * code + bias with 4-bit codes and
an fp16 scale and bias per token, KV head and group of 64 dims, the weight packs' affine format: 4.5 bits a value
where the fp16 cache takes 16.

    KV4Cache(pages, kv_heads, head_dim, page_size=64)   a new cache (KV4Cache.of wraps a caller's uint8 tensor)
    append(cache, qkv, positions, slots, cos, sin, heads, ...) -> q
                                    RoPE, q scale and the K/V write of `tokens` rows [q heads | k heads | v heads]: one
                                    row a sequence in a decode step, a whole prompt at once otherwise. Optional qkv
                                    bias (Qwen2) and QK-norm gains (Qwen3) are applied first. q is ready for attention
    attention(q, cache, page_table, lengths) -> out
                                    q [batch, heads, head_dim], or [batch, rows, heads, head_dim] for the last `rows`
                                    tokens of each sequence (drafts to verify, a prompt chunk): row i sees keys
                                    0 .. length - rows + i, and a row that sees none gives zeros
    KV4Cache.rows(slots) -> (k, v)  the fp16 values held at some slots

Everything is enqueued on torch's current stream. Shapes and types are checked on the host (ValueError); positions,
slots, lengths and page numbers live on the device and are checked there: one out of range is left out (a length:
clamped) and sets a bit of the context's error word, which `check_errors()` reads and raises.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from agxforge_b200 import _native as N

LOG2E = 1.4426950408889634
DTYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}


def _stream(index):
    """torch's current stream on the device; its default stream (handle 0) as cudaStreamLegacy (1), because the C ABI
    reads NULL as the context's own stream."""
    return C.c_void_p(torch.cuda.current_stream(index).cuda_stream or 1)


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _check(t, dtype, device, what):
    if t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError("%s: contiguous %s on the cache's device" % (what, str(dtype)[6:]))


def token_bytes(head_dim):
    """Bytes one token takes in one KV head: the codes of K and V and an fp16 scale and bias per 64 dims of each."""
    _need(head_dim in (64, 128), "kv4: head_dim 64 or 128")
    return head_dim + 8 * (head_dim // 64)


class KV4Cache:
    """`data` uint8 [pages, kv_heads, page_size * token_bytes(head_dim)], 16-token tiles in the library's byte order
    (include/agxc.h). Pages are the caller's to hand out; a page's bytes hold finite values from the start."""

    def __init__(self, pages, kv_heads, head_dim, page_size=64, device=0, data=None):
        _need(head_dim in (64, 128), "kv4: head_dim 64 or 128")
        _need(page_size >= 16 and page_size % 16 == 0, "kv4: page_size a positive multiple of 16")
        _need(pages >= 1 and kv_heads >= 1, "kv4: at least one page and one KV head")
        shape = (pages, kv_heads, page_size * token_bytes(head_dim))
        if data is None:
            data = torch.zeros(shape, dtype=torch.uint8, device="cuda:%d" % device)
        _need(data.dtype == torch.uint8 and tuple(data.shape) == shape and data.is_contiguous() and data.is_cuda,
              "kv4: data is contiguous uint8 %s on the GPU" % (shape,))
        self.data, self.pages, self.kv_heads, self.head_dim, self.page_size = data, pages, kv_heads, head_dim, page_size
        self.device, self.index = data.device, data.device.index
        self._c = N.Kv4Cache(data.data_ptr(), pages, kv_heads, head_dim, page_size)

    @classmethod
    def of(cls, data, head_dim, page_size=64):
        """The cache whose bytes are `data` [pages, kv_heads, page_size * token_bytes(head_dim)]."""
        _need(data.dim() == 3, "kv4: data is [pages, kv_heads, bytes]")
        return cls(data.shape[0], data.shape[1], head_dim, page_size, data=data)

    @property
    def nbytes(self):
        return self.data.numel()

    def rows(self, slots):
        """(k, v) fp16 [tokens, kv_heads, head_dim]: the values held at `slots` (int64); zeros for a negative slot."""
        _check(slots, torch.int64, self.device, "rows: slots")
        k, v = torch.empty((2, slots.numel(), self.kv_heads, self.head_dim), dtype=torch.float16, device=self.device)
        N.check(N.lib().agxc_kv4_rows_dev(N.context(self.index), C.byref(self._c), slots.data_ptr(), slots.numel(),
                                          k.data_ptr(), v.data_ptr(), _stream(self.index)), "rows")
        return k, v


def append(cache, qkv, positions, slots, cos, sin, heads, bias=None, q_norm=None, k_norm=None, eps=1e-6, qscale=None,
           q_dtype=None, out=None):
    """Rotate and scale q, rotate, quantise and write k, quantise and write v. qkv [tokens, (heads + 2 kv_heads) *
    head_dim] fp32, fp16 or bf16 (rows may be strided); positions int32 [tokens] index the fp32 RoPE tables cos and sin
    [n, head_dim / 2]; slots int64 [tokens], each at most once, negative = not written. bias fp16
    [(heads + 2 kv_heads) * head_dim], q_norm and k_norm fp16 [head_dim]. qscale defaults to log2(e) / sqrt(head_dim)
    (the attention's softmax is base 2). Returns q [tokens, heads, head_dim], bf16 for bf16 rows and fp16 otherwise
    unless q_dtype says which."""
    dev, hd, idx = cache.device, cache.head_dim, cache.index
    width = (heads + 2 * cache.kv_heads) * hd
    _need(heads >= 1 and heads % cache.kv_heads == 0, "append: heads a positive multiple of kv_heads")
    _need(qkv.dim() == 2 and qkv.shape[1] == width,
          "append: qkv is [tokens, (heads + 2 kv_heads) * head_dim] = [tokens, %d]" % width)
    _need(qkv.dtype in DTYPES and qkv.device == dev and (qkv.stride(1) == 1 or width == 1),
          "append: qkv fp32, fp16 or bf16 on the cache's device, its rows contiguous")
    T = qkv.shape[0]
    _check(positions, torch.int32, dev, "append: positions")
    _check(slots, torch.int64, dev, "append: slots")
    _need(positions.numel() == T and slots.numel() == T, "append: one position and one slot a token")
    _check(cos, torch.float32, dev, "append: cos")
    _check(sin, torch.float32, dev, "append: sin")
    _need(cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] == hd // 2 and cos.shape[0] >= 1,
          "append: cos and sin are [n, head_dim / 2]")
    if bias is not None:
        _check(bias, torch.float16, dev, "append: bias")
        _need(bias.numel() == width, "append: bias is [(heads + 2 kv_heads) * head_dim]")
    _need((q_norm is None) == (k_norm is None), "append: q_norm and k_norm, or neither")
    if q_norm is not None:
        for g in (q_norm, k_norm):
            _check(g, torch.float16, dev, "append: q_norm and k_norm")
            _need(g.numel() == hd, "append: q_norm and k_norm are [head_dim]")
    if out is None:
        if q_dtype is None:
            q_dtype = torch.bfloat16 if qkv.dtype == torch.bfloat16 else torch.float16
        out = torch.empty((T, heads, hd), dtype=q_dtype, device=dev)
    else:
        _check(out, out.dtype, dev, "append: out")
        _need(out.shape == (T, heads, hd), "append: out is [tokens, heads, head_dim]")
    _need(out.dtype in (torch.float16, torch.bfloat16), "append: q fp16 or bf16")
    if qscale is None:
        qscale = float(np.float32(LOG2E / math.sqrt(hd)))
    a = N.Kv4AppendArgs(cache._c, qkv.data_ptr(), qkv.stride(0) if T > 1 else width, DTYPES[qkv.dtype], T, heads,
                        positions.data_ptr(), slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                        None if bias is None else bias.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
                        None if k_norm is None else k_norm.data_ptr(), eps, qscale, out.data_ptr(), DTYPES[out.dtype])
    N.check(N.lib().agxc_kv4_append_dev(N.context(idx), C.byref(a), _stream(idx)), "append")
    return out


def attention(q, cache, page_table, lengths, out=None):
    """Base-2 softmax attention of q (as append returns it: scaled by log2(e) / sqrt(head_dim)), fp16 or bf16
    [batch, heads, head_dim] or [batch, rows, heads, head_dim], over the cache: page_table int32 [batch, max_pages]
    (its rows may be strided), lengths int32 [batch], the tokens held with the rows' own among them. Returns out of
    q's shape and type."""
    dev, idx = cache.device, cache.index
    _need(q.dim() in (3, 4) and q.shape[-1] == cache.head_dim,
          "attention: q is [batch, heads, head_dim] or [batch, rows, heads, head_dim] with head_dim %d" % cache.head_dim)
    _need(q.dtype in (torch.float16, torch.bfloat16) and q.device == dev, "attention: q fp16 or bf16 on the cache's device")
    B, n, H = q.shape[0], 1 if q.dim() == 3 else q.shape[1], q.shape[-2]
    _need(H >= 1 and H % cache.kv_heads == 0, "attention: heads a positive multiple of kv_heads")
    _check(lengths, torch.int32, dev, "attention: lengths")
    _need(lengths.numel() == B, "attention: one length a sequence")
    _need(page_table.dim() == 2 and page_table.shape[0] == B and page_table.dtype == torch.int32 and
          page_table.device == dev and (page_table.stride(1) == 1 or page_table.shape[1] <= 1),
          "attention: page_table int32 [batch, max_pages] on the cache's device, its rows contiguous")
    if not q.is_contiguous():
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out, q.dtype, dev, "attention: out")
        _need(out.shape == q.shape, "attention: out has q's shape")
    mp = page_table.shape[1]
    a = N.Kv4AttentionArgs(cache._c, q.data_ptr(), out.data_ptr(), DTYPES[q.dtype], B, n, H, page_table.data_ptr(),
                           page_table.stride(0) if B > 1 else mp, mp, lengths.data_ptr(), None, 0)
    L, ctx = N.lib(), N.context(idx)
    need = L.agxc_kv4_attention_workspace(ctx, C.byref(a))
    if need < 0:
        N.check(N.EINVAL, "attention")
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace_dev, a.workspace_bytes = ws.data_ptr(), need
    N.check(L.agxc_kv4_attention_dev(ctx, C.byref(a), _stream(idx)), "attention")
    return out


def check_errors(device=0):
    """Wait for the device, read and clear the context's error word, and raise RuntimeError if a call since the last
    check met a position, slot, length or page out of range."""
    torch.cuda.synchronize(device)
    w = C.c_uint32()
    N.check(N.lib().agxc_ctx_error_word(N.context(device), C.byref(w)), "error_word")
    if w.value:
        raise RuntimeError("kv4: a position, slot, length or page was out of range (error word 0x%x)" % w.value)
