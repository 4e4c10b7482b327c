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

Everything is enqueued on torch's current stream of the cache's device, whichever device is current. Shapes and types are
checked on the host (ValueError); positions, slots, lengths and page numbers live on the device and are checked there: one
out of range is left out (a length: clamped) and sets a bit of the context's error word, which `check_errors()` reads and
raises.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from agxforge_b200 import _native as N

LOG2E = 1.4426950408889634
_QSCALE = {hd: float(np.float32(LOG2E / math.sqrt(hd))) for hd in (64, 128)}
DTYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}


# the handle of torch's current stream on a device, without a Stream object around it (1.2 us a call less)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(index):
    """torch's current stream on the device; its default stream (handle 0) as cudaStreamLegacy (1), because the C ABI
    reads NULL as the context's own stream."""
    return _raw_stream(index) or 1


def _need(ok, text):
    if not ok:
        raise ValueError(text)


def _check(t, dtype, index, what):
    if t.dtype is not dtype or t.get_device() != index or not t.is_contiguous():
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
        self._workspace = {}        # bytes that an attention call of a shape needs

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
        idx, T = self.index, slots.numel()
        _check(slots, torch.int64, idx, "rows: slots")
        kv = torch.empty(2, T, self.kv_heads, self.head_dim, dtype=torch.float16, device=self.device)
        at = kv.data_ptr()
        rc = N.lib().agxc_kv4_rows_dev(N.context(idx), C.byref(self._c), slots.data_ptr(), T, at,
                                       at + 2 * T * self.kv_heads * self.head_dim, _stream(idx))
        if rc:
            N.check(rc, "rows")
        return kv.unbind(0)


def append(cache, qkv, positions, slots, cos, sin, heads, bias=None, q_norm=None, k_norm=None, eps=1e-6, qscale=None,
           q_dtype=None, out=None):
    """Rotate and scale q, rotate, quantise and write k, quantise and write v. qkv [tokens, (heads + 2 kv_heads) *
    head_dim] fp32, fp16 or bf16 (rows may be strided); positions int32 [tokens] index the fp32 RoPE tables cos and sin
    [n, head_dim / 2]; slots int64 [tokens], each at most once, negative = not written. bias fp16
    [(heads + 2 kv_heads) * head_dim], q_norm and k_norm fp16 [head_dim]. qscale defaults to log2(e) / sqrt(head_dim)
    (the attention's softmax is base 2). Returns q [tokens, heads, head_dim], bf16 for bf16 rows and fp16 otherwise
    unless q_dtype says which."""
    hd, idx = cache.head_dim, cache.index
    width = (heads + 2 * cache.kv_heads) * hd
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError("append: heads a positive multiple of kv_heads")
    shape = qkv.shape
    if len(shape) != 2 or shape[1] != width:
        raise ValueError("append: qkv is [tokens, (heads + 2 kv_heads) * head_dim] = [tokens, %d]" % width)
    T = shape[0]
    ld, inner = qkv.stride()
    kind = DTYPES.get(qkv.dtype)
    if kind is None or qkv.get_device() != idx or inner != 1:
        raise ValueError("append: qkv fp32, fp16 or bf16 on the cache's device, its rows contiguous")
    _check(positions, torch.int32, idx, "append: positions")
    _check(slots, torch.int64, idx, "append: slots")
    if positions.numel() != T or slots.numel() != T:
        raise ValueError("append: one position and one slot a token")
    _check(cos, torch.float32, idx, "append: cos")
    _check(sin, torch.float32, idx, "append: sin")
    shape = cos.shape
    if len(shape) != 2 or shape != sin.shape or shape[1] != hd // 2 or shape[0] < 1:
        raise ValueError("append: cos and sin are [n, head_dim / 2]")
    if bias is not None:
        _check(bias, torch.float16, idx, "append: bias")
        _need(bias.numel() == width, "append: bias is [(heads + 2 kv_heads) * head_dim]")
    _need((q_norm is None) == (k_norm is None), "append: q_norm and k_norm, or neither")
    if q_norm is not None:
        for g in (q_norm, k_norm):
            _check(g, torch.float16, idx, "append: q_norm and k_norm")
            _need(g.numel() == hd, "append: q_norm and k_norm are [head_dim]")
    if out is None:
        if q_dtype is None:
            q_dtype = torch.bfloat16 if kind == N.BF16 else torch.float16
        _need(q_dtype is torch.float16 or q_dtype is torch.bfloat16, "append: q fp16 or bf16")
        out = torch.empty(T, heads, hd, dtype=q_dtype, device=cache.device)
        q_kind = DTYPES[q_dtype]
    else:
        _need(out.dtype in (torch.float16, torch.bfloat16), "append: q fp16 or bf16")
        _check(out, out.dtype, idx, "append: out")
        _need(out.shape == (T, heads, hd), "append: out is [tokens, heads, head_dim]")
        q_kind = DTYPES[out.dtype]
    if qscale is None:
        qscale = _QSCALE[hd]
    a = N.Kv4AppendArgs(cache._c, qkv.data_ptr(), ld if T > 1 else width, kind, T, heads, positions.data_ptr(),
                        slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), shape[0],
                        None if bias is None else bias.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
                        None if k_norm is None else k_norm.data_ptr(), eps, qscale, out.data_ptr(), q_kind)
    rc = N.lib().agxc_kv4_append_dev(N.context(idx), C.byref(a), _stream(idx))
    if rc:
        N.check(rc, "append")
    return out


def attention(q, cache, page_table, lengths, out=None):
    """Base-2 softmax attention of q (as append returns it: scaled by log2(e) / sqrt(head_dim)), fp16 or bf16
    [batch, heads, head_dim] or [batch, rows, heads, head_dim], over the cache: page_table int32 [batch, max_pages]
    (its rows may be strided), lengths int32 [batch], the tokens held with the rows' own among them. Returns out of
    q's shape and type."""
    hd, idx = cache.head_dim, cache.index
    shape = q.shape
    if len(shape) not in (3, 4) or shape[-1] != hd:
        raise ValueError("attention: q is [batch, heads, head_dim] or [batch, rows, heads, head_dim] with head_dim %d" % hd)
    kind = DTYPES.get(q.dtype)
    if kind is None or kind == N.F32 or q.get_device() != idx:
        raise ValueError("attention: q fp16 or bf16 on the cache's device")
    B, n, H = shape[0], 1 if len(shape) == 3 else shape[1], shape[-2]
    if H < 1 or H % cache.kv_heads:
        raise ValueError("attention: heads a positive multiple of kv_heads")
    _check(lengths, torch.int32, idx, "attention: lengths")
    if lengths.numel() != B:
        raise ValueError("attention: one length a sequence")
    pages = page_table.shape
    if len(pages) != 2 or pages[0] != B or page_table.dtype is not torch.int32 or \
            page_table.get_device() != idx or (page_table.stride(1) != 1 and pages[1] > 1):
        raise ValueError("attention: page_table int32 [batch, max_pages] on the cache's device, its rows contiguous")
    if not q.is_contiguous():
        q = q.contiguous()
    if out is None:
        out = torch.empty_like(q)
    else:
        _check(out, q.dtype, idx, "attention: out")
        _need(out.shape == shape, "attention: out has q's shape")
    mp = pages[1]
    ld = page_table.stride(0) if B > 1 else mp
    if ld > 0x7fffffff:
        raise ValueError("attention: page_table rows less than 2^31 entries apart")
    a = N.Kv4AttentionArgs(cache._c, q.data_ptr(), out.data_ptr(), kind, B, n, H, page_table.data_ptr(), ld, mp,
                           lengths.data_ptr(), None, 0)
    L, ctx = N.lib(), N.context(idx)
    need = cache._workspace.get((kind, B, n, H, mp))
    if need is None:
        need = L.agxc_kv4_attention_workspace(ctx, C.byref(a))
        if need < 0:
            N.check(N.EINVAL, "attention")
        if len(cache._workspace) >= 1024:
            cache._workspace.clear()
        cache._workspace[kind, B, n, H, mp] = need
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=cache.device)
        a.workspace_dev, a.workspace_bytes = ws.data_ptr(), need
    rc = L.agxc_kv4_attention_dev(ctx, C.byref(a), _stream(idx))
    if rc:
        N.check(rc, "attention")
    return out


def check_errors(device=0):
    """Wait for the device, read and clear the error word of its context (the operators of a context share it), and raise if
    anything set it since the last check: TimeoutError where a bounded wait gave up, RuntimeError otherwise (a position,
    slot, length or page out of range)."""
    torch.cuda.synchronize(device)
    w = C.c_uint32()
    N.check(N.lib().agxc_ctx_error_word(N.context(device), C.byref(w)), "error_word")
    if w.value:
        what = [text for bit, text in N.ERRORS.items() if w.value & bit] or ["an error"]
        raise (TimeoutError if w.value & N.ERR_WAITS else RuntimeError)(
            "kv4: %s (error word 0x%x)" % ("; ".join(what), w.value))
