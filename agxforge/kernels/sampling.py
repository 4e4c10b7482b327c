"""The choice of a token from logits with temperature, top-k, top-p and min-p, at given uniform random numbers (the
reference chooses greedily, agxforge/kernels/argmax.py; greedy rows are temperature 0 here).

    sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> (tokens, probs)

Each option is one number for all rows or a device tensor with one a row. Per row: tokens are ranked by logit, equal
logits by index (NaN ranks as -inf); weights are exp((l - max) / T) in whole units of 2^-40, so sums are exact and a row
gives the same token whatever batch it is in. Kept are the first `top_k` ranks (top_k <= 0: all), of those the ranks
whose weight before them is below top_p of the total (top_p >= 1: all; the first always), of those the weights >=
min_p (of the largest). The token is the first kept index at which the cumulative weight exceeds u of the total, and
prob its share of the kept weight. Temperature 0 takes the first maximum; a row with no finite logit, or that keeps nothing
(min_p above 1), gives -1 and 0. So does a temperature of an array that is below 0 or NaN, and it sets a bit of the error
word that kv4.check_errors reads; a number like that is refused (ValueError).
"""
from __future__ import annotations

import ctypes as C

import torch

from agxforge_b200 import _native as N
from agxforge.kernels.kv4 import DTYPES, _stream


def _option(v, dtype, B, index, name):
    """(number, device pointer): a number for all rows, or a tensor with one a row."""
    if type(v) is not float and type(v) is not int and isinstance(v, torch.Tensor):  # torch's own check takes a while
        if v.dtype is not dtype or v.get_device() != index or v.numel() != B or not v.is_contiguous():
            raise ValueError("sample: %s is a number or contiguous %s [batch] on the logits' device" % (name, str(dtype)[6:]))
        return 0, v.data_ptr()
    return v, None


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Tokens int32 [batch] and their probabilities fp32 [batch] for logits [batch, vocab] fp32, fp16 or bf16 (rows may
    be strided, vocab at most 1,048,576) and u fp32 [batch] in [0, 1). temperature, top_p and min_p: numbers or fp32 [batch]; top_k: a number or
    int32 [batch]."""
    kind, idx = DTYPES.get(logits.dtype), logits.get_device()
    if logits.dim() != 2 or kind is None or idx < 0 or logits.shape[1] < 1 or \
            (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("sample: logits are [batch, vocab] fp32, fp16 or bf16 on the GPU, their rows contiguous")
    B, V = logits.shape
    if u.dtype is not torch.float32 or u.get_device() != idx or u.numel() != B or not u.is_contiguous():
        raise ValueError("sample: u is contiguous float32 [batch] on the logits' device")
    t, td = _option(temperature, torch.float32, B, idx, "temperature")
    k, kd = _option(top_k, torch.int32, B, idx, "top_k")
    p, pd = _option(top_p, torch.float32, B, idx, "top_p")
    m, md = _option(min_p, torch.float32, B, idx, "min_p")
    if not t >= 0:
        raise ValueError("sample: temperature >= 0")
    if not -1 <= k <= V:           # all of them; the call takes 32 bits
        k = 0
    dev = logits.device
    tokens = torch.empty(B, dtype=torch.int32, device=dev)
    probs = torch.empty(B, dtype=torch.float32, device=dev)
    a = N.SampleArgs(logits.data_ptr(), logits.stride(0) if B > 1 else V, kind, B, V, u.data_ptr(), t, p, m, k, td, kd, pd,
                     md, tokens.data_ptr(), probs.data_ptr())
    rc = N.lib().agxc_sample_dev(N.context(idx), C.byref(a), _stream(idx))
    if rc:
        N.check(rc, "sample")
    return tokens, probs
