"""Next-token sampling from given uniform numbers: CUDA tensors run ``csrc/sample.cu`` (one launch, nothing read by the host; it may be
captured into a graph), CPU tensors the plain statement of ``reference``."""
from __future__ import annotations

import ctypes as C

import torch

from . import reference as ref

BF16, F32 = torch.bfloat16, torch.float32
MAX_VOCAB = 8 * 40 * 1024


class _Sample(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("ld", C.c_longlong), ("V", C.c_int), ("per", C.c_int)] + \
               [(n, C.c_void_p) for n in ("uniform", "temperature", "top_p", "min_p", "top_k")] + [(n, C.c_float) for n in ("t", "p", "m")] + \
               [("k", C.c_int), ("out", C.c_void_p)]


_fns = None


def _k():
    global _fns
    if _fns is None:
        from . import cuda as K

        _fns = (K, K._sig("b200_sample", [C.POINTER(_Sample), C.c_int, C.c_int, C.c_void_p]))
    return _fns


def _setting(x, name: str, logits, dtype, low, high):
    """(tensor or None, number) of a setting given as a number or as one per row."""
    if torch.is_tensor(x):
        if x.shape != logits.shape[:1] or x.dtype != dtype or x.device != logits.device or not x.is_contiguous():
            raise ValueError(f"{name}: a number or a contiguous {dtype} tensor [{logits.shape[0]}] on the logits' device")
        return x, 0
    x = 0 if x is None else x
    if not low <= x <= high:
        raise ValueError(f"{name} lies in {low} .. {high}: got {x}")
    return None, x


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """One token (int64) per row of ``logits`` [B, vocab] (bf16 or fp32) from the row's number ``uniform[b]`` in [0, 1) (fp32): the first
    index, in the vocabulary's order, at which the sum of the kept probabilities exceeds ``uniform`` times their total (a number below 0 or
    NaN counts as 0, one of 1 or more gives the last kept token).

    Kept is what all filters keep, as in ``models.sampling``: ``top_k`` (0: off) drops what is below the k-th largest logit, ``top_p`` (0 or
    1: off) keeps the longest prefix of the descending order (equal logits: lowest index first) whose probabilities sum to at most
    ``top_p`` and at least one token, ``min_p`` (0: off) drops what has less than ``min_p`` times the largest probability.  Every setting is a number
    or a tensor with one value per row (fp32, ``top_k`` int32).  A ``temperature`` of 0 picks the largest logit, the lowest index among
    equal ones.  NaN logits count as -inf; a row without any logit above -inf gives -1."""
    if logits.dim() != 2 or logits.dtype not in (BF16, F32) or logits.shape[1] == 0 or logits.stride(1) != 1:
        raise ValueError("logits are bf16 or fp32 [B, vocab] with contiguous rows")
    B, V = logits.shape
    if V > MAX_VOCAB:
        raise ValueError(f"vocabularies of up to {MAX_VOCAB}: got {V}")
    if B > 1 and logits.stride(0) < V:
        raise ValueError("rows of logits do not overlap")
    if uniform.shape != (B,) or uniform.dtype != F32 or uniform.device != logits.device or not uniform.is_contiguous():
        raise ValueError(f"uniform is a contiguous fp32 tensor [{B}] on the logits' device")
    inf = float("inf")
    t, t0 = _setting(temperature, "temperature", logits, F32, 0, inf)
    p, p0 = _setting(top_p, "top_p", logits, F32, 0, 1)
    m, m0 = _setting(min_p, "min_p", logits, F32, 0, 1)
    k, k0 = _setting(top_k, "top_k", logits, torch.int32, 0, 2 ** 31 - 1)
    if B == 0:
        return torch.empty(0, dtype=torch.int64, device=logits.device)
    if not logits.is_cuda:
        return ref.sample_tokens(logits, uniform, t0 if t is None else t, k0 if k is None else k, p0 if p is None else p, m0 if m is None else m)
    from .kv8 import _On

    K, fn = _k()
    out = torch.empty(B, dtype=torch.int64, device=logits.device)
    a = _Sample(logits.data_ptr(), max(logits.stride(0), V), V, 0, uniform.data_ptr(), K._ptr(t), K._ptr(p), K._ptr(m), K._ptr(k), t0, p0, m0, int(k0),
                out.data_ptr())
    with _On(logits.device):
        K._check(fn(C.byref(a), B, logits.dtype == BF16, K._stream()), "sample")
    return out
