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
    NaN counts as 0, one of 1 or more gives the last kept token that has a weight: what has less than 2^-44
    of the largest probability is never drawn).

    Kept is what all filters keep, as in ``models.sampling``: ``top_k`` (0: off) drops what is below the k-th largest logit, ``top_p`` (0 or
    1: off) keeps the longest prefix of the descending order (equal logits: lowest index first) whose probabilities sum to at most
    ``top_p`` and at least one token, ``min_p`` (0: off) drops what has less than ``min_p`` times the largest probability.  Every setting is a number
    or a tensor with one value per row (fp32, ``top_k`` int32).  A ``temperature`` of 0 picks the largest logit, the lowest index among
    equal ones; an infinite one weighs all logits alike that are not infinitely far below the largest.  NaN logits count as -inf; a row without any logit above -inf gives -1."""
    key = (logits.shape, logits.stride(), logits.dtype, logits.device, uniform.shape, uniform.stride(), uniform.dtype, uniform.device,
           *(_kind(x) for x in (temperature, top_k, top_p, min_p)))
    call = _calls.get(key)
    if call is None:
        if len(_calls) >= 256:
            _calls.clear()
        call = _calls[key] = _checked(logits, uniform, temperature, top_k, top_p, min_p)
    return call(logits, uniform, temperature, top_k, top_p, min_p)


_calls: dict = {}       # kinds of calls (shapes, pitches, types, numbers), checked once


def _kind(x):
    return (x.shape, x.stride(), x.dtype, x.device) if torch.is_tensor(x) else x


def _checked(logits, uniform, temperature, top_k, top_p, min_p):
    """Checks a kind of call and returns the function that makes it."""
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
    device = logits.device
    if B == 0:
        return lambda *a: torch.empty(0, dtype=torch.int64, device=device)
    if not logits.is_cuda:
        return lambda x, u, t, k, p, m: ref.sample_tokens(x, u, *(0 if a is None else a for a in (t, k, p, m)))
    K, fn = _k()
    ld, is_bf16, k0 = max(logits.stride(0), V), logits.dtype == BF16, int(k0)
    check, stream, current, byref = K._check, K._stream, torch._C._cuda_getDevice, C.byref
    like = torch.empty(B, dtype=torch.int64, device=device)
    ptr = lambda given, x: 0 if given is None else x.data_ptr()  # noqa: E731

    def run(x, u, temperature, top_k, top_p, min_p):
        out = torch.empty_like(like)
        a = _Sample(x.data_ptr(), ld, V, 0, u.data_ptr(), ptr(t, temperature), ptr(p, top_p), ptr(m, min_p), ptr(k, top_k), t0, p0, m0, k0, out.data_ptr())
        if device.index == current():
            check(fn(byref(a), B, is_bf16, stream()), "sample")
        else:
            with torch.cuda.device(device):
                check(fn(byref(a), B, is_bf16, stream()), "sample")
        return out

    return run
