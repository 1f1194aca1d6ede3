"""Operators of an 8-bit key / value cache: CUDA tensors run the kernels of ``csrc/kv8.cu`` and ``csrc/kv8_attention.cu`` (long
prompts: ``csrc/latent_attention.cu`` behind a pass that turns codes into bf16), CPU tensors the plain statements of ``reference``.
A CUDA tensor never takes the plain path.

The cache holds e4m3 codes ``[B, kv_heads, capacity, dim]`` and one int8 exponent per head and block of tokens ``[B, kv_heads,
capacity / block]``; a value is ``code * 2**exponent``.  The exponent of a block is the least that brings its largest magnitude to
448 or less; it never falls below -40, so values below 2**-49 are stored as zero.  A position's block is begun when its
first position is written, so rows of an earlier sequence need no clearing; a sequence is written in order, and writing at a position
again forgets what lies behind it in the block.  Infinities are stored as the block's largest code, NaN as NaN.

Sequences are described by int32 tensors on the cache's device and never read by the host: positions outside the cache are left out by
the kernels (nothing is written) and recorded in the device status word (``cuda.check_device_status``), lengths are cut to the capacity.
Calls run on the current stream and allocate through PyTorch's allocator.  They belong to decoding: their results carry no
gradient, whatever requires one."""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

import torch

from . import reference as ref

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
BLOCKS = (16, 32, 64, 128)
# Bytes of bf16 keys, values and partial sums that a long prompt's attention may hold at a time (one key head of one sequence may take more).
# Smaller groups leave the machine idle at their ends: 32 sequences of 16384 keys, 8 key heads of 128, 128 tokens of 32 heads take 2054 us
# all at once, 2073 with 2 GiB, 2186 with 1 and 2559 with a quarter; of 500 keys in that capacity 236, 311, 403 and 542.
PROMPT_SCRATCH = 2 << 30


def streams(n: int, dim: int) -> bool:
    """Whether n query tokens per sequence are answered by streaming the codes, 32 rows (tokens x heads of a key head) at a time, and not from
    bf16 rows by the prompt attention, whose tiles are filled by the tokens of one head.  Microseconds of both ways at 8 sequences of 4096 keys
    and 8 key heads: dim 64, 4 heads per key head: 64 tokens 95 / 124, 128 tokens 176 / 126; dim 128, 1 head: 64 tokens 64 / 70, 128 tokens
    99 / 72; 16 heads: 32 tokens 281 / 446, 64 tokens 537 / 447.  They are equal at about 105 (94), 95 (75), 80 (64) and 62 (52) tokens
    for dims of 32, 64, 96 and 128 with 4 (16) heads per key head.  Neither batch nor length enters, so few tiles
    of long sequences are answered later than they could be: 1 sequence of 65536 keys, 16 key heads of 128, 1 head each: 64 tokens 160 / 357, 128 tokens
    280 / 355, 256 tokens 516 / 374."""
    return n <= 112 - dim // 2


class _Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "ke", "ve")] + [(n, C.c_longlong) for n in ("sb", "sh", "eb", "eh")] + \
               [(n, C.c_int) for n in ("B", "Hkv", "cap", "D", "log2_block")]


class _Attn(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "ke", "ve")] + [(n, C.c_longlong) for n in ("sb", "sh", "eb", "eh")] + \
               [(n, C.c_int) for n in ("B", "Hkv", "cap", "D", "log2_block")] + [("q", C.c_void_p)] + \
               [(n, C.c_longlong) for n in ("q_sb", "q_sn", "q_sh")] + [(n, C.c_void_p) for n in ("lens", "out", "part")] + \
               [(n, C.c_int) for n in ("n", "group", "rows", "tiles_r", "most")] + [("scale_log2", C.c_float), ("ctas", C.c_int), ("group_magic", C.c_uint32), ("whole", C.c_int)]


_fns = None


def _k():
    global _fns
    if _fns is None:
        from types import SimpleNamespace

        from . import cuda as K

        vp, i, ll = C.c_void_p, C.c_int, C.c_longlong
        _fns = SimpleNamespace(
            K=K, check=K._check, stream=K._stream,
            append=K._sig("b200_kv8_append", [C.POINTER(_Cache), vp, vp, C.POINTER(ll), vp, vp, i, vp, vp]),
            rope=K._sig("b200_kv8_rope_append", [C.POINTER(_Cache), vp, ll, i, i, vp, vp, vp, vp, vp, i, vp, vp]),
            decode=K._sig("b200_kv8_decode", [C.POINTER(_Cache), vp, vp, vp, i, i, vp, i, vp]),
            plan=K._sig("b200_kv8_attention_plan", [i] * 5 + [C.POINTER(i)]),
            attn=K._sig("b200_kv8_attention", [C.POINTER(_Attn)] + [vp] * 5),
            scratch=K._sig("b200_kv8_prompt_scratch", [i] * 6 + [ll]),
            prompt=K._sig("b200_kv8_prompt", [C.POINTER(_Cache)] + [vp] * 4 + [i] * 3 + [C.c_float, ll, vp, vp]),
        )
        _fns.scratch.restype = C.c_longlong
    return _fns


_device = torch._C._cuda_getDevice
_MOST_CALLS = 256       # remembered kinds of calls per cache


def _on(device: torch.device):
    """A guard that makes ``device`` the current one, or None where it is."""
    return None if device.index == _device() else torch.cuda.device(device)


def _guarded(device: torch.device, fn, *args):
    guard = _on(device)
    if guard is None:
        return fn(*args)
    with guard:
        return fn(*args)


@dataclass(eq=False)
class KV8Cache:
    """Codes and exponents of one layer's keys and values.  The tensors may be views (of a cache with more slots, say): a head's
    positions and channels have to be contiguous, codes and exponents of keys and values laid out alike."""

    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor

    def __post_init__(self):
        k, v, ke, ve = self.k, self.v, self.k_exp, self.v_exp
        if k.dim() != 4 or k.dtype != E4M3 or v.dtype != E4M3 or v.shape != k.shape:
            raise ValueError("codes are two float8_e4m3fn tensors [B, kv_heads, capacity, dim]")
        if ke.dim() != 3 or ke.dtype != torch.int8 or ve.dtype != torch.int8 or ve.shape != ke.shape or ke.shape[:2] != k.shape[:2]:
            raise ValueError("exponents are two int8 tensors [B, kv_heads, capacity / block]")
        if len({t.device for t in (k, v, ke, ve)}) != 1:
            raise ValueError("codes and exponents lie on one device")
        self.batch, self.kv_heads, self.capacity, self.dim = k.shape
        blocks = ke.shape[2]
        self.block = self.capacity // blocks if blocks else 0
        if self.block not in BLOCKS or self.block * blocks != self.capacity:
            raise ValueError(f"blocks of {BLOCKS} tokens: got {blocks} exponents for {self.capacity} positions")
        if self.dim % 32 or not 32 <= self.dim <= 128:
            raise ValueError(f"head dims of 32, 64, 96 and 128: got {self.dim}")
        if min(k.shape) == 0:
            raise ValueError("a cache has at least one sequence, head and position")
        if k.stride()[2:] != (self.dim, 1) or v.stride() != k.stride() or ke.stride(2) != 1 or ve.stride() != ke.stride():
            raise ValueError("a head's positions are contiguous, and keys and values laid out alike")
        if not (_apart(k, self.capacity * self.dim) and _apart(ke, blocks)):
            raise ValueError("heads do not overlap")
        if k.is_cuda and ((k.data_ptr() | v.data_ptr() | k.stride(0) | k.stride(1)) & 15):
            raise ValueError("heads start on 16-byte boundaries")
        self.device = k.device
        if k.is_cuda:
            _k().K.err_word(k.device)   # the status word is there before a call is captured
        self._calls: dict = {}          # what a kind of call (shapes, pitches, types, numbers) needs: checked once, then looked up
        self._c = _Cache(k.data_ptr(), v.data_ptr(), ke.data_ptr(), ve.data_ptr(), k.stride(0), k.stride(1), ke.stride(0), ke.stride(1),
                         *k.shape, self.block.bit_length() - 1)

    @classmethod
    def empty(cls, batch: int, kv_heads: int, capacity: int, dim: int, device=None, block: int = 32) -> "KV8Cache":
        """A cache for ``capacity`` positions (rounded up to whole blocks) per sequence."""
        if block not in BLOCKS:
            raise ValueError(f"blocks of {BLOCKS} tokens: got {block}")
        n = (capacity + block - 1) // block
        codes = [torch.zeros(batch, kv_heads, n * block, dim, dtype=torch.uint8, device=device).view(E4M3) for _ in range(2)]
        return cls(*codes, *(torch.full((batch, kv_heads, n), ref.KV8_EMIN, dtype=torch.int8, device=device) for _ in range(2)))

    def decoded(self, length: Optional[int] = None) -> tuple:
        """Keys and values of the first ``length`` positions (all by default) as bf16 [B, length, kv_heads, dim] (exact)."""
        n = self.capacity if length is None else int(length)
        if not 0 < n <= self.capacity:
            raise ValueError(f"length lies in 1 .. {self.capacity}")
        if not self.k.is_cuda:
            blocks = (n + self.block - 1) // self.block
            return tuple(ref.kv8_decode(c[:, :, :blocks * self.block], e[:, :, :blocks])[:, :, :n].transpose(1, 2).to(BF16, memory_format=torch.contiguous_format)
                         for c, e in ((self.k, self.k_exp), (self.v, self.v_exp)))
        k, v = (torch.empty(self.batch, n, self.kv_heads, self.dim, dtype=BF16, device=self.device) for _ in range(2))
        f = _k()
        _guarded(self.device, lambda: f.K._check(f.decode(C.byref(self._c), 0, k.data_ptr(), v.data_ptr(), n, n, 0, 0, f.K._stream()), "kv8_decode"))
        return k, v

    def _call(self, key: tuple, make, *args):
        call = self._calls.get(key)
        if call is None:
            if len(self._calls) >= _MOST_CALLS:
                self._calls.clear()
            call = self._calls[key] = make(self, *args)
        return call


def _apart(t: torch.Tensor, extent: int) -> bool:
    """Whether the heads [B, kv_heads] of ``extent`` elements each lie in places of their own."""
    for stride, n in sorted(zip(t.stride()[:2], t.shape[:2])):
        if n > 1:
            if stride < extent:
                return False
            extent = stride * (n - 1) + extent
    return True


def _index(t: torch.Tensor, cache: KV8Cache, what: str) -> None:
    if t.dtype != torch.int32 or t.shape != (cache.batch,) or t.device != cache.device or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 tensor [{cache.batch}] on the cache's device")


def _kind(t: torch.Tensor) -> tuple:
    return t.shape, t.stride(), t.dtype, t.device


def _pitch(x: torch.Tensor) -> list:
    """Strides of all but the last dimension; those of single entries do not matter."""
    return [0 if n == 1 else st for n, st in zip(x.shape[:-1], x.stride())]


def _aligned(x: torch.Tensor) -> bool:
    """Whether contiguous head vectors start on 16-byte boundaries, apart from the tensor's address."""
    return x.stride(-1) == 1 and not any(s & 7 for s in _pitch(x))


def _copy(x: torch.Tensor) -> torch.Tensor:
    return x.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------
def _append_call(cache, k, v, start, counts):
    if k.dim() != 4 or k.dtype != BF16 or v.dtype != BF16 or k.shape != v.shape or k.device != cache.device or v.device != cache.device:
        raise ValueError("keys and values are bf16 [B, n, kv_heads, dim] on the cache's device")
    B, n, H, D = k.shape
    if (B, H, D) != (cache.batch, cache.kv_heads, cache.dim):
        raise ValueError(f"keys {tuple(k.shape)} do not fit a cache of {cache.batch} sequences, {cache.kv_heads} heads of {cache.dim}")
    _index(start, cache, "start")
    if counts is not None:
        _index(counts, cache, "counts")
    if not cache.k.is_cuda or n == 0:
        return n, False, None, None, 0
    ok = _aligned(k) and _aligned(v)
    return n, ok, C.byref(cache._c), (C.c_longlong * 6)(*_pitch(k), *_pitch(v)) if ok else None, _k().K.err_word(cache.device).data_ptr()


def append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
    """Write keys and values [B, n, kv_heads, dim] (bf16, any pitches) of positions ``start[b] .. start[b] + n - 1`` into the cache;
    ``counts``: only the first ``counts[b]`` of a sequence's n."""
    n, ok, c, pitch, err = cache._call(("append", _kind(k), _kind(v), _kind(start), None if counts is None else _kind(counts)), _append_call, k, v, start,
                                    counts)
    if n == 0:
        return
    if err == 0:
        return ref.kv8_append(cache, k, v, start, counts)
    kp, vp = k.data_ptr(), v.data_ptr()
    if not ok or (kp | vp) & 15:
        return append(cache, _copy(k), _copy(v), start, counts)
    f, cp = _fns, 0 if counts is None else counts.data_ptr()
    if cache.device.index == _device():
        f.check(f.append(c, kp, vp, pitch, start.data_ptr(), cp, n, err, f.stream()), "kv8_append")
    else:
        with torch.cuda.device(cache.device):
            f.check(f.append(c, kp, vp, pitch, start.data_ptr(), cp, n, err, f.stream()), "kv8_append")


# ------------------------------------------------------------------------------------------
# rotate and append
# ------------------------------------------------------------------------------------------
def _rope_call(cache, qkv, cos, sin, pos, heads, bias, clear):
    B, D, Hkv = cache.batch, cache.dim, cache.kv_heads
    W = (heads + 2 * Hkv) * D
    if heads <= 0 or heads % Hkv:
        raise ValueError(f"{heads} query heads do not share {Hkv} key heads evenly")
    if qkv.dim() != 2 or tuple(qkv.shape) != (B, W) or qkv.dtype not in (BF16, F32) or qkv.device != cache.device or qkv.stride(1) != 1:
        raise ValueError(f"qkv is bf16 or fp32 [{B}, {W}] with contiguous rows on the cache's device")
    for t, what in ((cos, "cos"), (sin, "sin")):
        if t.dtype != F32 or t.dim() != 2 or t.shape[1] != D // 2 or t.shape[0] < cache.capacity or not t.is_contiguous() or t.device != cache.device:
            raise ValueError(f"{what} is a contiguous fp32 table [>= {cache.capacity}, {D // 2}] on the cache's device")
    if bias is not None and (bias.dtype != F32 or bias.numel() != (heads + Hkv) * D or not bias.is_contiguous() or bias.device != cache.device):
        raise ValueError(f"bias is a contiguous fp32 tensor of {(heads + Hkv) * D} values on the cache's device")
    if clear and (qkv.dtype != F32 or (B > 1 and qkv.stride(0) < W)):
        raise ValueError("only an fp32 accumulator whose rows do not overlap is handed back zeroed")
    _index(pos, cache, "pos")
    ld = 0 if B == 1 else qkv.stride(0)
    err = _k().K.err_word(cache.device).data_ptr() if cache.k.is_cuda else 0
    like = torch.empty(1, dtype=BF16, device=cache.device).expand(B, heads, D)        # a template of one element: an engine has many caches
    return like, C.byref(cache._c), ld, int(qkv.dtype == F32), not (ld * qkv.element_size() & 15), err


def rope_append(cache: KV8Cache, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor, heads: int,
                bias: Optional[torch.Tensor] = None, clear: bool = False) -> torch.Tensor:
    """The new token of every sequence: ``qkv`` [B, (heads + 2 kv_heads) dim] (bf16 or fp32) holds its packed projection.  Adds the fp32
    ``bias`` [(heads + kv_heads) dim] to q and k, turns their neighbouring pairs by the angles of position ``pos[b]`` (``cos`` / ``sin``: fp32
    [>= capacity, dim / 2]), writes k and v into the cache and returns q as bf16 [B, heads, dim].  Rows whose position lies outside the
    cache keep an undefined q.  ``clear`` hands an fp32 ``qkv`` back zeroed (the accumulator of a decode step's product)."""
    like, c, ld, f32, ok, err = cache._call(("rope", _kind(qkv), _kind(cos), _kind(sin), _kind(pos), heads, None if bias is None else _kind(bias), clear), _rope_call,
                                          qkv, cos, sin, pos, heads, bias, clear)
    if err == 0:
        return ref.kv8_rope_append(cache, qkv, cos, sin, pos, heads, bias, clear)
    x, cp, sp = qkv.data_ptr(), cos.data_ptr(), sin.data_ptr()
    if not ok or x & 15:
        if clear:
            raise ValueError("an accumulator that is cleared has rows on 16-byte boundaries")
        return rope_append(cache, _copy(qkv), cos, sin, pos, heads, bias)
    if (cp | sp) & 15:
        return rope_append(cache, qkv, cos.clone(), sin.clone(), pos, heads, bias, clear)
    f, q, bp = _fns, torch.empty_like(like, memory_format=torch.contiguous_format), 0 if bias is None else bias.data_ptr()
    if cache.device.index == _device():
        f.check(f.rope(c, x, ld, f32, clear, bp, cp, sp, pos.data_ptr(), q.data_ptr(), heads, err, f.stream()), "kv8_rope_append")
    else:
        with torch.cuda.device(cache.device):
            f.check(f.rope(c, x, ld, f32, clear, bp, cp, sp, pos.data_ptr(), q.data_ptr(), heads, err, f.stream()), "kv8_rope_append")
    return q


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
def _attention_call(cache, q, lens, scale, max_len):
    if q.dim() != 4 or q.dtype != BF16 or q.device != cache.device:
        raise ValueError("q is bf16 [B, n, heads, dim] on the cache's device")
    B, n, H, D = q.shape
    if (B, D) != (cache.batch, cache.dim) or H == 0 or H % cache.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {cache.batch} sequences, {cache.kv_heads} heads of {cache.dim}")
    _index(lens, cache, "lens")
    most = cache.capacity if max_len is None else int(max_len)
    if not 0 < most <= cache.capacity:
        raise ValueError(f"max_len lies in 1 .. {cache.capacity}")
    scale = D ** -0.5 if scale is None else float(scale)
    if n == 0:
        return lambda cache, q, lens: torch.empty_like(q)
    if not cache.k.is_cuda:
        return lambda cache, q, lens: ref.kv8_attention(q, cache, lens, scale, most)
    group = H // cache.kv_heads
    if not streams(n, D) and scale > 0:
        call = _prompt_call(cache, q, scale, most)
        if call is not None:
            return call
    ok = _aligned(q)
    f, c, device = _k(), cache._c, cache.device
    plan = (C.c_int * 5)()
    rc = _guarded(device, lambda: f.plan(B, cache.kv_heads, D, n * group, most, plan))
    if rc:
        raise RuntimeError(f"kv8_attention_plan failed with code {rc}")
    rows, tiles_r, ctas, scratch, whole = plan
    p = _Attn(c.k, c.v, c.ke, c.ve, c.sb, c.sh, c.eb, c.eh, B, c.Hkv, c.cap, D, c.log2_block, 0, *(_pitch(q) if ok else (0, 0, 0)), 0, 0, 0, n, group, rows,
              tiles_r, most, scale * 1.4426950408889634, ctas, 0, whole)
    ref_p, check, attn, stream, empty_like = C.byref(p), f.check, f.attn, f.stream, torch.empty_like
    out_like, part_like = (torch.empty(1, dtype=t, device=device).expand(n) for t, n in ((BF16, q.shape), (F32, (scratch,))))

    def run(cache, q, lens):            # holds no reference to the cache, which holds this
        qp = q.data_ptr()
        if not ok or qp & 15:
            return attention(_copy(q), cache, lens, scale, most)
        out, part = empty_like(out_like, memory_format=torch.contiguous_format), empty_like(part_like, memory_format=torch.contiguous_format)
        if device.index == _device():
            check(attn(ref_p, qp, lens.data_ptr(), out.data_ptr(), part.data_ptr(), stream()), "kv8_attention")
        else:
            with torch.cuda.device(device):
                check(attn(ref_p, qp, lens.data_ptr(), out.data_ptr(), part.data_ptr(), stream()), "kv8_attention")
        return out

    run.keep = p
    return run


def attention(q: torch.Tensor, cache: KV8Cache, lens: torch.Tensor, scale: Optional[float] = None, max_len: Optional[int] = None) -> torch.Tensor:
    """Causal attention of each sequence's n newest tokens: ``q`` [B, n, heads, dim] (bf16), the last one sees the first ``lens[b]`` positions
    of the cache, the one before it one fewer, and so on; one that sees nothing gets zeros.  Returns bf16 [B, n, heads, dim].
    Scores and sums are fp32; the weights enter their product with V in 11 bits where codes are streamed, in bf16's 8 where ``streams`` says no (long
    prompts: 0.0022 off the result in 64 bits, of which rounding the output is 0.0017).
    ``scale``: factor of the scores, dim ** -0.5 by default.  ``max_len``: no length is larger (longer ones are cut); the capacity by
    default.  A smaller bound makes short calls cheaper, and those of many tokens take scratch memory for as many keys, at most ``PROMPT_SCRATCH``
    bytes at a time."""
    if scale is not None:
        scale = float(scale)
    return cache._call((_kind(q), _kind(lens), scale, max_len), _attention_call, q, lens, scale, max_len)(cache, q, lens)


def _prompt_call(cache, q, scale, most):
    """Many query rows per key: the codes become bf16 rows once (exactly), and the prompt attention on the tensor cores reads those, a group of
    sequences and key heads at a time.  None: more tokens than that attention takes."""
    B, n, H, D = q.shape
    f, device, c, empty_like, limit = _k(), cache.device, C.byref(cache._c), torch.empty_like, PROMPT_SCRATCH
    nbytes = _guarded(device, lambda: f.scratch(B, cache.kv_heads, H, D, n, most, limit))
    if not nbytes:
        return None
    like, mem_like = (torch.empty(1, dtype=t, device=device).expand(s) for t, s in ((BF16, q.shape), (torch.uint8, (nbytes,))))
    err, contiguous, layout = f.K.err_word(device).data_ptr(), q.is_contiguous(), torch.contiguous_format

    def run(cache, q, lens):            # holds no reference to the cache, which holds this
        if not contiguous or q.data_ptr() & 15:
            q = _copy(q)
        out, mem = empty_like(like, memory_format=layout), empty_like(mem_like, memory_format=layout)
        if device.index == _device():
            f.check(f.prompt(c, q.data_ptr(), lens.data_ptr(), out.data_ptr(), mem.data_ptr(), H, n, most, scale, limit, err, f.stream()), "kv8_prompt")
        else:
            with torch.cuda.device(device):
                f.check(f.prompt(c, q.data_ptr(), lens.data_ptr(), out.data_ptr(), mem.data_ptr(), H, n, most, scale, limit, err, f.stream()), "kv8_prompt")
        return out

    return run
