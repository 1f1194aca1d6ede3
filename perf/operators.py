"""Cases of the operators of a decode step with an 8-bit key / value cache: writing keys and values into the cache, rotating and
writing one new token, attention over the cache, and drawing the next token from given random numbers.

The cache holds e4m3 codes ``[B, kv_heads, capacity, dim]`` and one power-of-two exponent (int8) per head and block of tokens
``[B, kv_heads, capacity / block]``: a value is ``code * 2**exponent``.  Since the exponents are powers of two, codes and
exponents together say the values exactly; updated caches are returned as those tensors.

``own`` false: the plain statement of each operator; true: this package's operators (``ops/kv8.py``, ``ops/sampling.py``).
"""
import math

import torch

own = False

E_MIN, E_MAX, CODE_MAX = -40, 119, 448.0
DEV = "cuda"


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # a prompt of 1024 tokens per sequence of the 55 x 96 model enters the cache after the prefill of one layer
        dict(name="append prompt", op="append", B=4, n=1024, Hkv=55, D=96, cap=1024, block=32, start=0, ragged=False),
        # portions of unequal length continue sequences in the middle of blocks, grouped heads
        dict(name="append ragged", op="append", B=13, n=77, Hkv=8, D=128, cap=1184, block=32, start=1003, ragged=True),
        # the new token of a single sequence, one layer: the smallest call, bound by its latency
        dict(name="rope append 1", op="rope", B=1, H=55, Hkv=55, D=96, cap=512, block=32, start=301, bias=True),
        # the new tokens of a full batch, one layer
        dict(name="rope append 64", op="rope", B=64, H=32, Hkv=8, D=128, cap=512, block=64, start=130, bias=False),
        # one token of a single sequence behind a short prompt: latency
        dict(name="attention 1 x 512", op="attention", B=1, n=1, H=55, Hkv=55, D=96, cap=1024, block=32, L=512, spread=0.0),
        # a serving batch of unequal lengths, as many key heads as query heads
        dict(name="attention 8 x 4096", op="attention", B=8, n=1, H=55, Hkv=55, D=96, cap=4096, block=32, L=4001, spread=0.5),
        # a long context and a few short ones in one batch, grouped heads
        dict(name="attention 3 x 65536", op="attention", B=3, n=1, H=32, Hkv=8, D=128, cap=65536, block=64, L=65501, spread=0.98),
        # five drafted tokens per sequence are checked at once
        dict(name="attention drafts", op="attention", B=16, n=5, H=32, Hkv=8, D=64, cap=8192, block=32, L=6007, spread=0.7),
        # a prompt goes on behind what the cache holds
        dict(name="attention prompt", op="attention", B=1, n=1500, H=32, Hkv=8, D=128, cap=8192, block=32, L=7777, spread=0.0),
        # the next token of a single sequence: latency
        dict(name="sample 1", op="sample", B=1, V=65536, dtype="float32", t=0.8, k=0, p=0.95, m=0.0, mixed=False),
        # a full batch whose rows have settings of their own
        dict(name="sample 64", op="sample", B=64, V=65536, dtype="float32", t=0.7, k=50, p=0.9, m=0.02, mixed=True),
        # 16-bit logits, many of them equal, an odd vocabulary
        dict(name="sample bf16", op="sample", B=24, V=32003, dtype="bfloat16", t=1.0, k=0, p=0.8, m=0.0, mixed=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "rope", "attention", "attention", "sample", "sample"])
    if op == "sample":
        V = _log(rng, 1000, 131072)
        B = _log(rng, 1, max(1, min(96, (64 * 65536) // V)))
        return dict(op=op, B=B, V=V, dtype=rng.choice(["float32", "bfloat16"]), t=rng.choice([0.3, 0.7, 1.0, 1.5]),
                    k=rng.choice([0, 0, 1, 40, 500]), p=rng.choice([1.0, 0.95, 0.7, 0.2]), m=rng.choice([0.0, 0.0, 0.01, 0.2]),
                    mixed=rng.random() < 0.5)
    D, block = rng.choice([32, 64, 96, 128]), rng.choice([16, 32, 64, 128])
    group, Hkv = rng.choice([(1, 55), (1, 16), (2, 12), (4, 8), (5, 3), (8, 4), (16, 1)])
    if op == "rope":
        cap = block * rng.randint(1, 8)
        return dict(op=op, B=_log(rng, 1, 64), H=group * Hkv, Hkv=Hkv, D=D, cap=cap, block=block, start=rng.randint(0, cap - 1),
                    bias=rng.random() < 0.5)
    if op == "append":
        B, n = _log(rng, 1, 16), _log(rng, 1, 1200)
        n = max(1, min(n, (4 * 1024 * 55 * 96) // (B * Hkv * D)))
        start = rng.choice([0, rng.randint(0, 600)])
        return dict(op=op, B=B, n=n, Hkv=Hkv, D=D, cap=(start + n + block - 1) // block * block, block=block, start=start,
                    ragged=rng.random() < 0.5)
    most_keys, most_scores = 3 * 65536 * 8 * 128, 1500 * 32 * 8192
    L, B = _log(rng, 1, 65536), _log(rng, 1, 64)
    n = rng.choice([1, 1, 1, 2, 3, 7, _log(rng, 8, 1024)])
    L = min(L, most_keys // (Hkv * D) - 512)
    cap = (L + rng.randint(0, 300) + block - 1) // block * block
    B = max(1, min(B, most_keys // (cap * Hkv * D)))
    n = max(1, min(n, most_scores // (cap * group * Hkv)))
    B = max(1, min(B, most_scores // (cap * group * Hkv * n)))
    return dict(op=op, B=B, n=n, H=group * Hkv, Hkv=Hkv, D=D, cap=cap, block=block, L=L, spread=rng.choice([0.0, 0.5, 1.0]))


def _lens(c):
    """Visible keys of each sequence's last query: from L down to L (1 - spread), in a mixed order."""
    return [int(round(c["L"] * (1 - c["spread"] * ((b * 5) % c["B"]) / max(1, c["B"] - 1)))) for b in range(c["B"])]


def _counts(c):
    return [c["n"] - (b * 7) % c["n"] if c["ragged"] else c["n"] for b in range(c["B"])]


def work(c):
    if c["op"] == "append":
        t = sum(_counts(c)) * c["Hkv"] * c["D"]
        return dict(bytes=2 * t * (2 + 1), flops=6 * t)
    if c["op"] == "rope":
        q, kv = c["B"] * c["H"] * c["D"], 2 * c["B"] * c["Hkv"] * c["D"]
        return dict(bytes=2 * (q + kv) + 2 * q + kv + 4 * c["D"] * c["B"], flops=6 * (q + kv))
    if c["op"] == "attention":
        lens, n = _lens(c), c["n"]
        seen = sum(sum(max(0, x - i) for i in range(n)) for x in lens)
        return dict(bytes=2 * sum(lens) * c["Hkv"] * (c["D"] + 1 / c["block"]) + 4 * c["B"] * n * c["H"] * c["D"], flops=4 * c["H"] * c["D"] * seen)
    return dict(bytes=c["B"] * c["V"] * (4 if c["dtype"] == "float32" else 2), flops=8 * c["B"] * c["V"])


# ------------------------------------------------------------------------------------------
# the cache in its plain form
# ------------------------------------------------------------------------------------------
def _pow2(e):
    """2**e in fp32, exactly, for whole e in -126 .. 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The least exponent that brings amax to at most the largest code."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > CODE_MAX / 512).int()
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _encode(x, e):
    """fp32 values -> codes under the exponents e (broadcast), to nearest, at most the largest code."""
    return (x * _pow2(-e)).clamp(-CODE_MAX, CODE_MAX).to(torch.float8_e4m3fn)


def _finite_amax(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dims)


def _decode(codes, exps, block):
    """fp32 values of codes [..., T, D] with exponents [..., T / block]."""
    return codes.float() * _pow2(exps).repeat_interleave(block, -1)[..., None]


def _write(codes, exps, x, start, counts, block):
    """Positions start[b] .. start[b] + counts[b] - 1 become x [B, n, Hkv, D] (fp32).  A block that is begun takes the exponent of its
    new tokens; one that goes on keeps the larger exponent, and what it holds in front of them is encoded again."""
    B, Hkv, cap, D = codes.shape
    n = x.shape[1]
    nb = min((n + block - 2) // block + 1, cap // block)
    first = torch.minimum(start // block, torch.tensor(cap // block - nb, device=start.device))
    blocks = first[:, None] + torch.arange(nb, device=start.device)                             # [B, nb]
    pos = blocks[:, :, None] * block + torch.arange(block, device=start.device)                 # [B, nb, block]
    flat = pos.reshape(B, nb * block)
    off = flat - start[:, None]
    new = (off >= 0) & (off < counts[:, None])
    xn = x.gather(1, off.clamp(0, n - 1)[:, :, None, None].expand(B, nb * block, Hkv, D)).permute(0, 2, 1, 3)
    at = flat[:, None, :, None].expand(B, Hkv, nb * block, D)
    old = codes.view(torch.uint8).gather(2, at)
    be = blocks[:, None, :].expand(B, Hkv, nb)
    old_e = exps.gather(2, be).int()
    touched = new.view(B, nb, block).any(-1)[:, None, :]
    fresh = (blocks * block >= start[:, None])[:, None, :]
    xv = torch.where(new[:, None, :, None], xn, 0.0)
    e_new = _exponent(_finite_amax(xv.view(B, Hkv, nb, block, D), (-1, -2)))
    e = torch.where(fresh, e_new, torch.maximum(e_new, old_e))
    e = torch.where(touched, e, old_e)
    et = e.repeat_interleave(block, -1)[..., None]
    kept = old.view(torch.float8_e4m3fn).float() * _pow2(old_e).repeat_interleave(block, -1)[..., None]
    vals = torch.where(new[:, None, :, None], xv, kept)
    moved = new[:, None, :, None] | ((off < 0)[:, None, :, None] & touched.repeat_interleave(block, -1)[..., None])
    got = torch.where(moved, _encode(vals, et).view(torch.uint8), old)
    codes.view(torch.uint8).scatter_(2, at, got)
    exps.scatter_(2, be, e.to(torch.int8))


def _rotate(x, cos, sin):
    """Neighbouring pairs (x[2i], x[2i + 1]) turned by the angles of their position: x [B, heads, D], tables [B, D / 2]."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None], sin[:, None]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _keys(g, B, Hkv, T, D):
    """Keys or values as a model makes them: heads and channels of unequal size, a first token that stands out."""
    head = torch.exp(0.5 * torch.randn(Hkv, 1, 1, device=DEV, generator=g))
    chan = torch.exp(0.4 * torch.randn(Hkv, 1, D, device=DEV, generator=g))
    return torch.randn(B, Hkv, T, D, device=DEV, generator=g) * head * chan


def _filled(g, c):
    """A cache whose positions are all written."""
    k, v = (_keys(g, c["B"], c["Hkv"], c["cap"], c["D"]) for _ in range(2))
    out = {}
    for name, x in (("k", k), ("v", v)):
        e = _exponent(x.view(c["B"], c["Hkv"], -1, c["block"], c["D"]).abs().amax((-1, -2)))
        out[name] = _encode(x, e.repeat_interleave(c["block"], -1)[..., None])
        out[name + "_exp"] = e.to(torch.int8)
    return out


def prepare(c, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(c)
    if c["op"] == "sample":
        x = 2.5 * torch.randn(c["B"], c["V"], device=DEV, generator=g)
        x[:, : max(1, c["V"] // 100)] += 3.0
        x = x[:, torch.randperm(c["V"], device=DEV, generator=g)]
        s["logits"] = x.to(getattr(torch, c["dtype"]))
        s["uniform"] = torch.rand(c["B"], device=DEV, generator=g)
        if c["mixed"]:      # rows of a batch ask for different things, some for nothing
            r = torch.arange(c["B"], device=DEV)
            s["t"] = torch.where(r % 7 == 6, 0.0, c["t"] + 0.1 * (r % 5))
            s["k"] = torch.where(r % 3 == 0, c["k"], 0).int()
            s["p"] = torch.where(r % 4 < 2, c["p"], 1.0)
            s["m"] = torch.where(r % 5 == 0, c["m"], 0.0)
        return s
    s.update(_filled(g, c))
    if c["op"] == "attention":
        s["q"] = torch.randn(c["B"], c["n"], c["H"], c["D"], device=DEV, generator=g).to(torch.bfloat16)
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
        return s
    s["start"] = torch.full((c["B"],), c["start"], dtype=torch.int32, device=DEV)
    if c["op"] == "append":
        # views of one packed projection, as the model hands them over
        kv = torch.cat([_keys(g, c["B"], c["Hkv"], c["n"], c["D"]).transpose(1, 2) for _ in range(2)], 2).to(torch.bfloat16)
        s["k_new"], s["v_new"] = kv[:, :, : c["Hkv"]], kv[:, :, c["Hkv"]:]
        s["counts"] = torch.tensor(_counts(c), dtype=torch.int32, device=DEV)
        return s
    W = (c["H"] + 2 * c["Hkv"]) * c["D"]
    s["qkv"] = torch.randn(c["B"], W, device=DEV, generator=g).to(torch.bfloat16)
    s["bias"] = 0.3 * torch.randn((c["H"] + c["Hkv"]) * c["D"], device=DEV, generator=g) if c["bias"] else None
    f = 50000.0 ** (-torch.arange(0, c["D"], 2, device=DEV, dtype=torch.float64) / c["D"])
    angle = torch.arange(c["cap"], device=DEV, dtype=torch.float64)[:, None] * f
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def _handle(s):
    """The cache object that a program keeps for its tensors."""
    if "cache" not in s:
        from recurrent_pretraining_b200.ops.kv8 import KV8Cache

        s["cache"] = KV8Cache(s["k"], s["v"], s["k_exp"], s["v_exp"])
    return s["cache"]


def run(s):
    if s["op"] == "sample":
        return _sample(s)
    if s["op"] == "attention":
        return _attention(s)
    if s["op"] == "append":
        if own:
            from recurrent_pretraining_b200.ops import kv8

            kv8.append(_handle(s), s["k_new"], s["v_new"], s["start"], s["counts"])
        else:
            for x, name in ((s["k_new"], "k"), (s["v_new"], "v")):
                _write(s[name], s[name + "_exp"], x.float(), s["start"].long(), s["counts"].long(), s["block"])
        return s["k"], s["v"], s["k_exp"], s["v_exp"]
    return _rope(s)


def _rope(s):
    if own:
        from recurrent_pretraining_b200.ops import kv8

        q = kv8.rope_append(_handle(s), s["qkv"], s["cos"], s["sin"], s["start"], s["H"], bias=s["bias"])
        return q, s["k"], s["v"], s["k_exp"], s["v_exp"]
    B, H, Hkv, D = s["B"], s["H"], s["Hkv"], s["D"]
    x = s["qkv"].float()
    qk = x[:, : (H + Hkv) * D]
    if s["bias"] is not None:
        qk = qk + s["bias"]
    pos = s["start"].long()
    qk = _rotate(qk.view(B, H + Hkv, D), s["cos"][pos], s["sin"][pos])
    one = torch.ones_like(pos)
    _write(s["k"], s["k_exp"], qk[:, None, H:], pos, one, s["block"])
    _write(s["v"], s["v_exp"], x[:, (H + Hkv) * D:].view(B, 1, Hkv, D), pos, one, s["block"])
    return qk[:, :H].to(torch.bfloat16), s["k"], s["v"], s["k_exp"], s["v_exp"]


def _attention(s):
    if own:
        from recurrent_pretraining_b200.ops import kv8

        return kv8.attention(s["q"], _handle(s), s["lens"])
    B, n, H, D = s["q"].shape
    Hkv, cap = s["Hkv"], s["cap"]
    G = H // Hkv
    lens = s["lens"].long()
    key = torch.arange(cap, device=lens.device)
    held = key < lens[:, None]                                                                   # [B, cap]
    k, v = (torch.where(held[:, None, :, None], _decode(s[x], s[x + "_exp"], s["block"]), 0.0) for x in ("k", "v"))
    q = s["q"].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    sc = (torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5).view(B, Hkv, G, n, cap)
    limit = lens[:, None] - (n - 1) + torch.arange(n, device=lens.device)                        # keys that query i sees
    seen = (key < limit[:, :, None])[:, None, None]
    sc = torch.where(seen, sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    w = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)                                             # a query without keys: zeros
    o = torch.matmul(w.view(B, Hkv, G * n, cap), v).view(B, Hkv, G, n, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(torch.bfloat16)


def _sample(s):
    t, k, p, m = s["t"], s["k"], s["p"], s["m"]
    if own:
        from recurrent_pretraining_b200.ops.sampling import sample_tokens

        return sample_tokens(s["logits"], s["uniform"], temperature=t, top_k=k, top_p=p, min_p=m)
    x = s["logits"].double()
    B, V = x.shape
    row = lambda a: (a.double() if torch.is_tensor(a) else torch.full((B,), float(a), dtype=torch.float32, device=x.device).double())[:, None]  # noqa: E731
    t, k, p, m = row(t), row(k), row(p), row(m)
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)                              # equal ones: lowest index first
    w = torch.exp((xs - xs[:, :1]) / torch.where(t > 0, t, 1.0))
    kth = xs.gather(1, (torch.where(k > 0, k, V).clamp(1, V) - 1).long())
    keep = xs >= kth                                                                             # ties with the k-th stay
    total = w.sum(-1, keepdim=True)
    inside = w.cumsum(-1) <= p * total
    inside[:, 0] = True
    keep &= inside | (p >= 1) | (p <= 0)
    keep &= (w >= m) | (m <= 0)
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w).cumsum(-1)                                     # in the vocabulary's order
    target = s["uniform"].double()[:, None] * w[:, -1:]
    got = (w <= target).sum(-1).clamp_max(V - 1)
    return torch.where(t[:, 0] > 0, got, order[:, 0])


# ------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------
def exact(c, seed):
    if c["op"] == "sample":
        return None                 # whole numbers
    s = prepare(c, seed)
    if c["op"] == "attention":
        B, n, H, Hkv, D = c["B"], c["n"], c["H"], c["Hkv"], c["D"]
        out = torch.zeros(B, n, H, D, dtype=torch.float64, device=DEV)
        for b, length in enumerate(_lens(c)):
            if length <= 0:
                continue
            ex = torch.arange(length, device=DEV) // c["block"]
            lim = torch.arange(length - n + 1, length + 1, device=DEV)
            hide = torch.arange(length, device=DEV)[None] >= lim[:, None]
            for h in range(H):
                kv = h // (H // Hkv)
                K = s["k"][b, kv, :length].double() * torch.exp2(s["k_exp"][b, kv, ex].double())[:, None]
                V = s["v"][b, kv, :length].double() * torch.exp2(s["v_exp"][b, kv, ex].double())[:, None]
                a = (s["q"][b, :, h].double() @ K.T / math.sqrt(D)).masked_fill(hide, -math.inf)
                a = torch.softmax(a, -1)
                a[lim <= 0] = 0
                out[b, :, h] = a @ V
        return out
    # a cache in 64 bits: the values that the codes would stand for without rounding, in units of their blocks
    k, v = s["k"].double(), s["v"].double()
    q = None
    if c["op"] == "append":
        new = {"k": s["k_new"].double(), "v": s["v_new"].double()}
        counts = _counts(c)
    else:
        H, Hkv, D = c["H"], c["Hkv"], c["D"]
        x = s["qkv"].double().view(c["B"], H + 2 * Hkv, D)
        y = x.clone()
        if s["bias"] is not None:
            y[:, : H + Hkv] += s["bias"].double().view(H + Hkv, D)
        z = torch.complex(y[..., ::2].contiguous(), y[..., 1::2].contiguous())
        z = z * torch.complex(s["cos"][c["start"]].double(), s["sin"][c["start"]].double())
        y = torch.view_as_real(z).flatten(-2)
        q = y[:, :H]
        new = {"k": y[:, None, H:H + Hkv], "v": x[:, None, H + Hkv:]}
        counts = [1] * c["B"]
    blk = c["block"]
    for name, codes in (("k", k), ("v", v)):
        exps = s[name + "_exp"].double()
        for b, cnt in enumerate(counts):
            at, end = c["start"], c["start"] + cnt
            for i in range(at // blk, (end - 1) // blk + 1):
                lo, hi = max(at, i * blk), min(end, (i + 1) * blk)
                x = new[name][b, lo - at:hi - at].transpose(0, 1)                                # [Hkv, tokens, D]
                e = torch.ceil(torch.log2(x.abs().amax((1, 2)) / CODE_MAX) - 1e-12).clamp(E_MIN, E_MAX)   # a whole power stays one
                if lo > i * blk:
                    was = exps[b, :, i]
                    e = torch.maximum(e, was)
                    codes[b, :, i * blk:lo] *= torch.exp2(was - e)[:, None, None]
                codes[b, :, lo:hi] = x * torch.exp2(-e)[:, None, None]
    return (k, v, None, None) if q is None else (q, k, v, None, None)
