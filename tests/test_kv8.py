"""The 8-bit key / value cache (``ops/kv8.py``) against statements in 64 bits: the same tests on CPU tensors (plain path) and on the GPU
(kernels).  Codes and exponents of given bf16 values are exact; tolerances of the rest are sums of the roundings on the way."""
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from recurrent_pretraining_b200.ops import kv8
from recurrent_pretraining_b200.ops.kv8 import KV8Cache

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16_HALF, F16_HALF = 2.0 ** -8, 2.0 ** -11       # half a step, relative


# ------------------------------------------------------------------------------------------
# oracle
# ------------------------------------------------------------------------------------------
def e4m3_round(x):
    """fp64 -> nearest e4m3 value, ties to even, at most 448; NaN stays."""
    a = x.abs().clamp(max=448.0)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
    return torch.copysign(torch.clamp(torch.round(a / step) * step, max=448.0), x)


def least_exponent(amax):
    e = -40
    while amax > 448.0 * 2.0 ** e and e < 119:
        e += 1
    return e


def oracle_write(state, x, start, block):
    """state: {"val": fp64 values [H, cap, D], "exp": [H][blocks]} of one sequence; x [n, H, D] fp64."""
    val, exp = state["val"], state["exp"]
    for h in range(val.shape[0]):
        for i in range(start // block, (start + x.shape[0] - 1) // block + 1):
            lo, hi = max(start, i * block), min(start + x.shape[0], (i + 1) * block)
            new = x[lo - start:hi - start, h]
            fin = new[torch.isfinite(new)].abs()
            e = least_exponent(float(fin.max()) if fin.numel() else 0.0)
            if lo > i * block:
                e = max(e, exp[h][i])
                val[h, i * block:lo] = e4m3_round(val[h, i * block:lo] * 2.0 ** -e) * 2.0 ** e
            val[h, lo:hi] = e4m3_round(new * 2.0 ** -e) * 2.0 ** e
            exp[h][i] = e


def values(cache, which="k"):
    c, e = (cache.k, cache.k_exp) if which == "k" else (cache.v, cache.v_exp)
    return c.double().cpu() * torch.exp2(e.double().cpu()).repeat_interleave(cache.block, -1)[..., None]


def states(cache, which):
    val, exp = values(cache, which), (cache.k_exp if which == "k" else cache.v_exp).tolist()
    return [{"val": val[b].clone(), "exp": [list(r) for r in exp[b]]} for b in range(cache.batch)]


def check(cache, which, want, upto):
    got = values(cache, which)
    exps = (cache.k_exp if which == "k" else cache.v_exp).tolist()
    for b, st in enumerate(want):
        n = upto[b]
        assert torch.equal(torch.nan_to_num(got[b, :, :n], nan=1e30), torch.nan_to_num(st["val"][:, :n], nan=1e30))
        blocks = (n + cache.block - 1) // cache.block
        assert [r[:blocks] for r in exps[b]] == [r[:blocks] for r in st["exp"]]


def attend(q, k, v, lens, scale):
    """q [B, n, H, D], k / v [B, Hkv, L, D] in fp64 -> outputs, sum of |w v| and largest sum |q k| scale per row."""
    B, n, H, D = q.shape
    group = H // k.shape[1]
    out, mag, big = (torch.zeros(B, n, H, D, dtype=torch.float64), torch.zeros(B, n, H, D, dtype=torch.float64),
                     torch.zeros(B, n, H, 1, dtype=torch.float64))
    for b in range(B):
        for i in range(n):
            m = min(max(int(lens[b]), 0), k.shape[2]) - (n - 1 - i)
            for h in range(H):
                if m <= 0:
                    continue
                K, V = k[b, h // group, :m], v[b, h // group, :m]
                w = torch.softmax(K @ q[b, i, h] * scale, 0)
                out[b, i, h], mag[b, i, h] = w @ V, w @ V.abs()
                big[b, i, h] = (K.abs() @ q[b, i, h].abs()).max() * abs(scale)
    return out, mag, big


def tolerance(out, mag, big, D, weight_half):
    """Output rounding + rounding of the weights + scores (fp32 sums of D products, twice the error in the exponent for numerator and
    denominator) + exp2 and the division."""
    return BF16_HALF * out.abs() + (weight_half + 2 * (D + 4) * 2.0 ** -23 * big + 2.0 ** -18) * mag + 1e-30


def filled(B, Hkv, cap, D, block, device, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    cache = KV8Cache.empty(B, Hkv, cap, D, device, block)
    k, v = (torch.randn(B, cache.capacity, Hkv, D, generator=g).mul(scale).to(torch.bfloat16).to(device) for _ in range(2))
    kv8.append(cache, k, v, torch.zeros(B, dtype=torch.int32, device=device))
    return cache


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("block,D,Hkv,cap,steps", [
    (32, 96, 5, 128, [(0, 70), (70, 1), (71, 30), (101, 27)]),       # a prompt, tokens, a portion that ends with the cache
    (16, 32, 3, 48, [(0, 1), (1, 1), (2, 1), (3, 13), (16, 32)]),
    (128, 128, 2, 256, [(5, 200), (205, 51)]),                       # begins inside a block
    (64, 64, 1, 64, [(0, 64), (10, 3), (13, 51)]),                   # goes back and on from there
    (32, 64, 4, 96, [(33, 1), (34, 62)]),
])
def test_append_matches_its_definition_bit_for_bit(device, block, D, Hkv, cap, steps):
    B = 3
    g = torch.Generator().manual_seed(1)
    cache = KV8Cache.empty(B, Hkv, cap, D, device, block)
    for t in (cache.k, cache.v):             # what lay there before does not matter where a block is begun
        t.view(torch.uint8).random_(0, 127)
    want = {w: states(cache, w) for w in "kv"}
    for step, (start, n) in enumerate(steps):
        size = 2.0 ** (3 * step - 4)         # growing values: blocks that go on are encoded again
        kv = torch.randn(B, n, 2 * Hkv, D, generator=g) * size
        kv[1] *= 1e-3
        kv = kv.to(torch.bfloat16)
        d = kv.to(device)
        kv8.append(cache, d[:, :, :Hkv], d[:, :, Hkv:], i32([start] * B, device))
        for w, x in (("k", kv[:, :, :Hkv]), ("v", kv[:, :, Hkv:])):
            for b in range(B):
                oracle_write(want[w][b], x[b].double(), start, block)
            check(cache, w, want[w], [start + n] * B)


@pytest.mark.parametrize("device", DEVICES)
def test_append_ragged_counts_leave_everything_else_alone(device):
    B, Hkv, D, block, n = 4, 2, 64, 16, 40
    cache = filled(B, Hkv, 96, D, block, device)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
    want = states(cache, "k")
    k = torch.randn(B, n, Hkv, D).to(torch.bfloat16).to(device) * 4
    start, counts = [3, 0, 56, 17], [40, 0, 40, 1]
    kv8.append(cache, k, k, i32(start, device), i32(counts, device))
    for b in range(B):
        if counts[b]:
            oracle_write(want[b], k[b, :counts[b]].double().cpu(), start[b], block)
    check(cache, "k", want, [s + c for s, c in zip(start, counts)])
    for now, old in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8)), (before[0].view(torch.uint8), before[1].view(torch.uint8))):
        for b in range(B):
            end = start[b] + counts[b]
            assert torch.equal(now[b, :, end:], old[b, :, end:])
            assert torch.equal(now[b, :, :start[b] // block * block], old[b, :, :start[b] // block * block])


@pytest.mark.parametrize("device", DEVICES)
def test_append_again_changes_nothing(device):
    cache = filled(2, 3, 64, 32, 32, device)
    k, v = (torch.randn(2, 9, 3, 32, generator=torch.Generator().manual_seed(s)).mul(7).to(torch.bfloat16).to(device) for s in (3, 4))
    kv8.append(cache, k, v, i32([20, 27], device))
    first = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
    kv8.append(cache, k, v, i32([20, 27], device))
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(first, (cache.k, cache.v, cache.k_exp, cache.v_exp)))


@pytest.mark.parametrize("device", DEVICES)
def test_append_of_extreme_values(device):
    """Zeros, NaN, infinities, the largest and the smallest bf16 values, magnitudes at the border of an exponent."""
    D, block = 32, 16
    big, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    rows = [[0.0], [float("nan"), 1.0], [float("inf"), 3.0, -float("inf")], [big, -big / 2, 1.0], [tiny], [448.0, 1.0], [450.0, 1.0], [447.0], [2.0 ** -49, 2.0 ** -31],
            [float("nan")], [-0.0, 7.0]]
    cache = KV8Cache.empty(1, 1, block * len(rows), D, device, block)
    x = torch.zeros(1, block * len(rows), 1, D)
    for i, r in enumerate(rows):
        x[0, i * block, 0, :len(r)] = torch.tensor(r)
    x = x.to(torch.bfloat16)
    want = states(cache, "k")
    oracle_write(want[0], x[0].double(), 0, block)
    kv8.append(cache, x.to(device), x.to(device), i32([0], device))
    check(cache, "k", want, [cache.capacity])
    check(cache, "v", want, [cache.capacity])


@pytest.mark.parametrize("device", DEVICES)
def test_sequences_that_do_not_fit_are_left_out(device):
    cache = filled(5, 2, 64, 32, 32, device)
    old = [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
    k = torch.ones(5, 8, 2, 32, dtype=torch.bfloat16, device=device)
    kv8.append(cache, k, k, i32([-1, 57, 2 ** 31 - 1, 64, 0], device), i32([8, 8, 8, 1, 9], device))
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(old, (cache.k, cache.v, cache.k_exp, cache.v_exp)))
    kv8.rope_append(cache, torch.ones(5, 6 * 32, dtype=torch.bfloat16, device=device), *tables(64, 32, device), i32([-1, 64, 2 ** 31 - 1, -2 ** 31, 65], device), 2)
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(old, (cache.k, cache.v, cache.k_exp, cache.v_exp)))
    if device == "cuda":
        from recurrent_pretraining_b200.ops import cuda as K

        assert K.check_device_status() == 8 and K.check_device_status() == 0
    out = kv8.attention(torch.ones(5, 1, 2, 32, dtype=torch.bfloat16, device=device), cache, i32([64, 65, 2 ** 31 - 1, -5, 0], device))
    assert torch.equal(out[0].cpu(), kv8.attention(torch.ones(5, 1, 2, 32, dtype=torch.bfloat16, device=device), cache, i32([64] * 5, device))[0].cpu())
    assert out[1].isfinite().all() and out[2].isfinite().all() and not out[3:].any()


# ------------------------------------------------------------------------------------------
# rotate and append
# ------------------------------------------------------------------------------------------
def tables(length, D, device):
    a = torch.arange(length, dtype=torch.float64)[:, None] * 50000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return a.cos().float().to(device), a.sin().float().to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hkv,D,block,bias", [(1, 5, 5, 96, 32, True), (7, 8, 2, 64, 16, False), (3, 6, 3, 128, 128, True), (33, 4, 1, 32, 64, True)])
def test_rope_append(device, dtype, B, H, Hkv, D, block, bias):
    g = torch.Generator().manual_seed(5)
    cache = filled(B, Hkv, 2 * block, D, block, device)
    want = {w: states(cache, w) for w in "kv"}
    pos = [(block - 2 + 3 * b) % cache.capacity for b in range(B)]
    pos[0] = block                                                    # a block is begun
    cos, sin = tables(cache.capacity, D, device)
    qkv = (torch.randn(B, (H + 2 * Hkv) * D, generator=g) * torch.exp(torch.randn(B, 1, generator=g))).to(dtype)
    bvec = torch.randn((H + Hkv) * D, generator=g) if bias else None
    dev = torch.zeros(B, qkv.shape[1] + 8, dtype=dtype, device=device)[:, :qkv.shape[1]]       # rows with a pitch of their own
    dev.copy_(qkv)
    q = kv8.rope_append(cache, dev, cos, sin, i32(pos, device), H, bias=None if bvec is None else bvec.to(device))
    x = qkv.double().view(B, H + 2 * Hkv, D)
    qk = x[:, :H + Hkv] + (bvec.double().view(H + Hkv, D) if bias else 0.0)
    c, s = cos.double().cpu()[pos][:, None], sin.double().cpu()[pos][:, None]
    a, b2 = qk[..., ::2], qk[..., 1::2]
    rot = torch.stack([a * c - b2 * s, a * s + b2 * c], -1).flatten(2)
    noise = 4 * 2.0 ** -24 * (qk.abs().unflatten(-1, (-1, 2)).sum(-1).repeat_interleave(2, -1) + 1e-30)     # sum, two products, sum in fp32
    assert ((q.double().cpu() - rot[:, :H]).abs() <= BF16_HALF * rot[:, :H].abs() + 2 * noise[:, :H]).all()
    for w, new, eps in (("k", rot[:, H:], noise[:, H:]), ("v", x[:, H + Hkv:], torch.zeros(1))):
        got, exps = values(cache, w), (cache.k_exp if w == "k" else cache.v_exp).cpu()
        for b in range(B):
            p0 = pos[b] // block * block
            e = exps[b, :, pos[b] // block].double()[:, None]
            amax = new[b].abs().amax(-1, keepdim=True)
            old = torch.tensor([h[pos[b] // block] for h in want[w][b]["exp"]], dtype=torch.float64)[:, None] if pos[b] > p0 else torch.full((Hkv, 1), -40.0, dtype=torch.float64)
            slack = 1 + 2.0 ** -20                                    # the fp32 value may lie just across a border
            assert (amax <= 448 * torch.exp2(e) * slack).all() and ((e == old) | (amax * slack > 448 * torch.exp2(e - 1))).all() and (e >= old).all()
            err = (got[b, :, pos[b]] - new[b]).abs()
            assert (err <= 2.0 ** -4 * new[b].abs() + 2.0 ** -10 * torch.exp2(e) + 2 * (eps[b] if eps.numel() > 1 else 0)).all()
            if pos[b] > p0:                                           # older tokens of the block under its exponent
                old_val = want[w][b]["val"][:, p0:pos[b]]
                assert torch.equal(got[b, :, p0:pos[b]], e4m3_round(old_val * torch.exp2(-e)[..., None]) * torch.exp2(e)[..., None])
            keep = torch.ones(cache.capacity, dtype=torch.bool)
            keep[p0:p0 + block] = False
            assert torch.equal(got[b][:, keep], want[w][b]["val"][:, keep])


@pytest.mark.parametrize("device", DEVICES)
def test_rope_append_hands_an_accumulator_back(device):
    cache = filled(2, 2, 32, 32, 32, device)
    qkv = torch.randn(2, 8 * 32, device=device)
    cos, sin = tables(32, 32, device)
    plain = kv8.rope_append(cache, qkv.clone(), cos, sin, i32([3, 4], device), 4)
    other = kv8.rope_append(cache, qkv, cos, sin, i32([3, 4], device), 4, clear=True)
    assert torch.equal(plain, other) and not qkv.any()


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
CASES = [  # B, n, H, Hkv, D, block, cap, lens
    (3, 1, 5, 5, 96, 32, 320, [1, 0, 320]),
    (4, 1, 8, 8, 64, 16, 608, [607, 513, 512, 33]),
    (2, 1, 8, 2, 128, 64, 2048, [2047, 130]),          # several CTAs share a range
    (2, 1, 16, 1, 32, 128, 1280, [1279, 1]),
    (40, 1, 2, 2, 32, 16, 640, [(37 * b) % 641 for b in range(40)]),
    (3, 2, 4, 2, 96, 32, 160, [2, 1, 159]),            # the first token sees one key, none, 158
    (2, 5, 12, 3, 64, 32, 1024, [1001, 4]),
    (1, 7, 4, 1, 128, 32, 640, [640]),                 # 28 rows
    (2, 9, 6, 2, 128, 16, 96, [96, 8]),                # 27 rows
    (2, 11, 12, 3, 96, 16, 560, [559, 10]),            # 44 rows: two row tiles
    (1, 64, 2, 2, 96, 64, 640, [631]),                 # 64 rows
    (2, 33, 4, 2, 64, 32, 352, [345, 33]),             # 66 rows
    (2, 9, 28, 2, 96, 32, 640, [640, 5]),              # 126 rows, tiles of 32 that begin inside a token
    (1, 48, 6, 2, 128, 32, 1280, [1270]),
    (1, 49, 6, 2, 128, 32, 1280, [1270]),              # from here on the prompt kernel
    (2, 65, 4, 2, 96, 16, 352, [345, 66]),
    (3, 100, 6, 6, 96, 16, 304, [300, 99, 0]),
    (1, 300, 4, 2, 128, 32, 608, [601]),
    (2, 270, 2, 1, 32, 32, 320, [320, 13]),
    (2, 257, 4, 1, 128, 128, 1664, [1650, 258]),       # a tile of one query
    (1, 160, 2, 2, 96, 16, 1008, [1000]),
    (3, 400, 20, 10, 64, 32, 480, [433, 401, 127]),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B,n,H,Hkv,D,block,cap,lens", CASES)
def test_attention(device, B, n, H, Hkv, D, block, cap, lens):
    g = torch.Generator().manual_seed(7)
    cache = filled(B, Hkv, cap, D, block, device, seed=8)
    q = torch.randn(B, n, H, D, generator=g).to(torch.bfloat16)
    for b in range(B):                       # what lies behind the last key may be anything
        cache.k.view(torch.uint8)[b, :, lens[b]:] = 0x7F
        cache.v.view(torch.uint8)[b, :, lens[b]:] = 0xFF
        cache.v_exp[b, :, (lens[b] + block - 1) // block:] = 127
    out = kv8.attention(q.to(device), cache, i32(lens, device)).double().cpu()
    k, v = (torch.nan_to_num(values(cache, w)) for w in "kv")
    want, mag, big = attend(q.double(), k, v, lens, D ** -0.5)
    tol = tolerance(want, mag, big, D, F16_HALF if kv8.streams(n, D) else BF16_HALF)
    bad = (out - want).abs() > tol
    assert not bad.any(), ((out - want).abs() / tol).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 3])
def test_attention_with_sizes_far_apart(device, n):
    """Blocks of very different exponents, a first token that draws most of the weight, large and tiny queries, a negative scale."""
    B, H, Hkv, D, block, cap = 2, 4, 2, 64, 16, 640
    g = torch.Generator().manual_seed(9)
    cache = KV8Cache.empty(B, Hkv, cap, D, device, block)
    size = torch.exp2(torch.randint(-12, 13, (B, cap // block, Hkv, 1), generator=g).double()).repeat_interleave(block, 1)
    k = torch.randn(B, cap, Hkv, D, generator=g).double()
    k[:, 0] *= 4
    v = torch.randn(B, cap, Hkv, D, generator=g).double() * size
    v[1, :16] = 0                                                      # the reference exponent is that of an empty block
    kv8.append(cache, k.to(torch.bfloat16).to(device), v.to(torch.bfloat16).to(device), i32([0] * B, device))
    q = (torch.randn(B, n, H, D, generator=g) * torch.tensor([1.0, 30.0, 1e-3, 1e-20]).view(1, 1, H, 1)).to(torch.bfloat16)
    for scale in (D ** -0.5, -0.2):
        out = kv8.attention(q.to(device), cache, i32([cap, 77], device), scale=scale).double().cpu()
        want, mag, big = attend(q.double(), values(cache, "k"), values(cache, "v"), [cap, 77], scale)
        tol = tolerance(want, mag, big, D, F16_HALF)
        assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_takes_views(device):
    """A slot of a larger cache, heads of a packed row as queries, a bound on the lengths."""
    S, B, Hkv, D, cap, H = 3, 2, 2, 64, 256, 4
    whole = KV8Cache.empty(S * B, Hkv, cap, D, device)
    k = torch.randn(S * B, cap, Hkv, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(device)
    kv8.append(whole, k, k.flip(1), i32([0] * (S * B), device))
    parts = [t.view(B, S, *t.shape[1:])[:, 1] for t in (whole.k, whole.v, whole.k_exp, whole.v_exp)]
    view = KV8Cache(*parts)
    same = KV8Cache(*(t.contiguous() for t in parts))
    packed = torch.randn(B, 2, 8 * D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)
    q = packed[:, :, 2 * D:6 * D].view(B, 2, H, D)
    odd = torch.empty(B * 2 * H * D + 1, dtype=torch.bfloat16, device=device)[1:].view(B, 2, H, D).copy_(q)
    lens = i32([255, 90], device)
    want = kv8.attention(q.contiguous(), same, lens)
    assert torch.equal(kv8.attention(q, view, lens), want)
    assert torch.equal(kv8.attention(odd, view, lens), want)
    cut = kv8.attention(q, view, lens, max_len=100)
    exact, mag, big = attend(q.cpu().double(), values(view, "k"), values(view, "v"), [100, 90], D ** -0.5)       # (a bound may change the order of the sums)
    assert ((cut.double().cpu() - exact).abs() <= tolerance(exact, mag, big, D, F16_HALF)).all()
    dk, dv = view.decoded()
    assert torch.equal(dk.double().cpu(), values(view, "k").transpose(1, 2)) and torch.equal(dv.double().cpu(), values(view, "v").transpose(1, 2))
    assert kv8.attention(q[:, :0], view, lens).shape == (B, 0, H, D)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_nan_reaches_only_those_who_see_it(device):
    B, n, H, Hkv, D, cap = 1, 4, 2, 2, 64, 160
    cache = filled(B, Hkv, cap, D, 32, device)
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)
    clean = kv8.attention(q, cache, i32([150], device))
    cache.v.view(torch.uint8)[0, 0, 148, 5] = 0x7F          # seen by the last two tokens
    cache.k.view(torch.uint8)[0, 1, 149, 9] = 0xFF          # seen by the last one
    out = kv8.attention(q, cache, i32([150], device))
    nan = torch.zeros(B, n, H, D, dtype=torch.bool)
    nan[0, 2:, 0, 5] = True
    nan[0, 3, 1] = True
    assert torch.equal(out.isnan().cpu(), nan)
    assert torch.equal(out[~out.isnan()], clean[~out.isnan()])


@pytest.mark.parametrize("device", DEVICES)
def test_long_attention_nan_reaches_only_those_who_see_it(device):
    B, n, H, Hkv, D, cap = 2, 70, 4, 2, 128, 416
    assert not kv8.streams(n, D)
    cache = filled(B, Hkv, cap, D, 32, device)
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)
    lens = i32([400, 75], device)
    clean = kv8.attention(q, cache, lens)
    q[0, 3, 1] = float("nan")
    v, k = cache.v.view(torch.uint8), cache.k.view(torch.uint8)
    v[0, 0, 390, 5] = v[0, 0, 395, 5] = 0x7F                # seen by the last ten tokens
    v[0, 0, 20, 6] = 0xFF                                   # by all
    k[0, 1, 399, 9] = 0xFF                                  # by the last one
    v[1, 1, 74, 0] = v[1, 1, 5, 1] = 0x7F                   # by the last one; by all
    out = kv8.attention(q, cache, lens)
    nan = torch.zeros(B, n, H, D, dtype=torch.bool)
    nan[0, 3, 1] = True
    nan[0, 60:, :2, 5] = nan[0, :, :2, 6] = nan[0, 69, 2:] = nan[1, 69, 2:, 0] = nan[1, :, 2:, 1] = True
    assert torch.equal(out.isnan().cpu(), nan)
    assert torch.equal(out[~out.isnan()], clean[~out.isnan()])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,group", [(1, 1), (3, 2)])
@pytest.mark.parametrize("order", ["small first", "large first"])
def test_attention_with_exponents_at_both_ends(device, n, group, order):
    """A block of the largest values next to blocks of the smallest: every key counts in the sum of the weights."""
    B, Hkv, D, block, cap = 2, 2, 64, 16, 640
    g = torch.Generator().manual_seed(11)
    cache = KV8Cache.empty(B, Hkv, cap, D, device, block)
    k, v = (torch.randn(B, cap, Hkv, D, generator=g) for _ in range(2))
    v = v.clamp(0.1, 3.0) * 2.0 ** -45
    at = 0 if order == "large first" else 320
    v[:, at:at + block] = v[:, at:at + block] * 2.0 ** 45 * 2.0 ** 124
    kv8.append(cache, k.to(torch.bfloat16).to(device), v.to(torch.bfloat16).to(device), i32([0] * B, device))
    assert cache.v_exp.max() > 115 and cache.v_exp.min() == -40
    q = torch.randn(B, n, Hkv * group, D, generator=g).to(torch.bfloat16)
    lens = [cap, 330]
    out = kv8.attention(q.to(device), cache, i32(lens, device)).double().cpu()
    want, mag, big = attend(q.double(), values(cache, "k"), values(cache, "v"), lens, D ** -0.5)
    tol = tolerance(want, mag, big, D, F16_HALF)
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()


def test_refusals():
    cache = KV8Cache.empty(2, 2, 64, 32)
    k, p = torch.zeros(2, 4, 2, 32, dtype=torch.bfloat16), i32([0, 0], "cpu")
    qkv, (cos, sin) = torch.zeros(2, 8 * 32), tables(64, 32, "cpu")
    q = torch.zeros(2, 1, 4, 32, dtype=torch.bfloat16)
    bad = [
        lambda: KV8Cache.empty(2, 2, 64, 48), lambda: KV8Cache.empty(2, 2, 64, 32, block=24), lambda: KV8Cache.empty(2, 2, 64, 160),
        lambda: KV8Cache.empty(0, 2, 64, 32), lambda: KV8Cache.empty(2, 2, 0, 32),
        lambda: KV8Cache(cache.k, cache.v, cache.k_exp, cache.v_exp[:, :, :1]),
        lambda: KV8Cache(cache.k.float(), cache.v, cache.k_exp, cache.v_exp),
        lambda: KV8Cache(cache.k, cache.v, cache.k_exp.int(), cache.v_exp),
        lambda: KV8Cache(cache.k.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn), cache.v, cache.k_exp, cache.v_exp),
        lambda: kv8.append(cache, k.float(), k, p), lambda: kv8.append(cache, k, k[:, :3], p), lambda: kv8.append(cache, k[:1], k[:1], p),
        lambda: kv8.append(cache, k, k, p.long()), lambda: kv8.append(cache, k, k, p[:1]), lambda: kv8.append(cache, k, k, p, i32([1, 1, 1], "cpu")),
        lambda: kv8.rope_append(cache, qkv, cos, sin, p, 3), lambda: kv8.rope_append(cache, qkv[:, :-1], cos, sin, p, 4),
        lambda: kv8.rope_append(cache, qkv.half(), cos, sin, p, 4), lambda: kv8.rope_append(cache, qkv, cos[:63], sin, p, 4),
        lambda: kv8.rope_append(cache, qkv, cos.double(), sin, p, 4), lambda: kv8.rope_append(cache, qkv, cos, sin, p, 4, bias=torch.zeros(3)),
        lambda: kv8.rope_append(cache, qkv.bfloat16(), cos, sin, p, 4, clear=True), lambda: kv8.rope_append(cache, qkv, cos, sin, p.long(), 4),
        lambda: kv8.attention(q.float(), cache, p), lambda: kv8.attention(q[:, :, :3], cache, p), lambda: kv8.attention(q[:1], cache, p),
        lambda: kv8.attention(q, cache, p.long()), lambda: kv8.attention(q, cache, p, max_len=0), lambda: kv8.attention(q, cache, p, max_len=65),
        lambda: kv8.attention(q[..., :16], cache, p),
        lambda: KV8Cache(*(t[:1].expand(2, *t.shape[1:]) for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_exp, cache.v_exp))),
        lambda: KV8Cache(*(t[:1].expand(2, *t.shape[1:]) for t in (cache.k, cache.v, cache.k_exp, cache.v_exp))),      # two sequences in one place
        lambda: KV8Cache(cache.k, cache.v, *(t[:, :1].expand(2, 2, 2) for t in (cache.k_exp, cache.v_exp))),
        lambda: kv8.rope_append(cache, qkv[:1].expand(2, -1), cos, sin, p, 4, clear=True),
        lambda: kv8.rope_append(cache, torch.zeros(300).as_strided((2, 256), (32, 1)), cos, sin, p, 4, clear=True),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    kv8.append(cache, k[:, :0], k[:, :0], p)      # nothing to write
    KV8Cache(*(t.transpose(0, 1) for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)))       # heads in any order


# ------------------------------------------------------------------------------------------
# GPU only
# ------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_results_repeat_and_do_not_depend_on_the_batch():
    cache = filled(6, 3, 1500, 96, 32, "cuda")
    q = torch.randn(6, 2, 6, 96, device="cuda", dtype=torch.float32).to(torch.bfloat16)
    lens = i32([1500, 3, 900, 0, 1024, 77], "cuda")
    first = kv8.attention(q, cache, lens)
    for _ in range(5):
        assert torch.equal(kv8.attention(q, cache, lens), first)


FIRST_CALLS = """
import torch
from recurrent_pretraining_b200.ops import kv8
from recurrent_pretraining_b200.ops.sampling import sample_tokens
B, H, D, cap = 2, 4, 64, 2048
cache, other = kv8.KV8Cache.empty(B, H, cap, D, "cuda"), kv8.KV8Cache.empty(B, H, cap, D, "cuda")
k = torch.randn(B, 1500, H, D, device="cuda").to(torch.bfloat16)
qkv, logits = torch.randn(B, 3 * H * D, device="cuda"), torch.randn(B, 9000, device="cuda")
cos, start, pos, lens = torch.ones(cap, D // 2, device="cuda"), *(torch.full((B,), x, dtype=torch.int32, device="cuda") for x in (0, 1500, 1501))
u = torch.tensor([0.2, 0.7], device="cuda")
sin = torch.zeros_like(cos)

def step(cache):
    kv8.append(cache, k, k, start)
    q = kv8.rope_append(cache, qkv, cos, sin, pos, H)
    return kv8.attention(q[:, None], cache, lens), kv8.attention(k[:, :200], cache, lens), kv8.attention(q[:, None], cache, lens, max_len=300), sample_tokens(logits, u, top_p=0.9)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step(cache)
graph.replay()
want = step(other)
assert all(torch.equal(a, b) for a, b in zip(got, want))
pos[1] = cap
graph.replay()
from recurrent_pretraining_b200.ops import cuda as K
assert K.check_device_status() != 0 and K.check_device_status() == 0
"""


@pytest.mark.gpu
def test_first_calls_may_be_captured():
    subprocess.run([sys.executable, "-c", FIRST_CALLS], check=True, timeout=300, cwd=Path(__file__).parents[1])


@pytest.mark.gpu
def test_a_step_in_a_graph_follows_the_device_tensors():
    """Append, attention and the next position captured once and replayed, against the same calls one by one; on a side stream."""
    B, H, Hkv, D, cap = 3, 4, 2, 64, 704
    cos, sin = tables(cap, D, "cuda")
    g = torch.Generator().manual_seed(11)
    steps = torch.randn(6, B, (H + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()

    def step(cache, qkv, pos, lens):
        q = kv8.rope_append(cache, qkv, cos, sin, pos, H)
        return kv8.attention(q[:, None], cache, lens)

    want, cache = [], filled(B, Hkv, cap, D, 16, "cuda")
    for i in range(6):
        pos = i32([510 + i, 30 + i, 15 + i], "cuda")
        want.append(step(cache, steps[i], pos, pos + 1))
    cache = filled(B, Hkv, cap, D, 16, "cuda")
    qkv, pos = steps[0].clone(), i32([510, 30, 15], "cuda")
    lens = pos + 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, qkv, pos, lens)                     # plans and attributes; writing it again changes nothing
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(cache, qkv, pos, lens)
        for i in range(6):
            qkv.copy_(steps[i])
            graph.replay()
            assert torch.equal(out, want[i])
            pos.add_(1)
            lens.add_(1)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.gpu
def test_offsets_beyond_two_gigabytes():
    Hkv, D, cap = 2, 128, 9 * 2 ** 20
    codes = torch.zeros(1, Hkv, cap, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    exps = torch.zeros(1, Hkv, cap // 128, dtype=torch.int8, device="cuda")
    cache = KV8Cache(codes, codes, exps, exps)
    assert codes.numel() > 2 ** 31
    n, start = 200, cap - 300
    k = torch.randn(1, n, Hkv, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    kv8.append(cache, k.cuda(), k.cuda(), i32([start], "cuda"))
    tail = codes[:, :, start:start + n].double().cpu() * torch.exp2(exps[:, :, torch.arange(start, start + n) // 128].double().cpu())[..., None]
    q = torch.randn(1, 1, Hkv, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = kv8.attention(q.cuda(), cache, i32([start + n], "cuda"), scale=1.0).double().cpu()
    for h in range(Hkv):                        # every other key is zero: weight exp(0), value 0
        s = tail[0, h] @ q[0, 0, h].double()
        top = max(0.0, float(s.max()))
        w = torch.exp(s - top)
        z = w.sum() + start * math.exp(-top)
        want, mag = w @ tail[0, h] / z, w @ tail[0, h].abs() / z
        big = (tail[0, h].abs() @ q[0, 0, h].double().abs()).max()
        # the sum of 9.4 million weights of zero scores adds fp32 roundings of partial sums: 2^-24 per addition of a lane, at most 2^-9 in all
        assert ((out[0, 0, h] - want).abs() <= tolerance(want, mag, big, D, F16_HALF + 2.0 ** -9)).all()


# ------------------------------------------------------------------------------------------
# scratch memory of the prompt path
# ------------------------------------------------------------------------------------------
def run_in_groups(monkeypatch, limit, B, n, H, Hkv, D, block, cap, lens, device="cuda"):
    monkeypatch.setattr(kv8, "PROMPT_SCRATCH", limit)
    cache = filled(B, Hkv, cap, D, block, device, seed=8)
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16)
    for b in range(B):
        cache.k.view(torch.uint8)[b, :, lens[b]:] = 0x7F
        cache.v.view(torch.uint8)[b, :, lens[b]:] = 0xFF
    out = kv8.attention(q.to(device), cache, i32(lens, device)).double().cpu()
    k, v = (torch.nan_to_num(values(cache, w)) for w in "kv")
    want, mag, big = attend(q.double(), k, v, lens, D ** -0.5)
    tol = tolerance(want, mag, big, D, BF16_HALF)
    assert ((out - want).abs() <= tol).all(), ((out - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("limit", [1, 400_000, 2_000_000])     # a key head of a sequence at a time, a few of them, whole sequences
@pytest.mark.parametrize("B,n,H,Hkv,D,block,cap,lens", [
    (3, 100, 6, 6, 96, 16, 304, [300, 99, 0]),
    (5, 65, 6, 3, 128, 32, 352, [345, 66, 1, 352, 130]),
    (2, 270, 4, 2, 32, 32, 320, [320, 13]),
])
def test_long_attention_in_groups(monkeypatch, limit, B, n, H, Hkv, D, block, cap, lens):
    """Sequences and key heads answered one group after the other through the same scratch memory, the last group a smaller one."""
    run_in_groups(monkeypatch, limit, B, n, H, Hkv, D, block, cap, lens)


@pytest.mark.gpu
def test_long_attention_in_groups_nan_reaches_only_those_who_see_it(monkeypatch):
    monkeypatch.setattr(kv8, "PROMPT_SCRATCH", 1)
    test_long_attention_nan_reaches_only_those_who_see_it("cuda")


def test_prompt_scratch_is_bounded():
    """Whatever the sizes are, up to what one key head of one sequence takes."""
    f = kv8._k()
    for B, Hkv, H, D, n, most in [(64, 8, 32, 128, 64, 32768), (16, 55, 55, 96, 300, 65536), (1, 8, 32, 128, 1500, 8192), (16400, 1, 1, 128, 49, 64),
                                  (65535, 2, 4, 64, 100, 128), (4, 3, 3, 32, 5000, 1 << 20), (1, 1, 16, 128, 64, 1 << 21), (40000, 1, 1, 128, 50, 1 << 17)]:
        got = f.scratch(B, Hkv, H, D, n, most, kv8.PROMPT_SCRATCH)
        least = 2 * ((most + 127) // 128 * 128) * D * 2
        assert 0 < got <= max(kv8.PROMPT_SCRATCH, least + (64 << 20)), (B, Hkv, n, most, got)
    assert f.scratch(1, 1, 1, 128, 1 << 23, 1 << 23, kv8.PROMPT_SCRATCH) == 0         # more query tiles than a grid holds: streamed


@pytest.mark.gpu
def test_scratch_of_long_attention_follows_no_capacity():
    B, n, H, Hkv, D, cap = 64, 64, 8, 8, 128, 16384
    cache = KV8Cache.empty(B, Hkv, cap, D, "cuda")
    k = torch.randn(B, 200, Hkv, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    kv8.append(cache, k, k, i32([0] * B, "cuda"))
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    lens = i32([200 - b for b in range(B)], "cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = kv8.attention(q, cache, lens)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before < 1.1 * kv8.PROMPT_SCRATCH
    for b in (0, 31, 63):
        part = KV8Cache(*(t[b:b + 1, :, :256 if t.dim() == 4 else 8].contiguous() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)))
        want, mag, big = attend(q[b:b + 1].double().cpu(), values(part, "k"), values(part, "v"), [200 - b], D ** -0.5)
        assert ((out[b:b + 1].double().cpu() - want).abs() <= tolerance(want, mag, big, D, BF16_HALF)).all()


@pytest.mark.gpu
def test_long_attention_of_more_sequences_than_a_grid_of_tiles_holds():
    B, n, D, cap = 16400, 49, 128, 64
    assert not kv8.streams(n, D)
    cache = KV8Cache.empty(B, 1, cap, D, "cuda")
    k, v = (torch.randn(B, cap, 1, D, device="cuda", generator=torch.Generator("cuda").manual_seed(s)).to(torch.bfloat16) for s in (1, 2))
    kv8.append(cache, k, v, torch.zeros(B, dtype=torch.int32, device="cuda"))
    q = torch.randn(B, n, 1, D, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).to(torch.bfloat16)
    lens = (torch.arange(B, device="cuda") % (cap + 1)).int()
    out = kv8.attention(q, cache, lens)
    for b in (0, 1, 63, 8200, 16383, 16384, 16399):
        part = KV8Cache(*(t[b:b + 1].contiguous() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)))
        want, mag, big = attend(q[b:b + 1].double().cpu(), values(part, "k"), values(part, "v"), [b % (cap + 1)], D ** -0.5)
        assert ((out[b:b + 1].double().cpu() - want).abs() <= tolerance(want, mag, big, D, BF16_HALF)).all()


@pytest.mark.gpu
def test_what_the_tiles_do_not_take_is_streamed(monkeypatch):
    monkeypatch.setattr(kv8, "_prompt_call", lambda *a: None)
    B, n, H, Hkv, D, block, cap = 2, 100, 4, 2, 128, 32, 352
    assert not kv8.streams(n, D)
    cache = filled(B, Hkv, cap, D, block, "cuda", seed=8)
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16)
    out = kv8.attention(q.cuda(), cache, i32([345, 66], "cuda")).double().cpu()
    want, mag, big = attend(q.double(), values(cache, "k"), values(cache, "v"), [345, 66], D ** -0.5)
    assert ((out - want).abs() <= tolerance(want, mag, big, D, F16_HALF)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 60])
def test_results_carry_no_gradient(device, n):
    """On either device, whatever requires one; an accumulator that requires one may be cleared."""
    B, H, Hkv, D = 2, 4, 2, 128
    cache = filled(B, Hkv, 96, D, 32, device)
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device).requires_grad_()
    assert not kv8.attention(q, cache, i32([90, 70], device)).requires_grad
    assert not kv8.attention(q[:, :0], cache, i32([90, 70], device)).requires_grad
    cos, sin = tables(96, D, device)
    qkv = torch.randn(B, (H + 2 * Hkv) * D, device=device, requires_grad=True)
    bias = torch.randn((H + Hkv) * D, device=device, requires_grad=True)
    assert not kv8.rope_append(cache, qkv, cos, sin, i32([3, 4], device), H, bias=bias).requires_grad
    assert not kv8.rope_append(cache, qkv, cos, sin, i32([5, 6], device), H, bias=bias, clear=True).requires_grad
    assert not qkv.detach().any()
    k = torch.randn(B, 3, Hkv, D, device=device).to(torch.bfloat16).requires_grad_()
    kv8.append(cache, k, k, i32([7, 8], device))
    assert not any(t.requires_grad for t in (cache.k, cache.v, cache.k_exp, cache.v_exp, *cache.decoded()))


@pytest.mark.parametrize("device", DEVICES)
def test_what_a_cache_remembers_of_its_calls_is_small(device):
    """Plans and templates, no buffers of a call's size: an engine keeps a cache per layer and recurrence."""
    B, H, Hkv, D = 8, 16, 4, 64
    cache = filled(B, Hkv, 96, D, 32, device)
    cos, sin = tables(96, D, device)
    q = kv8.rope_append(cache, torch.randn(B, (H + 2 * Hkv) * D, device=device), cos, sin, i32([3] * B, device), H)
    kv8.attention(q[:, None], cache, i32([4] * B, device))
    kept = [x for call in cache._calls.values() if isinstance(call, tuple) for x in call if torch.is_tensor(x)]
    assert sum(t.untyped_storage().nbytes() for t in kept) <= 64
    assert q.shape == (B, H, D) and q.is_contiguous()


@pytest.mark.parametrize("device", DEVICES)
def test_decoded_positions(device):
    """Keys and values of the first positions only: memory for those, whatever the capacity is."""
    cache = filled(2, 3, 320, 96, 32, device)
    whole = cache.decoded()
    for length in (1, 31, 130, 320):
        for got, all_, which in zip(cache.decoded(length), whole, "kv"):
            assert got.shape == (2, length, 3, 96) and got.untyped_storage().nbytes() == 2 * 2 * length * 3 * 96
            assert torch.equal(got, all_[:, :length]) and torch.equal(got.double().cpu(), values(cache, which)[:, :, :length].transpose(1, 2))
    for bad in (0, -1, 321):
        with pytest.raises(ValueError):
            cache.decoded(bad)


@pytest.mark.gpu
def test_a_sequence_alone_and_in_a_batch():
    """Shares are cut from the lengths of all sequences, so the order of a sum follows the batch; the result stays within its tolerance."""
    B, n, H, Hkv, D, cap = 6, 2, 6, 3, 96, 1504
    cache = filled(B, Hkv, cap, D, 32, "cuda")
    q = torch.randn(B, n, H, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    lens = [1500, 3, 900, 0, 1024, 77]
    whole = kv8.attention(q.cuda(), cache, i32(lens, "cuda")).double().cpu()
    for b in range(B):
        alone = KV8Cache(*(t[b:b + 1] for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)))
        one = kv8.attention(q[b:b + 1].cuda(), alone, i32(lens[b:b + 1], "cuda")).double().cpu()
        want, mag, big = attend(q[b:b + 1].double(), values(alone, "k"), values(alone, "v"), lens[b:b + 1], D ** -0.5)
        tol = tolerance(want, mag, big, D, F16_HALF)
        assert ((one - want).abs() <= tol).all() and ((whole[b:b + 1] - want).abs() <= tol).all()
