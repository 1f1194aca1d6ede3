"""``ops/sampling.py: sample_tokens`` against its definition in 64 bits: the same tests on CPU tensors (plain path) and on the GPU (kernel)."""
import math

import numpy as np
import pytest
import torch

from recurrent_pretraining_b200.ops.sampling import MAX_VOCAB, sample_tokens

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def oracle(x, u, t, k, p, m):
    """One row: x fp64 [V] (numpy), settings as the numbers that fp32 holds."""
    t, p, m, u = (float(np.float32(a)) for a in (t, p, m, u))
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1
    if not t > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(x == top, 0.0, (x - top) / t))
    order = np.lexsort((np.arange(x.size), -x))
    keep = np.ones(x.size, bool)
    if 0 < k < x.size:
        keep &= x >= x[order[k - 1]]
    if 0 < p < 1:
        inside = np.cumsum(w[order]) <= p * math.fsum(w)
        inside[0] = True
        keep[order] &= inside
    if m > 0:
        keep &= w >= min(m, 1.0)
    w = np.where(keep, w, 0.0)
    c = np.cumsum(w)
    hit = np.nonzero(c > u * c[-1])[0]
    return int(hit[0]) if hit.size else int(np.nonzero(keep)[0][-1])


def compare(logits, u, device, t=1.0, k=0, p=1.0, m=0.0):
    def to(a, dtype):
        return torch.tensor(a, dtype=dtype, device=device) if isinstance(a, list) else a

    got = sample_tokens(logits.to(device), u.to(device), temperature=to(t, torch.float32), top_k=to(k, torch.int32), top_p=to(p, torch.float32),
                        min_p=to(m, torch.float32))
    assert got.dtype == torch.int64 and got.device.type == device
    row = lambda a, b: a[b] if isinstance(a, list) else a  # noqa: E731
    x = logits.double().numpy()
    want = [oracle(x[b], float(u[b]), row(t, b), row(k, b), row(p, b), row(m, b)) for b in range(len(x))]
    assert got.tolist() == want


def numbers(B, seed=0):
    u = torch.rand(B, generator=torch.Generator().manual_seed(seed))
    u[0] = 0.0
    if B > 1:
        u[1] = 1 - 2.0 ** -24
    return u


FILTERS = [dict(), dict(t=0.6), dict(k=1), dict(k=40, t=1.3), dict(p=0.9), dict(p=1e-6), dict(p=0.999999, t=2.0), dict(m=0.05), dict(m=1.0), dict(k=500, p=0.7, m=0.01, t=0.8),
           dict(k=3, p=0.99), dict(t=0.0), dict(t=1e-6), dict(t=1e30), dict(t=100.0, p=0.5, k=10000)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("setting", FILTERS, ids=str)
@pytest.mark.parametrize("B,V,dtype", [(5, 1000, torch.float32), (3, 32003, torch.bfloat16), (2, 65536, torch.float32)])
def test_filters(device, B, V, dtype, setting):
    x = (2.5 * torch.randn(B, V, generator=torch.Generator().manual_seed(V))).to(dtype)
    compare(x, numbers(B), device, **setting)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [1, 2, 7, 31, 512, 513, 1024, 1025, 4097, 8193, 16384, 65537, 100003, MAX_VOCAB])
def test_vocabulary_sizes(device, V):
    B = 4
    x = torch.randn(B, V, generator=torch.Generator().manual_seed(V)) * 3
    compare(x, numbers(B, V), device, t=[1.0, 0.7, 0.0, 1.0], k=[0, 20, 0, V], p=[1.0, 0.95, 1.0, 0.4], m=[0.0, 0.0, 0.0, 0.03])
    compare(x.to(torch.bfloat16), numbers(B, V), device, p=0.9)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [1000, 40000])
@pytest.mark.parametrize("setting", [dict(), dict(p=0.37), dict(k=10), dict(k=10, p=0.5), dict(p=0.001, m=0.5), dict(p=1e-7), dict(k=39999, p=0.75)], ids=str)
def test_equal_logits(device, V, setting):
    """One value, two values, and a few: prefixes end inside runs of equal logits, in index order."""
    g = torch.Generator().manual_seed(3)
    x = torch.stack([torch.zeros(V), torch.randint(0, 2, (V,), generator=g).float(), torch.randint(-3, 4, (V,), generator=g).float() * 0.5,
                     torch.where(torch.randint(0, 2, (V,), generator=g).bool(), torch.zeros(V), -torch.zeros(V))])
    compare(x, numbers(4), device, **setting)
    compare(x.to(torch.bfloat16), numbers(4, 1), device, **setting)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("setting", [dict(p=0.5), dict(k=7000), dict(k=7000, p=0.3), dict(p=0.9, k=30000)], ids=str)
def test_many_different_logits_close_together(device, setting):
    """Thousands of candidates inside one bin of the first histogram: it is divided again."""
    g = torch.Generator().manual_seed(4)
    x = torch.stack([torch.rand(40000, generator=g) * 1e-3, torch.rand(40000, generator=g) * 0.03 - 5, (torch.rand(40000, generator=g) * 64).round() / 4096])
    x[1, 17] = 0.0
    compare(x, numbers(3), device, **setting)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [64, 20000])
def test_rows_with_infinities_and_nan(device, V):
    inf, nan = float("inf"), float("nan")
    x = torch.randn(7, V, generator=torch.Generator().manual_seed(5))
    x[0] = -inf
    x[1] = nan
    x[2, :] = -inf
    x[2, V // 2] = -1e30
    x[3, ::2] = -inf
    x[4, 5], x[4, V - 3] = inf, inf
    x[5, ::3] = nan
    x[6, 1:] = -3e38
    for setting in (dict(), dict(p=0.8), dict(k=5), dict(m=0.1), dict(t=0.0), dict(k=V - 1, p=0.9, m=0.01)):
        compare(x, numbers(7), device, **setting)


@pytest.mark.parametrize("device", DEVICES)
def test_greedy_rows_take_the_lowest_index(device):
    x = torch.zeros(3, 30000)
    x[0, [29999, 777, 20000]] = 5.0
    x[1, [0, 29999]] = 5.0
    assert sample_tokens(x.to(device), torch.full((3,), 0.9, device=device), temperature=0.0).tolist() == [777, 0, 0]


@pytest.mark.parametrize("device", DEVICES)
def test_rows_with_a_pitch_and_numbers_outside(device):
    wide = torch.randn(4, 5003, generator=torch.Generator().manual_seed(6))
    for lo in (0, 1, 4):
        x = wide.to(device)[:, lo:lo + 4999]
        u = torch.tensor([0.3, 1.0, -0.5, float("nan")])
        got = sample_tokens(x, u.to(device), top_p=0.9).tolist()
        first = oracle(wide[2, lo:lo + 4999].double().numpy(), 0.0, 1.0, 0, 0.9, 0.0)
        assert got[0] == oracle(wide[0, lo:lo + 4999].double().numpy(), 0.3, 1.0, 0, 0.9, 0.0) and got[2] == first
        assert got[3] == oracle(wide[3, lo:lo + 4999].double().numpy(), 0.0, 1.0, 0, 0.9, 0.0)
        assert got[1] == oracle(wide[1, lo:lo + 4999].double().numpy(), 1 - 2.0 ** -24, 1.0, 0, 0.9, 0.0)
    assert sample_tokens(wide[:0].to(device), torch.zeros(0, device=device)).shape == (0,)


@pytest.mark.parametrize("device", DEVICES)
def test_the_share_of_each_token_is_its_probability(device):
    """Equally spaced numbers: every token comes as often as its probability says, to one part in their count on either side."""
    n = 4096
    x = torch.randn(1, 50, generator=torch.Generator().manual_seed(8))
    u = (torch.arange(n).float() + 0.5) / n
    got = sample_tokens(x.expand(n, 50).contiguous().to(device), u.to(device), temperature=0.9).cpu()
    share = torch.bincount(got, minlength=50).double() / n
    assert (share - torch.softmax(x[0].double() / float(np.float32(0.9)), -1)).abs().max() <= 1.0 / n + 1e-9


def test_refusals():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    bad = [lambda: sample_tokens(x.double(), u), lambda: sample_tokens(x[0], u), lambda: sample_tokens(x, u[:1]), lambda: sample_tokens(x, u.double()),
           lambda: sample_tokens(x.t(), torch.zeros(8)), lambda: sample_tokens(x[:, :0], u), lambda: sample_tokens(x, u, temperature=-1.0),
           lambda: sample_tokens(x, u, temperature=float("nan")), lambda: sample_tokens(x, u, top_p=1.5), lambda: sample_tokens(x, u, min_p=-0.1),
           lambda: sample_tokens(x, u, top_k=-1), lambda: sample_tokens(x, u, top_k=torch.tensor([1, 2])), lambda: sample_tokens(x, u, top_p=torch.ones(3)),
           lambda: sample_tokens(torch.zeros(1, MAX_VOCAB + 1), u[:1]), lambda: sample_tokens(x[:1].expand(2, 8), u)]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")


@pytest.mark.gpu
def test_captured_calls_follow_their_tensors():
    B, V = 6, 20011
    g = torch.Generator().manual_seed(9)
    x, u = torch.randn(B, V, device="cuda"), torch.rand(B, device="cuda")
    k = torch.tensor([0, 1, 50, 0, 0, 7], dtype=torch.int32, device="cuda")
    p = torch.tensor([1.0, 1.0, 0.9, 0.5, 1.0, 0.99], device="cuda")
    sample_tokens(x, u, top_k=k, top_p=p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, u, top_k=k, top_p=p)
    for _ in range(4):
        x.copy_(torch.randn(B, V, generator=g))
        u.copy_(torch.rand(B, generator=g))
        graph.replay()
        rows = x.double().cpu().numpy()
        assert out.tolist() == [oracle(rows[b], float(u[b]), 1.0, int(k[b]), float(p[b]), 0.0) for b in range(B)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("V", [6, 20011])
def test_an_infinite_temperature_weighs_finite_logits_alike(device, per_row, V):
    """The limit of high temperatures: weight 1, or 0 at an infinite distance from the largest."""
    inf = float("inf")
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(2))
    x[0, 1] = x[1, ::2] = x[1, 5] = -inf
    x[2, [3, V - 2]] = inf
    t = torch.full((3,), inf, device=device) if per_row else inf
    for u in (0.0, 0.1, 0.5, 0.99):
        for setting in (dict(), dict(min_p=0.3), dict(min_p=1.0), dict(top_k=2), dict(top_p=0.5), dict(top_p=0.5, min_p=1.0)):
            got = sample_tokens(x.to(device), torch.full((3,), u, device=device), temperature=t, **setting).tolist()
            for b in range(3):
                w = (x[b] == inf if b == 2 else x[b] > -inf).numpy()
                order = np.lexsort((np.arange(V), -x[b].numpy()))
                keep = w.copy()
                if "top_k" in setting:
                    keep &= x[b].numpy() >= x[b].numpy()[order[1]]
                if "top_p" in setting:
                    keep[order[max(1, int(0.5 * w.sum())):]] = False
                kept = np.nonzero(keep)[0]
                assert got[b] == kept[int(float(np.float32(u)) * kept.size)], (u, setting, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [50, 5000])
@pytest.mark.parametrize("setting", [dict(), dict(p=0.6), dict(k=20), dict(k=30, p=0.4), dict(m=0.1)], ids=str)
def test_logits_further_apart_than_the_largest_number(device, V, setting):
    """Distances of more than 3.4e38 under a temperature that makes weights of them."""
    x = torch.rand(4, V, generator=torch.Generator().manual_seed(12)) * 2 - 1
    compare(x * 3.4e38, numbers(4, 3), device, t=1e38, **setting)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("setting", [dict(), dict(p=0.6), dict(k=20), dict(m=0.1)], ids=str)
def test_temperatures_below_the_smallest_normal_number(device, setting):
    x = torch.rand(4, 3001, generator=torch.Generator().manual_seed(13)) * 1e-38
    compare(x, numbers(4, 4), device, t=2e-39, **setting)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [4, 9000])
def test_numbers_from_one_on_take_the_last_kept_token_with_a_weight(device, V):
    """Tokens below 2^-44 of the largest weigh nothing and are never drawn."""
    x = torch.full((4, V), -2000.0)
    x[:, 0], x[:, 1], x[:, 2] = 5.0, 0.0, -200.0
    x[2, V - 1] = 5 - 30.0                  # e^-30 = 2^-43.3
    x[3, V - 1] = 5 - 31.2                  # 2^-45.01
    for u in (1.0, 7.0, float("inf")):
        got = sample_tokens(x.to(device), torch.full((4,), u, device=device)).tolist()
        assert got == [1, 1, V - 1, 1]
        assert sample_tokens(x.to(device), torch.full((4,), u, device=device), top_k=1).tolist() == [0] * 4
        assert sample_tokens(x.to(device), torch.full((4,), u, device=device), temperature=1000.0).tolist() == [V - 1] * 4


@pytest.mark.parametrize("device", DEVICES)
def test_a_min_p_of_one_keeps_the_largest_alone(device):
    """However close the next one is: its weight is below the largest's, although the difference is lost when weights are numbers near one."""
    x = torch.full((2, 3000), -5.0)
    x[0, [10, 2000]] = torch.tensor([1e-30, 2e-30])
    x[1, [10, 2000, 2500]] = torch.tensor([4.0, 4.0, 3.9999998])
    for u, want in ((0.0, [2000, 10]), (0.4, [2000, 10]), (0.9, [2000, 2000])):
        assert sample_tokens(x.to(device), torch.full((2,), u, device=device), min_p=1.0).tolist() == want


def test_ctas_of_a_row_follow_the_device():
    import ctypes as C

    from recurrent_pretraining_b200.ops import cuda as K

    ctas = K._sig("b200_sample_ctas", [C.c_int] * 4)
    for sms in (148, 74, 1):
        for wide in (0, 1):
            for B in (1, 4, 5, 18, 64, 5000):
                for V in (1, 1024, 1025, 32003, 65536, MAX_VOCAB):
                    c = ctas(B, V, sms, wide)
                    assert c in (1, 2, 4, 8, 16) and (c < 16 or (wide and B <= 4)) and -(-V // c) <= 40960
                    assert c == 1 or -(-V // (c // 2)) > 1024                          # no slices that are not worth a CTA
                    assert B * c <= 2 * sms or c in (1, 16) or -(-V // (c // 2)) > 40960
    assert [ctas(b, 65536, 148, 1) for b in (1, 4, 5, 18, 64, 200)] == [16, 16, 8, 8, 4, 2]
