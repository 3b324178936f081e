"""Sampling with temperature, top-k, top-p and min-p from given random numbers, against the definition in whole numbers (weights in units of
2^-44 of the largest) and 64-bit arithmetic: equal tokens, at sizes around the kernel's lanes, waves and places, with ties, masked and
other odd logits, and each filter at its ends."""
import math

import numpy as np
import pytest
import torch

from swifttransformer_amd.ops import kernels as K

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def drawn(x, u, t, k, p, least):
    """One row's token by the definition; x float32, the others Python numbers that float32 holds."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if not t > 0 or k == 1 or not p > 0 or top == -np.inf:
        return int(order[0])
    if top == np.inf:
        w = (x == top).astype(np.float64)
    else:
        w = np.where(x == -np.inf, 0.0, np.exp((np.maximum(x, -1e300) - top) / t))
    w = np.floor(w * 2.0 ** 44 + 0.5).astype(np.int64)
    kept = order[:k] if k > 0 else order
    if p < 1:
        sums = np.cumsum(w[kept])
        share = min(max(math.ceil(p * float(sums[-1])), 1), int(sums[-1]))
        kept = kept[:int(np.searchsorted(sums, share, side="left")) + 1]
    kept = np.sort(kept[w[kept] >= min(least, 1.0) * 2.0 ** 44])
    sums = np.cumsum(w[kept])
    total = int(sums[-1])
    below = min(max(int(math.floor(u * float(total))), 0), total - 1)
    return int(kept[int(np.searchsorted(sums, below + 1, side="left"))])


def floats(values):
    return torch.tensor(values, dtype=torch.float32)


def check(logits, u, t, k, p, least, **kw):
    want = [drawn(logits[r].numpy(), float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(least[r])) for r in range(len(logits))]
    got = K.sample_filtered(logits.to(DEV), u.to(DEV), t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), min_p=least.to(DEV), **kw)
    assert got.dtype == torch.int32 and got.cpu().tolist() == want


def settings(rows, vocab, g):
    pick = lambda options: floats([options[int(torch.randint(len(options), (1,), generator=g))] for _ in range(rows)])  # noqa: E731
    k = pick([0, 0, -1, 1, 2, 5, 50, 700, vocab - 1, vocab, vocab + 5]).int()
    return (torch.where(torch.rand(rows, generator=g) < 0.2, pick([0.0, 1.0 - 2.0 ** -24]), torch.rand(rows, generator=g)),
            pick([0.0, 0.05, 0.7, 1.0, 1.5, 30.0]), k, pick([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 1.0]), pick([0.0, 0.0, 0.02, 0.5, 1.0]))


@pytest.mark.parametrize("kind", ["normal", "peaked", "halves", "equal", "two", "masked", "lowest", "infinite", "nan"])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 256, 257, 1023, 1025, 4099, 20011])
def test_rows(vocab, kind):
    g = torch.Generator().manual_seed(vocab)
    rows = 24
    x = 3 * torch.randn(rows, vocab, generator=g)
    if kind == "peaked":
        x = x + 9 * (torch.rand(rows, vocab, generator=g) < 8.0 / vocab)
    elif kind == "halves":
        x = torch.round(2 * x) / 2
    elif kind == "equal":
        x = torch.full_like(x, 1.25)
    elif kind == "two":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.3, 2.0, -1.0)
    elif kind == "masked":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.9, -math.inf, x)
        x[0] = -math.inf
    elif kind == "lowest":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.9, torch.finfo(torch.float32).min, x)
    elif kind == "infinite":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 3.0 / vocab, math.inf, x)
    elif kind == "nan":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.3, math.nan, x)
        x[0] = math.nan
    check(x, *settings(rows, vocab, g))


@pytest.mark.parametrize("vocab", [50272, 65536, 131075, 262144])
def test_wide(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.cat([3 * torch.randn(9, vocab, generator=g), torch.randn(3, vocab, generator=g).bfloat16().float(), torch.zeros(2, vocab)])
    check(x, *settings(len(x), vocab, g))


@pytest.mark.parametrize("temperature", [1e-38, 1e-6, 1e6, 3e38, math.inf, -1.0, math.nan])
def test_temperatures(temperature):
    g = torch.Generator().manual_seed(3)
    x = torch.cat([4 * torch.randn(4, 3000, generator=g), 1e38 * torch.randn(4, 3000, generator=g), 1e-40 * torch.randn(4, 3000, generator=g)])
    n = len(x)
    check(x, torch.rand(n, generator=g), torch.full((n,), temperature), torch.tensor([0, 7, 100, 0] * 3).int(), floats([0.9, 1.0, 0.5, 1.0] * 3),
          floats([0.0, 0.0, 0.1, 0.0] * 3))


@pytest.mark.parametrize("temperature", [1e37, 1.2e37, 6e37, 1e38, 3.4e38, math.inf])
@pytest.mark.parametrize("vocab", [700, 3000, 20000])
def test_differences_that_no_float_holds(vocab, temperature):
    """Finite logits further apart than the largest number, at temperatures that give all of them weight."""
    g = torch.Generator().manual_seed(vocab)
    n = 24
    x = 3.3e38 * (2 * torch.rand(n, vocab, generator=g) - 1)
    x[::3] = torch.where(torch.rand(n // 3, vocab, generator=g) < 0.01, x[::3], -x[::3].abs())
    k = torch.tensor([0, 0, 600, vocab // 2] * 6).int()
    check(x, torch.rand(n, generator=g), torch.full((n,), temperature), k, floats([0.2, 0.6, 0.9, 0.99, 1.0 - 2.0 ** -20, 1.0] * 4), floats([0.0, 0.0, 0.0, 0.1] * 6))


def test_a_step_that_holds_most_of_the_row():
    """Nearly all logits within one step of the histogram, then within one step of that one, down to values a bit apart."""
    g = torch.Generator().manual_seed(9)
    n, V = 12, 9000
    x = 1.0 + torch.randint(0, 40, (n, V), generator=g) * 2.0 ** -23
    x[:, ::50] += torch.rand(n, V // 50, generator=g) * 1e-3
    x[:, 17] = 9.0
    check(x, torch.rand(n, generator=g), torch.ones(n), torch.tensor([0, 2000, 5000, 8990] * 3).int(), floats([0.3, 0.5, 0.7, 0.99] * 3), torch.zeros(n))


def test_filters_left_out():
    g = torch.Generator().manual_seed(2)
    x, u, t = torch.randn(6, 777, generator=g), torch.rand(6, generator=g), floats([0.0, 0.5, 1.0, 2.0, 1.0, 1.0])
    got = K.sample_filtered(x.to(DEV), u.to(DEV), t.to(DEV))
    assert got.cpu().tolist() == [drawn(x[r].numpy(), float(u[r]), float(t[r]), 0, 1.0, 0.0) for r in range(6)]
    assert K.sample_filtered(x[:0].to(DEV), u[:0].to(DEV), t[:0].to(DEV)).shape == (0,)


@pytest.mark.parametrize("stride,offset", [(1003, 0), (1004, 1), (2000, 3)])
def test_strided_rows(stride, offset):
    g = torch.Generator().manual_seed(stride)
    base = torch.full((5 * stride + 8,), 99.0)
    rows = base.as_strided((5, 1003), (stride, 1), offset)
    rows.copy_(torch.randn(5, 1003, generator=g))
    u, t, k, p, least = settings(5, 1003, g)
    want = [drawn(rows[r].numpy(), float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(least[r])) for r in range(5)]
    there = base.to(DEV).as_strided((5, 1003), (stride, 1), offset)
    out = torch.full((5,), -7, dtype=torch.int32, device=DEV)
    got = K.sample_filtered(there, u.to(DEV), t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV), min_p=least.to(DEV), out=out)
    assert got.data_ptr() == out.data_ptr() and got.cpu().tolist() == want


def test_recorded_and_on_another_stream():
    g = torch.Generator().manual_seed(4)
    V, n = 5000, 8
    x, u = torch.zeros(n, V, device=DEV), torch.zeros(n, device=DEV)
    t, k, p, least = torch.ones(n), torch.tensor([0, 5, 50, 900] * 2).int(), floats([1.0, 0.9, 0.8, 0.5] * 2), floats([0.0, 0.0, 0.1, 0.0] * 2)
    on = [v.to(DEV) for v in (t, k, p, least)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.sample_filtered(x, u, on[0], top_k=on[1], top_p=on[2], min_p=on[3])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = K.sample_filtered(x, u, on[0], top_k=on[1], top_p=on[2], min_p=on[3])
    torch.cuda.synchronize()
    for seed in range(4):
        g.manual_seed(seed)
        a, b = 4 * torch.randn(n, V, generator=g), torch.rand(n, generator=g)
        x.copy_(a)
        u.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = [drawn(a[r].numpy(), float(b[r]), float(t[r]), int(k[r]), float(p[r]), float(least[r])) for r in range(n)]
        assert got.cpu().tolist() == want
        assert K.sample_filtered(x, u, on[0], top_k=on[1], top_p=on[2], min_p=on[3]).cpu().tolist() == want


def test_frequencies():
    """Random numbers spread evenly over [0, 1) give every kept token its share of them, to one of them a border."""
    n = 4096
    x = floats([2.0, 0.5, 1.0, -1.0, 1.5, 0.0])
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    got = K.sample_filtered(x.expand(n, 6).contiguous().to(DEV), u.to(DEV), torch.ones(n, device=DEV), top_k=torch.full((n,), 4, dtype=torch.int32, device=DEV))
    share = torch.softmax(torch.where(x >= 0.5, x, -math.inf).double(), 0)
    counts = torch.bincount(got.cpu().long(), minlength=6)
    assert (counts - n * share).abs().max() <= 2


def test_refusals():
    x, r = torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV)
    ok = dict(top_k=torch.zeros(2, dtype=torch.int32, device=DEV))
    K.sample_filtered(x, r, r, **ok)
    for bad in (lambda: K.sample_filtered(x.double(), r, r), lambda: K.sample_filtered(x, r[:1], r), lambda: K.sample_filtered(x, r, r.int()),
                lambda: K.sample_filtered(x.t(), r, r), lambda: K.sample_filtered(x, r, r, top_k=r), lambda: K.sample_filtered(x, r.cpu(), r),
                lambda: K.sample_filtered(x, r, r, top_p=r[:1]), lambda: K.sample_filtered(x[:1].expand(2, 8), r, r),
                lambda: K.sample_filtered(x, r, r, out=torch.zeros(2, dtype=torch.int64, device=DEV)),
                lambda: K.sample_filtered(torch.zeros(2, (1 << 18) + 1, device=DEV), r, r)):
        with pytest.raises(K.KernelError):
            bad()
