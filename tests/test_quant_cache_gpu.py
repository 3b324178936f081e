"""The cache in 8 bits: entries and exponents equal, bit for bit, to the definition (one rounding to e4m3, to nearest even, under the smallest power of two
that keeps the largest at most 448), and back; page sizes, heads, strides, values from zero to the largest and not finite, padding rows
and pages that are none."""
import math

import pytest
import torch

from swifttransformer_amd.ops import kernels as K

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


def small(x):
    """(bits, exponents) of heads [..., head_dim] by the definition, in 64 bits."""
    x = x.double()
    big = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    e = torch.full(big.shape, 127)
    for at in range(1, 255):
        fits = big <= 448 * 2.0 ** (at - 127)
        if at == 1:
            e = torch.where(fits, 1, 254)
            done = fits
        else:
            e = torch.where(fits & ~done, at, e)
            done = done | fits
    e = torch.where(big == 0, 127, e)
    y = torch.where(torch.isfinite(x), x, torch.full_like(x, math.nan)) * torch.exp2(127.0 - e.double())[..., None]
    return y.float().to(E4M3).view(torch.uint8), e.to(torch.uint8)


def pools(pages, heads, page, hd, strided):
    extra = 2 if strided else 0
    k, v = (torch.randint(0, 255, (pages, heads + extra, page, hd), dtype=torch.uint8).to(DEV) for _ in range(2))
    ke, ve = (torch.randint(0, 255, (pages, heads + extra, page), dtype=torch.uint8).to(DEV) for _ in range(2))
    cut = lambda t: t[:, :heads]  # noqa: E731
    return cut(k).view(E4M3), cut(v).view(E4M3), cut(ke), cut(ve)


def bits(t):
    return t.view(torch.uint8).cpu()


def source(T, heads, hd, g, dtype):
    x = torch.randn(T, 2, heads, hd, generator=g) * torch.exp2(torch.randint(-20, 20, (T, 2, heads, 1), generator=g).float())
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hd,page", [(1, 16, 1), (3, 32, 7), (12, 64, 16), (5, 80, 12), (2, 112, 32), (40, 128, 16), (2, 256, 5)])
@pytest.mark.parametrize("strided", [False, True])
def test_write_and_read(heads, hd, page, dtype, strided):
    g = torch.Generator().manual_seed(hd + page)
    items, width = 3, 4
    lens = [1, 2 * page + 1 if page > 1 else 3, width * page]
    table = torch.randperm(items * width + 2, generator=g)[:items * width].int().view(items, width)
    item = torch.tensor([r for r, n in enumerate(lens) for _ in range(n)] + [-1, 0]).int()
    position = torch.tensor([p for n in lens for p in range(n)] + [0, -1]).int()
    T = len(item)
    kv = source(T, heads, hd, g, dtype)
    kv[0, 0, 0] = 0
    flat = kv.view(T, 2 * heads * hd).to(DEV)
    k_src, v_src = flat[:, :heads * hd], flat[:, heads * hd:]
    torch.manual_seed(1)
    cache = pools(items * width + 2, heads, page, hd, strided)
    before = [bits(c).clone() for c in cache]
    put = lambda t: t.to(DEV)  # noqa: E731
    K.quant_kv_write(*cache, k_src, v_src, put(item), put(position), put(table), page)
    for n, (c, e) in enumerate(((0, 2), (1, 3))):
        want_c, want_e = before[c].clone(), before[e].clone()
        entry, exponent = small(kv[:, n])
        for t in range(T - 2):
            at = (int(table[item[t], position[t] // page]), slice(None), int(position[t] % page))
            want_c[at], want_e[at] = entry[t], exponent[t]
        assert torch.equal(bits(cache[c]), want_c) and torch.equal(bits(cache[e]), want_e)
    back = K.quant_kv_read(*cache, put(item), put(position), put(table), dtype)
    for n in range(2):
        entry, exponent = small(kv[:, n])
        want = (entry.view(E4M3).double() * torch.exp2(exponent.double() - 127)[..., None]).to(dtype)
        want[T - 2:] = 0
        assert back[n].dtype == dtype and torch.equal(back[n].cpu(), want.view(T, heads * hd))


def test_values_at_their_ends():
    """Zeros, the smallest numbers, the largest, infinities and NaN, and largest values on both sides of 448 times a power of two."""
    hd = 16
    rows = [torch.zeros(hd), torch.full((hd,), 1e-45), torch.full((hd,), 2.0 ** -126), torch.linspace(-3.4e38, 3.4e38, hd),
            torch.tensor([math.inf] + [1.0] * (hd - 1)), torch.tensor([math.nan, -math.inf] + [3.0] * (hd - 2)), torch.full((hd,), math.nan)]
    for top in (448.0, math.nextafter(448.0, 1e9), 447.0, 7.0, 7.5, 1.75, 1.7500001, 224.0):
        rows.append(torch.linspace(-top, top, hd))
    for step in (2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 2.0 ** -6, 0.9 * 2.0 ** -6):          # beside 448: what is stored with fewer bits, ties
        rows.append(torch.cat([torch.tensor([448.0]), step * torch.arange(1, hd).float()]))
    x = torch.stack(rows)
    T = len(x)
    cache = pools(T, 1, 1, hd, False)
    table = torch.arange(T).int().view(1, T).to(DEV)
    item, position = torch.zeros(T).int().to(DEV), torch.arange(T).int().to(DEV)
    K.quant_kv_write(*cache, x.to(DEV), (-x).to(DEV), item, position, table, 1)
    for c, e, src in ((0, 2, x), (1, 3, -x)):
        entry, exponent = small(src)
        got, want = bits(cache[c]).view(T, hd), entry
        nan = (want & 0x7f) == 0x7f
        assert torch.equal((got & 0x7f) == 0x7f, nan) and torch.equal(got[~nan], want[~nan])
        assert torch.equal(bits(cache[e]).view(T), exponent)


def test_errors_within_half_a_step():
    """Of an element down to 2^-14 of its head's largest at most 2^-4 of itself."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(64, 4 * 128, generator=g) * torch.exp(2 * torch.randn(64, 4 * 128, generator=g))
    cache = pools(64, 4, 1, 128, False)
    ids = [t.to(DEV) for t in (torch.arange(64).int(), torch.zeros(64).int(), torch.arange(64).int().view(64, 1))]
    K.quant_kv_write(*cache, x.to(DEV), x.to(DEV), *ids, 1)
    got = K.quant_kv_read(*cache, *ids, torch.float32)[1].cpu().double()
    heads = x.double().view(64, 4, 128)
    large = (heads.abs() >= heads.abs().amax(-1, keepdim=True) * 2.0 ** -14).view(64, -1)
    assert ((got - x.double()).abs()[large] <= 2.0 ** -4 * x.double().abs()[large]).all()


def test_pages_that_are_none_are_left_out():
    cache = pools(2, 1, 4, 16, False)
    before = [bits(c).clone() for c in cache]
    table = torch.tensor([[0, -1, 7], [2, 1, 1 << 30]], dtype=torch.int32, device=DEV)
    item = torch.tensor([0, 0, 1, 1, 1, 2, 5], dtype=torch.int32, device=DEV)
    position = torch.tensor([4, 8, 0, 8, 12, 0, 0], dtype=torch.int32, device=DEV)      # (12: past the table's width)
    x = torch.ones(7, 16, device=DEV)
    K.quant_kv_write(*cache, x, x, item, position, table, 4)
    assert all(torch.equal(bits(c), b) for c, b in zip(cache, before))
    k, v = K.quant_kv_read(*cache, item, position, table, torch.bfloat16)
    assert not k.any() and not v.any()
    K.quant_kv_write(*cache, x[:0], x[:0], item[:0], position[:0], table, 4)
    assert K.quant_kv_read(*cache, item[:0], position[:0], table, torch.float32)[0].shape == (0, 16)


def test_recorded():
    g = torch.Generator().manual_seed(5)
    cache = pools(6, 4, 16, 64, False)
    table = torch.randperm(6, generator=g).int().view(2, 3).to(DEV)
    x = torch.zeros(4, 512, device=DEV, dtype=torch.bfloat16)
    item, position = torch.tensor([0, 0, 1, 1]).int().to(DEV), torch.zeros(4).int().to(DEV)
    call = lambda: (K.quant_kv_write(*cache, x[:, :256], x[:, 256:], item, position, table, 16),  # noqa: E731
                    K.quant_kv_read(*cache, item, position, table, torch.bfloat16))[1]
    position.copy_(torch.tensor([0, 1, 2, 3]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call()
    torch.cuda.synchronize()
    for n in range(3):
        a = torch.randn(4, 512, generator=g).bfloat16()
        x.copy_(a)
        position.copy_(torch.tensor([5 * n, 40 - n, 17 + n, n]))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            entry, exponent = small(a.view(4, 2, 4, 64)[:, i])
            want = (entry.view(E4M3).double() * torch.exp2(exponent.double() - 127)[..., None]).bfloat16().view(4, 256)
            assert torch.equal(got[i].cpu(), want)


def test_refusals():
    cache = pools(2, 2, 4, 32, False)
    k, v, ke, ve = cache
    x = torch.zeros(3, 64, device=DEV)
    i = torch.zeros(3, dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    K.quant_kv_write(*cache, x, x, i, torch.arange(3, device=DEV).int(), table, 4)
    odd = torch.zeros(3, 65, device=DEV)[:, 1:]
    for bad in (lambda: K.quant_kv_write(k.view(torch.uint8), v, ke, ve, x, x, i, i, table, 4), lambda: K.quant_kv_write(k, v, ke.int(), ve, x, x, i, i, table, 4),
                lambda: K.quant_kv_write(*cache, x.half(), x.half(), i, i, table, 4), lambda: K.quant_kv_write(*cache, x, x, i, i, table, 5),
                lambda: K.quant_kv_write(*cache, x[:, :32], x, i, i, table, 4), lambda: K.quant_kv_write(*cache, odd, odd, i, i, table, 4),
                lambda: K.quant_kv_write(*cache, x, x, i[:2], i, table, 4), lambda: K.quant_kv_write(*cache, x, x, i, i, table[0], 4),
                lambda: K.quant_kv_write(*cache, x, x, i.cpu(), i, table, 4), lambda: K.quant_kv_read(*cache, i, i, table.long(), torch.float32),
                lambda: K.quant_kv_write(k.transpose(1, 2), v.transpose(1, 2), ke, ve, x, x, i, i, table, 4),
                lambda: K.quant_kv_write(*(c[..., :24] if c.dim() == 4 else c for c in cache), x[:, :48], x[:, :48], i, i, table, 4)):
        with pytest.raises((K.KernelError, TypeError)):
            bad()
    with pytest.raises(TypeError):
        K.quant_kv_read(*cache, i, i, table, torch.float16)
