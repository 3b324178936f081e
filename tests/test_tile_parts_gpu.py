"""Attention by tiles whose keys are split into many parts, up to the 64 that a row may have, at heads that do not fill the lanes which join them."""
import pytest
import torch

from swifttransformer_amd.ops import kernels as K
from test_tile_attention_gpu import DEV, E4M3, compare, ints, queries, reference

pytestmark = pytest.mark.gpu


def paged(n, kv, hd, page, dtype, quant, g):
    """One request's entries in pages of any order: (table [1, pages], arguments of the cache, keys and values [n, kv, hd] in 64 bits)."""
    pages = -(-n // page)
    order = torch.randperm(pages, generator=g)
    x = torch.randn(2, pages * page, kv, hd, generator=g)
    held = (40 * x).to(E4M3) if quant else x.to(dtype)
    exps = torch.full((2, pages, kv, page), 121, dtype=torch.uint8)
    pool = torch.zeros((2, pages, kv, page, hd), dtype=torch.uint8 if quant else dtype)
    pool[:, order] = (held.view(torch.uint8) if quant else held).view(2, pages, page, kv, hd).permute(0, 1, 3, 2, 4).contiguous()
    on = pool.to(DEV)
    cache = [on[0].view(E4M3), on[1].view(E4M3), exps[0].to(DEV), exps[1].to(DEV)] if quant else [on[0], on[1], None, None]
    values = held.double()[:, :n] * (2.0 ** -6 if quant else 1.0)
    return order.int().view(1, pages), cache, values[0], values[1]


def check(got, q, k, v, lens, heads, scale):
    want = [reference(q[t], k[:n], v[:n], heads, scale) for t, n in enumerate(lens)]
    compare(got, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))


HEADS = [(2, 1, 16), (2, 1, 32), (3, 1, 48), (4, 2, 80), (4, 2, 96), (1, 1, 112), (2, 1, 128), (2, 2, 144), (1, 1, 160), (1, 1, 208)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd", HEADS)
def test_single_rows(heads, kv, hd, dtype):
    g = torch.Generator().manual_seed(hd)
    lens = [2061, 2048, 40]
    table, cache, k, v = paged(max(lens), kv, hd, 16, dtype, True, g)
    q = queries(len(lens), heads, hd, dtype, g)
    for splits in (16, 17, 32, 33, 64):
        got = K.attention_rows_quant(q.to(DEV), *cache, torch.zeros(3, dtype=torch.int32, device=DEV), ints([n - 1 for n in lens]).to(DEV), table.to(DEV), heads,
                                     hd ** -0.5, num_splits=splits)
        check(got, q, k, v, lens, heads, hd ** -0.5)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd", HEADS[::2] + HEADS[3::4])
def test_behind_prefixes(heads, kv, hd, dtype, quant):
    g = torch.Generator().manual_seed(hd + 1)
    prefix, lens = 1100, [1100 + 1060, 1100 + 3, 700]
    table, cache, k, v = paged(max(lens), kv, hd, 16, dtype, quant, g)
    q = queries(len(lens), heads, hd, dtype, g)
    n = torch.zeros(3, dtype=torch.int32, device=DEV)
    for shared, own in ((16, 1), (1, 16), (31, 2), (32, 32), (17, 40)):
        got = K.attention_shared(q.to(DEV), cache[0], cache[1], n, ints([m - 1 for m in lens]).to(DEV), table.to(DEV), heads, hd ** -0.5, n + prefix,
                                 ints([0, 1, 2]).to(DEV), ints([0, 3]).to(DEV), k_exp=cache[2], v_exp=cache[3], shared_splits=shared, own_splits=own)
        check(got, q, k, v, lens, heads, hd ** -0.5)


@pytest.mark.parametrize("heads,kv,hd,n", [(8, 8, 80, 4865), (8, 8, 80, 8201), (4, 1, 16, 9001), (24, 8, 96, 8193)])
def test_parts_by_the_rule(heads, kv, hd, n):
    g = torch.Generator().manual_seed(n)
    units = torch.cuda.get_device_properties(0).multi_processor_count
    assert K.tile_splits(kv, n, units) > 16
    table, cache, k, v = paged(n, kv, hd, 16, torch.float32, True, g)
    q = queries(1, heads, hd, torch.float32, g)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = K.attention_rows_quant(q.to(DEV), *cache, zero, zero + (n - 1), table.to(DEV), heads, hd ** -0.5)
    check(got, q, k, v, [n], heads, hd ** -0.5)
    prefix = n - n // 3
    got = K.attention_shared(q.to(DEV), cache[0], cache[1], zero, zero + (n - 1), table.to(DEV), heads, hd ** -0.5, zero + prefix, zero, ints([0, 1]).to(DEV),
                             k_exp=cache[2], v_exp=cache[3])
    check(got, q, k, v, [n], heads, hd ** -0.5)
