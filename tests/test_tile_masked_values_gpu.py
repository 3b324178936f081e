"""What a row does not read does not reach it, whatever lies there: entries of its own pages before its own keys begin, values that only other rows
of its tile or group see.  And what it does read arrives, infinities as infinities."""
import math

import pytest
import torch

from swifttransformer_amd.ops import kernels as K
from test_tile_attention_gpu import DEV, Pool, compare, ints, queries, reference, shared_batch

pytestmark = pytest.mark.gpu

SHAPES = [(4, 2, 64, 16), (4, 2, 64, 12), (6, 2, 80, 16), (3, 1, 256, 16), (8, 2, 96, 7), (8, 2, 128, 32)]


def spoil(pool, page, rows):
    """NaN in entries of a page."""
    if pool.quant:
        pool.k[page, :, rows], pool.v[page, :, rows], pool.ke[page, :, rows], pool.ve[page, :, rows] = 0x7f, 0xff, 255, 255
    else:
        pool.k[page, :, rows], pool.v[page, :, rows] = math.nan, math.nan


@pytest.mark.parametrize("waves", [1, 4])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_own_pages_before_the_own_keys(heads, kv, hd, page, dtype, quant, waves):
    """A prefix that ends inside a page: only the first row of the group holds that part of it."""
    g = torch.Generator().manual_seed(hd + page)
    pool, table, lens, start, shared, off, q = shared_batch([(53, 3), (6, 2)], [1, 17, 40], heads, kv, hd, page, dtype, quant, g, alone=(12,))
    n = len(lens)
    entries = [pool.entries(table, t, lens[t]) for t in range(n)]
    for i in range(len(off) - 1):
        for r in shared[off[i] + 1:off[i + 1]]:
            assert start[r] % page
            spoil(pool, int(table[r, start[r] // page]), slice(0, start[r] % page))
    units = torch.cuda.get_device_properties(0).multi_processor_count
    T = n if waves == 4 else -(-4 * units // kv) + 3                # batch row t is request t % n once more
    listed, at = [], [0]
    for i in range(len(off) - 1):
        listed += [t for r in shared[off[i]:off[i + 1]] for t in range(r, T, n)]
        at.append(len(listed))
    assert K.tile_waves(T * kv, table.shape[1] * page, units) == waves
    q = queries(T, heads, hd, dtype, g)
    k, v, ke, ve = pool.put()
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    got = K.attention_shared(q.to(DEV), k, v, put([t % n for t in range(T)]), put([lens[t % n] - 1 for t in range(T)]), table.to(DEV), heads, hd ** -0.5,
                             put([start[t % n] for t in range(T)]), put(listed), put(at), k_exp=ke, v_exp=ve, shared_splits=2, own_splits=1).cpu()
    for t in list(range(0, T, 1 if waves == 4 else 11)) + [T - 1]:
        want, bound = reference(q[t], *entries[t % n], heads, hd ** -0.5)
        compare(got[t], want, bound)


def compare_with_holes(got, q, k, v, heads, scale):
    """A row of results over keys of which some values are not finite: the others as if there were none, these as the sum gives them (p > 0)."""
    bad = ~torch.isfinite(v)                                       # [n, kv, hd]
    group = heads // v.shape[1]
    sums = torch.where(bad, v, torch.zeros_like(v)).sum(0)         # inf, -inf, NaN or 0
    want, bound = reference(q, k, torch.where(bad, torch.zeros_like(v), v), heads, scale)
    holes = bad.any(0).repeat_interleave(group, 0).reshape(-1)
    what = sums.repeat_interleave(group, 0).reshape(-1)
    got = got.cpu().double()
    compare(torch.where(holes, torch.zeros_like(got), got), torch.where(holes, torch.zeros_like(want), want), bound)
    assert torch.equal(got[holes].isnan(), what[holes].isnan())
    some = ~what[holes].isnan()
    assert torch.equal(got[holes][some], what[holes][some])


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_rows_of_a_portion_before_a_value_that_is_no_number(heads, kv, hd, page, dtype, splits):
    g = torch.Generator().manual_seed(hd)
    cached, T = 21, 70
    table = torch.full((1, -(-(cached + T) // page)), -1, dtype=torch.int32)
    pool = Pool(table.shape[1] + 1, kv, page, hd, dtype, True, g)
    pool.fill(table, 0, 0, cached + T)
    for key, head, dim in ((cached + 3, 0, 5), (cached + 18, kv - 1, 11), (cached + 18, kv - 1, hd - 1), (cached + 40, 0, 0), (cached + 69, 0, 8)):
        pool.v[int(table[0, key // page]), head, key % page, dim] = 0x7f if dim else 0xff
    q = queries(T, heads, hd, dtype, g)
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    got = K.attention_prefill_quant(q.to(DEV), *pool.put(), put([0, 0]), put([0, 64]), put([0]), put([cached]), put([T]), table.to(DEV), heads, hd ** -0.5,
                                    num_splits=splits)
    k, v = pool.entries(table, 0, cached + T)
    for t in range(T):
        compare_with_holes(got[t], q[t], k[:cached + t + 1], v[:cached + t + 1], heads, hd ** -0.5)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_rows_of_a_group_that_end_before_a_value_that_is_not_finite(heads, kv, hd, page, dtype, quant):
    """Rows whose positions lie in the prefix, before and behind values of it that are NaN and infinite; requests that share all of it."""
    g = torch.Generator().manual_seed(hd)
    prefix = 75
    table = torch.full((1, -(-90 // page)), -1, dtype=torch.int32)
    pool = Pool(table.shape[1] + 1, kv, page, hd, dtype, quant, g)
    pool.fill(table, 0, 0, 90)
    for key, dim, bits, value in ((20, 3, 0x7f, math.inf), (37, 3, 0x7f, math.inf), (38, 9, 0xff, -math.inf), (64, 12, 0x7f, math.nan), (64, 3, 0x7f, -math.inf),
                                  (74, 1, 0x7f, math.inf)):
        pool.v[int(table[0, key // page]), kv - 1, key % page, dim] = bits if quant else value
    ends = [1, 19, 20, 21, 36, 37, 38, 39, 60, 64, 65, 74, 75, 76, 90]
    T = len(ends)
    q = queries(T, heads, hd, dtype, g)
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    on = pool.put()
    k, v = pool.entries(table, 0, 90)
    for splits in (1, 2):
        got = K.attention_shared(q.to(DEV), on[0], on[1], put([0] * T), put([n - 1 for n in ends]), table.to(DEV), heads, hd ** -0.5, put([prefix] * T),
                                 put(range(T)), put([0, T]), k_exp=on[2], v_exp=on[3], shared_splits=splits, own_splits=1)
        for t, n in enumerate(ends):
            compare_with_holes(got[t], q[t], k[:n], v[:n], heads, hd ** -0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("waves", [1, 4])
def test_a_last_value_that_is_infinite(dtype, waves):
    """(What lies behind the last key of a block stands for nothing, not for that key once more.)"""
    g = torch.Generator().manual_seed(2)
    heads, kv, hd, page, n = 2, 1, 64, 16, 45
    table = torch.full((1, 3), -1, dtype=torch.int32)
    pool = Pool(4, kv, page, hd, dtype, False, g)
    pool.fill(table, 0, 0, n)
    pool.v[int(table[0, 44 // page]), 0, 44 % page, 7] = math.inf
    T = 1 if waves == 4 else 4 * torch.cuda.get_device_properties(0).multi_processor_count
    q = queries(1, heads, hd, dtype, g)
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    on = pool.put()
    k, v = pool.entries(table, 0, n)
    for start in (16, 33):
        got = K.attention_shared(q.expand(T, -1).contiguous().to(DEV), on[0], on[1], put([0] * T), put([n - 1] * T), table.to(DEV), heads, 0.125, put([start] * T),
                                 put(range(T)), put([0, T]), shared_splits=1, own_splits=1)
        compare_with_holes(got[0], q[0], k, v, heads, 0.125)
        compare_with_holes(got[T - 1], q[0], k, v, heads, 0.125)


@pytest.mark.parametrize("quant", [False, True])
def test_rows_with_a_prefix_that_no_group_lists(quant):
    """They read their own keys from where these begin, and nothing that the workspace held before."""
    g = torch.Generator().manual_seed(6)
    batch = shared_batch([(70, 4), (33, 3)], [20, 5], 4, 2, 64, 16, torch.float32, quant, g)
    pool, table, lens, start, shared, off, q = batch
    left_out = [shared[1], shared[6]]
    listed = [-1 if r in left_out else r for r in shared]
    k, v, ke, ve = pool.put()
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    n = len(lens)
    for rows, at in ((listed, off), (listed + [left_out[0]], off), ([left_out[1]] + listed, [1 + o for o in off]), (listed + [-1] * 300, [0, 4, 307])):
        # (lists that go on behind the last group, or begin before the first one, and a long one)
        workspace = torch.full((n * 4 * 4 * 66,), math.nan, device=DEV)
        got = K.attention_shared(q.to(DEV), k, v, put(range(n)), put([m - 1 for m in lens]), table.to(DEV), 4, 0.125, put(start), put(rows), put(at), k_exp=ke,
                                 v_exp=ve, shared_splits=2, own_splits=2, workspace=workspace)
        for t in range(n):
            kk, vv = pool.entries(table, t, lens[t])
            first = start[t] if t in left_out else 0
            compare(got[t], *reference(q[t], kk[first:], vv[first:], 4, 0.125))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 80, 128])
def test_rows_that_see_nothing_beside_rows_that_see_all(hd, dtype, quant):
    """Padding rows, and rows without a prefix, that a group lists: whatever their queries are, they get zeros (their own keys only), the others their results."""
    g = torch.Generator().manual_seed(hd)
    batch = shared_batch([(150, 9), (33, 4)], [20, 5, 1], 4, 2, hd, 16, dtype, quant, g)
    pool, table, lens, start, shared, off, q = batch
    k, v, ke, ve = pool.put()
    n = len(lens)
    item = list(range(n))
    padding, plain = [shared[0], shared[4], shared[12]], shared[6]
    for r in padding:
        item[r] = -1
        q[r] = math.nan
    start = list(start)
    start[plain] = 0
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    for a, b in ((1, 1), (3, 2)):
        got = K.attention_shared(q.to(DEV), k, v, put(item), put([m - 1 for m in lens]), table.to(DEV), 4, 0.125, put(start), put(shared), put(off), k_exp=ke,
                                 v_exp=ve, shared_splits=a, own_splits=b)
        for t in range(n):
            if t in padding:
                assert bool((got[t] == 0).all())
            else:
                compare(got[t], *reference(q[t], *pool.entries(table, t, lens[t]), 4, 0.125))
