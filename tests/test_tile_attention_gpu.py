"""Attention over the 8-bit cache (single tokens, prompt portions) and over shared prefixes, against 64-bit arithmetic on the values that the cache
holds: head layouts, sizes and pages of every kind, lengths around the blocks of 32 keys and the four waves' rounds of them, splits, rows
without keys, entries that no row sees filled with NaN.

The bound of an element: with A = sum_j p_j |v_j|, bfloat16 rounds the probabilities and the result, 2^-8 each, of A at most; a score of float sums of
d products is off by (d + 4) 2^-24 sum |q_i k_i| scale, a probability by that much of itself and its normaliser again; sums over n keys by 2^-24 n."""
import math

import pytest
import torch

from swifttransformer_amd.ops import kernels as K

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


class Pool:
    """A paged cache on the host with NaN wherever nothing is written; ``put`` sends it to the GPU."""

    def __init__(self, pages, heads, page, hd, dtype, quant, g):
        self.page, self.quant, self.dtype, self.g = page, quant, dtype, g
        shape = (pages, heads, page, hd)
        if quant:
            self.k, self.v = (torch.full(shape, 0x7f, dtype=torch.uint8) for _ in range(2))
            self.ke, self.ve = (torch.full(shape[:3], 255, dtype=torch.uint8) for _ in range(2))
        else:
            self.k, self.v = (torch.full(shape, math.nan, dtype=dtype) for _ in range(2))
        self.order = torch.randperm(pages, generator=g).tolist()

    def fill(self, table, row, begin, end):
        """Random entries at positions [begin, end) of a table's row, whose pages it names (as far as they are not)."""
        heads, hd = self.k.shape[1], self.k.shape[3]
        for p in range(begin, end):
            if table[row, p // self.page] < 0:
                table[row, p // self.page] = self.order.pop()
            at = (int(table[row, p // self.page]), slice(None), p % self.page)
            if self.quant:
                for c, e in ((self.k, self.ke), (self.v, self.ve)):
                    x = torch.randn(heads, hd, generator=self.g) * 64
                    c[at] = x.to(E4M3).view(torch.uint8)
                    e[at] = torch.randint(120, 123, (heads,), generator=self.g).to(torch.uint8)
            else:
                self.k[at], self.v[at] = (torch.randn(heads, hd, generator=self.g).to(self.dtype) for _ in range(2))

    def entries(self, table, row, n):
        """Keys and values [n, heads, hd] in 64 bits."""
        at = torch.arange(n)
        page, r = table[row, at // self.page].long(), at % self.page
        if not self.quant:
            return self.k[page, :, r].double(), self.v[page, :, r].double()
        return tuple(c[page, :, r].view(E4M3).double() * torch.exp2(e[page, :, r].double() - 127)[..., None] for c, e in ((self.k, self.ke), (self.v, self.ve)))

    def put(self):
        if not self.quant:
            return self.k.to(DEV), self.v.to(DEV), None, None
        return self.k.to(DEV).view(E4M3), self.v.to(DEV).view(E4M3), self.ke.to(DEV), self.ve.to(DEV)


def reference(q, k, v, heads, scale):
    """(result, bound) of one query row [heads * hd] over keys [n, kv heads, hd]."""
    n, nkv, hd = k.shape
    if n == 0:
        return torch.zeros(heads * hd, dtype=torch.float64), torch.zeros(heads * hd, dtype=torch.float64)
    qh = q.double().view(nkv, heads // nkv, hd)
    s = torch.einsum("hgd,nhd->hgn", qh, k) * scale
    p = torch.softmax(s, -1)
    size = torch.einsum("hgd,nhd->hgn", qh.abs(), k.abs()).amax(-1, keepdim=True) * scale
    o = torch.einsum("hgn,nhd->hgd", p, v)
    a = torch.einsum("hgn,nhd->hgd", p, v.abs())
    off = 2 * (hd + 8) * 2.0 ** -24 * size + (2 * n + 64) * 2.0 ** -24
    if q.dtype == torch.bfloat16:
        off = off + 2 * 2.0 ** -8
    return o.reshape(-1), (a * off).reshape(-1)


def queries(T, heads, hd, dtype, g):
    return (1.5 * torch.randn(T, heads * hd, generator=g)).to(dtype)


def compare(got, want, bound):
    off = (got.cpu().double() - want).abs()
    assert bool((off <= bound).all()), f"off by {off.max().item()}, {(off / bound.clamp(min=1e-30)).max().item()} of the bound"


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


SHAPES = [(4, 4, 64, 16), (4, 4, 16, 1), (6, 2, 32, 7), (8, 8, 80, 16), (12, 3, 96, 12), (8, 2, 128, 16), (20, 1, 64, 32), (5, 5, 112, 16), (6, 2, 144, 8),
          (3, 1, 256, 16), (64, 1, 48, 16), (17, 1, 128, 5)]


@pytest.mark.parametrize("splits", [0, 1, 5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_single_tokens_quant(heads, kv, hd, page, dtype, splits):
    g = torch.Generator().manual_seed(heads + hd)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 161, 300, 0]
    width = -(-max(lens) // page) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    pool = Pool(sum(-(-n // page) for n in lens) + 2, kv, page, hd, dtype, True, g)
    for r, n in enumerate(lens):
        pool.fill(table, r, 0, n)
    T = len(lens) + 1
    wide = queries(T, heads + 1, hd, dtype, g).to(DEV)
    q = wide[:, :heads * hd]                                     # rows with a stride
    item = ints(list(range(len(lens))) + [-1])
    position = ints([n - 1 for n in lens] + [5])
    scale = hd ** -0.5
    k, v, ke, ve = pool.put()
    got = K.attention_rows_quant(q, k, v, ke, ve, item.to(DEV), position.to(DEV), table.to(DEV), heads, scale, num_splits=splits)
    want = [reference(q[t].cpu(), *pool.entries(table, t, n), heads, scale) for t, n in enumerate(lens + [0]) if t < len(lens)] + \
           [reference(q[0].cpu(), torch.zeros(0, kv, hd).double(), torch.zeros(0, kv, hd).double(), heads, scale)]
    compare(got, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))


@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_many_short_rows(heads, kv, hd, page, dtype, splits):
    """So many rows that each is a wave's own: several tokens of the same requests, padding rows between."""
    g = torch.Generator().manual_seed(heads * hd)
    lens = [1, 9, 33, 64, 70]
    table = torch.full((len(lens), -(-max(lens) // page) + 1), -1, dtype=torch.int32)
    pool = Pool(table.numel() + 2, kv, page, hd, dtype, True, g)
    for r, n in enumerate(lens):
        pool.fill(table, r, 0, n)
    T = -(-4 * torch.cuda.get_device_properties(0).multi_processor_count // (kv * splits)) + 3
    item = torch.randint(-1, len(lens), (T,), generator=g, dtype=torch.int32)
    position = torch.tensor([int(torch.randint(0, lens[i], (1,), generator=g)) if i >= 0 else 3 for i in item.tolist()], dtype=torch.int32)
    q = queries(T, heads, hd, dtype, g)
    k, v, ke, ve = pool.put()
    assert K.tile_waves(T * kv * splits, table.shape[1] * page, torch.cuda.get_device_properties(0).multi_processor_count) == 1
    got = K.attention_rows_quant(q.to(DEV), k, v, ke, ve, item.to(DEV), position.to(DEV), table.to(DEV), heads, hd ** -0.5, num_splits=splits).cpu()
    for t in list(range(0, T, 7)) + [T - 2, T - 1]:
        n = int(position[t]) + 1 if item[t] >= 0 else 0
        want, bound = reference(q[t], *pool.entries(table, int(item[t]), n), heads, hd ** -0.5)
        compare(got[t], want, bound)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_many_short_rows_behind_prefixes(heads, kv, hd, page, dtype, quant):
    g = torch.Generator().manual_seed(heads + 3 * hd)
    pool, table, lens, start, shared, off, q = shared_batch([(50, 3), (19, 2)], [1, 17, 40], heads, kv, hd, page, dtype, quant, g, alone=(12,))
    n = len(lens)
    T = -(-4 * torch.cuda.get_device_properties(0).multi_processor_count // kv) + 3
    rows = [[t for t in range(T) if t % n == r] for r in range(n)]                 # batch row t is request t % n once more
    listed, at = [], [0]
    for i in range(len(off) - 1):
        listed += [t for r in shared[off[i]:off[i + 1]] for t in rows[r]]
        at.append(len(listed))
    item, position = ints([t % n for t in range(T)]), ints([lens[t % n] - 1 for t in range(T)])
    q = queries(T, heads, hd, dtype, g)
    k, v, ke, ve = pool.put()
    put = lambda x: x.to(DEV)  # noqa: E731
    got = K.attention_shared(put(q), k, v, put(item), put(position), put(table), heads, hd ** -0.5, put(ints([start[t % n] for t in range(T)])), put(ints(listed)),
                             put(ints(at)), k_exp=ke, v_exp=ve, shared_splits=2, own_splits=1).cpu()
    for t in list(range(0, T, 11)) + [T - 1]:
        want, bound = reference(q[t], *pool.entries(table, t % n, lens[t % n]), heads, hd ** -0.5)
        compare(got[t], want, bound)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 2.0])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_of_any_size_and_sign(dtype, quant, scale):
    g = torch.Generator().manual_seed(12)
    batch = shared_batch([(37, 3)], [1, 40, 77], 4, 2, 80, 16, dtype, quant, g)
    pool, table, lens, _, _, _, q = batch
    got = run_shared(batch, 4, scale, shared_splits=2, own_splits=2)
    for t, n in enumerate(lens):
        k, v = pool.entries(table, t, n)
        want, bound = reference(q[t] if scale >= 0 else -q[t], k, v, 4, abs(scale))
        compare(got[t], want, bound)


def test_some_rows_only():
    g = torch.Generator().manual_seed(1)
    table = torch.full((6, 20), -1, dtype=torch.int32)
    pool = Pool(80, 2, 16, 64, torch.bfloat16, True, g)
    for r in range(6):
        pool.fill(table, r, 0, 40 * r + 3)
    q = queries(6, 4, 64, torch.bfloat16, g)
    rows = ints([4, -1, 0, 5, -1])
    for splits in (1, 3):
        out = torch.full((6, 256), 7.0, dtype=torch.bfloat16, device=DEV)
        K.attention_rows_quant(q.to(DEV), *pool.put(), ints(range(6)).to(DEV), ints([40 * r + 2 for r in range(6)]).to(DEV), table.to(DEV), 4, 0.125,
                               row_ids=rows.to(DEV), out=out, num_splits=splits)
        for r in (0, 4, 5):
            want, bound = reference(q[r], *pool.entries(table, r, 40 * r + 3), 4, 0.125)
            compare(out[r], want, bound)
        assert bool((out[[1, 2, 3]] == 7).all())


def test_pages_that_are_none_hold_no_keys():
    g = torch.Generator().manual_seed(2)
    table = torch.full((2, 9), -1, dtype=torch.int32)
    pool = Pool(20, 1, 16, 64, torch.float32, True, g)
    pool.fill(table, 0, 0, 140)
    pool.fill(table, 1, 0, 20)
    q = queries(2, 2, 64, torch.float32, g)
    k, v = pool.entries(table, 0, 140)
    bad = table.clone()
    bad[0, 2], bad[0, 4], bad[0, 8] = -1, 20, 1 << 30
    bad[1] = -5
    seen = torch.ones(140, dtype=torch.bool)
    seen[32:48] = seen[64:80] = seen[128:] = False
    for splits in (1, 4):
        got = K.attention_rows_quant(q.to(DEV), *pool.put(), ints([0, 1]).to(DEV), ints([139, 19]).to(DEV), bad.to(DEV), 2, 0.125, num_splits=splits)
        want, bound = reference(q[0], k[seen], v[seen], 2, 0.125)
        compare(got[0], want, bound)
        assert not got[1].any()
    # positions past the table end there, items past it have no keys
    got = K.attention_rows_quant(q.to(DEV), *pool.put(), ints([0, 7]).to(DEV), ints([10 ** 9, 19]).to(DEV), table[:, :3].contiguous().to(DEV), 2, 0.125, num_splits=2)
    want, bound = reference(q[0], k[:48], v[:48], 2, 0.125)
    compare(got[0], want, bound)
    assert not got[1].any()


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_portions_quant(heads, kv, hd, page, dtype, splits):
    g = torch.Generator().manual_seed(hd)
    items = [(0, 1), (0, 65), (37, 40), (100, 131), (5, 0)]       # (cached before, tokens)
    T = sum(n for _, n in items) + 2
    width = -(-300 // page)
    table = torch.full((len(items), width), -1, dtype=torch.int32)
    pool = Pool(sum(-(-(a + n) // page) for a, n in items) + 1, kv, page, hd, dtype, True, g)
    for r, (a, n) in enumerate(items):
        pool.fill(table, r, 0, a + n)
    q = queries(T, heads, hd, dtype, g)
    off, at = [], 1                                               # (batch rows 0 and the last belong to no tile)
    for _, n in items:
        off.append(at)
        at += n
    tiles = [(-1, 0)] + [(r, q0) for r, (_, n) in enumerate(items) for q0 in range(0, n, 64)]
    out = torch.full((T, heads * hd), 3.0, dtype=dtype, device=DEV)
    put = lambda v: ints(v).to(DEV)  # noqa: E731
    scale = hd ** -0.5
    K.attention_prefill_quant(q.to(DEV), *pool.put(), put([r for r, _ in tiles]), put([q0 for _, q0 in tiles]), put(off), put([a for a, _ in items]),
                              put([n for _, n in items]), table.to(DEV), heads, scale, out=out, num_splits=splits, max_keys=300)
    want, bound = torch.full((T, heads * hd), 3.0, dtype=torch.float64), torch.zeros(T, heads * hd, dtype=torch.float64)
    for r, (a, n) in enumerate(items):
        k, v = pool.entries(table, r, a + n)
        for i in range(n):
            want[off[r] + i], bound[off[r] + i] = reference(q[off[r] + i], k[:a + i + 1], v[:a + i + 1], heads, scale)
    compare(out, want, bound)


def shared_batch(groups, own, heads, kv, hd, page, dtype, quant, g, alone=(), shift=0):
    """Requests of groups (prefix length, requests) with their own entries behind; a prefix that ends inside a page is copied there.  Returns
    (pool, table, lens, row_start, shared_rows, group_off, q)."""
    n = sum(c for _, c in groups) + len(alone)
    lens_own = [own[i % len(own)] for i in range(n - len(alone))] + list(alone)
    longest = max([p for p, _ in groups] + [0]) + max(lens_own) + page
    table = torch.full((n, -(-longest // page)), -1, dtype=torch.int32)
    pool = Pool(n * table.shape[1] + 4, kv, page, hd, dtype, quant, g)
    order = torch.randperm(n, generator=g).tolist()              # batch rows in any order
    lens, start, shared, off = [0] * n, [0] * n, [], [0]
    at = 0
    for prefix, count in groups:
        rows = [order[at + i] for i in range(count)]
        pool.fill(table, rows[0], 0, prefix)
        for r in rows[1:]:
            whole = prefix // page
            table[r, :whole] = table[rows[0], :whole]
            if prefix % page:
                table[r, whole] = pool.order.pop()
                a, b = int(table[rows[0], whole]), int(table[r, whole])
                pool.k[b, :, :prefix % page], pool.v[b, :, :prefix % page] = pool.k[a, :, :prefix % page], pool.v[a, :, :prefix % page]
                if quant:
                    pool.ke[b, :, :prefix % page], pool.ve[b, :, :prefix % page] = pool.ke[a, :, :prefix % page], pool.ve[a, :, :prefix % page]
        for i, r in enumerate(rows):
            lens[r], start[r] = prefix + lens_own[at + i], prefix
            pool.fill(table, r, prefix, lens[r])
        shared += rows
        off.append(len(shared))
        at += count
    for i in range(len(alone)):
        r = order[at + i]
        lens[r] = alone[i]
        pool.fill(table, r, 0, lens[r])
    return pool, table, lens, start, shared, off, queries(n, heads, hd, dtype, g)


def run_shared(batch, heads, scale, **kw):
    pool, table, lens, start, shared, off, q = batch
    k, v, ke, ve = pool.put()
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    return K.attention_shared(q.to(DEV), k, v, put(range(len(lens))), put([n - 1 for n in lens]), table.to(DEV), heads, scale, put(start), put(shared), put(off),
                              k_exp=ke, v_exp=ve, **kw)


def check_shared(batch, heads, scale, **kw):
    pool, table, lens, start, shared, off, q = batch
    got = run_shared(batch, heads, scale, **kw)
    want = [reference(q[t], *pool.entries(table, t, n), heads, scale) for t, n in enumerate(lens)]
    compare(got, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))


@pytest.mark.parametrize("splits", [(0, 0), (1, 1), (5, 2)])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd,page", SHAPES)
def test_shared(heads, kv, hd, page, dtype, quant, splits):
    g = torch.Generator().manual_seed(heads * hd)
    batch = shared_batch([(100, 5), (33, 1), (64, 3)], [1, 2, 40, 17, 0], heads, kv, hd, page, dtype, quant, g, alone=(1, 50))
    check_shared(batch, heads, hd ** -0.5, shared_splits=splits[0], own_splits=splits[1])


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("groups", [[(1, 2)], [(40, 70)], [(200, 33), (31, 40), (7, 2)], [(20, 1)] * 70 + [(50, 3)]])
def test_shared_groups(groups, quant):
    """Groups that fill tiles of rows and do not, prefixes from one token on, more groups than a wave has lanes."""
    g = torch.Generator().manual_seed(len(groups))
    batch = shared_batch(groups, [1, 9], 4, 2, 64, 16, torch.bfloat16, quant, g)
    check_shared(batch, 4, 0.125, max_shared=200, max_own=9)


def test_rows_inside_the_prefix_and_padding_rows():
    """A row whose position lies in the prefix sees the keys up to it, a padding row none, wherever in its group it stands."""
    g = torch.Generator().manual_seed(8)
    batch = shared_batch([(90, 6)], [10], 4, 2, 64, 16, torch.float32, False, g)
    pool, table, lens, start, shared, off, q = batch
    first, inside, padding = shared[0], shared[2], shared[4]
    k, v, _, _ = pool.put()
    item, position = ints(range(6)), ints([n - 1 for n in lens])
    position[inside] = 41
    item[padding] = -1
    item[first] = -1
    put = lambda x: x.to(DEV)  # noqa: E731
    got = K.attention_shared(put(q), k, v, put(item), put(position), put(table), 4, 0.125, put(ints(start)), put(ints(shared)), put(ints(off)), shared_splits=2,
                             own_splits=1)
    for t in range(6):
        n = 0 if t in (padding, first) else int(position[t]) + 1
        kk, vv = pool.entries(table, t, n)
        want, bound = reference(q[t], kk, vv, 4, 0.125)
        compare(got[t], want, bound)
    # a list of nothing but places that are none: rows read what is theirs
    nobody = torch.full((6,), -1, dtype=torch.int32)
    got = K.attention_shared(put(q), k, v, put(ints(range(6))), put(ints([n - 1 for n in lens])), put(table), 4, 0.125, put(ints([0] * 6)), put(nobody),
                             put(ints([0, 6])))
    want = [reference(q[t], *pool.entries(table, t, n), 4, 0.125) for t, n in enumerate(lens)]
    compare(got, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))


@pytest.mark.parametrize("nobody", [63, 64, 150])
def test_a_group_that_begins_with_many_padding_rows(nobody):
    """The prefix's pages come from the first row with a request, however far behind in the list it stands."""
    g = torch.Generator().manual_seed(4)
    pool, table, lens, start, shared, off, q = shared_batch([(70, 3)], [9], 4, 2, 64, 16, torch.float32, False, g)
    k, v, _, _ = pool.put()
    put = lambda x: x.to(DEV)  # noqa: E731
    rows = [-1] * (nobody - 1) + [3] + list(shared)
    item = ints([0, 1, 2, -1])
    got = K.attention_shared(put(torch.cat((q, q[:1]))), k, v, put(item), put(ints([n - 1 for n in lens] + [50])), put(table), 4, 0.125,
                             put(ints(list(start) + [70])), put(ints(rows)), put(ints([0, len(rows)])), shared_splits=2, own_splits=1)
    for t, n in enumerate(lens):
        want, bound = reference(q[t], *pool.entries(table, t, n), 4, 0.125)
        compare(got[t], want, bound)
    assert (got[3] == 0).all()


def test_a_value_that_is_no_number_reaches_its_rows_only():
    g = torch.Generator().manual_seed(3)
    batch = shared_batch([(70, 4)], [20], 2, 2, 64, 16, torch.bfloat16, False, g)
    pool, table, lens, start, shared, off, q = batch
    r = shared[1]
    pool.v[int(table[r, 80 // 16]), 1, 80 % 16, 5] = math.nan
    pool.v[int(table[r, 81 // 16]), 0, 81 % 16, 9] = math.inf
    got = run_shared(batch, 2, 0.125, shared_splits=2, own_splits=2).cpu()
    for t in range(4):
        hit = torch.zeros(128, dtype=torch.bool)
        if t == r:
            hit[64 + 5] = hit[9] = True
        assert torch.equal(~torch.isfinite(got[t]), hit)
    assert got[r, 69].isnan() and got[r, 9] == math.inf


def test_results_do_not_depend_on_the_batch():
    """A row's result in a group is bit for bit the same from call to call, and for equal splits whatever the other rows are."""
    g = torch.Generator().manual_seed(6)
    batch = shared_batch([(150, 9)], [30], 8, 2, 64, 16, torch.bfloat16, True, g)
    a = run_shared(batch, 8, 0.125, shared_splits=3, own_splits=2)
    assert all(torch.equal(a, run_shared(batch, 8, 0.125, shared_splits=3, own_splits=2)) for _ in range(3))


@pytest.mark.parametrize("kind", ["rows", "portion", "shared"])
def test_recorded(kind):
    """Recorded calls follow positions, tables, groups and queries that change under them, and leave nothing of a call for the next."""
    g = torch.Generator().manual_seed(12)
    heads, kv, hd, page, n = 4, 2, 64, 16, 6
    table = torch.full((n, 20), -1, dtype=torch.int32)
    pool = Pool(n * 20 + 1, kv, page, hd, torch.bfloat16, True, g)
    for r in range(n):
        pool.fill(table, r, 0, 320)
    on = pool.put()
    q = torch.zeros(n, heads * hd, dtype=torch.bfloat16, device=DEV)
    item, position, start, rows, off = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (n, n, n, n, 3))
    tables = table.to(DEV)
    tile_item, tile_q0, tok, first, length = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (2, 2, n, n, n))
    if kind == "rows":
        call = lambda: K.attention_rows_quant(q, *on, item, position, tables, heads, 0.125, num_splits=4)  # noqa: E731
    elif kind == "portion":
        call = lambda: K.attention_prefill_quant(q, *on, tile_item, tile_q0, tok, first, length, tables, heads, 0.125, num_splits=3)  # noqa: E731
    else:
        call = lambda: K.attention_shared(q, on[0], on[1], item, position, tables, heads, 0.125, start, rows, off, k_exp=on[2], v_exp=on[3],  # noqa: E731
                                          shared_splits=3, own_splits=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call()
    torch.cuda.synchronize()
    for turn in range(4):
        qq = queries(n, heads, hd, torch.bfloat16, g)
        q.copy_(qq)
        lens = [1 + 50 * turn + 7 * r for r in range(n)]
        tab = table.clone()
        if kind == "portion":
            # items 0 and 1: four and two rows behind what is cached
            at = 37 * turn
            tile_item.copy_(ints([1, 0])); tile_q0.zero_(); tok.copy_(ints([0, 4, 0, 0, 0, 0])); first.copy_(ints([at, 2 * at, 0, 0, 0, 0]))
            length.copy_(ints([4, 2, 0, 0, 0, 0]))
            where = [(0, at + i + 1) for i in range(4)] + [(1, 2 * at + i + 1) for i in range(2)]
        else:
            item.copy_(ints(range(n)))
            position.copy_(ints([m - 1 for m in lens]))
            where = list(enumerate(lens))
            if kind == "shared" and turn:
                prefix = 32 * turn
                tab[1, :prefix // 16] = tab[0, :prefix // 16]
                tab[5, :prefix // 16] = tab[0, :prefix // 16]
                start.copy_(ints([prefix if prefix and r in (0, 1, 5) else 16 if r in (2, 4) else 0 for r in range(n)]))
                tab[4, 0] = tab[2, 0]
                rows.copy_(ints([5, 0, 1, 4, 2, -1])); off.copy_(ints([0, 3, 5]))
        tables.copy_(tab)
        graph.replay()
        torch.cuda.synchronize()
        want = [reference(qq[t], *pool.entries(tab, r, m), heads, 0.125) for t, (r, m) in enumerate(where)]
        want, bound = torch.stack([w for w, _ in want]), torch.stack([b for _, b in want])
        compare(got, want, bound)
        assert torch.equal(got, call())


def test_long_tables_with_far_pages():
    """Page numbers whose first element lies past 2^31 elements: 8-bit and bfloat16 pools of more than that."""
    g = torch.Generator().manual_seed(5)
    heads, kv, hd, page = 4, 4, 128, 16
    pages = (1 << 31) // (kv * page * hd) + 40
    for quant in (True, False):
        dtype = E4M3 if quant else torch.bfloat16
        k, v = (torch.zeros((pages, kv, page, hd), dtype=torch.uint8 if quant else dtype, device=DEV) for _ in range(2))
        exps = [torch.full((pages, kv, page), 121, dtype=torch.uint8, device=DEV) for _ in range(2)] if quant else [None, None]
        far = pages - 1 - torch.randperm(20, generator=g)
        kk, vv = (torch.randn(20, kv, page, hd, generator=g) for _ in range(2))
        if quant:
            kk, vv = (40 * kk).to(E4M3), (40 * vv).to(E4M3)
            k[far.to(DEV)], v[far.to(DEV)] = kk.view(torch.uint8).to(DEV), vv.view(torch.uint8).to(DEV)
            k, v = k.view(E4M3), v.view(E4M3)
        else:
            kk, vv = kk.bfloat16(), vv.bfloat16()
            k[far.to(DEV)], v[far.to(DEV)] = kk.to(DEV), vv.to(DEV)
        unit = 2.0 ** -6 if quant else 1.0
        ek, ev = ((x.double() * unit).permute(0, 2, 1, 3).reshape(320, kv, hd) for x in (kk, vv))
        q = queries(2, heads, hd, torch.bfloat16, g)
        table = far.int().view(1, 20).expand(2, 20).contiguous().to(DEV)
        item, position = ints([0, 1]).to(DEV), ints([299, 317]).to(DEV)
        if quant:
            got = K.attention_rows_quant(q.to(DEV), k, v, *exps, item, position, table, heads, 0.09)
        else:
            got = K.attention_shared(q.to(DEV), k, v, item, position, table, heads, 0.09, ints([160, 160]).to(DEV), ints([0, 1]).to(DEV), ints([0, 2]).to(DEV))
        for t, n in enumerate((300, 318)):
            want, bound = reference(q[t], ek[:n], ev[:n], heads, 0.09)
            compare(got[t], want, bound)
        del k, v, exps
        torch.cuda.empty_cache()


def test_refusals():
    g = torch.Generator().manual_seed(0)
    batch = shared_batch([(20, 2)], [3], 4, 2, 64, 16, torch.bfloat16, True, g)
    pool, table, lens, start, shared, off, q = batch
    k, v, ke, ve = pool.put()
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    q, table, item, position = q.to(DEV), table.to(DEV), put([0, 1]), put([n - 1 for n in lens])
    rows = lambda **kw: K.attention_rows_quant(**{**dict(q=q, k_cache=k, v_cache=v, k_exp=ke, v_exp=ve, token_item=item, positions=position,  # noqa: E731
                                                         block_table=table, num_q_heads=4, scale=0.1), **kw})
    both = lambda **kw: K.attention_shared(**{**dict(q=q, k_cache=k, v_cache=v, k_exp=ke, v_exp=ve, token_item=item, positions=position, block_table=table,  # noqa: E731
                                                     num_q_heads=4, scale=0.1, row_start=put(start), shared_rows=put(shared), group_off=put(off)), **kw})
    tile = lambda **kw: K.attention_prefill_quant(**{**dict(q=q, k_cache=k, v_cache=v, k_exp=ke, v_exp=ve, tile_item=put([0]), tile_q0=put([0]),  # noqa: E731
                                                            item_tok_off=put([0, 1]), item_start=put([0, 0]), item_len=put([1, 1]), block_table=table,
                                                            num_q_heads=4, scale=0.1), **kw})
    rows(), both(), tile()
    small = torch.zeros(3, device=DEV)
    for bad in (lambda: rows(q=q.half()), lambda: rows(q=q[:, :192]), lambda: rows(num_q_heads=3), lambda: rows(k_cache=k.view(torch.uint8)),
                lambda: rows(token_item=item.long()), lambda: rows(positions=position[:1]), lambda: rows(num_splits=65), lambda: rows(block_table=table[0]),
                lambda: rows(num_splits=2, workspace=small), lambda: rows(k_exp=ke[:1]), lambda: rows(token_item=item.cpu()),
                lambda: rows(out=torch.zeros(2, 256, device=DEV)), lambda: rows(q=torch.zeros(2, 257, dtype=torch.bfloat16, device=DEV)[:, 1:]),
                lambda: both(k_exp=None), lambda: both(k_exp=None, v_exp=None), lambda: both(row_start=put([0])), lambda: both(group_off=put([0])),
                lambda: both(shared_rows=put([])), lambda: both(shared_splits=60, own_splits=5), lambda: both(shared_rows=put(shared).long()),
                lambda: tile(item_len=put([1])), lambda: tile(tile_rows=0), lambda: tile(tile_q0=put([0, 0])), lambda: tile(tile_item=put([0]).long())):
        with pytest.raises((K.KernelError, TypeError)):
            bad()
