"""Attention by tiles at scores of any size that floats hold: from 10^9 on, where a rounding of a score is more than an exponent's range, up to 10^34,
of either sign.  Scores are powers of two times small whole numbers, so they are exact and the keys with the largest share the result evenly; sums over n of
them are off by n 2^-24 of what they add, and bfloat16 rounds the result by 2^-8 of it at most (and probabilities of one or nothing not at all)."""
import pytest
import torch

from swifttransformer_amd.ops import kernels as K
from test_tile_attention_gpu import DEV, compare, ints
from test_tile_parts_gpu import paged

pytestmark = pytest.mark.gpu


def batch(power, n, heads, kv, hd, dtype, quant, g):
    """Queries with one dim of +-2^power, keys with 1, 1.5 or 2 there: (q, table, cache, results for all lengths up to n by definition)."""
    table, cache, k, v = paged(n, kv, hd, 16, dtype, quant, g)
    unit = 2.0 ** -6 if quant else 1.0
    pages = table[0].long()
    first = torch.randint(2, 5, (n, kv), generator=g) / 2                     # 1, 1.5, 2
    first[0], first[n // 2:] = 1.5, torch.where(first[n // 2:] == 2, 1.0, first[n // 2:])
    for j in range(n):
        at = (pages[j // 16], slice(None), j % 16, 0)
        if quant:
            cache[0].view(torch.uint8)[at] = (first[j] / unit).to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
        else:
            cache[0][at] = first[j].to(dtype).to(DEV)
    sign = torch.where(torch.arange(heads) % 2 == 0, 1.0, -1.0)
    q = torch.zeros(1, heads, hd)
    q[:, :, 0] = sign * 2.0 ** power
    group = heads // kv

    def wanted(m):
        out, size = [], []
        for h in range(heads):
            s = first[:m, h // group] * sign[h]
            best = s == s.max()
            out.append(v[:m, h // group][best].mean(0))
            size.append(v[:m, h // group][best].abs().mean(0))
        return torch.cat(out), torch.cat(size) * ((2 * m + 64) * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0))
    return q.view(1, heads * hd).to(dtype), table, cache, wanted


@pytest.mark.parametrize("scale", [1.0, -0.125])
@pytest.mark.parametrize("power", [20, 31, 60, 113])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 64), (6, 2, 80), (2, 1, 256)])
def test_large_scores(heads, kv, hd, dtype, quant, power, scale):
    g = torch.Generator().manual_seed(power)
    lens = [1, 2, 40, 301]
    q, table, cache, wanted = batch(power, 301, heads, kv, hd, dtype, quant, g)
    if scale < 0:
        q = -q
    T = len(lens)
    q = q.expand(T, -1).contiguous().to(DEV)
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    item, position, table = put([0] * T), put([n - 1 for n in lens]), table.to(DEV)
    want = [wanted(n) for n in lens]
    want, bound = torch.stack([w for w, _ in want]), torch.stack([b for _, b in want])
    for shared, own in ((1, 1), (3, 2)):
        got = K.attention_shared(q, cache[0], cache[1], item, position, table, heads, scale, put([100] * T), put(range(T)), put([0, T]), k_exp=cache[2],
                                 v_exp=cache[3], shared_splits=shared, own_splits=own)
        compare(got, want, bound)
        if quant:
            compare(K.attention_rows_quant(q, *cache, item, position, table, heads, scale, num_splits=own), want, bound)
            last = lens[-1]
            got = K.attention_prefill_quant(q[:3], *cache, put([0]), put([0]), put([0]), put([last - 3]), put([3]), table, heads, scale, num_splits=own)
            some = [wanted(last - 2 + i) for i in range(3)]
            compare(got, torch.stack([w for w, _ in some]), torch.stack([b for _, b in some]))


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores_of_rows_a_wave_each(dtype, quant):
    g = torch.Generator().manual_seed(3)
    heads, kv, hd, n = 4, 2, 64, 70
    q, table, cache, wanted = batch(60, n, heads, kv, hd, dtype, quant, g)
    T = 4 * torch.cuda.get_device_properties(0).multi_processor_count // kv + 1
    put = lambda x: ints(x).to(DEV)  # noqa: E731
    lens = [1 + (7 * t) % n for t in range(T)]
    got = K.attention_shared(q.expand(T, -1).contiguous().to(DEV), cache[0], cache[1], put([0] * T), put([m - 1 for m in lens]), table.to(DEV), heads, 1.0,
                             put([16] * T), put(range(T)), put([0, T]), k_exp=cache[2], v_exp=cache[3], shared_splits=1, own_splits=1)
    for t in range(0, T, 23):
        w, b = wanted(lens[t])
        compare(got[t], w, b)
