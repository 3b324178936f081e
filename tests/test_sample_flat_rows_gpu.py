"""Filtered sampling where most of a row weighs the same as its largest, up to rows of 2^18 logits whose sums of weights are the largest that there are,
and logits that are signalling NaN."""
import math

import numpy as np
import pytest
import torch

from test_sample_filtered_gpu import check, floats, settings

pytestmark = pytest.mark.gpu

US = [0.0, 0.2, 0.73, 1.0 - 2.0 ** -24]


def table(options):
    """Every combination of lists, as columns."""
    columns = list(zip(*[(u, t, k, p, least) for u in US for t in options[0] for k in options[1] for p in options[2] for least in options[3]]))
    return [floats(c) for c in columns[:2]] + [torch.tensor(columns[2], dtype=torch.int32)] + [floats(c) for c in columns[3:]]


@pytest.mark.parametrize("vocab", [261119, 261120, 261121, 262143, 262144])
def test_equal_logits(vocab):
    u, t, k, p, least = table(([1.0, math.inf], [0, 200000], [1.0, 0.5, 0.999], [0.0, 1.0]))
    check(torch.full((len(u), vocab), -2.5), u, t, k, p, least)


@pytest.mark.parametrize("vocab", [261120, 262143, 262144])
def test_temperatures_that_make_all_alike(vocab):
    g = torch.Generator().manual_seed(vocab)
    u, t, k, p, least = table(([1e30, math.inf], [0], [1.0, 0.7], [0.0, 0.5]))
    check(3 * torch.randn(len(u), vocab, generator=g), u, t, k, p, least)


@pytest.mark.parametrize("vocab", [50272, 262144])
def test_stretches_of_largest_and_of_smaller(vocab):
    """The border of a top p in the smaller ones, behind stretches that are all of the largest."""
    u, t, k, p, least = table(([1.0], [0], [1.0, 0.8, 0.9], [0.0, 0.1, 1.0]))
    x = torch.zeros(len(u), vocab)
    x[:, vocab * 5 // 8:] = -0.5
    x[1::2] = x[1::2].flip(1)
    check(x, u, t, k, p, least)


@pytest.mark.parametrize("bits", [0x7f800001, 0x7fa00000, 0x7fbfffff, -0x7fffff, -0x600000])
@pytest.mark.parametrize("vocab", [3, 700, 5003])
def test_signalling_nan(vocab, bits):
    g = torch.Generator().manual_seed(vocab)
    rows = 24
    x = 3 * torch.randn(rows, vocab, generator=g)
    at = torch.rand(rows, vocab, generator=g) < 0.3
    x.view(torch.int32)[at] = bits
    x.view(torch.int32)[0] = bits
    assert bool(np.isnan(x.numpy()[0]).all())
    check(x, *settings(rows, vocab, g))
