"""Filters through the sampler, the engine and the command line: the tokens are those of the definition for the hash's random numbers,
whatever batch a request is in, and requests without filters keep theirs."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_opt
import tiny
from test_sample_filtered_gpu import drawn
from swifttransformer_amd.ops import kernels as K
from swifttransformer_amd.sampling import Sampler, SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PARAMS = [SamplingParams(temperature=0.7, seed=3, top_k=5), SamplingParams(temperature=1.2, seed=1 << 40, top_p=0.8), SamplingParams(),
          SamplingParams(temperature=0.9, seed=7), SamplingParams(temperature=1.0, seed=9, min_p=0.1), SamplingParams(seed=2, top_k=3),
          SamplingParams(temperature=0.5, seed=11, top_k=40, top_p=0.9, min_p=0.02), SamplingParams(temperature=2.0, seed=12)]


def wanted(x, p, d):
    if p.filtered:
        u = K.hash_uniform(p.seed & 0xffffffff, p.seed >> 32, d, 0xffffffff)
        return drawn(x, float(np.float32(u)), float(np.float32(p.temperature)), p.top_k, float(np.float32(p.top_p)), float(np.float32(p.min_p)))
    return plain_opt.choose(x, p.temperature, p.seed, d)


def test_sampler():
    g = torch.Generator().manual_seed(1)
    sampler = Sampler(DEV)
    for draws in ([0] * 8, [3, 1, 4, 1, 5, 9, 2, 6], [1000 + i for i in range(8)]):
        x = 2 * torch.randn(8, 3001, generator=g)
        got = sampler.sample(x.to(DEV), PARAMS, draws)
        assert got == [wanted(x[i].numpy(), p, d) for i, (p, d) in enumerate(zip(PARAMS, draws))]
        # each alone, and the ones without filters among themselves
        assert got == [sampler.sample(x[i:i + 1].to(DEV), [PARAMS[i]], [draws[i]])[0] for i in range(8)]
        plain = [i for i, p in enumerate(PARAMS) if not p.filtered]
        assert [got[i] for i in plain] == sampler.sample(x[plain].to(DEV), [PARAMS[i] for i in plain], [draws[i] for i in plain])


def test_engine(tmp_path):
    from swifttransformer_amd.engine.engine import Engine
    d = tiny.write_model("B", str(tmp_path), seed=11)
    cfg, _w = plain_opt.load_folder(d)
    prompts = [tiny.prompt(n, cfg["vocab_size"], 40 + i) for i, n in enumerate((1, 9, 40, 20))]
    params = [SamplingParams(temperature=0.8, seed=50, max_new_tokens=10, ignore_eos=True, top_k=8), SamplingParams(max_new_tokens=10, ignore_eos=True),
              SamplingParams(temperature=1.5, seed=51, max_new_tokens=10, ignore_eos=True, top_p=0.7, min_p=0.01),
              SamplingParams(temperature=0.8, seed=52, max_new_tokens=10, ignore_eos=True)]
    make = lambda **kw: Engine(d, dtype="fp32", page_size=8, num_pages=60, **kw)  # noqa: E731
    outs = make(max_seqs=4).generate(prompts, params)
    assert outs == make(max_seqs=2, prefill_chunk=7, max_batched_tokens=20).generate(prompts, params)
    assert outs == [make(max_seqs=1).generate([p], [sp])[0] for p, sp in zip(prompts, params)]
    # a k of one is greedy, whatever the temperature
    one = make(max_seqs=4).generate(prompts, SamplingParams(temperature=1.3, top_k=1, max_new_tokens=6, ignore_eos=True))
    assert one == make(max_seqs=4).generate(prompts, SamplingParams(max_new_tokens=6, ignore_eos=True))


def test_command_line(tmp_path):
    d = tiny.write_model("A", str(tmp_path), seed=11)
    prompts = tmp_path / "prompts.txt"
    prompts.write_text("2 5 9\n7 7\n")
    run = lambda *more: subprocess.run([sys.executable, os.path.join(ROOT, "bin", "run_opt"), d, "auto", "fp32", str(prompts), "--max-new-tokens", "5",  # noqa: E731
                                        "--ignore-eos", "--num-blocks", "16", *more], capture_output=True, text=True, timeout=100)
    greedy, one = run(), run("--temperature", "1.5", "--top-k", "1", "--top-p", "0.9", "--min-p", "0.1")
    lines = lambda r: [x for x in r.stdout.splitlines() if x.startswith("[")]  # noqa: E731
    assert greedy.returncode == 0 and one.returncode == 0, one.stderr
    assert len(lines(greedy)) == 2 and lines(greedy) == lines(one)


def test_operators_together():
    """A decode loop as a server of many answers to few prompts runs it: new entries go into the 8-bit cache, every answer attends over its group's
    prompt and its own entries, and draws its next token with filters of its own; each step against the definitions."""
    from test_tile_attention_gpu import Pool, compare, ints, reference
    g = torch.Generator().manual_seed(21)
    heads, kv, hd, page, vocab = 8, 2, 64, 16, 997
    prompts, answers = (70, 33), (5, 3)
    B = sum(answers)
    table = torch.full((B, 8), -1, dtype=torch.int32)
    pool = Pool(B * 8 + 1, kv, page, hd, torch.float32, True, g)
    start, groups, at = [], [], 0
    for n, count in zip(prompts, answers):
        rows = list(range(at, at + count))
        pool.fill(table, rows[0], 0, n)
        for r in rows:
            table[r, :n // page] = table[rows[0], :n // page]
            if r != rows[0] and n % page:                        # the page that the prompt ends in: each has its own
                table[r, n // page] = pool.order.pop()
                a, b = int(table[rows[0], n // page]), int(table[r, n // page])
                for c in (pool.k, pool.v, pool.ke, pool.ve):
                    c[b, :, :n % page] = c[a, :, :n % page]
        start += [n] * count
        groups.append(rows)
        at += count
    for r in range(B):                                           # pages for what is to come
        for i in range(start[r] // page, 8):
            if table[r, i] < 0:
                table[r, i] = pool.order.pop()
    k, v, ke, ve = pool.put()
    put = lambda t: t.to(DEV)  # noqa: E731
    tables, item, row_start = put(table), put(ints(range(B))), put(ints(start))
    rows, off = put(ints([r for rs in groups for r in rs])), put(ints([0, answers[0], B]))
    head, embed = torch.randn(heads * hd, vocab, generator=g) * 0.2, torch.randn(vocab, (heads + 2 * kv) * hd, generator=g)
    head_dev, embed_dev = put(head), put(embed)
    t, top_k, top_p, min_p = torch.rand(B, generator=g) + 0.5, ints([0, 5, 20, 0, 3, 0, 50, 2]), torch.tensor([0.9, 1.0, 0.8, 0.5] * 2), torch.tensor([0.0, 0.05] * 4)
    filters = [put(x) for x in (t, top_k, top_p, min_p)]
    tokens = put(ints([3 * r for r in range(B)]))
    for step in range(6):
        qkv = embed_dev[tokens.long()]
        position = put(ints([s + step for s in start]))
        K.quant_kv_write(k, v, ke, ve, qkv[:, heads * hd:(heads + kv) * hd], qkv[:, (heads + kv) * hd:], item, position, tables, page)
        o = K.attention_shared(qkv[:, :heads * hd], k, v, item, position, tables, heads, hd ** -0.5, row_start, rows, off, k_exp=ke, v_exp=ve,
                               max_shared=max(prompts), max_own=step + 1)
        logits = o @ head_dev
        u = torch.rand(B, generator=g)
        nxt = K.sample_filtered(logits, put(u), filters[0], top_k=filters[1], top_p=filters[2], min_p=filters[3])
        # against the definitions, from what the device's cache holds
        pool.k, pool.v, pool.ke, pool.ve = k.view(torch.uint8).cpu(), v.view(torch.uint8).cpu(), ke.cpu(), ve.cpu()
        want = [reference(qkv[r, :heads * hd].cpu(), *pool.entries(table, r, start[r] + step + 1), heads, hd ** -0.5) for r in range(B)]
        compare(o, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))
        alone = K.attention_rows_quant(qkv[:, :heads * hd], k, v, ke, ve, item, position, tables, heads, hd ** -0.5)
        compare(alone, torch.stack([w for w, _ in want]), torch.stack([b for _, b in want]))
        x = logits.cpu().numpy()
        assert nxt.tolist() == [drawn(x[r], float(u[r]), float(t[r]), int(top_k[r]), float(top_p[r]), float(min_p[r])) for r in range(B)]
        tokens = nxt
