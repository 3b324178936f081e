"""What the speed of the operators behind shared prompts, the cache in 8 bits and filtered sampling is measured on: one call of each, as a
serving step makes it, over paged caches with pages in any order.

  op "sample"   a token for each of ``rows`` rows of ``vocab`` float logits: temperature, then the ``top_k`` largest, of those the fewest that
                hold ``top_p`` of the weight, of those the ones with ``min_p`` of the largest's weight, then the given random number's
                place among them in the order of their indices.  ``filters`` says which of the three the rows use; ``coarse``: logits that
                come out of 16 bits, many of them alike.
  op "write"    keys and values of ``tokens`` tokens of ``requests`` requests go into the 8-bit cache, and are read back from there.
  op "read"     attention of the last ``new`` tokens of each request over its own entries in the 8-bit cache (``tokens`` over all requests).
  op "shared"   attention of one token of each request over a prefix of ``prefix`` tokens, which the requests of a group share, and
                over entries of its own; ``cache`` says in which form the entries are held ("same": the queries' type, or "e4m3").

An entry in 8 bits is e4m3 times a power of two that a token's head has in common: the smallest with which its largest value is at most 448.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _sample(name, rows, vocab, filters="all", coarse=False):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "filters": filters, "coarse": coarse}


def _write(name, requests, tokens, kv_heads, head_dim, dtype="bf16", page=16):
    return {"name": name, "op": "write", "requests": requests, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "page": page}


def _read(name, requests, tokens, new, heads, kv_heads, head_dim, dtype="bf16", page=16):
    return {"name": name, "op": "read", "requests": requests, "tokens": tokens, "new": new, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "page": page}


def _shared(name, requests, groups, prefix, tokens, heads, kv_heads, head_dim, cache="same", dtype="bf16", page=16):
    return {"name": name, "op": "shared", "requests": requests, "groups": groups, "prefix": prefix, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "cache": cache, "dtype": dtype, "page": page}


def listed():
    return [
        # one user's next token
        _sample("sample 1", 1, 50272),
        # a full server's next tokens, every row with filters of its own
        _sample("sample 64", 64, 50272),
        # many answers at once over a large vocabulary of odd size, by the weight that they hold alone, logits of a 16-bit head
        _sample("sample 256 wide", 256, 128007, "top_p", True),
        # the entries of one decode step of 8 requests
        _write("write 8", 8, 8, 32, 64),
        # a prompt's entries at wide layers
        _write("write 2047", 1, 2047, 40, 128),
        # the headline decode step: 8 requests half way from 1,024-token prompts to the 2,048-token context
        _read("read 8", 8, 8 * 1536, 1, 32, 32, 64),
        # a full server with grouped heads: 64 requests of very different lengths
        _read("read 64 grouped", 64, 64 * 1000 + 9, 1, 32, 8, 128),
        # a portion of a prompt behind what is cached of it
        _read("read portion", 1, 1536, 512, 32, 32, 128),
        # a short exchange in 32 bits
        _read("read fp32", 3, 701, 1, 12, 12, 64, "fp32"),
        # several answers to a prompt
        _shared("shared 16", 16, 1, 1024, 16 * 101, 32, 32, 64),
        # a busy server: three long system prompts with grouped heads, in the small cache
        _shared("shared 200 e4m3", 200, 3, 6007, 200 * 301, 32, 8, 128, "e4m3"),
        # several answers in 32 bits, at a head size that fills no power of two
        _shared("shared fp32", 40, 1, 500, 40 * 63, 32, 32, 80, dtype="fp32"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case: 1 to 256 rows of 1,000 to 128,000 logits; 1 to 4,096 tokens written; 1 to 64 requests of 1 to 4,000 tokens, single tokens
    or portions of up to 600; 2 to 256 requests behind prefixes of 16 to 8,000 tokens; pages of 8 to 32."""
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("sample", "write", "read", "shared"))
        heads, kv_heads, head_dim = rng.choice(((12, 12, 64), (32, 32, 64), (32, 32, 80), (32, 32, 128), (32, 8, 128), (16, 2, 64), (8, 1, 256), (24, 8, 96)))
        dtype = "fp32" if rng.random() < 0.25 else "bf16"
        page = rng.choice((16, 16, 8, 32, 12))
        if op == "sample":
            case = _sample("", _log(rng, 1, 256), _log(rng, 1000, 128000), rng.choice(("all", "top_k", "top_p", "min_p", "none")), rng.random() < 0.3)
        elif op == "write":
            tokens = _log(rng, 1, 4096)
            case = _write("", rng.choice((1, min(tokens, 4), tokens)), tokens, kv_heads, head_dim, dtype, page)
        elif op == "read":
            requests = _log(rng, 1, 64)
            new = rng.choice((1, 1, _log(rng, 8, 600)))
            requests = requests if new == 1 else min(requests, 4)
            case = _read("", requests, requests * (new + _log(rng, 1, 4000)), new, heads, kv_heads, head_dim, dtype, page)
        else:
            requests = _log(rng, 2, 256)
            case = _shared("", requests, rng.randint(1, min(4, requests)), _log(rng, 16, 8000), requests * _log(rng, 1, 600), heads, kv_heads, head_dim,
                           rng.choice(("same", "e4m3")), dtype, page)
        del case["name"]
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / (1e14 if case.get("dtype") == "fp32" else 1e15)


def _share(n, total, least, tag):
    """``total`` in ``n`` ragged parts of at least ``least``."""
    rng = random.Random(f"{n} parts of {total} {tag}")
    share = [rng.uniform(0.3, 1.7) for _ in range(n)] if n > 1 else [1.0]
    parts = [max(least, int(total * s / sum(share))) for s in share]
    parts[0] = max(least, parts[0] + total - sum(parts))
    return parts


def _lengths(case):
    """Tokens of each request (of its own ones, behind a prefix)."""
    if case["op"] == "write":
        return _share(case["requests"], case["tokens"], 1, "write")
    if case["op"] == "read":
        return _share(case["requests"], case["tokens"], case["new"], "read")
    return _share(case["requests"], case["tokens"], 1, "shared")


def _prefixes(case):
    """A group's prefix length and its requests, which are dealt out in turn."""
    lens = _share(case["groups"], case["groups"] * case["prefix"], 1, "prefix")
    return [(lens[g], list(range(g, case["requests"], case["groups"]))) for g in range(case["groups"])]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + 24.0 * case["rows"], "flops": 4.0 * n}
    elem = 4 if case["dtype"] == "fp32" else 2
    w = case["kv_heads"] * case["head_dim"]
    small = 2.0 * (w + case["kv_heads"])                              # an entry's keys and values in 8 bits
    if case["op"] == "write":
        return {"bytes": case["tokens"] * (2.0 * w * elem + 2 * small + 2.0 * w * elem), "flops": 4.0 * case["tokens"] * w}
    lens, rows = _lengths(case), case["requests"]
    if case["op"] == "read":
        rows *= case["new"]
        entries = sum(lens)
        pairs = sum(case["new"] * n - case["new"] * (case["new"] - 1) // 2 for n in lens)
    else:
        groups = _prefixes(case)
        entries = sum(lens) + sum(n for n, _ in groups)
        pairs = sum(lens) + sum(n * len(r) for n, r in groups)
    entry = small if case["op"] == "read" or case["cache"] == "e4m3" else 2.0 * w * elem
    wide = case["heads"] * case["head_dim"]
    return {"bytes": entries * entry + 2.0 * rows * wide * elem, "flops": 4.0 * pairs * wide}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _to_small(x):
    """Heads' vectors [..., head_dim] as e4m3 and the exponents (biased by 127) of their powers of two."""
    big = x.float().abs().amax(-1)
    m, e = torch.frexp(big)                                            # big = m * 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9)                           # 448 = 0.875 * 2^9
    e = torch.where(big > 0, e + 127, torch.full_like(e, 127)).clamp(1, 254)
    power = torch.exp2(127.0 - e.double())[..., None]
    return (x.double() * power).float().to(torch.float8_e4m3fn), e.to(torch.uint8)


def _from_small(x, e):
    return x.float() * torch.exp2(e.double() - 127.0).float()[..., None]


def _tables(lens, page, gen, groups=()):
    """(block table, pages of the pool): ``groups`` of (whole prefix pages, requests) name the same pages."""
    counts = [-(-n // page) for n in lens]
    total = sum(counts) + sum(p for p, _ in groups)
    order = torch.randperm(total + 3, generator=gen).tolist()
    shared = {}
    for pages, requests in groups:
        first = [order.pop() for _ in range(pages)]
        for r in requests:
            shared[r] = first
    table = torch.zeros((len(lens), max(counts)), dtype=torch.int32)
    for r, c in enumerate(counts):
        first = shared.get(r, [])
        table[r, :c] = torch.tensor(first + [order.pop() for _ in range(c - len(first))], dtype=torch.int32)
    return table.to(DEV), total + 3


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=dev, device=DEV)  # noqa: E731
    if case["op"] == "sample":
        R, V = case["rows"], case["vocab"]
        # few likely words over a broad rest, sharper for some rows than for others
        logits = randn(R, V) * (1.0 + 2.0 * torch.rand((R, 1), generator=dev, device=DEV))
        logits += 6.0 * (torch.rand((R, V), generator=dev, device=DEV) < 20.0 / V) * torch.rand((R, V), generator=dev, device=DEV)
        if case["coarse"]:
            logits = logits.bfloat16().float()
        rng = random.Random(seed)
        use = lambda name: case["filters"] in ("all", name)  # noqa: E731
        temperature = [0.0 if R > 4 and rng.random() < 0.1 else rng.uniform(0.4, 1.5) for _ in range(R)]
        top_k = [rng.choice((20, 50, 200, 0)) if use("top_k") else 0 for _ in range(R)]
        top_p = [rng.choice((0.5, 0.8, 0.9, 0.95, 1.0)) if use("top_p") else 1.0 for _ in range(R)]
        min_p = [rng.choice((0.0, 0.02, 0.05, 0.1)) if use("min_p") else 0.0 for _ in range(R)]
        floats = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
        return {"op": "sample", "logits": logits, "uniforms": torch.rand((R,), generator=dev, device=DEV), "temperature": floats(temperature),
                "top_k": torch.tensor(top_k, dtype=torch.int32, device=DEV), "top_p": floats(top_p), "min_p": floats(min_p)}
    dtype, page, nkv, hd = DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["head_dim"]
    lens = _lengths(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    outliers = 1.0 + 3.0 * (torch.rand((hd,), generator=dev, device=DEV) < 0.04)     # channels that keys are large in
    if case["op"] == "write":
        table, pages = _tables(lens, page, gen)
        T = sum(lens)
        kv = randn(T, 2, nkv, hd) * torch.exp(0.7 * randn(T, 2, nkv, 1))
        kv[:, 0] *= outliers
        kv = kv.to(dtype).view(T, 2 * nkv * hd)
        return {"op": "write", "k": kv[:, :nkv * hd], "v": kv[:, nkv * hd:], "table": table, "page": page, "dtype": dtype,
                "k_cache": torch.zeros((pages, nkv, page, hd), device=DEV).to(torch.float8_e4m3fn),
                "v_cache": torch.zeros((pages, nkv, page, hd), device=DEV).to(torch.float8_e4m3fn),
                "k_exp": torch.zeros((pages, nkv, page), dtype=torch.uint8, device=DEV),
                "v_exp": torch.zeros((pages, nkv, page), dtype=torch.uint8, device=DEV),
                "item": ints([r for r, n in enumerate(lens) for _ in range(n)]), "position": ints([p for n in lens for p in range(n)])}
    heads, new = case["heads"], case.get("new", 1)
    groups, start = [], [0] * len(lens)
    if case["op"] == "shared":
        groups = _prefixes(case)
        for n, requests in groups:
            for r in requests:
                start[r] = n
                lens[r] += n
    # (where a prefix ends inside a page, every request has its own copy of what is in that page)
    table, pages = _tables(lens, page, gen, [(n // page, requests) for n, requests in groups])
    k = (randn(pages, nkv, page, hd) * outliers).to(dtype)
    v = randn(pages, nkv, page, hd).to(dtype)
    for n, requests in groups:
        if n % page:
            rest = table[requests, n // page].long()
            k[rest, :, :n % page], v[rest, :, :n % page] = k[rest[0], :, :n % page], v[rest[0], :, :n % page]
    T = len(lens) * new
    s = {"op": case["op"], "q": (1.5 * randn(T, heads * hd)).to(dtype), "table": table, "heads": heads, "scale": hd ** -0.5, "page": page,
         "item": ints([r for r in range(len(lens)) for _ in range(new)]), "position": ints([n - new + i for n in lens for i in range(new)]),
         "k_cache": k, "v_cache": v, "k_exp": None, "v_exp": None, "new": new, "longest": max(lens)}
    if case["op"] == "read" or case["cache"] == "e4m3":
        s["k_cache"], s["k_exp"] = _to_small(k)
        s["v_cache"], s["v_exp"] = _to_small(v)
    if case["op"] == "read":
        s["tile_item"] = ints([r for r in range(len(lens)) for _ in range(0, new, 64)])
        s["tile_q0"] = ints([q for _ in lens for q in range(0, new, 64)])
        s["item_tok_off"], s["item_start"], s["item_len"] = ints([r * new for r in range(len(lens))]), ints([n - new for n in lens]), ints([new] * len(lens))
    else:
        s["row_start"] = ints(start)
        s["shared_rows"] = ints([r for _, requests in groups for r in requests])
        at = [0]
        for _, requests in groups:
            at.append(at[-1] + len(requests))
        s["group_off"] = ints(at)
        s["max_shared"], s["max_own"] = max(n for n, _ in groups), max(n - b for n, b in zip(lens, start))
    return s


# -------------------------------------------------------------------------------------------------------------- plain forms
def _plain_sample(s):
    x = s["logits"].double()
    T = s["temperature"].double()[:, None]
    R, V = x.shape
    w = torch.exp((x - x.amax(1, keepdim=True)) / torch.where(T > 0, T, torch.ones_like(T)))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = torch.gather(w, 1, order)
    rank = torch.arange(V, device=x.device)[None]
    k = s["top_k"].long()[:, None]
    ranked = torch.where((k <= 0) | (rank < k), ranked, torch.zeros_like(ranked))
    sums = torch.cumsum(ranked, 1)
    kept = (sums - ranked < s["top_p"].double()[:, None] * sums[:, -1:]) | (rank == 0)
    kept &= ranked >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, ranked, torch.zeros_like(ranked)))
    sums = torch.cumsum(w, 1)
    drawn = ((sums > s["uniforms"].double()[:, None] * sums[:, -1:]) & (w > 0)).to(torch.uint8).argmax(1)
    return torch.where(T[:, 0] > 0, drawn, order[:, 0]).int()


def _plain_write(s):
    nkv, hd = s["k_cache"].shape[1], s["k_cache"].shape[3]
    page = s["table"][s["item"].long(), (s["position"] // s["page"]).long()].long()
    row = (s["position"] % s["page"]).long()
    back = []
    for name in ("k", "v"):
        small, e = _to_small(s[name].view(-1, nkv, hd))
        s[name + "_cache"].view(torch.uint8)[page, :, row] = small.view(torch.uint8)
        s[name + "_exp"][page, :, row] = e
        read = _from_small(s[name + "_cache"].view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn), s[name + "_exp"][page, :, row])
        back.append(read.to(s["dtype"]).view(-1, nkv * hd))
    return back


def _plain_attention(s):
    B, hd, nkv, new = s["table"].shape[0], s["k_cache"].shape[3], s["k_cache"].shape[1], s["new"]
    group = s["heads"] // nkv
    at = torch.arange(s["longest"], device=s["q"].device)
    page = s["table"][:, at // s["page"]].long()
    row = (at % s["page"])[None].expand(B, -1)
    entries = []
    for name in ("k", "v"):
        pool = s[name + "_cache"]
        if s[name + "_exp"] is None:
            x = pool[page, :, row].float()
        else:
            x = _from_small(pool.view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn), s[name + "_exp"][page, :, row])
        entries.append(x.permute(0, 2, 1, 3).contiguous())                          # [B, kv heads, longest, head_dim]
    k, v = entries
    q = s["q"].float().view(B, new, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(B, nkv, group * new, hd)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    seen = at[None, None, :] <= s["position"].view(B, new)[:, :, None]               # [B, new, longest]
    scores = scores.view(B, nkv, group, new, -1).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, nkv, group * new, -1)
    out = torch.matmul(p, v).view(B, nkv, group, new, hd).permute(0, 3, 1, 2, 4)
    return out.reshape(B * new, s["heads"] * hd).to(s["q"].dtype)


def run(s):
    if own:
        from swifttransformer_amd.ops import kernels as K
        if s["op"] == "sample":
            return K.sample_filtered(s["logits"], s["uniforms"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
        if s["op"] == "write":
            cache = (s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"])
            K.quant_kv_write(*cache, s["k"], s["v"], s["item"], s["position"], s["table"], s["page"])
            return K.quant_kv_read(*cache, s["item"], s["position"], s["table"], s["dtype"])
        if s["op"] == "shared":
            return K.attention_shared(s["q"], s["k_cache"], s["v_cache"], s["item"], s["position"], s["table"], s["heads"], s["scale"],
                                      s["row_start"], s["shared_rows"], s["group_off"], k_exp=s["k_exp"], v_exp=s["v_exp"],
                                      max_shared=s["max_shared"], max_own=s["max_own"])
        if s["new"] == 1:
            return K.attention_rows_quant(s["q"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["item"], s["position"], s["table"], s["heads"],
                                          s["scale"], max_keys=s["longest"])
        return K.attention_prefill_quant(s["q"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["tile_item"], s["tile_q0"], s["item_tok_off"],
                                         s["item_start"], s["item_len"], s["table"], s["heads"], s["scale"], max_keys=s["longest"])
    if s["op"] == "sample":
        return _plain_sample(s)
    if s["op"] == "write":
        return _plain_write(s)
    return _plain_attention(s)


# ------------------------------------------------------------------------------------------------------- definitions in 64 bits
def _exact_entries(x, e):
    return x.double() if e is None else torch.ldexp(x.float().double(), e.int()[..., None] - 127)


def _exact_small(x):
    """x [..., head_dim] in 64 bits as the value that its entry stands for: rounded to a multiple of the step that e4m3 has there."""
    big = x.abs().amax(-1, keepdim=True)
    unit = torch.ones_like(big)
    for _ in range(300):
        unit = torch.where(big > 448 * unit, unit * 2, torch.where((big > 0) & (big <= 224 * unit), unit / 2, unit))
    unit = unit.clamp(2.0 ** -126, 2.0 ** 127)
    y = (x / unit).abs()
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        ids = []
        columns = (s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniforms"])
        for x, t, k, p, least, u in zip(s["logits"].double(), *(c.tolist() for c in columns)):
            value, index = torch.sort(x, descending=True, stable=True)
            if t <= 0:
                ids.append(int(index[0]))
                continue
            if k > 0:
                value, index = value[:k], index[:k]
            w = torch.exp((value - value[0]) / t)
            sums = torch.cumsum(w, 0)
            count = max(1, int((sums < p * sums[-1]).sum()) + 1)
            w, index = w[:count], index[:count]
            w, index = w[w >= least], index[w >= least]
            index, by = torch.sort(index)
            sums = torch.cumsum(w[by], 0)
            ids.append(int(index[min(int((sums <= u * sums[-1]).sum()), len(index) - 1)]))
        return torch.tensor(ids, dtype=torch.int32)
    if case["op"] == "write":
        nkv, hd = case["kv_heads"], case["head_dim"]
        return [_exact_small(s[n].double().view(-1, nkv, hd)).view(-1, nkv * hd) for n in ("k", "v")]
    hd, nkv, heads, new = case["head_dim"], case["kv_heads"], case["heads"], s["new"]
    out = []
    for r in range(s["table"].shape[0]):
        n = int(s["position"][(r + 1) * new - 1]) + 1
        at = torch.arange(n, device=DEV)
        page, row = s["table"][r, at // s["page"]].long(), at % s["page"]
        k, v = (_exact_entries(s[c + "_cache"].view(torch.uint8)[page, :, row].view(torch.float8_e4m3fn), s[c + "_exp"][page, :, row])
                if s[c + "_exp"] is not None else s[c + "_cache"][page, :, row].double() for c in ("k", "v"))
        q = s["q"][r * new:(r + 1) * new].double().view(new, heads, hd)
        hidden = at[None] > s["position"][r * new:(r + 1) * new, None]
        for h in range(heads):
            scores = (q[:, h] @ k[:, h * nkv // heads].T.contiguous()) * s["scale"]
            scores[hidden] = -math.inf
            out.append(torch.softmax(scores, 1) @ v[:, h * nkv // heads].contiguous())
    rows = torch.stack(out).view(-1, heads, new, hd)
    return rows.permute(0, 2, 1, 3).reshape(-1, heads * hd)
