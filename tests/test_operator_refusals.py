"""What the C entries of filtered sampling, the 8-bit cache and tile attention refuse before they launch anything, and what their faces refuse
before they ask for the library's device: no GPU is needed for either."""
import ctypes

import pytest
import torch

from swifttransformer_amd.ops import kernels as K


def error(rc):
    assert rc != 0
    return K._lib().st_last_error().decode()


def test_sample_filtered():
    lib = K._lib()
    p = 4096
    ok = dict(out=p, logits=p, stride=10, rows=0, vocab=10, uniforms=p, temperature=p)
    call = lambda **kw: lib.st_sample_filtered(*[{**ok, **kw}[n] for n in ok], None, None, None, None)  # noqa: E731
    assert call() == 0
    for bad, says in ((dict(rows=-1), "bad sizes"), (dict(vocab=0), "bad sizes"), (dict(stride=9), "bad sizes"), (dict(vocab=1 << 19, stride=1 << 19), "logits a row"),
                      (dict(rows=1 << 22), "at once"), (dict(rows=1, logits=None), "null"), (dict(rows=1, uniforms=None), "null"), (dict(rows=1, temperature=None), "null")):
        assert says in error(call(**bad))


def test_quant_cache():
    lib = K._lib()
    p = 4096
    sizes = dict(num_items=1, max_pages=2, page_size=16, num_pages=3, tokens=0, heads=2, head_dim=64, dtype=1)
    strides = dict(page=2 * 16 * 64, exp=32, src=256)

    def write(src=p, **kw):
        z, s = {**sizes, **kw}, {**strides, **kw}
        return lib.st_quant_kv_write(p, p, s["page"], p, p, s["exp"], src, p, s["src"], p, p, p, *[z[n] for n in sizes], None)

    def read(to=p, **kw):
        z, s = {**sizes, **kw}, {**strides, **kw}
        return lib.st_quant_kv_read(to, p, p, p, s["page"], p, p, s["exp"], p, p, p, *[z[n] for n in sizes], None)
    for call in (write, read):
        assert call() == 0
        for bad, says in ((dict(head_dim=24), "multiple of 16"), (dict(head_dim=272), "multiple of 16"), (dict(page=2000), "page stride"), (dict(page=2056), "page stride"),
                          (dict(exp=31), "overlap"), (dict(tokens=-1), "bad sizes"), (dict(num_pages=0), "bad sizes"), (dict(dtype=3), "dtype"),
                          (dict(tokens=0x7fffffff, heads=4096, page=4096 * 1024, exp=65536), "too many")):
            assert says in error(call(**bad))
    assert "aligned" in error(write(src=4104))
    assert "aligned" in error(read(to=4104))


def test_tile_attention():
    lib = K._lib()
    p = 4096
    ok = dict(out=p, part_o=p, part_ml=p, q=p, q_stride=256, k_cache=p, v_cache=p, page_stride=2 * 16 * 64, k_exp=p, v_exp=p, exp_stride=32, token_item=p,
              positions=p, block_table=p, num_rows=0, num_entries=0, num_items=1, max_pages=4, page_size=16, num_pages=9, heads=4, kv_heads=2, head_dim=64,
              scale=1.0, own_splits=1, slots=1, dtype=1, cache_dtype=2, own_waves=4)
    call = lambda **kw: lib.st_tile_attention(bytes(K._TileAttention(**{**ok, **kw})), None)  # noqa: E731
    assert call() == 0
    one = dict(num_rows=1, num_entries=1)
    shared = dict(row_start=p, shared_rows=p, group_off=p, num_groups=1, num_shared=2, shared_splits=1, slots=2)
    for bad, says in ((dict(heads=5), "divide"), (dict(head_dim=40), "multiple of 16"), (dict(head_dim=512), "multiple of 16"), (dict(page_size=0), "bad sizes"),
                      (dict(num_items=0), "bad sizes"), (dict(max_pages=1 << 28), "2^31"), (dict(dtype=7), "dtype"), (dict(cache_dtype=0), "cache of type"),
                      (dict(cache_dtype=1), "kernels of their own"), (dict(k_exp=None), "exponents"), (dict(exp_stride=3), "exponents"),
                      (dict(page_stride=1024), "page stride"), (dict(page_stride=2 * 16 * 64 + 8), "page stride"), (dict(page_stride=1 << 32), "page stride"),
                      (dict(own_splits=0, slots=0), "splits"), (dict(own_splits=70, slots=70), "splits"), (dict(own_splits=2, slots=1), "splits"),
                      (dict(one, own_splits=2, slots=2, part_o=None), "null"), (dict(one, q=None), "null"), (dict(one, q=4104), "aligned"),
                      (dict(one, q_stride=257), "aligned"), (dict(one, out=None), "null"),
                      (dict(num_tiles=1, tile_rows=64), "tiles need"), (dict(own_waves=2), "waves"), (dict(shared, row_start=None), "lists"), (dict(shared, shared_splits=0, slots=1), "splits"),
                      (dict(shared, row_ids=p), "lists"), (dict(num_rows=1 << 30, num_entries=1 << 30), "at once"),
                      (dict(num_rows=1 << 24, num_entries=1 << 24, own_splits=2, slots=2, own_waves=1), "at once"),
                      (dict(num_rows=1, num_tiles=1 << 20, tile_rows=65536, tile_item=p, tile_q0=p, item_tok_off=p, item_start=p, item_len=p), "at once")):
        assert says in error(call(**bad)), bad


def test_packed_arguments_are_the_structure():
    """Every field in its place: numbers that say which one they are."""
    n = len(K._TileAttention._fields_)
    values = list(range(1, n + 1))
    assert K._pack_tiles(*values) == bytes(K._TileAttention(*values))[:len(K._pack_tiles(*values))]
    assert len(bytes(K._TileAttention())) - len(K._pack_tiles(*values)) < 8      # (padding at the end)


def test_faces_want_gpu_tensors():
    x, r = torch.zeros(2, 8), torch.zeros(2)
    i = torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(1, 1, 4, 16).to(torch.float8_e4m3fn)
    e = torch.zeros(1, 1, 4, dtype=torch.uint8)
    table = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(K.KernelError, match="GPU tensor"):
        K.sample_filtered(x, r, r)
    with pytest.raises(K.KernelError, match="GPU tensor"):
        K.quant_kv_write(k, k, e, e, x, x, i, i, table, 4)
    with pytest.raises(K.KernelError, match="GPU tensor"):
        K.quant_kv_read(k, k, e, e, i, i, table, torch.float32)
    with pytest.raises(K.KernelError, match="GPU tensor"):
        K.attention_rows_quant(x, k, k, e, e, i, i, table, 1, 1.0)


def test_splits_follow_the_sizes():
    assert K.tile_splits(1, 100, 256) == 1 and K.tile_splits(10 ** 6, 10 ** 6, 256) == 1
    assert all(1 <= K.tile_splits(w, m, 256) <= 32 for w in (0, 1, 7, 255, 256, 999) for m in (0, 1, 127, 128, 4096, 10 ** 6))
