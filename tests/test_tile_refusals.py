"""Lists of shared prefixes, and block tables, that the C entry refuses before it launches anything: no GPU is needed."""
import pytest

from swifttransformer_amd.ops import kernels as K

P = 4096
ONE = dict(out=P, part_o=P, part_ml=P, q=P, q_stride=256, k_cache=P, v_cache=P, page_stride=2 * 16 * 64, k_exp=P, v_exp=P, exp_stride=32, token_item=P,
           positions=P, block_table=P, num_rows=0, num_entries=0, num_items=1, max_pages=4, page_size=16, num_pages=9, heads=4, kv_heads=2, head_dim=64,
           scale=1.0, own_splits=1, slots=1, dtype=1, cache_dtype=2, own_waves=4)
SHARED = dict(ONE, row_start=P, shared_rows=P, group_off=P, num_groups=1, num_shared=2, shared_splits=1, slots=2)


def call(**kw):
    return K._lib().st_tile_attention(bytes(K._TileAttention(**kw)), None)


def test_lists_that_are_whole():
    assert call(**ONE) == 0 and call(**SHARED) == 0


@pytest.mark.parametrize("kw", [dict(SHARED, num_shared=0), dict(SHARED, shared_rows=None), dict(SHARED, group_off=None), dict(ONE, row_start=P)])
def test_lists_that_are_not(kw):
    """(The join looks for a row in the groups' lists: an empty one, or starts without groups, leave it nothing to look at.)"""
    assert call(**kw) != 0 and "lists" in K._lib().st_last_error().decode()


@pytest.mark.parametrize("max_pages,page_size,fits", [((1 << 27) - 1, 16, False), ((1 << 31) - 2, 1, False), ((1 << 31) - 513, 1, True), ((1 << 27) - 32, 16, False),
                                                      ((1 << 27) - 33, 16, True), ((1 << 27) - 31, 16, False), (1 << 20, 1 << 11, False)])
def test_tables_whose_last_keys_are_close_to_what_an_int_holds(max_pages, page_size, fits):
    """(A wave's next blocks of keys are looked up ahead, behind the last key too.)"""
    kw = dict(ONE, max_pages=max_pages, page_size=page_size, page_stride=2 * page_size * 64 if page_size <= 16 else 1 << 30, exp_stride=2 * page_size)
    rc = call(**kw)
    assert (rc == 0) == fits and (fits or "2^31" in K._lib().st_last_error().decode())
