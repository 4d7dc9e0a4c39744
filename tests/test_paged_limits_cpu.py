"""CPU tier: the extents at which the paged attention's 32-bit counters end. The decoding kernel deals
units to its CTAs, an item (sequence, KV head) having its key blocks' and 384 / head_dim more, and keeps their
total, a CTA's first unit and its last one in 32 bits."""
import ctypes as C

import pytest

I32 = 2 ** 31 - 1


def desc(lvb, batch, heads_kv, D, width, page, group=1, max_q=1):
    d = lvb.lvb_paged_desc()
    d.dtype, d.causal, d.scale = lvb.BF16, 1, 0.1
    d.batch, d.heads_q, d.heads_kv, d.head_dim = batch, group * heads_kv, heads_kv, D
    d.tokens, d.max_q = batch * max_q, max_q
    d.page_size, d.num_pages, d.table_width = page, 1000, width
    return d


def attention_check(lvb, *a, **k):
    st = lvb.lib.lvb_attention_paged_check(C.byref(desc(lvb, *a, **k)))
    return st, lvb.lib.lvb_last_error().decode()


@pytest.mark.parametrize("batch,heads,D,width,page", [
    (49_000_000, 8, 64, 1, 8),          # 392 million items of one block and six more units
    (4_194_304, 74, 64, 1, 128),
    (2 ** 20, 512, 128, 1, 8),
    (1000, 8, 128, 2 ** 22, 128),       # long tables: the blocks themselves
])
def test_more_units_than_the_counters_hold(lvb, batch, heads, D, width, page):
    units = batch * heads * (-(-width * page // 128) + 384 // D)
    assert units > I32
    st, msg = attention_check(lvb, batch, heads, D, width, page)
    assert st == lvb.LVB_ERR_UNSUPPORTED and "split the batch" in msg
    p = lvb.lvb_paged_plan()
    d = desc(lvb, batch, heads, D, width, page)
    assert lvb.lib.lvb_attention_paged_plan_for(C.byref(d), 148, C.byref(p)) == lvb.LVB_ERR_UNSUPPORTED


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [1, 8, 74])
@pytest.mark.parametrize("width,page", [(1, 8), (1, 128), (3, 48), (8, 128), (100, 64), (2 ** 22, 256)])
def test_the_largest_batch_fits(lvb, D, heads, width, page):
    """At the last batch that is taken every counter of the kernel is below 2^31, one more is refused;
    no batch whose counters fit by a third of 2^31 is."""
    per = heads * (-(-width * page // 128) + 384 // D)
    lo, hi = 1, I32 // max(heads, 1)
    while lo < hi:
        mid = (lo + hi + 1) // 2
        lo, hi = (mid, hi) if attention_check(lvb, mid, heads, D, width, page)[0] == 0 else (lo, mid - 1)
    assert attention_check(lvb, lo + 1, heads, D, width, page)[0] == lvb.LVB_ERR_UNSUPPORTED
    total = lo * per
    assert I32 * 2 // 3 - 2 * per < total <= I32
    for ctas in (1, 2, 3, 80, 132, 148):
        assert total + ctas - 1 <= I32
        share = (total + ctas - 1) // ctas
        firsts = [min(i, total // share + 1) * share for i in range(ctas)]
        assert max(firsts) + share <= I32


def test_other_calls_do_not_count_units(lvb):
    """The append and the flash kernel have no such sum."""
    a = lvb.lvb_append_desc()
    a.paged = desc(lvb, 49_000_000, 8, 64, 1, 8)
    a.rot.n_axes = 1
    assert lvb.lib.lvb_kv_append_check(C.byref(a)) == 0
    assert attention_check(lvb, 10_000_000, 8, 64, 2, 256, max_q=17)[0] == 0


@pytest.mark.parametrize("heads_kv", [2 ** 62, 2 ** 32 + 1, 2 ** 31])
def test_heads_without_queries_are_bounded(lvb, heads_kv):
    """An append without queries has no heads_q that would bound its KV heads: four sequences of 2^62
    heads are 2^64 items, 0 in 64 bits."""
    a = lvb.lvb_append_desc()
    a.paged = desc(lvb, 4, heads_kv, 64, 1, 8, group=0)
    a.rot.n_axes = 1
    assert lvb.lib.lvb_kv_append_check(C.byref(a)) == lvb.LVB_ERR_UNSUPPORTED
    assert "2^31" in lvb.lib.lvb_last_error().decode()
