"""Sizes whose sums or grids do not fit the kernels' 32 bits are refused on the
host (with addresses that are never read: no call here gets to a launch)."""
from test_paged_refusals import PTR, SHAPE, _append, _attention, _batch, _kv


def test_table_rows_end_below_2_to_the_31():
    for page in (1, 16, 256):
        kv = _kv(page_size=page, table_width=(2 ** 31 - 1) // page, page_stride=2 * page * 128, head_stride=page * 128)
        assert _attention(kv, _batch()) == SHAPE
        assert _append(kv, _batch()) == SHAPE


def test_sums_of_tiles_fit():
    """4,096 sequences of up to 2^25 positions have more than 2^31 tiles."""
    kv = _kv(slots=4096, table_width=1 << 21)
    assert _attention(kv, _batch(seqs=4096, tokens=4096, max_new=1)) == SHAPE


def test_rows_of_a_sample_fit_a_grid():
    from hy_mt_rs_b200._native import lib
    for rows in (2 ** 31 - 1, 2 ** 28):
        assert lib.hyq_sample(PTR, 100, 100, rows, None, None, None, None, PTR, PTR, None, None) == SHAPE


def test_entries_of_histories_and_biases_end_below_2_to_the_31():
    """The adjust kernel's loops over a row's history and biases count in 32 bits, some
    turns past the last entry."""
    from test_paged8_refusals import _adjust
    for n in (2 ** 31 - 1, 2 ** 31 - 2048, 2 ** 31 - 65536):
        assert _adjust(width=n, history_stride=n) == SHAPE
        assert _adjust(bias_count=n) == SHAPE
