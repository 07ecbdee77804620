"""CPU: sizes at the ends of 32 bits, refused before any launch"""
import ctypes as C

import pytest

from adaptivepnp_sci_amd import _lib

P = 256                                                           # an aligned address that is never followed
TOP = 2 ** 31 - 1


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


def refused(lib, rc, word):
    assert rc in (-1, -2, -4) and word in lib.scipnp_last_error().decode(), (rc, lib.scipnp_last_error())


@pytest.mark.parametrize('Lk, block', [(TOP, 64), (TOP, 1), (TOP - 5, 2), (8193, 1), (TOP, 262143)])
def test_selection_counts_its_blocks_in_64_bits(lib, Lk, block):
    st = (C.c_int64 * 3)(64 * 4, 64, 64)
    a = _lib.SelectArgs(dtype=1, B=1, Lq=4, Lk=Lk, Hq=2, Hk=1, D=64, block=block, query_block=4, n_sel=1, q=P, summary=P, sel=P, q_stride=st)
    refused(lib, lib.scipnp_select_blocks(C.byref(a), None), 'key blocks')


@pytest.mark.parametrize('Lk, block, newest', [(TOP, 1, 0), (TOP, 2, 0), (1 << 24, 1, 0), (TOP, 100, TOP)])
def test_summary_counts_its_blocks_in_64_bits(lib, Lk, block, newest):
    st = (C.c_int64 * 3)(64 * 4, 64, 64)
    refused(lib, lib.scipnp_block_summary(P, st, 1, None, P, 1, Lk, 1, 64, block, newest, None), 'blocks')


def test_heads_are_counted_in_64_bits(lib):
    st = (C.c_int64 * 3)(64 * 4, 64, 64)
    refused(lib, lib.scipnp_block_summary(P, st, 1, None, P, 1, 64, 1 << 28, 128, 64, 0, None), 'key heads')
    a = _lib.BlockAttnArgs(dtype=1, B=1, Lq=1, Lk=64, Hq=1 << 26, Hk=1, D=64, block=64, query_block=1, n_sel=1, scale=1.0, q=P, k=P, v=P, out=P, sel=P,
                           num_buckets=64, max_distance=4, bias=P, bucket_of=P, q_stride=st, k_stride=st, v_stride=st, out_stride=st)
    refused(lib, lib.scipnp_block_attn(C.byref(a), None), 'at most 2048')
