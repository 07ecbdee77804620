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
    full = dict(dout=P, dq=P, dk=P, dv=P, lse=P, lse_rest=P, out32=P, dbias=P, dout_stride=st)
    a = _lib.BlockAttnArgs(dtype=1, B=1, Lq=1, Lk=64, Hq=32 * 40000, Hk=40000, D=64, block=64, query_block=1, n_sel=1, scale=1.0, q=P, k=P, v=P, out=P, sel=P,
                           num_buckets=64, max_distance=4, bias=P, bucket_of=P, q_stride=st, k_stride=st, v_stride=st, out_stride=st, **full)
    refused(lib, lib.scipnp_block_attn_backward(C.byref(a), None), 'buckets and query heads')


# ------------------------------------------------------------------ results that share memory
def test_results_in_the_memory_of_something_else_are_refused():
    import torch
    from adaptivepnp_sci_amd import attention as A
    q, k, v, w = torch.zeros(2, 64, 2, 64), torch.zeros(2, 64, 2, 64), torch.zeros(2, 64, 2, 64), torch.ones(64)
    sel = torch.zeros(2, 2, 16, 1, dtype=torch.int32)
    flat = torch.zeros(2 * 64 * 2 * 64 + 64)
    part = flat[64:].view(2, 64, 2, 64)                           # overlaps flat[:-64] by all but a row
    whole = flat[:-64].view(2, 64, 2, 64)
    one = torch.zeros(2, 1, 2, 64).expand(2, 64, 2, 64)
    for call, word in (
            (lambda: A.block_attention(q, k, v, sel, query_block=4, out=k), 'out shares memory with k'),
            (lambda: A.block_attention(q, k, v, sel, query_block=4, out=v), 'out shares memory with v'),
            (lambda: A.block_attention(part, k, v, sel, query_block=4, out=whole), 'out shares memory with q'),
            (lambda: A.block_attention(q, k, v, sel, query_block=4, out=one), 'out has several places'),
            (lambda: A.block_attention(q, part, v, sel, query_block=4, out=whole), 'out shares memory with k'),
            (lambda: A.head_norm_rotate(q, k, w, w, out_q=k), 'out_q shares memory with k'),
            (lambda: A.head_norm_rotate(q, k, w, w, out_k=q), 'out_k shares memory with q'),
            (lambda: A.head_norm_rotate(q, k, w, w, out_q=v, out_k=v), 'out_k shares memory with out_q'),
            (lambda: A.head_norm_rotate(part, None, w, out_q=whole), 'out_q shares memory with q'),
            (lambda: A.head_norm_rotate(q, None, w, out_q=one), 'out_q has several places'),
            (lambda: A.head_norm_rotate(q, k, w, w, out_k=torch.zeros_like(k), v=v, out_v=k), 'out_v shares memory with k'),
            (lambda: A.head_norm_rotate(q, k, w, w, out_k=v, v=v, out_v=torch.zeros_like(v)), 'out_k shares memory with v'),
            (lambda: A.head_norm_rotate(q, k[:, :1], w, w, out_k=v, v=v[:, :1], out_v=k, slots=torch.zeros(2, 1, dtype=torch.int32)), 'shares memory'),
            (lambda: (lambda t: A.block_summary(t, 1, out=t))(torch.zeros(1, 64, 1, 8)), 'out shares memory with k')):
        with pytest.raises((ValueError, _lib.ScipnpError), match=word):
            call()
    packed = torch.zeros(2, 64, 6, 64)                            # views of one projection, in place: not refused for their memory
    for call in (lambda: A.head_norm_rotate(packed[:, :, :2], packed[:, :, 2:4], w, w, out_q=packed[:, :, :2], out_k=packed[:, :, 2:4]),
                 lambda: A.block_attention(packed[:, :, :2], packed[:, :, 2:4], packed[:, :, 4:], sel, query_block=4, out=packed[:, :, :2]),
                 lambda: A.head_norm_rotate(q, k, w, w, out_q=q, out_k=k, v=v, out_v=v)):
        with pytest.raises(_lib.ScipnpError, match='no CPU fallback'):
            call()


# ------------------------------------------------------------------ the build
def test_the_libraries_build_without_python(tmp_path):
    """a C host has no torch: plain make asks for the libraries alone there, and for the Python module as well where it can be built"""
    import os
    import subprocess
    csrc = os.path.join(os.path.dirname(_lib.__file__), 'csrc')
    for python, built in (('false', False), ('python3', True)):
        r = subprocess.run(['make', '-n', '-C', csrc, f'PYTHON={python}', f'BIND_OUT={tmp_path}/none.so'], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, r.stderr
        assert ('-ltorch_python' in r.stdout) == built, r.stdout


def test_a_module_of_another_torch_is_refused(monkeypatch):
    from adaptivepnp_sci_amd import attention as A
    have = A.torch.__version__.split('+')[0]
    monkeypatch.setattr(A, '_bound', None)
    monkeypatch.setattr(A.torch, '__version__', '1.0.0+other')
    with pytest.raises(_lib.ScipnpError, match='built for torch'):
        A._bind()
    monkeypatch.setattr(A.torch, '__version__', have + 'a0+git123')           # (a build of the same three numbers)
    assert A._bind().built_for == have
