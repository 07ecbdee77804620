"""CPU: argument errors of the block-attention operators (before any launch), the plans they take, and the definitions they are
tested against (oracle/attention.py) held to a second form of each formula and to differences."""
import ctypes as C
import math

import pytest
import torch

from adaptivepnp_sci_amd import _lib
from adaptivepnp_sci_amd import attention as A
from oracle import attention as O

P = 256                                                           # an aligned address that is never followed


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return _lib.load()


def refused(lib, rc, word):
    assert rc in (-1, -2, -4) and word in lib.scipnp_last_error().decode(), lib.scipnp_last_error()


def attn(**kw):
    st = (C.c_int64 * 3)(64 * 4, 64, 64)
    a = dict(dtype=1, B=2, Lq=8, Lk=64, Hq=4, Hk=2, D=64, block=64, query_block=4, n_sel=1, scale=1.0, q=P, k=P, v=P, out=P, sel=P,
             q_stride=st, k_stride=st, v_stride=st, out_stride=st, dout_stride=st)
    a.update(kw)
    return _lib.BlockAttnArgs(**a)


@pytest.mark.parametrize('change, word', [
    (dict(struct_size=8), 'struct_size'), (dict(dtype=2), 'dtype'), (dict(Lq=0), 'positive'), (dict(Hq=3), 'multiple'), (dict(D=20), 'head size'),
    (dict(D=136), 'head size'), (dict(block=32), 'multiple of 64'), (dict(query_block=0), 'query_block'), (dict(query_block=2000), 'query_block'),
    (dict(n_sel=0), 'n_sel'), (dict(n_sel=1025), 'n_sel'), (dict(sel=0), 'null'), (dict(q=0), 'null'), (dict(q=P + 2), 'aligned'),
    (dict(k_stride=(C.c_int64 * 3)(3, 64, 64)), 'stride'), (dict(v_stride=(C.c_int64 * 3)(64, -64, 64)), 'stride'), (dict(num_buckets=65, bias=P, bucket_of=P), 'buckets'),
    (dict(num_buckets=8), 'bias'), (dict(num_buckets=8, bias=P, bucket_of=P, max_distance=5000), 'max_distance'), (dict(out=0), 'out'),
    (dict(Hq=128, Hk=1, num_buckets=64, bias=P, bucket_of=P, max_distance=4), 'at most 2048'), (dict(Lq=1 << 30, query_block=1), 'groups'),
])
def test_attention_refusals(lib, change, word):
    size = change.pop('struct_size', None)
    a = attn(**change)
    if size:
        a.struct_size = size
    refused(lib, lib.scipnp_block_attn(C.byref(a), None), word)
    if word != 'out':
        refused(lib, lib.scipnp_block_attn_backward(C.byref(a), None), word)
        assert lib.scipnp_block_attn_workspace_bytes(C.byref(a), 1) == 0


def test_attention_backward_refusals(lib):
    refused(lib, lib.scipnp_block_attn_backward(C.byref(attn()), None), 'backward needs')
    full = dict(dout=P, dq=P, dk=P, dv=P, lse=P, lse_rest=P, out32=P)
    refused(lib, lib.scipnp_block_attn_backward(C.byref(attn(**full, num_buckets=8, bias=P, bucket_of=P, max_distance=9)), None), 'dbias')
    a = attn(**full)
    need = lib.scipnp_block_attn_workspace_bytes(C.byref(a), 1)
    assert need > 0
    refused(lib, lib.scipnp_block_attn_backward(C.byref(a), None), 'workspace')
    a.workspace, a.workspace_bytes = P, need - 1
    refused(lib, lib.scipnp_block_attn_backward(C.byref(a), None), 'workspace')
    # few groups with many keys are split over workgroups, which needs a workspace too
    b = attn(Lq=1, Lk=65536, query_block=1, n_sel=512)
    assert lib.scipnp_block_attn_workspace_bytes(C.byref(b), 0) > 0
    refused(lib, lib.scipnp_block_attn(C.byref(b), None), 'workspace')
    refused(lib, lib.scipnp_block_attn(None, None), 'null')


def test_norm_summary_and_selection_refusals(lib):
    st = (C.c_int64 * 3)(64 * 4, 64, 64)
    base = dict(dtype=1, B=1, L=4, Hq=2, Hk=1, D=64, eps=1e-6, q=P, k=P, out_q=P, out_k=P, wq=P, wk=P, q_stride=st, k_stride=st, out_q_stride=st, out_k_stride=st)
    for change, word in ((dict(D=12), 'head size'), (dict(D=264), 'head size'), (dict(rot=12), 'rotated'), (dict(rot=128), 'rotated'), (dict(rot=16), 'turns'),
                         (dict(wq=0), 'null'), (dict(k=0), 'Hk'), (dict(v=P), 'out_v'), (dict(slots=P), 'Lout'), (dict(eps=-1.0), 'eps'),
                         (dict(q=P + 8), 'aligned'), (dict(out_q_stride=(C.c_int64 * 3)(1, 64, 64)), 'stride'), (dict(L=0), 'positive')):
        refused(lib, lib.scipnp_head_norm_rotate(C.byref(_lib.HeadNormArgs(**{**base, **change})), None), word)
    refused(lib, lib.scipnp_head_norm_rotate_backward(C.byref(_lib.HeadNormArgs(**base)), None), 'backward needs')
    refused(lib, lib.scipnp_head_norm_rotate_backward(C.byref(_lib.HeadNormArgs(**base, g_q=P, g_k=P, dwq=P, dwk=P, g_q_stride=st, g_k_stride=st)), None), 'workspace')
    for args, word in (((None, st, 1, None, P, 1, 64, 1, 64, 64, 0), 'null'), ((P, st, 1, None, P, 1, 64, 1, 60, 64, 0), 'head size'),
                       ((P, st, 3, None, P, 1, 64, 1, 64, 64, 0), 'dtype'), ((P, st, 1, None, P, 1, 64, 1, 64, 0, 0), 'block'), ((P + 4, st, 1, None, P, 1, 64, 1, 64, 64, 0), 'aligned')):
        refused(lib, lib.scipnp_block_summary(*args, None), word)
    sel = dict(dtype=1, B=1, Lq=4, Lk=64, Hq=2, Hk=1, D=64, block=64, query_block=4, n_sel=1, q=P, summary=P, sel=P, q_stride=st)
    for change, word in ((dict(Hk=4), 'multiple'), (dict(Lk=1 << 20, block=64), 'key blocks'), (dict(n_sel=0), 'n_sel'), (dict(sink=-1), 'sink'), (dict(q=0), 'null'),
                         (dict(query_block=1025), 'query_block')):
        refused(lib, lib.scipnp_select_blocks(C.byref(_lib.SelectArgs(**{**sel, **change})), None), word)


def test_python_refusals_name_the_argument():
    q, k = torch.zeros(2, 8, 4, 64), torch.zeros(2, 64, 2, 64)
    sel = torch.zeros(2, 2, 2, 1, dtype=torch.int32)
    w = torch.ones(64)
    for call, word in (
            (lambda: A.head_norm_rotate(q[0], k, w, w), r'q must be a \(B, L, H, D\)'), (lambda: A.head_norm_rotate(q.half(), None, w), 'float16'),
            (lambda: A.head_norm_rotate(q.transpose(2, 3), None, w), 'last dimension'), (lambda: A.head_norm_rotate(q[:, :0], None, w), 'empty'),
            (lambda: A.block_summary(k, 0), 'block'), (lambda: A.block_summary(k, 64, newest=1), 'newest needs out'),
            (lambda: A.select_blocks(q, torch.zeros(2, 1, 3, 64), 1), 'summary'), (lambda: A.select_blocks(q, torch.zeros(2, 1, 2, 64), 1, keys=65), '65 keys'),
            (lambda: A.block_attention(q, k[:1], k[:1], sel), 'same batch'), (lambda: A.block_attention(q, k, k, sel, query_block=0), 'query_block'),
            (lambda: A.block_attention(q, k, k, sel[0], query_block=4), 'sel must be')):
        with pytest.raises(ValueError, match=word):
            call()
    with pytest.raises(_lib.ScipnpError, match='no CPU fallback'):
        A.block_attention(q, k, k, sel, query_block=4)
    for bad in ((1, 8, False), (66, 100, True), (5, 100, True), (8, 2, True), (8, 5000, True)):
        with pytest.raises(ValueError):
            A.bucket_table(*bad)
    with pytest.raises(ValueError):
        A.rotary_turns(12)


def test_bucket_table_against_logarithms():
    """away from the exact steps the whole-number rule is the floor of the logarithm"""
    for n, md, both in ((32, 128, True), (32, 128, False), (16, 500, True), (64, 4096, False), (4, 9, True)):
        t = A.bucket_table(n, md, both)
        side = n // 2 if both else n
        e = side // 2
        for rel in range(-md, md + 1):
            d = abs(rel) if both else max(-rel, 0)
            x = (side - e) * math.log(d / e) / math.log(md / e) if d >= e else 0.0
            if d >= e and abs(x - round(x)) < 1e-9:
                continue
            want = d if d < e else min(side - 1, e + math.floor(x))
            assert t[rel + md] == want + (n // 2 if both and rel > 0 else 0), (n, md, rel)


def test_the_definition_has_the_gradients_of_differences():
    gen = torch.Generator().manual_seed(0)
    B, Lq, Lk, Hq, Hk, D, qb, block = 1, 5, 9, 2, 1, 8, 2, 4
    q, k, v, g = (torch.randn(B, L, H, D, generator=gen) for L, H in ((Lq, Hq), (Lk, Hk), (Lk, Hk), (Lq, Hq)))
    sel = torch.tensor([[0, 2], [1, -1], [0, 1]], dtype=torch.int32)[None, None].repeat(B, Hk, 1, 1)
    table, bias = A.bucket_table(8, 6), torch.randn(8, Hq, generator=gen).double()

    def f(q, k, v, bias):
        return (O.attention(q, k, v, sel, block, qb, 0.4, True, None, None, table, bias, dout=None)['out'][0] * g.double()).sum()

    got = O.attention(q, k, v, sel, block, qb, 0.4, True, None, None, table, bias, dout=g)
    for name, i in (('dq', 0), ('dk', 1), ('dv', 2), ('dbias', 3)):
        args = [t.double() for t in (q, k, v)] + [bias]
        O.U[torch.float64] = 2.0 ** -53
        d = torch.randn(args[i].shape, generator=gen, dtype=torch.float64)
        up, down = list(args), list(args)
        h = 1e-5
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        diff = (f(*up) - f(*down)) / (2 * h)
        assert abs(float(diff - (got[name][0] * d).sum())) < 1e-7 * max(1.0, abs(float(diff))), name      # truncation h^2, cancellation 2^-53 / h
