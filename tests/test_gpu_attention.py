"""-m gpu: the block-attention operators (adaptivepnp_sci_amd/attention.py) against their plain definitions in 64 bits
(oracle/attention.py).  Tolerances are element-wise bounds of the roundings that the kernels make: half a step of the output's type,
of the probabilities' type in front of the second product, and of every fp32 sum (see `attention` there); nothing is fitted."""
import math

import pytest
import torch

from oracle import attention as O

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def A():
    from adaptivepnp_sci_amd import attention
    return attention


def randn(gen, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=gen) * std).to(dtype)


def cu(t):
    return None if t is None else t.cuda()


def within(got, val, err, what):
    got = got.double().cpu()
    assert got.shape == val.shape, what
    fin = torch.isfinite(val)
    assert torch.equal(torch.isfinite(got), fin), what
    assert torch.equal(got[~fin], val[~fin]), what
    d = (got[fin] - val[fin]).abs()
    over = d > err[fin] + 1e-37
    assert not over.any(), f'{what}: {int(over.sum())} of {over.numel()} over the bound, worst {float((d / (err[fin] + 1e-37)).max()):.3g} x'


# ------------------------------------------------------------------ norm and rotation
NORM = [  # B, L, Hq, Hk, D, rot
    (1, 1, 1, 1, 8, 0), (2, 3, 5, 1, 16, 8), (1, 7, 4, 4, 48, 48), (3, 1, 8, 2, 128, 128), (2, 65, 6, 3, 40, 16),
    (1, 300, 2, 2, 256, 64), (1, 1500, 3, 1, 96, 96), (2, 33, 7, 7, 72, 72), (1, 2, 2, 1, 24, 24),
]


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('case', NORM)
def test_head_norm_rotate_and_its_gradient(A, case, dt):
    B, L, Hq, Hk, D, rot = case
    T = DT[dt]
    gen = torch.Generator().manual_seed(B * 1000 + L)
    q, k, gq, gk = (randn(gen, B, L, H, D, dtype=T, std=s) for H, s in ((Hq, 3.0), (Hk, 0.1), (Hq, 1.0), (Hk, 1.0)))
    wq, wk = 1 + 0.3 * randn(gen, D), 1 + 0.3 * randn(gen, D)
    pos = torch.randint(0, 1 << 20, (B, L), generator=gen, dtype=torch.int32)
    turns = A.rotary_turns(rot) if rot else None
    oq, ok = A.head_norm_rotate(cu(q), cu(k), cu(wq), cu(wk), cu(turns), cu(pos))
    # fp64 throughout, one rounding; 2^-40 covers the fp64 roundings and the angle's (2^-52 * 2^20 * 2 pi)
    for got, x, w in ((oq, q, wq), (ok, k, wk)):
        val = O.norm_rotate(x, w, turns, pos)
        size = O.norm_rotate(x, w, None, pos).abs().amax(-1, keepdim=True)
        within(got, val, O.U[T] * (1 + 2 ** -7) * val.abs() + 2.0 ** -29 * size, 'norm')
    dq, dk, dwq, dwk = A.head_norm_rotate_backward(cu(gq), cu(gk), cu(q), cu(k), cu(wq), cu(wk), cu(turns), cu(pos))
    for got, gw, x, w, g in ((dq, dwq, q, wq, gq), (dk, dwk, k, wk, gk)):
        xx, ww = x.double().requires_grad_(), w.double().requires_grad_()
        y = xx * torch.rsqrt(xx.square().mean(-1, keepdim=True) + 1e-6) * ww
        if rot:
            h = rot // 2
            ang = pos.double()[..., None] * turns
            ang = 2 * math.pi * (ang - ang.floor())
            c, s = ang.cos()[:, :, None], ang.sin()[:, :, None]
            y = torch.cat([y[..., :h] * c - y[..., h:rot] * s, y[..., h:rot] * c + y[..., :h] * s, y[..., rot:]], -1)
        y.backward(g.double())
        size = xx.grad.abs().amax(-1, keepdim=True)
        within(got, xx.grad, O.U[T] * (1 + 2 ** -7) * xx.grad.abs() + 2.0 ** -29 * size, 'dx')
        within(gw, ww.grad, O.U32 * 1.01 * ww.grad.abs() + 2.0 ** -40 * (g.double().abs().sum((0, 1, 2)).amax() * 40), 'dw')


def test_head_norm_rotate_into_a_cache(A):
    """slots scatter keys and values; a slot outside the cache drops its row; the rest of the cache stays as it was; strided inputs"""
    gen = torch.Generator().manual_seed(3)
    B, L, Hq, Hk, D, rows = 2, 3, 4, 2, 64, 10
    packed = randn(gen, B, L, Hq + 2 * Hk, D, dtype=torch.bfloat16).cuda()
    q, k, v = packed[:, :, :Hq], packed[:, :, Hq:Hq + Hk], packed[:, :, Hq + Hk:]
    ck, cv = (randn(gen, B, rows, Hk, D, dtype=torch.bfloat16).cuda() for _ in range(2))
    ck0, cv0 = ck.clone(), cv.clone()
    w = torch.ones(D).cuda()
    slots = torch.tensor([[4, -1, 9], [0, 10, 3]], dtype=torch.int32).cuda()
    turns = A.rotary_turns(64, device='cuda')
    oq, ok = A.head_norm_rotate(q, k, w, w, turns, slots, out_k=ck, v=v, out_v=cv, slots=slots)
    rq, rk = A.head_norm_rotate(q.contiguous(), k.contiguous(), w, w, turns, slots)
    assert ok is ck and torch.equal(oq, rq)
    for b in range(B):
        for l in range(L):
            s = int(slots[b, l])
            if 0 <= s < rows:
                ck0[b, s], cv0[b, s] = rk[b, l], v[b, l]
    assert torch.equal(ck, ck0) and torch.equal(cv, cv0)
    # in place, and without keys
    q2 = q.contiguous()
    A.head_norm_rotate(q2, None, w, out_q=q2)
    assert torch.equal(q2, A.head_norm_rotate(q, None, w)[0])


# ------------------------------------------------------------------ summary and selection
SELECT = [  # B, Lq, Lk, Hq, Hk, D, block, qb, n, causal, ragged
    (1, 1, 1, 1, 1, 8, 64, 1, 1, True, False), (2, 1, 700, 8, 2, 64, 64, 1, 4, True, True), (1, 130, 130, 4, 4, 48, 64, 16, 2, True, False),
    (2, 65, 300, 6, 3, 40, 32, 8, 5, False, True), (1, 200, 1000, 4, 1, 128, 1, 64, 300, False, False), (1, 31, 4097, 2, 1, 256, 64, 7, 64, True, False),
    (3, 50, 20, 2, 2, 32, 64, 16, 3, True, True), (1, 5, 8192, 1, 1, 16, 1, 5, 1000, True, False),
]


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('case', SELECT)
def test_summary_and_selection(A, case, dt):
    B, Lq, Lk, Hq, Hk, D, block, qb, n, causal, ragged = case
    gen = torch.Generator().manual_seed(Lk + D)
    q, k = randn(gen, B, Lq, Hq, D, dtype=DT[dt]), randn(gen, B, Lk, Hk, D, dtype=DT[dt])
    klen = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32) if ragged else None
    qlen = torch.randint(0, Lq + 1, (B,), generator=gen, dtype=torch.int32) if ragged else None
    if ragged:
        for b in range(B):
            k[b, int(klen[b]):] = math.nan                        # never read
            q[b, int(qlen[b]):] = math.inf
    want = O.summary(k, block, klen)
    got = A.block_summary(cu(k), block, cu(klen))
    within(got, want, O.U32 * want.abs() + 1e-15, 'summary')
    for sink, local in ((1, 1), (0, 0), (2, 3)):
        sel = A.select_blocks(cu(q), got, n, block, qb, keys=Lk, causal=causal, qlen=cu(qlen), klen=cu(klen), sink=sink, local=local)
        assert torch.equal(sel.cpu(), O.select(q, got.cpu(), n, block, qb, Lk, causal, qlen, klen, sink, local)), (sink, local)


def test_selection_ties_nan_and_infinities(A):
    q = torch.ones(1, 4, 1, 8).cuda()
    s = torch.zeros(1, 600, 1, 8)
    s[0, 5, 0] = math.nan
    s[0, 7, 0, 0] = math.inf
    s[0, 9, 0, 0] = -math.inf
    s[0, 300:310] = 2.0
    s[0, 11, 0] = -0.0
    for n in (1, 3, 12, 500, 598, 599, 600, 700):
        got = A.select_blocks(q, s.cuda(), n, block=1, query_block=4, sink=0, local=0)
        assert torch.equal(got.cpu(), O.select(q.cpu(), s, n, 1, 4, 600, False, None, None, 0, 0)), n


@pytest.mark.parametrize('step', [2.0 ** -30, 2.0 ** -45])
def test_selection_of_scores_that_one_float32_holds(A, step):
    """neighbours in the order closer than fp32 can tell, a few of them and hundreds"""
    gen = torch.Generator().manual_seed(5)
    q = torch.ones(1, 2, 1, 8)
    s = torch.zeros(1, 700, 1, 8)
    s[0, :, 0, 0] = 1.0
    s[0, :, 0, 1] = torch.randperm(700, generator=gen).float() * step
    s[0, 100:200, 0, 0] = 3.0
    for n in (1, 50, 99, 101, 400, 699):
        got = A.select_blocks(cu(q), cu(s), n, block=1, query_block=2, sink=0, local=0)
        assert torch.equal(got.cpu(), O.select(q, s, n, 1, 2, 700, False, None, None, 0, 0)), n


def test_summary_of_the_newest_tokens(A):
    gen = torch.Generator().manual_seed(9)
    B, Lk, Hk, D, block = 3, 500, 2, 64, 64
    k = randn(gen, B, Lk, Hk, D, dtype=torch.bfloat16).cuda()
    for newest, lens in ((1, (1, 64, 500)), (1, (65, 0, 128)), (70, (70, 130, 500)), (600, (3, 200, 500))):
        klen = torch.tensor(lens, dtype=torch.int32).cuda()
        before = torch.full((B, 8, Hk, D), 7.0).cuda()
        got = A.block_summary(k, block, klen, newest=newest, out=before.clone())
        full = A.block_summary(k, block, klen)
        want = before.clone()
        for b, n in enumerate(lens):
            if n:
                lo, hi = max(0, n - newest) // block, (n - 1) // block
                want[b, lo:hi + 1] = full[b, lo:hi + 1]
        assert torch.equal(got, want)


# ------------------------------------------------------------------ attention
ATTN = [  # B, Lq, Lk, Hq, Hk, D, block, qb, n, causal, ragged, buckets, maxd, frames
    (1, 1, 1, 1, 1, 8, 64, 1, 1, True, False, 0, 0, False),
    (2, 1, 700, 8, 2, 128, 64, 1, 5, True, True, 32, 128, False),
    (1, 130, 130, 4, 4, 48, 64, 16, 3, True, False, 32, 100, False),
    (2, 65, 300, 6, 3, 40, 64, 8, 4, False, True, 16, 16, True),
    (1, 200, 200, 8, 1, 64, 64, 64, 4, True, False, 32, 128, False),
    (1, 96, 257, 5, 1, 96, 128, 7, 3, False, False, 8, 500, False),
    (2, 33, 10, 3, 3, 16, 64, 16, 2, True, True, 4, 16, False),
    (1, 150, 150, 2, 2, 128, 64, 32, 2, True, False, 0, 0, False),
    (1, 64, 640, 1, 1, 48, 64, 64, 10, False, False, 16, 16, True),
    (3, 4, 90, 7, 1, 112, 64, 1, 2, True, True, 2, 300, False),
    (1, 17, 1100, 2, 1, 72, 64, 17, 18, False, False, 64, 4096, False),
    (1, 40, 300, 4, 2, 24, 192, 3, 2, True, False, 16, 64, False),
]


def problem(case, dt, gen):
    B, Lq, Lk, Hq, Hk, D, block, qb, n, causal, ragged, buckets, maxd, frames = case
    T = DT[dt]
    q, k, v, g = randn(gen, B, Lq, Hq, D, dtype=T, std=1.5), randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lq, Hq, D, dtype=T)
    klen = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32) if ragged else None
    qlen = torch.randint(0, Lq + 1, (B,), generator=gen, dtype=torch.int32) if ragged else None
    nb, ng = -(-Lk // block), -(-Lq // qb)
    sel = torch.full((B, Hk, ng, n), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(Hk):
            for i in range(ng):
                m = int(torch.randint(0, min(n, nb) + 1, (1,), generator=gen)) if i % 5 == 4 else min(n, nb)     # some groups choose little or nothing
                sel[b, h, i, :m] = torch.randperm(nb, generator=gen)[:m].sort().values.to(torch.int32)
    how = dict(block=block, query_block=qb, scale=0.7 / math.sqrt(D), causal=causal, qlen=qlen, klen=klen, bucket_of=None, bias=None, q_pos=None, k_pos=None)
    if buckets:
        from adaptivepnp_sci_amd.attention import bucket_table
        how['bucket_of'] = bucket_table(buckets, maxd, bidirectional=not causal and buckets % 2 == 0)
        how['bias'] = randn(gen, buckets, Hq)
        if frames:
            how['q_pos'] = torch.arange(Lq, dtype=torch.int32).div(20, rounding_mode='floor').to(torch.int32).repeat(B, 1)
            how['k_pos'] = torch.arange(Lk, dtype=torch.int32).div(64, rounding_mode='floor').to(torch.int32).repeat(B, 1)
    if ragged:                                                    # what lies behind the sequences is never used
        for b in range(B):
            q[b, int(qlen[b]):], g[b, int(qlen[b]):] = math.nan, math.inf
            k[b, int(klen[b]):], v[b, int(klen[b]):] = math.nan, math.nan
    return q, k, v, g, sel, how


def reference(q, k, v, sel, how, dout=None):
    names = ('scale', 'causal', 'qlen', 'klen', 'bucket_of', 'bias', 'q_pos', 'k_pos')
    return O.attention(q, k, v, sel, how['block'], how['query_block'], *(how[n] for n in names), dout=dout)


def on_gpu(how):
    return {n: cu(t) if isinstance(t, torch.Tensor) else t for n, t in how.items()}


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('case', ATTN)
def test_block_attention(A, case, dt):
    q, k, v, _, sel, how = problem(case, dt, torch.Generator().manual_seed(case[1] + case[2]))
    want = reference(q, k, v, sel, how)
    out, (lse, *_) = A.block_attention(cu(q), cu(k), cu(v), cu(sel), save=True, **on_gpu(how))
    qlen = how['qlen']
    live = torch.ones(q.shape[:2], dtype=torch.bool) if qlen is None else torch.arange(q.shape[1])[None] < qlen[:, None]
    within(out, *want['out'], 'out')
    within(lse.cpu().transpose(1, 2)[live], want['lse'][0].transpose(1, 2)[live], want['lse'][1].transpose(1, 2)[live], 'lse')
    plain = A.block_attention(cu(q), cu(k), cu(v), cu(sel), **on_gpu(how))
    within(plain, *want['out'], 'out without save')
    assert torch.equal(plain, A.block_attention(cu(q), cu(k), cu(v), cu(sel), **on_gpu(how)))
    if dt == 'f32':
        assert torch.equal(plain, out)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('B,L,Hq,Hk,D,qb,new', [(1, 130, 2, 1, 64, 16, 0), (2, 96, 1, 1, 128, 64, 0), (1, 70, 3, 3, 48, 8, 0), (1, 200, 2, 2, 96, 200, 0),
                                                (2, 90, 8, 2, 128, 1, 3), (1, 300, 4, 1, 8, 3, 5)])
def test_what_a_later_key_holds_does_not_reach_an_earlier_query(A, B, L, Hq, Hk, D, qb, new, dt):
    """infinities and NaN in keys and values of causal sequences: the queries that see them, and only those, show them"""
    gen = torch.Generator().manual_seed(L)
    Lq, T = new or L, DT[dt]
    q, k, v = randn(gen, B, Lq, Hq, D, dtype=T), randn(gen, B, L, Hk, D, dtype=T), randn(gen, B, L, Hk, D, dtype=T)
    at = [L - 2, L - 1] if new else [L // 2, L // 2 + 1, L - 1]
    v[0, at[0], 0, 3], v[0, at[1], 0, D - 1], v[-1, at[-1], -1, 0] = math.inf, -math.inf, math.nan
    k[0, L - 1, -1, 1] = math.nan
    nb, ng = -(-L // 64), -(-Lq // qb)
    sel = torch.arange(nb, dtype=torch.int32).expand(B, Hk, ng, nb).contiguous()
    from adaptivepnp_sci_amd.attention import bucket_table
    how = dict(block=64, query_block=qb, scale=0.3 / math.sqrt(D), causal=True, qlen=None, klen=None, bucket_of=bucket_table(8, 40, False),
               bias=0.3 * randn(gen, 8, Hq), q_pos=None, k_pos=None)
    val, err = reference(q, k, v, sel, how)['out']
    assert torch.isfinite(val).any() and not torch.isfinite(val).all()
    got = A.block_attention(cu(q), cu(k), cu(v), cu(sel), **on_gpu(how)).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(val)) and torch.equal(torch.isinf(got), torch.isinf(val))
    within(got.nan_to_num(nan=0.0), val.nan_to_num(nan=0.0), err.nan_to_num(nan=0.0), 'out')


def again(t, times):
    return t.repeat(times, *[1] * (t.dim() - 1))


def of_all(how, times):
    return on_gpu({n: again(t, times) if n in ('qlen', 'klen', 'q_pos', 'k_pos') and t is not None else t for n, t in how.items()})


@pytest.mark.parametrize('times,case', [
    (37, (2, 100, 300, 8, 2, 128, 64, 16, 4, True, True, 32, 128, False)),
    (210, (1, 65, 257, 3, 1, 112, 64, 16, 3, False, True, 16, 16, True)),
    (33, (1, 200, 300, 8, 2, 128, 64, 64, 3, True, False, 0, 0, False)),
    (26, (2, 130, 400, 5, 1, 96, 128, 32, 3, True, True, 8, 60, False)),
    (86, (1, 150, 150, 4, 1, 72, 64, 13, 3, True, False, 4, 16, False)),
])
def test_more_workgroups_than_two_a_cu(A, times, case):
    """wide bf16 heads have a kernel of their own there: the same sequences many times over, each with the result of the first"""
    q, k, v, _, sel, how = problem(case, 'bf16', torch.Generator().manual_seed(case[1] + case[2]))
    want = reference(q, k, v, sel, how)['out']
    args = [cu(again(t, times)) for t in (q, k, v, sel)]
    for save in (False, True):
        got = A.block_attention(*args, save=save, **of_all(how, times))
        got = (got[0] if save else got).unflatten(0, (times, q.shape[0]))
        within(got[0], *want, 'out')
        assert torch.equal(got, got[:1].expand_as(got))


@pytest.mark.parametrize('times,L,Hq,Hk,D,qb', [(58, 130, 8, 2, 128, 16), (90, 140, 4, 1, 96, 64), (60, 130, 4, 1, 128, 64)])
def test_values_that_are_not_numbers_with_more_workgroups_than_two_a_cu(A, times, L, Hq, Hk, D, qb):
    gen = torch.Generator().manual_seed(L)
    q, k, v = (randn(gen, 1, L, h, D, dtype=torch.bfloat16) for h in (Hq, Hk, Hk))
    v[0, L // 2, 0, 3], v[0, L // 2 + 1, 0, D - 1], v[0, L - 1, -1, 0] = math.inf, -math.inf, math.nan
    nb, ng = -(-L // 64), -(-L // qb)
    sel = torch.arange(nb, dtype=torch.int32).expand(1, Hk, ng, nb).contiguous()
    from adaptivepnp_sci_amd.attention import bucket_table
    how = dict(block=64, query_block=qb, scale=0.3 / math.sqrt(D), causal=True, qlen=None, klen=None, bucket_of=bucket_table(8, 40, False),
               bias=0.3 * randn(gen, 8, Hq), q_pos=None, k_pos=None)
    val, err = reference(q, k, v, sel, how)['out']
    assert torch.isfinite(val).any() and not torch.isfinite(val).all()
    got = A.block_attention(*(cu(again(t, times)) for t in (q, k, v, sel)), **of_all(how, times)).double().cpu()
    for one in (got[:1], got[-1:]):
        assert torch.equal(torch.isnan(one), torch.isnan(val)) and torch.equal(torch.isinf(one), torch.isinf(val))
        within(one.nan_to_num(nan=0.0), val.nan_to_num(nan=0.0), err.nan_to_num(nan=0.0), 'out')
    assert torch.equal(got.nan_to_num(nan=0.0), got[:1].nan_to_num(nan=0.0).expand_as(got))


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('low', [-math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min])
def test_a_bias_of_the_lowest_value_masks(A, low, dt):
    """some buckets masked for one head, every one for another: zeros there, and no gradient"""
    gen = torch.Generator().manual_seed(17)
    T = DT[dt]
    q, k, v, g = randn(gen, 1, 100, 2, 64, dtype=T), randn(gen, 1, 100, 1, 64, dtype=T), randn(gen, 1, 100, 1, 64, dtype=T), randn(gen, 1, 100, 2, 64, dtype=T)
    sel = torch.tensor([0, 1], dtype=torch.int32).expand(1, 1, 7, 2).contiguous()
    from adaptivepnp_sci_amd.attention import bucket_table
    bias = randn(gen, 8, 2)
    bias[2:, 0], bias[:, 1] = low, low
    how = dict(block=64, query_block=16, scale=0.2, causal=False, qlen=None, klen=None, bucket_of=bucket_table(8, 20), bias=bias, q_pos=None, k_pos=None)
    want = reference(q, k, v, sel, how, dout=g)
    args = [cu(t) for t in (q, k, v, sel)]
    out, saved = A.block_attention(*args, save=True, **on_gpu(how))
    within(out, *want['out'], 'out')
    assert not out[:, :, 1].any() and torch.equal(saved[0][:, 1].cpu(), torch.full((1, 100), -math.inf))
    for name, t in zip(('dq', 'dk', 'dv', 'dbias'), A.block_attention_backward(cu(g), *args, saved, **on_gpu(how))):
        within(t, *want[name], name)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('case', ATTN)
def test_block_attention_backward(A, case, dt):
    q, k, v, g, sel, how = problem(case, dt, torch.Generator().manual_seed(case[1] * 3 + case[2]))
    want = reference(q, k, v, sel, how, dout=g)
    args = [cu(t) for t in (q, k, v, sel)]
    _, saved = A.block_attention(*args, save=True, **on_gpu(how))
    got = A.block_attention_backward(cu(g), *args, saved, **on_gpu(how))
    for name, t in zip(('dq', 'dk', 'dv', 'dbias'), got):
        if t is None:
            assert name == 'dbias' and how['bias'] is None
            continue
        within(t, *want[name], name)
    again = A.block_attention_backward(cu(g), *args, saved, **on_gpu(how))
    assert all(x is None or torch.equal(x, y) for x, y in zip(got, again))
