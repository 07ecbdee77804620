"""-m gpu: the block-attention operators at the edges of what they take: large biases beside rows that do not exist, keys that a bias masks
and what they hold, the digits of the weights.  Tolerances as in test_gpu_attention.py: bounds of the roundings (oracle/attention.py)."""
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


def on_gpu(how):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in how.items()}


def reference(q, k, v, sel, how, dout=None, **kw):
    names = ('scale', 'causal', 'qlen', 'klen', 'bucket_of', 'bias', 'q_pos', 'k_pos')
    return O.attention(q, k, v, sel, how['block'], how['query_block'], *(how.get(n) for n in names), dout=dout, **kw)


def within(got, val, err, what):
    """where a value is none of the real numbers, the same one; elsewhere inside the bound"""
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(val)) and torch.equal(torch.isinf(got), torch.isinf(val)), what
    fin = torch.isfinite(val)
    d = (got[fin] - val[fin]).abs()
    assert not (d > err[fin] + 1e-37).any(), f'{what}: worst {float((d / (err[fin] + 1e-37)).max()):.3g} x the bound'


def every_block(B, Hk, Lq, Lk, qb, block=64):
    nb = -(-Lk // block)
    return torch.arange(nb, dtype=torch.int32).expand(B, Hk, -(-Lq // qb), nb).contiguous()


# ------------------------------------------------------------------ rows that do not exist
@pytest.mark.parametrize('add', [100.0, 1e4, -1e4])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('B,Lq,Lk,Hq,Hk,D,qb,causal,ragged', [
    (2, 50, 300, 6, 2, 64, 8, False, True),                       # 24 rows a group, lengths
    (1, 33, 130, 3, 1, 48, 16, True, False),                      # 48 rows: half of a wave
    (1, 70, 200, 1, 1, 56, 64, False, False),                     # a last group of 6 rows
    (2, 3, 100, 4, 1, 128, 1, False, True),                       # 4 rows, single queries
])
def test_large_biases_beside_rows_that_do_not_exist(A, B, Lq, Lk, Hq, Hk, D, qb, causal, ragged, dt, add):
    """a constant on every bias changes no weight, however large: no row that does not exist may show its exponential"""
    gen, T = torch.Generator().manual_seed(Lq + D), DT[dt]
    q, g = randn(gen, B, Lq, Hq, D, dtype=T), randn(gen, B, Lq, Hq, D, dtype=T)
    k, v = randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T)
    qlen = torch.tensor([Lq - 2, 1][:B], dtype=torch.int32) if ragged else None
    klen = torch.tensor([Lk, Lk - 30][:B], dtype=torch.int32) if ragged else None
    how = dict(block=64, query_block=qb, scale=0.7 / math.sqrt(D), causal=causal, qlen=qlen, klen=klen, bucket_of=A.bucket_table(8, 20, not causal),
               bias=randn(gen, 8, Hq) + add, q_pos=None, k_pos=None)
    sel = every_block(B, Hk, Lq, Lk, qb)
    want = reference(q, k, v, sel, how, dout=g)
    args = [t.cuda() for t in (q, k, v, sel)]
    out, saved = A.block_attention(*args, save=True, **on_gpu(how))
    within(out, *want['out'], 'out')
    for name, t in zip(('dq', 'dk', 'dv', 'dbias'), A.block_attention_backward(g.cuda(), *args, saved, **on_gpu(how))):
        within(t, *want[name], name)


# ------------------------------------------------------------------ keys that a bias masks
def spoil(gen, k, v, at):
    """infinities and NaN in the keys and values at those places"""
    for i, x in enumerate(at):
        k[..., x, :, i % k.shape[-1]] = (math.nan, math.inf, -math.inf)[i % 3]
        v[..., x, :, (3 * i + 1) % k.shape[-1]] = (math.inf, math.nan, -math.inf)[i % 3]


MASKED = [  # times, B, Lq, Lk, Hq, Hk, D, qb
    (1, 1, 150, 150, 2, 1, 64, 16), (1, 2, 70, 70, 1, 1, 48, 64), (1, 1, 90, 90, 6, 2, 128, 8), (1, 1, 64, 64, 1, 1, 8, 200), (1, 1, 100, 100, 3, 3, 112, 32),
    (90, 1, 130, 130, 8, 2, 128, 16), (90, 1, 140, 140, 4, 1, 96, 64),      # (more than two workgroups a CU)
]


@pytest.mark.parametrize('low', [-math.inf, torch.finfo(torch.float32).min])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('times,B,Lq,Lk,Hq,Hk,D,qb', MASKED)
def test_what_a_key_masked_by_its_bias_holds_does_not_reach_a_query(A, times, B, Lq, Lk, Hq, Hk, D, qb, dt, low):
    """buckets of the keys behind a query masked, for one head or for all: a causal mask in another form"""
    gen, T = torch.Generator().manual_seed(Lq * D), DT[dt]
    q, k, v = randn(gen, B, Lq, Hq, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T)
    spoil(gen, k, v, [Lk // 2, Lk // 2 + 1, Lk - 2, Lk - 1])
    for some in (False, True):
        bias = 0.3 * randn(gen, 8, Hq)
        bias[4:, :1 if some else None] = low
        how = dict(block=64, query_block=qb, scale=0.3 / math.sqrt(D), causal=False, qlen=None, klen=None, bucket_of=A.bucket_table(8, 40), bias=bias,
                   q_pos=None, k_pos=None)
        sel = every_block(B, Hk, Lq, Lk, qb)
        val, err = reference(q, k, v, sel, how)['out']
        assert torch.isfinite(val).any() and not torch.isfinite(val).all()
        got = A.block_attention(*(t.repeat(times, 1, 1, 1).cuda() for t in (q, k, v, sel)), **on_gpu(how))
        within(got[:B], val, err, 'out')
        within(got[-B:], val, err, 'out of the last')


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('at', [[300, 301, 700, 1279], [300, 301, 1279]])        # (head 0 sees key 700)
@pytest.mark.parametrize('Lq,qb,D', [(128, 64, 56), (128, 16, 128), (2, 1, 128), (1, 1, 64)])
def test_frames_masked_by_their_distance(A, Lq, qb, D, at, dt):
    """whole tiles of one bucket, masked; the keys split over workgroups where there are few queries"""
    gen, T, Lk = torch.Generator().manual_seed(Lq + D), DT[dt], 1280
    q, k, v = randn(gen, 1, Lq, 2, D, dtype=T), randn(gen, 1, Lk, 1, D, dtype=T), randn(gen, 1, Lk, 1, D, dtype=T)
    spoil(gen, k, v, at)
    table = torch.arange(9, dtype=torch.int32)                                # a bucket for every distance up to four frames
    bias = 0.3 * randn(gen, 9, 2)
    bias[torch.tensor([0, 1, 7, 8]), 0] = -math.inf                          # head 0 sees two frames around its own
    bias[torch.tensor([0, 3, 6, 8]), 1] = -math.inf
    how = dict(block=64, query_block=qb, scale=0.3 / math.sqrt(D), causal=False, qlen=None, klen=None, bucket_of=table, bias=bias,
               q_pos=torch.full((1, Lq), 5, dtype=torch.int32), k_pos=(torch.arange(Lk, dtype=torch.int32) // 128)[None].contiguous())
    sel = every_block(1, 1, Lq, Lk, qb)
    val, err = reference(q, k, v, sel, how)['out']
    assert 700 in at or torch.isfinite(val[:, :, 0]).all()
    within(A.block_attention(q.cuda(), k.cuda(), v.cuda(), sel.cuda(), **on_gpu(how)), val, err, 'out')


@pytest.mark.parametrize('save', [False, True])
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('times,B,Lq,Lk,Hq,Hk,D,qb,causal', [
    (1, 1, 100, 300, 2, 1, 64, 16, False), (1, 2, 130, 130, 2, 2, 128, 32, True), (1, 1, 1, 900, 4, 1, 128, 1, False), (1, 1, 70, 130, 1, 1, 56, 64, False),
    (90, 1, 130, 130, 8, 2, 128, 16, True), (90, 1, 140, 140, 4, 1, 96, 64, False), (60, 1, 130, 200, 4, 1, 128, 64, False),
])
def test_an_infinite_value_arrives_as_one(A, times, B, Lq, Lk, Hq, Hk, D, qb, causal, dt, save):
    """infinities and NaN among values that are seen: in their columns, and in no other"""
    gen, T = torch.Generator().manual_seed(Lq + Lk + D), DT[dt]
    q, k, v = randn(gen, B, Lq, Hq, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T)
    v[0, 0, 0, 1], v[0, Lk // 2, 0, 5], v[-1, 3, -1, D - 1] = math.inf, -math.inf, math.nan
    how = dict(block=64, query_block=qb, scale=0.3 / math.sqrt(D), causal=causal, bucket_of=A.bucket_table(8, 40, not causal), bias=0.3 * randn(gen, 8, Hq))
    sel = every_block(B, Hk, Lq, Lk, qb)
    val, err = reference(q, k, v, sel, how)['out']
    assert torch.isfinite(val).any() and torch.isinf(val).any() and torch.isnan(val).any()
    got = A.block_attention(*(t.repeat(times, 1, 1, 1).cuda() for t in (q, k, v, sel)), save=save, **on_gpu(how))
    got = got[0] if save else got
    within(got[:B], val, err, 'out')
    within(got[-B:], val, err, 'out of the last')


# ------------------------------------------------------------------ sizes at the ends of 32 bits
@pytest.mark.parametrize('block', [2 ** 31 - 1, 2 ** 31 - 64, 2 ** 30])
def test_one_block_of_any_length(A, block):
    """a block as long as a 32-bit number goes: all keys are its own"""
    gen = torch.Generator().manual_seed(4)
    q, k = randn(gen, 2, 9, 2, 16), randn(gen, 2, 100, 1, 16)
    klen, qlen = torch.tensor([100, 3], dtype=torch.int32), torch.tensor([9, 5], dtype=torch.int32)
    summ = A.block_summary(k.cuda(), block, klen.cuda())
    val = O.summary(k, block, klen)
    within(summ, val, O.U32 * val.abs() + 1e-15, 'summary')
    for causal in (False, True):
        for sink, local in ((0, 0), (1, 1), (0, 2)):
            got = A.select_blocks(q.cuda(), summ, 2, block, 4, keys=100, causal=causal, qlen=qlen.cuda(), klen=klen.cuda(), sink=sink, local=local)
            assert torch.equal(got.cpu(), O.select(q, summ.cpu(), 2, block, 4, 100, causal, qlen, klen, sink, local)), (causal, sink, local)
    got = A.select_blocks(q.cuda(), summ, 2, block, 4)              # (keys: as many as the block)
    assert torch.equal(got.cpu(), torch.tensor([0, -1], dtype=torch.int32).expand(2, 1, 3, 2))


@pytest.mark.parametrize('newest', [2 ** 31 - 1, 2 ** 31 - 64, 500])
def test_every_token_is_among_the_newest(A, newest):
    gen = torch.Generator().manual_seed(6)
    k, klen = randn(gen, 3, 500, 2, 64).cuda(), torch.tensor([500, 0, 65], dtype=torch.int32).cuda()
    got, want = A.block_summary(k, 64, klen, newest=newest, out=torch.full((3, 8, 2, 64), 7.0).cuda()), A.block_summary(k, 64, klen)
    for b, n in enumerate((8, 0, 2)):
        assert torch.equal(got[b, :n], want[b, :n]) and (got[b, n:] == 7).all()


# ------------------------------------------------------------------ the digits of the weights
DIGITS = [  # times, B, Lq, Lk, Hq, Hk, D, qb, causal
    (1, 1, 96, 257, 4, 1, 64, 16, False), (1, 2, 130, 130, 2, 2, 128, 16, True), (1, 1, 3, 700, 8, 2, 128, 1, True), (1, 1, 1, 1500, 4, 1, 40, 1, False),
    (1, 1, 200, 200, 1, 1, 96, 64, False), (90, 1, 130, 130, 8, 2, 128, 16, True), (90, 1, 140, 140, 4, 1, 96, 64, False),
]


@pytest.mark.parametrize('times,B,Lq,Lk,Hq,Hk,D,qb,causal', DIGITS)
def test_bf16_weights_keep_sixteen_digits(A, times, B, Lq, Lk, Hq, Hk, D, qb, causal):
    """only the result is rounded to bf16: where the values cancel, a weight of eight digits is off by far more than that.  Two bf16 numbers
    hold a weight to 2^-8 of 2^-8 of it (half a step of what the first left over)"""
    gen, T = torch.Generator().manual_seed(Lq + D), torch.bfloat16
    q, k, v = randn(gen, B, Lq, Hq, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T), randn(gen, B, Lk, Hk, D, dtype=T)
    how = dict(block=64, query_block=qb, scale=0.5 / math.sqrt(D), causal=causal, bucket_of=A.bucket_table(8, 20, not causal), bias=randn(gen, 8, Hq))
    sel = every_block(B, Hk, Lq, Lk, qb)
    val, err = reference(q, k, v, sel, how, parts=2)['out']
    args = [t.repeat(times, 1, 1, 1).cuda() for t in (q, k, v, sel)]
    for save in (False, True):
        got = A.block_attention(*args, save=save, **on_gpu(how))
        got = got[0] if save else got
        within(got[:B], val, err, f'out, save {save}')
        within(got[-B:], val, err, f'out of the last, save {save}')


@pytest.mark.parametrize('B,Lq,Lk,Hq,Hk,D,qb,causal', [c[1:] for c in DIGITS[:5]])
def test_bf16_gradients_keep_sixteen_digits(A, B, Lq, Lk, Hq, Hk, D, qb, causal):
    gen, T = torch.Generator().manual_seed(Lq + D), torch.bfloat16
    q, k, v, g = (randn(gen, B, L, h, D, dtype=T) for L, h in ((Lq, Hq), (Lk, Hk), (Lk, Hk), (Lq, Hq)))
    how = dict(block=64, query_block=qb, scale=0.5 / math.sqrt(D), causal=causal, bucket_of=A.bucket_table(8, 20, not causal), bias=randn(gen, 8, Hq))
    sel = every_block(B, Hk, Lq, Lk, qb)
    want = reference(q, k, v, sel, how, dout=g, parts=2)
    args = [t.cuda() for t in (q, k, v, sel)]
    _, saved = A.block_attention(*args, save=True, **on_gpu(how))
    for name, t in zip(('dq', 'dk', 'dv', 'dbias'), A.block_attention_backward(g.cuda(), *args, saved, **on_gpu(how))):
        within(t, *want[name], name)


# ------------------------------------------------------------------ results in place
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('Lq,Lk,qb', [(150, 150, 16), (2, 2000, 1)])
def test_results_in_the_queries_own_memory(A, Lq, Lk, qb, dt):
    """views of one projection, written in place: keys split over workgroups, and not"""
    gen, T = torch.Generator().manual_seed(Lq), DT[dt]
    packed = randn(gen, 2, Lq, 6, 64, dtype=T).cuda()
    k, v = randn(gen, 2, Lk, 2, 64, dtype=T).cuda(), randn(gen, 2, Lk, 2, 64, dtype=T).cuda()
    q = packed[:, :, 1:5]
    sel, how = every_block(2, 2, Lq, Lk, qb).cuda(), dict(block=64, query_block=qb, causal=True)
    want, before = A.block_attention(q, k, v, sel, **how), packed.clone()
    assert A.block_attention(q, k, v, sel, out=q, **how) is q
    assert torch.equal(q, want) and torch.equal(packed[:, :, [0, 5]], before[:, :, [0, 5]])
    w, turns = torch.ones(64).cuda(), A.rotary_turns(32, device='cuda')
    a, b = packed[:, :, :4], packed[:, :, 4:]
    wa, wb = A.head_norm_rotate(a, b, w, w, turns)
    A.head_norm_rotate(a, b, w, w, turns, out_q=a, out_k=b)
    assert torch.equal(a, wa) and torch.equal(b, wb)


# ------------------------------------------------------------------ beside autograd
def test_results_beside_autograd(A):
    """results require no gradient; a given one that autograd had saved is noticed"""
    w = torch.ones(64, device='cuda', requires_grad=True)
    q, k = (torch.randn(1, 64, 2, 64, device='cuda', requires_grad=True) for _ in range(2))
    sel = every_block(1, 2, 64, 64, 16).cuda()
    results = [*A.head_norm_rotate(q, k, w, w), A.block_summary(k), A.block_attention(q, k, k, sel, query_block=16),
               *A.block_attention(q, k, k, sel, query_block=16, save=True)[1]]
    assert not any(t.requires_grad for t in results)
    for write in (lambda t: A.head_norm_rotate(q, k, w, w, out_q=t), lambda t: A.head_norm_rotate(q, k, w, w, out_k=t),
                  lambda t: A.head_norm_rotate(q, k, w, w, out_k=torch.empty_like(t), v=k, out_v=t),
                  lambda t: A.block_attention(q, k, k, sel, query_block=16, out=t), lambda t: A.block_summary(k, 1, out=t)):
        t = torch.zeros(1, 64, 2, 64, device='cuda')
        loss = (t * q).sum()                              # (saves t for the gradient of q)
        write(t)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
    with torch.inference_mode():
        t = torch.zeros(1, 64, 2, 64, device='cuda')
    assert A.block_attention(q, k, k, sel, query_block=16, out=t) is t and torch.equal(t, results[3])


# ------------------------------------------------------------------ grids past 2^24 workgroups
def room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f'{gib} GiB of free memory needed')


def test_a_norm_of_more_tokens_than_a_row_of_the_grid(A):
    """2^28 tokens and a few, one head of 8"""
    room(12)
    L = (1 << 28) + 5
    x = torch.full((1, L, 1, 8), 7.0, dtype=torch.bfloat16, device='cuda')
    w, turns = torch.arange(1.0, 9.0, device='cuda'), A.rotary_turns(8, device='cuda')
    at = [0, 1, (1 << 26) - 1, 1 << 26, (1 << 28) - 1, 1 << 28, L - 1]
    gen = torch.Generator().manual_seed(1)
    rows = randn(gen, 1, len(at), 1, 8, dtype=torch.bfloat16).cuda()
    x[:, at] = rows
    pos = torch.tensor([at], dtype=torch.int32, device='cuda')
    want = A.head_norm_rotate(rows, None, w, None, turns, pos)[0]
    A.head_norm_rotate(x, None, w, None, turns, out_q=x)
    assert torch.equal(x[:, at], want) and not (x[0, -1000:-5] == 7).all(-1).any()
    del x
    torch.cuda.empty_cache()


def test_gradients_of_more_blocks_than_a_row_of_the_grid(A):
    """2^20 blocks of 64 keys and a few, 128 wide: 16 workgroups each join a block's chunks"""
    room(150)
    B, Lk, D, T = 32, (1 << 21) + 64, 128, torch.bfloat16
    gen = torch.Generator().manual_seed(2)
    k0, v0 = randn(gen, 1, 64, 1, D, dtype=T).cuda(), randn(gen, 1, 64, 1, D, dtype=T).cuda()
    k, v = torch.zeros(1, Lk, 1, D, dtype=T, device='cuda'), torch.zeros(1, Lk, 1, D, dtype=T, device='cuda')
    k[:, -64:], v[:, -64:] = k0, v0
    q, g = randn(gen, B, 1, 1, D, dtype=T).cuda(), randn(gen, B, 1, 1, D, dtype=T).cuda()
    how = dict(block=64, query_block=1)

    def grads(k, v, last):
        sel = torch.full((B, 1, 1, 1), last, dtype=torch.int32, device='cuda')
        args = (q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), sel)
        saved = A.block_attention(*args, save=True, **how)[1]
        return A.block_attention_backward(g, *args, saved, **how)[:3]
    want = grads(k0, v0, 0)
    got = grads(k, v, Lk // 64 - 1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][:, -64:], want[1]) and torch.equal(got[2][:, -64:], want[2])
    for t in got[1:]:
        assert not any(t[b, i:i + (1 << 19)].any() for b in range(B) for i in range(0, Lk - 64, 1 << 19) if i + (1 << 19) <= Lk - 64)
    del got, t
    torch.cuda.empty_cache()


# ------------------------------------------------------------------ views
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
@pytest.mark.parametrize('Lq,Lk,Hq,Hk,D,qb', [(190, 190, 4, 2, 40, 16), (150, 150, 8, 2, 128, 16), (3, 1500, 4, 1, 64, 1), (70, 70, 1, 1, 48, 64)])
def test_a_strided_result_holds_the_bits_of_a_tight_one(A, Lq, Lk, Hq, Hk, D, qb, dt):
    """columns and heads of a wider tensor, and (B, H, L, D) storage: every row in its place, nothing beside it"""
    gen, T = torch.Generator().manual_seed(Lq + D), DT[dt]
    q, k, v = randn(gen, 2, Lq, Hq, D, dtype=T).cuda(), randn(gen, 2, Lk, Hk, D, dtype=T).cuda(), randn(gen, 2, Lk, Hk, D, dtype=T).cuda()
    sel = every_block(2, Hk, Lq, Lk, qb).cuda()
    how = dict(block=64, query_block=qb, causal=True, bucket_of=A.bucket_table(8, 20, False, device='cuda'), bias=randn(gen, 8, Hq).cuda())
    for save in (False, True):
        want = A.block_attention(q, k, v, sel, save=save, **how)
        want = want[0] if save else want
        assert want.float().abs().amax() > 0
        wide = torch.full((2, Lq, Hq + 2, 2 * D), 3.0, dtype=T).cuda()
        A.block_attention(q, k, v, sel, out=wide[:, :, 1:-1, :D], save=save, **how)
        assert torch.equal(wide[:, :, 1:-1, :D], want)
        assert (wide[..., D:] == 3).all() and (wide[:, :, [0, -1]] == 3).all()
        heads = torch.full((2, Hq, Lq + 1, D), 3.0, dtype=T).cuda()
        A.block_attention(q, k, v, sel, out=heads.transpose(1, 2)[:, :Lq], save=save, **how)
        assert torch.equal(heads.transpose(1, 2)[:, :Lq], want) and (heads[:, :, Lq] == 3).all()
