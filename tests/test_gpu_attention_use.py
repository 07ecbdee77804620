"""-m gpu: the block-attention operators the way programs use them: a cache that grows token by token, a training step, captured graphs,
other streams, views, long caches, lists with odd entries.  Tolerances as in test_gpu_attention.py: bounds of the roundings."""
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


def randn(seed, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def within(got, val, err, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    d = (got - val).abs()
    assert not (d > err + 1e-37).any(), f'{what}: worst {float((d / (err + 1e-37)).max()):.3g} x the bound'


# ------------------------------------------------------------------ a run of them together
class Decoder:
    """a layer's cache and one step of it: norm and rotation into the cache, summary of the touched block, selection, attention"""

    def __init__(self, A, B, Lmax, Hq, Hk, D, T, n, buckets=8, maxd=60):
        self.A, self.n, self.D, self.T = A, n, D, T
        self.kc, self.vc = (torch.zeros(B, Lmax, Hk, D, dtype=T).cuda() for _ in range(2))
        self.summary = torch.zeros(B, -(-Lmax // 64), Hk, D).cuda()
        self.wq, self.wk = 1 + 0.2 * randn(1, D).cuda(), 1 + 0.2 * randn(2, D).cuda()
        self.turns = A.rotary_turns(D // 16 * 8, device='cuda')
        self.bucket_of, self.bias = A.bucket_table(buckets, maxd, False, device='cuda'), randn(3, buckets, Hq).cuda()

    def how(self, klen):
        return dict(block=64, query_block=1, scale=0.6 / math.sqrt(self.D), causal=True, klen=klen, bucket_of=self.bucket_of, bias=self.bias)

    def step(self, q, k, v, klen):
        """one new token a sequence, at position klen (before it)"""
        slots = klen[:, None].contiguous()
        q, _ = self.A.head_norm_rotate(q, k, self.wq, self.wk, self.turns, slots, out_k=self.kc, v=v, out_v=self.vc, slots=slots)
        now = klen + 1
        self.A.block_summary(self.kc, 64, now, newest=1, out=self.summary)
        sel = self.A.select_blocks(q, self.summary, self.n, 64, 1, keys=self.kc.shape[1], causal=True, klen=now)
        return q, sel, now, self.A.block_attention(q, self.kc, self.vc, sel, **self.how(now))


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_a_cache_that_grows(A, dt):
    B, Lmax, Hq, Hk, D, T = 3, 330, 6, 2, 64, DT[dt]
    d = Decoder(A, B, Lmax, Hq, Hk, D, T, 3)
    klen = torch.tensor([0, 63, 250], dtype=torch.int32)
    for b in range(B):                                    # what the sequences hold already
        for t in range(int(klen[b])):
            d.kc[b, t], d.vc[b, t] = (randn(1000 * b + t + s, Hk, D, dtype=T).cuda() for s in (0, 500000))
    d.summary.copy_(A.block_summary(d.kc, 64, klen.cuda()))
    for i in range(70):
        new = [randn(7000 + 10 * i + s, B, 1, h, D, dtype=T).cuda() for s, h in ((0, Hq), (1, Hk), (2, Hk))]
        q, sel, now, out = d.step(*new, klen.cuda())
        if i % 9 == 0 or i > 66:
            kc, vc, now_ = d.kc.cpu(), d.vc.cpu(), now.cpu()
            val = O.norm_rotate(new[1].cpu(), d.wk.cpu(), d.turns.cpu(), klen[:, None])
            got = torch.stack([kc[b, int(klen[b])] for b in range(B)])[:, None]
            within(got, val, O.U[T] * (1 + 2 ** -7) * val.abs() + 2.0 ** -29 * val.abs().amax(-1, keepdim=True) * 2, 'key in the cache')
            assert all(torch.equal(vc[b, int(klen[b])], new[2][b, 0].cpu()) for b in range(B))
            assert torch.equal(d.summary, A.block_summary(d.kc, 64, now))
            assert torch.equal(sel.cpu(), O.select(q.cpu(), d.summary.cpu(), 3, 64, 1, Lmax, True, None, now_))
            want = O.attention(q.cpu(), kc, vc, sel.cpu(), 64, 1, 0.6 / math.sqrt(D), True, None, now_, d.bucket_of.cpu(), d.bias.cpu())
            within(out, *want['out'], f'step {i}')
        klen = klen + 1


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_a_training_step(A, dt):
    """norm, rotation, selection, attention and all the way back, shared key heads; the gradients of the raw queries and keys against
    64 bits, the bounds of the attention's gradients carried through the norm's"""
    B, L, Hq, Hk, D, T, rot = 2, 200, 4, 2, 48, DT[dt], 32
    q0, k0, v, g = randn(1, B, L, Hq, D, dtype=T, std=2), randn(2, B, L, Hk, D, dtype=T), randn(3, B, L, Hk, D, dtype=T), randn(4, B, L, Hq, D, dtype=T)
    wq, wk, turns = 1 + 0.2 * randn(5, D), 1 + 0.2 * randn(6, D), A.rotary_turns(rot)
    bucket_of, bias = A.bucket_table(8, 60, False), randn(7, 8, Hq)
    c = [t.cuda() for t in (q0, k0, v, g, wq, wk, turns, bucket_of, bias)]
    q, k = A.head_norm_rotate(c[0], c[1], c[4], c[5], c[6])
    sel = A.select_blocks(q, A.block_summary(k, 64), 2, 64, 16, keys=L, causal=True)
    how = dict(block=64, query_block=16, scale=0.5 / math.sqrt(D), causal=True, bucket_of=c[7], bias=c[8])
    out, saved = A.block_attention(q, k, c[2], sel, save=True, **how)
    dq, dk, dv, dbias = A.block_attention_backward(c[3], q, k, c[2], sel, saved, **how)
    dq0, dk0, dwq, dwk = A.head_norm_rotate_backward(dq, dk, c[0], c[1], c[4], c[5], c[6])
    ref = O.attention(q.cpu(), k.cpu(), v, sel.cpu(), 64, 16, how['scale'], True, None, None, bucket_of, bias, dout=g)
    for name, t in (('out', out), ('dv', dv), ('dbias', dbias)):
        within(t, *ref[name], name)
    h = rot // 2
    ang = torch.arange(L).double()[None, :, None] * turns
    ang = 2 * math.pi * (ang - ang.floor())
    co, si = ang.cos()[:, :, None], ang.sin()[:, :, None]
    for name, x, w, got, gw in (('dq', q0, wq, dq0, dwq), ('dk', k0, wk, dk0, dwk)):
        val, err = ref[name]
        xx, ww = x.double().requires_grad_(), w.double().requires_grad_()
        r = torch.rsqrt(xx.square().mean(-1, keepdim=True) + 1e-6)
        y = xx * r * ww
        y = torch.cat([y[..., :h] * co - y[..., h:rot] * si, y[..., h:rot] * co + y[..., :h] * si, y[..., rot:]], -1)
        y.backward(val)
        r, xd, wd = r.detach(), x.double().abs(), w.double().abs()
        e = torch.cat([co.abs() * err[..., :h] + si.abs() * err[..., h:rot], co.abs() * err[..., h:rot] + si.abs() * err[..., :h], err[..., rot:]], -1)
        slack = r * (wd * e + xd * r * (wd * xd * r * e).mean(-1, keepdim=True))
        size = xx.grad.abs().amax(-1, keepdim=True)
        within(got, xx.grad, slack * (1 + 2 ** -7) + O.U[T] * (1 + 2 ** -7) * xx.grad.abs() + 2.0 ** -29 * size, name + ' raw')
        within(gw, ww.grad, (e * xd * r).sum((0, 1, 2)) + 2.0 ** -22 * (val.abs() * xd.amax() * r).sum((0, 1, 2)), 'dw of ' + name)


# ------------------------------------------------------------------ graphs and streams
def test_a_captured_step_replays(A):
    """the whole step in a graph: every replay against the eager step, other work and other inputs between them"""
    B, Lmax, Hq, Hk, D, T = 2, 400, 8, 2, 64, torch.bfloat16
    fast, slow = Decoder(A, B, Lmax, Hq, Hk, D, T, 3), Decoder(A, B, Lmax, Hq, Hk, D, T, 3)
    ins = [torch.zeros(B, 1, h, D, dtype=T).cuda() for h in (Hq, Hk, Hk)]
    klen = torch.zeros(B, dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fast.step(*ins, klen)                             # (first calls allocate and set attributes outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fast.step(*ins, klen)
    for t in (fast.kc, fast.vc, fast.summary):
        t.zero_()
    for i in range(6):
        new = [randn(40 + 3 * i + s, *x.shape, dtype=T).cuda() for s, x in enumerate(ins)]
        at = torch.tensor([60 + i, 130 + i], dtype=torch.int32).cuda()
        for x, y in zip(ins, new):
            x.copy_(y)
        klen.copy_(at)
        graph.replay()
        noise = torch.randn(1 << 20, device='cuda').sum()              # eager work on the same stream in between
        want = slow.step(*new, at)
        torch.cuda.synchronize()
        assert torch.isfinite(noise)
        for x, y in zip(got, want):
            assert torch.equal(x, y), i
        assert torch.equal(fast.kc, slow.kc) and torch.equal(fast.summary, slow.summary)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_a_captured_training_step_replays(A, dt):
    B, L, Hq, Hk, D, T = 1, 260, 4, 1, 64, DT[dt]
    q, k, v, g = (torch.zeros(B, L, h, D, dtype=T).cuda() for h in (Hq, Hk, Hk, Hq))
    w, turns = torch.ones(D).cuda(), A.rotary_turns(D, device='cuda')
    bucket_of, bias = A.bucket_table(16, 64, device='cuda'), randn(1, 16, Hq).cuda()

    def step():
        qn, kn = A.head_norm_rotate(q, k, w, w, turns)
        sel = A.select_blocks(qn, A.block_summary(kn, 64), 3, 64, 32, keys=L)
        how = dict(block=64, query_block=32, bucket_of=bucket_of, bias=bias)
        out, saved = A.block_attention(qn, kn, v, sel, save=True, **how)
        dq, dk, dv, db = A.block_attention_backward(g, qn, kn, v, sel, saved, **how)
        return (out, dv, db) + A.head_norm_rotate_backward(dq, dk, q, k, w, w, turns)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for s, x in enumerate((q, k, v, g)):
            x.copy_(randn(10 * i + s, *x.shape, dtype=T).cuda())
        graph.replay()
        want = step()                                     # (eager, the same inputs, while the graph's results live)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


def test_streams_side_by_side(A):
    """two calls at once on two streams, each with its workspace: the same bits as one after the other"""
    T = torch.bfloat16
    q, k, v = randn(1, 2, 1, 8, 128, dtype=T).cuda(), randn(2, 2, 4000, 2, 128, dtype=T).cuda(), randn(3, 2, 4000, 2, 128, dtype=T).cuda()
    sel = torch.arange(0, 60, 2, dtype=torch.int32).cuda().expand(2, 2, 1, 30).contiguous()
    how = dict(block=64, query_block=1, causal=True)
    want = [A.block_attention(q * s, k, v, sel, **how) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(A.block_attention(q * (i + 1), k, v, sel, **how))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


# ------------------------------------------------------------------ views, long caches, odd lists and lengths
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_views(A, dt):
    """packed projections, (B, H, L, D) storage, a cache longer than the keys, a given strided output"""
    B, L, Hq, Hk, D, T = 2, 190, 4, 2, 40, DT[dt]
    packed = randn(1, B, L, Hq + 2 * Hk, D + 8, dtype=T).cuda()
    q, k, v = packed[:, :, :Hq, :D], packed[:, :, Hq:Hq + Hk, :D], packed[:, :, Hq + Hk:, 8:]
    hm = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    cache = torch.full((B, 2 * L, Hk, D), math.nan, dtype=T).cuda()
    cache[:, 5:5 + L] = k
    tight = [x.contiguous() for x in (q, k, v)]
    bucket_of, bias = A.bucket_table(8, 20, device='cuda'), randn(2, 8, Hq).cuda()
    sel = torch.tensor([0, 1, 2], dtype=torch.int32).cuda().expand(B, Hk, -(-L // 16), 3).contiguous()
    how = dict(block=64, query_block=16, causal=True, bucket_of=bucket_of, bias=bias)
    want, saved = A.block_attention(*tight, sel, save=True, **how)
    for x in ((q, k, v), tuple(hm), (tight[0], cache[:, 5:5 + L], v)):
        assert torch.equal(A.block_attention(*x, sel, **how, save=True)[0], want)
    wide = torch.full((B, L, Hq, 2 * D), 3.0, dtype=T).cuda()
    A.block_attention(q, k, v, sel, out=wide[..., :D], **how)
    if dt == 'f32':
        assert torch.equal(wide[..., :D], want)
    assert (wide[..., D:] == 3).all()
    g = randn(5, B, L, Hq, 2 * D, dtype=T).cuda()
    one = A.block_attention_backward(g[..., :D], q, k, v, sel, saved, **how)
    two = A.block_attention_backward(g[..., :D].contiguous(), *tight, sel, saved, **how)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    # a row broadcast over the batch (stride 0), keys and values one tensor
    shared = tight[1][:1].expand(B, L, Hk, D)
    assert torch.equal(A.block_attention(tight[0], shared, shared, sel, **how), A.block_attention(tight[0], shared.contiguous(), shared.contiguous(), sel, **how))
    assert torch.equal(A.block_summary(k, 64), A.block_summary(tight[1], 64))
    assert torch.equal(A.select_blocks(q, A.block_summary(k, 64), 2, 64, 16, keys=L, causal=True),
                       A.select_blocks(tight[0], A.block_summary(tight[1], 64), 2, 64, 16, keys=L, causal=True))


def test_offsets_past_32_bits(A):
    """a cache whose last token begins 3.3e9 elements behind its first; a norm over 2.2e9 elements"""
    L, D, T = 200000, 128, torch.bfloat16
    buf = torch.empty(L * 16384, dtype=T, device='cuda').view(1, L, 128, D)
    k, v = buf[:, :, 3:4], buf[:, :, 90:91]
    gen = torch.Generator(device='cuda').manual_seed(1)
    tight = [torch.randn(1, L, 1, D, generator=gen, device='cuda').to(T) for _ in range(2)]
    k.copy_(tight[0]), v.copy_(tight[1])
    nb = -(-L // 64)
    q = randn(2, 1, 3, 4, D, dtype=T).cuda()
    summary = A.block_summary(k, 64)
    assert torch.equal(summary, A.block_summary(tight[0], 64))
    sel = A.select_blocks(q, summary, 40, 64, 1, keys=L, causal=True)
    assert int(sel.max()) == nb - 1 and int((sel > nb // 2).sum()) > 20
    how = dict(block=64, query_block=1, causal=True)
    a, sa = A.block_attention(q, k, v, sel, save=True, **how)
    b, sb = A.block_attention(q, *tight, sel, save=True, **how)
    assert torch.equal(a, b)
    g = randn(4, 1, 3, 4, D, dtype=T).cuda()
    for x, y in zip(A.block_attention_backward(g, q, k, v, sel, sa, **how)[:3], A.block_attention_backward(g, q, *tight, sel, sb, **how)[:3]):
        assert torch.equal(x, y)
    new = randn(5, 1, 1, 1, D, dtype=T).cuda()
    w, slots = torch.ones(D).cuda(), torch.tensor([[L - 1]], dtype=torch.int32).cuda()
    _, kc = A.head_norm_rotate(new, new, w, w, out_k=k, slots=slots)
    assert torch.equal(kc[:, -1:], A.head_norm_rotate(new, None, w)[0]) and torch.equal(kc[:, -2], tight[0][:, -2])
    del k, v, kc
    x = buf[:, :135000]                                   # 2.2e9 elements
    x[:, -2:] = randn(6, 1, 2, 128, D, dtype=T).cuda()
    want = A.head_norm_rotate(x[:, -2:].contiguous(), None, w, turns=A.rotary_turns(D, device='cuda'), first=x.shape[1] - 2)[0]
    A.head_norm_rotate(x, None, w, turns=A.rotary_turns(D, device='cuda'), out_q=x)
    assert torch.equal(x[:, -2:], want)


@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_lists_with_odd_entries(A, dt):
    """out of range, negative in the middle, twice the same, descending: ignored as documented, forward and backward"""
    T = DT[dt]
    q, k, v, g = randn(1, 1, 96, 2, 64, dtype=T), randn(2, 1, 400, 1, 64, dtype=T), randn(3, 1, 400, 1, 64, dtype=T), randn(4, 1, 96, 2, 64, dtype=T)
    lists = [[0, 0, 3, 3, 5, 6], [5, 2, 1, 0, -1, -1], [-7, 2, -1, 4, 99, 3], [7, 8, 2 ** 31 - 1, -2 ** 31, 0, 1], [-1] * 6, [6, 6, 6, 6, 6, 6]]
    sel = torch.tensor(lists, dtype=torch.int32).view(1, 1, 6, 6)
    for causal in (False, True):
        want = O.attention(q, k, v, sel, 64, 16, 0.1, causal, None, None, dout=g)
        args = [t.cuda() for t in (q, k, v, sel)]
        how = dict(block=64, query_block=16, scale=0.1, causal=causal)
        out, saved = A.block_attention(*args, save=True, **how)
        within(out, *want['out'], 'out')
        for name, t in zip(('dq', 'dk', 'dv'), A.block_attention_backward(g.cuda(), *args, saved, **how)):
            within(t, *want[name], name)


@pytest.mark.parametrize('Lq,qb,n', [(3, 1, 40), (100, 16, 3)])          # keys split over workgroups and joined; one workgroup a group
@pytest.mark.parametrize('dt', ['f32', 'bf16'])
def test_lengths_of_zero_and_rows_left_as_they_were(A, Lq, qb, n, dt):
    """no queries, no keys, more queries than keys; rows behind qlen: zeros in a new output, untouched in a given one"""
    T, B, Lk = DT[dt], 5, 2600
    q, k, v, g = randn(1, B, Lq, 4, 64, dtype=T), randn(2, B, Lk, 2, 64, dtype=T), randn(3, B, Lk, 2, 64, dtype=T), randn(4, B, Lq, 4, 64, dtype=T)
    qlen = torch.tensor([0, Lq, Lq - 1, Lq, 1], dtype=torch.int32)
    klen = torch.tensor([Lk, 0, 1, Lk - 5, 64], dtype=torch.int32)
    sel = torch.arange(n, dtype=torch.int32).expand(B, 2, -(-Lq // qb), n).contiguous()
    args, kw = [t.cuda() for t in (q, k, v, sel)], dict(block=64, query_block=qb, scale=0.1, causal=True)
    want = O.attention(q, k, v, sel, 64, qb, 0.1, True, qlen, klen, dout=g)
    out, saved = A.block_attention(*args, qlen=qlen.cuda(), klen=klen.cuda(), save=True, **kw)
    within(out, *want['out'], 'out')
    given = torch.full_like(out, 7.0)
    assert A.block_attention(*args, qlen=qlen.cuda(), klen=klen.cuda(), out=given, **kw) is given
    behind = torch.arange(Lq)[None] >= qlen[:, None]
    assert (given.cpu()[behind] == 7).all() and not out.cpu()[behind].any()
    within(given.cpu()[~behind], want['out'][0][~behind], want['out'][1][~behind], 'given')
    for name, t in zip(('dq', 'dk', 'dv'), A.block_attention_backward(g.cuda(), *args, saved, qlen=qlen.cuda(), klen=klen.cuda(), **kw)):
        within(t, *want[name], name)
    got = A.select_blocks(q.cuda(), A.block_summary(k.cuda(), 64, klen.cuda()), n, 64, qb, keys=Lk, causal=True, qlen=qlen.cuda(), klen=klen.cuda())
    assert torch.equal(got.cpu(), O.select(q, A.block_summary(k.cuda(), 64, klen.cuda()).cpu(), n, 64, qb, Lk, True, qlen, klen))


@pytest.mark.parametrize('D,G,qb', [(64, 1, 2), (40, 3, 1)])
def test_gradients_against_differences(A, D, G, qb):
    """fp32: a step of the raw inputs along the gradient's direction, forward differences of the kernel's own fp32 result summed in
    fp64; the bound is the forward's error bound over the step, and the remainder seen between two steps"""
    B, L, Hk, n = 1, 70, 1, 2
    q, k, v, g = (randn(s, B, L, h, D).cuda() for s, h in ((1, Hk * G), (2, Hk), (3, Hk), (4, Hk * G)))
    bucket_of, bias = A.bucket_table(8, 20, device='cuda'), randn(5, 8, Hk * G).cuda()
    sel = torch.tensor([0, 1], dtype=torch.int32).cuda().expand(B, Hk, -(-L // qb), n).contiguous()
    base = dict(q=q, k=k, v=v, bias=bias)

    def run(x, save=False):
        return A.block_attention(x['q'], x['k'], x['v'], sel, block=64, query_block=qb, causal=True, bucket_of=bucket_of, bias=x['bias'], save=save)

    def loss(x):
        return float((run(x).double() * g.double()).sum())
    _, saved = run(base, True)
    grads = dict(zip(('q', 'k', 'v', 'bias'), A.block_attention_backward(g, q, k, v, sel, saved, block=64, query_block=qb, causal=True,
                                                                         bucket_of=bucket_of, bias=bias)))
    ref = O.attention(q.cpu(), k.cpu(), v.cpu(), sel.cpu(), 64, qb, 1 / math.sqrt(D), True, None, None, bucket_of.cpu(), bias.cpu())
    noise = float((ref['out'][1] * g.double().cpu().abs()).sum())
    for i, name in enumerate(base):
        way = randn(20 + i, *base[name].shape).cuda()
        way = way / way.norm()

        def central(h):
            hi, lo = dict(base), dict(base)
            hi[name], lo[name] = base[name] + h * way, base[name] - h * way
            real = float(((hi[name].double() - lo[name].double()) * way.double()).sum() / (way.double() ** 2).sum())       # the step that fp32 took
            return (loss(hi) - loss(lo)) / real, 2 * noise / real
        (fine, e1), (coarse, e2) = central(0.02), central(0.04)
        exact = float((grads[name].double() * way.double()).sum())
        # remainder of a central difference goes with h^2: a third of what two steps differ by; their noise with it
        assert abs(fine - exact) <= abs(coarse - fine) + e1 + e2 + 1e-5 * abs(exact), name
