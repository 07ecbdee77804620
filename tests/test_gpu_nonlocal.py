"""-m gpu: the non-local prior of the solver (adaptivepnp_sci_amd/nonlocal_prior.py): the attention operators one after the other, as a
pass of the prior uses them, its gradients, its online adaptation and its place in the solver.  Tolerances are the element-wise
bounds of the operators' roundings (oracle/attention.py), carried through the chain where one result feeds the next."""
import numpy as np
import pytest
import torch

from adaptivepnp_sci_amd import synth
from oracle import attention as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def N():
    from adaptivepnp_sci_amd import nonlocal_prior
    return nonlocal_prior


def clip(B, H, W, seed=0):
    """smooth moving frames with noise, in [0, 1]"""
    g = torch.Generator().manual_seed(seed)
    y, x = torch.meshgrid(torch.arange(H).float(), torch.arange(W).float(), indexing='ij')
    base = torch.stack([torch.stack([0.5 + 0.4 * torch.sin((x + 3 * t) / (7 + c)) * torch.cos(y / (9 - c)) for c in range(3)]) for t in range(B)])
    return (base + 0.05 * torch.randn(B, 3, H, W, generator=g)).clamp(0, 1)


def plain_tokens(frames, units, shifts, constant, scale, replicate):
    """indices written out: tokens (units * shifts, L, 1, 56)"""
    B, _, H, W = frames.shape
    T, more = B // units, 2 if shifts > 1 else 0
    ty, tx = -(-(H + more) // 32), -(-(W + more) // 32)
    out = torch.zeros(units * shifts, T, ty, tx, 8, 8, 56)
    for u in range(units):
        for s, (oy, ox) in enumerate([(0, 0), (2, 2), (0, 2), (2, 0)][:shifts]):
            rows, cols = torch.arange(ty * 32) - oy, torch.arange(tx * 32) - ox
            ry, rx = rows.clamp(0, H - 1), cols.clamp(0, W - 1)
            img = frames[u::units][:, :, ry][:, :, :, rx] * scale
            if not replicate:
                img = img * ((rows == ry)[:, None] & (cols == rx)[None])
            v = img.reshape(T, 3, ty, 8, 4, tx, 8, 4).permute(0, 2, 5, 3, 6, 1, 4, 7)
            out[u * shifts + s][..., :48] = v.reshape(T, ty, tx, 8, 8, 48)
            out[u * shifts + s][..., 48] = constant
    return out.reshape(units * shifts, -1, 1, 56)


@pytest.mark.parametrize('B,H,W,units,shifts', [(1, 1, 1, 1, 1), (2, 32, 32, 1, 1), (4, 31, 66, 2, 2), (3, 40, 36, 1, 4), (6, 64, 30, 3, 2)])
def test_patch_tokens_and_back(N, B, H, W, units, shifts):
    from adaptivepnp_sci_amd import ops
    x = clip(B, H, W)
    want = plain_tokens(x, units, shifts, 2.5, 0.25, True)
    tok = torch.full(want.shape, 9.0).cuda()
    ops.patch_tokens(x.cuda(), tok, units, shifts, 2.5, 0.25)
    assert torch.equal(tok.cpu(), want)
    # frames and back: the mean of equal values (a sum of up to four of them, divided: exact)
    ops.patch_tokens(x.cuda(), tok, units, shifts, 1.0)
    back = ops.patch_frames(tok, torch.empty(B, 3, H, W).cuda(), units, shifts)
    assert torch.equal(back.cpu(), x) if shifts != 4 else (back.cpu() - x).abs().max() <= 3 * 2.0 ** -24
    # adjoint: <A t, x> = <t, A' x>, in fp64 of fp32 results; (a sum of four terms and its quotient: 4 roundings of 2^-24 a term)
    g = torch.Generator().manual_seed(1)
    t = torch.randn(tok.shape, generator=g)
    fr = ops.patch_frames(t.cuda(), torch.empty(B, 3, H, W).cuda(), units, shifts).cpu().double()
    adj = torch.empty_like(tok)
    ops.patch_tokens(x.cuda(), adj, units, shifts, 0.0, 1.0 / shifts, replicate=False)
    assert torch.equal(adj.cpu(), plain_tokens(x, units, shifts, 0.0, 1.0 / shifts, False))
    a, b = (fr * x.double()).sum(), (adj.cpu().double() * t.double()).sum()
    assert (a - b).abs() <= 4 * 2.0 ** -24 * (adj.cpu().double().abs() * t.double().abs()).sum()


def within(got, val, err, what):
    d = (got.double().cpu() - val).abs()
    assert not (d > err + 1e-37).any(), f'{what}: worst {float((d / (err + 1e-37)).max()):.3g} x the bound'


def prior(N, **kw):
    m = N.NonLocalPrior(**kw)
    g = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for p, s in ((m.wq, 0.1), (m.wk, 0.1), (m.bias, 0.5)):
            p.add_(s * torch.randn(p.shape, generator=g))
    return m


@pytest.mark.parametrize('B,H,W,shifts,n_sel', [(2, 40, 36, 2, 3), (3, 32, 64, 1, 5), (1, 20, 20, 4, 2)])
@pytest.mark.parametrize('limit', [8192, 3])
def test_a_pass_operator_by_operator(N, B, H, W, shifts, n_sel, limit, monkeypatch):
    """every operator's result, given what the one before it left; limit: the blocks of a selection, past which they get larger"""
    monkeypatch.setattr(N, 'MAX_BLOCKS', limit)
    m = prior(N, n_sel=n_sel, shifts=shifts)
    eng = N.NonLocalEngine(m, B, H, W, torch.device('cuda'))
    x, sigma = clip(B, H, W), 0.2
    out, (tensors, how, saved) = eng.forward(x.cuda(), sigma, save=True)
    q, k, tok, sel = (t.cpu() for t in tensors)
    assert torch.equal(tok, plain_tokens(x, 1, shifts, N.LIFT, 1.0, True))
    for got, w in ((q, m.wq), (k, m.wk)):
        val = O.norm_rotate(tok, w.detach(), None, None)
        within(got, val, O.U32 * 1.01 * val.abs() + 2.0 ** -29 * val.abs().amax(-1, keepdim=True), 'norm')
    many = -(-tok.shape[1] // 64 // limit)
    block, n_sel = 64 * many, max(1, n_sel // many)
    assert how['block'] == block and sel.shape[-1] == n_sel
    want = O.summary(k, block, None)
    within(eng.summary, want, O.U32 * want.abs() + 1e-15, 'summary')
    L = tok.shape[1]
    assert torch.equal(sel, O.select(q, eng.summary.cpu(), n_sel, block, 64, L, False, None, None, 0, 1))
    h = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in how.items()}
    ref = O.attention(q, k, tok, sel, block, 64, h['scale'], False, None, None, h['bucket_of'], h['bias'], h['q_pos'], h['k_pos'])
    within(eng.o, *ref['out'], 'attention')
    # the mean over the grids of values with those errors, plus its own roundings
    val, err = (torch.zeros(B, 3, H, W, dtype=torch.float64) for _ in range(2))
    from adaptivepnp_sci_amd import ops
    for src, dst in ((ref['out'][0], val), (ref['out'][1], err)):
        for s in range(shifts):
            one = torch.zeros_like(eng.o)
            one[s] = src[s].cuda().float()
            dst += ops.patch_frames(one, torch.empty(B, 3, H, W).cuda(), 1, shifts).cpu().double()
    within(out, val, err * (1 + 2.0 ** -20) + 8 * O.U32 * (val.abs() + 1), 'frames')
    assert torch.equal(out, m(x.cuda(), sigma)), 'the module, without saving'


def test_a_flat_clip_stays_as_it_is(N):
    """every key is the query's own token: the weights sum to one whatever they are"""
    x = torch.full((2, 3, 32, 48), 0.625)
    got = N.NonLocalPrior(n_sel=4)(x.cuda(), 0.1).cpu()
    assert (got - x).abs().max() <= 0.625 * 2.0 ** -24 * (4 * 64 + 8)      # (256 products, their sum, the quotient)


def test_gradients_of_the_parameters(N):
    """against the formulas in 64 bits, and against differences of the 64-bit pass with the chosen blocks held"""
    B, H, W, shifts, n_sel, sigma = 2, 40, 36, 2, 3, 0.3
    m = prior(N, n_sel=n_sel, shifts=shifts)
    eng = N.NonLocalEngine(m, B, H, W, torch.device('cuda'))
    x = clip(B, H, W)
    _, kept = eng.forward(x.cuda(), sigma, save=True)
    g = torch.randn(B, 3, H, W, generator=torch.Generator().manual_seed(3))
    got = dict(zip(('wq', 'wk', 'bias'), (t.cpu() for t in eng.backward(g.cuda(), kept))))
    q, k, tok, sel = (t.cpu() for t in kept[0])
    h = {n: t.cpu() if isinstance(t, torch.Tensor) else t for n, t in kept[1].items()}
    do = plain_tokens(g, 1, shifts, 0.0, 1.0 / shifts, False)
    ref = O.attention(q, k, tok, sel, 64, 64, h['scale'], False, None, None, h['bucket_of'], h['bias'], h['q_pos'], h['k_pos'], dout=do)
    within(got['bias'], *ref['dbias'], 'dbias')
    n = tok.double() * torch.rsqrt(tok.double().square().mean(-1, keepdim=True) + 1e-6)
    for name, d in (('wq', 'dq'), ('wk', 'dk')):
        val, err = ref[d]
        want, slack = (val * n).sum((0, 1, 2)), (err * n.abs()).sum((0, 1, 2))
        within(got[name], want, slack + O.U32 * 1.01 * want.abs() + 2.0 ** -40 * (val.abs() * n.abs()).sum((0, 1, 2)), name)

    def loss(p):                                          # the pass in 64 bits, dense over the chosen keys
        nq, nk = n * p['wq'], n * p['wk']
        total = 0.0
        L = tok.shape[1]
        for b in range(tok.shape[0]):
            for gi in range(L // 64):
                rows = slice(gi * 64, gi * 64 + 64)
                keys = torch.cat([torch.arange(e * 64, e * 64 + 64) for e in sel[b, 0, gi].tolist() if e >= 0])
                dist = (h['k_pos'][b, keys][None] - h['q_pos'][b, rows][:, None]).clamp(-16, 16) + 16
                s = h['scale'] * nq[b, rows, 0] @ nk[b, keys, 0].T + p['bias'][h['bucket_of'][dist].long(), 0]
                total = total + (torch.softmax(s, -1) @ tok.double()[b, keys, 0] * do.double()[b, rows, 0]).sum()
        return total
    at = {k_: getattr(m, k_).detach().double() for k_ in ('wq', 'wk', 'bias')}
    gen = torch.Generator().manual_seed(11)
    for name in at:
        way = torch.randn(at[name].shape, generator=gen, dtype=torch.float64)

        def central(step):
            hi, lo = dict(at), dict(at)
            hi[name], lo[name] = at[name] + step * way, at[name] - step * way
            return (loss(hi) - loss(lo)) / (2 * step)
        fine, coarse = central(1e-5), central(2e-5)
        # the kernels' q, k are fp32: each off by half a step, which moves the 64-bit gradient by about 2^-23 of its terms' sizes
        err = (ref['dbias'][1].abs() * way.abs()).sum() if name == 'bias' else (ref['dq' if name == 'wq' else 'dk'][1] * (n * way).abs()).sum()
        size = (got[name].double().abs() * way.abs()).sum()
        logit = h['scale'] * q.double().abs().amax() * k.double().abs().amax() * 56
        assert (fine - (got[name].double() * way).sum()).abs() <= err + (coarse - fine).abs() + 2.0 ** -22 * (1 + logit) * size, name


def solve(N, model, U=1, update=False, two_stage=True, iters=3, seed=5, **kw):
    from adaptivepnp_sci_amd.solver import AdmmRun
    pr = [synth.make_problem(64, 96, 4, seed=seed + i) for i in range(U)]
    args = [[p[i] for p in pr] for i in range(3)] if U > 1 else list(pr[0])
    if U > 1:
        kw['units'] = U
    return AdmmRun(args[0], args[1], 'nonlocal_color', two_stage, X_orig=args[2], model=model, update_=update, inital_iter=0, interval_iter=2, lr_=1e-2,
                   update_per_iter=3, **kw), pr


@pytest.mark.parametrize('two_stage', [True, False])
def test_solver_iterations_and_adaptation(N, two_stage):
    from adaptivepnp_sci_amd import finetune as F
    m = N.NonLocalPrior(n_sel=6)
    run, _ = solve(N, m, update=True, two_stage=two_stage)
    seen = []
    F.GRAD_HOOK = lambda g: seen.append(g)
    try:
        for k in range(4):
            run.step(25 / 255, last=(k == 3))
    finally:
        F.GRAD_HOOK = None
    assert len(seen) == 1 and set(seen[0]) == {'wq', 'wk', 'bias'} and all(torch.isfinite(t).all() and t.abs().max() > 0 for t in seen[0].values())
    # three Adam steps: |m| / sqrt(v) of a step is at most sqrt(sum a_i^2 / b_i) for the weights a (0.9), b (0.999) of its gradients:
    # 1, 1.001, 1.004
    for p, start in ((m.wq, 1.0), (m.wk, 1.0)):
        d = (p.detach() - start).abs()
        assert d.max() > 0 and d.max() <= 3 * 1e-2 * 1.01
    assert torch.equal(run.eng.flat.cpu(), torch.cat([p.detach().reshape(-1) for p in (m.wq, m.wk, m.bias)]))
    assert torch.isfinite(run.out_rgb).all() and all(np.isfinite(run.psnr_all()))


@pytest.mark.parametrize('close_form', [False, True])
def test_unit_batch_equals_single_runs(N, close_form):
    m = prior(N, n_sel=5)
    batch, pr = solve(N, m, U=3, close_form_demosaic=close_form)
    from adaptivepnp_sci_amd.solver import AdmmRun
    single = [AdmmRun(y, Phi, 'nonlocal_color', True, X_orig=orig, model=m, close_form_demosaic=close_form) for y, Phi, orig in pr]
    for k in range(2):
        for r in single + [batch]:
            r.step(25 / 255)
        for u, t in enumerate(batch.result_mosaic()):
            assert torch.equal(t, single[u].result_mosaic()), (k, u)
    for u, r in enumerate(batch.split()):
        for x in (r, single[u]):
            x.step(25 / 255, last=True)
        assert torch.equal(r.result_mosaic(), single[u].result_mosaic()) and torch.equal(r.out_rgb, single[u].out_rgb)


def test_entry_points_and_plug_in(N):
    import adaptivepnp_sci_amd as P
    y, Phi, orig = synth.make_problem(64, 64, 4, seed=9)
    m = N.NonLocalPrior(n_sel=4)
    rgb, mosaic, psnr, ssim, allp, model, dm = P.twoStageAdmm_denoise_bayer(y, Phi, denoiser='nonlocal_color', iter_max=[2], noise_estimate=False,
                                                                             sigma=[25 / 255], X_orig=orig, model_denoise=m)
    assert model is m and rgb.shape == (64, 64, 3, 4) and mosaic.shape == y.shape + (4,) and len(allp) == 2 and np.isfinite(allp).all()
    res = P.admm_denoise_bayer_demosaic_pre(y, Phi, denoiser='nonlocal_color', iter_max=[2], noise_estimate=False, sigma=[25 / 255], X_orig=orig, model=m)
    assert np.isfinite(res[4]).all()
    x = clip(2, 40, 36).cuda()
    cube = P.nonlocal_denoiser_full_tensor(x.permute(2, 3, 1, 0).contiguous(), 0.1, model=m)
    assert torch.equal(cube.permute(3, 2, 0, 1), m(x, 0.1))
    with pytest.raises(ValueError, match='NonLocalPrior'):
        P.twoStageAdmm_denoise_bayer(y, Phi, denoiser='nonlocal_color', iter_max=[1], sigma=[0.1], model_denoise=torch.nn.Linear(2, 2))


def test_a_large_cube(N):
    """1024 x 1024 x 16: more tiles than a selection takes; a constant clip with one odd tile stays a constant clip elsewhere"""
    x = torch.full((16, 3, 1024, 1024), 0.25, device='cuda')
    x[3, :, 256:288, 320:352] = 0.75
    m = N.NonLocalPrior(n_sel=6)
    got = m(x, 0.02)
    assert torch.isfinite(got).all()
    # a weight across the two kinds is below exp(-|x - x'|^2 / (48 s^2) (about)): their cosine is 0.96, the scale 2500, nothing is left of it;
    # the rest is the sum over 384 equal values and its quotient
    far = torch.ones(1024, 1024, dtype=torch.bool, device='cuda')
    far[224:320, 288:384] = False
    assert (got[:, :, far] - 0.25).abs().max() <= 0.25 * 2.0 ** -24 * (4 * 64 * 6 + 8)
