"""Non-local colour prior of the PnP solver ('nonlocal_color'): every patch of a clip becomes a mean of the patches that resemble it,
anywhere in the clip, by attention over selected blocks (attention.py).

A frame is cut into 4 x 4 x 3 patches, 8 x 8 of them are one block of 64 tokens; a constant entry is put behind a token's 48 values,
so that the norm keeps its brightness.  Per pass, for each clip and each of `shifts` patch grids (moved by half a patch and averaged):

    q, k = norm(token) * wq, norm(token) * wk                                     head_norm_rotate
    blocks of the most similar mean key, the block itself always among them       block_summary, select_blocks
    softmax(q k / (D sigma^2) + bias[frame distance]) token                       block_attention

With wq = wk = 1 and no bias the weight of a patch pair is exp(-|x - x'|^2 / (48 sigma^2)) for patches of middle brightness: non-local
means.  wq, wk and the bias adapt online to the measurement, like the weights of the network denoisers: nonlocal_online_finetune.
Not part of the solvers' reference (parity unpinned).
"""
import ctypes as C

import torch
from torch import nn

from . import _lib, attention as A, ops

F32 = torch.float32
VALUES, DIMS, BLOCK, TILE = 48, 56, 64, 32
LIFT = 0.5 * VALUES ** 0.5               # the constant entry: as long as a patch of middle brightness
MIN_SIGMA = 1e-3
MAX_BLOCKS = 8192                        # of a selection
_EPS = 1e-6


class NonLocalPrior(nn.Module):
    """parameters (wq, wk: weight of each token entry; bias: by bucketed frame distance) and the sizes of the prior"""

    def __init__(self, n_sel=16, shifts=2, num_buckets=16, max_distance=16):
        super().__init__()
        if n_sel < 1 or n_sel > 1024 or shifts not in (1, 2, 4):
            raise ValueError(f'n_sel {n_sel}: 1 to 1024; shifts {shifts}: 1, 2 or 4')
        self.n_sel, self.shifts, self.num_buckets, self.max_distance = n_sel, shifts, num_buckets, max_distance
        A.bucket_table(num_buckets, max_distance)             # (refuses what it cannot be)
        self.wq, self.wk = nn.Parameter(torch.ones(DIMS)), nn.Parameter(torch.ones(DIMS))
        self.bias = nn.Parameter(torch.zeros(num_buckets, 1))

    def forward(self, frames, sigma):
        """frames (B,3,H,W) CUDA tensor of one clip -> denoised (B,3,H,W); HIP kernels only"""
        B, _, H, W = frames.shape
        return NonLocalEngine(self, B, H, W, frames.device).forward(frames.float().contiguous(), float(sigma))


class NonLocalEngine:
    """the prior on B frames of H x W in `units` clips, frame t of clip u at t * units + u (like FastDVDEngine)"""
    precision = 'f32'

    def __init__(self, model, B, H, W, device, units=1):
        if not isinstance(model, NonLocalPrior):
            raise ValueError(f'nonlocal_color needs a NonLocalPrior as its model, got {type(model).__name__}')
        if B % units:
            raise ValueError(f'{B} frames do not split into {units} units')
        self.B, self.H, self.W, self.units, self.device = B, H, W, units, device
        self.shifts = model.shifts
        more = 2 if self.shifts > 1 else 0
        tiles = -(-(H + more) // TILE) * -(-(W + more) // TILE)
        T, self.L = B // units, B // units * tiles * BLOCK
        many = -(-T * tiles // MAX_BLOCKS)      # (a clip of more tiles, e.g. 1024 x 1024 x 16: blocks of several tiles, fewer of them)
        self.block, self.n_sel = BLOCK * many, max(1, model.n_sel // many)
        seqs = units * self.shifts
        self.tokens = torch.empty(seqs, self.L, 1, DIMS, dtype=F32, device=device)
        self.q, self.k, self.o = (torch.empty_like(self.tokens) for _ in range(3))
        self.summary = torch.empty(seqs, -(-self.L // self.block), 1, DIMS, dtype=F32, device=device)
        self.frame = torch.arange(T, dtype=torch.int32, device=device).repeat_interleave(tiles * BLOCK).expand(seqs, -1).contiguous()
        self.bucket_of = A.bucket_table(model.num_buckets, model.max_distance, device=device)
        self.flat = torch.empty(2 * DIMS + model.num_buckets, dtype=F32, device=device)
        self.wq, self.wk, self.bias = self.flat[:DIMS], self.flat[DIMS:2 * DIMS], self.flat[2 * DIMS:].view(-1, 1)
        self.out = torch.empty(B, 3, H, W, dtype=F32, device=device)
        self.refresh(model)

    def refresh(self, model):
        from .finetune import _upload_flat
        _upload_flat(self.flat, [p.detach() for p in (model.wq, model.wk, model.bias)])

    def _clip(self, u, sigma, sel):
        s = slice(u * self.shifts, (u + 1) * self.shifts)
        return ((self.q[s], self.k[s], self.tokens[s], sel[s]),
                dict(block=self.block, query_block=BLOCK, scale=1.0 / (DIMS * max(float(sigma), MIN_SIGMA) ** 2), bucket_of=self.bucket_of, bias=self.bias,
                     q_pos=self.frame[s], k_pos=self.frame[s]), self.o[s])

    def forward(self, frames, sigma, save=False):
        """frames planar (B,3,H,W) -> denoised planar (B,3,H,W), owned by the engine and overwritten by the next call.  save: also what
        the backward pass needs (a single clip)"""
        if tuple(frames.shape) != tuple(self.out.shape):
            raise ValueError(f'frames must be {tuple(self.out.shape)}, got {tuple(frames.shape)}')
        ops.patch_tokens(frames, self.tokens, self.units, self.shifts, LIFT)
        A.head_norm_rotate(self.tokens, self.tokens, self.wq, self.wk, eps=_EPS, out_q=self.q, out_k=self.k)
        A.block_summary(self.k, self.block, out=self.summary)
        sel = A.select_blocks(self.q, self.summary, self.n_sel, self.block, BLOCK, keys=self.L, sink=0, local=1)
        kept = None
        for u in range(self.units):      # (a clip a call: how its work is split, and so its bits, does not depend on the other clips)
            tensors, how, o = self._clip(u, sigma, sel)
            res = A.block_attention(*tensors, out=o, save=save, **how)
            kept = (tensors, how, res[1]) if save else None
        ops.patch_frames(self.o, self.out, self.units, self.shifts)
        return (self.out, kept) if save else self.out

    def backward(self, dout, kept):
        """(dwq, dwk, dbias) for the gradient of the output frames, behind forward(save=True)"""
        tensors, how, saved = kept
        do = torch.empty_like(self.tokens)
        ops.patch_tokens(dout, do, self.units, self.shifts, 0.0, scale=1.0 / self.shifts, replicate=False)      # adjoint of patch_frames
        dq, dk, _, dbias = A.block_attention_backward(do, *tensors, saved, **how)
        _, _, dwq, dwk = A.head_norm_rotate_backward(dq, dk, self.tokens, self.tokens, self.wq, self.wk, eps=_EPS)
        return dwq, dwk, dbias


def nonlocal_online_finetune(model, eng, frames, y_pm, Phi_pm, sigma, lr_, update_per_iter, logf=None, trace=None):
    """`update_per_iter` Adam steps of wq, wk and the bias on the measurement loss MSE(y, sum_t Phi_t out_t at the CFA sites) for the
    input `frames` (B,3,H,W), the loss of the network denoisers' online finetunes; y_pm [4][M][N], Phi_pm [B][4][M][N] plane-major.
    The module's parameters and the engine's are the updated ones afterwards; a new Adam each event."""
    from . import finetune as F
    if eng.units != 1:
        raise ValueError('the finetune needs weights of its own for every clip: one unit')
    M, N = eng.H // 2, eng.W // 2
    if eng.H % 2 or eng.W % 2:
        raise ValueError(f'{eng.H}x{eng.W} frames have no whole Bayer cells: the finetune needs even sizes')
    for name, t, shape in (('frames', frames, (eng.B, 3, eng.H, eng.W)), ('y_pm', y_pm, (4, M, N)), ('Phi_pm', Phi_pm, (eng.B, 4, M, N))):
        if tuple(t.shape) != shape or t.dtype != F32 or not t.is_contiguous():
            raise ValueError(f'{name} must be contiguous float32 {shape}, got {t.dtype} {tuple(t.shape)} contiguous={t.is_contiguous()}')
        if t.device != eng.out.device:
            raise ValueError(f'{name} is on {t.device}, the engine on {eng.out.device}')
    _lib.require_gpu()
    if update_per_iter <= 0:
        return model
    lib = _lib.load()
    nblocks = C.c_int(0)
    size = (M, N, eng.B, C.byref(nblocks))
    _lib.check(lib.scipnp_fastdvd_loss_grad(None, None, None, None, None, *size, None), 'size')
    part = torch.empty(nblocks.value, dtype=torch.float64, device=eng.device)
    dout, (m, v) = torch.empty_like(eng.out), (torch.zeros_like(eng.flat) for _ in range(2))
    params = [model.wq, model.wk, model.bias]
    eng.refresh(model)
    losses = []
    for step in range(1, update_per_iter + 1):
        out, kept = eng.forward(frames, sigma, save=True)
        _lib.check(lib.scipnp_fastdvd_loss_grad(F._ptr(out), F._ptr(Phi_pm), F._ptr(y_pm), F._ptr(dout), F._ptr(part), *size, F._s()),
                   'scipnp_fastdvd_loss_grad')
        losses.append(F._DeviceMean(ops.sum_rows_f64(part), float(eng.H * eng.W)))
        grads = eng.backward(dout, kept)
        if step == 1 and F.GRAD_HOOK is not None:
            F.GRAD_HOOK(dict(zip(('wq', 'wk', 'bias'), (g.clone() for g in grads))))
        grad = torch.cat([g.reshape(-1) for g in grads])
        _lib.check(lib.scipnp_adam_step(F._ptr(eng.flat), F._ptr(grad), F._ptr(m), F._ptr(v), eng.flat.numel(), float(lr_), 0.9, 0.999, 1e-8, step, F._s()),
                   'scipnp_adam_step')
    F._download_flat(eng.flat, params)
    for loss in losses:
        val = float(loss.item())
        print('loss:', val)
        if trace is not None:
            trace.append(val)
    return model
