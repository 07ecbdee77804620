"""Non-local attention over selected key blocks: thin wrappers over the C ABI (include/scipnp.h), like ops.py.

A query group picks the key blocks that resemble it by a cheap score and attends to those blocks only: the block matching of
non-local video restoration in the form of attention, for tokens of any kind.  Four operators, used together:

    head_norm_rotate   norm of every query and key head with its learned weight, and the rotation by the token's position, in one
                       pass; writes into a cache when given slots                          (+ head_norm_rotate_backward)
    block_summary      mean key of every block (or of the blocks that the newest tokens touched)
    select_blocks      each query group's n blocks with the largest score (group's summed queries) . (mean key)
    block_attention    softmax attention over the selected blocks with a learned relative position bias by buckets
                                                                                           (+ block_attention_backward)

Tensors are (B, L, H, D), float32 or bfloat16, last dimension contiguous, the other strides free (views of a packed projection or of a
cache); q has Hq heads, k and v Hk, Hq a multiple of Hk.  float32 inputs are multiplied in exact fp32 products; sums, norms and
softmax statistics are fp32 or fp64 in either type.  Sequence b has qlen[b] queries and klen[b] keys (int32, None: all); query i
stands at key position klen - qlen + i, so a cache with one new token needs klen only.  Every call is asynchronous on the current
stream of the tensors' device, allocates its workspace from torch, gives the same bits for the same inputs, and can be captured.
"""
import ctypes as C
import math

import torch

from . import _lib
from ._lib import BlockAttnArgs, HeadNormArgs, SelectArgs, ScipnpError

_DT = {torch.float32: 0, torch.bfloat16: 1}
_st3 = C.c_int64 * 3


def rotary_turns(dims, base=10000.0, device=None):
    """turns of the circle per position of each rotated pair, base^(-2i/dims) / (2 pi), in fp64: (dims / 2,)"""
    if dims <= 0 or dims % 8:
        raise ValueError(f'{dims} rotated dimensions: a positive multiple of 8')
    return torch.tensor([base ** (-2.0 * i / dims) / (2.0 * math.pi) for i in range(dims // 2)], dtype=torch.float64, device=device)


def bucket_table(num_buckets, max_distance, bidirectional=True, device=None):
    """bucket of every relative position key - query from -max_distance to max_distance (further ones belong to the ends), int32.

    Distances up to half the buckets of a side have one of their own, the others share buckets that widen by equal factors up to
    max_distance: the last step reached is the largest s with (dist / e)^m >= (max_distance / e)^s, decided in whole numbers.
    bidirectional: the upper half of the buckets for keys behind the query; otherwise such keys share the query's own bucket."""
    per_side = num_buckets // 2 if bidirectional else num_buckets
    if num_buckets < 2 or num_buckets > 64 or per_side < 2 or (bidirectional and num_buckets % 2):
        raise ValueError(f'{num_buckets} buckets: 2 to 64, and an even number from 4 on for both directions')
    e = per_side // 2
    if max_distance <= e or max_distance > 4096:
        raise ValueError(f'max_distance {max_distance}: above {e} (distances with a bucket of their own), at most 4096')
    m, side, step = per_side - e, [], 0
    for dist in range(max_distance + 1):
        while dist >= e and step + 1 < m and dist ** m * e ** (step + 1) >= e ** m * max_distance ** (step + 1):
            step += 1
        side.append(dist if dist < e else e + step)
    behind = [(num_buckets // 2 if bidirectional else 0) + (side[d] if bidirectional else 0) for d in range(1, max_distance + 1)]
    return torch.tensor(side[::-1] + behind, dtype=torch.int32, device=device)


# ------------------------------------------------------------------ argument checks
def _tokens(t, name, shape=None, dtype=None):
    """a (B, L, H, D) tensor: its pointer and element strides"""
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f'{name} must be a (B, L, H, D) tensor')
    if t.dtype not in _DT or (dtype is not None and t.dtype != dtype):
        raise ValueError(f'{name} is {t.dtype}: expected {dtype or "float32 or bfloat16"}')
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f'{name} has shape {tuple(t.shape)}, expected {shape}')
    n, s = t.shape, t.stride()
    if s[3] != 1 and n[3] != 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')
    _on_device(t, name)
    return t.data_ptr(), _st3(s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _array(t, name, shape, dtype):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        got = (t.dtype, tuple(t.shape)) if isinstance(t, torch.Tensor) else type(t)
        raise ValueError(f'{name} must be a contiguous {dtype} tensor of shape {shape}, got {got}')
    _on_device(t, name)
    return t.data_ptr()


def _on_device(t, name):
    if not t.is_cuda:
        raise ScipnpError(f'{name} must be a CUDA/ROCm tensor (the hot path has no CPU fallback)')
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f'{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}')


def _call(name, *args):
    lib = _lib.load()
    _lib.require_gpu()
    _lib.check(getattr(lib, name)(*args, _lib.stream_ptr()), name)


def _shape4(t, name):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f'{name} must be a (B, L, H, D) tensor')
    if 0 in t.shape:
        raise ValueError(f'{name} has an empty dimension: {tuple(t.shape)}')
    return tuple(t.shape)


def _heads(q, k):
    B, Lq, Hq, D = _shape4(q, 'q')
    Bk, Lk, Hk, Dk = _shape4(k, 'k')
    if Bk != B or Dk != D or Hq % Hk:
        raise ValueError(f'q {tuple(q.shape)} and k {tuple(k.shape)}: same batch and head size, query heads a multiple of key heads')
    return B, Lq, Lk, Hq, Hk, D


# ------------------------------------------------------------------ norm and rotation
def _norm_args(q, k, wq, wk, turns, positions, first, eps):
    B, L, Hq, D = _shape4(q, 'q')
    a = HeadNormArgs(dtype=_DT.get(q.dtype, -1), B=B, L=L, Hq=Hq, D=D, first=int(first), eps=float(eps))
    a.q, a.q_stride = _tokens(q, 'q')
    if k is not None:
        a.Hk = _shape4(k, 'k')[2]
        a.k, a.k_stride = _tokens(k, 'k', (B, L, a.Hk, D), q.dtype)
        a.wk = _array(wk, 'wk', (D,), torch.float32)
    a.wq = _array(wq, 'wq', (D,), torch.float32)
    if turns is not None:
        a.rot = 2 * turns.numel()
        a.turns = _array(turns, 'turns', (turns.numel(),), torch.float64)
    a.positions = _array(positions, 'positions', (B, L), torch.int32)
    return a


def head_norm_rotate(q, k=None, wq=None, wk=None, turns=None, positions=None, first=0, eps=1e-6, out_q=None, out_k=None, v=None,
                     out_v=None, slots=None):
    """(q', k'): every head normalised by its root mean square, times the weight wq / wk (D,), its first 2 * turns.numel() dimensions
    turned by the token's position (positions (B, L) int32, None: first + index); pair i is dimensions i and i + turns.numel().
    Computed in fp64 and rounded once.  With out_k (and v, out_v) the keys (and values, unchanged) go there; with slots (B, L) int32
    to row slots[b, l] of it -- a cache (B, Lmax, Hk, D).  A slot outside the cache drops the row; two tokens of a sequence with the
    same slot leave either.  out_q / out_k may be q / k themselves."""
    a = _norm_args(q, k, wq, wk, turns, positions, first, eps)
    B, L, _, D = q.shape
    out_q = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out_q is None else out_q
    a.out_q, a.out_q_stride = _tokens(out_q, 'out_q', tuple(q.shape), q.dtype)
    if k is not None:
        if slots is not None:
            if out_k is None:
                raise ValueError('slots need out_k (a cache)')
            a.slots = _array(slots, 'slots', (B, L), torch.int32)
            a.Lout = _shape4(out_k, 'out_k')[1]
        out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device) if out_k is None else out_k
        rows = a.Lout if slots is not None else L
        a.out_k, a.out_k_stride = _tokens(out_k, 'out_k', (B, rows, a.Hk, D), q.dtype)
        if v is not None:
            if out_v is None:
                raise ValueError('v needs out_v')
            a.v, a.v_stride = _tokens(v, 'v', tuple(k.shape), q.dtype)
            a.out_v, a.out_v_stride = _tokens(out_v, 'out_v', (B, rows, a.Hk, D), q.dtype)
    elif out_k is not None or v is not None or slots is not None:
        raise ValueError('out_k, v and slots need k')
    _call('scipnp_head_norm_rotate', C.byref(a))
    return out_q, out_k


def head_norm_rotate_backward(g_q, g_k, q, k, wq, wk, turns=None, positions=None, first=0, eps=1e-6):
    """(dq, dk, dwq, dwk) of head_norm_rotate from the gradients of its two results (k None: dk, dwk None)"""
    a = _norm_args(q, k, wq, wk, turns, positions, first, eps)
    a.g_q, a.g_q_stride = _tokens(g_q, 'g_q', tuple(q.shape), q.dtype)
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    a.out_q, a.out_q_stride = _tokens(dq, 'dq')
    dwq = torch.empty_like(wq)
    a.dwq = dwq.data_ptr()
    dk = dwk = None
    if k is not None:
        a.g_k, a.g_k_stride = _tokens(g_k, 'g_k', tuple(k.shape), q.dtype)
        dk, dwk = torch.empty(k.shape, dtype=k.dtype, device=k.device), torch.empty_like(wk)
        a.out_k, a.out_k_stride = _tokens(dk, 'dk')
        a.dwk = dwk.data_ptr()
    ws = torch.empty(_lib.load().scipnp_head_norm_rotate_backward_workspace_bytes(C.byref(a)), dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _call('scipnp_head_norm_rotate_backward', C.byref(a))
    return dq, dk, dwq, dwk


# ------------------------------------------------------------------ summary and selection
def block_summary(k, block=64, klen=None, newest=0, out=None):
    """mean key of every block of `block` keys over its live ones: (B, ceil(Lk / block), Hk, D) float32, zeros behind klen.  newest=n
    writes only the blocks that the last n live keys touch (out: the summary of the cache before them)."""
    B, Lk, Hk, D = _shape4(k, 'k')
    if block < 1 or newest < 0:
        raise ValueError(f'block {block} must be positive, newest {newest} not negative')
    if newest and out is None:
        raise ValueError('newest needs out')
    p, st = _tokens(k, 'k')
    shape = (B, -(-Lk // block), Hk, D)
    out = torch.empty(shape, dtype=torch.float32, device=k.device) if out is None else out
    _call('scipnp_block_summary', p, st, _DT[k.dtype], _array(klen, 'klen', (B,), torch.int32), _array(out, 'out', shape, torch.float32),
          B, Lk, Hk, D, int(block), int(newest))
    return out


def select_blocks(q, summary, n_sel, block=64, query_block=64, keys=None, causal=False, qlen=None, klen=None, sink=1, local=1):
    """the n_sel key blocks of every group of query_block queries (and the query heads of a key head): (B, Hk, groups, n_sel) int32,
    ascending, -1 behind the last.  Score: (sum of the group's queries) . (mean key), in fp64; ties to the lower block.  The `sink`
    first blocks and the blocks within local - 1 of the group's last query come before every score.  keys: length of the key
    sequence (None: the summary's blocks are full); causal: only blocks that begin at or before the group's last query."""
    B, Lq, Hq, D = _shape4(q, 'q')
    if not isinstance(summary, torch.Tensor) or summary.dim() != 4 or summary.shape[0] != B or summary.shape[3] != D or Hq % max(1, summary.shape[2]):
        raise ValueError(f'summary must be (B, blocks, Hk, D) of q {tuple(q.shape)}')
    nb, Hk = summary.shape[1:3]
    Lk = nb * block if keys is None else int(keys)
    if block < 1 or query_block < 1 or n_sel < 1 or -(-Lk // block) != nb:
        raise ValueError(f'{Lk} keys in blocks of {block} are not the {nb} blocks of the summary (n_sel {n_sel}, query_block {query_block})')
    a = SelectArgs(dtype=_DT.get(q.dtype, -1), B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=D, block=int(block), query_block=int(query_block),
                   n_sel=int(n_sel), sink=int(sink), local=int(local), causal=int(bool(causal)))
    a.q, a.q_stride = _tokens(q, 'q')
    a.summary = _array(summary, 'summary', (B, nb, Hk, D), torch.float32)
    a.qlen, a.klen = _array(qlen, 'qlen', (B,), torch.int32), _array(klen, 'klen', (B,), torch.int32)
    sel = torch.empty(B, Hk, -(-Lq // query_block), n_sel, dtype=torch.int32, device=q.device)
    a.sel = sel.data_ptr()
    _call('scipnp_select_blocks', C.byref(a))
    return sel


# ------------------------------------------------------------------ attention
def _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos):
    B, Lq, Lk, Hq, Hk, D = _heads(q, k)
    if block < 1 or query_block < 1:
        raise ValueError(f'block {block} and query_block {query_block} must be positive')
    groups = -(-Lq // query_block)
    if not isinstance(sel, torch.Tensor) or sel.dim() != 4:
        raise ValueError(f'sel must be (B, Hk, groups, n) = ({B}, {Hk}, {groups}, n)')
    a = BlockAttnArgs(dtype=_DT.get(q.dtype, -1), B=B, Lq=Lq, Lk=Lk, Hq=Hq, Hk=Hk, D=D, block=int(block), query_block=int(query_block),
                      n_sel=sel.shape[3], causal=int(bool(causal)), scale=1.0 / math.sqrt(D) if scale is None else float(scale))
    a.q, a.q_stride = _tokens(q, 'q')
    a.k, a.k_stride = _tokens(k, 'k', dtype=q.dtype)
    a.v, a.v_stride = _tokens(v, 'v', tuple(k.shape), q.dtype)
    a.sel = _array(sel, 'sel', (B, Hk, groups, sel.shape[3]), torch.int32)
    a.qlen, a.klen = _array(qlen, 'qlen', (B,), torch.int32), _array(klen, 'klen', (B,), torch.int32)
    if (bias is None) != (bucket_of is None):
        raise ValueError('bias and bucket_of belong together')
    if bias is not None:
        if bias.dim() != 2 or bucket_of.dim() != 1 or bucket_of.numel() % 2 == 0:
            raise ValueError('bias must be (buckets, Hq), bucket_of (2 * max_distance + 1,)')
        a.num_buckets, a.max_distance = bias.shape[0], bucket_of.numel() // 2
        a.bias = _array(bias, 'bias', (bias.shape[0], Hq), torch.float32)
        a.bucket_of = _array(bucket_of, 'bucket_of', (bucket_of.numel(),), torch.int32)
        a.q_pos, a.k_pos = _array(q_pos, 'q_pos', (B, Lq), torch.int32), _array(k_pos, 'k_pos', (B, Lk), torch.int32)
    elif q_pos is not None or k_pos is not None:
        raise ValueError('q_pos and k_pos are positions for the bias')
    return a


def _workspace(a, backward, device):
    n = _lib.load().scipnp_block_attn_workspace_bytes(C.byref(a), backward)
    if not n:
        return None
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    return ws


def block_attention(q, k, v, sel, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None, bucket_of=None, bias=None,
                    q_pos=None, k_pos=None, out=None, save=False):
    """softmax(scale * q k^T + bias) v over the keys of each group's selected blocks (select_blocks; an entry outside the blocks, or
    not greater than those before it, is ignored).  scale None: 1 / sqrt(D).  causal: keys behind the query are masked.  bias
    (buckets, Hq) float32 by the relative position of key and query, bucket_of from bucket_table; q_pos (B, Lq), k_pos (B, Lk) int32
    name the positions (None: the key positions), e.g. the frame of each token of a video; differences must fit 32 bits.  A query
    without a visible key gives zeros.  Rows behind qlen are zeros, or left as they were in a given `out`.
    save=True returns (out, saved) for block_attention_backward; bfloat16 probabilities are then multiplied whole, not rounded, so that
    the saved fp32 result carries the gradient (out is the same up to its rounding)."""
    a = _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos)
    if out is None:
        out = (torch.empty if qlen is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    a.out, a.out_stride = _tokens(out, 'out', tuple(q.shape), q.dtype)
    saved = None
    if save:
        saved = (torch.empty(a.B, a.Hq, a.Lq, dtype=torch.float32, device=q.device), torch.empty(q.shape, dtype=torch.float32, device=q.device))
        a.lse, a.out32 = saved[0].data_ptr(), saved[1].data_ptr()
    ws = _workspace(a, 0, q.device)                                     # noqa: F841 (alive until the call is enqueued)
    _call('scipnp_block_attn', C.byref(a))
    return (out, saved) if save else out


def block_attention_backward(dout, q, k, v, sel, saved, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None,
                             bucket_of=None, bias=None, q_pos=None, k_pos=None):
    """(dq, dk, dv, dbias) of block_attention called with the same arguments and save=True; rows behind qlen / klen are zeros, dbias
    (buckets, Hq) float32 is None without a bias.  The selection is not differentiated."""
    a = _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos)
    a.dout, a.dout_stride = _tokens(dout, 'dout', tuple(q.shape), q.dtype)
    lse, out32 = saved
    a.lse = _array(lse, 'saved[0]', (a.B, a.Hq, a.Lq), torch.float32)
    a.out32 = _array(out32, 'saved[1]', tuple(q.shape), torch.float32)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    dbias = None
    if bias is not None:
        dbias = torch.empty_like(bias)
        a.dbias = dbias.data_ptr()
    ws = _workspace(a, 1, q.device)                                     # noqa: F841
    _call('scipnp_block_attn_backward', C.byref(a))
    return dq, dk, dv, dbias
