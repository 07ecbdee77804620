"""Non-local attention over selected key blocks: thin wrappers over the C ABI (include/scipnp.h), like ops.py.

A query group picks the key blocks that resemble it by a cheap score and attends to those blocks only: the block matching of
non-local video restoration in the form of attention, for tokens of any kind (the solver's 'nonlocal_color' prior is built of them,
nonlocal_prior.py).  Four operators, used together:

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
import struct

import torch

from . import _lib
from ._lib import ScipnpError

_DT = {torch.float32: 0, torch.bfloat16: 1}
_F32, _F64, _I32 = torch.float32, torch.float64, torch.int32

# The argument blocks of include/scipnp.h as one struct.pack each: a call of a few microseconds on the GPU should not wait for
# forty ctypes assignments (a decoding step is five such calls).
_NORM = struct.Struct('@N9if10P24q6PN')
_SELECT = struct.Struct('@N13iP3q4P')
_ATTN = struct.Struct('@N14if4P12q10P3q5PN')
assert (_NORM.size, _SELECT.size, _ATTN.size) == tuple(C.sizeof(s) for s in (_lib.HeadNormArgs, _lib.SelectArgs, _lib.BlockAttnArgs))
_NONE4 = (0, 0, 0, 0)


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
    """pointer and element strides (batch, token, head) of a (B, L, H, D) tensor"""
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f'{name} must be a (B, L, H, D) tensor')
    n, s = t.shape, t.stride()
    if (t.dtype is not dtype) if dtype is not None else (t.dtype not in _DT):
        raise ValueError(f'{name} is {t.dtype}: expected {dtype or "float32 or bfloat16"}')
    if shape is not None and n != shape:
        raise ValueError(f'{name} has shape {tuple(n)}, expected {tuple(shape)}')
    if s[3] != 1 and n[3] != 1:
        raise ValueError(f'{name}: the last dimension must be contiguous')
    return t.data_ptr(), s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0


def _array(t, name, shape, dtype):
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        got = (t.dtype, tuple(t.shape)) if isinstance(t, torch.Tensor) else type(t)
        raise ValueError(f'{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}, got {got}')
    return t.data_ptr()


def _on_device(*named):
    """every tensor is on the current device: its stream is the one the call goes to"""
    dev = -1
    for name, t in named:
        if t is None:
            continue
        d = t.get_device()
        if d < 0:
            raise ScipnpError(f'{name} must be a CUDA/ROCm tensor (the hot path has no CPU fallback)')
        if dev < 0:
            dev = torch.cuda.current_device()
        if d != dev:
            raise ValueError(f'{name} is on cuda:{d}, the current device is cuda:{dev}')


_FN = {}


def _call(name, *args):
    fn = _FN.get(name)
    if fn is None:
        lib = _lib.load()
        _lib.require_gpu()
        fn = _FN[name] = getattr(lib, name)
    rc = fn(*args, _lib.stream_ptr())
    if rc:
        _lib.check(rc, name)


def _shape4(t, name):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f'{name} must be a (B, L, H, D) tensor')
    n = t.shape
    if 0 in n:
        raise ValueError(f'{name} has an empty dimension: {tuple(n)}')
    return n


# ------------------------------------------------------------------ norm and rotation
def head_norm_rotate(q, k=None, wq=None, wk=None, turns=None, positions=None, first=0, eps=1e-6, out_q=None, out_k=None, v=None,
                     out_v=None, slots=None):
    """(q', k'): every head normalised by its root mean square, times the weight wq / wk (D,), its first 2 * turns.numel() dimensions
    turned by the token's position (positions (B, L) int32, None: first + index); pair i is dimensions i and i + turns.numel().
    Computed in fp64 and rounded once.  With out_k (and v, out_v) the keys (and values, unchanged) go there; with slots (B, L) int32
    to row slots[b, l] of it -- a cache (B, Lmax, Hk, D).  A slot outside the cache drops the row; two tokens of a sequence with the
    same slot leave either.  out_q / out_k may be q / k themselves."""
    n = _shape4(q, 'q')
    B, L, Hq, D = n
    dt = q.dtype
    qa = _tokens(q, 'q')
    wq_ = _array(wq, 'wq', (D,), _F32)
    if out_q is None:
        out_q = torch.empty_like(q)
    oq = _tokens(out_q, 'out_q', n, dt)
    ka = va = ok = ov = _NONE4
    Hk = rows = wk_ = slots_ = 0
    if k is not None:
        Hk = _shape4(k, 'k')[2]
        kn = (B, L, Hk, D)
        ka = _tokens(k, 'k', kn, dt)
        wk_ = _array(wk, 'wk', (D,), _F32)
        rows = L
        if slots is not None:
            if out_k is None:
                raise ValueError('slots need out_k (a cache)')
            slots_ = _array(slots, 'slots', (B, L), _I32)
            rows = _shape4(out_k, 'out_k')[1]
        if out_k is None:
            out_k = torch.empty_like(k)
        ok = _tokens(out_k, 'out_k', (B, rows, Hk, D), dt)
        if v is not None:
            if out_v is None:
                raise ValueError('v needs out_v')
            va, ov = _tokens(v, 'v', kn, dt), _tokens(out_v, 'out_v', (B, rows, Hk, D), dt)
    elif out_k is not None or v is not None or slots is not None:
        raise ValueError('out_k, v and slots need k')
    rot = 0 if turns is None else 2 * turns.numel()
    turns_, pos_ = _array(turns, 'turns', (rot // 2,), _F64), _array(positions, 'positions', (B, L), _I32)
    _on_device(('q', q), ('k', k), ('v', v), ('wq', wq), ('wk', wk), ('turns', turns), ('positions', positions), ('slots', slots),
               ('out_q', out_q), ('out_k', out_k), ('out_v', out_v))
    _call('scipnp_head_norm_rotate', _NORM.pack(
        _NORM.size, _DT[dt], B, L, Hq, Hk, D, rot, first, rows if slots is not None else 0, eps, qa[0], ka[0], va[0], oq[0], ok[0], ov[0],
        0, 0, 0, 0, *qa[1:], *ka[1:], *va[1:], *oq[1:], *ok[1:], *ov[1:], 0, 0, 0, 0, 0, 0, wq_, wk_, turns_, pos_, slots_, 0, 0))
    return out_q, out_k


def head_norm_rotate_backward(g_q, g_k, q, k, wq, wk, turns=None, positions=None, first=0, eps=1e-6):
    """(dq, dk, dwq, dwk) of head_norm_rotate from the gradients of its two results (k None: dk, dwk None)"""
    n = _shape4(q, 'q')
    B, L, Hq, D = n
    dt = q.dtype
    qa, ga = _tokens(q, 'q'), _tokens(g_q, 'g_q', n, dt)
    wq_ = _array(wq, 'wq', (D,), _F32)
    rot = 0 if turns is None else 2 * turns.numel()
    turns_, pos_ = _array(turns, 'turns', (rot // 2,), _F64), _array(positions, 'positions', (B, L), _I32)
    ka = gk = ok = _NONE4
    Hk = wk_ = dwk_ = 0
    dk = dwk = None
    if k is not None:
        Hk = _shape4(k, 'k')[2]
        kn = (B, L, Hk, D)
        ka, gk = _tokens(k, 'k', kn, dt), _tokens(g_k, 'g_k', kn, dt)
        wk_ = _array(wk, 'wk', (D,), _F32)
        dk, dwk = torch.empty(kn, dtype=dt, device=q.device), torch.empty_like(wk)
        ok, dwk_ = _tokens(dk, 'dk'), dwk.data_ptr()
    _on_device(('q', q), ('k', k), ('g_q', g_q), ('g_k', g_k if k is not None else None), ('wq', wq), ('wk', wk), ('turns', turns), ('positions', positions))
    dq, dwq = torch.empty(n, dtype=dt, device=q.device), torch.empty_like(wq)
    oq = _tokens(dq, 'dq')

    def block(ws, size):
        return _NORM.pack(_NORM.size, _DT[dt], B, L, Hq, Hk, D, rot, first, 0, eps, qa[0], ka[0], 0, oq[0], ok[0], 0, ga[0], gk[0], dwq.data_ptr(), dwk_,
                          *qa[1:], *ka[1:], 0, 0, 0, *oq[1:], *ok[1:], 0, 0, 0, *ga[1:], *gk[1:], wq_, wk_, turns_, pos_, 0, ws, size)
    size = _lib.load().scipnp_head_norm_rotate_backward_workspace_bytes(block(0, 0))
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    _call('scipnp_head_norm_rotate_backward', block(ws.data_ptr(), size))
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
    ka = _tokens(k, 'k')
    shape = (B, -(-Lk // block), Hk, D)
    if out is None:
        out = torch.empty(shape, dtype=_F32, device=k.device)
    args = (ka[0], (C.c_int64 * 3)(*ka[1:]), _DT[k.dtype], _array(klen, 'klen', (B,), _I32), _array(out, 'out', shape, _F32), B, Lk, Hk, D, block, newest)
    _on_device(('k', k), ('klen', klen), ('out', out))
    _call('scipnp_block_summary', *args)
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
    if block < 1 or query_block < 1 or n_sel < 1:
        raise ValueError(f'block {block}, query_block {query_block} and n_sel {n_sel} must be positive')
    Lk = nb * block if keys is None else int(keys)
    if -(-Lk // block) != nb:
        raise ValueError(f'{Lk} keys in blocks of {block} are not the {nb} blocks of the summary')
    qa = _tokens(q, 'q')
    su, ql, kl = _array(summary, 'summary', (B, nb, Hk, D), _F32), _array(qlen, 'qlen', (B,), _I32), _array(klen, 'klen', (B,), _I32)
    _on_device(('q', q), ('summary', summary), ('qlen', qlen), ('klen', klen))
    sel = torch.empty((B, Hk, -(-Lq // query_block), n_sel), dtype=_I32, device=q.device)
    _call('scipnp_select_blocks', _SELECT.pack(_SELECT.size, _DT[q.dtype], B, Lq, Lk, Hq, Hk, D, block, query_block, n_sel, sink, local, bool(causal),
                                               qa[0], *qa[1:], su, ql, kl, sel.data_ptr()))
    return sel


# ------------------------------------------------------------------ attention
def _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos):
    """the argument block as a function of out, the saved tensors, the gradients and the workspace"""
    B, Lq, Hq, D = _shape4(q, 'q')
    kn = _shape4(k, 'k')
    Lk, Hk = kn[1], kn[2]
    if kn[0] != B or kn[3] != D or Hq % Hk:
        raise ValueError(f'q {tuple(q.shape)} and k {tuple(kn)}: same batch and head size, query heads a multiple of key heads')
    if block < 1 or query_block < 1:
        raise ValueError(f'block {block} and query_block {query_block} must be positive')
    groups = -(-Lq // query_block)
    if not isinstance(sel, torch.Tensor) or sel.dim() != 4:
        raise ValueError(f'sel must be (B, Hk, groups, n) = ({B}, {Hk}, {groups}, n)')
    dt, n = q.dtype, sel.shape[3]
    qa, ka, va = _tokens(q, 'q'), _tokens(k, 'k', None, dt), _tokens(v, 'v', kn, dt)
    sel_ = _array(sel, 'sel', (B, Hk, groups, n), _I32)
    ql, kl = _array(qlen, 'qlen', (B,), _I32), _array(klen, 'klen', (B,), _I32)
    if (bias is None) != (bucket_of is None):
        raise ValueError('bias and bucket_of belong together')
    nbuckets = maxd = bias_ = bucket_ = qp = kp = 0
    if bias is not None:
        if bias.dim() != 2 or bucket_of.dim() != 1 or bucket_of.shape[0] % 2 == 0:
            raise ValueError('bias must be (buckets, Hq), bucket_of (2 * max_distance + 1,)')
        nbuckets, maxd = bias.shape[0], bucket_of.shape[0] // 2
        bias_, bucket_ = _array(bias, 'bias', (nbuckets, Hq), _F32), _array(bucket_of, 'bucket_of', (2 * maxd + 1,), _I32)
        qp, kp = _array(q_pos, 'q_pos', (B, Lq), _I32), _array(k_pos, 'k_pos', (B, Lk), _I32)
    elif q_pos is not None or k_pos is not None:
        raise ValueError('q_pos and k_pos are positions for the bias')
    _on_device(('q', q), ('k', k), ('v', v), ('sel', sel), ('qlen', qlen), ('klen', klen), ('bias', bias), ('bucket_of', bucket_of), ('q_pos', q_pos), ('k_pos', k_pos))
    front = (_ATTN.size, _DT[dt], B, Lq, Lk, Hq, Hk, D, block, query_block, n, bool(causal), nbuckets, maxd)
    inputs = (1.0 / math.sqrt(D) if scale is None else scale, qa[0], ka[0], va[0])
    strides = (*qa[1:], *ka[1:], *va[1:])
    middle = (sel_, ql, kl, bucket_, qp, kp, bias_)

    def pack(out=_NONE4, lse=0, out32=0, dout=_NONE4, grads=_NONE4, ws=0, size=0, zero_rest=False):
        return _ATTN.pack(*front, zero_rest, *inputs, out[0], *strides, *out[1:], *middle, lse, out32, *dout, *grads, ws, size)
    return pack, front


_BYTES = {}


def _forward_bytes(pack, front):
    """the forward workspace of these sizes (asked of the library once for each)"""
    key = front[1:11]
    size = _BYTES.get(key)
    if size is None:
        if len(_BYTES) > 4096:
            _BYTES.clear()
        size = _lib.load().scipnp_block_attn_workspace_bytes(pack(), 0)
        if size or _lib.load().scipnp_block_attn_workspace_bytes(pack(), 1):       # (0 for both: refused, nothing to remember)
            _BYTES[key] = size
    return size


def block_attention(q, k, v, sel, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None, bucket_of=None, bias=None,
                    q_pos=None, k_pos=None, out=None, save=False):
    """softmax(scale * q k^T + bias) v over the keys of each group's selected blocks (select_blocks; an entry outside the blocks, or
    not greater than those before it, is ignored).  scale None: 1 / sqrt(D).  causal: keys behind the query are masked.  bias
    (buckets, Hq) float32 by the relative position of key and query, bucket_of from bucket_table; q_pos (B, Lq), k_pos (B, Lk) int32
    name the positions (None: the key positions), e.g. the frame of each token of a video; differences must fit 32 bits.  A bias below
    -1e30 (-inf, a type's lowest value) masks its keys.  A query without a visible key gives zeros; what a key holds that a query does
    not see -- NaN, infinity -- does not reach it.  Rows behind qlen are zeros, or left as they were in a given `out`.
    save=True returns (out, saved) for block_attention_backward; bfloat16 probabilities are then multiplied whole, not rounded, so that
    the saved fp32 result carries the gradient (out is the same up to its rounding)."""
    pack, front = _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos)
    n, dt, dev = q.shape, q.dtype, q.device
    fresh = out is None
    if fresh:
        out = torch.empty_like(q)
    oa = _tokens(out, 'out', n, dt)
    _on_device(('out', out))
    saved = None
    lse = out32 = ws_ = 0
    if save:
        saved = (torch.empty((n[0], n[2], n[1]), dtype=_F32, device=dev), torch.empty(n, dtype=_F32, device=dev))
        lse, out32 = saved[0].data_ptr(), saved[1].data_ptr()
    size = _forward_bytes(pack, front)
    if size:
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        ws_ = ws.data_ptr()
    _call('scipnp_block_attn', pack(oa, lse, out32, ws=ws_, size=size, zero_rest=fresh))
    return (out, saved) if save else out


def block_attention_backward(dout, q, k, v, sel, saved, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None,
                             bucket_of=None, bias=None, q_pos=None, k_pos=None):
    """(dq, dk, dv, dbias) of block_attention called with the same arguments and save=True; rows behind qlen / klen are zeros, dbias
    (buckets, Hq) float32 is None without a bias.  The selection is not differentiated.  q, k, v and dout of the live rows must be finite:
    here a NaN or an infinity reaches every gradient of its block of 64."""
    pack, _ = _attn_args(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos)
    n, dev = q.shape, q.device
    da = _tokens(dout, 'dout', n, q.dtype)
    lse, out32 = saved
    lse_, out32_ = _array(lse, 'saved[0]', (n[0], n[2], n[1]), _F32), _array(out32, 'saved[1]', n, _F32)
    _on_device(('dout', dout), ('saved[0]', lse), ('saved[1]', out32))
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    dbias = torch.empty_like(bias) if bias is not None else None
    grads = (dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 0 if dbias is None else dbias.data_ptr())
    size = _lib.load().scipnp_block_attn_workspace_bytes(pack(_NONE4, lse_, out32_, da, grads), 1)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _call('scipnp_block_attn_backward', pack(_NONE4, lse_, out32_, da, grads, ws.data_ptr(), size))
    return dq, dk, dv, dbias
