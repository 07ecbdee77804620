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

Like every kernel of this package the calls are outside autograd: results require no gradient whatever the inputs do, forward-mode tangents
are dropped, and the *_backward functions are called by hand or from a torch.autograd.Function of the program.  A given result that is
written raises its version counter, so autograd refuses a backward pass that had saved what was there.
"""
import ctypes as C
import importlib
import math
import re

import torch

from . import _lib
from ._lib import ScipnpError

_ENTRIES = ('scipnp_head_norm_rotate', 'scipnp_head_norm_rotate_backward', 'scipnp_head_norm_rotate_backward_workspace_bytes', 'scipnp_block_summary',
            'scipnp_select_blocks', 'scipnp_block_attn_workspace_bytes', 'scipnp_block_attn', 'scipnp_block_attn_backward')
_bound = None


def _bind():
    """csrc/attn_bind.cpp, which checks the tensors, allocates the results and makes the C call, bound to the loaded library"""
    global _bound
    lib = _lib.load()
    try:
        mod = importlib.import_module('._attn_bind', __package__)
    except ImportError as e:
        raise ScipnpError(f'{e}: build it with `make -C adaptivepnp_sci_amd/csrc`') from e
    if mod.built_for != '.'.join(re.findall(r'\d+', torch.__version__)[:3]):          # (the headers know the three numbers)
        raise ScipnpError(f'_attn_bind.so was built for torch {mod.built_for}, this is {torch.__version__}: build it again with `make -C adaptivepnp_sci_amd/csrc`')
    mod.bind(*(C.cast(getattr(lib, n), C.c_void_p).value for n in _ENTRIES), _lib.check, ScipnpError, torch.cuda.current_device,
             getattr(torch._C, '_cuda_getCurrentRawStream', None) or _raw_stream)
    if torch.cuda.is_available():
        _lib.require_gpu()
    _bound = mod
    return mod


def _raw_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


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


# ------------------------------------------------------------------ norm and rotation
def head_norm_rotate(q, k=None, wq=None, wk=None, turns=None, positions=None, first=0, eps=1e-6, out_q=None, out_k=None, v=None,
                     out_v=None, slots=None):
    """(q', k'): every head normalised by its root mean square, times the weight wq / wk (D,), its first 2 * turns.numel() dimensions
    turned by the token's position (positions (B, L) int32, None: first + index); pair i is dimensions i and i + turns.numel().
    Computed in fp64 and rounded at the end (bfloat16 by way of float32).  With out_k (and v, out_v) the keys (and values, unchanged) go
    there; with slots (B, L) int32 to row slots[b, l] of it -- a cache (B, Lmax, Hk, D).  A slot outside the cache drops the row; two tokens of a sequence with the
    same slot leave either.  out_q / out_k / out_v may be q / k / v themselves; results that share memory in another way are refused."""
    return (_bound or _bind()).head_norm_rotate(q, k, wq, wk, turns, positions, first, eps, out_q, out_k, v, out_v, slots)


def head_norm_rotate_backward(g_q, g_k, q, k, wq, wk, turns=None, positions=None, first=0, eps=1e-6):
    """(dq, dk, dwq, dwk) of head_norm_rotate from the gradients of its two results (k None: dk, dwk None)"""
    return (_bound or _bind()).head_norm_rotate_backward(g_q, g_k, q, k, wq, wk, turns, positions, first, eps)


# ------------------------------------------------------------------ summary and selection
def block_summary(k, block=64, klen=None, newest=0, out=None):
    """mean key of every block of `block` keys over its live ones: (B, ceil(Lk / block), Hk, D) float32, zeros behind klen.  newest=n
    writes only the blocks that the last n live keys touch (out: the summary of the cache before them)."""
    return (_bound or _bind()).block_summary(k, block, klen, newest, out)


def select_blocks(q, summary, n_sel, block=64, query_block=64, keys=None, causal=False, qlen=None, klen=None, sink=1, local=1):
    """the n_sel key blocks of every group of query_block queries (and the query heads of a key head): (B, Hk, groups, n_sel) int32,
    ascending, -1 behind the last.  Score: (sum of the group's queries) . (mean key), in fp64; ties to the lower block.  The `sink`
    first blocks and the blocks within local - 1 of the group's last query come before every score.  keys: length of the key
    sequence (None: the summary's blocks are full); causal: only blocks that begin at or before the group's last query."""
    return (_bound or _bind()).select_blocks(q, summary, n_sel, block, query_block, keys, causal, qlen, klen, sink, local)


# ------------------------------------------------------------------ attention
def block_attention(q, k, v, sel, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None, bucket_of=None, bias=None,
                    q_pos=None, k_pos=None, out=None, save=False):
    """softmax(scale * q k^T + bias) v over the keys of each group's selected blocks (select_blocks; an entry outside the blocks, or
    not greater than those before it, is ignored).  scale None: 1 / sqrt(D).  causal: keys behind the query are masked.  bias
    (buckets, Hq) float32 by the relative position of key and query, bucket_of from bucket_table; q_pos (B, Lq), k_pos (B, Lk) int32
    name the positions (None: the key positions), e.g. the frame of each token of a video; differences must fit 32 bits.  A bias below
    -1e30 (-inf, a type's lowest value) masks its keys.  A query without a visible key gives zeros; what a key holds that a query does
    not see -- NaN, infinity -- does not reach it.  Rows behind qlen are zeros, or left as they were in a given `out` (q itself, or memory of its own).
    bfloat16 probabilities go into the product with v in two numbers, off by 2^-16.  save=True returns (out, saved) for
    block_attention_backward, saved = (log-sum-exp (B, Hq, Lq), fp32 result, what the first was rounded by; rows behind qlen are not written);
    the probabilities are then multiplied whole, in three, because the saved result carries the gradient: out can differ by a rounding."""
    return (_bound or _bind()).block_attention(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos, out, save)


def block_attention_backward(dout, q, k, v, sel, saved, block=64, query_block=64, scale=None, causal=False, qlen=None, klen=None,
                             bucket_of=None, bias=None, q_pos=None, k_pos=None):
    """(dq, dk, dv, dbias) of block_attention called with the same arguments and save=True; rows behind qlen / klen are zeros, dbias
    (buckets, Hq) float32 is None without a bias.  The selection is not differentiated.  q, k, v and dout of the live rows must be finite:
    here a NaN or an infinity reaches every gradient of its block of 64."""
    lse, out32, rest = saved
    return (_bound or _bind()).block_attention_backward(q, k, v, sel, block, query_block, scale, causal, qlen, klen, bucket_of, bias, q_pos, k_pos, dout, lse,
                                                        out32, rest)
