"""CPU: what the non-local prior refuses before it touches the GPU, and its C entries' argument checks"""
import pytest
import torch

from adaptivepnp_sci_amd import NonLocalPrior, _lib
from adaptivepnp_sci_amd.nonlocal_prior import NonLocalEngine


@pytest.mark.parametrize('kw', [dict(n_sel=0), dict(n_sel=1025), dict(shifts=3), dict(shifts=0), dict(num_buckets=3), dict(num_buckets=65),
                                dict(num_buckets=16, max_distance=4), dict(max_distance=4097)])
def test_prior_sizes(kw):
    with pytest.raises(ValueError):
        NonLocalPrior(**kw)


def test_engine_arguments():
    with pytest.raises(ValueError, match='NonLocalPrior'):
        NonLocalEngine(torch.nn.Linear(2, 2), 4, 32, 32, 'cpu')
    with pytest.raises(ValueError, match='units'):
        NonLocalEngine(NonLocalPrior(), 4, 32, 32, 'cpu', units=3)


@pytest.mark.parametrize('bad', [dict(B=0), dict(H=0), dict(W=-1), dict(units=3), dict(units=0), dict(shifts=3), dict(shifts=0), dict(H=1 << 21)])
def test_entries_refuse_shapes(bad):
    lib = _lib.load()
    a = dict(B=4, H=32, W=32, units=1, shifts=2)
    a.update(bad)
    n = (a['B'], a['H'], a['W'], a['units'], a['shifts'])
    assert lib.scipnp_patch_tokens(64, 64, *n, 1.0, 1.0, 1, None) != 0 and b'shape' in lib.scipnp_last_error()
    assert lib.scipnp_patch_frames(64, 64, *n, None) != 0


def test_entries_refuse_pointers():
    lib = _lib.load()
    assert lib.scipnp_patch_tokens(None, 64, 1, 32, 32, 1, 1, 1.0, 1.0, 1, None) != 0
    assert lib.scipnp_patch_tokens(64, 68, 1, 32, 32, 1, 1, 1.0, 1.0, 1, None) != 0
    assert lib.scipnp_patch_frames(64, None, 1, 32, 32, 1, 1, None) != 0
