"""CPU: tensors that do not fit each other or the engine are refused before any launch"""
import pytest
import torch

from adaptivepnp_sci_amd import NonLocalPrior, _lib, ops
from adaptivepnp_sci_amd.nonlocal_prior import NonLocalEngine, nonlocal_online_finetune


@pytest.mark.parametrize('shape', [(2, 4 * 64 * 4, 1, 56), (2, 2 * 64 * 4, 1, 56), (1, 4 * 64, 1, 56), (2, 4 * 64, 1, 48)])
@pytest.mark.parametrize('call', [lambda f, t: ops.patch_tokens(f, t, 1, 2, 1.0), lambda f, t: ops.patch_frames(t, f, 1, 2)])
def test_tokens_of_another_size(call, shape):
    """4 frames of 30 x 30, two grids: one tile a frame, (2, 256, 1, 56)"""
    with pytest.raises(ValueError, match='tokens of 4 frames'):
        call(torch.zeros(4, 3, 30, 30), torch.zeros(shape))
    with pytest.raises(ValueError, match='frames must be'):
        call(torch.zeros(4, 30, 30), torch.zeros(2, 256, 1, 56))
    with pytest.raises(_lib.ScipnpError, match='no CPU fallback'):
        call(torch.zeros(4, 3, 30, 30), torch.zeros(2, 256, 1, 56))


def test_frames_of_another_size():
    eng = NonLocalEngine(NonLocalPrior(), 4, 64, 64, 'cpu')
    for shape in ((4, 3, 128, 128), (3, 3, 64, 64), (4, 3, 32, 64), (4, 1, 64, 64)):
        with pytest.raises(ValueError, match='frames must be'):
            eng.forward(torch.zeros(shape), 0.1)


@pytest.mark.parametrize('size', [(63, 64), (64, 31)])
def test_adaptation_needs_whole_bayer_cells(size):
    eng = NonLocalEngine(NonLocalPrior(), 2, *size, 'cpu')
    M, N = size[0] // 2, size[1] // 2
    with pytest.raises(ValueError, match='even sizes'):
        nonlocal_online_finetune(NonLocalPrior(), eng, torch.zeros(2, 3, *size), torch.zeros(4, M, N), torch.zeros(2, 4, M, N), 0.1, 1e-3, 1)


@pytest.mark.parametrize('bad, word', [
    (dict(frames=torch.zeros(3, 3, 64, 64)), 'frames'), (dict(frames=torch.zeros(2, 3, 64, 64).double()), 'frames'), (dict(y=torch.zeros(4, 64, 64)), 'y_pm'),
    (dict(y=torch.zeros(32, 32, 4).permute(2, 0, 1)), 'y_pm'), (dict(y=torch.zeros(4, 32, 32).double()), 'y_pm'), (dict(Phi=torch.zeros(1, 4, 32, 32)), 'Phi_pm'),
    (dict(Phi=torch.zeros(2, 4, 32, 32).half()), 'Phi_pm')])
def test_adaptation_needs_a_measurement_that_fits(bad, word):
    eng = NonLocalEngine(NonLocalPrior(), 2, 64, 64, 'cpu')
    a = dict(frames=torch.zeros(2, 3, 64, 64), y=torch.zeros(4, 32, 32), Phi=torch.zeros(2, 4, 32, 32))
    a.update(bad)
    with pytest.raises(ValueError, match=f'{word} must be'):
        nonlocal_online_finetune(NonLocalPrior(), eng, a['frames'], a['y'], a['Phi'], 0.1, 1e-3, 1)
