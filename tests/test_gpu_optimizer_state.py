"""optim.AdamW on the GPU: copies go on like their original, states change hands with the torch classes."""
import copy
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


def _params(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).cuda().requires_grad_(True) for s in ((13, 7), (300,), (5, 4, 6), (1,))]


def _step(opt, k):
    for i, p in enumerate(p for group in opt.param_groups for p in group['params']):
        p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i)).cuda()
    opt.step()


@pytest.mark.parametrize('through', [copy.deepcopy, lambda opt: pickle.loads(pickle.dumps(opt))], ids=['copy', 'pickle'])
@pytest.mark.parametrize('bits', [32, 8])
def test_a_copy_steps_like_its_original(gpu, bits, through):
    from paccmann_generator_amd import AdamW
    ps = _params()
    opt = AdamW([dict(params=ps[:2], lr=1e-2), dict(params=ps[2:])], state_bits=bits, max_grad_norm=0.5)
    _step(opt, 0)
    again = through(opt)
    for k in (1, 2):
        _step(opt, k)
        _step(again, k)
    assert torch.equal(opt.grad_norm, again.grad_norm)
    for a, b in zip(opt.param_groups, again.param_groups):
        for p, q in zip(a['params'], b['params']):
            assert p is not q and torch.equal(p, q) and int(again.state[q]['step']) == 3
            assert all(torch.equal(x, again.state[q][n]) for n, x in opt.state[p].items())
