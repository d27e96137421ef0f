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


@pytest.mark.parametrize('foreach', [False, True])
@pytest.mark.parametrize('decoupled', [False, True])
def test_torch_goes_on_from_our_checkpoint(gpu, decoupled, foreach):
    """Three steps here, two there, against five steps here: the classes make the same update up to roundings."""
    from paccmann_generator_amd import AdamW
    a, b = _params(1), _params(1)
    kw = dict(lr=1e-2, weight_decay=0.1)
    opt, ref = AdamW(a, decoupled=decoupled, **kw), AdamW(b, decoupled=decoupled, **kw)
    for k in range(3):
        _step(opt, k)
        _step(ref, k)
    theirs = (torch.optim.AdamW if decoupled else torch.optim.Adam)(a, foreach=foreach, **kw)
    theirs.load_state_dict(opt.state_dict())
    for g in theirs.param_groups:
        g['foreach'] = foreach
    for k in (3, 4):
        _step(theirs, k)
        _step(ref, k)
    assert all(float(theirs.state[p]['step']) == 5 for p in a)
    for x, y in zip(a, b):
        # a step moves by at most lr / (1 - 0.9^4) |m| / sqrt(v) < 10 lr, off by up to 32 roundings (moments, root, quotient);
        # the parameter's own two roundings a step
        assert float((x - y).detach().abs().max()) <= 2 * (10 * 1e-2 * 32 + 2 * float(y.detach().abs().max())) * 2.0 ** -24


def test_clipping_of_a_flat_buffer_with_empty_tensors(gpu):
    """Views of one buffer, empty ones at the start of others and inside them."""
    from paccmann_generator_amd import ops
    flat = torch.randn(1000, device='cuda')
    want = flat.double()
    got = [flat[0:0], flat[0:400], flat[200:200], flat[400:1000].view(20, 30), flat[400:400].view(0, 7), flat[1000:]]
    norm = ops.clip_grad_norm_(got, 2.0)
    exact = float(want.norm())
    # the norm and the factor rounded to fp32, the product
    assert abs(float(norm) - exact) <= 1.001 * 2.0 ** -24 * exact
    want = want * (2.0 / (exact + 1e-6))
    assert bool(((flat.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all())
