"""pmg::embedding and its gradient against the 64-bit plain form: element types, odd and large sizes, strides and
alignments, frequent tokens, padding, empty batches, repeated and captured calls, autograd."""
import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ids(n, V, seed, kind='mixed'):
    g = torch.Generator().manual_seed(seed)
    if kind == 'one':
        return torch.full((n,), V - 1)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return (u.pow(3) * V).long().clamp_(max=V - 1)


def _tol(t, exact):
    """One rounding of the product to fp32 and one to the type; half a step of the subnormals."""
    f = torch.finfo(t)
    return exact.abs() * (f.eps / 2 + 2.0 ** -23) + f.tiny * f.eps


def _check_grad(got, grad, ids, V, scale, pad=-1):
    exact, size, count = lm.embedding_grad(grad.cpu(), ids.cpu(), V, scale, pad)
    got = got.cpu().double()
    # every position enters through at most `count` additions in fp32, then one product and one rounding
    bound = size * ((count.double() + 2) * 2.0 ** -24).unsqueeze(1) + _tol(grad.dtype, exact)
    assert bool(((got - exact).abs() <= bound).all()), float(((got - exact).abs() - bound).max())
    assert not got[count == 0].any()


SIZES = [(1, 1, 1), (1, 5, 3), (2, 3, 4), (63, 7, 8), (64, 60, 128), (65, 1, 33), (700, 100000, 20), (2048, 300, 16),
         (2049, 300, 17), (4096, 511, 264), (4097, 512, 8), (20001, 3, 40), (33000, 70001, 12), (9000, 600, 4104)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('n,V,E', SIZES)
def test_forward_and_gradient(gpu, dtype, n, V, E):
    from paccmann_generator_amd import ops
    torch.manual_seed(n + V + E)
    weight = torch.randn(V, E).to(dtype)
    ids = _ids(n, V, n)
    grad = torch.randn(n, E).to(dtype)
    for scale, pad, kind in ((1.0, None, torch.int64), (3.7, 0, torch.int32)):
        scale = float(torch.tensor(scale))
        w = weight.cuda().requires_grad_(True)
        out = ops.embedding(w, ids.to(kind).cuda(), scale=scale, padding_idx=pad)
        exact = lm.embedding(weight, ids, scale)
        assert out.dtype == dtype and out.shape == (n, E)
        assert bool(((out.detach().cpu().double() - exact).abs() <= _tol(dtype, exact)).all())
        got, = torch.autograd.grad(out, w, grad.cuda())
        _check_grad(got, grad, ids, V, scale, -1 if pad is None else pad)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_one_token_in_every_position(gpu, dtype):
    """A run that spans all chunks, wide and narrow rows."""
    for n, V, E in ((70000, 9, 40), (3000, 2, 2000), (2500, 4, 1)):
        torch.manual_seed(0)
        grad = torch.randn(n, E).to(dtype)
        ids = _ids(n, V, 0, 'one')
        got = torch.ops.pmg.embedding_bwd(grad.cuda(), ids.cuda(), V, 1.0, -1)
        _check_grad(got, grad, ids, V, 1.0)


def test_runs_that_end_at_chunk_borders(gpu):
    """Sorted ids whose runs have every length around the chunk sizes 8 to 64."""
    lens = [1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1]
    for times in (1, 4, 40, 120):
        ids = torch.cat([torch.full((k,), i) for i, k in enumerate(lens * times)])
        ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(times))]
        V = len(lens) * times + 3
        torch.manual_seed(times)
        grad = torch.randn(ids.numel(), 20)
        got = torch.ops.pmg.embedding_bwd(grad.cuda(), ids.cuda(), V, 1.0, 5)
        _check_grad(got, grad, ids, V, 1.0, 5)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_strides_offsets_and_shapes(gpu, dtype):
    from paccmann_generator_amd import ops
    torch.manual_seed(1)
    V, E = 50, 24
    base = torch.randn(V * 40 + 8).to(dtype).cuda()
    ids = _ids(6 * 35, V, 3).view(6, 35).cuda()
    for off, ld in ((0, 40), (1, 33), (3, 25), (8, 24)):
        w = base[off:off + V * ld].view(V, ld)[:, :E].detach().requires_grad_(True)
        out = ops.embedding(w, ids)
        assert out.shape == (6, 35, E) and torch.equal(out, w.detach()[ids])
        wide = torch.randn(6, 35, E + 5, device='cuda').to(dtype)
        for g in (wide[..., :E], wide[..., 5:], torch.randn(35, 6, E, device='cuda').to(dtype).transpose(0, 1),
                  torch.randn(1, 1, E, device='cuda').to(dtype).expand(6, 35, E),
                  torch.randn(6, 35, 1, device='cuda').to(dtype).expand(6, 35, E)):
            got, = torch.autograd.grad(ops.embedding(w, ids, padding_idx=V - 1), w, g)
            assert got.shape == (V, E)
            _check_grad(got, g.contiguous(), ids, V, 1.0, V - 1)
    t = torch.randn(E, V, device='cuda').to(dtype).t()          # a transposed table
    assert torch.equal(ops.embedding(t, ids), t[ids])
    odd = ids.t()                                               # ids in another order
    assert torch.equal(ops.embedding(t, odd), t[odd])


def test_empty_batch_and_single_token(gpu):
    from paccmann_generator_amd import ops
    w = torch.randn(30, 12, device='cuda', requires_grad=True)
    out = ops.embedding(w, torch.zeros(0, 4, dtype=torch.long, device='cuda'))
    assert out.shape == (0, 4, 12)
    got, = torch.autograd.grad(out.sum(), w)
    assert got.shape == (30, 12) and not got.any()
    one = ops.embedding(w, torch.tensor(7, device='cuda'))
    assert one.shape == (12,) and torch.equal(one, w[7])
    pad_only = torch.ops.pmg.embedding_bwd(torch.randn(5000, 12, device='cuda'),
                                           torch.full((5000,), 3, device='cuda'), 30, 1.0, 3)
    assert not pad_only.any()


def test_ids_out_of_range(gpu):
    """Checked on the host; trusted ones that are wrong after all are loud and harmless."""
    from paccmann_generator_amd import _ffi, ops
    w = torch.randn(10, 8, device='cuda')
    bad = torch.tensor([1, 10, -1, 9], device='cuda')
    with pytest.raises(_ffi.PmgError):
        ops.embedding(w, bad)
    out = ops.embedding(w, bad, trusted_tokens=True)
    assert out[[1, 2]].isnan().all() and torch.equal(out[[0, 3]], w[[1, 9]])
    g = torch.randn(4, 8, device='cuda')
    got = torch.ops.pmg.embedding_bwd(g, bad, 10, 1.0, -1)
    assert torch.equal(got[1], g[0]) and torch.equal(got[9], g[3]) and int(got.any(1).sum()) == 2


def test_repeats_are_bit_identical_and_replays_equal_eager(gpu):
    from paccmann_generator_amd import ops
    for n, V, E in ((300, 50, 16), (30000, 900, 72)):
        w = torch.randn(V, E, device='cuda')
        ids, grad = _ids(n, V, 5).cuda(), torch.randn(n, E, device='cuda')

        def both():
            return (ops.embedding(w, ids, 0.5, trusted_tokens=True), torch.ops.pmg.embedding_bwd(grad, ids, V, 0.5, 2))

        eager = both()
        assert all(torch.equal(a, b) for a, b in zip(eager, both()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        for k in range(3):
            ids.copy_(_ids(n, V, 20 + k))
            grad.normal_()
            graph.replay()
            torch.cuda.synchronize()
            now = [x.clone() for x in held]
            assert all(torch.equal(a, b) for a, b in zip(now, both()))


def test_opcheck_and_differences(gpu):
    from paccmann_generator_amd import ops
    w = torch.randn(11, 8, device='cuda', requires_grad=True)
    ids = torch.tensor([[1, 5, 5], [0, 10, 1]], device='cuda')
    torch.library.opcheck(torch.ops.pmg.embedding, (w, ids, 2.0, 0))
    torch.library.opcheck(torch.ops.pmg.embedding_bwd, (torch.randn(2, 3, 8, device='cuda'), ids, 11, 2.0, 0))
    # the operator is linear in the table: a difference along any direction equals the gradient's product with it
    probe, along = torch.randn(2, 3, 8, device='cuda'), torch.randn(11, 8, device='cuda')
    got, = torch.autograd.grad((ops.embedding(w, ids, 2.0) * probe).sum(), w)
    with torch.no_grad():
        diff = ((ops.embedding(along, ids, 2.0) * probe).double().sum())
    assert abs(float((got * along).double().sum() - diff)) < 1e-5 * float(probe.abs().sum() * 4)


def test_offsets_beyond_32_bits(gpu):
    """A table of 4.9 GB and its gradient."""
    from paccmann_generator_amd import ops
    V, E = 1200000, 1024
    table = torch.zeros(V, E, device='cuda')
    ids = torch.cat([torch.tensor([V - 1, 0, V - 2, V - 1]), torch.randint(0, V, (3000,), generator=torch.Generator().manual_seed(1))])
    rows = torch.randn(len(ids), E, generator=torch.Generator().manual_seed(2))
    first = {int(v): n for n, v in reversed(list(enumerate(ids.tolist())))}
    there = torch.tensor([first[int(v)] for v in ids])
    table[ids.cuda()] = rows[there].cuda()
    table.requires_grad_(True)
    y = ops.embedding(table, ids.cuda())
    assert torch.equal(y.detach().cpu(), rows[there])
    slope = torch.randn(len(ids), E, generator=torch.Generator().manual_seed(3))
    dw, = torch.autograd.grad(y, table, slope.cuda())
    unique, place = ids.unique(return_inverse=True)
    exact = torch.zeros(len(unique), E, dtype=torch.float64).index_add_(0, place, slope.double())
    size = torch.zeros_like(exact).index_add_(0, place, slope.double().abs())
    count = torch.bincount(place).double().unsqueeze(1)
    assert bool(((dw[unique.cuda()].cpu().double() - exact).abs() <= size * (count + 2) * 2.0 ** -24 + exact.abs() * 2.0 ** -23).all())
    dw[unique.cuda()] = 0.0
    assert not bool(dw.any())


def test_the_gradient_is_not_differentiated_again(gpu):
    from paccmann_generator_amd import ops
    w = torch.randn(9, 5, device='cuda', requires_grad=True)
    y = ops.embedding(w, torch.tensor([1, 2, 1], device='cuda'))
    d, = torch.autograd.grad((y * y).sum(), w, create_graph=True)
    assert bool((d[1] - 4 * w[1]).abs().max() <= 1e-5) and not d[0].any()
    with pytest.raises(RuntimeError, match='not differentiable'):
        torch.autograd.grad(d.sum(), w)
