"""pmg::linear_cross_entropy against the 64-bit plain form: forward and gradients, both types, every tile shape, odd
and large sizes, ignored and masked rows, strides, scales, reductions, slopes of both outputs, captured calls."""
import math

import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _data(N, V, H, dtype, seed=0, bias=False, weighted=False, ignored=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    w = (torch.randn(V, H, generator=g) * 2 / math.sqrt(H)).to(dtype)
    b = (torch.randn(V, generator=g) * 0.3).to(dtype) if bias else None
    t = torch.randint(0, V, (N,), generator=g)
    if ignored:
        t[torch.rand(N, generator=g) < ignored] = -100
    r = torch.rand(N, generator=g) - 0.3 if weighted else None
    return x, w, b, t, r


def _cuda(*ts):
    return [t.cuda() if t is not None else None for t in ts]


def _check(x, w, b, t, r, scale=1.0, reduction='mean', lse_slope=None, ignore=-100):
    """Runs the operator on CPU data moved to the GPU and checks every output against its bound."""
    from paccmann_generator_amd import ops
    dx, dw, db, dt, dr = _cuda(x, w, b, t, r)
    leaves = [z.requires_grad_(True) for z in (dx, dw, db) if z is not None]
    loss, lse = ops.linear_cross_entropy(dx, dw, dt, bias=db, row_weight=dr, ignore_index=ignore, logit_scale=scale,
                                         reduction=reduction)
    e = lm.linear_ce(x, w, t, b, r, scale, reduction, ignore)
    H, V = x.shape[-1], w.shape[0]
    # a logit: H products summed in fp32 (exact products of bf16; of fp32 one rounding more), bias and scale; log and
    # exp add a few steps relative to the logits' size
    size = e['size']                       # [N] largest sum of magnitudes over the row's logits
    tol = (H + 16) * U * size + 8 * U
    assert bool(((lse.detach().cpu().double() - e['lse']).abs() <= tol + 2 * U * e['lse'].abs()).all())
    per_row = (2 * tol + 4 * U * e['lse'].abs()) * e['w'].abs()
    got = loss.detach().cpu().double()
    if reduction == 'none':
        assert bool(((got - e['loss']).abs() <= per_row + 2 * U * e['loss'].abs()).all())
    else:
        total = per_row.sum() / (max(1, e['count']) if reduction == 'mean' else 1)
        assert abs(float(got - e['loss'])) <= float(total) + 2 * U * abs(float(e['loss'])) + 1e-12
    slope = torch.randn(got.shape, generator=torch.Generator().manual_seed(9)) if reduction == 'none' else torch.tensor(1.7)
    out = (loss * slope.cuda()).sum()
    if lse_slope is not None:
        out = out + (lse * lse_slope.cuda()).sum()
    got = torch.autograd.grad(out, leaves)
    grads = lm.linear_ce_grads(x, w, t, b, r, scale, reduction, ignore, slope, lse_slope)
    f = torch.finfo(x.dtype)
    # dl: the exponential's error, relative, and its rounding to the operands' type; then a sum in fp32 and a rounding
    rel = float(4 * tol.max()) + 16 * U + (0 if x.dtype == torch.float32 else f.eps / 2)
    for name, g in zip(('x', 'w', 'b'), got):
        exact, mag = grads[name], grads['|' + name + '|']
        # the split product sums in fp32: at most its length in roundings, relative to the sum of magnitudes
        length = {'x': V, 'w': x.reshape(-1, H).shape[0], 'b': x.reshape(-1, H).shape[0]}[name]
        bound = mag * (rel + (length + 8) * U) + exact.abs() * f.eps / 2 * 1.01
        off = (g.cpu().double() - exact).abs()
        assert g.dtype == x.dtype and g.shape == exact.shape
        assert bool((off <= bound + 1e-30).all()), (name, float((off - bound).max()))
    return loss, lse


TYPES = [torch.float32, torch.bfloat16]
SIZES = [  # tokens, vocabulary, hidden: every tile shape, sizes around the tiles' and stages' edges
    (1, 2, 1), (1, 1, 8), (3, 60, 16), (16, 130, 64), (17, 300, 40), (33, 65, 24), (64, 1000, 32), (65, 64, 128),
    (100, 60, 256), (255, 257, 64), (256, 256, 128), (257, 511, 72), (300, 129, 33), (1, 5000, 96), (700, 4097, 56),
    (5000, 60, 128), (70000, 23, 32), (2, 70001, 16), (1025, 1030, 520)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,V,H', SIZES)
def test_against_the_definition(gpu, dtype, N, V, H):
    _check(*_data(N, V, H, dtype, seed=N + V + H))
    _check(*_data(N, V, H, dtype, seed=N, bias=True, weighted=True, ignored=0.3), scale=0.7, reduction='sum')


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
def test_reductions_and_slopes_of_both_outputs(gpu, dtype, reduction):
    for N, V, H in ((40, 90, 48), (300, 700, 64)):
        x, w, b, t, r = _data(N, V, H, dtype, seed=3, bias=True, weighted=True, ignored=0.2)
        z = torch.randn(N, generator=torch.Generator().manual_seed(1))
        z[5] = 0.0
        _check(x, w, b, t, r, scale=1.3, reduction=reduction, lse_slope=z)


def test_large_vocabulary_in_pieces(gpu):
    """Several pieces of the vocabulary: gradients of hidden summed over them, a short last piece."""
    from paccmann_generator_amd import ops
    N, V, H = 4096, 40000 + 17, 64
    x, w, b, t, r = _data(N, V, H, torch.bfloat16, seed=2, bias=True, ignored=0.1)
    dx, dw, db, dt, _ = _cuda(x, w, b, t, r)
    for z in (dx, dw, db):
        z.requires_grad_(True)
    loss, _ = ops.linear_cross_entropy(dx, dw, dt, bias=db)
    got = torch.autograd.grad(loss, (dx, dw, db))
    e = lm.linear_ce_grads(*(z.cuda() if z is not None else None for z in (x, w, t, b, r)), 1.0, 'mean', -100,
                           torch.tensor(1.0).cuda(), None)
    for name, g in zip('xwb', got):
        exact, mag = e[name], e['|' + name + '|']
        assert bool(((g.double() - exact).abs() <= mag * (2.0 ** -8 + 4096 * U) + exact.abs() * 2.0 ** -8 * 1.01).all()), name


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_strides_alignments_and_shapes(gpu, dtype):
    from paccmann_generator_amd import ops
    N, V, H = 60, 150, 40
    x, w, b, t, _ = _data(N, V, H, dtype, seed=5, bias=True)
    want = _check(x, w, b, t, None)
    base = torch.zeros(200 * 64 + 16, dtype=dtype, device='cuda')

    def place(src, off, ld):
        v = base.new_zeros(base.shape)[off:off + src.shape[0] * ld].view(src.shape[0], ld)[:, :H]
        v.copy_(src.cuda())
        return v

    for off, ld in ((0, 40), (0, 48), (8, 56), (1, 40), (0, 41), (3, 47), (4, 44)):
        xs, ws = place(x, off, ld).requires_grad_(True), place(w, off, ld).requires_grad_(True)
        loss, lse = ops.linear_cross_entropy(xs, ws, t.cuda().to(torch.int32), bias=b.cuda())
        assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
        g = torch.autograd.grad(loss, (xs, ws))
        assert g[0].shape == x.shape and g[1].shape == w.shape and all(z.isfinite().all() for z in g)
    # [batch, time, H] in another order of its dimensions, targets alike; a transposed weight; an expanded hidden
    x3, t3 = x.view(6, 10, H).cuda(), t.view(6, 10).cuda()
    loss, lse = ops.linear_cross_entropy(x3.transpose(0, 1), w.cuda(), t3.t(), bias=b.cuda())
    assert lse.shape == (10, 6) and torch.equal(lse.t().reshape(-1), want[1])
    wt = w.t().contiguous().cuda().t()
    assert torch.equal(ops.linear_cross_entropy(x.cuda(), wt, t.cuda(), bias=b.cuda())[1], want[1])
    one = x[:1].cuda().requires_grad_(True)
    _, lse = ops.linear_cross_entropy(one.expand(N, H), w.cuda(), t.cuda(), bias=b.cuda())
    assert torch.equal(lse, lse[:1].expand(N)) and abs(float((lse[0] - want[1][0]).detach())) < 1e-5
    g, = torch.autograd.grad(lse.sum(), one)
    assert g.shape == (1, H)


def test_rows_that_are_masked(gpu):
    """Batches without targets, ignored rows of any content, a vocabulary masked to one entry or to none."""
    from paccmann_generator_amd import ops
    for dtype in TYPES:
        x, w, b, t, _ = _data(50, 80, 32, dtype, seed=6, bias=True)
        dx, dw, db = (z.cuda().requires_grad_(True) for z in (x, w, b))
        for reduction in ('mean', 'sum'):
            loss, lse = ops.linear_cross_entropy(dx, dw, torch.full((50,), -1, device='cuda'), bias=db, ignore_index=-1,
                                                 reduction=reduction)
            assert float(loss.detach()) == 0.0 and lse.isfinite().all()
            assert not any(g.any() for g in torch.autograd.grad(loss, (dx, dw, db)))
        # an entry of -inf in the bias is out of the vocabulary: no probability, no gradient
        b2 = b.clone()
        b2[10:] = -float('inf')
        t2 = t % 10
        db2 = b2.cuda().requires_grad_(True)
        loss, lse = ops.linear_cross_entropy(dx, dw, t2.cuda(), bias=db2)
        g = torch.autograd.grad(loss, (dx, dw, db2))
        ref, rl = ops.linear_cross_entropy(x.cuda(), dw[:10], t2.cuda(), bias=db2[:10])
        assert torch.allclose(lse, rl, rtol=1e-5) and abs(float(loss - ref)) < 1e-5
        assert not g[1][10:].any() and not g[2][10:].any() and all(z.isfinite().all() for z in g)
        # masked by the type's lowest value
        b3 = b.clone()
        b3[10:] = torch.finfo(dtype).min
        _, l3 = ops.linear_cross_entropy(x.cuda(), w.cuda(), t2.cuda(), bias=b3.cuda())
        assert torch.allclose(l3, rl, rtol=1e-5)
        # everything masked: the log of nothing
        _, l4 = ops.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), bias=torch.full_like(b, -float('inf')).cuda())
        assert bool((l4 == -float('inf')).all())
        # ignored rows that hold NaN or infinities touch no other row's loss and no gradient of the others
        t5 = t.clone()
        t5[[3, 40]] = -100
        x5 = x.clone()
        x5[3], x5[40] = float('nan'), float('inf')
        clean = ops.linear_cross_entropy(dx, dw, t5.cuda(), bias=db)
        want = torch.autograd.grad(clean[0], (dx, dw, db))
        d5 = x5.cuda().requires_grad_(True)
        loss, lse = ops.linear_cross_entropy(d5, dw, t5.cuda(), bias=db)
        assert float(loss) == float(clean[0])
        got = torch.autograd.grad(loss, (d5, dw, db))
        assert all(torch.equal(a, b_) for a, b_ in zip(got, want))


def test_targets_out_of_range(gpu):
    from paccmann_generator_amd import _ffi, ops
    x, w, _, t, _ = _data(20, 30, 16, torch.float32)
    bad = t.clone()
    bad[4] = 30
    with pytest.raises(_ffi.PmgError):
        ops.linear_cross_entropy(x.cuda(), w.cuda(), bad.cuda())
    bad[5] = -7
    loss, lse = ops.linear_cross_entropy(x.cuda(), w.cuda(), bad.cuda(), reduction='none', trusted_tokens=True)
    assert loss[[4, 5]].isnan().all() and loss.isnan().sum() == 2 and lse.isfinite().all()


def test_large_logits_do_not_overflow(gpu):
    for dtype in TYPES:
        x, w, b, t, _ = _data(70, 200, 64, dtype, seed=8)
        x = x * 60
        _check(x, w, None, t, None)
        x[:, :] = 0
        _check(x, w, None, t, None)


def test_gradients_against_differences(gpu):
    """A central difference of the loss in fp32 along random directions: 2 h slope, an error of h^2 times the third
    derivative (below 1 here) and the losses' rounding over 2 h."""
    from paccmann_generator_amd import ops
    x, w, b, t, r = (z.cuda() for z in _data(30, 50, 24, torch.float32, seed=4, bias=True, weighted=True))
    for z in (x, w, b):
        z.requires_grad_(True)
    call = lambda x, w, b: ops.linear_cross_entropy(x, w, t, bias=b, row_weight=r, logit_scale=0.9)[0]      # noqa: E731
    grads = torch.autograd.grad(call(x, w, b), (x, w, b))
    for k in range(3):
        d = torch.randn(grads[k].shape, device='cuda')
        d /= d.norm()
        h = 2e-2
        args = [z.detach() for z in (x, w, b)]
        hi, lo = list(args), list(args)
        hi[k], lo[k] = args[k] + h * d, args[k] - h * d
        diff = float(call(*hi).double() - call(*lo).double()) / (2 * h)
        assert abs(diff - float((grads[k] * d).sum())) < h * h + 50 * U / h


def test_repeats_and_replays(gpu):
    from paccmann_generator_amd import ops
    for dtype, (N, V, H) in ((torch.float32, (90, 60, 64)), (torch.bfloat16, (300, 3000, 128)), (torch.bfloat16, (3, 900, 64))):
        x, w, b, t, r = (z.cuda() for z in _data(N, V, H, dtype, seed=7, bias=True, weighted=True, ignored=0.2))

        def both():
            loss, lse, count = torch.ops.pmg.linear_cross_entropy(x, w, b, t, r, -100, 1.0, 2)
            return (loss, lse, *torch.ops.pmg.linear_cross_entropy_bwd(torch.ones_like(loss), None, x, w, b, t, r, lse, count,
                                                                      -100, 1.0, 2, [True] * 3))

        eager = both()
        assert all(torch.equal(a, c) for a, c in zip(eager, both()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = both()
        for k in range(3):
            x.normal_()
            t.copy_(torch.randint(0, V, (N,)))
            t[k] = -100
            graph.replay()
            torch.cuda.synchronize()
            now = [z.clone() for z in held]
            assert all(torch.equal(a, c) for a, c in zip(now, both()))


def test_partial_gradients_opcheck_and_empty(gpu):
    from paccmann_generator_amd import ops
    x, w, b, t, r = (z.cuda() for z in _data(20, 30, 16, torch.float32, bias=True, weighted=True))
    full = [z.clone().requires_grad_(True) for z in (x, w, b)]
    want = torch.autograd.grad(ops.linear_cross_entropy(full[0], full[1], t, bias=full[2], row_weight=r)[0], full)
    for k in range(3):
        z = [v.clone().requires_grad_(i == k) for i, v in enumerate((x, w, b))]
        got, = torch.autograd.grad(ops.linear_cross_entropy(z[0], z[1], t, bias=z[2], row_weight=r)[0], z[k])
        assert torch.equal(got, want[k])
    torch.library.opcheck(torch.ops.pmg.linear_cross_entropy, (full[0], full[1], full[2], t, r, -100, 1.0, 2))
    torch.library.opcheck(torch.ops.pmg.linear_cross_entropy, (full[0], full[1], None, t, None, -100, 0.5, 0))
    e = torch.zeros(0, 16, device='cuda', requires_grad=True)
    loss, lse = ops.linear_cross_entropy(e, full[1], torch.zeros(0, dtype=torch.long, device='cuda'))
    assert float(loss) == 0.0 and lse.shape == (0,)
    g = torch.autograd.grad(loss, (e, full[1]))
    assert g[0].shape == (0, 16) and not g[1].any()


def test_refusals(gpu):
    from paccmann_generator_amd import _ffi, ops
    x, w, b, t, r = (z.cuda() for z in _data(20, 30, 16, torch.float32, bias=True, weighted=True))
    bad = [(x[:, :15], w, t, {}), (x, w, t[:19], {}), (x.half(), w.half(), t, {}), (x.bfloat16(), w, t, {}), (x, w[0], t, {}),
           (x, w, t.float(), dict(trusted_tokens=True)), (x, w, t, dict(bias=b[:29])), (x, w, t, dict(bias=b.bfloat16())),
           (x, w, t, dict(row_weight=r[:19])), (x, w, t, dict(row_weight=r.double())), (x, w, t, dict(reduction='avg')),
           (x.cpu(), w, t, {}), (x, w, t.cpu(), dict(trusted_tokens=True)), (x, w[:0], t, dict(trusted_tokens=True))]
    for a, c, d, kw in bad:
        with pytest.raises(_ffi.PmgError):
            ops.linear_cross_entropy(a, c, d, **kw)


# Few vocabulary entries against the hidden size: training keeps the logits (16 V <= bytes of a hidden row)
KEPT = [(1, 1, 64), (70, 3, 48), (300, 60, 480), (2000, 17, 296), (33, 129, 1056), (20000, 61, 504), (65, 128, 1024)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,V,H', KEPT)
def test_logits_kept_for_the_backward(gpu, dtype, N, V, H):
    if 16 * V > H * dtype.itemsize:
        V = H * dtype.itemsize // 16
    _check(*_data(N, V, H, dtype, seed=N + V + H))
    z = torch.randn(N, generator=torch.Generator().manual_seed(1))
    z[N // 2] = 0.0
    _check(*_data(N, V, H, dtype, seed=N, bias=True, weighted=True, ignored=0.3), scale=0.7, reduction='none', lse_slope=z)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,V,H', [(524288, 603, 16), (50, 700, 32), (20, 5, 16)])
def test_kept_logits_give_the_gradients_of_formed_ones(gpu, dtype, N, V, H):
    """In pieces of the vocabulary, over listed rows: the slopes are those of logits formed again (equal products; the
    tiles' shapes may sum them in another order)."""
    x, w, b, t, r = _cuda(*_data(N, V, H, dtype, seed=4, bias=True, weighted=True, ignored=0.4))
    call = (x, w, b, t, r, -100, 0.8, 1)
    loss, lse, count = torch.ops.pmg.linear_cross_entropy(*call)
    l2, e2, c2, logits = torch.ops.pmg.linear_cross_entropy_keep(*call, True)
    assert torch.equal(loss, l2) and torch.equal(lse, e2) and torch.equal(count, c2) and logits.shape == (N, (V + 3) // 4 * 4)
    empty = torch.ops.pmg.linear_cross_entropy_keep(*call, False)[3]
    back = lambda k: torch.ops.pmg.linear_cross_entropy_bwd(torch.ones_like(loss), None, *call[:5], lse, count, *call[5:],   # noqa: E731
                                                            [True] * 3, k)
    want, same = back(None), back(empty)
    got = back(logits)
    size = (H + 16) * U * float((x.float().abs().amax(0) * w.float().abs().amax(0)).sum() + 2)
    for a, c, d, other in zip(got, want, same, (w, x, None)):
        assert torch.equal(c, d)
        # dl differs by its relative error at most (a logit's rounding, dl's own), in a sum of at most this many terms
        terms = {0: V, 1: N, None: N}[0 if other is w else 1 if other is x else None]
        most = (1.3 if terms == N else 1.0) * 0.8 * (float(other.float().abs().max()) if other is not None else 1.0)
        step = torch.finfo(dtype).eps / 2
        scale = most * (2.0 if terms == V else float(r.abs().sum()) * 2)
        assert bool(((a.float() - c.float()).abs() <= scale * (4 * size + 2 * step) + 2 * step * c.float().abs()).all())
    with pytest.raises(RuntimeError, match='logits must be'):
        back(logits[:, :-1] if V > 4 else logits[:-1])


@pytest.mark.parametrize('V', [40, 300])
def test_offsets_beyond_32_bits(gpu, V):
    """Hidden rows of 4.9 GB; the rows with a slope lie at both ends."""
    from paccmann_generator_amd import ops
    N, H = 1200000, 1024
    g = torch.Generator(device='cuda').manual_seed(5)
    x = torch.randn(N, H, device='cuda', generator=g).requires_grad_(True)
    w = (torch.randn(V, H, device='cuda', generator=g) / 16).requires_grad_(True)
    t = torch.randint(0, V, (N,), device='cuda', generator=g)
    rows = torch.cat([torch.arange(0, 300, 3), torch.arange(N - 200, N)])
    r = torch.zeros(N, device='cuda')
    r[rows.cuda()] = torch.rand(len(rows), device='cuda', generator=g) + 0.5
    loss, lse = ops.linear_cross_entropy(x, w, t, row_weight=r, reduction='sum')
    dx, dw = torch.autograd.grad(loss, (x, w))
    part = x.detach()[rows.cuda()].cpu(), w.detach().cpu(), t[rows.cuda()].cpu(), None, r[rows.cuda()].cpu()
    e = lm.linear_ce(*part, 1.0, 'sum', -100)
    tol = (H + 16) * U * e['size'] + 8 * U
    assert bool(((lse.detach()[rows.cuda()].cpu().double() - e['lse']).abs() <= tol + 2 * U * e['lse'].abs()).all())
    grads = lm.linear_ce_grads(*part, 1.0, 'sum', -100, torch.tensor(1.0), None)
    rel = 4 * float(tol.max()) + 16 * U
    for got, name, length in ((dx[rows.cuda()], 'x', V), (dw, 'w', len(rows))):
        bound = grads['|' + name + '|'] * (rel + (length + 8) * U) + grads[name].abs() * U * 1.01
        assert bool(((got.cpu().double() - grads[name]).abs() <= bound).all()), name
    dx[rows.cuda()] = 0.0
    assert not bool(dx.any())


def test_gradients_are_not_differentiated_again(gpu):
    from paccmann_generator_amd import ops
    x, w, b, t, _ = _cuda(*_data(20, 30, 16, torch.float32, seed=1, bias=True))
    z = [v.requires_grad_(True) for v in (x, w, b)]
    want = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b)[0], z)
    got = torch.autograd.grad(ops.linear_cross_entropy(x, w, t, bias=b)[0], z, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    for p in got:
        with pytest.raises(RuntimeError, match='not differentiable'):
            torch.autograd.grad(p.sum(), z, allow_unused=True, retain_graph=True)


# Few tiles and a long hidden size: the products are split over it
LONG = [(1, 3, 2000), (16, 100, 4096), (17, 300, 1032), (64, 1030, 2048), (300, 300, 2001), (5, 12000, 1032), (700, 60, 1024)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,V,H', LONG)
def test_hidden_size_split(gpu, dtype, N, V, H):
    _check(*_data(N, V, H, dtype, seed=N + V + H))
    _check(*_data(N, V, H, dtype, seed=N, bias=True, weighted=True, ignored=0.3), scale=0.7, reduction='none')


def test_masked_rows_of_a_split_hidden_size(gpu):
    """Masked entries, rows without any entry, and rows with NaN that stay apart."""
    from paccmann_generator_amd import ops
    N, V, H = 20, 90, 2048
    x, w, b, t, _ = _data(N, V, H, torch.float32, seed=6, bias=True)
    t = t % 40
    b[40:] = -float('inf')
    with torch.no_grad():
        _, lse = ops.linear_cross_entropy(*_cuda(x, w, t), bias=b.cuda())
        _, want = ops.linear_cross_entropy(*_cuda(x, w[:40], t), bias=b[:40].cuda())
        assert torch.allclose(lse, want, rtol=1e-6, atol=0)
        _, lse = ops.linear_cross_entropy(*_cuda(x, w, t), bias=torch.full((V,), torch.finfo(torch.float32).min).cuda())
        assert bool((lse <= torch.finfo(torch.float32).min * 0.99).all())
        _, lse = ops.linear_cross_entropy(*_cuda(x, w, t), bias=torch.full((V,), -float('inf')).cuda())
        assert bool((lse == -float('inf')).all())
        x[3] = float('nan')
        loss, lse = ops.linear_cross_entropy(*_cuda(x, w, t), bias=b.cuda(), reduction='none')
        rest = torch.arange(N) != 3
        assert bool(lse[3].isnan()) and bool(loss[3].isnan()) and torch.equal(lse.cpu()[rest].isnan(), torch.zeros(N - 1, dtype=torch.bool))
        assert torch.allclose(lse.cpu()[rest], want.cpu()[rest], rtol=1e-6, atol=0)
    # ignored, the row with NaN leaves every gradient alone
    t[3] = -100
    z = [v.requires_grad_(True) for v in _cuda(x, w, b)]
    got = torch.autograd.grad(ops.linear_cross_entropy(z[0], z[1], t.cuda(), bias=z[2])[0], z)
    assert not any(bool(g.isnan().any()) for g in got) and not got[0][3].any()
