"""pmg::linear_cross_entropy at the ends of what its arguments allow: infinite logits."""
import math

import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16]


def _data(N, V, H, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, H, generator=g).to(dtype)
    w = (torch.randn(V, H, generator=g) * 2 / math.sqrt(H)).to(dtype)
    return x, w, (torch.randn(V, generator=g) * 0.3).to(dtype), torch.randint(0, V, (N,), generator=g)


# one wave's tile, several waves and tiles, few tokens over many words, a hidden size that is split, kept logits
SIZES = [(20, 30, 16), (300, 700, 64), (5, 5000, 96), (20, 90, 2048), (3000, 60, 512)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('N,V,H', SIZES)
def test_infinite_logits(gpu, dtype, N, V, H):
    """lse is +inf where a logit is, NaN where one is NaN, and untouched in the other rows; the loss follows from it."""
    from paccmann_generator_amd import ops
    x, w, b, t = _data(N, V, H, dtype, seed=N)
    x[:, 0] = 0
    w[:, 0] = 0
    up = [7, V - 2 if V % 3 == 1 else V - 1]        # no multiples of 3: those are masked out below
    w[up, 0] = 16.0
    hot, nan = [3, N - 2], 4
    x[hot, 0] = 3e38                    # 16 x 3e38 leaves fp32 in the columns `up`, and no other
    x[nan, 0], x[nan, 1] = 3e38, float('nan')
    t[3], t[N - 2] = 7, 5
    rest = torch.ones(N, dtype=torch.bool)
    rest[hot + [nan]] = False
    for bias in (b, b.masked_fill(torch.arange(V) % 3 == 0, -float('inf'))):      # and with others masked out
        t = torch.where(t % 3 == 0, (t + 1) % V, t) if bias is not b else t
        t = torch.where(t % 3 == 0, torch.ones_like(t), t) if bias is not b else t
        e = lm.linear_ce(x[rest], w, t[rest], bias, None, 1.0, 'none', -100)
        size = lm.linear_ce(x[rest], w, t[rest], b, None, 1.0, 'none', -100)['size']
        tol = (H + 16) * U * size + 8 * U
        for train in (False, True):
            z = [v.cuda().requires_grad_(train) for v in (x, w, bias)]
            loss, lse = ops.linear_cross_entropy(z[0], z[1], t.cuda(), bias=z[2], reduction='none')
            lse, loss = lse.detach().cpu(), loss.detach().cpu()
            assert bool((lse[hot] == float('inf')).all()) and bool(lse[nan].isnan())
            for n in hot:                       # inf - inf, or inf - finite
                assert bool(loss[n].isnan()) if int(t[n]) in up else float(loss[n]) == float('inf')
            assert bool(((lse[rest].double() - e['lse']).abs() <= tol + 2 * U * e['lse'].abs()).all())
            assert bool(((loss[rest].double() - e['loss']).abs() <= 2 * tol + 4 * U * (e['lse'].abs() + e['loss'].abs())).all())
    # a bias of +inf is in every row
    b2 = b.clone()
    b2[V // 2] = float('inf')
    _, lse = ops.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), bias=b2.cuda())
    keep = torch.arange(N) != nan
    assert bool((lse.cpu()[keep] == float('inf')).all()) and bool(lse[nan].isnan())
    b2[V // 3] = float('nan')
    assert bool(ops.linear_cross_entropy(x.cuda(), w.cuda(), t.cuda(), bias=b2.cuda())[1].isnan().all())
    # ignored, such rows leave the loss and the gradients alone
    t[hot + [nan]] = -100
    z = [v.cuda().requires_grad_(True) for v in (x, w, b)]
    loss, _ = ops.linear_cross_entropy(z[0], z[1], t.cuda(), bias=z[2])
    g = torch.autograd.grad(loss, z)
    assert bool(loss.isfinite()) and all(bool(v.isfinite().all()) for v in g) and not g[0][hot + [nan]].any()


def _in_64_bits(x, w, b, t, step):
    """(lse, logit of the target, largest sum of magnitudes) of every row, a block of rows at a time, on the GPU."""
    out = []
    wd, bd = w.double(), b.double()
    for n in range(0, len(x), step):
        xd = x[n:n + step].double()
        logits = torch.mm(xd, wd.t().contiguous()).add_(bd)
        size = xd.abs().sum(1) * wd.abs().max() + bd.abs().max()
        out.append((logits.logsumexp(1), logits.gather(1, t[n:n + step].clamp(min=0).unsqueeze(1)).squeeze(1), size))
    return [torch.cat(c) for c in zip(*out)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_tokens_in_blocks(gpu, dtype):
    """More statistics of tiles than the scratch holds at a time: the last block is shorter, rows and sums run through."""
    from paccmann_generator_amd import ops
    N, V, H = 70001, 128000, 16
    x, w, b, t = _data(N, V, H, dtype, seed=1)
    t[torch.rand(N, generator=torch.Generator().manual_seed(2)) < 0.3] = -100
    r = torch.rand(N, generator=torch.Generator().manual_seed(3)) - 0.3
    x, w, b, t, r = (v.cuda() for v in (x, w, b, t, r))
    lse, hit, size = _in_64_bits(x, w, b, t, 8192)
    used = t != -100
    tol = (H + 16) * U * size + 8 * U
    nll = torch.where(used, (lse - hit) * r, torch.zeros_like(lse))
    off = (2 * tol + 4 * U * lse.abs()) * r.abs() * used
    for ids in (t, t.int()):
        got, l = ops.linear_cross_entropy(x, w, ids, bias=b, row_weight=r, reduction='none')
        assert bool(((l.double() - lse).abs() <= tol + 2 * U * lse.abs()).all())
        assert bool(((got.double() - nll).abs() <= off + 2 * U * nll.abs()).all())
        total, l2 = ops.linear_cross_entropy(x, w, ids, bias=b, row_weight=r, reduction='sum')
        mean, l3 = ops.linear_cross_entropy(x, w, ids, bias=b, row_weight=r, reduction='mean')
        assert torch.equal(l, l2) and torch.equal(l, l3)
        assert abs(float(total) - float(nll.sum())) <= float(off.sum()) + 2 * U * abs(float(nll.sum()))
        # the same sum, divided: rounded once more each
        assert abs(float(mean) - float(total) / int(used.sum())) <= 2 * U * abs(float(mean))


def test_tokens_in_blocks_with_kept_logits(gpu):
    """Few words, so that a block is 33.5 million tokens; training keeps the logits of both blocks."""
    from paccmann_generator_amd import ops
    N, V, H = (1 << 25) + 5003, 2, 8
    g = torch.Generator(device='cuda').manual_seed(4)
    x = torch.randn(N, H, device='cuda', generator=g)
    w, b = torch.randn(V, H, device='cuda', generator=g), torch.randn(V, device='cuda', generator=g)
    t = torch.randint(0, V, (N,), device='cuda', generator=g)
    x.requires_grad_(True)
    loss, lse = ops.linear_cross_entropy(x, w, t, bias=b, trusted_tokens=True)
    dx, = torch.autograd.grad(loss, x)
    xd = x.detach()
    want, hit, size = _in_64_bits(xd, w, b, t, 1 << 24)
    tol = (H + 16) * U * size + 8 * U
    assert bool(((lse.double() - want).abs() <= tol + 2 * U * want.abs()).all())
    nll = want - hit
    assert abs(float(loss) - float(nll.mean())) <= float((2 * tol + 4 * U * want.abs()).mean()) + 2 * U * float(nll.mean())
    # dx = (p - onehot) W / N: the exponential's error, relative; a product, two sums and a factor
    rel = 4 * float(tol.max()) + 32 * U
    wd = w.double()
    for n in range(0, N, 1 << 24):
        p = (torch.mm(xd[n:n + (1 << 24)].double(), wd.t().contiguous()) + b.double() - want[n:n + (1 << 24)].unsqueeze(1)).exp()
        one = torch.nn.functional.one_hot(t[n:n + (1 << 24)], V)
        exact, most = torch.mm(p - one, wd) / N, torch.mm(p + one, wd.abs()) / N
        assert bool(((dx[n:n + (1 << 24)].double() - exact).abs() <= most * rel).all())


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('weight', [1e-38, 1e-30, 1e-12, 1e12, 1e30])
def test_losses_of_any_weight_beside_the_log_sum_exp(gpu, dtype, weight):
    """weight * loss + sum(z lse): the gradients are sums of both, whichever is the smaller by far.  Ignored rows have the
    slope of the log-sum-exp alone."""
    from paccmann_generator_amd import ops
    N, V, H = 40, 90, 48
    x, w, b, t = _data(N, V, H, dtype, seed=5)
    t[:10] = -100
    z = torch.randn(N, generator=torch.Generator().manual_seed(6))
    for reduction in ('mean', 'sum'):
        leaves = [v.cuda().requires_grad_(True) for v in (x, w, b)]
        loss, lse = ops.linear_cross_entropy(leaves[0], leaves[1], t.cuda(), bias=leaves[2], reduction=reduction)
        got = torch.autograd.grad((loss, lse), leaves, (torch.tensor(weight, device='cuda'), z.cuda()))
        grads = lm.linear_ce_grads(x, w, t, b, None, 1.0, reduction, -100, torch.tensor(weight, dtype=torch.float64), z)
        size = lm.linear_ce(x, w, t, b)['size']
        f = torch.finfo(dtype)
        rel = 4 * ((H + 16) * U * float(size.max()) + 8 * U) + 16 * U + (0 if dtype == torch.float32 else f.eps / 2)
        for name, length, g in zip('xwb', (V, N, N), got):
            exact, mag = grads[name], grads['|' + name + '|']
            bound = mag * (rel + (length + 8) * U) + exact.abs() * f.eps / 2 * 1.01
            assert bool(((g.cpu().double() - exact).abs() <= bound + 1e-30).all()), (name, reduction)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_kept_logits_over_pieces_of_the_vocabulary(gpu, dtype):
    """Gradients from kept logits and from logits formed again, three pieces of the vocabulary, against 64 bits: every
    element within its own sum of magnitudes.  Hidden states and rewards are positive and targets are a few words, so that
    the sums of the others do not cancel: a gradient of zeros, or one with its pieces in another order, is far outside."""
    import paccmann_generator_amd  # noqa: F401  (registers the operators)
    N, V, H = 524288, 603, 16
    x, w, b, _ = _data(N, V, H, dtype, seed=7)
    x = x.abs()
    g = torch.Generator().manual_seed(8)
    t, r = torch.randint(0, 37, (N,), generator=g) * 16 + 5, torch.rand(N, generator=g) + 0.1
    t[torch.rand(N, generator=g) < 0.4] = -100
    x, w, b, t, r = (v.cuda() for v in (x, w, b, t, r))
    call = (x, w, b, t, r, -100, 0.8, 1)
    loss, lse, count, logits = torch.ops.pmg.linear_cross_entropy_keep(*call, True)
    runs = [torch.ops.pmg.linear_cross_entropy_bwd(torch.ones_like(loss), None, *call[:5], lse, count, *call[5:], [True] * 3, k)
            for k in (logits, None)]
    size = lm.linear_ce(x, w, t, b, r, 0.8, 'sum')['size']
    grads = lm.linear_ce_grads(x, w, t, b, r, 0.8, 'sum', -100, torch.tensor(1.0).cuda(), None)
    f = torch.finfo(dtype)
    rel = 4 * ((H + 16) * U * float(size.max()) + 8 * U) + 16 * U + (0 if dtype == torch.float32 else f.eps / 2)
    for k, (name, length) in enumerate((('x', V), ('w', N), ('b', N))):
        exact, mag = grads[name], grads['|' + name + '|']
        bound = mag * (rel + (length + 8) * U) + exact.abs() * f.eps / 2 * 1.01
        for got in runs:
            assert bool(((got[k].double() - exact).abs() <= bound).all()), name
        if name == 'x':          # rows without a slope are zeros; in the others nearly all elements stand out
            assert float((exact.abs() > bound)[t != -100].double().mean()) > 0.9
        else:
            stands, targets = exact.abs() > 2 * bound, torch.unique(t[t != -100])
            assert float(stands.double().mean()) > 0.95, name
            stands[targets] = True
            assert bool(stands.all()), name
            turned = exact.roll(256, 0)
            assert float(((turned - exact).abs() > 2 * bound).double().mean()) > 0.5, name
