"""pmg::grad_norm, pmg::clip_grad_norm_ and pmg::adamw_step_: against the 64-bit formulas within the roundings of
their arithmetic, and, for a state held in 8 bits, code by code against the same formulas evaluated in fp32."""
import math

import pytest
import torch

from oracle import lm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [(3, 70), (1,), (255,), (256,), (257,), (0,), (4096,), (4097,), (33, 129), (5, 7, 11), (70001,), (2, 0, 3)]
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.98, eps=1e-8, wd=0.03)


def _make(shapes, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * std).to(dtype) for s in shapes]


@pytest.mark.parametrize('dtypes', [(torch.float32,), (torch.bfloat16,), (torch.float16,),
                                    (torch.float32, torch.bfloat16, torch.float16)], ids=str)
def test_norm_and_clipping(gpu, dtypes):
    from paccmann_generator_amd import ops
    grads = [x.to(dtypes[i % len(dtypes)]) for i, x in enumerate(_make(SHAPES * 20, 1))]      # over one launch's table
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    dev = [g.cuda() for g in grads]
    norm = ops.grad_norm(dev)
    # fp64 sums, one rounding of the result
    assert norm.shape == () and abs(float(norm) - exact) <= 1.001 * U * exact + 1e-12 * exact
    for max_norm in (1e9, 3.0):
        again = [g.clone() for g in dev]
        got = ops.clip_grad_norm_(again, max_norm)
        assert float(got) == float(norm)
        c = lm.clip_factor(exact, max_norm)
        for a, g in zip(again, grads):
            if c == 1.0:
                assert torch.equal(a.cpu(), g)
                continue
            want, f = g.double() * c, torch.finfo(g.dtype)
            # the norm and the factor rounded to fp32, the product, the store
            bound = want.abs() * (4 * U + f.eps / 2) + f.tiny * f.eps
            assert bool(((a.cpu().double() - want).abs() <= bound).all())


def test_norm_range_and_special_values(gpu):
    from paccmann_generator_amd import ops
    for v in (1e-30, 1e30):        # squares leave fp32
        x = torch.full((1000,), v, device='cuda')
        assert abs(float(ops.grad_norm([x])) / (v * math.sqrt(1000)) - 1) < 1e-6
    x = torch.ones(5000, device='cuda')
    for bad, is_bad in ((float('inf'), torch.isinf), (float('nan'), torch.isnan)):
        y = x.clone()
        y[4321] = bad
        assert bool(is_bad(ops.grad_norm([x, y])))
    y = x.clone()
    y[3] = float('nan')
    ops.clip_grad_norm_([x, y], 1.0)
    assert bool(x.isnan().all())                         # as a NaN norm does in the reference's clipping
    z = torch.zeros(10, device='cuda')
    assert float(ops.clip_grad_norm_([z], 1.0)) == 0.0 and not z.any()
    assert float(ops.grad_norm([torch.zeros(0, device='cuda')])) == 0.0


def test_norm_of_strided_and_misaligned_gradients(gpu):
    from paccmann_generator_amd import ops
    base = torch.randn(9000, device='cuda')
    wide = torch.randn(40, 60, device='cuda')
    grads = [base[1:2000], base[2003:4096], wide.t(), wide[:, ::2], wide[:1, :1].expand(30, 30)]
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(float(ops.grad_norm(grads)) - exact) <= 2 * U * exact
    clip = [base[1:2000], base[2003:4096], wide.t()]
    want = [g.double() for g in clip]
    n = float(ops.clip_grad_norm_(clip, 2.0))
    for a, w in zip(clip, want):
        w = w * lm.clip_factor(n, 2.0)
        assert bool(((a.double() - w).abs() <= 3 * U * w.abs()).all())


def _state(params, bits, seed):
    m, v = _make([p.shape for p in params], seed, 0.1), [x.square() + 1e-4 for x in _make([p.shape for p in params], seed + 1, 0.3)]
    if bits == 32:
        return m, v, None, None
    cm, cv = [lm.state_codes(x, True) for x in m], [lm.state_codes(x, False) for x in v]
    return [c for c, _ in cm], [c for c, _ in cv], [t for _, t in cm], [t for _, t in cv]


@pytest.mark.parametrize('decoupled', [True, False])
@pytest.mark.parametrize('clip', [False, True])
@pytest.mark.parametrize('dtype,grad_dtype,with_master', [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, True),
    (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True), (torch.float16, torch.float32, False)],
    ids=str)
@pytest.mark.parametrize('bits', [32, 8])
def test_update_against_the_formulas(gpu, bits, dtype, grad_dtype, with_master, clip, decoupled):
    from paccmann_generator_amd import ops
    h = HYPER
    shapes = SHAPES + [(40,)] * 70                       # over one launch's table
    params = _make(shapes, 3, 0.5, dtype)
    grads = _make(shapes, 4, 0.2, grad_dtype)
    master = [p.float() + 1e-4 * x for p, x in zip(params, _make(shapes, 5))] if with_master else None
    m, v, mt, vt = _state(params, bits, 6)
    cuda = lambda xs: [x.cuda() for x in xs] if xs is not None else None      # noqa: E731
    dp, dg, dm, dv, dmt, dvt, dw = (cuda(x) for x in (params, grads, m, v, mt, vt, master))
    step = torch.full((1,), 6, dtype=torch.int64, device='cuda')
    norm = ops.grad_norm(dg) if clip else None
    ops.adamw_step(dp, dg, dm, dv, step, lr=h['lr'], betas=(h['beta1'], h['beta2']), eps=h['eps'], weight_decay=h['wd'],
                   decoupled=decoupled, exp_avg_top=dmt, exp_avg_sq_top=dvt, master=dw, grad_norm=norm,
                   max_norm=0.7 if clip else 0.0)
    assert int(step) == 7
    factor = lm.clip_factor(norm, 0.7) if clip else 1.0
    for i, p in enumerate(params):
        assert torch.equal(dg[i].cpu(), grads[i])        # the gradients stay as they are
        p0 = master[i] if with_master else p.float()
        m0 = m[i] if bits == 32 else lm.state_values(m[i], mt[i])
        v0 = v[i] if bits == 32 else lm.state_values(v[i], vt[i])
        args = (7, h['lr'], h['beta1'], h['beta2'], h['eps'], h['wd'], decoupled, factor)
        # fp32, operation by operation: the same bits, so the same codes
        p32, m32, v32 = lm.adamw(p0, grads[i].float(), m0, v0, *args)
        same = lambda a, b: int((a.cpu() != b).sum()) == 0       # noqa: E731
        assert same(dp[i], p32.to(dtype))
        if with_master:
            assert same(dw[i], p32)
        if bits == 32:
            assert same(dm[i], m32) and same(dv[i], v32)
        else:
            (cm, tm), (cv, tv) = lm.state_codes(m32, True), lm.state_codes(v32, False)
            assert torch.equal(dm[i].cpu(), cm) and torch.equal(dmt[i].cpu(), tm)
            assert torch.equal(dv[i].cpu(), cv) and torch.equal(dvt[i].cpu(), tv)
            assert torch.equal(ops.adamw_state_values(dm[i], dmt[i]).cpu(), lm.state_values(cm, tm))
            assert torch.equal(ops.adamw_state_values(dv[i], dvt[i]).cpu(), lm.state_values(cv, tv))
        # fp64: m is two products and a sum of a gradient with up to three roundings; p - keep p is one product
        # and one difference of a quotient with up to nine
        pe, me, ve = lm.adamw(p0.double(), grads[i].double(), m0.double(), v0.double(), *args)
        G = grads[i].double().abs() * factor + (0 if decoupled else h['wd'] * p0.double().abs())
        dm_ = 6 * U * (h['beta1'] * m0.double().abs() + (1 - h['beta1']) * G)
        if bits == 32:
            assert bool(((dm[i].cpu().double() - me).abs() <= dm_).all())
            assert bool(((dv[i].cpu().double() - ve).abs() <= 8 * U * (h['beta2'] * v0.double() + (1 - h['beta2']) * G * G)).all())
        den = ve.sqrt() / math.sqrt(1 - h['beta2'] ** 7) + h['eps']
        slope = h['lr'] / (1 - h['beta1'] ** 7) / den
        rel_v = 8 * U * (h['beta2'] * v0.double() + (1 - h['beta2']) * G * G) / ve.clamp(min=1e-30)
        bound = slope * (dm_ + me.abs() * (9 * U + rel_v)) + 3 * U * p0.double().abs()
        f = torch.finfo(dtype)
        store = 0 if dtype == torch.float32 else pe.abs() * f.eps / 2 * 1.01 + f.tiny * f.eps
        assert bool(((dp[i].cpu().double() - pe).abs() <= bound * 1.01 + store).all())


def test_misaligned_and_permuted_tensors(gpu):
    """Gradients cut from one flat buffer at any offset (as the data-parallel step leaves them), parameters in another
    memory order, gradients in another order than their parameters."""
    from paccmann_generator_amd import ops
    h = HYPER
    for bits in (32, 8):
        flat = torch.randn(20001, device='cuda')
        p = [torch.randn(3, 70, device='cuda'), torch.randn(60, 50, device='cuda').t(),
             torch.randn(8001, device='cuda')[1:], torch.randn(4, 6, 5, device='cuda').permute(2, 0, 1)]
        g = [flat[1:211].view(3, 70), flat[211:3211].view(50, 60), flat[3211:11211], flat[11213:11333].view(5, 4, 6)]
        state = [ops.adamw_state(x, bits) for x in p]
        ref = [(x.cpu().clone(), torch.zeros(x.shape), torch.zeros(x.shape)) for x in p]
        step = torch.zeros(1, dtype=torch.int64, device='cuda')
        for t in (1, 2):
            ops.adamw_step(p, g, [s[0] for s in state], [s[1] for s in state], step, lr=h['lr'],
                           betas=(h['beta1'], h['beta2']), weight_decay=h['wd'],
                           exp_avg_top=[s[2] for s in state] if bits == 8 else None,
                           exp_avg_sq_top=[s[3] for s in state] if bits == 8 else None)
            for i in range(len(p)):
                rp, rm, rv = lm.adamw(*ref[i][:1], g[i].cpu(), *ref[i][1:], t, h['lr'], h['beta1'], h['beta2'], 1e-8,
                                      h['wd'], True)
                assert torch.equal(p[i].cpu(), rp)
                if bits == 8:       # blocks follow the memory order
                    order = sorted(range(p[i].dim()), key=lambda d: -p[i].stride(d))
                    back = [order.index(d) for d in range(p[i].dim())]
                    rm, rv = (lm.state_values(*lm.state_codes(x.permute(order).contiguous(), s)).permute(back)
                              for x, s in ((rm, True), (rv, False)))
                ref[i] = (rp, rm, rv)


def test_state_of_special_blocks(gpu):
    """Zeros, magnitudes below the normal numbers, one value far above the others, infinities and NaN."""
    from paccmann_generator_amd import ops
    n = 256 * 6 + 10
    g = torch.zeros(n)
    g[256:512] = 1e-30                       # squares vanish, first moments are held
    g[512:768] = 1e-3 * torch.randn(256)
    g[600] = 1e4
    g[800] = float('inf')
    g[1100] = float('nan')
    g[1300:] = torch.randn(n - 1300)
    p = torch.zeros(n, device='cuda')
    m, v, mt, vt = ops.adamw_state(p, 8)
    step = torch.zeros(1, dtype=torch.int64, device='cuda')
    ops.adamw_step([p], [g.cuda()], [m], [v], step, exp_avg_top=[mt], exp_avg_sq_top=[vt])
    rp, rm, rv = lm.adamw(torch.zeros(n), g, torch.zeros(n), torch.zeros(n), 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, True)
    (cm, tm), (cv, tv) = lm.state_codes(rm, True), lm.state_codes(rv, False)
    assert torch.equal(m.cpu(), cm) and torch.equal(v.cpu(), cv)
    assert torch.equal(mt.cpu(), tm, ) or torch.equal(mt.cpu().nan_to_num(7.0), tm.nan_to_num(7.0))
    assert torch.equal(vt.cpu().nan_to_num(7.0), tv.nan_to_num(7.0))
    assert torch.equal(p.cpu().nan_to_num(7.0), rp.nan_to_num(7.0))
    vals = ops.adamw_state_values(v, vt).cpu()
    assert not vals[:512].any() and bool((vals[512:768] > 0).all())       # a positive square keeps a positive value
    assert not vals[768:1280].isfinite().any() and bool((vals[1300:] > 0).all())


def test_state_codes_cover_their_range(gpu):
    from paccmann_generator_amd import ops
    code = torch.arange(-127, 128, dtype=torch.int8)
    got = ops.adamw_state_values(code.cuda(), torch.tensor([2.0], device='cuda')).cpu().double()
    c = torch.arange(-127, 128).double() / 127
    assert bool(((got - 2 * c * c.abs()).abs() <= 5 * U * 2 * c * c).all())
    code = torch.arange(0, 256, dtype=torch.uint8)
    got = ops.adamw_state_values(code.cuda(), torch.tensor([3.0], device='cuda')).cpu().double()
    assert bool(((got - 3 * (torch.arange(256).double() / 255) ** 4).abs() <= 8 * U * 3).all())
    # values survive a round trip through their codes
    m, top = lm.state_codes(ops.adamw_state_values(torch.arange(-127, 128, dtype=torch.int8).cuda(),
                                                   torch.tensor([2.0], device='cuda')).cpu(), True)
    assert torch.equal(m, torch.arange(-127, 128, dtype=torch.int8)) and float(top) == 2.0


def test_captured_update_counts_on(gpu):
    """Norm, update and step counter in one graph: every replay equals the eager update, also with another learning
    rate in its tensor."""
    from paccmann_generator_amd import ops
    shapes = [(300, 40), (257,), (5000,)]
    for bits in (32, 8):
        def fresh():
            p = [x.cuda() for x in _make(shapes, 1)]
            s = [ops.adamw_state(x, bits) for x in p]
            return dict(p=p, s=s, step=torch.zeros(1, dtype=torch.int64, device='cuda'),
                        lr=torch.tensor([1e-3], device='cuda'))

        g = [x.cuda() for x in _make(shapes, 2)]

        def update(a):
            norm = ops.grad_norm(g)
            ops.adamw_step(a['p'], g, [s[0] for s in a['s']], [s[1] for s in a['s']], a['step'], weight_decay=0.1,
                           exp_avg_top=[s[2] for s in a['s']] if bits == 8 else None,
                           exp_avg_sq_top=[s[3] for s in a['s']] if bits == 8 else None, grad_norm=norm, max_norm=1.0,
                           lr_tensor=a['lr'])

        a, b = fresh(), fresh()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            update(b)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            update(b)
        assert int(b['step']) == 1
        update(a)
        for k in range(4):
            for x in g:
                x.normal_()
            for q in (a, b):
                q['lr'].fill_(1e-3 * (k + 1))
            graph.replay()
            update(a)
            torch.cuda.synchronize()
            assert int(a['step']) == int(b['step']) == k + 2
            assert all(torch.equal(x, y) for x, y in zip(a['p'], b['p']))
            assert all(torch.equal(x, y) for u, w in zip(a['s'], b['s']) for x, y in zip(u, w) if x is not None)


def test_versions_and_opcheck(gpu):
    from paccmann_generator_amd import ops
    p = torch.randn(40, device='cuda', requires_grad=True)
    out = (p * p).sum()
    m, v, _, _ = ops.adamw_state(p)
    step = torch.zeros(1, dtype=torch.int64, device='cuda')
    g = torch.randn(40, device='cuda')
    ops.adamw_step([p], [g], [m], [v], step)
    with pytest.raises(RuntimeError):            # autograd notices that a saved tensor was changed in place
        out.backward()
    utils = ('test_schema', 'test_faketensor')
    torch.library.opcheck(torch.ops.pmg.grad_norm, ([g, m],), test_utils=utils)
    torch.library.opcheck(torch.ops.pmg.clip_grad_norm_, ([g.clone(), m.clone()], 1.0), test_utils=utils)
    torch.library.opcheck(torch.ops.pmg.adamw_step_, ([p.detach().clone()], [g], [m], [v], [], [], [], step, None, None,
                                                     1e-3, 0.9, 0.99, 1e-8, 0.0, 0.0, True), test_utils=utils)


def test_device_side_refusals(gpu):
    from paccmann_generator_amd import _ffi, ops
    p, g = torch.randn(64, device='cuda'), torch.randn(64, device='cuda')
    m, v, _, _ = ops.adamw_state(p)
    step = torch.zeros(1, dtype=torch.int64, device='cuda')
    bad = [
        dict(params=[p, p], grads=[g, g], exp_avg=[m, m.clone()], exp_avg_sq=[v, v.clone()]),     # twice the same
        dict(params=[p[:40], p[30:]], grads=[g[:40], g[30:]], exp_avg=[m[:40].clone(), m[30:].clone()],
             exp_avg_sq=[v[:40].clone(), v[30:].clone()]),
        dict(params=[p], grads=[p], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[m]),
        dict(params=[p], grads=[g[:63]], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[p], grads=[g.half()], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[p], grads=[g], exp_avg=[m.double()], exp_avg_sq=[v]),
        dict(params=[p], grads=[g], exp_avg=[m[:32]], exp_avg_sq=[v]),
        dict(params=[p], grads=[g, g], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[torch.randn(128, device='cuda')[::2]], grads=[g], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], master=[p.clone()]),             # fp32 needs no copy
        dict(params=[p], grads=[g.cpu()], exp_avg=[m], exp_avg_sq=[v]),
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], grad_norm=torch.ones(1, device='cuda')),   # no max_norm
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], betas=(1.0, 0.9)),
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], lr=-1.0),
        dict(params=[p], grads=[g], exp_avg=[m], exp_avg_sq=[v], lr=float('nan')),
        dict(params=[p], grads=[g], exp_avg=[m.to(torch.int8)], exp_avg_sq=[v.to(torch.uint8)],
             exp_avg_top=[torch.ones(2, device='cuda')], exp_avg_sq_top=[torch.ones(1, device='cuda')]),
    ]
    before = p.clone()
    for kw in bad:
        with pytest.raises(_ffi.PmgError):
            ops.adamw_step(step=step, **kw)
    with pytest.raises(_ffi.PmgError):
        ops.adamw_step([p], [g], [m], [v], torch.zeros(1, device='cuda'))
    with pytest.raises(_ffi.PmgError):
        ops.clip_grad_norm_([g, g], 1.0)
    with pytest.raises(_ffi.PmgError):
        ops.clip_grad_norm_([g[:1].expand(5)], 1.0)
    with pytest.raises(_ffi.PmgError):
        ops.clip_grad_norm_([g], 0.0)
    torch.cuda.synchronize()
    assert int(step) == 0 and torch.equal(p, before)
