"""The training operators as they are used together: optim.AdamW against its formulas over several steps (missing
gradients, groups, types, checkpoints), a token model trained through embedding, cross entropy, clipping and update --
eager against a plain fp64 model, and captured in one graph -- and the learners with the fused update."""
import copy

import pytest
import torch
import torch.nn as nn

from oracle import lm
from tests import test_gpu_harness as H

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------- optimizer
def _params(seed=0, dtypes=(torch.float32,)):
    g = torch.Generator().manual_seed(seed)
    shapes = [(13, 7), (300,), (5, 4, 6), (1,)]
    return [torch.randn(s, generator=g).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


@pytest.mark.parametrize('decoupled', [True, False])
@pytest.mark.parametrize('bits', [32, 8])
def test_optimizer_follows_the_formulas(gpu, bits, decoupled):
    """Five steps, bit for bit; the third parameter has no gradient in steps 2 and 3 and keeps its count."""
    from paccmann_generator_amd import AdamW
    ref = [dict(p=p.clone(), m=torch.zeros_like(p), v=torch.zeros_like(p), t=0) for p in _params()]
    ps = [p.cuda().requires_grad_(True) for p in _params()]
    opt = AdamW([dict(params=ps[:2], lr=1e-2), dict(params=ps[2:], weight_decay=0.2, betas=(0.8, 0.95))], weight_decay=0.1,
                decoupled=decoupled, state_bits=bits)
    for k in range(5):
        for i, p in enumerate(ps):
            g = torch.randn(p.shape, generator=torch.Generator().manual_seed(10 * k + i))
            skip = i == 2 and k in (1, 2)
            p.grad = None if skip else g.cuda()
            if skip:
                continue
            r = ref[i]
            r['t'] += 1
            lr, betas, wd = (1e-2, (0.9, 0.999), 0.1) if i < 2 else (1e-3, (0.8, 0.95), 0.2)
            r['p'], r['m'], r['v'] = lm.adamw(r['p'], g, r['m'], r['v'], r['t'], lr, *betas, 1e-8, wd, decoupled)
            if bits == 8:
                r['m'], r['v'] = (lm.state_values(*lm.state_codes(r[x], x == 'm')) for x in 'mv')
        assert opt.step() is None
        for p, r in zip(ps, ref):
            assert torch.equal(p.detach().cpu(), r['p'])
    assert [int(opt.state[p]['step']) for p in ps] == [5, 5, 3, 5]


def test_optimizer_with_mixed_types_copies_and_clipping(gpu):
    from paccmann_generator_amd import AdamW
    dtypes = (torch.float32, torch.bfloat16, torch.float16, torch.bfloat16)
    for master in (False, True):
        ps = [p.cuda().requires_grad_(True) for p in _params(1, dtypes)]
        start = [p.detach().cpu().float() for p in ps]
        opt = AdamW(ps, lr=1e-2, master_weights=master, max_grad_norm=0.5)
        w, m, v = list(start), [torch.zeros_like(x) for x in start], [torch.zeros_like(x) for x in start]
        for t in (1, 2, 3):
            for i, p in enumerate(ps):
                p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(7 * t + i)).cuda().to(p.dtype)
            opt.step()
            factor = lm.clip_factor(opt.grad_norm, 0.5)
            assert factor < 1.0
            for i, p in enumerate(ps):
                w[i], m[i], v[i] = lm.adamw(w[i], p.grad.cpu().float(), m[i], v[i], t, 1e-2, 0.9, 0.999, 1e-8, 1e-2, True, factor)
                if not master:
                    w[i] = w[i].to(p.dtype).float()
                assert torch.equal(p.detach().cpu(), w[i].to(p.dtype))
                if master and p.dtype != torch.float32:
                    assert torch.equal(opt.state[p]['master'].cpu(), w[i])


def test_optimizer_checkpoints(gpu, tmp_path):
    from paccmann_generator_amd import AdamW, _ffi
    for bits in (32, 8):
        a = [p.cuda().requires_grad_(True) for p in _params(2, (torch.float32, torch.bfloat16))]
        opt = AdamW(a, state_bits=bits, master_weights=True)
        grads = [torch.randn_like(p) for p in a]
        for p, g in zip(a, grads):
            p.grad = g
        opt.step()
        torch.save(opt.state_dict(), tmp_path / 'o.pt')
        b = [p.detach().clone().requires_grad_(True) for p in a]
        again = AdamW(b, state_bits=bits, master_weights=True)
        again.load_state_dict(torch.load(tmp_path / 'o.pt', weights_only=True))
        for p, q, g in zip(a, b, grads):
            for k, x in opt.state[p].items():
                assert torch.equal(x, again.state[q][k]) and x.dtype == again.state[q][k].dtype
            q.grad = g
        assert len({id(again.state[q]['step']) for q in b}) == 1         # counters that agree are one again
        opt.step(), again.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    # 8 bits read back into 32; not the other way round
    wide = AdamW([p.detach().clone().requires_grad_(True) for p in a], state_bits=32)
    wide.load_state_dict(torch.load(tmp_path / 'o.pt', weights_only=True))
    for q in wide.param_groups[0]['params']:
        assert wide.state[q]['exp_avg'].dtype == torch.float32 and 'exp_avg_top' not in wide.state[q]
    with pytest.raises(_ffi.PmgError):
        again.load_state_dict(wide.state_dict())
    for kw in (dict(state_bits=4), dict(max_grad_norm=0.0)):
        with pytest.raises(_ffi.PmgError):
            AdamW(b, **kw)


# ------------------------------------------------------------------------------------ a model trained
class TokenModel(nn.Module):
    """Embedding, one hidden layer, projection; ``plain`` computes the same in torch (any type and device)."""

    def __init__(self, V, E, Hd):
        super().__init__()
        self.table = nn.Parameter(torch.randn(V, E))
        self.mid = nn.Linear(E, Hd)
        self.head = nn.Parameter(torch.randn(V, Hd) / Hd ** 0.5)
        self.bias = nn.Parameter(torch.zeros(V))

    def forward(self, tokens, targets, reward):
        from paccmann_generator_amd import ops
        x = torch.tanh(self.mid(ops.embedding(self.table, tokens, scale=0.5, padding_idx=0, trusted_tokens=True)))
        return ops.linear_cross_entropy(x, self.head, targets, bias=self.bias, row_weight=reward, ignore_index=0,
                                        logit_scale=0.8, trusted_tokens=True)[0]

    def plain(self, tokens, targets, reward):
        x = torch.tanh(self.mid(nn.functional.embedding(tokens, self.table, padding_idx=0) * 0.5))
        logp = torch.log_softmax((x @ self.head.t() + self.bias) * 0.8, -1)
        keep = targets != 0
        nll = -logp.gather(-1, targets.unsqueeze(-1)).squeeze(-1) * reward
        return (nll * keep).sum() / keep.sum()


def _batch(seed, V, shape=(12, 25)):
    g = torch.Generator().manual_seed(seed)
    tokens, targets = torch.randint(1, V, shape, generator=g), torch.randint(1, V, shape, generator=g)
    lens = torch.randint(1, shape[1], (shape[0],), generator=g).unsqueeze(1)
    pad = torch.arange(shape[1]).unsqueeze(0) >= lens
    return tokens.masked_fill(pad, 0), targets.masked_fill(pad, 0), torch.rand(shape, generator=g)


@pytest.mark.parametrize('V,E,Hd', [(23, 16, 24), (700, 33, 40)])
def test_training_steps_equal_a_plain_model(gpu, V, E, Hd):
    """Gradients within 1e-4 relative of the fp64 model's (fp32 sums of at most V or 300 terms: 700 x 2^-24 relative to
    the sum of magnitudes, which is within a factor 2 of the result's largest element), parameters after clipping and an
    update of size lr within 2 % of lr, three steps in a row from the fp64 model's parameters."""
    from paccmann_generator_amd import AdamW, ops
    torch.manual_seed(0)
    ref = TokenModel(V, E, Hd).double()
    for k in range(3):
        net = copy.deepcopy(ref).float().cuda()
        names = [n for n, _ in net.named_parameters()]
        opt = AdamW(net.parameters(), lr=1e-3, weight_decay=0.01)
        tokens, targets, reward = _batch(k, V)
        loss = net(tokens.cuda(), targets.cuda(), reward.cuda())
        loss.backward()
        want = ref.plain(tokens, targets, reward.double())
        grads = torch.autograd.grad(want, list(ref.parameters()))
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
        for n, p, g in zip(names, net.parameters(), grads):
            assert float((p.grad.cpu().double() - g).abs().max()) <= 1e-4 * float(g.abs().max()), n
        norm = ops.clip_grad_norm_([p.grad for p in net.parameters()], 0.05)
        exact = float(sum(g.square().sum() for g in grads) ** 0.5)
        assert abs(float(norm) - exact) <= 1e-5 * exact
        opt.step()
        with torch.no_grad():
            for n, p, r, g in zip(names, net.parameters(), ref.parameters(), grads):
                g = g * lm.clip_factor(exact, 0.05)
                new, _, _ = lm.adamw(r, g, torch.zeros_like(r), torch.zeros_like(r), 1, 1e-3, 0.9, 0.999, 1e-8, 0.01, True)
                # the first update is lr g / |g|: where g is a rounding of zero, its sign is free
                sure = g.abs() > 1e-3 * g.abs().max()
                off = (p.detach().cpu().double() - new).abs()
                assert float(off[sure].max()) <= 0.02 * 1e-3 and float(off.max()) <= 2.01 * 1e-3, n
                r.copy_(new)


@pytest.mark.parametrize('bits', [32, 8])
def test_whole_step_in_a_graph(gpu, bits):
    """Forward, backward, norm, clipped update in one captured graph: replays with new batches equal eager steps bit for
    bit (the eager graph's tensors are gone before the capture)."""
    from paccmann_generator_amd import AdamW
    V = 300

    def fresh():
        torch.manual_seed(1)
        net = TokenModel(V, 32, 48).cuda()
        return net, AdamW(net.parameters(), lr=1e-3, weight_decay=0.01, state_bits=bits, max_grad_norm=0.1)

    def step(net, opt, batch):
        opt.zero_grad(set_to_none=True)
        loss = net(*batch)
        loss.backward()
        opt.step()
        return loss.detach()

    (a, oa), (b, ob) = fresh(), fresh()
    held = [x.cuda() for x in _batch(0, V)]
    step(a, oa, held)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b, ob, held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lb = step(b, ob, held)
    for k in range(1, 5):
        for x, y in zip(held, _batch(k, V)):
            x.copy_(y)
        graph.replay()
        la = step(a, oa, held)
        torch.cuda.synchronize()
        assert torch.equal(la, lb)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    assert int(ob.state[b.table]['step']) == 5


def test_two_streams_at_once(gpu):
    """Two steps issued side by side on two streams share nothing: both equal the step alone."""
    nets, losses = [], []
    V = 500
    torch.manual_seed(2)
    base = TokenModel(V, 64, 72).cuda()
    batches = [[x.cuda() for x in _batch(k, V, (40, 60))] for k in (0, 1)]
    alone = []
    for bt in batches:
        net = copy.deepcopy(base)
        loss = net(*bt)
        loss.backward()
        alone.append((loss.detach(), [p.grad for p in net.parameters()]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    for bt, st in zip(batches, streams):
        net = copy.deepcopy(base)
        nets.append(net)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(3):
                for p in net.parameters():
                    p.grad = None
                loss = net(*bt)
                loss.backward()
            losses.append(loss.detach())
    torch.cuda.synchronize()
    for net, loss, (want, grads) in zip(nets, losses, alone):
        assert torch.equal(loss, want) and all(torch.equal(p.grad, g) for p, g in zip(net.parameters(), grads))


def test_decoder_methods(gpu):
    """StackGRUDecoder.embed and token_loss: the module's own lookup and output_layer + log_softmax + gather."""
    from tests import parity as P
    _, dec = P.make_pair(dict(P.TINY, pad_index=0), seed=0)
    tokens = P.synthetic_tokens(9, 14, P.TINY['vocab_size']).cuda()
    assert torch.equal(dec.embed(tokens).detach(), dec.embedding(tokens).detach())
    x = torch.tanh(torch.randn(9, 14, P.TINY['rnn_cell_size'], device='cuda')).requires_grad_(True)
    reward = torch.rand(9, 14, device='cuda')
    loss = dec.token_loss(x, tokens, reward=reward, ignore_index=0, temperature=0.7)
    got = torch.autograd.grad(loss, [x, dec.output_layer.weight, dec.output_layer.bias])
    w, b = (q.detach().cpu().double().requires_grad_(True) for q in (dec.output_layer.weight, dec.output_layer.bias))
    xd, t = x.detach().cpu().double().requires_grad_(True), tokens.cpu()
    logp = torch.log_softmax((xd @ w.t() + b) / 0.7, -1).gather(-1, t.unsqueeze(-1)).squeeze(-1)
    keep = t != 0
    want = -(logp * reward.cpu().double() * keep).sum() / keep.sum()
    assert abs(float(loss.detach()) - float(want)) <= 1e-5 * abs(float(want))
    for g, e in zip(got, torch.autograd.grad(want, [xd, w, b])):
        assert float((g.cpu().double() - e).abs().max()) <= 1e-4 * float(e.abs().max())


# ------------------------------------------------------------------------------------------- learners
def test_learner_with_the_fused_update_matches_the_oracle(gpu, tmp_path, monkeypatch):
    from paccmann_generator_amd import AdamW
    hp = H.HP
    monkeypatch.setattr(H, 'HP', dict(hp, optimizer='fused_adam'))
    H.test_policy_gradient_step_matches_oracle(gpu, tmp_path, 'omic')
    learner, *_ = H._setup(tmp_path / 'again')
    assert isinstance(learner.optimizer, AdamW) and learner.optimizer.state_bits == 32
    monkeypatch.setattr(H, 'HP', dict(hp, optimizer='sgd'))
    with pytest.raises(ValueError):
        H._setup(tmp_path / 'bad')


def test_learner_default_is_unchanged_and_8_bits_learn_alike(gpu, tmp_path, monkeypatch):
    """Three steps of the default learner, of the fused one and of the fused one with an 8-bit state from one seed: the
    first two agree to a few roundings of the update, the third to the codes' steps (half a step of the first moment's
    code is 1/127 of the block's largest, so an update is off by at most a few per cent of lr a step)."""
    hp, got = H.HP, {}
    for kind in ({}, dict(optimizer='fused_adam'), dict(optimizer='fused_adam', optimizer_state_bits=8)):
        monkeypatch.setattr(H, 'HP', dict(hp, **kind))
        learner, *_ = H._setup(tmp_path / str(len(got)))
        if not kind:
            assert type(learner.optimizer) is torch.optim.Adam
        learner.generator.seed(3)
        first = [p.detach().clone() for p in learner.generator.decoder.parameters()]
        for _ in range(3):
            rew, loss = learner.policy_gradient('cl1', 1, hp['batch_size'])
        got[len(got)] = ([p.detach() for p in learner.generator.decoder.parameters()], float(rew), loss)
    lr = hp['learning_rate']
    for a, b, c, z in zip(got[0][0], got[1][0], got[2][0], first):
        assert float((a - b).abs().max()) <= 0.02 * lr * 3
        assert float((b - c).abs().max()) <= 3 * lr and (not (a != z).any() or bool((c != z).any()))


def test_states_of_torch_and_of_several_groups_load(gpu):
    """A state of torch's Adam goes on as it would there; groups whose counters agree keep a counter each."""
    from paccmann_generator_amd import AdamW
    start = [torch.randn(300, generator=torch.Generator().manual_seed(k)).cuda() for k in range(3)]
    slopes = [[torch.randn(300, generator=torch.Generator().manual_seed(10 * n + k)).cuda() for k in range(3)] for n in range(6)]
    groups = lambda ps: [dict(params=ps[:1], lr=1e-2), dict(params=ps[1:], lr=3e-3)]         # noqa: E731

    def run(opt, ps, steps):
        for n in steps:
            for p, g in zip(ps, slopes[n]):
                p.grad = g.clone()
            opt.step()

    a = [s.clone().requires_grad_(True) for s in start]
    theirs = torch.optim.Adam(groups(a), weight_decay=0.01)
    run(theirs, a, range(3))
    b = [p.detach().clone().requires_grad_(True) for p in a]
    ours = AdamW(groups(b), decoupled=False, weight_decay=0.01)
    ours.load_state_dict(theirs.state_dict())
    assert [g['lr'] for g in ours.param_groups] == [1e-2, 3e-3] and not any(g['decoupled'] for g in ours.param_groups)
    c = [p.detach().clone().requires_grad_(True) for p in a]
    again = AdamW(groups(c), decoupled=False, weight_decay=0.01)
    again.load_state_dict(ours.state_dict())
    run(theirs, a, range(3, 6))
    run(ours, b, range(3, 6))
    run(again, c, range(3, 6))
    for x, y, z in zip(a, b, c):
        assert int(ours.state[y]['step']) == 6 == int(again.state[z]['step'])
        assert torch.equal(y, z)
        # three steps of at most lr (1 + decay) each, every step's quotient off by a few roundings
        assert float((x - y).abs().max()) <= 3 * 1e-2 * 32 * 2.0 ** -24 + float(x.abs().max()) * 6 * 2.0 ** -24
    bad = theirs.state_dict()
    bad['param_groups'][0]['amsgrad'] = True
    with pytest.raises(Exception, match='amsgrad'):
        ours.load_state_dict(bad)


def test_what_must_not_be_captured_is_refused(gpu, monkeypatch):
    from paccmann_generator_amd import AdamW
    from paccmann_generator_amd._ffi import PmgError
    ps = [torch.randn(40, device='cuda', requires_grad=True) for _ in range(2)]
    for p in ps:
        p.grad = torch.ones_like(p)
    fresh, used = AdamW(ps), AdamW(ps)
    used.step()
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    before = [p.detach().clone() for p in ps]
    with pytest.raises(PmgError, match='state of a parameter'):
        fresh.step()
    ps[1].grad = None
    with pytest.raises(PmgError, match='counter'):
        used.step()
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
