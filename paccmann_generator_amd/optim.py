"""Adam / AdamW over ``ops.adamw_step``: one pass over every parameter, its gradient and its state, for all parameters
of a type at once, with the state in 32 or 8 bits.

The reference updates the decoder with ``torch.optim.Adam`` (reinforce.py:44-49); ``AdamW(decoupled=False)`` makes the
same update.  The learners use it where ``params['optimizer']`` is ``'fused_adam'``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _ffi, ops


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (``decoupled=False``: ``torch.optim.Adam``) for parameters on one GPU.

    state_bits:      32, or 8: the moments are held as 8-bit codes with an fp32 scale per 256 values (2.03 bytes a
                     parameter instead of 8), the update itself is computed in fp32
    master_weights:  keep fp32 copies of bf16 / fp16 parameters; they take the update, the parameters are rounded copies
    max_grad_norm:   scale the gradients by min(1, max_grad_norm / (norm + 1e-6)) on the way, norm over all groups; the
                     gradients themselves stay as they are; the norm of the last step is ``self.grad_norm``
    lr:              a number, or an fp32 tensor of one element on the device (schedules under a captured step)

    Steps are counted on the device, so ``step`` can be captured into a graph once the state exists (after one eager
    step with the same gradients present; else the capture is refused); parameters that always step together share a
    counter, as in the torch classes a parameter without a gradient keeps its count.  States of the torch classes load, and
    states of 32 bits load there."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 decoupled: bool = True, state_bits: int = 32, master_weights: bool = False,
                 max_grad_norm: Optional[float] = None):
        if state_bits not in (32, 8):
            raise _ffi.PmgError('pmg: an Adam state has 32 or 8 bits')
        if max_grad_norm is not None and not max_grad_norm > 0:
            raise _ffi.PmgError('pmg: max_grad_norm must be positive')
        self.state_bits, self.master_weights, self.max_grad_norm = int(state_bits), bool(master_weights), max_grad_norm
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=float(eps), weight_decay=float(weight_decay),
                                      decoupled=bool(decoupled)))

    def __getstate__(self):
        """What copies and pickles carry: the base class names its own attributes only."""
        return dict(super().__getstate__(), state_bits=self.state_bits, master_weights=self.master_weights,
                    max_grad_norm=self.max_grad_norm, grad_norm=self.grad_norm)

    def _init_state(self, p, step):
        s = self.state[p]
        s['step'] = step
        m, v, mt, vt = ops.adamw_state(p.detach(), self.state_bits)
        s['exp_avg'], s['exp_avg_sq'] = m, v
        if self.state_bits == 8:
            s['exp_avg_top'], s['exp_avg_sq_top'] = mt, vt
        if self.master_weights and p.dtype != torch.float32:
            s['master'] = p.detach().to(torch.float32)

    @staticmethod
    def _not_captured(what):
        """What happens once must not be recorded: every replay would do it again."""
        if torch.cuda.is_current_stream_capturing():
            raise _ffi.PmgError(f'pmg: {what} while a graph is captured; make an eager step with the same gradients first')

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = [(group, [p for p in group['params'] if p.grad is not None]) for group in self.param_groups]
        grads = [p.grad for _, ps in todo for p in ps]
        if not grads:
            return loss
        if any(g.is_sparse for g in grads):
            raise _ffi.PmgError('pmg: sparse gradients are not supported')
        self.grad_norm = norm = ops.grad_norm(grads) if self.max_grad_norm is not None else None
        for group, ps in todo:
            for bucket in self._buckets(group, ps):
                self._update(group, bucket, norm)
        return loss

    def _buckets(self, group, ps):
        """The parameters of a group that one call updates: of one type, with gradients of one type and one counter."""
        fresh, buckets = {}, {}
        for p in ps:
            s = self.state[p]
            if not s:
                self._not_captured('the state of a parameter is made')
                step = fresh.get(p.device)
                if step is None:
                    step = fresh[p.device] = torch.zeros(1, dtype=torch.int64, device=p.device)
                self._init_state(p, step)
            buckets.setdefault((p.dtype, p.grad.dtype, id(s['step']), 'master' in s), []).append(p)
        # a counter belongs to one bucket: the others that hold it (no gradient this time, another type) get a copy
        owner = {}
        for key, members in buckets.items():
            step = self.state[members[0]]['step']
            if owner.setdefault(id(step), key) != key:
                self._not_captured('a step counter is divided')
                own = step.clone()
                for p in members:
                    self.state[p]['step'] = own
        stepping = set(ps)
        for p in group['params']:
            if p not in stepping and self.state.get(p) and id(self.state[p]['step']) in owner:
                self._not_captured('a step counter is divided')
                self.state[p]['step'] = self.state[p]['step'].clone()
        return buckets.values()

    def _update(self, group, ps, norm):
        states = [self.state[p] for p in ps]
        of = lambda name: [s[name] for s in states] if name in states[0] else None      # noqa: E731
        lr = group['lr']
        ops.adamw_step(ps, [p.grad for p in ps], of('exp_avg'), of('exp_avg_sq'), states[0]['step'],
                       lr=0.0 if torch.is_tensor(lr) else lr, lr_tensor=lr if torch.is_tensor(lr) else None,
                       betas=group['betas'], eps=group['eps'], weight_decay=group['weight_decay'],
                       decoupled=group['decoupled'], exp_avg_top=of('exp_avg_top'), exp_avg_sq_top=of('exp_avg_sq_top'),
                       master=of('master'), grad_norm=norm, max_norm=self.max_grad_norm or 0.0)

    def state_dict(self):
        """As the torch classes write it: a counter of its own per parameter, fp32 on the host (counters shared by a group
        would be counted up once per parameter there), so that a state of 32 bits loads into ``torch.optim.Adam`` and
        ``AdamW``.  Reading the counters synchronises."""
        out = super().state_dict()
        counts = {id(s['step']): s['step'] for s in out['state'].values() if 'step' in s}
        counts = {k: float(x) for k, x in counts.items()}
        out['state'] = {i: dict(s, step=torch.tensor(counts[id(s['step'])], dtype=torch.float32)) if 'step' in s else s
                        for i, s in out['state'].items()}
        return out

    def load_state_dict(self, state_dict):
        """States keep their types (the base class would cast them to their parameter's).  A state of 8 bits loads into
        an optimizer of 32; the other way round is refused.  States of ``torch.optim.Adam`` and ``AdamW`` load with what
        this class alone has (``decoupled``) as it is here."""
        state, groups = state_dict['state'], state_dict['param_groups']
        if any(g.get('amsgrad') or g.get('maximize') for g in groups):
            raise _ffi.PmgError('pmg: amsgrad and maximize are not supported')
        # all states are converted before anything is replaced: a refused load leaves the optimizer as it was
        loaded, shared = {}, {}
        if [len(g['params']) for g in groups] == [len(g['params']) for g in self.param_groups]:    # else the base class refuses
            for k, (given, mine) in enumerate(zip(groups, self.param_groups)):
                for i, p in zip(given['params'], mine['params']):
                    if state.get(i):
                        s = loaded[p] = self._converted(p, state[i])
                        # parameters of a group whose counters agree share one again
                        s['step'] = shared.setdefault((k, p.device, int(s['step'])), s['step'])
        before = [dict(g) for g in self.param_groups]
        super().load_state_dict(dict(state={}, param_groups=groups))
        for g, old in zip(self.param_groups, before):
            for key, value in old.items():
                g.setdefault(key, value)
        self.state.update(loaded)

    def _converted(self, p, given):
        """The state of a checkpoint for ``p`` as this optimizer holds it."""
        s = {name: torch.as_tensor(v).detach().to(p.device, copy=True) for name, v in given.items()}
        moments = ('exp_avg', 'exp_avg_sq')
        if any(name not in s for name in ('step', *moments)) or s['step'].numel() != 1:
            raise _ffi.PmgError(f'pmg: a state needs a step, exp_avg and exp_avg_sq, got {sorted(given)}')
        coded = [name + '_top' in s for name in moments]
        for name, signed in zip(moments, (True, False)):
            m, top = s[name], s.get(name + '_top')
            if m.shape != p.shape:
                raise _ffi.PmgError(f'pmg: {name} of shape {tuple(m.shape)} for a parameter {tuple(p.shape)}')
            if any(coded) and (not all(coded) or m.dtype != (torch.int8 if signed else torch.uint8) or top.dtype != torch.float32
                               or top.numel() != -(-p.numel() // _ffi.PMG_STATE_BLOCK)):
                raise _ffi.PmgError('pmg: a state of 8 bits needs int8 and uint8 codes and a scale per block of each')
            if not any(coded) and not m.is_floating_point():
                raise _ffi.PmgError(f'pmg: {name} of 32 bits must be a floating-point tensor, got {m.dtype}')
        if self.state_bits == 8 and not all(coded):
            raise _ffi.PmgError('pmg: a state of 32 bits does not load into an optimizer with 8')
        s['step'] = s['step'].to(torch.int64).reshape(1)
        like = torch.empty_like(p.detach(), dtype=torch.float32)     # in the parameter's memory order, as the update asks for
        if self.state_bits == 32:
            for name in moments:
                m = ops.adamw_state_values(s[name], s.pop(name + '_top')) if all(coded) else s[name]
                s[name] = torch.empty_like(like).copy_(m)
        elif any(s[name].stride() != like.stride() and not (s[name].is_contiguous() and like.is_contiguous()) for name in moments):
            raise _ffi.PmgError('pmg: the blocks of a state of 8 bits follow the memory order, which is another than the parameter\'s')
        if self.master_weights and p.dtype != torch.float32:
            master = s.get('master', p.detach())
            if master.shape != p.shape:
                raise _ffi.PmgError(f'pmg: a copy of shape {tuple(master.shape)} for a parameter {tuple(p.shape)}')
            s['master'] = like.copy_(master)
        else:
            s.pop('master', None)
        return s
