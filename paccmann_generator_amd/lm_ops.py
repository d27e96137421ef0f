"""Training operators around the decoder's vocabulary, over the C ABI of include/pmg_lm.h.

    torch.ops.pmg.embedding                -> pmg_embedding_fwd   rows of a table by token id, scaled; differentiable
    torch.ops.pmg.embedding_bwd            -> pmg_embedding_bwd   the gradient of the table, by sorted tokens
    torch.ops.pmg.linear_cross_entropy     -> pmg_linear_ce_fwd   loss over a vocabulary, large logits not kept; differentiable
    torch.ops.pmg.linear_cross_entropy_bwd -> pmg_linear_ce_bwd   its gradients
    torch.ops.pmg.grad_norm                -> pmg_grad_norm       norm over many gradients
    torch.ops.pmg.clip_grad_norm_          -> pmg_grad_norm, pmg_grad_clip   and their scaling, in place
    torch.ops.pmg.adamw_step_              -> pmg_adamw_step      the Adam / AdamW update of many parameters
    torch.ops.pmg.adamw_state_values       -> pmg_adamw_values    what an 8-bit state stands for

Re-exported by ``ops``.  Schemas, argument checks and autograd are in csrc/pmg_torch.cpp (lib/libpmg_torch.so); here
are the functions a user calls, with what they check on the host, and the fake (meta) implementations.  Only a HIP
implementation exists; CPU tensors raise.  Every call runs on the current stream of the device its tensors live on, with
a workspace of its own.
"""
from __future__ import annotations

import functools
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _ffi

STATE_BLOCK = _ffi.PMG_STATE_BLOCK
_ops = torch.ops.pmg


def _refusals(fn):
    """Errors of the operators' own checks as PmgError, like those of every entry point of this package."""
    @functools.wraps(fn)
    def call(*args, **kwargs):
        try:
            return fn(*args, **kwargs)
        except RuntimeError as e:
            text = str(e)
            if isinstance(e, _ffi.PmgError) or not text.startswith('pmg'):
                raise
            raise _ffi.PmgError(text.split('\n', 1)[0]) from None
    return call


def _need_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise _ffi.PmgError('pmg: tensors must live on the GPU (there is no CPU path)')


def check_ids(ids: Tensor, V: int, what: str, ignore: Optional[int] = None) -> None:
    """Host-side validation of token ids (one device->host round trip)."""
    if ids.numel() == 0:
        return
    bad = (ids < 0) | (ids >= V)
    if ignore is not None:
        bad &= ids != ignore
    if bool(bad.any()):
        raise _ffi.PmgError(f'pmg: {what} must lie in [0, {V}), got [{int(ids.min())}, {int(ids.max())}]')


# ------------------------------------------------------------------------------------------- embedding
@torch.library.register_fake('pmg::embedding')
def _(weight, ids, scale, padding_idx):
    return weight.new_empty((*ids.shape, weight.shape[1]))


@torch.library.register_fake('pmg::embedding_bwd')
def _(grad, ids, vocab_size, scale, padding_idx):
    return grad.new_empty((vocab_size, grad.shape[-1]))


@_refusals
def embedding(weight: Tensor, tokens: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              trusted_tokens: bool = False) -> Tensor:
    """``scale * weight[tokens]``: [..., E] in the type of the table [V, E] (fp32, bf16, fp16), differentiable w.r.t.
    the table.  The rows of its gradient are sums in fp32 over a token's positions, in one order whatever the launch
    (no atomics); ``padding_idx`` gets a zero row, a negative one counts from the table's end.  ``tokens``: int64 or int32
    of any shape.  ``trusted_tokens`` skips the id range check, which synchronises (captured graphs need it skipped): an id
    out of range then gives NaN."""
    if padding_idx is not None:
        padding_idx, V = int(padding_idx), weight.shape[0]
        if not -V <= padding_idx < V:
            raise _ffi.PmgError(f'pmg::embedding: padding_idx must lie in [{-V}, {V}), got {padding_idx}')
        padding_idx %= V
    _need_cuda(weight, tokens)
    if not trusted_tokens:
        check_ids(tokens, weight.shape[0], 'token ids')
    return _ops.embedding.default(weight, tokens, float(scale), -1 if padding_idx is None else padding_idx)


# --------------------------------------------------------------------------- linear cross entropy
@torch.library.register_fake('pmg::linear_cross_entropy')
def _(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction):
    f32 = dict(dtype=torch.float32)
    return (hidden.new_empty(() if reduction else targets.shape, **f32), hidden.new_empty(targets.shape, **f32),
            hidden.new_empty(() if reduction else (0,), **f32))


@torch.library.register_fake('pmg::linear_cross_entropy_keep')
def _(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction, keep):
    f32 = dict(dtype=torch.float32)
    return (hidden.new_empty(() if reduction else targets.shape, **f32), hidden.new_empty(targets.shape, **f32),
            hidden.new_empty(() if reduction else (0,), **f32),
            hidden.new_empty((targets.numel() if keep else 0, (weight.shape[0] + 3) // 4 * 4), **f32))


@torch.library.register_fake('pmg::linear_cross_entropy_bwd')
def _(grad_loss, grad_lse, hidden, weight, bias, targets, row_weight, lse, count, ignore_index, logit_scale, reduction,
      wanted, logits=None):
    return (hidden.new_empty(hidden.shape if wanted[0] else (0,)), weight.new_empty(weight.shape if wanted[1] else (0,)),
            weight.new_empty((weight.shape[0],) if wanted[2] else (0,)))


@_refusals
def linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, bias: Optional[Tensor] = None,
                         row_weight: Optional[Tensor] = None, ignore_index: int = -100, logit_scale: float = 1.0,
                         reduction: str = 'mean', trusted_tokens: bool = False) -> Tuple[Tensor, Tensor]:
    """(loss, lse) of ``logit_scale * (hidden @ weight.T + bias)`` against ``targets``, without keeping the logits: for
    training at most 256 MB of them are, in fp32, or any number whose rows take a quarter of the bytes of a hidden row.

    ``hidden`` [..., H], ``weight`` [V, H] and ``bias`` [V] are all fp32 or all bf16; ``targets`` [...] int64 or int32.
    The loss of a row is its negative log-probability times ``row_weight`` (fp32 [...], a reward say; it gets no
    gradient) and 0 where the target is ``ignore_index``.  ``reduction``: 'none' ([...]), 'sum', or 'mean' over the rows
    with a target (0 without any).  ``lse`` [...] is the log-sum-exp of every row's logits.  Differentiable through both
    w.r.t. hidden, weight and bias: logits that were not kept are formed again, a piece of the vocabulary at a time, for
    the rows whose loss or lse has a slope; the others have zero gradients and add nothing, whatever they hold.
    ``trusted_tokens`` skips the range check of the targets, which synchronises (captured graphs need it skipped): a
    target out of range then gives NaN."""
    if reduction not in _ffi.PMG_REDUCE:
        raise _ffi.PmgError(f'pmg::linear_cross_entropy: reduction must be none, sum or mean, got {reduction!r}')
    _need_cuda(hidden, weight, targets, bias, row_weight)
    if not trusted_tokens:
        check_ids(targets, weight.shape[0], 'targets', ignore=int(ignore_index))
    loss, lse, _ = _ops.linear_cross_entropy.default(hidden, weight, bias, targets, row_weight, int(ignore_index),
                                                     float(logit_scale), _ffi.PMG_REDUCE[reduction])
    return loss, lse


# --------------------------------------------------------------------------------- norm and clipping
@torch.library.register_fake('pmg::grad_norm')
def _(grads):
    return grads[0].new_empty((), dtype=torch.float32)


@torch.library.register_fake('pmg::clip_grad_norm_')
def _(grads, max_norm):
    return grads[0].new_empty((), dtype=torch.float32)


@_refusals
def grad_norm(grads: Sequence[Tensor]) -> Tensor:
    """The 2-norm of all elements of all tensors together, a 0-dim fp32 tensor (no synchronisation): squares are
    summed in fp64.  Tensors of fp32, bf16 and fp16 may be mixed; without tensors the norm is 0."""
    grads = list(grads)
    if not grads:
        return torch.zeros((), dtype=torch.float32)
    _need_cuda(*grads)
    with torch.no_grad():
        return _ops.grad_norm.default(grads)


@_refusals
def clip_grad_norm_(grads: Sequence[Tensor], max_norm: float) -> Tensor:
    """``torch.nn.utils.clip_grad_norm_`` (reinforce_omics.py:336-340) over a list of gradients: multiplies every
    gradient by min(1, max_norm / (norm + 1e-6)) in place and returns the norm before that.  Two passes over the
    gradients, no synchronisation; gradients must be dense and must not overlap."""
    grads = list(grads)
    if not max_norm > 0:
        raise _ffi.PmgError('pmg::clip_grad_norm_: max_norm must be positive')
    if not grads:
        return torch.zeros((), dtype=torch.float32)
    _need_cuda(*grads)
    with torch.no_grad():
        return _ops.clip_grad_norm_.default(grads, float(max_norm))


def clip_param_grads_(params: Sequence[Tensor], max_norm: float) -> Tensor:
    """``clip_grad_norm_`` of the gradients of ``params`` that have one."""
    return clip_grad_norm_([p.grad for p in params if p.grad is not None], max_norm)


# ------------------------------------------------------------------------------------------- AdamW
@torch.library.register_fake('pmg::adamw_step_')
def _(*args):
    return None


@torch.library.register_fake('pmg::adamw_state_values')
def _(code, top):
    return torch.empty_like(code, dtype=torch.float32)


@_refusals
def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avg: Sequence[Tensor],
               exp_avg_sq: Sequence[Tensor], step: Tensor, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 0.0, decoupled: bool = True,
               exp_avg_top: Optional[Sequence[Tensor]] = None, exp_avg_sq_top: Optional[Sequence[Tensor]] = None,
               master: Optional[Sequence[Tensor]] = None, grad_norm: Optional[Tensor] = None, max_norm: float = 0.0,
               lr_tensor: Optional[Tensor] = None) -> None:
    """One Adam update of many parameters in place (include/pmg_lm.h spells the formulas out).

    ``step``: int64 tensor of one element on the device, the number of updates so far; incremented, so that a
    captured update counts on when it is replayed.  ``decoupled``: AdamW; False adds the decay to the gradient, as
    the Adam of reinforce.py:44-49 does.  ``grad_norm`` and ``max_norm``: scale the gradients by
    min(1, max_norm / (norm + 1e-6)) on the way (the gradients stay as they are).  ``master``: fp32 copies of bf16 or
    fp16 parameters, which take the update; the parameters are written rounded.  ``exp_avg_top`` and
    ``exp_avg_sq_top``: given, the state is held in 8 bits (``adamw_state``).  ``lr_tensor``: fp32 value on the device
    that replaces ``lr`` (schedules under a captured update).  Gradients have the parameters' type or fp32."""
    params = list(params)
    if not params:
        return
    _need_cuda(step, params[0])
    with torch.no_grad():
        _ops.adamw_step_.default(params, list(grads), list(exp_avg), list(exp_avg_sq), list(exp_avg_top or ()),
                                 list(exp_avg_sq_top or ()), list(master or ()), step, lr_tensor, grad_norm, float(lr),
                                 float(betas[0]), float(betas[1]), float(eps), float(weight_decay), float(max_norm),
                                 bool(decoupled))


def adamw_state(param: Tensor, bits: int = 32):
    """A zero state for ``param``: (exp_avg, exp_avg_sq, exp_avg_top, exp_avg_sq_top); the last two are None with 32
    bits."""
    if bits == 32:
        return (torch.zeros_like(param, dtype=torch.float32), torch.zeros_like(param, dtype=torch.float32), None, None)
    if bits != 8:
        raise _ffi.PmgError('pmg: an Adam state has 32 or 8 bits')
    tops = [torch.zeros(-(-param.numel() // STATE_BLOCK), dtype=torch.float32, device=param.device) for _ in range(2)]
    return torch.zeros_like(param, dtype=torch.int8), torch.zeros_like(param, dtype=torch.uint8), *tops


@_refusals
def adamw_state_values(code: Tensor, top: Tensor) -> Tensor:
    """The fp32 values that a state held in 8 bits stands for (int8 codes: exp_avg, uint8: exp_avg_sq)."""
    _need_cuda(code, top)
    return _ops.adamw_state_values.default(code, top)
