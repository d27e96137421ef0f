"""Training operators around the decoder's vocabulary, over the C ABI of include/pmg_lm.h.

    torch.ops.pmg.embedding     -> pmg_embedding_fwd   rows of a table by token id, scaled; differentiable
    torch.ops.pmg.embedding_bwd -> pmg_embedding_bwd   the gradient of the table, by sorted tokens
    torch.ops.pmg.linear_cross_entropy     -> pmg_linear_ce_fwd   loss over a vocabulary, logits not kept; differentiable
    torch.ops.pmg.linear_cross_entropy_bwd -> pmg_linear_ce_bwd   its gradients
    torch.ops.pmg.grad_norm     -> pmg_grad_norm       norm over many gradients
    torch.ops.pmg.clip_grad_norm_ -> pmg_grad_norm, pmg_grad_clip   and their scaling, in place
    torch.ops.pmg.adamw_step_   -> pmg_adamw_step      the Adam / AdamW update of many parameters
    torch.ops.pmg.adamw_state_values -> pmg_adamw_values   what an 8-bit state stands for

Re-exported by ``ops``; registered in the namespace ``pmg`` with schemas and fake implementations like the
operators there.  They are defined through ``torch.library.Library`` rather than ``custom_op``: the update of
a decoder takes about 20 us on the device, and ``custom_op`` spends three times as long on the lists
of tensors alone (59 us for four lists of 15 tensors, 13 us this way).  Only a HIP implementation exists;
CPU tensors raise.  Every call runs on the current stream of the device its tensors live on.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _ffi

_lib = torch.library.Library('pmg', 'FRAGMENT')

DTYPES = {torch.float32: _ffi.PMG_F32, torch.bfloat16: _ffi.PMG_BF16, torch.float16: _ffi.PMG_F16}
STATE_BLOCK = _ffi.PMG_STATE_BLOCK


def _dtype_code(t: Tensor) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise _ffi.PmgError(f'pmg: fp32, bf16 or fp16 tensors required, got {t.dtype}')
    return code


class _on:
    """The device of a call: entered around its launches, so that a tensor of another device than the current one
    is worked on where it lives; gives that device's current stream."""

    def __init__(self, index: int):
        self.index = index
        self.prev = -1

    def __enter__(self):
        self.prev = torch.cuda._exchange_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        torch.cuda._maybe_exchange_device(self.prev)
        return False


def _one_device(tensors: Sequence[Tensor]) -> int:
    """The index of the GPU that all tensors live on."""
    index = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or not t.is_cuda:
            _need_cuda(tensors)
            raise _ffi.PmgError('pmg: the tensors of one call must live on one device')
    return index


def _need_cuda(tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise _ffi.PmgError('pmg: tensors must live on the GPU (there is no CPU path)')


def _dense(t: Tensor) -> bool:
    """Every element once, without gaps, in some order of the dimensions."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: (t.stride(d), t.size(d)), reverse=True)
    return t.permute(order).is_contiguous()


def _same_layout(a: Tensor, b: Tensor) -> bool:
    return a.shape == b.shape and ((a.is_contiguous() and b.is_contiguous()) or a.stride() == b.stride())


def _pointers(tensors: Sequence[Tensor]):
    return (C.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _numels(tensors: Sequence[Tensor]):
    return (C.c_int64 * len(tensors))(*[t.numel() for t in tensors])


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
_lib.define('embedding(Tensor weight, Tensor ids, float scale, int padding_idx) -> Tensor')
_lib.define('embedding_bwd(Tensor grad, Tensor ids, int vocab_size, float scale, int padding_idx) -> Tensor')
_ID_BITS = {torch.int64: 64, torch.int32: 32}


def _id_bits(ids: Tensor) -> int:
    bits = _ID_BITS.get(ids.dtype)
    if bits is None:
        raise _ffi.PmgError(f'pmg: token ids must be int64 or int32, got {ids.dtype}')
    return bits


def _rows(t: Tensor, width: int) -> Tuple[Tensor, int]:
    """``t`` [..., width] as rows of contiguous elements, and the elements from one row to the next; copied where it
    is not such rows (a stride of 0 of an expanded tensor among them)."""
    t = t.reshape(-1, width)
    if t.shape[0] > 1 and (t.stride(0) < width or (width > 1 and t.stride(1) != 1)) or \
            t.shape[0] == 1 and width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.shape[0] > 1 else width)


def _embedding(weight: Tensor, ids: Tensor, scale: float, padding_idx: int) -> Tensor:
    index = _one_device([weight, ids])
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise _ffi.PmgError(f'pmg::embedding: a table [V, E] required, got {tuple(weight.shape)}')
    V, E = weight.shape
    if not -1 <= padding_idx < V:
        raise _ffi.PmgError(f'pmg::embedding: padding_idx must lie in [0, {V}) or be -1 (none)')
    dtype, bits = _dtype_code(weight), _id_bits(ids)
    w, ld = _rows(weight, E)
    flat = ids.contiguous()
    out = torch.empty(*ids.shape, E, dtype=weight.dtype, device=weight.device)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_embedding_fwd(w.data_ptr(), ld, flat.data_ptr(), bits, flat.numel(), V, E, dtype, scale,
                                        out.data_ptr(), stream)
    _ffi.check(rc, 'pmg_embedding_fwd')
    return out


def _embedding_bwd(grad: Tensor, ids: Tensor, vocab_size: int, scale: float, padding_idx: int) -> Tensor:
    index = _one_device([grad, ids])
    E = grad.shape[-1]
    if grad.shape[:-1] != ids.shape:
        raise _ffi.PmgError(f'pmg::embedding_bwd: gradient {tuple(grad.shape)} for ids {tuple(ids.shape)}')
    dtype, bits = _dtype_code(grad), _id_bits(ids)
    g, ld = _rows(grad, E)
    flat = ids.contiguous()
    need = C.c_size_t(0)
    _ffi.check(_ffi.lib.pmg_embedding_bwd_workspace(flat.numel(), vocab_size, E, C.byref(need)),
               'pmg_embedding_bwd_workspace')
    ws = torch.empty(need.value, dtype=torch.uint8, device=grad.device)
    out = torch.empty(vocab_size, E, dtype=grad.dtype, device=grad.device)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_embedding_bwd(g.data_ptr(), ld, flat.data_ptr(), bits, flat.numel(), vocab_size, E, dtype, scale,
                                        padding_idx, out.data_ptr(), ws.data_ptr(), stream)
    _ffi.check(rc, 'pmg_embedding_bwd')
    return out


def _embedding_setup(ctx, inputs, output):
    weight, ids, ctx.scale, ctx.padding_idx = inputs
    ctx.vocab_size = weight.shape[0]
    ctx.save_for_backward(ids)


def _embedding_backward(ctx, grad):
    ids, = ctx.saved_tensors
    return torch.ops.pmg.embedding_bwd.default(grad, ids, ctx.vocab_size, ctx.scale, ctx.padding_idx), None, None, None


_lib.impl('embedding', _embedding, 'CUDA')
_lib.impl('embedding_bwd', _embedding_bwd, 'CUDA')
torch.library.register_fake('pmg::embedding', lambda weight, ids, scale, padding_idx:
                            weight.new_empty((*ids.shape, weight.shape[1])), lib=_lib)
torch.library.register_fake('pmg::embedding_bwd', lambda grad, ids, vocab_size, scale, padding_idx:
                            grad.new_empty((vocab_size, grad.shape[-1])), lib=_lib)
torch.library.register_autograd('pmg::embedding', _embedding_backward, setup_context=_embedding_setup, lib=_lib)


def embedding(weight: Tensor, tokens: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              trusted_tokens: bool = False) -> Tensor:
    """``scale * weight[tokens]``: [..., E] in the type of the table [V, E] (fp32, bf16, fp16), differentiable w.r.t.
    the table.  The rows of its gradient are sums in fp32 over a token's positions, in one order whatever the launch
    (no atomics); ``padding_idx`` gets a zero row.  ``tokens``: int64 or int32 of any shape.  ``trusted_tokens`` skips
    the id range check, which synchronises (captured graphs need it skipped): an id out of range then gives NaN."""
    _need_cuda([weight, tokens])
    if not trusted_tokens:
        check_ids(tokens, weight.shape[0], 'token ids')
    return torch.ops.pmg.embedding.default(weight, tokens, float(scale), -1 if padding_idx is None else int(padding_idx))


# --------------------------------------------------------------------------- linear cross entropy
_lib.define('linear_cross_entropy(Tensor hidden, Tensor weight, Tensor? bias, Tensor targets, Tensor? row_weight, '
            'int ignore_index, float logit_scale, int reduction) -> (Tensor, Tensor, Tensor)')
_lib.define('linear_cross_entropy_bwd(Tensor? grad_loss, Tensor? grad_lse, Tensor hidden, Tensor weight, Tensor? bias, '
            'Tensor targets, Tensor? row_weight, Tensor lse, Tensor count, int ignore_index, float logit_scale, '
            'int reduction, bool[3] wanted) -> (Tensor, Tensor, Tensor)')


def _ce_struct(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction):
    """(arguments of the C call without the outputs, device index, tensors that must outlive the call)."""
    tensors = [hidden, weight, targets, *(t for t in (bias, row_weight) if t is not None)]
    index = _one_device(tensors)
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise _ffi.PmgError(f'pmg::linear_cross_entropy: weight must be [V, H], got {tuple(weight.shape)}')
    V, H = weight.shape
    if hidden.dim() < 1 or hidden.shape[-1] != H or hidden.shape[:-1] != targets.shape:
        raise _ffi.PmgError(f'pmg::linear_cross_entropy: hidden [..., {H}] and targets [...] required, got '
                            f'{tuple(hidden.shape)} and {tuple(targets.shape)}')
    if hidden.dtype != weight.dtype or (bias is not None and bias.dtype != weight.dtype) or \
            hidden.dtype not in (torch.float32, torch.bfloat16):
        raise _ffi.PmgError('pmg::linear_cross_entropy: hidden, weight and bias must all be fp32 or all be bf16 (the '
                            'slopes of the logits leave the range of fp16)')
    if bias is not None and bias.shape != (V,):
        raise _ffi.PmgError(f'pmg::linear_cross_entropy: bias must be [{V}], got {tuple(bias.shape)}')
    if row_weight is not None and (row_weight.dtype != torch.float32 or row_weight.shape != targets.shape):
        raise _ffi.PmgError('pmg::linear_cross_entropy: row_weight must be fp32, one value per target')
    a = _ffi.PmgLinearCe()
    x, ld_x = _rows(hidden, H)
    w, ld_w = _rows(weight, H)
    t = targets.contiguous()
    b = bias.contiguous() if bias is not None else None
    r = row_weight.contiguous() if row_weight is not None else None
    a.N, a.V, a.H, a.dtype, a.id_bits = t.numel(), V, H, _dtype_code(weight), _id_bits(targets)
    a.reduction, a.logit_scale, a.ignore_index, a.ld_hidden, a.ld_weight = reduction, logit_scale, ignore_index, ld_x, ld_w
    a.hidden, a.weight, a.targets = x.data_ptr(), w.data_ptr(), t.data_ptr()
    a.bias = b.data_ptr() if b is not None else None
    a.row_weight = r.data_ptr() if r is not None else None
    return a, index, (x, w, t, b, r)


def _ce_workspace(a, backward: int, device) -> Tensor:
    need = C.c_size_t(0)
    _ffi.check(_ffi.lib.pmg_linear_ce_workspace(C.byref(a), backward, C.byref(need)), 'pmg_linear_ce_workspace')
    return torch.empty(need.value, dtype=torch.uint8, device=device)


def _ce_fwd(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction):
    a, index, keep = _ce_struct(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction)
    f32 = dict(dtype=torch.float32, device=hidden.device)
    if a.N == 0:
        return (torch.zeros(targets.shape if reduction == 0 else (), **f32), torch.zeros(targets.shape, **f32),
                torch.zeros(() if reduction else (0,), **f32))
    loss = torch.empty(targets.shape if reduction == 0 else (), **f32)
    lse, count = torch.empty(targets.shape, **f32), torch.empty(() if reduction else (0,), **f32)
    ws = _ce_workspace(a, 0, hidden.device)
    a.loss, a.lse, a.count = loss.data_ptr(), lse.data_ptr(), count.data_ptr()
    with _on(index) as stream:
        rc = _ffi.lib.pmg_linear_ce_fwd(C.byref(a), ws.data_ptr(), stream)
    _ffi.check(rc, 'pmg_linear_ce_fwd')
    return loss, lse, count


def _ce_bwd(grad_loss, grad_lse, hidden, weight, bias, targets, row_weight, lse, count, ignore_index, logit_scale, reduction,
            wanted):
    a, index, keep = _ce_struct(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction)
    dx = torch.empty(hidden.shape if wanted[0] else (0,), dtype=hidden.dtype, device=hidden.device)
    dw = torch.empty(weight.shape if wanted[1] else (0,), dtype=weight.dtype, device=hidden.device)
    db = torch.empty(bias.shape if wanted[2] else (0,), dtype=weight.dtype, device=hidden.device)
    if a.N == 0:
        return dx, dw.zero_(), db.zero_()
    slopes = []
    for name, g, like in (('grad_loss', grad_loss, () if reduction else targets.shape), ('grad_lse', grad_lse, targets.shape)):
        if g is not None:
            if g.shape != like:
                raise _ffi.PmgError(f'pmg::linear_cross_entropy_bwd: {name} must be {tuple(like)}, got {tuple(g.shape)}')
            g = g.to(torch.float32).contiguous()
            slopes.append(g)
            setattr(a, name, g.data_ptr())
    if lse.dtype != torch.float32 or lse.shape != targets.shape or not lse.is_contiguous() or count.dtype != torch.float32:
        raise _ffi.PmgError('pmg::linear_cross_entropy_bwd: lse and count must be those of the forward call')
    _one_device([hidden, lse, count, *slopes])
    a.lse, a.count = lse.data_ptr(), count.data_ptr()
    if wanted[0]:
        a.grad_hidden = dx.data_ptr()
    if wanted[1]:
        a.grad_weight = dw.data_ptr()
    if wanted[2]:
        a.grad_bias = db.data_ptr()
    ws = _ce_workspace(a, 1, hidden.device)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_linear_ce_bwd(C.byref(a), ws.data_ptr(), stream)
    _ffi.check(rc, 'pmg_linear_ce_bwd')
    return dx, dw, db


def _ce_setup(ctx, inputs, output):
    hidden, weight, bias, targets, row_weight, ctx.ignore_index, ctx.logit_scale, ctx.reduction = inputs
    _, lse, count = output
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(hidden, weight, bias, targets, row_weight, lse, count)


def _ce_backward(ctx, g_loss, g_lse, g_count):
    hidden, weight, bias, targets, row_weight, lse, count = ctx.saved_tensors
    wanted = [ctx.needs_input_grad[0], ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]]
    if (g_loss is None and g_lse is None) or not any(wanted):
        return (None,) * 8
    got = torch.ops.pmg.linear_cross_entropy_bwd.default(g_loss, g_lse, hidden, weight, bias, targets, row_weight, lse, count,
                                                         ctx.ignore_index, ctx.logit_scale, ctx.reduction, wanted)
    return tuple(g if w else None for g, w in zip(got, wanted)) + (None,) * 5


_lib.impl('linear_cross_entropy', _ce_fwd, 'CUDA')
_lib.impl('linear_cross_entropy_bwd', _ce_bwd, 'CUDA')


@torch.library.register_fake('pmg::linear_cross_entropy', lib=_lib)
def _(hidden, weight, bias, targets, row_weight, ignore_index, logit_scale, reduction):
    f32 = dict(dtype=torch.float32)
    return (hidden.new_empty(targets.shape if reduction == 0 else (), **f32), hidden.new_empty(targets.shape, **f32),
            hidden.new_empty(() if reduction else (0,), **f32))


@torch.library.register_fake('pmg::linear_cross_entropy_bwd', lib=_lib)
def _(grad_loss, grad_lse, hidden, weight, bias, targets, row_weight, lse, count, ignore_index, logit_scale, reduction, wanted):
    return (hidden.new_empty(hidden.shape if wanted[0] else (0,)), weight.new_empty(weight.shape if wanted[1] else (0,)),
            weight.new_empty((weight.shape[0],) if wanted[2] else (0,)))


torch.library.register_autograd('pmg::linear_cross_entropy', _ce_backward, setup_context=_ce_setup, lib=_lib)


def linear_cross_entropy(hidden: Tensor, weight: Tensor, targets: Tensor, bias: Optional[Tensor] = None,
                         row_weight: Optional[Tensor] = None, ignore_index: int = -100, logit_scale: float = 1.0,
                         reduction: str = 'mean', trusted_tokens: bool = False) -> Tuple[Tensor, Tensor]:
    """(loss, lse) of ``logit_scale * (hidden @ weight.T + bias)`` against ``targets``, without keeping the logits.

    ``hidden`` [..., H], ``weight`` [V, H] and ``bias`` [V] are all fp32 or all bf16; ``targets`` [...] int64 or int32.
    The loss of a row is its negative log-probability times ``row_weight`` (fp32 [...], a reward say; it gets no
    gradient) and 0 where the target is ``ignore_index``.  ``reduction``: 'none' ([...]), 'sum', or 'mean' over the rows
    with a target (0 without any).  ``lse`` [...] is the log-sum-exp of every row's logits.  Differentiable through both
    w.r.t. hidden, weight and bias: the logits are formed again, a piece of the vocabulary at a time.
    ``trusted_tokens`` skips the range check of the targets, which synchronises (captured graphs need it skipped): a
    target out of range then gives NaN."""
    if reduction not in _ffi.PMG_REDUCE:
        raise _ffi.PmgError(f'pmg::linear_cross_entropy: reduction must be none, sum or mean, got {reduction!r}')
    _need_cuda([hidden, weight, targets, bias, row_weight])
    if not trusted_tokens:
        check_ids(targets, weight.shape[0], 'targets', ignore=int(ignore_index))
    loss, lse, _ = torch.ops.pmg.linear_cross_entropy.default(hidden, weight, bias, targets, row_weight, int(ignore_index),
                                                              float(logit_scale), _ffi.PMG_REDUCE[reduction])
    return loss, lse


# --------------------------------------------------------------------------------- norm and clipping
_lib.define('grad_norm(Tensor[] grads) -> Tensor')
_lib.define('clip_grad_norm_(Tensor(a!)[] grads, float max_norm) -> Tensor')


def _norm_call(grads: List[Tensor], max_norm: Optional[float]) -> Tensor:
    index = _one_device(grads)
    n = len(grads)
    pointers, numel, dtype = _pointers(grads), _numels(grads), (C.c_int * n)(*[_dtype_code(g) for g in grads])
    need = C.c_size_t(0)
    _ffi.check(_ffi.lib.pmg_grad_norm_workspace(numel, n, C.byref(need)), 'pmg_grad_norm_workspace')
    ws = torch.empty(need.value, dtype=torch.uint8, device=grads[0].device)
    norm = torch.empty((), dtype=torch.float32, device=grads[0].device)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_grad_norm(pointers, numel, dtype, n, norm.data_ptr(), ws.data_ptr(), stream)
        _ffi.check(rc, 'pmg_grad_norm')
        if max_norm is not None:
            rc = _ffi.lib.pmg_grad_clip(pointers, numel, dtype, n, norm.data_ptr(), max_norm, stream)
            _ffi.check(rc, 'pmg_grad_clip')
    return norm


def _grad_norm(grads: List[Tensor]) -> Tensor:
    if len(grads) == 0:
        raise _ffi.PmgError('pmg::grad_norm: no tensors')
    return _norm_call([g if _dense(g) else g.contiguous() for g in grads], None)


def _clip_grad_norm(grads: List[Tensor], max_norm: float) -> Tensor:
    if len(grads) == 0:
        raise _ffi.PmgError('pmg::clip_grad_norm_: no tensors')
    if not max_norm > 0:
        raise _ffi.PmgError('pmg::clip_grad_norm_: max_norm must be positive')
    for g in grads:
        if not _dense(g):
            raise _ffi.PmgError('pmg::clip_grad_norm_: gradients must be dense (no gaps, no repeated elements)')
    return _norm_call(grads, max_norm)


_lib.impl('grad_norm', _grad_norm, 'CUDA')
_lib.impl('clip_grad_norm_', _clip_grad_norm, 'CUDA')
torch.library.register_fake('pmg::grad_norm', lambda grads: grads[0].new_empty((), dtype=torch.float32), lib=_lib)
torch.library.register_fake('pmg::clip_grad_norm_',
                            lambda grads, max_norm: grads[0].new_empty((), dtype=torch.float32), lib=_lib)


@torch.no_grad()
def grad_norm(grads: Sequence[Tensor]) -> Tensor:
    """The 2-norm of all elements of all tensors together, a 0-dim fp32 tensor (no synchronisation): squares are
    summed in fp64.  Tensors of fp32, bf16 and fp16 may be mixed; without tensors the norm is 0."""
    grads = list(grads)
    if not grads:
        return torch.zeros((), dtype=torch.float32)
    _need_cuda(grads)
    return torch.ops.pmg.grad_norm.default(grads)


@torch.no_grad()
def clip_grad_norm_(grads: Sequence[Tensor], max_norm: float) -> Tensor:
    """``torch.nn.utils.clip_grad_norm_`` (reinforce_omics.py:336-340) over a list of gradients: multiplies every
    gradient by min(1, max_norm / (norm + 1e-6)) in place and returns the norm before that.  Two passes over the
    gradients, no synchronisation; gradients must be dense and must not overlap."""
    grads = list(grads)
    if not max_norm > 0:
        raise _ffi.PmgError('pmg::clip_grad_norm_: max_norm must be positive')
    if not grads:
        return torch.zeros((), dtype=torch.float32)
    _need_cuda(grads)
    norm = torch.ops.pmg.clip_grad_norm_.default(grads, float(max_norm))
    torch.autograd.graph.increment_version(grads)
    return norm


# ------------------------------------------------------------------------------------------- AdamW
_lib.define('adamw_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avg, Tensor(c!)[] exp_avg_sq, '
            'Tensor(d!)[] exp_avg_top, Tensor(e!)[] exp_avg_sq_top, Tensor(f!)[] master, Tensor(g!) step, '
            'Tensor? lr_tensor, Tensor? grad_norm, float lr, float beta1, float beta2, float eps, float weight_decay, '
            'float max_norm, bool decoupled) -> ()')
_lib.define('adamw_state_values(Tensor code, Tensor top) -> Tensor')


def _adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_top, exp_avg_sq_top, master, step, lr_tensor, grad_norm,
                lr, beta1, beta2, eps, weight_decay, max_norm, decoupled) -> None:
    n = len(params)
    if n == 0:
        raise _ffi.PmgError('pmg::adamw_step_: no parameters')
    bits = 8 if exp_avg_top else 32
    lists = [params, grads, exp_avg, exp_avg_sq]
    if bits == 8:
        lists += [exp_avg_top, exp_avg_sq_top]
    elif exp_avg_sq_top:
        raise _ffi.PmgError('pmg::adamw_step_: scales of one half of the state only')
    if master:
        lists.append(master)
    if any(len(x) != n for x in lists):
        raise _ffi.PmgError('pmg::adamw_step_: lists of different lengths')
    index = _one_device([step, *params, *grads, *exp_avg, *exp_avg_sq, *exp_avg_top, *exp_avg_sq_top, *master])
    if step.dtype != torch.int64 or step.numel() != 1:
        raise _ffi.PmgError('pmg::adamw_step_: step must be one int64 value')
    for name, t in (('lr', lr_tensor), ('grad_norm', grad_norm)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != 1 or t.get_device() != index):
            raise _ffi.PmgError(f'pmg::adamw_step_: {name} must be one fp32 value on the device of the parameters')
    p_type, g_type = params[0].dtype, grads[0].dtype
    m_type, v_type = (torch.float32, torch.float32) if bits == 32 else (torch.int8, torch.uint8)
    dtype, grad_dtype = _dtype_code(params[0]), _dtype_code(grads[0])
    laid = []
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avg, exp_avg_sq)):
        if p.dtype != p_type or g.dtype != g_type or m.dtype != m_type or v.dtype != v_type:
            raise _ffi.PmgError('pmg::adamw_step_: one element type per list: parameters, gradients, fp32 states (or '
                                f'int8 and uint8 codes); got {p.dtype}, {g.dtype}, {m.dtype}, {v.dtype}')
        if p.shape != g.shape:
            raise _ffi.PmgError(f'pmg::adamw_step_: gradient of shape {tuple(g.shape)} for a parameter {tuple(p.shape)}')
        whole = p.is_contiguous()
        if not (whole and m.is_contiguous() and v.is_contiguous() and m.numel() == v.numel() == p.numel()) and \
                not (_dense(p) and _same_layout(p, m) and _same_layout(p, v)):
            raise _ffi.PmgError('pmg::adamw_step_: parameters must be dense (no gaps, no repeated elements) and states '
                                'must have their size and strides')
        if master and (master[i].dtype != torch.float32 or not _same_layout(p, master[i])):
            raise _ffi.PmgError('pmg::adamw_step_: 32-bit copies must be fp32 and have the strides of their parameter')
        if bits == 8:
            blocks = -(-p.numel() // STATE_BLOCK)
            for s in (exp_avg_top[i], exp_avg_sq_top[i]):
                if s.dtype != torch.float32 or s.numel() != blocks or not s.is_contiguous():
                    raise _ffi.PmgError(f'pmg::adamw_step_: {blocks} contiguous fp32 scales required for a state of '
                                        f'{p.numel()} values')
        # a gradient of another memory order than its parameter's is brought into that order
        if not (whole and g.is_contiguous()) and not _same_layout(p, g):
            g = torch.empty_like(p, dtype=g.dtype).copy_(g)
        laid.append(g)
    numel = _numels(params)
    keep = [_pointers(x) for x in (params, laid, exp_avg, exp_avg_sq)]
    a = _ffi.PmgAdamw()
    a.n, a.dtype, a.grad_dtype, a.state_bits, a.decoupled = n, dtype, grad_dtype, bits, int(decoupled)
    a.numel, a.param, a.grad, a.m, a.v = (C.addressof(x) for x in (numel, *keep))
    if bits == 8:
        keep += [_pointers(exp_avg_top), _pointers(exp_avg_sq_top)]
        a.m_top, a.v_top = C.addressof(keep[-2]), C.addressof(keep[-1])
    if master:
        keep.append(_pointers(master))
        a.master = C.addressof(keep[-1])
    a.step = step.data_ptr()
    a.lr_dev = lr_tensor.data_ptr() if lr_tensor is not None else None
    a.norm = grad_norm.data_ptr() if grad_norm is not None else None
    a.lr, a.beta1, a.beta2, a.eps, a.weight_decay, a.max_norm = lr, beta1, beta2, eps, weight_decay, max_norm
    ws = torch.empty(_ffi.PMG_ADAMW_WS, dtype=torch.uint8, device=step.device)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_adamw_step(C.byref(a), ws.data_ptr(), stream)
    _ffi.check(rc, 'pmg_adamw_step')


def _adamw_state_values(code: Tensor, top: Tensor) -> Tensor:
    index = _one_device([code, top])
    if code.dtype not in (torch.int8, torch.uint8) or top.dtype != torch.float32:
        raise _ffi.PmgError('pmg::adamw_state_values: int8 or uint8 codes and fp32 scales required')
    if not _dense(code) or not top.is_contiguous() or top.numel() != -(-code.numel() // STATE_BLOCK):
        raise _ffi.PmgError(f'pmg::adamw_state_values: dense codes with one scale per {STATE_BLOCK} required')
    out = torch.empty_like(code, dtype=torch.float32)
    with _on(index) as stream:
        rc = _ffi.lib.pmg_adamw_values(code.data_ptr(), top.data_ptr(), code.numel(), int(code.dtype == torch.int8),
                                       out.data_ptr(), stream)
    _ffi.check(rc, 'pmg_adamw_values')
    return out


_lib.impl('adamw_step_', _adamw_step, 'CUDA')
_lib.impl('adamw_state_values', _adamw_state_values, 'CUDA')
torch.library.register_fake('pmg::adamw_step_', lambda *a: None, lib=_lib)
torch.library.register_fake('pmg::adamw_state_values', lambda code, top: torch.empty_like(code, dtype=torch.float32),
                            lib=_lib)


@torch.no_grad()
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
    params, grads, exp_avg, exp_avg_sq = list(params), list(grads), list(exp_avg), list(exp_avg_sq)
    top_m = list(exp_avg_top) if exp_avg_top is not None else []
    top_v = list(exp_avg_sq_top) if exp_avg_sq_top is not None else []
    master = list(master) if master is not None else []
    if not params:
        return
    _need_cuda([step, params[0]])
    torch.ops.pmg.adamw_step_.default(params, grads, exp_avg, exp_avg_sq, top_m, top_v, master, step, lr_tensor, grad_norm,
                              float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
                              float(max_norm), bool(decoupled))
    torch.autograd.graph.increment_version([step, *params, *exp_avg, *exp_avg_sq, *top_m, *top_v, *master])


def adamw_state(param: Tensor, bits: int = 32):
    """A zero state for ``param``: (exp_avg, exp_avg_sq, exp_avg_top, exp_avg_sq_top); the last two are None with 32
    bits."""
    if bits == 32:
        return (torch.zeros_like(param, dtype=torch.float32), torch.zeros_like(param, dtype=torch.float32), None, None)
    if bits != 8:
        raise _ffi.PmgError('pmg: an Adam state has 32 or 8 bits')
    tops = [torch.zeros(-(-param.numel() // STATE_BLOCK), dtype=torch.float32, device=param.device) for _ in range(2)]
    return torch.zeros_like(param, dtype=torch.int8), torch.zeros_like(param, dtype=torch.uint8), *tops


@torch.no_grad()
def adamw_state_values(code: Tensor, top: Tensor) -> Tensor:
    """The fp32 values that a state held in 8 bits stands for (int8 codes: exp_avg, uint8: exp_avg_sq)."""
    _need_cuda([code, top])
    return torch.ops.pmg.adamw_state_values.default(code, top)
