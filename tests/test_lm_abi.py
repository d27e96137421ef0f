"""The C ABI of include/pmg_lm.h on a machine without a GPU: exported symbols, the header as plain C, structure
layouts, workspace sizes, and the refusals, which come before any launch.  No compute call is made."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, 'include', 'pmg_lm.h')
FAKE = 1 << 20          # an aligned address that no refused call touches


def test_header_exports_and_binding_agree():
    from paccmann_generator_amd import _ffi
    text = re.sub(r'/\*.*?\*/', '', open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r'\b(pmg_[a-z0-9_]+)\s*\(', text)))
    assert declared == sorted(_ffi.LM_EXPORTS)
    lib = C.CDLL(_ffi.LIB_PATH)
    assert all(hasattr(lib, name) for name in declared)


def test_header_compiles_as_plain_c_with_the_bound_layout(tmp_path):
    from paccmann_generator_amd import _ffi
    src = tmp_path / 't.c'
    src.write_text('#include "pmg_lm.h"\n#include <stdio.h>\n#include <stddef.h>\n'
                   'int main(void){printf("%d %d %d %d %d\\n",(int)sizeof(pmg_linear_ce),(int)offsetof(pmg_linear_ce,grad_bias),(int)sizeof(pmg_adamw),(int)offsetof(pmg_adamw,step),'
                   '(int)offsetof(pmg_adamw,max_norm));return 0;}\n')
    exe = tmp_path / 't'
    subprocess.check_call(['gcc', '-std=c99', '-Wall', '-Werror', '-I', os.path.join(ROOT, 'include'), str(src), '-o',
                           str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    a, c = _ffi.PmgAdamw, _ffi.PmgLinearCe
    assert got == [C.sizeof(c), c.grad_bias.offset, C.sizeof(a), a.step.offset, a.max_norm.offset]


def test_embedding_refusals_and_workspace():
    from paccmann_generator_amd import _ffi
    lib, size = _ffi.lib, C.c_size_t(0)
    fwd = lambda **k: lib.pmg_embedding_fwd(*[{**dict(w=FAKE, ld=8, ids=FAKE, bits=64, N=4, V=9, E=8, dt=0, s=1.0, out=FAKE,   # noqa: E731
                                                      st=None), **k}[x] for x in ('w', 'ld', 'ids', 'bits', 'N', 'V', 'E', 'dt', 's', 'out', 'st')])
    assert fwd(N=0) == 0
    for bad in (dict(w=None), dict(ids=None), dict(out=None), dict(ld=7), dict(bits=16), dict(N=-1), dict(V=0), dict(E=0),
                dict(dt=3), dict(dt=-1), dict(w=FAKE + 2), dict(ids=FAKE + 4), dict(N=1 << 31), dict(V=1 << 31), dict(E=1 << 23)):
        rc = fwd(**bad)
        assert rc < 0 and len(lib.pmg_strerror(rc)) > 3, bad
    bwd = lambda **k: lib.pmg_embedding_bwd(*[{**dict(g=FAKE, ld=8, ids=FAKE, bits=64, N=4, V=9, E=8, dt=0, s=1.0, pad=-1,     # noqa: E731
                                                      out=FAKE, ws=FAKE, st=None), **k}[x]
                                              for x in ('g', 'ld', 'ids', 'bits', 'N', 'V', 'E', 'dt', 's', 'pad', 'out', 'ws', 'st')])
    for bad in (dict(g=None), dict(ids=None), dict(out=None), dict(ws=None), dict(ld=7), dict(ws=FAKE + 8), dict(bits=8),
                dict(dt=5), dict(out=FAKE + 1)):
        assert bwd(**bad) < 0, bad
    last = 0
    for n in (0, 1, 2048, 2049, 100000, 1 << 20):
        assert lib.pmg_embedding_bwd_workspace(n, 32000, 512, 1, C.byref(size)) == 0
        assert size.value >= last and size.value >= 8 * n
        last = size.value
    assert lib.pmg_embedding_bwd_workspace(-1, 9, 8, 0, C.byref(size)) < 0
    assert lib.pmg_embedding_bwd_workspace(4, 9, 8, 0, None) < 0 and lib.pmg_embedding_bwd_workspace(4, 9, 8, 3, C.byref(size)) < 0


def test_linear_ce_refusals_and_workspace():
    from paccmann_generator_amd import _ffi
    lib, size = _ffi.lib, C.c_size_t(0)

    def args(**k):
        a = _ffi.PmgLinearCe()
        d = dict(N=40, V=90, H=16, dtype=0, id_bits=64, reduction=2, logit_scale=1.0, ignore_index=-100, ld_hidden=16, ld_weight=16,
                 hidden=FAKE, weight=FAKE, targets=FAKE, loss=FAKE, lse=FAKE, count=FAKE, grad_loss=FAKE, grad_hidden=FAKE)
        for name, x in {**d, **k}.items():
            setattr(a, name, x)
        return C.byref(a)

    shapes = [dict(N=0), dict(V=0), dict(H=0), dict(H=1 << 17, ld_hidden=1 << 17, ld_weight=1 << 17), dict(dtype=2), dict(dtype=-1),
              dict(id_bits=8), dict(ld_hidden=15), dict(ld_weight=3), dict(reduction=3), dict(hidden=FAKE + 2), dict(targets=FAKE + 4),
              dict(row_weight=FAKE + 1), dict(bias=FAKE + 3)]
    for k in shapes:
        for rc in (lib.pmg_linear_ce_fwd(args(**k), FAKE, None), lib.pmg_linear_ce_bwd(args(**k), FAKE, None),
                   lib.pmg_linear_ce_workspace(args(**k), 0, C.byref(size)), lib.pmg_linear_ce_workspace(args(**k), 1, C.byref(size))):
            assert rc < 0 and len(lib.pmg_strerror(rc)) > 3, k
    for k in (dict(hidden=None), dict(weight=None), dict(targets=None), dict(loss=None), dict(lse=None), dict(count=None), dict(loss=FAKE + 2)):
        assert lib.pmg_linear_ce_fwd(args(**k), FAKE, None) < 0, k
    for k in (dict(hidden=None), dict(lse=None), dict(count=None), dict(grad_bias=FAKE), dict(grad_weight=FAKE + 2), dict(grad_lse=FAKE + 2)):
        assert lib.pmg_linear_ce_bwd(args(**k), FAKE, None) < 0, k
    assert lib.pmg_linear_ce_fwd(args(), None, None) < 0 and lib.pmg_linear_ce_fwd(args(), FAKE + 8, None) < 0
    assert lib.pmg_linear_ce_bwd(args(), FAKE + 4, None) < 0 and lib.pmg_linear_ce_workspace(None, 0, C.byref(size)) < 0
    assert lib.pmg_linear_ce_bwd(args(grad_hidden=None), FAKE, None) == 0          # nothing wanted
    # the backward's scratch holds a piece of the vocabulary, not all logits
    for N, V, H in ((8192, 128000, 4096), (65536, 32000, 1024)):
        k = dict(N=N, V=V, H=H, ld_hidden=H, ld_weight=H, dtype=1)
        assert lib.pmg_linear_ce_workspace(args(**k), 1, C.byref(size)) == 0 and size.value < N * V
        assert lib.pmg_linear_ce_workspace(args(**k), 0, C.byref(size)) == 0 and size.value < N * V // 8


def test_norm_clip_and_update_refusals():
    from paccmann_generator_amd import _ffi
    lib, size = _ffi.lib, C.c_size_t(0)
    numel, ptr, dt = (C.c_int64 * 2)(10, 20), (C.c_void_p * 2)(FAKE, FAKE + 4096), (C.c_int * 2)(0, 1)
    assert lib.pmg_grad_norm_workspace(numel, 2, C.byref(size)) == 0 and size.value >= 16
    assert lib.pmg_grad_norm_workspace((C.c_int64 * 1)(-1), 1, C.byref(size)) < 0
    assert lib.pmg_grad_norm(ptr, numel, dt, 2, None, FAKE, None) < 0
    assert lib.pmg_grad_norm(ptr, numel, dt, 2, FAKE, None, None) < 0
    assert lib.pmg_grad_norm(ptr, numel, dt, 2, FAKE, FAKE + 4, None) < 0
    assert lib.pmg_grad_norm(ptr, numel, (C.c_int * 2)(0, 7), 2, FAKE, FAKE, None) < 0
    assert lib.pmg_grad_norm((C.c_void_p * 2)(FAKE, None), numel, dt, 2, FAKE, FAKE, None) < 0
    assert lib.pmg_grad_norm((C.c_void_p * 2)(FAKE + 2, FAKE), numel, dt, 2, FAKE, FAKE, None) < 0
    assert lib.pmg_grad_clip_check(ptr, numel, dt, 2, 1.0) == 0 and lib.pmg_grad_clip(ptr, numel, dt, 2, None, 1.0, None) < 0
    for m in (0.0, -1.0, float('nan')):
        assert lib.pmg_grad_clip_check(ptr, numel, dt, 2, m) < 0 and lib.pmg_grad_clip(ptr, numel, dt, 2, FAKE, m, None) < 0
    rc = lib.pmg_grad_clip((C.c_void_p * 2)(FAKE, FAKE + 36), numel, dt, 2, FAKE, 1.0, None)
    assert rc < 0 and b'overlap' in lib.pmg_strerror(rc)

    def update(ws=FAKE, **k):
        a = _ffi.PmgAdamw()
        d = dict(n=1, dtype=0, grad_dtype=0, state_bits=32, decoupled=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0,
                 max_norm=0.0, step=FAKE - 64, param=FAKE, grad=FAKE + 4096, m=FAKE + 8192, v=FAKE + 12288)
        d.update(k)
        keep = []
        for name, x in d.items():
            if name in ('param', 'grad', 'm', 'v', 'm_top', 'v_top', 'master'):
                keep.append((C.c_void_p * 1)(x))
                x = C.addressof(keep[-1])
            setattr(a, name, x)
        n = (C.c_int64 * 1)(d.get('numel', 10))
        a.numel = C.addressof(n)
        return lib.pmg_adamw_step(C.byref(a), ws, None)

    bad = [dict(ws=None), dict(ws=FAKE + 8), dict(step=None), dict(step=FAKE - 60), dict(state_bits=16), dict(state_bits=8),
           dict(dtype=3), dict(dtype=1, grad_dtype=2), dict(grad_dtype=1), dict(master=FAKE + 16384), dict(param=None),
           dict(param=FAKE + 2), dict(m=FAKE + 8193), dict(grad=FAKE + 4097), dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(lr=float('nan')),
           dict(weight_decay=-1.0), dict(norm=FAKE + 64), dict(grad=FAKE), dict(grad=FAKE + 39 - 3), dict(v=FAKE + 8192), dict(step=FAKE + 8),
           dict(numel=-1), dict(numel=1 << 50)]
    for k in bad:
        rc = update(**k)
        assert rc < 0 and len(lib.pmg_strerror(rc)) > 3, k
    assert lib.pmg_adamw_step(None, FAKE, None) < 0
    assert lib.pmg_adamw_values(None, FAKE, 5, 1, FAKE, None) < 0
    assert lib.pmg_adamw_values(FAKE, FAKE, -5, 1, FAKE, None) < 0
    assert lib.pmg_adamw_values(FAKE, FAKE + 1, 5, 1, FAKE, None) < 0


def test_operators_are_registered_and_refuse_cpu_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from paccmann_generator_amd import _ffi, ops
    for name in ('embedding', 'embedding_bwd', 'linear_cross_entropy', 'linear_cross_entropy_bwd', 'grad_norm', 'clip_grad_norm_', 'adamw_step_', 'adamw_state_values'):
        assert str(getattr(torch.ops.pmg, name).default._schema).startswith(f'pmg::{name}(')
    p, g = torch.randn(6, 4), torch.randn(6, 4)
    m, v, _, _ = ops.adamw_state(p)
    step = torch.zeros(1, dtype=torch.int64)
    for call in (lambda: ops.embedding(p, torch.tensor([1])), lambda: ops.grad_norm([g]), lambda: ops.clip_grad_norm_([g], 1.0),
                 lambda: ops.adamw_step([p], [g], [m], [v], step), lambda: ops.adamw_state_values(v.to(torch.uint8), torch.ones(1))):
        with pytest.raises(_ffi.PmgError):
            call()
    with pytest.raises(_ffi.PmgError):
        ops.adamw_state(p, 16)
    m, v, mt, vt = ops.adamw_state(torch.zeros(257), 8)
    assert (m.dtype, v.dtype, mt.numel(), vt.numel()) == (torch.int8, torch.uint8, 2, 2)
    with FakeTensorMode():
        w = torch.empty(9, 8)
        assert torch.ops.pmg.embedding(w, torch.empty(2, 3, dtype=torch.long), 1.0, -1).shape == (2, 3, 8)
        assert torch.ops.pmg.embedding_bwd(torch.empty(2, 3, 8), torch.empty(2, 3, dtype=torch.long), 9, 1.0, -1).shape == (9, 8)
        assert torch.ops.pmg.grad_norm([w]).shape == ()


def test_update_refuses_to_write_what_it_reads():
    """Workspace, norm and learning rate apart from everything the update writes."""
    from paccmann_generator_amd import _ffi
    a = _ffi.PmgAdamw()
    d = dict(n=1, dtype=0, grad_dtype=0, state_bits=32, decoupled=1, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, max_norm=1.0,
             step=FAKE - 64)
    keep = {name: (C.c_void_p * 1)(FAKE + 4096 * k) for k, name in enumerate(('param', 'grad', 'm', 'v'))}
    n = (C.c_int64 * 1)(10)
    for name, x in {**d, **{k: C.addressof(v) for k, v in keep.items()}, 'numel': C.addressof(n)}.items():
        setattr(a, name, x)
    for ws, norm, lr in ((FAKE + 4096 * 2, None, None), (FAKE + 16, None, None), (FAKE - 64, None, None), (FAKE + 65536, FAKE + 36, None),
                         (FAKE + 32768, FAKE + 4096 * 3, None), (FAKE + 32768, None, FAKE + 4096 * 2 + 8), (FAKE + 32768, FAKE + 32768 + 8, None)):
        a.norm, a.lr_dev = norm, lr
        rc = _ffi.lib.pmg_adamw_step(C.byref(a), ws, None)
        assert rc < 0 and b'overlap' in _ffi.lib.pmg_strerror(rc), (ws, norm, lr)
