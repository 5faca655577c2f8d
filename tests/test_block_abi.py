"""The C ABI of the gated recurrence, of the RMS norms either side of a block and of the projections: struct layouts, and arguments that are
refused before any CUDA call."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), '..'))


def test_struct_layouts_match_header(tmp_path):
    from b200gdn import _lib
    structs = {'b200gdn_gated_recurrence_args': _lib.GatedRecurrenceArgs, 'b200gdn_rms_norms_args': _lib.RmsNormsArgs, 'b200gdn_linear_args': _lib.LinearArgs}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    for name in ('NORMS_POST', 'NORMS_SIGMOID', 'NORMS_SILU', 'LINEAR_SILU', 'LINEAR_SIGMOID', 'LINEAR_GELU'):
        lines.append(f'printf("%d\\n", (int)B200GDN_{name});')
        want.append(getattr(_lib, name))
    prog = tmp_path / 'sz.c'
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b200gdn.h"\nint main(void){' + '\n'.join(lines) + 'return 0;}\n')
    exe = tmp_path / 'sz'
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(prog), '-o', str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want


def refused(fn, args, code, text):
    from b200gdn import _lib
    lib = _lib.load()
    args.struct_bytes = C.sizeof(args)
    assert getattr(lib, fn)(C.byref(args), None) == code
    assert text in lib.b200gdn_last_error().decode(), lib.b200gdn_last_error()


@pytest.mark.parametrize('name,cls', [('gated_recurrence', 'GatedRecurrenceArgs'), ('rms_norms', 'RmsNormsArgs'), ('linear', 'LinearArgs')])
def test_blocks_of_another_size(name, cls):
    from b200gdn import _lib
    for way in ('fwd', 'bwd'):
        fn = getattr(_lib.load(), f'b200gdn_{name}_{way}')
        assert fn(None, None) == -1
        a = getattr(_lib, cls)()
        a.struct_bytes = 8
        assert fn(C.byref(a), None) == -1 and b'ABI mismatch' in _lib.load().b200gdn_last_error()
        refused(f'b200gdn_{name}_{way}', getattr(_lib, cls)(), -1, 'empty problem')


def test_bad_arguments_of_the_recurrence():
    from b200gdn import _lib
    A = _lib.GatedRecurrenceArgs
    good = dict(rows=12, D=8, n_seq=3, seq_len=4, n_chunks=3, stride_x=8, stride_g=8, x=256, g=256)
    fwd, bwd = 'b200gdn_gated_recurrence_fwd', 'b200gdn_gated_recurrence_bwd'
    for fn in (fwd, bwd):
        for bad in (dict(D=0), dict(rows=0), dict(n_seq=0), dict(seq_len=-1)):
            refused(fn, A(**{**good, **bad}), -1, 'empty problem')
        refused(fn, A(**{**good, 'rows': (1 << 30) + 1}), -2, 'rows')
        refused(fn, A(**{**good, 'D': (1 << 23) + 1}), -2, 'D=')
        refused(fn, A(**{**good, 'rows': 11}), -1, 'sequences of 4 tokens')
        refused(fn, A(**{**good, 'seq_len': 0}), -1, 'chunk_meta is NULL')
        refused(fn, A(**{**good, 'seq_len': 0, 'chunk_meta': 256}), -1, 'seq_meta is NULL')
        for codes in ((3, 3), (0, 1), (1, 0), (2, 0), (-1, 2)):
            refused(fn, A(**{**good, 'dtype': codes[0], 'gate_dtype': codes[1]}), -1, 'dtype')
        refused(fn, A(**{**good, 'stride_x': 7}), -1, 'strides')
        refused(fn, A(**{**good, 'stride_g': 0}), -1, 'strides')
        refused(fn, A(**{**good, 'x': None}), -1, 'x is NULL')
        refused(fn, A(**{**good, 'g': None}), -1, 'g is NULL')
    refused(fwd, A(**good), -1, 'h is NULL')
    refused(bwd, A(**good), -1, 'states is NULL')
    refused(bwd, A(states=256, **good), -1, 'dx is NULL')
    for fn, more in ((fwd, dict(h=256, ht=256, h0=256, states=256)), (bwd, dict(states=256, dx=256, dg=256, dh=256, dht=256, dh0=256))):
        for name in list(more) + ['x', 'g']:
            for dtype, gate, at in ((0, 0, 257), (2, 2, 258), (0, 2, 258)):
                size = {'x': dtype, 'h': dtype, 'dh': dtype, 'dx': dtype, 'g': gate, 'dg': gate}.get(name, 2)
                if at % (4 if size == 2 else 2):
                    refused(fn, A(**{**good, **more, 'dtype': dtype, 'gate_dtype': gate, name: at}), -1, 'boundary')


def test_bad_arguments_of_the_norms():
    from b200gdn import _lib
    A = _lib.RmsNormsArgs
    fwd, bwd = 'b200gdn_rms_norms_fwd', 'b200gdn_rms_norms_bwd'
    good = dict(rows=4, D=8, y=256)
    for fn in (fwd, bwd):
        refused(fn, A(rows=(1 << 30) + 1, D=8), -2, 'rows')
        refused(fn, A(rows=4, D=(1 << 23) + 1), -2, 'D=')
        refused(fn, A(dtype=3, **good), -1, 'dtype')
        refused(fn, A(param_dtype=3, **good), -1, 'dtype')
        refused(fn, A(flags=6, **good), -1, 'flags')
        refused(fn, A(flags=8, **good), -1, 'flags')
        refused(fn, A(post_weight=256, **good), -1, 'NORMS_POST')
        refused(fn, A(rows=4, D=8), -1, 'y is NULL')
        refused(fn, A(rstd_y=256, **good), -1, 'come together')
    refused(fwd, A(**good), -1, 'out is NULL')
    refused(bwd, A(**good), -1, 'rstd_z is NULL')
    both = dict(rstd_y=256, rstd_z=256, **good)
    for name in ('dweight', 'dpost_weight', 'dscale'):
        refused(bwd, A(**{**both, name: 256}), -1, 'partials is NULL')
    refused(bwd, A(dgate=256, **both), -1, 'without a gate')
    every = dict(both, flags=1, residual=256, gate=256, weight=256, post_weight=256, scale=256, z=256, out=256, dout=256, dz=256, dy=256, dresidual=256,
                 dgate=256, dweight=256, dpost_weight=256, dscale=256, partials=256)
    params = ('weight', 'post_weight', 'scale', 'dweight', 'dpost_weight', 'dscale')
    for fn in (fwd, bwd):
        for name in every:
            if name in ('rows', 'D', 'flags'):
                continue
            for dtype, ptype, at in ((0, 1, 257), (2, 1, 258), (1, 0, 258)):
                size = 4 if name in ('rstd_y', 'rstd_z', 'partials') or (ptype == 0 if name in params else dtype == 2) else 2
                if at % size:
                    refused(fn, A(**{**every, 'dtype': dtype, 'param_dtype': ptype, name: at}), -1, 'boundary')
    lib = _lib.load()
    assert lib.b200gdn_rms_norms_partials(4, 64) >= 2 * 64 and lib.b200gdn_rms_norms_partials(400, 64) > lib.b200gdn_rms_norms_partials(4, 64)


def test_bad_arguments_of_the_projections():
    from b200gdn import _lib
    A = _lib.LinearArgs
    fwd, bwd = 'b200gdn_linear_fwd', 'b200gdn_linear_bwd'
    good = dict(rows=4, K=16, N=24)
    for fn in (fwd, bwd):
        for bad in (dict(K=0), dict(N=-1), dict(rows=0)):
            refused(fn, A(**{**good, **bad}), -1, 'empty problem')
        refused(fn, A(**{**good, 'rows': (1 << 30) + 1}), -2, 'rows')
        for k in ('K', 'N'):
            refused(fn, A(**{**good, k: (1 << 23) + 1}), -2, 'at most')
        refused(fn, A(dtype=2, **good), -1, 'dtype')
        refused(fn, A(activation=4, **good), -1, 'activation')
    for i, name in enumerate(('x', 'weight', 'y')):
        refused(fwd, A(**good, **dict.fromkeys(('x', 'weight', 'y')[:i], 256)), -1, f'{name} is NULL')
    refused(bwd, A(**good), -1, 'dy is NULL')
    refused(bwd, A(dy=256, dx=256, **good), -1, 'weight is NULL')
    refused(bwd, A(dy=256, dweight=256, **good), -1, 'x is NULL')
    refused(bwd, A(dy=256, activation=1, **good), -1, 'z is NULL')
    every = dict(x=256, weight=256, bias=256, residual=256, y=256, z=256, dy=256, dx=256, dweight=256, dbias=256, **good)
    for fn in (fwd, bwd):
        for name in every:
            if name not in good:
                refused(fn, A(**{**every, name: 257}), -1, 'boundary')
    lib = _lib.load()
    need = lib.b200gdn_linear_workspace_bytes(C.byref(A(**{**every, 'activation': 1})), 1)
    assert need > 0 and lib.b200gdn_linear_workspace_bytes(None, 1) == 0
    refused(bwd, A(activation=1, **every), -1, 'workspace is NULL')
    refused(bwd, A(activation=1, workspace=512, workspace_bytes=need - 1, **every), -1, 'are needed')
    refused(bwd, A(activation=1, workspace=384, workspace_bytes=need, **every), -1, 'boundary of 256')
    # rows that cannot be read in place are copied: room for that is counted
    many = dict(every, rows=1000)
    flat = lib.b200gdn_linear_workspace_bytes(C.byref(A(**many)), 0)
    assert lib.b200gdn_linear_workspace_bytes(C.byref(A(**{**many, 'x': 258})), 0) >= flat + 1000 * 16 * 2


def test_cpu_tensors_are_refused():
    import torch
    from b200gdn import B200GDNError, FusedLinear, ResidualRMSNorm, fused_linear, gated_recurrence, residual_rms_norm
    x = torch.zeros(2, 3, 8)
    for call in (lambda: gated_recurrence(x, x), lambda: residual_rms_norm(x), lambda: ResidualRMSNorm(8)(x), lambda: fused_linear(x, x[0]),
                 lambda: FusedLinear(8, 8)(x)):
        with pytest.raises(B200GDNError, match='CUDA device only'):
            call()


def test_the_restated_gradients_are_those_of_autograd():
    """oracle/block_oracle.py writes its gradients out: against torch.autograd in 64 bits, 1e-9 of the largest value."""
    import torch
    from oracle import block_oracle as O
    gen = torch.Generator().manual_seed(0)

    def rn(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)

    def same(a, b):
        assert (a - b).abs().max() <= 1e-9 * b.abs().max() + 1e-12
    bounds = [(0, 5), (5, 5), (5, 14)]
    x, g, h0, dh, dht = rn(14, 3), -rn(14, 3).abs(), rn(3, 3), rn(14, 3), rn(3, 3)
    leaves = [t.clone().requires_grad_(True) for t in (x, g, h0)]
    rows, last = [], []
    for n, (lo, hi) in enumerate(bounds):
        h = leaves[2][n]
        for t in range(lo, hi):
            h = torch.exp(leaves[1][t]) * h + leaves[0][t]
            rows.append(h)
        last.append(h)
    h, ht = torch.stack(rows), torch.stack(last)
    want = O.recurrence(x, g, h0, bounds, dh, dht)
    for name, got in zip(('h', 'ht', 'dx', 'dg', 'dh0'), [h, ht, *torch.autograd.grad([h, ht], leaves, [dh, dht])]):
        same(want[name], got.detach())
    N, D = 6, 11
    t = dict(y=rn(N, D), residual=rn(N, D), gate=rn(N, D), weight=rn(D), post_weight=rn(D), scale=rn(D))
    for act, post in (('silu', True), ('sigmoid', False), (None, True)):
        v = {k: a.clone().requires_grad_(True) for k, a in t.items()}
        p = v['y'] * torch.rsqrt(v['y'].square().mean(-1, keepdim=True) + 1e-3) * v['post_weight'] if post else v['y']
        gate = {'silu': torch.nn.functional.silu, 'sigmoid': torch.sigmoid, None: lambda q: q}[act](v['gate'])
        z = v['residual'] + v['scale'] * gate * p
        out = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-3) * v['weight']
        dout, dz = rn(N, D), rn(N, D)
        names = [k for k in t if post or k != 'post_weight']
        grads = torch.autograd.grad([out, z], [v[k] for k in names], [dout, dz])
        want = O.rms_norms(t['y'], t['weight'], t['residual'], post, t['post_weight'] if post else None, t['gate'], act, t['scale'], 1e-3, dout, dz)
        same(want['out'], out.detach())
        for k, got in zip(names, grads):
            same(want['d' + k], got)
    x, w, b, r, dy = (a.half() for a in (rn(5, 7), rn(9, 7), rn(9), rn(5, 9), rn(5, 9)))
    for act in (None, 'silu', 'sigmoid', 'gelu'):
        leaves = [a.double().requires_grad_(True) for a in (x, w, b, r)]
        z = torch.nn.functional.linear(*leaves[:3])
        y = {None: lambda q: q, 'silu': torch.nn.functional.silu, 'sigmoid': torch.sigmoid, 'gelu': torch.nn.functional.gelu}[act](z) + leaves[3]
        want = O.linear(x, w, b, r, act, dy)
        same(want['y'], y.detach())
        for k, got in zip(('dx', 'dweight', 'dbias'), torch.autograd.grad(y, leaves[:3], dy.double())):
            same(want[k], got)
