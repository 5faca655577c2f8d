"""The C ABI of layer norm and of the operators on logits: struct layouts, and arguments that are refused before any CUDA call."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), '..'))


def test_struct_layouts_match_header(tmp_path):
    from b200gdn import _lib
    structs = {'b200gdn_layer_norm_args': _lib.LayerNormArgs, 'b200gdn_logprob_args': _lib.LogprobArgs, 'b200gdn_distill_args': _lib.DistillArgs}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    lines += ['printf("%d\\n", B200GDN_MAX_TOP);', 'printf("%d\\n", B200GDN_MAX_LIST);']
    want += [_lib.MAX_TOP, _lib.MAX_LIST]
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


def test_bad_arguments_of_layer_norm():
    from b200gdn import _lib
    for fn in ('b200gdn_layer_norm_fwd', 'b200gdn_layer_norm_bwd'):
        assert getattr(_lib.load(), fn)(None, None) == -1
        refused(fn, _lib.LayerNormArgs(), -1, 'empty problem')
        refused(fn, _lib.LayerNormArgs(rows=1 << 31, D=8), -2, 'rows')
        refused(fn, _lib.LayerNormArgs(rows=4, D=8, dtype=3), -1, 'dtype')
        refused(fn, _lib.LayerNormArgs(rows=4, D=(1 << 23) + 1), -2, 'D=')
    refused('b200gdn_layer_norm_fwd', _lib.LayerNormArgs(rows=4, D=8), -1, 'a->x is NULL')
    refused('b200gdn_layer_norm_fwd', _lib.LayerNormArgs(rows=4, D=8, x=256, y=256, mean=256), -1, 'come together')
    refused('b200gdn_layer_norm_bwd', _lib.LayerNormArgs(rows=4, D=8, z=256, mean=256, rstd=256, dy=256, dx=256, dweight=256), -1, 'partials is NULL')
    a = _lib.LayerNormArgs(rows=4, D=8)
    a.struct_bytes = 8
    assert _lib.load().b200gdn_layer_norm_fwd(C.byref(a), None) == -1 and b'ABI mismatch' in _lib.load().b200gdn_last_error()
    assert _lib.load().b200gdn_layer_norm_ctas(1) >= 1


@pytest.mark.parametrize('name', ['logprob', 'distill'])
def test_bad_rows_of_logits(name):
    from b200gdn import _lib
    cls = {'logprob': _lib.LogprobArgs, 'distill': _lib.DistillArgs}[name]
    for way in ('fwd', 'bwd'):
        fn = f'b200gdn_{name}_{way}'
        assert getattr(_lib.load(), fn)(None, None) == -1
        refused(fn, cls(), -1, 'empty problem')
        refused(fn, cls(rows=2, V=5, inner=0), -1, 'empty problem')
        refused(fn, cls(rows=(1 << 27) + 1, V=5, inner=1), -2, 'rows')
        refused(fn, cls(rows=2, V=(1 << 30) + 1, inner=1), -2, 'entries')
        refused(fn, cls(rows=2, V=5, inner=1, dtype=4), -1, 'dtype')
        for scale in (0.0, -1.0, float('nan'), float('inf')):
            refused(fn, cls(rows=2, V=5, inner=1, scale=scale), -1, 'scale')
        refused(fn, cls(rows=2, V=5, inner=1, scale=1), -1, 'logits is NULL')
        refused(fn, cls(rows=2, V=5, inner=1, scale=1, logits=257), -1, 'boundary')
        refused(fn, cls(rows=2, V=5, inner=1, scale=1, dtype=2, logits=256, dlogits=258), -1, 'boundary')


def test_bad_arguments_of_logprob_and_distill():
    from b200gdn import _lib
    rows = dict(rows=2, V=50, inner=1, scale=1.0, logits=256)
    for k in (-1, 51, 129):
        refused('b200gdn_logprob_fwd', _lib.LogprobArgs(top_k=k, **rows), -2, 'top_k')
    refused('b200gdn_logprob_fwd', _lib.LogprobArgs(tokens=256, token_bytes=2, **rows), -1, 'token_bytes')
    refused('b200gdn_logprob_fwd', _lib.LogprobArgs(logprobs=256, **rows), -1, 'tokens is NULL')
    refused('b200gdn_logprob_fwd', _lib.LogprobArgs(top_k=3, **rows), -1, 'top_ids is NULL')
    refused('b200gdn_logprob_bwd', _lib.LogprobArgs(**rows), -1, 'stats is NULL')
    refused('b200gdn_logprob_bwd', _lib.LogprobArgs(stats=256, dlogits=256, dentropy=256, **rows), -1, 'entropy is NULL')
    for k in (0, 257):
        refused('b200gdn_distill_fwd', _lib.DistillArgs(K=k, **rows), -2, 'entries a row')
    refused('b200gdn_distill_fwd', _lib.DistillArgs(K=3, id_bytes=1, **rows), -1, 'id_bytes')
    refused('b200gdn_distill_fwd', _lib.DistillArgs(K=3, id_bytes=8, teacher_dtype=7, **rows), -1, 'teacher_dtype')
    refused('b200gdn_logprob_fwd', _lib.LogprobArgs(**rows), -1, 'workspace is NULL')
    lists = dict(K=3, id_bytes=8, teacher=256, ids=256, **rows)
    refused('b200gdn_distill_fwd', _lib.DistillArgs(**lists), -1, 'row_loss is NULL')
    refused('b200gdn_distill_fwd', _lib.DistillArgs(row_loss=256, **lists), -1, 'workspace is NULL')
    for fn, flags in (('b200gdn_distill_fwd', _lib.DISTILL_SKIP_ONE | _lib.DISTILL_SCALAR), ('b200gdn_distill_bwd', _lib.DISTILL_SKIP_ONE)):
        refused(fn, _lib.DistillArgs(row_loss=256, workspace=256, dloss=256, dlogits=256, flags=flags, **lists), -1, 'SKIP_ONE')
    refused('b200gdn_distill_bwd', _lib.DistillArgs(row_loss=256, workspace=256, **lists), -1, 'dloss is NULL')
    lib = _lib.load()
    assert lib.b200gdn_distill_workspace_bytes(4, 1000, 0, 8) > lib.b200gdn_distill_workspace_bytes(2, 1000, 0, 8) > 0
    assert lib.b200gdn_logprob_workspace_bytes(4, 1000, 0, 8) > lib.b200gdn_logprob_workspace_bytes(4, 1000, 0, 0) > 0


def test_cpu_tensors_are_refused():
    import torch
    from b200gdn import B200GDNError, LayerNorm, layer_norm, token_logprobs, topk_distill_loss
    x = torch.zeros(2, 8)
    for call in (lambda: layer_norm(x), lambda: LayerNorm(8)(x), lambda: token_logprobs(x, torch.zeros(2, dtype=torch.long)),
                 lambda: topk_distill_loss(x, x, x.long())):
        with pytest.raises(B200GDNError, match='CUDA device only'):
            call()


PIECES = r'''
#include <stdio.h>
#include "layer_norm_pieces.h"
int main() {   // dtype, param_dtype, D, addresses of rows, weight and bias; prints the elements that are moved at a time
  b200gdn_layer_norm_args a{};
  long x, w, b;
  while (scanf("%d %d %d %ld %ld %ld", &a.dtype, &a.param_dtype, &a.D, &x, &w, &b) == 6) {
    a.x = a.y = (void*)x;
    a.weight = (void*)w;
    a.bias = (void*)b;
    printf("%d\n", gdn::layer_norm_piece(a));
  }
}
'''


def test_layer_norm_moves_no_more_than_every_tensor_is_aligned_for(tmp_path):
    """The rule that chooses the kernels, by arithmetic: N elements of a row are one access, N parameters accesses of N times their
    own size, 16 bytes at most.  A slice of a flat buffer of fp32 parameters begins on any boundary of 4."""
    src, exe = tmp_path / 'pieces.cpp', tmp_path / 'pieces'
    src.write_text(PIECES)
    csrc = os.path.join(ROOT, 'flash-linear-attention_b200', 'csrc')
    subprocess.check_call(['g++', '-std=c++17', '-I', csrc, '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    base, cases = 1 << 12, []
    for dtype in (0, 1, 2):
        size = 4 if dtype == 2 else 2
        for ptype in (0, 1, 2):
            psize = 4 if ptype == 0 else 2
            for D in (1, 2, 7, 10, 1000, 1002, 2048, 2052):
                for x in (0, 1, 2, 4, 8):
                    for w, b in ((0, 0), (1, 0), (0, 1), (2, 2), (4, 0), (3, None), (None, 5), (None, None), (8, 8)):
                        cases.append((dtype, ptype, D, base + x * size, *(0 if o is None else base + o * psize for o in (w, b))))
    out = subprocess.run([str(exe)], input='\n'.join(' '.join(map(str, c)) for c in cases), capture_output=True, text=True, check=True).stdout.split()
    assert len(out) == len(cases)

    def fits(n, dtype, ptype, D, x, w, b):
        size, psize = 4 if dtype == 2 else 2, 4 if ptype == 0 else 2
        return D % n == 0 and x % (n * size) == 0 and all(p % min(16, n * psize) == 0 for p in (w, b))
    for got, c in zip(map(int, out), cases):
        assert fits(got, *c), (got, c)
        assert got == max(n for n in ((4, 1) if c[0] == 2 else (8, 2, 1)) if fits(n, *c)), (got, c)


def test_layer_norm_refuses_tensors_off_their_elements_boundary():
    from b200gdn import _lib
    fwd = dict(rows=4, D=8, x=256, y=256, residual=256, z=256, weight=256, bias=256, mean=256, rstd=256)
    bwd = dict(rows=4, D=8, z=256, mean=256, rstd=256, dy=256, dz=256, dx=256, weight=256, dweight=256, dbias=256, partials=256)
    for fn, good in (('b200gdn_layer_norm_fwd', fwd), ('b200gdn_layer_norm_bwd', bwd)):
        for name in good:
            if name in ('rows', 'D'):
                continue
            rows, params = name in ('x', 'y', 'residual', 'z', 'dy', 'dz', 'dx'), name in ('weight', 'bias', 'dweight', 'dbias')
            for dtype, ptype, at in ((0, 1, 257), (2, 1, 258), (1, 0, 258)):
                size = {'rows': 4 if dtype == 2 else 2, 'params': 4 if ptype == 0 else 2, 'sums': 4}['rows' if rows else 'params' if params else 'sums']
                if at % size:
                    refused(fn, _lib.LayerNormArgs(dtype=dtype, param_dtype=ptype, **{**good, name: at}), -1, 'boundary')


def test_logprob_and_distill_refuse_tensors_off_their_boundary():
    from b200gdn import _lib
    rows = dict(rows=2, V=50, inner=1, scale=1.0, logits=256, workspace=256)
    both = dict(tokens=256, token_bytes=8, entropy=256, top_k=3, top_ids=256, stats=256, **rows)
    fwd = dict(logprobs=256, top_logprobs=256, **both)
    bwd = dict(dlogprobs=256, dentropy=256, dtop_logprobs=256, dlogits=256, **both)
    for fn, good in (('b200gdn_logprob_fwd', fwd), ('b200gdn_logprob_bwd', bwd)):
        for name in ('logprobs', 'entropy', 'top_logprobs', 'stats', 'dlogprobs', 'dentropy', 'dtop_logprobs'):
            if name in good:
                refused(fn, _lib.LogprobArgs(**{**good, name: 258}), -1, 'boundary')
        for name in ('tokens', 'top_ids'):
            refused(fn, _lib.LogprobArgs(**{**good, name: 260}), -1, 'boundary')
        refused(fn, _lib.LogprobArgs(**{**good, 'token_bytes': 4, 'tokens': 258}), -1, 'boundary')
    refused('b200gdn_logprob_fwd', _lib.LogprobArgs(**{**fwd, 'workspace': 264}), -1, 'workspace')
    good = dict(K=3, id_bytes=8, teacher=256, ids=256, row_loss=256, loss=256, dloss=256, dlogits=256, **rows)
    for fn in ('b200gdn_distill_fwd', 'b200gdn_distill_bwd'):
        for name, at in (('teacher', 258), ('ids', 260), ('row_loss', 258), ('loss', 257), ('dloss', 258), ('workspace', 264)):
            refused(fn, _lib.DistillArgs(**{**good, name: at}), -1, 'boundary')
        refused(fn, _lib.DistillArgs(**{**good, 'teacher_dtype': 1, 'teacher': 257}), -1, 'boundary')
        refused(fn, _lib.DistillArgs(**{**good, 'id_bytes': 4, 'ids': 258}), -1, 'boundary')
