"""What layer norm, embedding, gate and 8-bit product refuse, on the CPU: the Python checks, and the C entry points' own (which return
before any launch)."""
import ctypes as C

import pytest
import torch

from mega_nerf import _native as N
from mega_nerf.embedding import embedding, embedding_backward, embedding_forward
from mega_nerf.gating import dispatch, route_topk, route_topk_backward, route_topk_forward
from mega_nerf.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
from mega_nerf.quantized import QuantizedRows, int8_linear, int8_product, quantize_rows

P = 1 << 12                    # an address that is never read: every call below is refused first


def refused(rc, text):
    assert rc == -1 and text in N.lib().mnr_last_error().decode(), (rc, N.lib().mnr_last_error())


def test_cpu_tensors_are_refused():
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    c = torch.zeros(4, 2, dtype=torch.int32)
    q = QuantizedRows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4))
    for call in (lambda: layer_norm(x), lambda: layer_norm_forward(x), lambda: layer_norm_backward(x, x, None, x[:, 0], x[:, 0]),
                 lambda: embedding(i, x), lambda: embedding_forward(i, x), lambda: embedding_backward(x, i, 4), lambda: route_topk(x, 2),
                 lambda: route_topk_forward(x, 2), lambda: route_topk_backward(x[:, :2], x, c), lambda: dispatch(c, 4), lambda: quantize_rows(x),
                 lambda: int8_linear(x, q), lambda: int8_product(q, q)):
        with pytest.raises(N.NativeError, match='HIP device'):
            call()


def test_other_types_are_refused():
    for t in (torch.float64, torch.int32, torch.float8_e4m3fn):
        x = torch.zeros(4, 8).to(t)
        for call in (lambda: layer_norm(x), lambda: embedding_forward(torch.zeros(2), x), lambda: route_topk_forward(x, 2), lambda: quantize_rows(x),
                     lambda: int8_linear(x, QuantizedRows(x, x))):
            with pytest.raises(N.NativeError, match='float32, float16 or bfloat16'):
                call()


def test_int8_linear_refuses_gradients():
    with pytest.raises(NotImplementedError):
        int8_linear(torch.zeros(2, 8, requires_grad=True), QuantizedRows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)))


def test_quantised_calls_refuse_what_a_recorded_computation_produced():
    """Its gradient would be lost; a parameter is a constant, and nothing is recorded under no_grad (those calls get as far as the device)."""
    leaf = torch.zeros(4, 8, requires_grad=True)
    values, scale, bias = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, requires_grad=True), torch.zeros(4, requires_grad=True)
    q, const = QuantizedRows(values, scale.detach()), torch.zeros(2, 8)
    for call in (lambda: quantize_rows(leaf * 2), lambda: int8_linear(const, q, bias * 2), lambda: int8_linear(const, QuantizedRows(values, scale * 2)),
                 lambda: int8_product(q, q, bias * 2), lambda: int8_product(QuantizedRows(values, scale * 2), q),
                 lambda: int8_product(q, QuantizedRows(values, scale * 2))):
        with pytest.raises(NotImplementedError, match='inference-only'):
            call()
        with torch.no_grad(), pytest.raises(N.NativeError, match='HIP device'):
            call()
    for call in (lambda: quantize_rows(leaf), lambda: int8_linear(const, QuantizedRows(values, scale), bias), lambda: int8_product(q, q, bias)):
        with pytest.raises(N.NativeError, match='HIP device'):
            call()


def test_a_plain_pair_is_a_quantised_operand():
    """(values, scale) without the name, as before: such calls get as far as the device."""
    pair = (torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4))
    for call in (lambda: int8_linear(torch.zeros(2, 8), pair), lambda: int8_product(pair, pair)):
        with pytest.raises(N.NativeError, match='HIP device'):
            call()


def test_counts_are_checked_before_anything_is_allocated():
    """... and as whole numbers: a C int takes the low 32 bits of a larger one, so 2^32 + 2 cells a row were two."""
    x, c = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int32)
    for how, text in ((dict(k=0), 'chooses'), (dict(k=-1), 'chooses'), (dict(k=9), 'chooses'), (dict(k=2 ** 32 + 2), 'chooses'),
                      (dict(k=1, n_groups=0), 'n_groups'), (dict(k=1, n_groups=3), 'n_groups'), (dict(k=1, n_groups=2 ** 32 + 1), 'n_groups'),
                      (dict(k=1, n_groups=4, k_groups=5), 'k_groups'), (dict(k=1, n_groups=4, k_groups=2 ** 32 + 1), 'k_groups'),
                      (dict(k=3, n_groups=4, k_groups=1), 'hold k'), (dict(k=1, group_top=3), 'group_top'), (dict(k=1, group_top=2 ** 32 + 1), 'group_top')):
        for call in (route_topk, route_topk_forward):
            with pytest.raises(N.NativeError, match=text):
                call(x, **how)
    with pytest.raises(N.NativeError, match='chooses'):
        route_topk_forward(torch.zeros(2, 64), 33)
    for n in (0, -1, 1 << 24, 2 ** 32 + 5):
        with pytest.raises(N.NativeError, match='dispatch needs'):
            dispatch(c, n)


def test_captured_backward_is_refused(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(N.NativeError, match='route_topk_backward'):
        N.refuse_captured_backward('route_topk')


def test_layer_norm_entry_refusals():
    lib = N.lib()
    fwd = lambda **k: lib.mnr_layer_norm_forward(*[{**dict(y=P, ldy=8, m=P, r=P, x=P, ldx=8, w=None, b=None, rows=4, cols=8, eps=1e-5, t=0, wt=0, st=None), **k}[a]  # noqa: E731
                                                   for a in ('y', 'ldy', 'm', 'r', 'x', 'ldx', 'w', 'b', 'rows', 'cols', 'eps', 't', 'wt', 'st')])
    refused(fwd(t=3), 'element type')
    refused(fwd(wt=-1), 'element type')
    refused(fwd(cols=0), 'cols')
    refused(fwd(cols=(1 << 24) + 1, ldx=1 << 25, ldy=1 << 25), 'cols')
    refused(fwd(rows=-1), 'rows')
    refused(fwd(x=None), 'null')
    refused(fwd(ldx=7), 'pitch')
    refused(fwd(ldy=7), 'pitch')
    assert fwd(rows=0) == 0
    assert lib.mnr_layer_norm_backward_workspace_bytes(100, 64, 7) == 0
    need = lib.mnr_layer_norm_backward_workspace_bytes(100, 64, 0)
    bwd = lambda **k: lib.mnr_layer_norm_backward(*[{**dict(dx=P, lddx=64, dw=P, db=P, dy=P, lddy=64, x=P, ldx=64, w=None, m=P, r=P, rows=100, cols=64, t=0,  # noqa: E731
                                                            wt=0, ws=P, n=need, st=None), **k}[a] for a in (
        'dx', 'lddx', 'dw', 'db', 'dy', 'lddy', 'x', 'ldx', 'w', 'm', 'r', 'rows', 'cols', 't', 'wt', 'ws', 'n', 'st')])
    refused(bwd(n=need - 1), 'workspace')
    refused(bwd(ws=None), 'workspace')
    refused(bwd(dy=None), 'null')
    refused(bwd(m=None), 'null')
    refused(bwd(lddx=63), 'pitch')
    assert bwd(rows=0, dw=None, db=None) == 0


def test_embedding_entry_refusals():
    lib = N.lib()
    fwd = lambda **k: lib.mnr_embedding_forward(*[{**dict(o=P, ldo=8, t=P, ldt=8, n=5, w=8, i=P, it=4, s=1.0, rows=3, ty=0, st=None), **k}[a]  # noqa: E731
                                                  for a in ('o', 'ldo', 't', 'ldt', 'n', 'w', 'i', 'it', 's', 'rows', 'ty', 'st')])
    refused(fwd(ty=4), 'element type')
    refused(fwd(it=1), 'indices')
    refused(fwd(n=0), 'count')
    refused(fwd(w=0), 'width')
    refused(fwd(rows=-1), 'rows')
    refused(fwd(rows=1 << 31), 'rows')
    refused(fwd(i=None), 'null')
    refused(fwd(ldo=7), 'pitch')
    refused(fwd(ldt=7), 'pitch')
    assert fwd(rows=0) == 0
    need = lib.mnr_embedding_backward_workspace_bytes(3, 5, 8)
    bwd = lambda **k: lib.mnr_embedding_backward(*[{**dict(g=P, gt=0, dy=P, ld=8, i=P, it=4, rows=3, n=5, w=8, pad=-1, s=1.0, ty=0, ws=P, size=need, st=None),  # noqa: E731
                                                    **k}[a] for a in ('g', 'gt', 'dy', 'ld', 'i', 'it', 'rows', 'n', 'w', 'pad', 's', 'ty', 'ws', 'size', 'st')])
    refused(bwd(gt=1), 'gradient')
    refused(bwd(pad=5), 'padding_idx')
    refused(bwd(pad=-2), 'padding_idx')
    refused(bwd(size=need - 1), 'workspace')
    refused(bwd(dy=None), 'null')
    refused(bwd(g=P + 2), 'multiple of 4')
    refused(bwd(ld=7), 'pitch')


def test_gate_entry_refusals():
    lib = N.lib()
    names = ('w', 'c', 'x', 'ld', 'b', 'm', 'ldm', 'rows', 'n', 'k', 'score', 'g', 'kg', 'top', 'ren', 's', 't', 'st')
    base = dict(w=P, c=P, x=P, ld=8, b=None, m=None, ldm=0, rows=3, n=8, k=2, score=0, g=1, kg=1, top=1, ren=1, s=1.0, t=0, st=None)
    fwd = lambda **k: lib.mnr_gate_forward(*[{**base, **k}[a] for a in names])      # noqa: E731
    refused(fwd(t=5), 'element type')
    refused(fwd(n=0), 'cells')
    refused(fwd(n=1025, ld=1025), 'cells')
    refused(fwd(k=0), 'chooses')
    refused(fwd(k=9), 'chooses')
    refused(fwd(n=64, ld=64, k=33), 'chooses')
    refused(fwd(score=2), 'score')
    refused(fwd(ld=7), 'pitch')
    refused(fwd(m=P, ldm=7), 'pitch')
    refused(fwd(g=3), 'groups')
    refused(fwd(g=0), 'groups')
    refused(fwd(g=4, kg=5), 'k_groups')
    refused(fwd(g=4, kg=0), 'k_groups')
    refused(fwd(g=4, kg=1, k=3), 'k cells')
    refused(fwd(top=3), 'best')
    refused(fwd(x=None), 'null')
    assert fwd(rows=0) == 0
    bwd = lambda **k: lib.mnr_gate_backward(*[{**dict(d=P, ldd=8, dw=P, lddw=2, x=P, ld=8, c=P, m=None, ldm=0, rows=3, n=8, k=2, score=0, ren=1, s=1.0, t=0,  # noqa: E731
                                                      st=None), **k}[a] for a in ('d', 'ldd', 'dw', 'lddw', 'x', 'ld', 'c', 'm', 'ldm', 'rows', 'n', 'k', 'score',
                                                                                  'ren', 's', 't', 'st')])
    refused(bwd(ldd=7), 'pitch')
    refused(bwd(lddw=1), 'pitch')
    refused(bwd(dw=None), 'null')
    need = lib.mnr_gate_dispatch_workspace_bytes(10, 4)
    refused(lib.mnr_gate_dispatch(P, P, P, 10, 0, P, need, None), 'cells')
    refused(lib.mnr_gate_dispatch(P, P, P, -1, 4, P, need, None), 'slots')
    refused(lib.mnr_gate_dispatch(P, P, P, 10, 4, P, need - 1, None), 'workspace')
    refused(lib.mnr_gate_dispatch(P, None, P, 10, 4, P, need, None), 'null')


def test_product_entry_refusals():
    lib = N.lib()
    quant = lambda **k: lib.mnr_quantize_rows(*[{**dict(v=P, p=128, s=P, x=P, ld=100, rows=3, cols=100, t=0, st=None), **k}[a]      # noqa: E731
                                                for a in ('v', 'p', 's', 'x', 'ld', 'rows', 'cols', 't', 'st')])
    refused(quant(p=120), 'pitch')
    refused(quant(p=96), 'pitch')
    refused(quant(v=P + 8), 'multiple of 16')
    refused(quant(cols=0), 'cols')
    refused(quant(ld=99), 'pitch')
    refused(quant(t=9), 'element type')
    assert quant(rows=0) == 0
    names = ('y', 'ldy', 'a', 'lda', 'sa', 'b', 'ldb', 'sb', 'bias', 'm', 'n', 'k', 'act', 't', 'st')
    base = dict(y=P, ldy=32, a=P, lda=128, sa=P, b=P, ldb=128, sb=P, bias=None, m=4, n=32, k=100, act=0, t=0, st=None)
    prod = lambda **k: lib.mnr_int8_product(*[{**base, **k}[a] for a in names])      # noqa: E731
    refused(prod(k=0), 'k <=')
    refused(prod(k=131072, lda=131072, ldb=131072), 'k <=')
    refused(prod(a=P + 4), 'multiples of 16')
    refused(prod(lda=120), 'multiples of 16')
    refused(prod(lda=96), 'pitch')
    refused(prod(ldb=96), 'pitch')
    refused(prod(ldy=31), 'pitch')
    refused(prod(act=2), 'activation')
    refused(prod(b=None), 'null')
    refused(prod(m=-1), 'm, n')
    refused(prod(lda=1 << 22), 'below 2^22')
    assert prod(m=0) == 0 and prod(n=0) == 0
    need = lib.mnr_int8_linear_workspace_bytes(4, 100)
    assert need == 4 * 128 + 16
    linear = lambda **k: lib.mnr_int8_linear(*[{**base, 'x': P, 'ldx': 100, 'xt': 0, 'ws': P, 'size': need, **k}[a] for a in (      # noqa: E731
        'y', 'ldy', 'x', 'ldx', 'xt', 'b', 'ldb', 'sb', 'bias', 'm', 'n', 'k', 'act', 't', 'ws', 'size', 'st')])
    refused(linear(size=need - 1), 'workspace')
    refused(linear(ws=P + 8), 'workspace')
    refused(linear(xt=3), 'element type')
    refused(linear(t=3), 'element type')
    refused(linear(ldx=99), 'pitch')
    refused(linear(k=131072), 'k <=')
    assert linear(m=0) == 0


def test_every_argument_list_matches_the_header():
    """The ctypes argument counts of the operators equal the C declarations'."""
    import re
    from pathlib import Path
    hdr = (Path(__file__).resolve().parent.parent / 'include' / 'mnr_api.h').read_text()
    lib = N.lib()
    for name in ('mnr_layer_norm_forward', 'mnr_layer_norm_backward', 'mnr_layer_norm_backward_workspace_bytes', 'mnr_embedding_forward', 'mnr_embedding_backward',
                 'mnr_embedding_backward_workspace_bytes', 'mnr_gate_forward', 'mnr_gate_backward', 'mnr_gate_dispatch', 'mnr_gate_dispatch_workspace_bytes',
                 'mnr_quantize_rows', 'mnr_int8_product', 'mnr_int8_linear', 'mnr_int8_linear_workspace_bytes'):
        args = re.search(r'\b%s\(([^;]*)\);' % name, hdr).group(1).split(',')
        want = [C.c_void_p if '*' in a else C.c_int64 if 'int64_t' in a else C.c_size_t if 'size_t' in a else C.c_float if 'float' in a else C.c_int for a in args]
        assert list(getattr(lib, name).argtypes) == want, name


def test_gate_kernels_are_the_ones_that_calls_reach():
    """A lane holds 8, 16 or 32 cells where the logits decide and in the gradient, 8 or 16 where scores do; up to that many cells are one
    lane's, beyond it lanes double up to 1024 cells.  No other shape is built."""
    import importlib.util
    import re
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    spec = importlib.util.spec_from_file_location('kernel_resources', root / 'mega-nerf_amd' / 'tools' / 'kernel_resources.py')
    kr = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(kr)
    if not kr.tools_available():
        pytest.skip('llvm-objdump not found')

    def shape(n, most):
        per = next(e for e in (8, 16, most) if n <= e or e == most)
        lanes = 1
        while lanes * per < n:
            lanes *= 2
        return lanes, per

    shapes = {most: {shape(n, most) for n in range(1, 1025)} for most in (16, 32)}
    built = {'k_gate_bwd': set(), False: set(), True: set()}
    for k in kr.kernel_resources(N.LIB_PATH):
        m = re.match(r'_ZN3mnr10(k_gate_[a-z]+)I(f|DF16_|DF16b|u6__bf16)Li(\d+)ELi(\d+)E(?:Lb([01])ELb[01]E)?E', k['symbol'])
        if m:
            built['k_gate_bwd' if m[1] == 'k_gate_bwd' else m[5] == '1'].add((int(m[3]), int(m[4])))
    assert built == {'k_gate_bwd': shapes[32], False: shapes[32], True: shapes[16]}


def test_no_kernel_holds_packed_fp32_arithmetic():
    """v_pk_add / mul / fma_f32 have given wrong values on these GPUs: no code object of the library holds one (the build forbids them;
    tgemm.hip, built without that flag, must be free of them by itself)."""
    import importlib.util
    import os
    import shutil
    import subprocess
    import tempfile
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    spec = importlib.util.spec_from_file_location('kernel_resources', root / 'mega-nerf_amd' / 'tools' / 'kernel_resources.py')
    kr = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(kr)
    if not kr.tools_available():
        pytest.skip('llvm-objdump not found')
    objdump = os.path.join(kr.LLVM_BIN, 'llvm-objdump')
    seen = 0
    with tempfile.TemporaryDirectory(prefix='mnr_pk_') as tmp:
        copy = os.path.join(tmp, 'lib.so')
        shutil.copy(N.LIB_PATH, copy)
        subprocess.run([objdump, '--offloading', copy], capture_output=True, check=True, cwd=tmp)
        for f in sorted(os.listdir(tmp)):
            if 'amdgcn' not in f:
                continue
            dis = subprocess.Popen([objdump, '-d', '--no-show-raw-insn', '--no-leading-addr', os.path.join(tmp, f)], stdout=subprocess.PIPE)
            found = subprocess.run(['grep', '-m', '1', '-E', r'v_pk_(add|mul|fma)_f32'], stdin=dis.stdout, capture_output=True, text=True)
            dis.stdout.close()
            dis.wait()
            assert found.stdout == '', (f, found.stdout)
            seen += 1
    assert seen > 20
