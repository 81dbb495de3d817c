"""
CPU tests of the policy operators: the definitions the GPU tests compare with (gradients against differences), the ABI of the
descriptors, and what is refused before anything reaches a GPU.
"""
import ctypes as C
import os
import subprocess

import pytest
import torch

from simurlacra_amd import _abi as abi, operators as ops
from simurlacra_amd.engine import load_library
from simurlacra_amd.utils.exceptions import ShapeErr, TypeErr, ValueErr
from tests import operators_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _differences(f, inputs, grads, weight):
    """ Each gradient against central differences of sum(weight * f) in random directions.  With step 1e-5 the difference is off by
    the third derivative times 1e-10 / 6 and by 1e-16 / 1e-5 of the value's rounding: below 1e-6 of the terms here. """
    gen = torch.Generator().manual_seed(1)
    for name, x in inputs.items():
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        v = [sum(float((w*o).sum()) for w, o in zip(weight, f(**{**inputs, name: x + s*1e-5*d}))) for s in (1, -1)]
        assert (v[0] - v[1])/2e-5 == pytest.approx(float((grads[name]*d).sum()), rel=1e-5, abs=1e-5), name


def test_definitions_gradients_are_those_of_differences():
    gen = torch.Generator().manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)
    off, grp = [0, 3, 3, 9], [0, 1, 3]
    x, w, b, dy = r(9, 4), r(3, 5, 4), r(3, 5), r(9, 5)
    for nl in (None, 'tanh', 'sigmoid'):
        o = ref.linear(x, w, b, off, nl, dy)
        _differences(lambda x, w, b: (ref.linear(x, w, b, off, nl)['y'],), dict(x=x, w=w, b=b), dict(x=o['dx'], w=o['dw'], b=o['db']), (dy,))
    x, w, b, st, dy, dl = r(9, 4), r(2, 4, 3), r(2, 4), r(3, 4, 2), r(9, 4), r(3, 4, 2)
    o = ref.conv(x, w, b, off, grp, st, True, dy, dl)
    _differences(lambda x, w, b, state: (lambda q: (q['y'], q['last']))(ref.conv(x, w, b, off, grp, state)), dict(x=x, w=w, b=b, state=st),
                 dict(x=o['dx'], w=o['dw'], b=o['db'], state=o['dstate']), (dy, dl))
    v = dict(u=r(9, 4), delta=r(9, 4), A=-r(2, 4, 3).abs(), B=r(9, 3), C=r(9, 3), D=r(2, 4), z=r(9, 4), bias=r(2, 4), state=r(3, 4, 3))
    dy, dl = r(9, 4), r(3, 4, 3)
    o = ref.scan(off=off, groups=grp, dy=dy, dlast=dl, **v)
    _differences(lambda **v: (lambda q: (q['y'], q['last']))(ref.scan(off=off, groups=grp, **v)), v, {k: o['d' + k] for k in v}, (dy, dl))


def test_magnitudes_bound_the_values():
    gen = torch.Generator().manual_seed(0)

    def r(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float64)
    off = [0, 5, 5, 9]
    v = dict(u=r(9, 4), delta=r(9, 4), A=-r(1, 4, 3).abs(), B=r(9, 3), C=r(9, 3), D=r(1, 4), z=r(9, 4), bias=r(1, 4), state=r(3, 4, 3))
    a, m = (ref.scan(off=off, dy=r(9, 4)*0 + 1, dlast=r(3, 4, 3)*0 - 1, mag=mag, **v) for mag in (False, True))
    for k in a:
        assert (a[k].abs() <= m[k]*(1 + 1e-12) + 1e-300).all(), k


def test_descriptors_match_the_c_compiler(tmp_path):
    structs = {'psh_linear_desc': abi.PshLinearDesc, 'psh_conv_desc': abi.PshConvDesc, 'psh_scan_desc': abi.PshScanDesc}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "pysimhip.h"', 'int main(void){',
             'printf("PSH_MAX_TAPS %d\\nPSH_MAX_MEM_STATES %d\\n", PSH_MAX_TAPS, PSH_MAX_MEM_STATES);']
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path/'layout.c', tmp_path/'layout'
    src.write_text('\n'.join(lines + ['return 0;}']))
    subprocess.check_call(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)]).decode().splitlines())
    assert int(got['PSH_MAX_TAPS']) == abi.PSH_MAX_TAPS and int(got['PSH_MAX_MEM_STATES']) == abi.PSH_MAX_MEM_STATES
    for cname, cls in structs.items():
        assert int(got[cname]) == C.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f'{cname}.{f}']) == getattr(cls, f).offset, f'{cname}.{f}'


def test_tensors_off_the_gpu_and_wrong_types_are_refused():
    off = torch.tensor([0, 4], dtype=torch.int32)
    x, w = torch.zeros(4, 3), torch.zeros(1, 2, 3)
    with pytest.raises(ValueErr, match='no CPU fallback'):
        ops.grouped_linear(x, w, None, off)
    with pytest.raises(ValueErr, match='no CPU fallback'):
        ops.causal_conv(x, torch.zeros(1, 3, 4), None, off)
    with pytest.raises(ValueErr, match='no CPU fallback'):
        ops.selective_scan_step(x, x, torch.zeros(4, 3, 2), torch.zeros(1, 3, 2), x[:, :2], x[:, :2], None, None, None)
    for f in (lambda: ops.grouped_linear([[1.]], w, None, off), lambda: ops.causal_conv(None, w, None, off)):
        with pytest.raises(TypeErr):
            f()
    with pytest.raises(ValueErr, match='in place'):
        ops.causal_conv_step(x.requires_grad_(), torch.zeros(4, 3, 3), torch.zeros(1, 3, 4), None)


def test_argument_helpers():
    cpu = torch.device('cpu')
    with pytest.raises(ShapeErr):
        ops._offsets('offsets', torch.zeros(1, dtype=torch.int32), cpu)
    with pytest.raises(TypeErr):
        ops._offsets('offsets', torch.zeros(3, dtype=torch.int64), cpu)
    with pytest.raises(ShapeErr):
        ops._policies(None, cpu, 2)
    with pytest.raises(ShapeErr):
        ops._policies(torch.zeros(3, dtype=torch.int32), cpu, 3)
    with pytest.raises(ShapeErr):
        ops._param('A', torch.zeros(2, 3), torch.float32, cpu, (3, 2))
    with pytest.raises(TypeErr):
        ops._param('A', torch.zeros(2, 3), torch.float64, cpu, (2, 3))
    t = torch.zeros(4, 2, 3)
    assert ops._state_arg('s', t, torch.float32, cpu, (4, 2, 3))[1] == 6
    long = torch.zeros(4, 10)
    view = long[:, 2:8].view(4, 2, 3)
    same, stride = ops._state_arg('s', view, torch.float32, cpu, (4, 2, 3))
    assert same is view and stride == 10
    flipped = torch.zeros(4, 3, 2).transpose(1, 2)
    assert ops._state_arg('s', flipped, torch.float32, cpu, (4, 2, 3))[0] is not flipped


def _lin(**kw):
    d = abi.PshLinearDesc()
    d.dtype, d.n_groups, d.rows, d.in_dim, d.out_dim, d.ld_x, d.ld_w, d.ld_dy = 0, 2, 100, 6, 64, 6, 6, 64
    d.offsets = d.x = d.weight = d.y = d.dy = d.dx = d.dweight = d.dbias = 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _conv(**kw):
    d = abi.PshConvDesc()
    d.n_policies, d.n_seqs, d.rows, d.channels, d.taps, d.ld_x, d.ld_dy = 1, 2, 100, 8, 4, 8, 8
    d.offsets = d.x = d.weight = d.y = d.dy = d.dx = d.dweight = d.dbias = 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _scan(**kw):
    d = abi.PshScanDesc()
    d.n_policies, d.n_seqs, d.rows, d.channels, d.states = 1, 2, 100, 8, 16
    d.ld_u = d.ld_delta = d.ld_dy = 8
    d.ld_B = d.ld_C = 16
    d.offsets = d.u = d.delta = d.A = d.B = d.C = d.y = d.check = d.dy = d.du = d.dA = d.dB = 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize('name,make,changes', [
    ('psh_grouped_linear', _lin, [dict(dtype=3), dict(nonlin=4), dict(n_groups=0), dict(rows=-1), dict(in_dim=0), dict(offsets=None), dict(x=None),
                                  dict(weight=None), dict(y=None), dict(ld_x=5), dict(ld_w=5), dict(stride_w=-1)]),
    ('psh_grouped_linear_grad', _lin, [dict(dy=None), dict(ld_dy=63), dict(nonlin=1, y=None), dict(nonlin=1)]),
    ('psh_causal_conv', _conv, [dict(dtype=-1), dict(taps=0), dict(taps=9), dict(channels=0), dict(n_policies=2), dict(offsets=None), dict(x=None),
                                dict(weight=None), dict(y=None), dict(ld_x=7), dict(step=1), dict(state=4096, stride_state=23), dict(last=4096, stride_last=0)]),
    ('psh_causal_conv_grad', _conv, [dict(dy=None), dict(ld_dy=7), dict(step=1, rows=2), dict()]),
    ('psh_selective_scan', _scan, [dict(dtype=7), dict(states=0), dict(states=65), dict(n_policies=0), dict(n_policies=3), dict(offsets=None), dict(u=None),
                                   dict(A=None), dict(B=None), dict(y=None), dict(ld_B=15), dict(ld_u=7), dict(z=4096, ld_z=0), dict(step=1),
                                   dict(state=4096, stride_state=127), dict(last=4096, stride_last=1)]),
    ('psh_selective_scan_grad', _scan, [dict(dy=None), dict(check=None), dict(step=1, rows=2), dict()]),
])
def test_the_c_entry_points_refuse_bad_descriptors(name, make, changes):
    """ Every one is turned away by the checks, before a device is touched: the context here has none. """
    lib = load_library()
    ctx = (C.c_char*8192)()
    for kw in changes:
        d = make(**kw)
        assert getattr(lib, name)(C.cast(ctx, C.c_void_p), C.byref(d)) == abi.PSH_ERR_ARG, kw
        assert lib.psh_last_error(C.cast(ctx, C.c_void_p)), kw
    assert getattr(lib, name)(None, C.byref(make())) == abi.PSH_ERR_ARG
    too_many = make(rows=(1 << 30) + 1)
    too_many.workspace, too_many.workspace_bytes = 4096, 1 << 62
    assert getattr(lib, name)(C.cast(ctx, C.c_void_p), C.byref(too_many)) == abi.PSH_ERR_UNSUPPORTED


def test_workspace_sizes():
    lib = load_library()
    assert lib.psh_grouped_linear_grad_workspace(C.byref(_lin(nonlin=1))) >= 100*64*8
    assert lib.psh_grouped_linear_grad_workspace(C.byref(_lin(rows=0))) == 0
    assert lib.psh_grouped_linear_grad_workspace(C.byref(_lin(in_dim=0))) < 0
    assert lib.psh_causal_conv_grad_workspace(C.byref(_conv(dweight=None, dbias=None))) == 0
    assert lib.psh_causal_conv_grad_workspace(C.byref(_conv())) > 0
    # states before every 8 (float64) or 16 rows of a sequence
    assert lib.psh_selective_scan_check(C.byref(_scan())) == (100//8 + 3)*8*16*8
    assert lib.psh_selective_scan_check(C.byref(_scan(dtype=1))) == (100//16 + 3)*8*16*4
    assert lib.psh_selective_scan_workspace(C.byref(_scan(step=1, rows=2))) == 0
    assert lib.psh_selective_scan_check(C.byref(_scan(states=0))) < 0


def test_memory_policy_is_described_without_a_gpu():
    from simurlacra_amd.environments.pysim.one_mass_oscillator import OneMassOscillatorSim
    from simurlacra_amd.policies import RecurrentPolicy, SSMPolicy
    spec = OneMassOscillatorSim(dt=0.02, max_steps=5).spec
    policy = SSMPolicy(spec, hidden_size=8, num_layers=2, num_states=4, num_taps=3, use_cuda=False)
    assert isinstance(policy, RecurrentPolicy) and policy.is_recurrent and policy.fused_spec() is None
    assert policy.hidden_size == 2*16*(2 + 4) and policy.init_hidden(3).shape == (3, policy.hidden_size)
    vals = policy.param_values.detach().clone()
    policy.init_param(2*vals)
    assert torch.equal(policy.param_values, 2*vals) and policy.param_values.dtype == torch.float64
    dt = torch.nn.functional.softplus(SSMPolicy(spec, use_cuda=False).layers[0].dt_bias)
    assert dt.min().item() >= 1e-3*(1 - 1e-9) and dt.max().item() <= 0.1*(1 + 1e-9)
    for kw in (dict(num_states=65), dict(num_taps=9), dict(num_layers=0), dict(dtype=torch.bfloat16)):
        with pytest.raises(ValueErr):
            SSMPolicy(spec, use_cuda=False, **kw)
    with pytest.raises(ValueErr, match='no CPU fallback'):
        policy(torch.zeros(2, dtype=torch.float64))
