"""
What torch keeps track of around the policy operators: saved tensors, derivatives, traces.  On the CPU, with an engine whose calls do
nothing: whatever a call returns is empty memory, and the tests are about what is refused and noticed.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode
from torch.utils.flop_counter import FlopCounterMode

from simurlacra_amd import operators as ops
from simurlacra_amd.engine import load_library
from simurlacra_amd.utils.exceptions import ValueErr


class _NoEngine:
    def __init__(self):
        self.lib, self.calls = load_library(), []

    def _stream(self):
        return 0

    def _call(self, name, *args):
        self.calls.append(name)


@pytest.fixture
def engine(monkeypatch):
    """ Tensors on the CPU count as those of a GPU, whose calls are noted down. """
    eng = _NoEngine()
    monkeypatch.setattr(ops, 'get_engine', lambda index: eng)
    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    return eng


def conv_args(S=3, D=4, K=3):
    return torch.randn(S, D), torch.randn(S, D, K - 1), torch.randn(1, D, K), torch.randn(1, D)


def scan_args(S=3, D=4, N=2):
    return dict(u=torch.randn(S, D), delta=torch.randn(S, D), A=-torch.rand(1, D, N), B=torch.randn(S, N), C=torch.randn(S, N),
                D=torch.randn(1, D), z=torch.randn(S, D), delta_bias=torch.randn(1, D))


# ------------------------------------------------------------------------------------------------- states in place
def test_a_state_that_a_backward_pass_needs_is_not_advanced_unnoticed(engine):
    x, state, w, b = conv_args()
    off = torch.arange(4, dtype=torch.int32)
    y = ops.causal_conv(x, w.requires_grad_(), b, off, state=state)
    with torch.no_grad():
        ops.causal_conv_step(x, state, w, b)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    v = scan_args()
    h = torch.randn(3, 4, 2)
    y = ops.selective_scan(**dict(v, A=v['A'].requires_grad_()), offsets=off, state=h)
    with torch.no_grad():
        ops.selective_scan_step(state=h, **v)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_steps_count_as_changes_of_the_memory_their_state_lies_in(engine):
    """ the states of a policy are slices of one vector per environment; those that anything else saved are noticed too """
    memory = torch.randn(3, 4*2 + 4*2)
    x, _, w, b = conv_args()
    v = scan_args()
    leaf = torch.randn(3, 16, requires_grad=True)
    product = memory*leaf
    before = memory._version
    ops.causal_conv_step(x, memory[:, :8].view(3, 4, 2), w, b)
    assert memory._version == before + 1
    ops.selective_scan_step(state=memory[:, 8:].view(3, 4, 2), **v)
    assert memory._version == before + 2
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        product.sum().backward()
    with torch.inference_mode():
        ops.causal_conv_step(x, torch.randn(3, 4, 2), w, b)


def test_a_refused_step_changes_nothing(engine):
    x, state, w, b = conv_args()
    before = state._version
    with pytest.raises(ValueError):
        ops.causal_conv_step(x, state, torch.randn(1, 4, 9), b)
    assert state._version == before and not engine.calls


# -------------------------------------------------------------------------------------------------- forward derivatives
def entry_points():
    """ Every call of the module with its tensors by name: [(name, function of the tensors, tensors)] """
    off = torch.arange(4, dtype=torch.int32)
    x, state, w, b = conv_args()
    v, h = scan_args(), torch.randn(3, 4, 2)
    dy, dlast = torch.randn(3, 4), torch.randn(3, 4, 2)
    lin = dict(x=torch.randn(3, 5), weight=torch.randn(3, 4, 5), bias=torch.randn(3, 4))
    check = torch.zeros(load_library().psh_selective_scan_check(ops.C.byref(
        ops.abi.PshScanDesc(ops.abi.DTYPE_F32, 0, 1, 3, 3, 4, 2))), dtype=torch.uint8)
    return [
        ('grouped_linear', lambda **t: ops.grouped_linear(**t, offsets=off, nonlin='tanh'), lin),
        ('grouped_linear_grad', lambda **t: ops.grouped_linear_grad(**t, offsets=off, nonlin='tanh'),
         dict(dy=dy, y=torch.randn(3, 4), x=lin['x'], weight=lin['weight'])),
        ('causal_conv', lambda **t: ops.causal_conv(**t, offsets=off), dict(x=x, weight=w, bias=b, state=state)),
        ('causal_conv_grad', lambda **t: ops.causal_conv_grad(**t, offsets=off),
         dict(dy=dy, dlast=state.clone(), x=x, weight=w, bias=b, state=state)),
        ('causal_conv_step', ops.causal_conv_step, dict(x=x, state=state, weight=w, bias=b)),
        ('selective_scan', lambda **t: ops.selective_scan(**t, offsets=off), dict(v, state=h)),
        ('selective_scan_check', lambda **t: ops.selective_scan_check(**t, offsets=off), dict(v, state=h)),
        ('selective_scan_grad', lambda **t: ops.selective_scan_grad(check=check, offsets=off, **t), dict(v, state=h, dy=dy, dlast=dlast)),
        ('selective_scan_step', ops.selective_scan_step, dict(v, state=h)),
    ]


NAMES = ['grouped_linear', 'grouped_linear_grad', 'causal_conv', 'causal_conv_grad', 'causal_conv_step', 'selective_scan',
         'selective_scan_check', 'selective_scan_grad', 'selective_scan_step']


def test_the_entry_points_run_here(engine):
    for name, f, tensors in entry_points():
        f(**tensors)
    assert [n for n, _, _ in entry_points()] == NAMES and len(engine.calls) == len(NAMES)


@pytest.mark.parametrize('k', range(len(NAMES)), ids=NAMES)
def test_forward_derivatives_are_refused_and_not_zero(engine, k):
    """ A tangent on any of the tensors; without one, calls inside a dual level are calls as usual. """
    name, f, tensors = entry_points()[k]
    for which in tensors:
        with fwd.dual_level():
            dual = fwd.make_dual(tensors[which], torch.ones_like(tensors[which]))
            for mode in (torch.no_grad, torch.enable_grad):
                with mode(), pytest.raises(ValueErr, match='forward'):
                    f(**dict(tensors, **{which: dual}))
    assert not engine.calls
    with fwd.dual_level():
        f(**tensors)
    assert len(engine.calls) == 1


def test_forward_derivatives_beside_those_that_are_differentiated_are_refused(engine):
    """ also where another tensor asks for a gradient, so that the call is autograd's """
    name, f, tensors = entry_points()[0]
    with fwd.dual_level():
        dual = fwd.make_dual(tensors['x'], torch.ones_like(tensors['x']))
        with pytest.raises(ValueErr, match='forward'):
            f(x=dual, weight=tensors['weight'].clone().requires_grad_(), bias=tensors['bias'])
    with pytest.raises(Exception):
        torch.func.jvp(lambda x: f(**dict(tensors, x=x)), (tensors['x'],), (torch.ones_like(tensors['x']),))
    assert not engine.calls


@pytest.mark.parametrize('k', [0, 2, 5], ids=[NAMES[k] for k in (0, 2, 5)])
def test_forward_derivatives_of_backward_passes_are_refused(engine, k):
    name, f, tensors = entry_points()[k]
    first = next(iter(tensors))
    y = f(**dict(tensors, **{first: tensors[first].requires_grad_()}))
    with fwd.dual_level(), pytest.raises(ValueErr, match='forward'):
        torch.autograd.grad(y, tensors[first], fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))
    assert len(engine.calls) == 1


# -------------------------------------------------------------------------------------------------------------- traces
TRACERS = {'jit.trace': lambda f, t: torch.jit.trace(f, t, check_trace=False),
           'make_fx': lambda f, t: make_fx(f)(*t),
           'make_fx before the dispatcher': lambda f, t: make_fx(f, pre_dispatch=True)(*t)}


@pytest.mark.parametrize('tracer', TRACERS)
@pytest.mark.parametrize('k', range(len(NAMES)), ids=NAMES)
def test_traces_are_refused(engine, k, tracer):
    """ A recorded call would be the allocation of its results and nothing else. """
    name, f, tensors = entry_points()[k]
    with pytest.raises(ValueErr, match='recorded'):
        TRACERS[tracer](lambda *t: f(**dict(zip(tensors, t))), tuple(tensors.values()))
    assert not engine.calls
    f(**tensors)
    assert len(engine.calls) == 1


@pytest.mark.parametrize('k', range(len(NAMES)), ids=NAMES)
def test_calls_for_their_shapes_alone_are_refused(engine, k):
    """ results without memory, of tensors that have some """
    name, f, tensors = entry_points()[k]
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(ValueErr, match='recorded'):
        f(**tensors)
    assert not engine.calls


def test_traces_of_differentiated_calls_are_refused(engine):
    name, f, tensors = entry_points()[0]
    with pytest.raises(ValueErr, match='recorded'):
        torch.jit.trace(lambda x: f(**dict(tensors, x=x)), tensors['x'].clone().requires_grad_(), check_trace=False)
    assert not engine.calls


def test_modes_that_only_watch_are_no_traces(engine):
    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    for mode in (Watch(), FlopCounterMode(display=False)):
        for name, f, tensors in entry_points():
            with mode:
                f(**tensors)
    assert len(engine.calls) == 2*len(NAMES)


@pytest.mark.parametrize('name,which', [('grouped_linear', 'bias'), ('causal_conv', 'bias'), ('causal_conv', 'state'), ('causal_conv_grad', 'dlast'),
                                        ('selective_scan', 'D'), ('selective_scan', 'z'), ('selective_scan', 'delta_bias'), ('selective_scan', 'state'),
                                        ('selective_scan_grad', 'dlast')])
def test_a_tensor_without_memory_is_not_an_absent_one(engine, name, which):
    """ What stands for a tensor while a program is being transformed has no address, which the kernels would take for 'not given'. """
    f, tensors = next((f, t) for n, f, t in entry_points() if n == name)
    mode = FakeTensorMode()
    fake = mode.from_tensor(tensors[which])
    with pytest.raises(ValueErr, match='no memory'):
        f(**dict(tensors, **{which: fake}))
    with pytest.raises(ValueErr, match='no memory'):
        torch.func.functionalize(lambda t: f(**dict(tensors, **{which: t})))(tensors[which])
    assert not engine.calls


# --------------------------------------------------------------------------------------------------------------- sizes
BIG = 2**32 + 5      # of which 32 bits keep 5


def test_sizes_that_32_bits_do_not_hold_are_refused(engine):
    """ The descriptors hold sizes in 32 bits.  (Nothing here is ever written, so the memory is never there.) """
    off = torch.arange(2, dtype=torch.int32)
    bf, f = torch.bfloat16, torch.float32
    long, short = torch.empty(BIG, 1, dtype=bf), torch.empty(3, 1, dtype=bf)
    many = torch.zeros(1, dtype=torch.int32).expand(BIG + 1)
    one = torch.zeros(1, 1, 1)
    rows = dict(delta=long, B=long, C=long, D=None, z=None, delta_bias=None)
    calls = {
        'rows': lambda: ops.grouped_linear(long, one.to(bf), None, off),
        'inputs': lambda: ops.grouped_linear(long.view(1, BIG), long.view(1, 1, BIG), None, off),
        'outputs': lambda: ops.grouped_linear(short, long.view(1, BIG, 1), None, off),
        'groups': lambda: ops.grouped_linear(short, one.to(bf).expand(BIG, 1, 1), None, many),
        'rows of a gradient': lambda: ops.grouped_linear_grad(long, None, long, one.to(bf), off),
        'rows of a convolution': lambda: ops.causal_conv(long, one, None, off),
        'channels': lambda: ops.causal_conv(long.view(1, BIG), torch.empty(1, 1, 1).expand(1, BIG, 1), None, off),
        'sequences': lambda: ops.causal_conv(short, one, None, many),
        'policies': lambda: ops.causal_conv(short, one.expand(BIG, 1, 1), None, off, groups=many),
        'taps': lambda: ops.causal_conv(short, one.expand(1, 1, BIG), None, off),
        'sequences of a step': lambda: ops.causal_conv_step(long, torch.empty(BIG, 1, 0, dtype=bf), one, None),
        'rows of a recurrence': lambda: ops.selective_scan(long, A=one, offsets=off, **rows),
        'sequences of a recurrence': lambda: ops.selective_scan(short, A=one, offsets=many, **dict(rows, delta=short, B=short, C=short)),
        'policies of a recurrence': lambda: ops.selective_scan(short, A=one.expand(BIG, 1, 1), offsets=off, groups=many,
                                                               **dict(rows, delta=short, B=short, C=short)),
        'sequences of its step': lambda: ops.selective_scan_step(long, state=torch.empty(1, 1, 1).expand(BIG, 1, 1), A=one, **rows),
    }
    for what, call in calls.items():
        with pytest.raises(ValueErr):
            call()
            pytest.fail(what)
        assert not engine.calls, what
