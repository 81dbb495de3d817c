"""
What torch keeps track of around the policy operators, on the GPU: states that change in place, traces, forward derivatives.
"""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from simurlacra_amd.utils.exceptions import ValueErr
from tests.test_gpu_operators import offs, rnd, scan_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from simurlacra_amd import operators
    return operators


def test_a_state_that_a_backward_pass_needs_is_not_advanced_unnoticed(ops):
    gen = torch.Generator().manual_seed(1)
    S, D, K, N = 5, 12, 4, 8
    x, w, st = rnd(gen, S, D), rnd(gen, 1, D, K), rnd(gen, S, D, K - 1)
    leaf = w.clone().requires_grad_()
    want, = torch.autograd.grad(ops.causal_conv(x, leaf, None, offs([1]*S), state=st).sum(), leaf)
    y = ops.causal_conv(x, leaf, None, offs([1]*S), state=st)
    kept = st.clone()
    with torch.no_grad():
        ops.causal_conv_step(x, kept, w, None)        # of another tensor: nothing happens to this one
    assert torch.equal(torch.autograd.grad(y.sum(), leaf, retain_graph=True)[0], want)
    with torch.no_grad():
        ops.causal_conv_step(x, st, w, None)
    assert torch.equal(st, kept)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y.sum(), leaf)
    v, off, _ = scan_inputs(gen, ops, torch.float64, [1]*S, D, N, None, tail=0)
    h = v.pop('state')
    product = h*torch.ones_like(h).requires_grad_()
    ops.selective_scan_step(state=h, **v)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        product.sum().backward()


def test_traces_and_forward_derivatives_are_refused(ops):
    gen = torch.Generator().manual_seed(2)
    x, w, off = rnd(gen, 30, 6), rnd(gen, 2, 5, 6), offs([10, 20])
    with pytest.raises(ValueErr, match='recorded'):
        torch.jit.trace(lambda t: ops.grouped_linear(t, w, None, off), x, check_trace=False)
    with fwd.dual_level(), pytest.raises(ValueErr, match='forward'):
        ops.grouped_linear(x, fwd.make_dual(w, w), None, off)
    assert ops.grouped_linear(x, w, None, off).isfinite().all()


def test_more_rows_than_can_be_counted_are_refused(ops):
    """ (2^32 + 5 rows of two bytes: memory that nobody touches) """
    x = torch.empty(2**32 + 5, 1, dtype=torch.bfloat16, device='cuda')
    w = torch.ones(1, 1, 1, dtype=torch.bfloat16, device='cuda')
    with pytest.raises(ValueErr, match='can count'):
        ops.grouped_linear(x, w, None, offs([5]))
    with pytest.raises(ValueErr, match='can count'):
        ops.causal_conv_step(x, x.view(-1, 1, 1)[:, :, :0], torch.ones(1, 1, 1, device='cuda'), None)


@pytest.mark.parametrize('name', ['grouped_linear', 'causal_conv', 'selective_scan', 'causal_conv_step', 'selective_scan_step'])
def test_compiled_functions_call_the_operators_between_their_graphs(ops, name):
    """ torch.compile leaves the calls as they are, differentiated ones too, and sees what the steps change """
    gen = torch.Generator().manual_seed(3)
    S, D, N = 6, 8, 4
    off = offs([1]*S)
    x, w, st, cw = rnd(gen, S, D), rnd(gen, S, 5, D), rnd(gen, S, D, 3), rnd(gen, 1, D, 4)
    v, _, _ = scan_inputs(gen, ops, torch.float64, [1]*S, D, N, None, tail=0)
    h = v.pop('state')
    rest = {k: t for k, t in v.items() if k != 'u'}
    calls = {'grouped_linear': lambda x, s: ops.grouped_linear(2*x, w, None, off, 'tanh') + 1,
             'causal_conv': lambda x, s: ops.causal_conv(2*x, cw, None, off, state=s) + 1,
             'selective_scan': lambda x, s: ops.selective_scan(2*x, **rest, offsets=off, state=s) + 1,
             'causal_conv_step': lambda x, s: ops.causal_conv_step(2*x, s, cw, None) + s.sum(),
             'selective_scan_step': lambda x, s: ops.selective_scan_step(2*x, state=s, **rest) + s.sum()}
    f, state = calls[name], h if 'scan' in name else st
    torch._dynamo.reset()
    for backend in ('eager', 'aot_eager'):
        compiled = torch.compile(f, backend=backend)
        for train in (False, True) if 'step' not in name else (False,):
            for turn in range(3):
                a, b = (x + turn).requires_grad_(train), (x + turn).requires_grad_(train)
                s, t = state.clone(), state.clone()
                want, got = f(a, s), compiled(b, t)
                assert torch.equal(want, got) and torch.equal(s, t)
                if train:
                    assert torch.equal(*(torch.autograd.grad(y.sum(), q)[0] for y, q in ((want, a), (got, b))))
    torch._dynamo.reset()
