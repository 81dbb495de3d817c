"""
What torch keeps track of around the policy operators: saved tensors, derivatives, traces.  On the CPU, with an engine whose calls do
nothing: whatever a call returns is empty memory, and the tests are about what is refused and noticed.
"""
import pytest
import torch

from simurlacra_amd import operators as ops
from simurlacra_amd.engine import load_library


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
