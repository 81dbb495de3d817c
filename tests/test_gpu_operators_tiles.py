"""
grouped_linear in bfloat16 with every kind of tile (tests/layer_cases.py) against its definition in float64, and that the calls take the tiles
they are meant to.  Tolerances: those of tests/test_gpu_operators.py, with |error| <= n u M + eps / 2 |value|, u = 2^-24, n = inputs + 8 for y,
outputs + 8 for dx and rows + 8 for the weights' and biases' gradients, and for the roundings of dp = dy f'(y), with a nonlinearity, another
(3 eps / 2 + 2 (K + 8) u max M) times the sums over |dy|.
"""
import pytest
import torch

from tests import layer_cases, linear_plan
from tests.test_gpu_operators import offs, rnd

pytestmark = pytest.mark.gpu
T, U, STEP = torch.bfloat16, 2.**-24, 2.**-8


@pytest.fixture(scope='module')
def ops():
    from simurlacra_amd import operators
    return operators


def definition(x, w, b, lengths, nonlin, dy, mag):
    """ y, dx, dw, db group by group, or (mag) the sums of the magnitudes of what is added up in them """
    m = torch.abs if mag else (lambda t: t)
    y, dx, dw, db = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    f = {None: lambda v: v, 'tanh': torch.tanh, 'sigmoid': torch.sigmoid}[nonlin]
    a = 0
    for g, n in enumerate(lengths):
        r = slice(a, a + n)
        a += n
        y[r] = torch.mm(m(x[r]), m(w[g]).t().contiguous()) + m(b[g])
        v = f(torch.mm(x[r], w[g].t().contiguous()) + b[g])
        dp = dy[r]*{None: torch.ones_like(v), 'tanh': 1 - v*v, 'sigmoid': v*(1 - v)}[nonlin]
        if not mag:
            y[r] = v
        dx[r], dw[g], db[g] = torch.mm(m(dp), m(w[g])), torch.mm(m(dp).t().contiguous(), m(x[r])), m(dp).sum(0)
    return dict(y=y, dx=dx, dw=dw, db=db)


def close(name, got, want, M, n, extra=None):
    tol = n*U*M + STEP*want.abs() + 1e-300 + (0. if extra is None else extra)
    worst = ((got.double() - want).abs()/tol).nan_to_num(float('inf')).max()
    assert float(worst) <= 1., f'{name}: {float(worst):.3g} of the tolerance'


@pytest.fixture
def plans(ops, monkeypatch):
    """ the plans of the calls that reach the library """
    from simurlacra_amd.engine import Engine
    seen, call = [], Engine._call

    def _call(self, what, *args):
        if what.startswith('psh_grouped_linear'):
            seen.append((what, linear_plan.plan(args[0]._obj)))
        return call(self, what, *args)
    monkeypatch.setattr(Engine, '_call', _call)
    return seen


@pytest.mark.parametrize('name', layer_cases.CASES)
def test_every_kind_of_tile(ops, plans, name):
    lengths, K, N, shift, nonlin, forward, dx, dw, joint = layer_cases.CASES[name]
    gen = torch.Generator().manual_seed(K + N)
    tail, G, off = 3, len(lengths), offs(lengths)
    R, ld = sum(lengths) + tail, (K + 7)//8*8 + 8
    x = rnd(gen, R, ld, T=T)[:, shift:shift + K]
    w = rnd(gen, G, N, ld, T=T, scale=K**-.5)[:, :, shift:shift + K]
    b, dy = rnd(gen, G, N, T=T), rnd(gen, R, (N + 7)//8*8, T=T)[:, :N]
    y, value = ops._linear_forward(x, w, b, off, nonlin, wide=True)
    got = dict(zip(('dx', 'dw', 'db'), ops.grouped_linear_grad(dy, value, x, w, off, nonlin)))
    assert plans[0][1].forward == forward and (plans[1][1].dx, plans[1][1].dw, plans[1][1].joint) == (dx, dw, joint)
    assert not y[R - tail:].any() and not got['dx'][R - tail:].any()
    wide = [t.double().contiguous() for t in (x, w, b, dy)]
    nl = nonlin
    if nonlin == 'relu':      # the side of zero is the kernel's own: its y for the slopes
        assert torch.equal(y, torch.relu(ops.grouped_linear(x, w, b, off)))
        wide[3], nl = wide[3]*(y > 0), None
    want, M = (definition(*wide[:3], lengths, nl, wide[3], mag) for mag in (False, True))
    if nonlin == 'relu':
        want['y'] = torch.relu(want['y'])
    close('y', y, want['y'], M['y'], K + 8)
    full, off_dp = M, 0.
    if nl is not None:
        full = definition(*wide[:3], lengths, None, wide[3], True)      # sums over |dy| itself
        off_dp = 3*STEP + 2*(K + 8)*U*float(M['y'].max())
    # the gradients together, and one by one, by launches of their own (which may add up in another order: a workgroup's place in the launch
    # decides where its sums begin)
    for j, (k, n) in enumerate((('dx', N + 8), ('dw', max(lengths) + 8), ('db', max(lengths) + 8))):
        alone = ops.grouped_linear_grad(dy, value, x, w, off, nonlin, tuple(i == j for i in range(3)))
        assert not plans[-1][1].joint and [g is not None for g in alone] == [i == j for i in range(3)]
        for g in (got[k], alone[j]):
            close(k, g, want[k], M[k], n, off_dp*full[k])


def test_the_largest_tiles_in_a_graph_against_the_definition(ops, plans):
    """ captured, and replayed with other inputs """
    lengths, K, N, shift, nonlin, forward, dx, dw, joint = layer_cases.CASES['wide']
    gen = torch.Generator().manual_seed(3)
    off, R = offs(lengths), sum(lengths)
    x, w, b, dy = rnd(gen, R, K, T=T), rnd(gen, len(lengths), N, K, T=T, scale=K**-.5), rnd(gen, len(lengths), N, T=T), rnd(gen, R, N, T=T)

    def run():
        return [ops.grouped_linear(x, w, b, off), *ops.grouped_linear_grad(dy, None, x, w, off)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    assert all(p.forward == forward if what == 'psh_grouped_linear' else (p.dx, p.dw, p.joint) == (dx, dw, joint) for what, p in plans) and len(plans) == 4
    for _ in range(3):
        for t in (x, dy):
            t.copy_(rnd(gen, *t.shape, T=T))
        eager = run()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))
    wide = [t.double() for t in (x, w, b, dy)]
    want, M = (definition(*wide[:3], lengths, None, wide[3], mag) for mag in (False, True))
    for k, t, n in zip(('y', 'dx', 'dw', 'db'), out, (K + 8, N + 8, max(lengths) + 8, max(lengths) + 8)):
        close(k, t, want[k], M[k], n)
