"""
The policy operators on the GPU against their definitions in float64 (tests/operators_ref.py).

Tolerances.  u is the unit roundoff of the sums (2^-53 for float64 rows, 2^-24 for the others), M the sum of the magnitudes
that make up a result, n the number of roundings on the longest chain to it; results are rounded once to the rows' type (half a
step, eps / 2, of their value).  So |error| <= n u M + eps / 2 |value|, with n from the sizes:
  grouped_linear   n = K + 8 for y (each product and sum rounds once; the nonlinearities have slopes of at most 1 and
                   are within a few ulp), and N + 8, rows + 8 for the gradients.  dp = dy f'(y) uses the rounded y and is itself
                   rounded to the rows' type: for tanh |d(1 - y^2)| <= 2 |y| eps / 2, sigmoid less, so dp is off by at
                   most (3 eps / 2 + 2 (K + 8) u max M) |dy|, the second part from y's own error: added, times the sums over |dy|.
  causal_conv      n = K + 12, times the rows for the parameters' gradients.
  selective_scan   a step's decay is off by (4 + 3 |dt A|) u relatively (product, scaling, exponential); a chain passes through at
                   most L steps with 3 roundings of their own each, forward and back; the sums over states, channels and
                   (parameters) rows, 40 for the element-wise functions.
"""
import pytest
import torch

from tests import operators_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float64, torch.float32, torch.bfloat16]
IDS = ['f64', 'f32', 'bf16']


@pytest.fixture(scope='module')
def ops():
    from simurlacra_amd import operators
    return operators


def unit(T):
    return 2.**-53 if T == torch.float64 else 2.**-24


def half_step(T):
    return torch.finfo(T).eps/2


def close(name, got, want, M, n, T, extra=None):
    """ |got - want| <= n u M + eps / 2 |want| (+ extra); T is the result's type """
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    if not got.numel():
        return
    tol = n*unit(T)*M + half_step(T)*want.abs() + 1e-300
    if extra is not None:
        tol = tol + extra
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f'{name}: {int(bad.sum())} of {bad.numel()} values off, worst '
                           f'{float(((got - want).abs()/tol).nan_to_num(float("inf")).max()):.3g} of the tolerance, first at '
                           f'{torch.nonzero(bad)[0].tolist()}')


def offs(lengths, dev='cuda'):
    o = [0]
    for n in lengths:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int32, device=dev)


def rnd(gen, *shape, T=torch.float64, scale=1.):
    return (torch.randn(*shape, generator=gen, dtype=torch.float64)*scale).to(T).cuda()


# ------------------------------------------------------------------------------------------------- grouped_linear
LINEAR = [
    # lengths of the groups, inputs, outputs
    ([1], 1, 1), ([0, 1, 0], 3, 2), ([5, 0, 17, 64, 65], 6, 64), ([0, 0], 4, 4), ([130, 1, 0, 63], 64, 65),
    ([7]*9, 33, 129), ([300, 20], 129, 31), ([2]*70, 8, 8), ([700], 16, 200), ([1, 2, 3, 4], 257, 16),
]


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('nonlin', [None, 'tanh', 'relu', 'sigmoid'])
@pytest.mark.parametrize('lengths,K,N', LINEAR)
def test_grouped_linear(ops, T, nonlin, lengths, K, N):
    gen = torch.Generator().manual_seed(len(lengths)*1000 + K)
    tail = 3
    G, R = len(lengths), sum(lengths) + tail
    off = offs(lengths)
    params = rnd(gen, G, N*K + N + 5, T=T, scale=K**-.5)          # layers are views into rows of whole parameter vectors
    w, b = params[:, 3:3 + N*K].view(G, N, K), params[:, 3 + N*K:3 + N*K + N]
    x, dy = rnd(gen, R, K, T=T), rnd(gen, R, N, T=T)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.grouped_linear(*leaves, off, nonlin)
    got = torch.autograd.grad(y, leaves, dy)
    want, M = (ref.linear(x, w, b, off, nonlin, dy, mag=m) for m in (False, True))
    eps = half_step(T)
    close('y', y, want['y'], M['y'], K + 8, T)
    assert not y[R - tail:].any() and not got[0][R - tail:].any()
    if nonlin == 'relu':     # the side of zero is the kernel's own: take its y for the slopes
        dyr = dy*(y.detach() > 0)
        want, M = (ref.linear(x, w, b, off, None, dyr, mag=m) for m in (False, True))
    full = ref.linear(x, w, b, off, None, dy, mag=True)           # sums over |dy| itself
    off_dp = 0. if nonlin in (None, 'relu') else 3*eps + 2*(K + 8)*unit(T)*float(M['y'].max())
    for name, g, n in zip(('dx', 'dw', 'db'), got, (N + 8, max(lengths) + 8, max(lengths) + 8)):
        close(name, g, want[name], M[name], n, T, off_dp*full[name])


@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_grouped_linear_strides_and_unwanted_gradients(ops, T):
    gen = torch.Generator().manual_seed(5)
    lengths, K, N = [9, 0, 40], 12, 20
    off, R = offs(lengths), 49
    big = rnd(gen, R, K + 7, T=T)
    for x in (big[:, 3:3 + K], rnd(gen, K, R, T=T).t(), big[:, :K], rnd(gen, 1, K, T=T).expand(R, K)):
        w, dy = rnd(gen, len(lengths), K, N, T=T).transpose(1, 2), rnd(gen, N, R, T=T).t()
        y = ops.grouped_linear(x, w, None, off, None)
        want, M = (ref.linear(x, w, None, off, None, dy, mag=m) for m in (False, True))
        close('y', y, want['y'], M['y'], K + 8, T)
        for want_these in ((True, False, False), (False, True, False), (False, False, True)):
            got = ops.grouped_linear_grad(dy, None, x, w, off, None, want_these)
            assert [g is not None for g in got] == list(want_these)
            for name, g, n in zip(('dx', 'dw', 'db'), got, (N + 8, 48, 48)):
                if g is not None:
                    close(name, g, want[name], M[name], n, T)


def test_grouped_linear_keeps_what_is_not_finite_in_its_row(ops):
    """ A NaN or an infinity in a row, or in a group's weights, reaches nothing outside that row, or group. """
    gen = torch.Generator().manual_seed(6)
    for T in TYPES:
        lengths, K, N = [10, 20, 0, 30], 24, 40
        off = offs(lengths)
        x, w, dy = rnd(gen, 62, K, T=T), rnd(gen, 4, N, K, T=T), rnd(gen, 62, N, T=T)
        clean = ops.grouped_linear(x, w, None, off)
        gclean = ops.grouped_linear_grad(dy, None, x, w, off)
        x2, w2, dy2 = x.clone(), w.clone(), dy.clone()
        x2[4, 3], x2[61, 0], w2[1, 2, 5], dy2[60, 1], x2[60, 2] = float('nan'), float('nan'), float('inf'), float('nan'), float('inf')
        y = ops.grouped_linear(x2, w2, None, off)
        same = torch.ones(62, dtype=torch.bool)
        same[4] = False
        same[10:30] = False
        assert torch.equal(y[same], clean[same]) and y[4].isnan().all() and not y[60:].any()
        dx, dw, db = ops.grouped_linear_grad(dy2, None, x2, w, off)
        assert torch.equal(dx, gclean[0]) and torch.equal(dw[1:], gclean[1][1:]) and torch.equal(db, gclean[2])
        assert dw[0, :, 3].isnan().all() and not dw[0].isnan()[:, :3].any()


# ---------------------------------------------------------------------------------------------------- causal_conv
CONV = [
    # lengths of the sequences, channels, taps, policies' shares of the sequences
    ([1], 1, 1, None), ([0, 1, 2, 3], 5, 4, None), ([40, 0, 17], 64, 4, [1, 2]), ([200], 24, 2, None), ([3]*20, 130, 8, [5, 0, 15]),
    ([70, 1, 33], 16, 3, [0, 2, 1]), ([0], 4, 4, None), ([600], 8, 5, None), ([35, 64], 256, 6, None), ([129], 72, 7, None),
]


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('carry,silu', [(True, True), (False, False), (False, True)])
@pytest.mark.parametrize('lengths,D,K,groups', CONV)
def test_causal_conv(ops, T, carry, silu, lengths, D, K, groups):
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    W = ops.wide_dtype(T)
    tail, S, P = 2, len(lengths), len(groups) if groups else 1
    R, off = sum(lengths) + tail, offs(lengths)
    grp = offs(groups) if groups else None
    x, dy = rnd(gen, R, D, T=T), rnd(gen, R, D, T=T)
    w, b = rnd(gen, P, D, K, T=W, scale=.5), rnd(gen, P, D, T=W)
    state = rnd(gen, S, D, K - 1, T=T) if carry else None
    dlast = rnd(gen, S, D, K - 1, T=T)
    leaves = [t.detach().requires_grad_() for t in (x, w, b) + ((state,) if carry else ())]
    y, last = ops.causal_conv(*leaves[:3], off, groups=grp, state=leaves[3] if carry else None, silu=silu, return_state=True)
    got = torch.autograd.grad((y, last), leaves, (dy, dlast))
    want, M = (ref.conv(x, w, b, off, grp, state, silu, dy, dlast, mag=m) for m in (False, True))
    close('y', y, want['y'], M['y'], K + 12, T)
    assert torch.equal(last.cpu().double(), want['last'])
    assert not y[R - tail:].any() and not got[0][R - tail:].any()
    n = K + 12
    close('dx', got[0], want['dx'], M['dx'], 2*n, T)
    # sums over the rows of a policy, wide results
    many = n + max(sum(lengths), 1)
    close('dw', got[1], want['dw'], M['dw'], many, W)
    close('db', got[2], want['db'], M['db'], many, W)
    if carry:
        close('dstate', got[3], want['dstate'], M['dstate'], 2*n, T)


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('S,D,K,groups', [(1, 1, 1, None), (1, 128, 4, None), (37, 65, 3, [10, 0, 27]), (300, 16, 8, None)])
def test_causal_conv_step_is_the_sequence_form(ops, T, S, D, K, groups):
    """ Steps one by one and the sequence form apply the same sums in the same order: equal bit for bit, rows and states. """
    gen = torch.Generator().manual_seed(S)
    W, L, P = ops.wide_dtype(T), 6, len(groups) if groups else 1
    grp = offs(groups) if groups else None
    x = rnd(gen, S, L, D, T=T)
    w, b = rnd(gen, P, D, K, T=W, scale=.5), rnd(gen, P, D, T=W)
    room = rnd(gen, S, D*(K - 1) + 5, T=T)                        # the states are slices of longer memory vectors
    state = room[:, 2:2 + D*(K - 1)].view(S, D, K - 1) if K > 1 else rnd(gen, S, D, 0, T=T)
    first, around = state.clone(), room.clone()
    want, last = ops.causal_conv(x.reshape(S*L, D), w, b, offs([L]*S), groups=grp, state=first, return_state=True)
    got = torch.stack([ops.causal_conv_step(x[:, t], state, w, b, groups=grp) for t in range(L)], 1)
    assert torch.equal(got.reshape(S*L, D), want) and torch.equal(state, last)
    assert torch.equal(room[:, :2], around[:, :2]) and torch.equal(room[:, 2 + D*(K - 1):], around[:, 2 + D*(K - 1):])


# ------------------------------------------------------------------------------------------------- selective_scan
SCAN = [
    # lengths, channels, states, policies' shares
    ([1], 1, 1, None), ([0, 1, 2], 3, 4, None), ([40, 0, 17, 16, 33], 64, 16, [1, 2, 0, 2]), ([100], 70, 16, None),
    ([5]*12, 20, 8, [4, 8]), ([33, 1], 17, 24, None), ([48], 9, 64, None), ([0], 4, 16, None), ([31, 32, 8, 7], 130, 12, [0, 1, 3]),
    ([20, 30], 33, 33, None), ([18], 65, 3, None),
]


def scan_inputs(gen, ops, T, lengths, D, N, groups, tail=2, gate=True, carry=True):
    W = ops.wide_dtype(T)
    S, P, R = len(lengths), len(groups) if groups else 1, sum(lengths) + tail
    low = rnd(gen, R, D + 2*N + 4, T=T)
    v = dict(u=rnd(gen, R, D, T=T), delta=low[:, 4:4 + D], A=-torch.rand(P, D, N, generator=gen, dtype=torch.float64).to(W).cuda()*4,
             B=low[:, 4 + D:4 + D + N], C=low[:, 4 + D + N:], D=rnd(gen, P, D, T=W), z=rnd(gen, R, D, T=T) if gate else None,
             delta_bias=rnd(gen, P, D, T=W) - 2, state=rnd(gen, S, D, N, T=W) if carry else None)
    return v, offs(lengths), offs(groups) if groups else None


def roundings(v, lengths, N, D):
    raw = v['delta'].double() + (v['delta_bias'].double().amax() if v['delta_bias'] is not None else 0)
    dtA = float(torch.nn.functional.softplus(raw).max()*v['A'].abs().max()) if raw.numel() else 0.
    return max(list(lengths) + [1])*(4 + 3*dtA + 3)*2 + N + 40


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('gate,carry', [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize('lengths,D,N,groups', SCAN)
def test_selective_scan(ops, T, gate, carry, lengths, D, N, groups):
    gen = torch.Generator().manual_seed(sum(lengths) + D + N)
    W = ops.wide_dtype(T)
    v, off, grp = scan_inputs(gen, ops, T, lengths, D, N, groups, gate=gate, carry=carry)
    if not gate:
        v['D'] = v['delta_bias'] = None
    R, S = v['u'].shape[0], len(lengths)
    dy, dlast = rnd(gen, R, D, T=T), rnd(gen, S, D, N, T=W)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    arg = {k: leaves.get(k) for k in v}
    state = arg.pop('state')
    y, last = ops.selective_scan(**arg, offsets=off, groups=grp, state=state, return_state=True)
    got = dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))))
    args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'], dy, dlast)
    want, M = (ref.scan(*args, mag=m) for m in (False, True))
    n = roundings(v, lengths, N, D)
    close('y', y, want['y'], M['y'], n, T)
    close('last', last, want['last'], M['last'], n, W)
    assert not y[R - 2:].any()
    for k in ('u', 'delta', 'z', 'B', 'C'):
        if k in got:
            assert not got[k][R - 2:].any(), k
            close('d' + k, got[k], want['d' + k], M['d' + k], 2*n + D, T)
    many = 2*n + max(sum(lengths), 1)
    for k, name in (('A', 'dA'), ('D', 'dD'), ('delta_bias', 'dbias')):
        if k in got:
            close(name, got[k], want[name], M[name], many, W)
    if carry:
        close('dstate', got['state'], want['dstate'], M['dstate'], 2*n, W)
    # the forward call without a gradient to prepare gives the same numbers
    with torch.no_grad():
        y2, last2 = ops.selective_scan(**{k: None if t is None else t.detach() for k, t in arg.items()}, offsets=off, groups=grp,
                                       state=v['state'], return_state=True)
    assert torch.equal(y, y2) and torch.equal(last, last2)


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('S,D,N,groups', [(1, 1, 1, None), (1, 128, 16, None), (37, 65, 12, [10, 0, 27]), (50, 16, 64, None), (9, 20, 5, None)])
def test_selective_scan_steps_follow_the_sequence(ops, T, S, D, N, groups):
    gen = torch.Generator().manual_seed(S + N)
    L, W = 5, ops.wide_dtype(T)
    v, off, grp = scan_inputs(gen, ops, T, [L]*S, D, N, groups, tail=0)
    args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'])
    want, M = (ref.scan(*args, mag=m) for m in (False, True))
    room = rnd(gen, S, D*N + 3, T=W)
    state = room[:, :D*N].view(S, D, N)
    state.copy_(v['state'])
    around = room.clone()
    step = {k: v[k].reshape(S, L, -1) for k in ('u', 'delta', 'B', 'C', 'z')}
    ys = [ops.selective_scan_step(step['u'][:, t], step['delta'][:, t], state, v['A'], step['B'][:, t], step['C'][:, t], v['D'],
                                  step['z'][:, t], v['delta_bias'], groups=grp) for t in range(L)]
    n = roundings(v, [L], N, D)
    close('y', torch.stack(ys, 1).reshape(S*L, D), want['y'], M['y'], n, T)
    close('state', state, want['last'], M['last'], n, W)
    assert torch.equal(room[:, D*N:], around[:, D*N:])


def test_selective_scan_far_values(ops):
    """ Step sizes from far below to far above what a type resolves, decays of 0 and of everything. """
    gen = torch.Generator().manual_seed(3)
    for T in (torch.float64, torch.float32):
        v, off, grp = scan_inputs(gen, ops, T, [24, 9], 8, 4, None, tail=0)
        v['delta'] = (torch.linspace(-60, 40, 33, dtype=torch.float64)[:, None] + torch.arange(8)).to(T).cuda()
        v['A'][:, :, 0] = 0.
        v['A'][:, :, 1] = -1e4
        v['delta_bias'] = None
        args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], None, off, None, v['state'])
        want, M = (ref.scan(*args, mag=m) for m in (False, True))
        y, last = ops.selective_scan(*args[:9], state=v['state'], return_state=True)
        # a decay of e^-x is off by 3 x u e^-x at most, and x e^-x < 0.4: the |dt A| of the chain counts as at most 1
        n = 24*(4 + 3 + 3)*2 + 44
        close('y', y, want['y'], M['y'], n, T)
        close('last', last, want['last'], M['last'], n, T)


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('lengths,K,N,shift', [
    # rows and sizes of the large tiles: whole and partial ones of every dimension, aligned and not
    ([9000, 0, 130, 17000], 72, 200, 0), ([12800, 12800], 264, 136, 0), ([20000, 5001], 100, 129, 0), ([16000], 256, 328, 1), ([6000, 127, 4001], 129, 520, 0),
    ([8192, 8193], 512, 264, 0), ([200]*40, 136, 1032, 0)])
def test_grouped_linear_large(ops, T, lengths, K, N, shift):
    """ as above, elements off their 16-byte places by `shift` """
    gen = torch.Generator().manual_seed(K)
    off, R, G = offs(lengths), sum(lengths) + 2, len(lengths)
    x, dy = rnd(gen, R, K + 8, T=T)[:, shift:shift + K], rnd(gen, R, N, T=T)
    w, b = rnd(gen, G, N, K + 8, T=T, scale=K**-.5)[:, :, shift:shift + K], rnd(gen, G, N, T=T)
    y = ops.grouped_linear(x, w, b, off)
    got = ops.grouped_linear_grad(dy, None, x, w, off)
    want, M = (ref.linear(x, w, b, off, None, dy, mag=m) for m in (False, True))
    close('y', y, want['y'], M['y'], K + 8, T)
    # a sum over n rows that is cut into pieces has fewer roundings than n on any chain
    for name, g, n in zip(('dx', 'dw', 'db'), got, (N + 8, max(lengths) + 8, max(lengths) + 8)):
        close(name, g, want[name], M[name], n, T)
    again = ops.grouped_linear_grad(dy, None, x, w, off)
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and torch.equal(y, ops.grouped_linear(x, w, b, off))


@pytest.mark.parametrize('T', TYPES, ids=IDS)
@pytest.mark.parametrize('lengths,D,N,groups', [([1500, 0, 700, 3], 40, 16, None), ([4000], 70, 5, None), ([900, 1, 64, 65, 1000], 12, 40, [1, 0, 4]),
                                                ([130]*9, 200, 16, [3, 6]), ([3 + i % 90 for i in range(400)], 24, 16, None)])
def test_long_sequences(ops, T, lengths, D, N, groups):
    """ The recurrence cut into pieces and joined, and the convolution over many runs of rows """
    gen = torch.Generator().manual_seed(sum(lengths))
    W, K = ops.wide_dtype(T), 4
    v, off, grp = scan_inputs(gen, ops, T, lengths, D, N, groups)
    S, R, P = len(lengths), v['u'].shape[0], len(groups) if groups else 1
    dy, dlast = rnd(gen, R, D, T=T), rnd(gen, S, D, N, T=W)
    args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'])
    y, last, check = ops.selective_scan_check(*args)
    got = dict(zip(('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'bias', 'state'), ops.selective_scan_grad(dy, dlast, check, *args)))
    want, M = (ref.scan(*args, dy, dlast, mag=m) for m in (False, True))
    n = roundings(v, lengths, N, D)
    close('y', y, want['y'], M['y'], n, T)
    close('last', last, want['last'], M['last'], n, W)
    for k in ('u', 'delta', 'z', 'B', 'C'):
        close('d' + k, got[k], want['d' + k], M['d' + k], 2*n + D, T)
    for k in ('A', 'D', 'bias'):
        close('d' + k, got[k], want['d' + k], M['d' + k], 2*n + sum(lengths), W)
    close('dstate', got['state'], want['dstate'], M['dstate'], 2*n, W)
    x, cy, cs = rnd(gen, R, D, T=T), rnd(gen, R, D, T=T), rnd(gen, S, D, K - 1, T=T)
    w, b = rnd(gen, P, D, K, T=W, scale=.5), rnd(gen, P, D, T=W)
    g = ops.causal_conv_grad(cy, cs, x, w, b, off, grp, cs)
    want, M = (ref.conv(x, w, b, off, grp, cs, True, cy, cs, mag=m) for m in (False, True))
    for name, t, k, T_ in zip(('dx', 'dw', 'db', 'dstate'), g, (2*(K + 12), K + 12 + sum(lengths), K + 12 + sum(lengths), 2*(K + 12)), (T, W, W, T)):
        close(name, t, want[name], M[name], k, T_)
    close('conv', ops.causal_conv(x, w, b, off, grp, cs), want['y'], M['y'], K + 12, T)
