"""
The policy operators the way programs use them: captured into graphs and replayed, on other streams and from several threads, with
offsets that make no sense, sizes beyond 32 bits, nothing at all, and calls that are refused.
"""
import threading

import pytest
import torch

from simurlacra_amd.utils.exceptions import ShapeErr, TypeErr, ValueErr
from tests.test_gpu_operators import IDS, TYPES, offs, rnd, scan_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from simurlacra_amd import operators
    return operators


def everything(ops, T, seed=0, lengths=(70, 0, 300, 33), D=24, N=16, K=40, M=72):
    """ One set of inputs for all operators, and a function that runs all of them: a list of results. """
    gen = torch.Generator().manual_seed(seed)
    W = ops.wide_dtype(T)
    v, off, _ = scan_inputs(gen, ops, T, list(lengths), D, N, None)
    S, R = len(lengths), sum(lengths) + 2
    x, w, b = rnd(gen, R, K, T=T), rnd(gen, S, M, K, T=T, scale=.2), rnd(gen, S, M, T=T)
    dyl, dy, dlast = rnd(gen, R, M, T=T), rnd(gen, R, D, T=T), rnd(gen, S, D, N, T=W)
    cw, cb, cs = rnd(gen, 1, D, 4, T=W), rnd(gen, 1, D, T=W), rnd(gen, S, D, 3, T=T)
    memory = [cs.clone(), v['state'].clone()]
    args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off)

    def run():
        y = ops.grouped_linear(x, w, b, off, 'tanh')
        out = [y, *ops.grouped_linear_grad(dyl, y, x, w, off, 'tanh')]
        out += ops.causal_conv(v['u'], cw, cb, off, state=cs, return_state=True)
        out += ops.causal_conv_grad(dy, cs, v['u'], cw, cb, off, state=cs)
        ys, last, check = ops.selective_scan_check(*args, state=v['state'])
        out += [ys, last, *ops.selective_scan_grad(dy, dlast, check, *args, state=v['state'])]
        for m, src in zip(memory, (cs, v['state'])):
            m.copy_(src)
        out.append(ops.causal_conv_step(v['u'][:S], memory[0], cw, cb))
        out.append(ops.selective_scan_step(v['u'][:S], v['delta'][:S], memory[1], v['A'], v['B'][:S], v['C'][:S], v['D'], v['z'][:S], v['delta_bias']))
        return out + [m.clone() for m in memory]
    return run, [x, w, b, dyl, dy, dlast, cw, cb, cs, *(t for t in v.values())]


@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_captured_and_replayed(ops, T):
    """ Two graphs of the same calls, replayed in turn with new inputs and eager work between: each replay is the eager result,
    bit for bit (no sum depends on the order in which workgroups finish). """
    run, inputs = everything(ops, T)
    other, _ = everything(ops, T, seed=1, lengths=(500, 9))
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(), other()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for f in (run, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = f()
        graphs.append(g)
        outs.append(o)
    gen = torch.Generator().manual_seed(9)
    for turn in range(4):
        for t in inputs[:6]:
            t.copy_(rnd(gen, *t.shape, T=t.dtype))
        want = [[t.clone() for t in f()] for f in (run, other)]
        torch.cuda.synchronize()
        for k in ((0, 1), (1, 0), (0, 0))[turn % 3]:
            graphs[k].replay()
            got = [t.clone() for t in outs[k]]
            torch.mm(torch.randn(64, 64, device='cuda'), torch.randn(64, 64, device='cuda'))
            torch.cuda.synchronize()
            for a, b in zip(got, want[k]):
                assert torch.equal(a.view(torch.uint8), b.contiguous().view(torch.uint8))


def test_captured_gradients_beside_a_live_eager_graph(ops):
    """ The *_grad calls in a capture have nothing to do with an autograd graph that holds the same tensors. """
    gen = torch.Generator().manual_seed(2)
    x, w, off = rnd(gen, 50, 8), rnd(gen, 2, 6, 8), offs([20, 30])
    x.requires_grad_()
    w.requires_grad_()
    y = ops.grouped_linear(x, w, None, off, 'tanh')      # stays alive
    dy = rnd(gen, 50, 6)
    want = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        ops.grouped_linear_grad(dy, y, x, w, off, 'tanh')
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        got = ops.grouped_linear_grad(dy, y, x, w, off, 'tanh')
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    again = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])


def test_other_streams_and_threads(ops):
    """ Calls of several threads on streams of their own at the same time give what they give alone. """
    runs = [everything(ops, T, seed=s, lengths=(200 + 10*s, 3, 40)) for s, T in enumerate(TYPES + TYPES[:1])]
    want = [[t.clone() for t in run()] for run, _ in runs]
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got = runs[k][0]()
            stream.synchronize()
            for a, b in zip(got, want[k]):
                assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        except BaseException as e:   # noqa: BLE001
            errors.append((k, e))
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(runs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize('bad', [[0, 50, 20, 1000000, 103], [5, 5, 5, 5, 5], [0, -7, 30, 2000000000, 60], [100, 80, 60, 40, 20], [0, 0, 0, 0, 0]])
def test_offsets_that_make_no_sense_stay_inside_the_arrays(ops, bad):
    """ Every row number the kernels form is limited to [0, rows] first, so the numbers are meaningless and nothing else happens:
    what lies around the results stays as it was. """
    for T in TYPES:
        run, inputs = everything(ops, T, lengths=(30, 20, 41, 10))
        gen = torch.Generator().manual_seed(3)
        W, R, D, N = ops.wide_dtype(T), 103, 24, 16
        off = torch.tensor(bad, dtype=torch.int32, device='cuda')
        grp = torch.tensor([bad[0], bad[2], bad[4]], dtype=torch.int32, device='cuda')
        v, _, _ = scan_inputs(gen, ops, T, [30, 20, 41, 10], D, N, [2, 2])
        x, w, dy = rnd(gen, R, 40, T=T), rnd(gen, 4, 72, 40, T=T), rnd(gen, R, 72, T=T)
        before = [t.clone() for t in (x, w, dy, *v.values())]
        ops.grouped_linear(x, w, None, off, 'relu')
        ops.grouped_linear_grad(dy, None, x, w, off)
        args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'])
        y, last, check = ops.selective_scan_check(*args)
        ops.selective_scan_grad(y, last, check, *args)
        cw, cs = rnd(gen, 2, D, 4, T=W), rnd(gen, 4, D, 3, T=T)
        yc, cl = ops.causal_conv(v['u'], cw, None, off, grp, cs, return_state=True)
        ops.causal_conv_grad(yc, cl, v['u'], cw, None, off, grp, cs)
        torch.cuda.synchronize()
        for a, b in zip((x, w, dy, *v.values()), before):
            assert torch.equal(a, b)


def test_more_than_two_to_the_31_elements(ops):
    T = torch.bfloat16
    R, K, N = 34_000_100, 64, 64
    x = torch.empty(R, K, dtype=T, device='cuda').normal_()
    gen = torch.Generator().manual_seed(4)
    w, off = rnd(gen, 3, N, K, T=T), torch.tensor([0, 1000, R - 100, R], dtype=torch.int32, device='cuda')
    y = ops.grouped_linear(x, w, None, off)
    for a, b, g in ((0, 1000, 0), (R - 100, R, 2), (R - 300, R - 100, 1)):
        part = torch.tensor([0, b - a], dtype=torch.int32, device='cuda')
        want = x[a:b].float() @ w[g].float().t()
        # two sums of 64 products in another order (64 x 2^-24 of terms of order 8 each), rounded to bf16: off by at most a step
        assert ((y[a:b].float() - want).abs() <= 2**-7*want.abs() + 64*8*8*2**-24).all()
        assert ops.grouped_linear(x[a:b], w[g:g + 1], None, part).shape == (b - a, N)
    dx, dw, _ = ops.grouped_linear_grad(y, None, x, w, off)
    want = y[R - 100:].float().t() @ x[R - 100:].float()
    assert ((dw[2].float() - want).abs() <= 2**-7*want.abs() + 2**-15*want.abs().max()).all()
    want = y[R - 100:].float() @ w[2].float()
    assert ((dx[R - 100:].float() - want).abs() <= 2**-7*want.abs() + 2**-15*want.abs().max()).all()
    del x, y, dx
    # the recurrence: the last sequence of many alone gives what it gives at the end (its pieces are cut alike, so bit for bit)
    D, S, L = 1024, 2200, 1000
    R = S*L
    u, delta, z = (torch.empty(R, D, dtype=T, device='cuda').normal_() for _ in range(3))
    B, C = (torch.empty(R, 4, dtype=T, device='cuda').normal_() for _ in range(2))
    A, skip = -torch.rand(1, D, 4, device='cuda'), torch.ones(1, D, device='cuda')
    off = torch.arange(S + 1, dtype=torch.int32, device='cuda')*L
    y, last = ops.selective_scan(u, delta, A, B, C, skip, z, None, off, return_state=True)
    a = R - L
    few = torch.arange(49, dtype=torch.int32, device='cuda')*L    # 48 sequences of 16 channel blocks: whole ones there too
    first = R - 48*L
    y2, last2 = ops.selective_scan(u[first:], delta[first:], A, B[first:], C[first:], skip, z[first:], None, few, return_state=True)
    assert torch.equal(y[a:], y2[-L:]) and torch.equal(last[-1], last2[-1])
    w = torch.rand(1, D, 4, device='cuda')
    c = ops.causal_conv(u, w, None, off)
    assert torch.equal(c[first:], ops.causal_conv(u[first:], w, None, few))


def test_nothing_at_all(ops):
    for T in TYPES:
        W = ops.wide_dtype(T)
        e = dict(dtype=T, device='cuda')
        off = torch.zeros(3, dtype=torch.int32, device='cuda')
        x, w = torch.empty(0, 5, **e), torch.ones(2, 4, 5, **e)
        assert ops.grouped_linear(x, w, None, off).shape == (0, 4)
        dx, dw, db = ops.grouped_linear_grad(torch.empty(0, 4, **e), None, x, w, off)
        assert dx.shape == (0, 5) and not dw.any() and not db.any()
        state = torch.ones(2, 5, 3, dtype=T, device='cuda')
        cw = torch.ones(1, 5, 4, dtype=W, device='cuda')
        y, last = ops.causal_conv(x, cw, None, off, state=state, return_state=True)
        assert y.shape == (0, 5) and torch.equal(last, state)
        g = ops.causal_conv_grad(x, 2*state, x, cw, None, off, state=state)
        assert not g[1].any() and torch.equal(g[3], 2*state)
        A, B = -torch.ones(1, 5, 6, dtype=W, device='cuda'), torch.empty(0, 6, **e)
        h = torch.randn(2, 5, 6, dtype=W, device='cuda')
        y, last, check = ops.selective_scan_check(x, x, A, B, B, None, None, None, off, state=h)
        assert y.shape == (0, 5) and torch.equal(last, h)
        g = ops.selective_scan_grad(x, 3*h, check, x, x, A, B, B, None, None, None, off, state=h)
        assert not g[2].any() and torch.equal(g[8], 3*h)
        assert ops.causal_conv_step(x, torch.empty(0, 5, 3, **e), cw, None).shape == (0, 5)
        assert ops.selective_scan_step(x, x, torch.empty(0, 5, 6, dtype=W, device='cuda'), A, B, B, None, None, None).shape == (0, 5)


def test_gradients_through_expanded_and_partial_graphs(ops):
    """ sum().backward() hands over an expanded gradient; only some inputs may want one; shared parameters collect both shares """
    gen = torch.Generator().manual_seed(7)
    x, w, off = rnd(gen, 30, 6), rnd(gen, 2, 5, 6).requires_grad_(), offs([10, 20])
    ops.grouped_linear(x, w, None, off).sum().backward()
    want = torch.stack([x[:10].sum(0).expand(5, 6), x[10:].sum(0).expand(5, 6)])
    assert torch.allclose(w.grad, want, rtol=1e-13, atol=1e-13)
    one = rnd(gen, 5, 6).requires_grad_()                  # one weight for both groups, by a stride of zero
    ops.grouped_linear(x, one.expand(2, 5, 6), None, off).sum().backward()
    assert torch.allclose(one.grad, want.sum(0), rtol=1e-13, atol=1e-13)
    v, off, _ = scan_inputs(gen, ops, torch.float64, [12, 5], 3, 2, None, tail=0)
    A = v['A'].clone().requires_grad_()
    y, last = ops.selective_scan(v['u'], v['delta'], A, v['B'], v['C'], None, None, None, off, return_state=True)
    both, = torch.autograd.grad(y.sum() + last.sum(), A, retain_graph=True)
    parts = [torch.autograd.grad(t.sum(), A, retain_graph=True)[0] for t in (y, last)]
    assert torch.allclose(both, parts[0] + parts[1], rtol=1e-12, atol=1e-12)
    with pytest.raises(ValueErr, match='second derivatives'):
        torch.autograd.grad(y.sum(), A, create_graph=True)


def test_refusals(ops):
    gen = torch.Generator().manual_seed(8)
    x, w, off = rnd(gen, 30, 6), rnd(gen, 2, 5, 6), offs([10, 20])
    b = rnd(gen, 2, 5)
    for error, call in [
            (ShapeErr, lambda: ops.grouped_linear(x, w[:1], None, off)), (ShapeErr, lambda: ops.grouped_linear(x[:, :4], w, None, off)),
            (ShapeErr, lambda: ops.grouped_linear(x, w, b[:, :3], off)), (TypeErr, lambda: ops.grouped_linear(x, w.float(), None, off)),
            (TypeErr, lambda: ops.grouped_linear(x.half(), w.half(), None, off)), (TypeErr, lambda: ops.grouped_linear(x, w, None, off.long())),
            (ValueErr, lambda: ops.grouped_linear(x, w, None, off.cpu())), (ValueErr, lambda: ops.grouped_linear(x, w, None, off, 'gelu')),
            (ValueErr, lambda: ops.grouped_linear(x, w.cpu(), None, off)), (ShapeErr, lambda: ops.grouped_linear(x[0], w, None, off)),
            (ShapeErr, lambda: ops.grouped_linear_grad(b, None, x, w, off)), (TypeErr, lambda: ops.grouped_linear_grad(x[:, :5], None, x, w, off, 'tanh'))]:
        with pytest.raises(error):
            call()
    cw, st = rnd(gen, 1, 6, 4), rnd(gen, 2, 6, 3)
    grp = offs([1, 1])
    for error, call in [
            (ShapeErr, lambda: ops.causal_conv(x, cw[:, :5], None, off)), (ValueErr, lambda: ops.causal_conv(x, rnd(gen, 1, 6, 9), None, off)),
            (ShapeErr, lambda: ops.causal_conv(x, cw, None, off, state=st[:1])), (TypeErr, lambda: ops.causal_conv(x, cw, None, off, state=st.float())),
            (TypeErr, lambda: ops.causal_conv(x, cw.float(), None, off)), (ShapeErr, lambda: ops.causal_conv(x, cw.expand(2, 6, 4), None, off)),
            (ShapeErr, lambda: ops.causal_conv(x, cw, None, off, groups=grp)), (TypeErr, lambda: ops.causal_conv_step(x, None, cw, None)),
            (ValueErr, lambda: ops.causal_conv_step(x[:2], st.transpose(1, 2).contiguous().transpose(1, 2), cw, None)),
            (ShapeErr, lambda: ops.causal_conv_step(x, st, cw, None))]:
        with pytest.raises(error):
            call()
    v, off, _ = scan_inputs(gen, ops, torch.float64, [12, 5], 3, 2, None, tail=0)
    args = [v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off]
    for k, bad, error in [(1, v['delta'][:, :2], ShapeErr), (2, v['A'][0], ShapeErr), (2, v['A'].float(), TypeErr), (3, v['B'][:5], ShapeErr), (4, v['u'], ShapeErr),
                          (5, v['D'][0], ShapeErr), (6, v['z'].float(), TypeErr), (7, v['D'].cpu(), ValueErr), (2, rnd(gen, 1, 3, 65), ValueErr), (8, None, TypeErr)]:
        wrong = list(args)
        wrong[k] = bad
        with pytest.raises(error):
            ops.selective_scan(*wrong)
    y, last, check = ops.selective_scan_check(*args)
    for bad in (None, check[:-8], check.float()):
        with pytest.raises(ValueErr):
            ops.selective_scan_grad(y, None, bad, *args)


@pytest.mark.parametrize('nonlin', ['tanh', 'sigmoid'])
def test_slopes_of_bfloat16_layers_where_they_are_flat(ops, nonlin):
    """ A layer's own bfloat16 result is too coarse for its slope (tanh at 3: a result of 1 - 2^-8 and a slope of 2^-7 in steps of half its
    size), so the gradient goes by the value before its rounding. """
    gen = torch.Generator().manual_seed(5)
    R, T = 4000, torch.bfloat16
    x = (torch.rand(R, 1, generator=gen)*6 - 3).to(T).cuda().requires_grad_()
    w, b, off = torch.ones(1, 1, 1, dtype=T, device='cuda'), torch.zeros(1, 1, dtype=T, device='cuda'), offs([R - 1])
    dy = rnd(gen, R, 1, T=T)
    y = ops.grouped_linear(x, w, b, off, nonlin)
    got, = torch.autograd.grad(y, x, dy)
    f = torch.tanh if nonlin == 'tanh' else torch.sigmoid
    v = f(x.detach().double())
    want = dy.double()*(1 - v*v if nonlin == 'tanh' else v*(1 - v))
    want[-1] = 0
    # the gradient before the layer and the result are rounded, 2^-8 each; the slope is at least 1/103 (tanh) or 1/23, and the
    # value's error, a few times 2^-24, twice that in the slope: less than 2^-13 of it
    assert ((got.double() - want).abs() <= (2*2**-8 + 2**-13)*want.abs()).all()
    wide = torch.zeros(R, 1, dtype=torch.float32, device='cuda')
    wide[:] = f(x.detach().float())
    same = ops.grouped_linear_grad(dy, wide, x.detach(), w, off, nonlin)[0]
    assert ((same.double() - want).abs() <= (2*2**-8 + 2**-13)*want.abs()).all()
    with pytest.raises(TypeErr):
        ops.grouped_linear_grad(dy, wide.double(), x.detach(), w, off, nonlin)


@pytest.mark.parametrize('K, N', [(8, 40), (64, 100), (256, 264), (40, 520)])
def test_values_before_their_rounding(ops, K, N):
    """ Every tile shape writes them, rounded they are the results, and rows behind the last group are zero in both. """
    gen = torch.Generator().manual_seed(6)
    for lengths in ([3, 0, 9], [300, 1, 1000], [5000, 4000]):
        R = sum(lengths) + 5
        x, w, b = rnd(gen, R, K, T=torch.bfloat16), rnd(gen, len(lengths), N, K, T=torch.bfloat16, scale=K**-.5), rnd(gen, len(lengths), N, T=torch.bfloat16)
        y, wide = ops._linear_forward(x, w, b, offs(lengths), 'sigmoid', wide=True)
        assert wide.dtype == torch.float32 and torch.equal(wide.to(torch.bfloat16), y) and not wide[-5:].any()
        assert torch.equal(y, ops.grouped_linear(x, w, b, offs(lengths), 'sigmoid'))


@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_states_without_memory(ops, T):
    """ A of minus infinity: exp(delta A) is 0, and neither the steps that fill up a tile nor the joining of pieces make a NaN of it. """
    gen = torch.Generator().manual_seed(10)
    lengths = [1, 33, 1900]
    v, off, _ = scan_inputs(gen, ops, T, lengths, 20, 8, None, tail=0)
    A = v['A'].clone()
    A[:, :5], A[:, 7, 3] = -float('inf'), -float('inf')
    args = (v['u'], v['delta'], A, v['B'], v['C'], None, None, None, off)
    y, last, check = ops.selective_scan_check(*args, state=v['state'])
    dt = torch.nn.functional.softplus(v['delta'].double())
    want = dt*v['u'].double()*(v['B'].double()*v['C'].double()).sum(1, keepdim=True)
    # a product of three and a sum of eight in T's wide type (20 roundings at the most, the step size's few among them), one rounding to T
    e, w = torch.finfo(T).eps/2, torch.finfo(ops.wide_dtype(T)).eps/2
    size = dt*v['u'].double().abs()*(v['B'].double()*v['C'].double()).abs().sum(1, keepdim=True)
    assert ((y.double() - want)[:, :5].abs() <= e*want[:, :5].abs() + 20*w*size[:, :5]).all()
    assert torch.isfinite(y).all() and torch.isfinite(last).all()
    grads = ops.selective_scan_grad(y, last, check, *args, state=v['state'])
    assert all(torch.isfinite(g).all() for g in grads if g is not None)
    assert not grads[8][:, :5].any()


@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_numbers_that_are_none_stay_in_their_sequence(ops, T):
    """ NaNs and infinities of one sequence and one group reach nothing of the others, and those behind the last row nothing at all. """
    gen = torch.Generator().manual_seed(11)
    W, D, N = ops.wide_dtype(T), 24, 16
    lengths = [50, 37, 400, 21]
    R = sum(lengths) + 4
    bad, grp = slice(50, 87), offs([1, 1, 2])
    v, off, _ = scan_inputs(gen, ops, T, lengths, D, N, [1, 1, 2], tail=4)
    cw, cb, cs, dy = rnd(gen, 3, D, 4, T=W), rnd(gen, 3, D, T=W), rnd(gen, 4, D, 3, T=T), rnd(gen, R, D, T=T)
    x, w, b, dyl = rnd(gen, R, 40, T=T), rnd(gen, 4, 72, 40, T=T, scale=.2), rnd(gen, 4, 72, T=T), rnd(gen, R, 72, T=T)
    dlast = rnd(gen, 4, D, N, T=W)

    def run():
        args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'])
        y, last, check = ops.selective_scan_check(*args)
        g = ops.selective_scan_grad(dy, dlast, check, *args)
        yc, lc = ops.causal_conv(v['u'], cw, cb, off, grp, cs, return_state=True)
        gc = ops.causal_conv_grad(dy, None, v['u'], cw, cb, off, grp, cs)
        yl = ops.grouped_linear(x, w, b, off, 'tanh')
        gl = ops.grouped_linear_grad(dyl, yl, x, w, off, 'tanh')
        rows = [y, g[0], g[1], g[3], g[4], yc, gc[0], yl, gl[0]]
        seqs = [last, lc, gc[3], gl[1], gl[2]]
        pols = [g[2], gc[1], gc[2]]
        return ([torch.cat([t[:50], t[87:]]) for t in rows] + [torch.cat([t[:1], t[2:]]) for t in seqs] + [torch.cat([t[:1], t[2:]]) for t in pols])
    want = [t.clone() for t in run()]
    for t in (v['u'], v['delta'], v['B'], v['C'], v['z'], x, dy, dyl):
        t[bad][::3] = float('nan')
        t[bad][1::3] = float('inf')
        t[-4:] = float('nan')
    for got, ref in zip(run(), want):
        assert torch.equal(got, ref)


def test_the_largest_tiles_in_a_graph(ops):
    """ Tiles that need more LDS than a kernel has without being asked: captured, replayed and against the eager call. """
    gen = torch.Generator().manual_seed(12)
    T, R, K, N = torch.bfloat16, 32768, 200, 768
    off = offs([20000, 0, R - 20007])
    x, w, dy = rnd(gen, R, K, T=T), rnd(gen, 3, N, K, T=T, scale=.1), rnd(gen, R, N, T=T)

    def run():
        return [ops.grouped_linear(x, w, None, off), *ops.grouped_linear_grad(dy, None, x, w, off)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for _ in range(3):
        x.copy_(rnd(gen, R, K, T=T))
        want = run()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_gradients_against_differences(ops):
    """ Central differences of every output over every input in fp64.  A step of 1e-6 leaves the third derivatives' 1e-12 and the
    outputs' rounding, a few hundred times 2^-53 of numbers of order 10, over 2e-6: well below 1e-6. """
    gen = torch.Generator().manual_seed(13)
    off, grp = offs([3, 0, 5, 1]), offs([1, 3])
    x, w, b = (t.requires_grad_() for t in (rnd(gen, 11, 3), rnd(gen, 4, 2, 3), rnd(gen, 4, 2)))
    for nonlin in (None, 'tanh', 'sigmoid'):
        assert torch.autograd.gradcheck(lambda *t: ops.grouped_linear(*t, off, nonlin), (x, w, b), eps=1e-6, atol=1e-6, rtol=1e-6)
    cw, cb, cs = (t.requires_grad_() for t in (rnd(gen, 2, 3, 4), rnd(gen, 2, 3), rnd(gen, 4, 3, 3)))
    assert torch.autograd.gradcheck(lambda a, ww, bb, ss: ops.causal_conv(a, ww, bb, off, grp, ss, return_state=True), (x, cw, cb, cs), eps=1e-6, atol=1e-6, rtol=1e-6)
    v, off, grp = scan_inputs(gen, ops, torch.float64, [3, 0, 5, 1], 3, 5, [1, 3], tail=2)
    names = ('u', 'delta', 'A', 'B', 'C', 'D', 'z', 'delta_bias', 'state')
    args = [v[n].detach().clone().requires_grad_() for n in names]
    assert torch.autograd.gradcheck(lambda *t: ops.selective_scan(*t[:8], off, grp, t[8], return_state=True), args, eps=1e-6, atol=1e-6, rtol=1e-6)


def test_autograd_in_a_capture_is_refused(ops):
    gen = torch.Generator().manual_seed(14)
    x, w, off = rnd(gen, 50, 8), rnd(gen, 2, 6, 8).requires_grad_(), offs([20, 30])
    cw = rnd(gen, 1, 8, 4).requires_grad_()
    v, soff, _ = scan_inputs(gen, ops, torch.float64, [40, 10], 8, 4, None, tail=0)
    A = v['A'].clone().requires_grad_()
    with torch.no_grad():
        want = ops.grouped_linear(x, w, None, off)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for call in (lambda: ops.grouped_linear(x, w, None, off), lambda: ops.causal_conv(x, cw, None, off),
                     lambda: ops.selective_scan(v['u'], v['delta'], A, v['B'], v['C'], None, None, None, soff)):
            with pytest.raises(ValueErr, match='captured'):
                call()
        with torch.no_grad():
            y = ops.grouped_linear(x, w, None, off)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
