"""
The policy operators write their results, their stored states and their scratch memory, each of exactly the size that they ask for, and
nothing beside them: for offsets that are in order and for such that make no sense.
"""
import contextlib
import math

import pytest
import torch

from tests import operators_ref as ref
from tests.test_gpu_operators import IDS, TYPES, close, offs, rnd, scan_inputs

pytestmark = pytest.mark.gpu
FENCE, MARK = 1 << 16, 0xA5


@pytest.fixture(scope='module')
def ops():
    from simurlacra_amd import operators
    return operators


class Fences:
    """ Gives out memory between stretches of marked bytes. """

    def __init__(self):
        self.given = []

    def empty(self, shape, dtype, device):
        n = math.prod(shape)*dtype.itemsize
        room = torch.full((2*FENCE + n,), MARK, dtype=torch.uint8, device=device)
        self.given.append((room, n))
        return room[FENCE:FENCE + n].view(dtype).view(shape) if n else room[:0].view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        assert self.given
        for room, n in self.given:
            around = torch.cat([room[:FENCE], room[FENCE + n:]])
            assert bool((around == MARK).all()), (n, torch.nonzero(around != MARK)[:4].flatten().tolist())

    @contextlib.contextmanager
    def around(self, monkeypatch):
        """ what the operators allocate while this lasts """
        def new_empty(t, *shape):
            return self.empty(shape, t.dtype, t.device)

        def empty(*shape, dtype, device):
            return self.empty(shape[0] if isinstance(shape[0], tuple) else shape, dtype, device)
        with monkeypatch.context() as m:
            m.setattr(torch.Tensor, 'new_empty', new_empty)
            m.setattr(torch, 'empty', empty)
            yield


BAD = [[0, 50, 20, 1000000, 103], [5, 5, 5, 5, 5], [0, -7, 30, 2000000000, 60], [100, 80, 60, 40, 20], [0, 0, 0, 0, 0], [0, 103, 0, 103, 0]]


def memory_calls(ops, v, off, grp, x, cw, cs, dy, dlast):
    """ every call of the memory operators, its results in a list """
    args = (v['u'], v['delta'], v['A'], v['B'], v['C'], v['D'], v['z'], v['delta_bias'], off, grp, v['state'])
    y, last, check = ops.selective_scan_check(*args)
    out = [y, last, *ops.selective_scan_grad(dy, dlast, check, *args)]
    out += ops.causal_conv(x, cw, None, off, grp, cs, return_state=True)
    return out + [g for g in ops.causal_conv_grad(dy, cs, x, cw, None, off, grp, cs)]


@pytest.mark.parametrize('bad', BAD + [None], ids=str)
@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_nothing_is_written_beside_the_results(ops, monkeypatch, T, bad):
    """ 103 rows whole, and 24 times as many, where sequences are cut into pieces and sums into segments """
    gen = torch.Generator().manual_seed(3)
    W, D, N = ops.wide_dtype(T), 24, 16
    for scale in (1, 24):
        lengths = [30*scale, 20*scale, 41*scale, 10*scale]
        R = sum(lengths) + 2
        v, off, grp = scan_inputs(gen, ops, T, lengths, D, N, [2, 2])
        if bad is not None:
            off = torch.tensor([min(o*scale, 2**31 - 1) for o in bad], dtype=torch.int32, device='cuda')
            grp = torch.tensor([bad[0], bad[2], bad[4]], dtype=torch.int32, device='cuda')
        x, w, b, dy = rnd(gen, R, 40, T=T), rnd(gen, 4, 72, 40, T=T), rnd(gen, 4, 72, T=T), rnd(gen, R, 72, T=T)
        memory = (v['u'], rnd(gen, 2, D, 4, T=W), rnd(gen, 4, D, 3, T=T), rnd(gen, R, D, T=T), rnd(gen, 4, D, N, T=W))

        def run():
            y, value = ops._linear_forward(x, w, b, off, 'tanh', wide=True)
            out = [y, value, *ops.grouped_linear_grad(dy, value, x, w, off, 'tanh')]
            return out + memory_calls(ops, v, off, grp, *memory)
        fences = Fences()
        with fences.around(monkeypatch):
            got = run()
        fences.check()
        if bad is None:      # in order: and everything that is a result has been written
            want = run()
            assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


@pytest.mark.parametrize('K, N', [(72, 200), (264, 136), (256, 520), (129, 520)])
@pytest.mark.parametrize('lengths', [[9000, 0, 130, 17000], [200]*40, 'bad'])
def test_nothing_is_written_beside_the_results_of_large_tiles(ops, monkeypatch, K, N, lengths):
    gen = torch.Generator().manual_seed(K)
    T = torch.bfloat16
    off = torch.tensor([0, 20000, 7000, 2000000000, 26000], dtype=torch.int32, device='cuda') if lengths == 'bad' else offs(lengths)
    R, G = 26133 if lengths == 'bad' else sum(lengths) + 3, off.shape[0] - 1
    x, w, b, dy = rnd(gen, R, K, T=T), rnd(gen, G, N, K, T=T, scale=.1), rnd(gen, G, N, T=T), rnd(gen, R, N, T=T)

    def run():
        return [*ops._linear_forward(x, w, b, off, 'sigmoid', wide=True), *ops.grouped_linear_grad(dy, None, x, w, off)]
    fences = Fences()
    with fences.around(monkeypatch):
        got = run()
    fences.check()
    if lengths != 'bad':
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_the_fences_see_a_byte():
    fences = Fences()
    t = fences.empty((3, 5), torch.float32, 'cuda')
    t.zero_()
    fences.check()
    for at in (FENCE - 1, FENCE + t.numel()*4):
        fences.given[0][0][at] = 0
        with pytest.raises(AssertionError):
            fences.check()
        fences.given[0][0][at] = MARK


@pytest.mark.parametrize('T', TYPES, ids=IDS)
def test_few_large_groups_among_many_small_ones(ops, monkeypatch, T):
    """ The sums of the large ones are cut into pieces, which alone have scratch memory: against the definition, and between fences. """
    gen = torch.Generator().manual_seed(8)
    lengths, K, N = [2]*150 + [1000] + [0, 3]*80 + [700, 129, 128], 40, 72
    off, R, G = offs(lengths), sum(lengths) + 2, len(lengths)
    x, w, dy = rnd(gen, R, K, T=T), rnd(gen, G, N, K, T=T, scale=K**-.5), rnd(gen, R, N, T=T)
    want, M = (ref.linear(x, w, None, off, None, dy, mag=m) for m in (False, True))
    fences = Fences()
    with fences.around(monkeypatch):
        got = ops.grouped_linear_grad(dy, None, x, w, off)
    fences.check()
    assert sum(n for _, n in fences.given) < 2*sum(t.numel()*t.element_size() for t in got)
    for name, g, n in zip(('dx', 'dw', 'db'), got, (N + 8, max(lengths) + 8, max(lengths) + 8)):
        close(name, g, want[name], M[name], n, T)
