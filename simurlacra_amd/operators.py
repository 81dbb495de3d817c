"""
Operators of policies on the GPU, differentiable where training needs it (kernels: csrc/ops_linear.hip and
csrc/ops_memory.hip, C ABI: psh_grouped_linear*, psh_causal_conv*, psh_selective_scan* of include/pysimhip.h).

  grouped_linear                            one layer of a population of networks, each on its own rows
  causal_conv, selective_scan               the recurrence of a policy with memory over whole sequences
  causal_conv_step, selective_scan_step     the same for one step of every sequence, the memory updated in place

Rows are steps.  The rows of a rollout follow one another, and so do the rollouts of a policy: `offsets` (int32, on the GPU,
[n + 1], beginning with 0) cut the rows into groups or sequences, of which any may be empty, and `groups` (int32,
on the GPU, [P + 1]) cut the sequences into the policies' shares.  Their values are not read on the host, so nothing waits
for the GPU; values that do not ascend or that leave the range give meaningless numbers, but no access outside the arrays.  Rows
behind the last offset belong to nobody: they are zero in the results and have zero gradients.

Element types are float64 (what the policies of this package use), float32 and bfloat16.  With bfloat16 rows the products and
sums run in fp32, and each result is rounded once.  Parameters and states of the recurrence are float64 for
float64 rows and float32 for the others.

All calls run on the current stream of the tensors' GPU and are ordered like any other work on it.  They can be captured
into graphs; for gradients inside a capture use the *_grad functions, which autograd's bookkeeping has no part in.  Without
a GPU every call raises: there is no CPU fallback.
"""
import ctypes as C

import torch

from . import _abi as abi
from .engine import get_engine
from .utils.exceptions import ShapeErr, TypeErr, ValueErr

_DTYPES = {torch.float64: abi.DTYPE_F64, torch.float32: abi.DTYPE_F32, torch.bfloat16: abi.DTYPE_BF16}
_NONLINS = {None: 0, 'tanh': 1, 'relu': 2, 'sigmoid': 3}


def wide_dtype(dtype: torch.dtype) -> torch.dtype:
    """ The type of the recurrence's parameters and states for rows of this type. """
    return torch.float64 if dtype == torch.float64 else torch.float32


# --------------------------------------------------------------------------------------------------------- checks
def _rows_arg(name, t, dtype=None, device=None, cols=None, rows=None):
    """ A [rows, cols] tensor whose columns are neighbours (copied if they are not): (tensor, row stride). """
    if not torch.is_tensor(t):
        raise TypeErr(given=t, given_name=name, expected_type=torch.Tensor)
    if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
        raise TypeErr(msg=f'{name} must be of type {"float64, float32 or bfloat16" if dtype is None else dtype}, but is {t.dtype}!')
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueErr(msg=f'{name} must be on {"a GPU" if device is None else device}, but is on {t.device}! There is no CPU fallback.')
    if t.dim() != 2 or (cols is not None and t.shape[1] != cols) or (rows is not None and t.shape[0] != rows):
        raise ShapeErr(msg=f'{name} must have the shape [{"rows" if rows is None else rows}, '
                           f'{"columns" if cols is None else cols}], but has {list(t.shape)}!')
    n, m = t.shape
    if m > 1 and t.stride(1) != 1 or n > 1 and t.stride(0) < m:
        t = t.contiguous()
    return t, (t.stride(0) if n > 1 else m)


def _param(name, t, dtype, device, shape):
    """ A parameter or state of the given shape, contiguous. """
    if not torch.is_tensor(t):
        raise TypeErr(given=t, given_name=name, expected_type=torch.Tensor)
    if t.dtype != dtype:
        raise TypeErr(msg=f'{name} must be of type {dtype}, but is {t.dtype}!')
    if t.device != device:
        raise ValueErr(msg=f'{name} must be on {device}, but is on {t.device}!')
    if tuple(t.shape) != tuple(shape):
        raise ShapeErr(msg=f'{name} must have the shape {list(shape)}, but has {list(t.shape)}!')
    return t.contiguous()


def _offsets(name, t, device):
    if not torch.is_tensor(t):
        raise TypeErr(given=t, given_name=name, expected_type=torch.Tensor)
    if t.dtype != torch.int32:
        raise TypeErr(msg=f'{name} must be of type torch.int32, but is {t.dtype}!')
    if t.device != device:
        raise ValueErr(msg=f'{name} must be on {device}, but is on {t.device}!')
    if t.dim() != 1 or t.shape[0] < 2:
        raise ShapeErr(msg=f'{name} must have one entry more than there are parts (at least two), but has the shape {list(t.shape)}!')
    return t.contiguous()


def _no_grad_args(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueErr(msg=f'{what} updates its state in place and has no gradient: call it under torch.no_grad(), and the '
                           f'form for whole sequences for training!')


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(bytes_, device):
    return torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ > 0 else None


def _size(eng, name, desc):
    n = getattr(eng.lib, name)(C.byref(desc))
    if n < 0:
        raise ValueErr(msg=f'{name}: invalid sizes')
    return int(n)


def _grad_tensor(t, like_dtype):
    """ An incoming gradient as the kernels take it. """
    return None if t is None else t.to(like_dtype).contiguous()


# ------------------------------------------------------------------------------------------------- grouped_linear
def _linear_desc(eng, x, weight, bias, offsets, nonlin):
    x, ld_x = _rows_arg('x', x)
    dev, dt = x.device, x.dtype
    offsets = _offsets('offsets', offsets, dev)
    if nonlin not in _NONLINS:
        raise ValueErr(msg=f'nonlin must be one of {list(_NONLINS)}, but is {nonlin!r}!')
    G, K = offsets.shape[0] - 1, x.shape[1]
    if not torch.is_tensor(weight):
        raise TypeErr(given=weight, given_name='weight', expected_type=torch.Tensor)
    if weight.dim() != 3 or weight.shape[0] != G or weight.shape[2] != K or weight.shape[1] < 1 or K < 1:
        raise ShapeErr(msg=f'weight must have the shape [{G}, outputs, {K}] with at least one input and output, but has {list(weight.shape)}!')
    N = weight.shape[1]
    for name, t in (('weight', weight), ('bias', bias)):
        if t is not None and (t.dtype != dt or t.device != dev):
            raise TypeErr(msg=f'{name} must be of type {dt} on {dev}, but is {t.dtype} on {t.device}!')
    if K > 1 and weight.stride(2) != 1 or N > 1 and weight.stride(1) < K:
        weight = weight.contiguous()
    if bias is not None:
        if tuple(bias.shape) != (G, N):
            raise ShapeErr(msg=f'bias must have the shape {[G, N]}, but has {list(bias.shape)}!')
        if N > 1 and bias.stride(1) != 1:
            bias = bias.contiguous()
    d = abi.PshLinearDesc()
    d.dtype, d.nonlin, d.n_groups, d.rows, d.in_dim, d.out_dim = _DTYPES[dt], _NONLINS[nonlin], G, x.shape[0], K, N
    d.offsets, d.x, d.weight, d.bias = offsets.data_ptr(), x.data_ptr(), weight.data_ptr(), _ptr(bias)
    d.ld_x, d.ld_w, d.stride_w = ld_x, (weight.stride(1) if N > 1 else K), (weight.stride(0) if G > 1 else 0)
    d.stride_b = 0 if bias is None or G == 1 else bias.stride(0)
    d.stream = eng._stream()
    return d, (x, weight, bias, offsets)    # the tensors have to outlive the call


def _engine_of(x, name='x'):
    if not torch.is_tensor(x):
        raise TypeErr(given=x, given_name=name, expected_type=torch.Tensor)
    if not x.is_cuda:
        raise ValueErr(msg=f'{name} must be on a GPU, but is on {x.device}! There is no CPU fallback.')
    return get_engine(x.device.index)


def _linear_forward(x, weight, bias, offsets, nonlin):
    eng = _engine_of(x)
    d, keep = _linear_desc(eng, x, weight, bias, offsets, nonlin)
    y = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype, device=x.device)
    d.y = y.data_ptr()
    eng._call('psh_grouped_linear', C.byref(d))
    del keep
    return y


def grouped_linear_grad(dy, y, x, weight, offsets, nonlin=None, want=(True, True, True)):
    """ The gradients (dx, dweight, dbias) of grouped_linear for the gradient dy of its result y; None where `want` is false.
    y is only read with a nonlinearity (its slope is taken from the value, in y's type). """
    eng = _engine_of(x)
    d, keep = _linear_desc(eng, x, weight, None, offsets, nonlin)
    (G, N, K), R, dev = weight.shape, x.shape[0], x.device
    dy, d.ld_dy = _rows_arg('dy', dy, x.dtype, dev, N, R)
    d.dy = dy.data_ptr()
    if nonlin is not None:
        y = _param('y', y, x.dtype, dev, (R, N))
        d.y = y.data_ptr()
    dx = torch.empty((R, K), dtype=x.dtype, device=dev) if want[0] else None
    dw = torch.empty((G, N, K), dtype=x.dtype, device=dev) if want[1] else None
    db = torch.empty((G, N), dtype=x.dtype, device=dev) if want[2] else None
    d.dx, d.dweight, d.dbias = _ptr(dx), _ptr(dw), _ptr(db)
    d.workspace_bytes = _size(eng, 'psh_grouped_linear_grad_workspace', d)
    space = _workspace(d.workspace_bytes, dev)
    d.workspace = _ptr(space)
    eng._call('psh_grouped_linear_grad', C.byref(d))
    del keep
    return dx, dw, db


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, nonlin):
        y = _linear_forward(x, weight, bias, offsets, nonlin)
        ctx.save_for_backward(x, weight, offsets, y if nonlin is not None else None)
        ctx.nonlin = nonlin
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, offsets, y = ctx.saved_tensors
        return grouped_linear_grad(dy, y, x, weight, offsets, ctx.nonlin, ctx.needs_input_grad[:3]) + (None, None)


def grouped_linear(x, weight, bias, offsets, nonlin: str = None):
    """ y[r] = f(weight[g] @ x[r] + bias[g]) for the rows r of group g, offsets[g] <= r < offsets[g + 1].

    x [R, K]; weight [G, N, K] and bias [G, N] (or None) of x's type, views into a matrix of whole parameter vectors
    included; nonlin None, 'tanh', 'relu' or 'sigmoid'.  Returns y [R, N]. """
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in (x, weight, bias)):
        return _GroupedLinear.apply(x, weight, bias, offsets, nonlin)
    return _linear_forward(x, weight, bias, offsets, nonlin)


# ---------------------------------------------------------------------------------------------------- causal_conv
def _policies(groups, dev, P):
    """ The policies' shares of the sequences, None for one policy. """
    if groups is None:
        if P != 1:
            raise ShapeErr(msg=f'parameters of {P} policies need groups that say which sequences are whose!')
        return None
    groups = _offsets('groups', groups, dev)
    if groups.shape[0] != P + 1:
        raise ShapeErr(msg=f'groups must have {P + 1} entries for {P} policies, but has {groups.shape[0]}!')
    return groups


def _state_arg(name, t, dtype, dev, shape):
    """ A [sequences, ...] state whose sequences may be apart: (tensor, stride). """
    if t is None:
        return None, 0
    if not torch.is_tensor(t):
        raise TypeErr(given=t, given_name=name, expected_type=torch.Tensor)
    if t.dtype != dtype or t.device != dev:
        raise TypeErr(msg=f'{name} must be of type {dtype} on {dev}, but is {t.dtype} on {t.device}!')
    if tuple(t.shape) != tuple(shape):
        raise ShapeErr(msg=f'{name} must have the shape {list(shape)}, but has {list(t.shape)}!')
    size = shape[1]*shape[2]
    if t.numel() and not (t[0].is_contiguous() and (shape[0] == 1 or t.stride(0) >= size)):
        return t.contiguous(), size
    return t, (t.stride(0) if shape[0] > 1 else size)


def _conv_desc(eng, x, weight, bias, offsets, groups, state, silu, step):
    x, ld_x = _rows_arg('x', x)
    dev, dt = x.device, x.dtype
    W = wide_dtype(dt)
    R, D = x.shape
    if not torch.is_tensor(weight) or weight.dim() != 3:
        raise ShapeErr(msg='weight must be a tensor of shape [policies, channels, taps]!')
    P, K = weight.shape[0], weight.shape[2]
    if not 1 <= K <= abi.PSH_MAX_TAPS or P < 1 or D < 1:
        raise ValueErr(msg=f'causal_conv takes 1 to {abi.PSH_MAX_TAPS} taps and at least one policy and channel, but weight is {list(weight.shape)}!')
    weight = _param('weight', weight, W, dev, (P, D, K))
    bias = None if bias is None else _param('bias', bias, W, dev, (P, D))
    groups = _policies(groups, dev, P)
    offsets = None if step else _offsets('offsets', offsets, dev)
    S = R if step else offsets.shape[0] - 1
    d = abi.PshConvDesc()
    d.dtype, d.silu, d.step, d.n_policies, d.n_seqs, d.rows, d.channels, d.taps = _DTYPES[dt], int(bool(silu)), int(step), P, S, R, D, K
    d.offsets, d.groups, d.x, d.weight, d.bias = _ptr(offsets), _ptr(groups), x.data_ptr(), weight.data_ptr(), _ptr(bias)
    d.ld_x = ld_x
    if state is not None:
        state, d.stride_state = _state_arg('state', state, dt, dev, (S, D, K - 1))
        d.state = state.data_ptr()
    d.stream = eng._stream()
    return d, (x, weight, bias, offsets, groups, state), S


def _conv_forward(x, weight, bias, offsets, groups, state, silu):
    eng = _engine_of(x)
    d, keep, S = _conv_desc(eng, x, weight, bias, offsets, groups, state, silu, False)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    last = torch.empty((S, x.shape[1], weight.shape[2] - 1), dtype=x.dtype, device=x.device)
    d.y, d.last, d.stride_last = y.data_ptr(), last.data_ptr(), last.shape[1]*last.shape[2]
    eng._call('psh_causal_conv', C.byref(d))
    del keep
    return y, last


def causal_conv_grad(dy, dlast, x, weight, bias, offsets, groups=None, state=None, silu: bool = True, want=(True,)*4):
    """ The gradients (dx, dweight, dbias, dstate) of causal_conv for those of its results (dlast may be None); None
    where `want` is false. """
    eng = _engine_of(x)
    d, keep, S = _conv_desc(eng, x, weight, bias, offsets, groups, state, silu, False)
    (R, D), (P, _, K), dev = x.shape, weight.shape, x.device
    dy, d.ld_dy = _rows_arg('dy', dy, x.dtype, dev, D, R)
    d.dy = dy.data_ptr()
    if dlast is not None:
        dlast = _param('dlast', dlast, x.dtype, dev, (S, D, K - 1))
        d.dlast = dlast.data_ptr()
    dx = torch.empty((R, D), dtype=x.dtype, device=dev) if want[0] else None
    dw = torch.empty((P, D, K), dtype=weight.dtype, device=dev) if want[1] else None
    db = torch.empty((P, D), dtype=weight.dtype, device=dev) if want[2] else None
    ds = torch.empty((S, D, K - 1), dtype=x.dtype, device=dev) if want[3] else None
    d.dx, d.dweight, d.dbias, d.dstate = _ptr(dx), _ptr(dw), _ptr(db), _ptr(ds)
    d.workspace_bytes = _size(eng, 'psh_causal_conv_grad_workspace', d)
    space = _workspace(d.workspace_bytes, dev)
    d.workspace = _ptr(space)
    eng._call('psh_causal_conv_grad', C.byref(d))
    del keep
    return dx, dw, db, ds


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, offsets, groups, silu):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, offsets, groups)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, offsets, groups, state, silu)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, offsets, groups = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        want = ctx.needs_input_grad[:4]
        return causal_conv_grad(dy, _grad_tensor(dlast, x.dtype), x, weight, bias, offsets, groups, state, ctx.silu,
                                want) + (None, None, None)


def causal_conv(x, weight, bias, offsets, groups=None, state=None, silu: bool = True, return_state: bool = False):
    """ A depthwise convolution along every sequence that looks K - 1 steps back, followed by v sigmoid(v) if `silu`:
    y[t, d] = f(bias[p, d] + sum_k weight[p, d, k] x[t - (K - 1) + k, d]).

    x [R, D]; weight [P, D, K] and bias [P, D] (or None) of policy p, whose sequences `groups` name; state [S, D, K - 1] the inputs
    before each sequence's first step, oldest first (None: zeros).  Returns y [R, D], with return_state also the state
    after each sequence's last step. """
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in (x, weight, bias, state)):
        y, last = _CausalConv.apply(x, weight, bias, state, offsets, groups, silu)
    else:
        y, last = _conv_forward(x, weight, bias, offsets, groups, state, silu)
    return (y, last) if return_state else y


def causal_conv_step(x, state, weight, bias, groups=None, silu: bool = True):
    """ causal_conv for one step of every sequence: x [S, D]; state [S, D, K - 1] is updated in place.  Returns y [S, D]. """
    _no_grad_args('causal_conv_step', *(t for t in (x, state, weight, bias) if torch.is_tensor(t)))
    eng = _engine_of(x)
    if state is None:
        raise TypeErr(given=state, given_name='state', expected_type=torch.Tensor)
    d, keep, S = _conv_desc(eng, x, weight, bias, None, groups, state, silu, True)
    if S and weight.shape[2] > 1 and keep[5] is not state:
        raise ValueErr(msg='state is updated in place: the values of each sequence have to be contiguous!')
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    d.y, d.last, d.stride_last = y.data_ptr(), state.data_ptr(), d.stride_state
    eng._call('psh_causal_conv', C.byref(d))
    del keep
    return y


# ------------------------------------------------------------------------------------------------- selective_scan
def _scan_desc(eng, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, step):
    u, ld_u = _rows_arg('u', u)
    dev, dt = u.device, u.dtype
    W = wide_dtype(dt)
    R, ch = u.shape
    if not torch.is_tensor(A) or A.dim() != 3:
        raise ShapeErr(msg='A must be a tensor of shape [policies, channels, states]!')
    P, N = A.shape[0], A.shape[2]
    if not 1 <= N <= abi.PSH_MAX_MEM_STATES or P < 1 or ch < 1:
        raise ValueErr(msg=f'selective_scan takes 1 to {abi.PSH_MAX_MEM_STATES} states and at least one policy and channel, but A is {list(A.shape)}!')
    delta, ld_delta = _rows_arg('delta', delta, dt, dev, ch, R)
    B, ld_B = _rows_arg('B', B, dt, dev, N, R)
    Cm, ld_C = _rows_arg('C', Cm, dt, dev, N, R)
    A = _param('A', A, W, dev, (P, ch, N))
    D = None if D is None else _param('D', D, W, dev, (P, ch))
    delta_bias = None if delta_bias is None else _param('delta_bias', delta_bias, W, dev, (P, ch))
    groups = _policies(groups, dev, P)
    offsets = None if step else _offsets('offsets', offsets, dev)
    S = R if step else offsets.shape[0] - 1
    d = abi.PshScanDesc()
    d.dtype, d.step, d.n_policies, d.n_seqs, d.rows, d.channels, d.states = _DTYPES[dt], int(step), P, S, R, ch, N
    d.offsets, d.groups = _ptr(offsets), _ptr(groups)
    d.u, d.delta, d.B, d.C = u.data_ptr(), delta.data_ptr(), B.data_ptr(), Cm.data_ptr()
    d.ld_u, d.ld_delta, d.ld_B, d.ld_C = ld_u, ld_delta, ld_B, ld_C
    if z is not None:
        z, d.ld_z = _rows_arg('z', z, dt, dev, ch, R)
        d.z = z.data_ptr()
    d.A, d.D, d.delta_bias = A.data_ptr(), _ptr(D), _ptr(delta_bias)
    if state is not None:
        state, d.stride_state = _state_arg('state', state, W, dev, (S, ch, N))
        d.state = state.data_ptr()
    d.stream = eng._stream()
    return d, (u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state), S


def _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, keep_check):
    eng = _engine_of(u, 'u')
    d, keep, S = _scan_desc(eng, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, False)
    dev = u.device
    y = torch.empty(u.shape, dtype=u.dtype, device=dev)
    last = torch.empty((S,) + tuple(A.shape[1:]), dtype=A.dtype, device=dev)
    d.y, d.last, d.stride_last = y.data_ptr(), last.data_ptr(), A.shape[1]*A.shape[2]
    check = _workspace(_size(eng, 'psh_selective_scan_check', d), dev) if keep_check else None
    d.check = _ptr(check)
    d.workspace_bytes = _size(eng, 'psh_selective_scan_workspace', d)
    space = _workspace(d.workspace_bytes, dev)
    d.workspace = _ptr(space)
    eng._call('psh_selective_scan', C.byref(d))
    del keep
    return y, last, check


def selective_scan_check(u, delta, A, B, C, D, z, delta_bias, offsets, groups=None, state=None):
    """ selective_scan for a gradient taken with selective_scan_grad: (y, last state, stored states). """
    return _scan_forward(u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, True)


def selective_scan_grad(dy, dlast, check, u, delta, A, B, C, D, z, delta_bias, offsets, groups=None, state=None, want=(True,)*9):
    """ The gradients (du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dstate) of selective_scan for those of its results
    (dlast may be None), from the states that selective_scan_check stored; None where `want` is false or there is no
    such input. """
    return _scan_grad(dy, dlast, check, u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, want)


def _scan_grad(dy, dlast, check, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, want):
    eng = _engine_of(u, 'u')
    d, keep, S = _scan_desc(eng, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, False)
    (R, ch), (P, _, N), dev, dt, W = u.shape, A.shape, u.device, u.dtype, A.dtype
    dy, d.ld_dy = _rows_arg('dy', dy, dt, dev, ch, R)
    d.dy = dy.data_ptr()
    if dlast is not None:
        dlast = _param('dlast', dlast, W, dev, (S, ch, N))
        d.dlast = dlast.data_ptr()
    need = _size(eng, 'psh_selective_scan_check', d)
    if check is None or check.dtype != torch.uint8 or check.device != dev or not check.is_contiguous() or check.numel() != need:
        raise ValueErr(msg='check must be the stored states that selective_scan_check returned for the same inputs!')
    d.check = check.data_ptr()

    def out(k, there, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=dev) if want[k] and there else None
    du, ddelta = out(0, True, (R, ch), dt), out(1, True, (R, ch), dt)
    dA, dB, dC = out(2, True, (P, ch, N), W), out(3, True, (R, N), dt), out(4, True, (R, N), dt)
    dD, dz = out(5, D is not None, (P, ch), W), out(6, z is not None, (R, ch), dt)
    dbias, dstate = out(7, delta_bias is not None, (P, ch), W), out(8, state is not None, (S, ch, N), W)
    d.du, d.ddelta, d.dA, d.dB, d.dC, d.dD, d.dz, d.ddelta_bias, d.dstate = (_ptr(t) for t in (du, ddelta, dA, dB, dC, dD, dz, dbias, dstate))
    d.workspace_bytes = _size(eng, 'psh_selective_scan_grad_workspace', d)
    space = _workspace(d.workspace_bytes, dev)
    d.workspace = _ptr(space)
    eng._call('psh_selective_scan_grad', C.byref(d))
    del keep
    return du, ddelta, dA, dB, dC, dD, dz, dbias, dstate


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, Cm, D, z, delta_bias, state, offsets, groups):
        ctx.set_materialize_grads(False)
        y, last, check = _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, True)
        ctx.save_for_backward(u, delta, A, B, Cm, D, z, delta_bias, state, offsets, groups, check)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        u, delta, A, B, Cm, D, z, delta_bias, state, offsets, groups, check = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(u)
        return _scan_grad(dy, _grad_tensor(dlast, A.dtype), check, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state,
                          ctx.needs_input_grad[:9]) + (None, None)


def selective_scan(u, delta, A, B, C, D, z, delta_bias, offsets, groups=None, state=None, return_state: bool = False):
    """ A linear recurrence whose decay and input depend on the step, along every sequence; channel d has N states:

        dt     = softplus(delta[t, d] + delta_bias[p, d])
        h_t[n] = exp(dt A[p, d, n]) h_{t-1}[n] + dt B[t, n] u[t, d]
        y[t,d] = (sum_n C[t, n] h_t[n] + D[p, d] u[t, d]) * z[t, d] sigmoid(z[t, d])

    u, delta, z [R, D]; B, C [R, N]; A [P, D, N], D and delta_bias [P, D] of policy p, whose sequences `groups` name; state [S, D, N]
    before each sequence's first step (None: zeros).  D, z and delta_bias may be None.  Returns y [R, D], with return_state
    also the state after each sequence's last step. """
    args = (u, delta, A, B, C, D, z, delta_bias, state)
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in args):
        y, last = _SelectiveScan.apply(*args, offsets, groups)
    else:
        y, last, _ = _scan_forward(u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, False)
    return (y, last) if return_state else y


def selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, groups=None):
    """ selective_scan for one step of every sequence: u [S, D] and so on; state [S, D, N] is updated in place.  Returns
    y [S, D]. """
    return _scan_step(u, delta, state, A, B, C, D, z, delta_bias, groups)


def _scan_step(u, delta, state, A, B, Cm, D, z, delta_bias, groups):
    _no_grad_args('selective_scan_step', *(t for t in (u, delta, state, A, B, Cm, D, z, delta_bias) if torch.is_tensor(t)))
    eng = _engine_of(u, 'u')
    if state is None:
        raise TypeErr(given=state, given_name='state', expected_type=torch.Tensor)
    d, keep, S = _scan_desc(eng, u, delta, A, B, Cm, D, z, delta_bias, None, groups, state, True)
    if S and keep[10] is not state:
        raise ValueErr(msg='state is updated in place: the values of each sequence have to be contiguous!')
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    d.y, d.last, d.stride_last = y.data_ptr(), state.data_ptr(), d.stride_state
    eng._call('psh_selective_scan', C.byref(d))
    del keep
    return y
