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
sums run in fp32, and each result is rounded once; with a nonlinearity, grouped_linear's gradient also rounds dy f'(y) to
bfloat16 before the products that read it.  Parameters and states of the recurrence are float64 for float64 rows and float32 for the others.

All calls run on the current stream of the tensors' GPU and are ordered like any other work on it.  They can be captured
into graphs; for gradients inside a capture use the *_grad functions, which autograd's bookkeeping has no part in (a call that autograd
would differentiate is refused there).  Without a GPU every call raises: there is no CPU fallback.

Torch does not see into the calls.  The single steps tell it that they have changed their state, so that a backward pass that needs the state as it
was raises; torch.compile leaves the calls as they are; recording them (torch.jit.trace, make_fx) and forward differentiation are refused.
"""
import ctypes as C

import torch
import torch.autograd.forward_ad as _forward

from . import _abi as abi
from .engine import get_engine
from .utils.exceptions import ShapeErr, TypeErr, ValueErr

_DTYPES = {torch.float64: abi.DTYPE_F64, torch.float32: abi.DTYPE_F32, torch.bfloat16: abi.DTYPE_BF16}
_NONLINS = {None: 0, 'tanh': 1, 'relu': 2, 'sigmoid': 3}


def wide_dtype(dtype: torch.dtype) -> torch.dtype:
    """ The type of the recurrence's parameters and states for rows of this type. """
    return torch.float64 if dtype == torch.float64 else torch.float32


# --------------------------------------------------------------------------------------------------------- checks
# (These run before every call, and a small call takes a few microseconds on the GPU: each check is one expression on the
# common path, and what is wrong is only worked out once something is.)
_Tensor = torch.Tensor
_MOST = 2**31 - 1    # what the descriptors' sizes hold (ctypes would keep the low bits of more)


def _refuse(name, t, dtype, device, shape):
    """ Raises for the first thing about t that is not as the call wants it (None in shape: any size). """
    if not isinstance(t, _Tensor):
        raise TypeErr(given=t, given_name=name, expected_type=_Tensor)
    if t.dtype not in _DTYPES or (dtype is not None and t.dtype != dtype):
        raise TypeErr(msg=f'{name} must be of type {"float64, float32 or bfloat16" if dtype is None else dtype}, but is {t.dtype}!')
    if not t.is_cuda and device is None:
        raise ValueErr(msg=f'{name} must be on a GPU, but is on {t.device}! There is no CPU fallback.')
    if device is not None and t.device != device:
        raise ValueErr(msg=f'{name} must be on {device}, but is on {t.device}!')
    raise ShapeErr(msg=f'{name} must have the shape [{", ".join("any" if n is None else str(n) for n in shape)}], but has {list(t.shape)}!')


def _too_large(name, n):
    raise ValueErr(msg=f'{name} has a size of {n}, more than the 2^31 - 1 that the operators can count!')


def _rows_arg(name, t, dtype, device, rows, cols):
    """ A [rows, cols] tensor whose columns are neighbours (copied if they are not): (tensor, row stride). """
    if not isinstance(t, _Tensor) or t.dtype != dtype or t.device != device or t.shape != (rows, cols):
        _refuse(name, t, dtype, device, (rows, cols))
    ld, step = t.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        t = t.contiguous()
        ld = cols
    return t, (ld if rows > 1 else cols)


def _first_rows_arg(name, t):
    """ The same for the tensor that decides about type, device and size, and the engine of its GPU. """
    if not isinstance(t, _Tensor) or t.dtype not in _DTYPES or not t.is_cuda or t.dim() != 2:
        _refuse(name, t, None, None, (None, None))
    rows, cols = t.shape
    if rows > _MOST or cols > _MOST:
        _too_large(name, max(rows, cols))
    ld, step = t.stride()
    if (step != 1 and cols > 1) or (ld < cols and rows > 1):
        t = t.contiguous()
        ld = cols
    device = t.device
    return t, (ld if rows > 1 else cols), rows, cols, t.dtype, device, get_engine(device.index)


def _param(name, t, dtype, device, shape):
    """ A parameter or state of the given shape, contiguous. """
    if not isinstance(t, _Tensor) or t.dtype != dtype or t.device != device or t.shape != shape:
        _refuse(name, t, dtype, device, shape)
    return t.contiguous()


def _offsets(name, t, device):
    if not isinstance(t, _Tensor):
        raise TypeErr(given=t, given_name=name, expected_type=_Tensor)
    if t.dtype != torch.int32:
        raise TypeErr(msg=f'{name} must be of type torch.int32, but is {t.dtype}!')
    if t.device != device:
        raise ValueErr(msg=f'{name} must be on {device}, but is on {t.device}!')
    shape = t.shape
    if len(shape) != 1 or shape[0] < 2:
        raise ShapeErr(msg=f'{name} must have one entry more than there are parts (at least two), but has the shape {list(shape)}!')
    if shape[0] > _MOST:
        _too_large(name, shape[0])
    return t.contiguous()


def _any_requires_grad(*tensors):
    for t in tensors:
        if isinstance(t, _Tensor) and t.requires_grad:
            return True
    return False


_is_tracing, _modes, _function_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack


def _recorded():
    """ Whether torch is recording: by jit.trace, by make_fx in one of the two places where it listens, or with tensors that have no memory. """
    modes = torch._C._TorchDispatchModeKey
    return (_is_tracing() or any(torch._C._get_dispatch_mode(m) is not None for m in (modes.PROXY, modes.FAKE))
            or torch._C._dispatch_tls_is_dispatch_key_included(torch._C.DispatchKey.PreDispatch))


def _seen_by_torch(*tensors):
    """ The kernels run past torch, which sees the tensors that come out and nothing of how they came about.  What it can only do with
    operations that it sees is refused: a recorded call would be empty memory whenever it is played back, and a tangent of forward
    differentiation would be dropped and the derivative read as zero. """
    if (_is_tracing() or _modes() or _function_modes()) and _recorded():
        raise ValueErr(msg='the policy operators cannot be recorded (torch.jit.trace, make_fx, FakeTensorMode): torch does not see what they do!')
    if _forward._current_level >= 0:
        for t in tensors:
            if isinstance(t, _Tensor) and _forward.unpack_dual(t).tangent is not None:
                raise ValueErr(msg='the policy operators have no forward derivatives!')


def _no_grad_args(what, *tensors):
    if torch.is_grad_enabled() and _any_requires_grad(*tensors):
        raise ValueErr(msg=f'{what} updates its state in place and has no gradient: call it under torch.no_grad(), and the '
                           f'form for whole sequences for training!')


def _ptr(t):
    """ The address of a tensor that need not be there, of which a null pointer tells the library (an empty tensor has none either). """
    if t is None:
        return None
    at = t.data_ptr()
    if at == 0 and t.numel():   # it stands for a tensor in a program that is being transformed
        raise ValueErr(msg=f'the policy operators need tensors that lie in memory, but {type(t).__name__} of shape {list(t.shape)} has no memory!')
    return at


def _size(eng, name, desc):
    n = getattr(eng.lib, name)(C.byref(desc))
    if n < 0:
        raise ValueErr(msg=f'{name}: invalid sizes')
    return n


def _workspace(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device) if n > 0 else None


def _give_workspace(eng, desc, name, like):
    """ The scratch memory of a call, on the GPU of `like`, written into its descriptor; it has to outlive the call. """
    n = _size(eng, name, desc)
    if n == 0:
        return None
    space = like.new_empty(-(-n//like.element_size()))   # (new_empty of plain sizes takes half the time of torch.empty with type and device)
    desc.workspace, desc.workspace_bytes = space.data_ptr(), n
    return space


def _advanced(state):
    """ The kernel has written the state past torch, whose count of its changes tells a backward pass that saved it. """
    torch.autograd.graph.increment_version(state)


def _first_derivative_only():
    if torch.is_grad_enabled():   # as it is in a backward pass with create_graph=True
        raise ValueErr(msg='the policy operators have no second derivatives!')


def _autograd(*tensors):
    """ Whether a call of these tensors is to be differentiated.  A backward pass in a capture waits for the streams of every autograd graph
    that its leaves are in, and where one of them lives outside the capture the process ends; so such a call is refused here. """
    if not (torch.is_grad_enabled() and _any_requires_grad(*tensors)):
        return False
    if torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        raise ValueErr(msg='an operator cannot be differentiated by autograd while it is captured into a graph: call it under '
                           'torch.no_grad(), and its *_grad function for the gradients!')
    return True


def _grad_tensor(t, like_dtype):
    """ An incoming gradient as the kernels take it. """
    return None if t is None else t.to(like_dtype).contiguous()


# ------------------------------------------------------------------------------------------------- grouped_linear
def _linear_desc(x, weight, bias, offsets, nonlin):
    x, ld_x, R, K, dt, dev, eng = _first_rows_arg('x', x)
    offsets = _offsets('offsets', offsets, dev)
    if nonlin not in _NONLINS:
        raise ValueErr(msg=f'nonlin must be one of {list(_NONLINS)}, but is {nonlin!r}!')
    G = offsets.shape[0] - 1
    if not isinstance(weight, _Tensor) or weight.dtype != dt or weight.device != dev or weight.dim() != 3:
        _refuse('weight', weight, dt, dev, (G, None, K))
    groups, N, cols = weight.shape
    if groups != G or cols != K or N < 1 or K < 1:
        raise ShapeErr(msg=f'weight must have the shape [{G}, outputs, {K}] with at least one input and output, but has {list(weight.shape)}!')
    if N > _MOST:
        _too_large('weight', N)
    stride_w, ld_w, step = weight.stride()
    if (step != 1 and K > 1) or (ld_w < K and N > 1):
        weight = weight.contiguous()
        stride_w, ld_w = N*K, K
    stride_b, b = 0, None
    if bias is not None:
        if not isinstance(bias, _Tensor) or bias.dtype != dt or bias.device != dev or bias.shape != (G, N):
            _refuse('bias', bias, dt, dev, (G, N))
        stride_b, step = bias.stride()
        if step != 1 and N > 1:
            bias = bias.contiguous()
            stride_b = N
        b = _ptr(bias)
    d = abi.PshLinearDesc(_DTYPES[dt], _NONLINS[nonlin], G, R, K, N, offsets.data_ptr(), x.data_ptr(), weight.data_ptr(), b, None, None, ld_x,
                          ld_w if N > 1 else K, stride_w if G > 1 else 0, stride_b if G > 1 else 0)
    d.stream = eng._stream()
    return eng, d, (x, weight, bias, offsets), R, K, G, N, dt, dev    # the tensors have to outlive the call


def _linear_forward(x, weight, bias, offsets, nonlin, wide=False):
    """ The layer's results, and with `wide` also what the gradient takes the nonlinearity's slope from: the results
    before their rounding where that makes a difference. """
    eng, d, keep, R, K, G, N, dt, dev = _linear_desc(x, weight, bias, offsets, nonlin)
    y = x.new_empty(R, N)
    d.y = y.data_ptr()
    value = y
    if wide and dt == torch.bfloat16 and nonlin in ('tanh', 'sigmoid'):
        value = torch.empty((R, N), dtype=torch.float32, device=dev)
        d.y_wide = value.data_ptr()
    eng._call('psh_grouped_linear', C.byref(d))
    del keep
    return (y, value) if wide else y


def grouped_linear_grad(dy, y, x, weight, offsets, nonlin=None, want=(True, True, True)):
    """ The gradients (dx, dweight, dbias) of grouped_linear for the gradient dy of its result y; None where `want` is false.
    y is only read with a nonlinearity, whose slope is taken from the value: of bfloat16 results, whose rounding is felt where a
    nonlinearity is flat, the values may be given in float32. """
    _seen_by_torch(dy, y, x, weight)
    eng, d, keep, R, K, G, N, dt, dev = _linear_desc(x, weight, None, offsets, nonlin)
    dy, d.ld_dy = _rows_arg('dy', dy, dt, dev, R, N)
    d.dy = dy.data_ptr()
    if nonlin is not None:
        wide = dt == torch.bfloat16 and isinstance(y, _Tensor) and y.dtype == torch.float32
        y = _param('y', y, torch.float32 if wide else dt, dev, (R, N))
        if wide:
            d.y_wide = _ptr(y)
        else:
            d.y = _ptr(y)
    dx = dw = db = None
    if want[0]:
        dx = x.new_empty(R, K)
        d.dx = dx.data_ptr()
    if want[1]:
        dw = x.new_empty(G, N, K)
        d.dweight = dw.data_ptr()
    if want[2]:
        db = x.new_empty(G, N)
        d.dbias = db.data_ptr()
    space = _give_workspace(eng, d, 'psh_grouped_linear_grad_workspace', x)
    eng._call('psh_grouped_linear_grad', C.byref(d))
    del keep, space
    return dx, dw, db


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, offsets, nonlin):
        y, value = _linear_forward(x, weight, bias, offsets, nonlin, wide=True)
        ctx.save_for_backward(x, weight, offsets, value if nonlin is not None else None)
        ctx.nonlin = nonlin
        return y

    @staticmethod
    def backward(ctx, dy):
        _first_derivative_only()
        x, weight, offsets, y = ctx.saved_tensors
        return grouped_linear_grad(dy, y, x, weight, offsets, ctx.nonlin, ctx.needs_input_grad[:3]) + (None, None)


def grouped_linear(x, weight, bias, offsets, nonlin: str = None):
    """ y[r] = f(weight[g] @ x[r] + bias[g]) for the rows r of group g, offsets[g] <= r < offsets[g + 1].

    x [R, K]; weight [G, N, K] and bias [G, N] (or None) of x's type, views into a matrix of whole parameter vectors
    included; nonlin None, 'tanh', 'relu' or 'sigmoid'.  Returns y [R, N]. """
    _seen_by_torch(x, weight, bias)
    if _autograd(x, weight, bias):
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
    if not isinstance(t, _Tensor):
        raise TypeErr(given=t, given_name=name, expected_type=_Tensor)
    if t.dtype != dtype or t.device != dev:
        raise TypeErr(msg=f'{name} must be of type {dtype} on {dev}, but is {t.dtype} on {t.device}!')
    if t.shape != shape:
        raise ShapeErr(msg=f'{name} must have the shape {list(shape)}, but has {list(t.shape)}!')
    size = shape[1]*shape[2]
    apart, line, step = t.stride()
    if (step != 1 and shape[2] > 1) or (line != shape[2] and shape[1] > 1) or (apart < size and shape[0] > 1):
        if size:
            return t.contiguous(), size
    return t, (apart if shape[0] > 1 else size)


def _conv_desc(x, weight, bias, offsets, groups, state, silu, step):
    x, ld_x, R, D, dt, dev, eng = _first_rows_arg('x', x)
    W = wide_dtype(dt)
    if not isinstance(weight, _Tensor) or weight.dim() != 3:
        raise ShapeErr(msg='weight must be a tensor of shape [policies, channels, taps]!')
    P, K = weight.shape[0], weight.shape[2]
    if not 1 <= K <= abi.PSH_MAX_TAPS or P < 1 or D < 1:
        raise ValueErr(msg=f'causal_conv takes 1 to {abi.PSH_MAX_TAPS} taps and at least one policy and channel, but weight is {list(weight.shape)}!')
    if P > _MOST:
        _too_large('weight', P)
    weight = _param('weight', weight, W, dev, (P, D, K))
    bias = None if bias is None else _param('bias', bias, W, dev, (P, D))
    groups = _policies(groups, dev, P)
    offsets = None if step else _offsets('offsets', offsets, dev)
    S = R if step else offsets.shape[0] - 1
    d = abi.PshConvDesc(_DTYPES[dt], 1 if silu else 0, 1 if step else 0, P, S, R, D, K, _ptr(offsets), _ptr(groups), x.data_ptr(), weight.data_ptr(),
                        _ptr(bias))
    d.ld_x = ld_x
    stride = 0
    if state is not None:
        state, stride = _state_arg('state', state, dt, dev, (S, D, K - 1))
        d.state, d.stride_state = _ptr(state), stride
    d.stream = eng._stream()
    return eng, d, (x, weight, bias, offsets, groups, state, stride), S, R, D, P, K, dt, dev


def _conv_forward(x, weight, bias, offsets, groups, state, silu):
    eng, d, keep, S, R, D, P, K, dt, dev = _conv_desc(x, weight, bias, offsets, groups, state, silu, False)
    y = x.new_empty(R, D)
    last = x.new_empty(S, D, K - 1)
    d.y, d.last, d.stride_last = y.data_ptr(), last.data_ptr(), D*(K - 1)
    eng._call('psh_causal_conv', C.byref(d))
    del keep
    return y, last


def causal_conv_grad(dy, dlast, x, weight, bias, offsets, groups=None, state=None, silu: bool = True, want=(True,)*4):
    """ The gradients (dx, dweight, dbias, dstate) of causal_conv for those of its results (dlast may be None); None
    where `want` is false. """
    _seen_by_torch(dy, dlast, x, weight, bias, state)
    eng, d, keep, S, R, D, P, K, dt, dev = _conv_desc(x, weight, bias, offsets, groups, state, silu, False)
    dy, d.ld_dy = _rows_arg('dy', dy, dt, dev, R, D)
    d.dy = dy.data_ptr()
    if dlast is not None:
        dlast = _param('dlast', dlast, dt, dev, (S, D, K - 1))
        d.dlast = _ptr(dlast)
    dx = x.new_empty(R, D) if want[0] else None
    dw = weight.new_empty(P, D, K) if want[1] else None
    db = weight.new_empty(P, D) if want[2] else None
    ds = x.new_empty(S, D, K - 1) if want[3] else None
    d.dx, d.dweight, d.dbias, d.dstate = _ptr(dx), _ptr(dw), _ptr(db), _ptr(ds)
    space = _give_workspace(eng, d, 'psh_causal_conv_grad_workspace', x)
    eng._call('psh_causal_conv_grad', C.byref(d))
    del keep, space
    return dx, dw, db, ds


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, offsets, groups, silu):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, offsets, groups)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, offsets, groups, state, silu)

    @staticmethod
    def backward(ctx, dy, dlast):
        _first_derivative_only()
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
    _seen_by_torch(x, weight, bias, state)
    if _autograd(x, weight, bias, state):
        y, last = _CausalConv.apply(x, weight, bias, state, offsets, groups, silu)
    else:
        y, last = _conv_forward(x, weight, bias, offsets, groups, state, silu)
    return (y, last) if return_state else y


def causal_conv_step(x, state, weight, bias, groups=None, silu: bool = True):
    """ causal_conv for one step of every sequence: x [S, D]; state [S, D, K - 1] is updated in place.  Returns y [S, D]. """
    _seen_by_torch(x, state, weight, bias)
    _no_grad_args('causal_conv_step', x, state, weight, bias)
    if state is None:
        raise TypeErr(given=state, given_name='state', expected_type=_Tensor)
    eng, d, keep, S, R, D, P, K, dt, dev = _conv_desc(x, weight, bias, None, groups, state, silu, True)
    if S and K > 1 and keep[5] is not state:
        raise ValueErr(msg='state is updated in place: the values of each sequence have to be contiguous!')
    y, stride = x.new_empty(R, D), keep[6]
    d.y, d.last, d.stride_last = y.data_ptr(), state.data_ptr(), stride
    eng._call('psh_causal_conv', C.byref(d))
    _advanced(state)
    del keep
    return y


# ------------------------------------------------------------------------------------------------- selective_scan
def _scan_desc(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, step):
    u, ld_u, R, ch, dt, dev, eng = _first_rows_arg('u', u)
    W = wide_dtype(dt)
    if not isinstance(A, _Tensor) or A.dim() != 3:
        raise ShapeErr(msg='A must be a tensor of shape [policies, channels, states]!')
    P, _, N = A.shape
    if not 1 <= N <= abi.PSH_MAX_MEM_STATES or P < 1 or ch < 1:
        raise ValueErr(msg=f'selective_scan takes 1 to {abi.PSH_MAX_MEM_STATES} states and at least one policy and channel, but A is {list(A.shape)}!')
    if P > _MOST:
        _too_large('A', P)
    delta, ld_delta = _rows_arg('delta', delta, dt, dev, R, ch)
    B, ld_B = _rows_arg('B', B, dt, dev, R, N)
    Cm, ld_C = _rows_arg('C', Cm, dt, dev, R, N)
    ld_z = 0
    if z is not None:
        z, ld_z = _rows_arg('z', z, dt, dev, R, ch)
    A = _param('A', A, W, dev, (P, ch, N))
    D = None if D is None else _param('D', D, W, dev, (P, ch))
    delta_bias = None if delta_bias is None else _param('delta_bias', delta_bias, W, dev, (P, ch))
    groups = _policies(groups, dev, P)
    offsets = None if step else _offsets('offsets', offsets, dev)
    S = R if step else offsets.shape[0] - 1
    stride = 0
    if state is not None:
        state, stride = _state_arg('state', state, W, dev, (S, ch, N))
    d = abi.PshScanDesc(_DTYPES[dt], 1 if step else 0, P, S, R, ch, N, 0, _ptr(offsets), _ptr(groups), u.data_ptr(), delta.data_ptr(), _ptr(z), B.data_ptr(),
                        Cm.data_ptr(), A.data_ptr(), _ptr(D), _ptr(delta_bias), _ptr(state), None, None, ld_u, ld_delta, ld_z, ld_B, ld_C, stride)
    d.stream = eng._stream()
    return eng, d, (u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, stride), S, R, ch, P, N, dt, W, dev


def _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, keep_check):
    eng, d, keep, S, R, ch, P, N, dt, W, dev = _scan_desc(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, False)
    y = u.new_empty(R, ch)
    last = A.new_empty(S, ch, N)
    d.y, d.last, d.stride_last = y.data_ptr(), last.data_ptr(), ch*N
    check = None
    if keep_check:
        check = _workspace(_size(eng, 'psh_selective_scan_check', d), dev)
        d.check = check.data_ptr()
    space = _give_workspace(eng, d, 'psh_selective_scan_workspace', u)
    eng._call('psh_selective_scan', C.byref(d))
    del keep, space
    return y, last, check


def selective_scan_check(u, delta, A, B, C, D, z, delta_bias, offsets, groups=None, state=None):
    """ selective_scan for a gradient taken with selective_scan_grad: (y, last state, stored states). """
    _seen_by_torch(u, delta, A, B, C, D, z, delta_bias, state)
    return _scan_forward(u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, True)


def selective_scan_grad(dy, dlast, check, u, delta, A, B, C, D, z, delta_bias, offsets, groups=None, state=None, want=(True,)*9):
    """ The gradients (du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dstate) of selective_scan for those of its results
    (dlast may be None), from the states that selective_scan_check stored; None where `want` is false or there is no
    such input. """
    return _scan_grad(dy, dlast, check, u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, want)


def _scan_grad(dy, dlast, check, u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, want):
    _seen_by_torch(dy, dlast, u, delta, A, B, Cm, D, z, delta_bias, state)
    eng, d, keep, S, R, ch, P, N, dt, W, dev = _scan_desc(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, False)
    dy, d.ld_dy = _rows_arg('dy', dy, dt, dev, R, ch)
    d.dy = dy.data_ptr()
    if dlast is not None:
        dlast = _param('dlast', dlast, W, dev, (S, ch, N))
        d.dlast = _ptr(dlast)
    need = _size(eng, 'psh_selective_scan_check', d)
    if check is None or check.dtype != torch.uint8 or check.device != dev or not check.is_contiguous() or check.numel() != need:
        raise ValueErr(msg='check must be the stored states that selective_scan_check returned for the same inputs!')
    d.check = check.data_ptr()

    rows, wide = u.new_empty, A.new_empty
    du = rows(R, ch) if want[0] else None
    ddelta = rows(R, ch) if want[1] else None
    dA = wide(P, ch, N) if want[2] else None
    dB = rows(R, N) if want[3] else None
    dC = rows(R, N) if want[4] else None
    dD = wide(P, ch) if want[5] and D is not None else None
    dz = rows(R, ch) if want[6] and z is not None else None
    dbias = wide(P, ch) if want[7] and delta_bias is not None else None
    dstate = wide(S, ch, N) if want[8] and state is not None else None
    d.du, d.ddelta, d.dA, d.dB, d.dC, d.dD, d.dz, d.ddelta_bias, d.dstate = (_ptr(t) for t in (du, ddelta, dA, dB, dC, dD, dz, dbias, dstate))
    space = _give_workspace(eng, d, 'psh_selective_scan_grad_workspace', u)
    eng._call('psh_selective_scan_grad', C.byref(d))
    del keep, space
    return du, ddelta, dA, dB, dC, dD, dz, dbias, dstate


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, Cm, D, z, delta_bias, state, offsets, groups):
        ctx.set_materialize_grads(False)
        y, last, check = _scan_forward(u, delta, A, B, Cm, D, z, delta_bias, offsets, groups, state, True)
        ctx.save_for_backward(u, delta, A, B, Cm, D, z, delta_bias, state, offsets, groups, check)
        return y, last

    @staticmethod
    def backward(ctx, dy, dlast):
        _first_derivative_only()
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
    _seen_by_torch(*args)
    if _autograd(*args):
        y, last = _SelectiveScan.apply(*args, offsets, groups)
    else:
        y, last, _ = _scan_forward(u, delta, A, B, C, D, z, delta_bias, offsets, groups, state, False)
    return (y, last) if return_state else y


def selective_scan_step(u, delta, state, A, B, C, D, z, delta_bias, groups=None):
    """ selective_scan for one step of every sequence: u [S, D] and so on; state [S, D, N] is updated in place.  Returns
    y [S, D]. """
    return _scan_step(u, delta, state, A, B, C, D, z, delta_bias, groups)


def _scan_step(u, delta, state, A, B, Cm, D, z, delta_bias, groups):
    _seen_by_torch(u, delta, state, A, B, Cm, D, z, delta_bias)
    _no_grad_args('selective_scan_step', u, delta, state, A, B, Cm, D, z, delta_bias)
    if state is None:
        raise TypeErr(given=state, given_name='state', expected_type=_Tensor)
    eng, d, keep, S, R, ch, P, N, dt, W, dev = _scan_desc(u, delta, A, B, Cm, D, z, delta_bias, None, groups, state, True)
    if S and keep[10] is not state:
        raise ValueErr(msg='state is updated in place: the values of each sequence have to be contiguous!')
    y, stride = u.new_empty(R, ch), keep[11]
    d.y, d.last, d.stride_last = y.data_ptr(), state.data_ptr(), stride
    eng._call('psh_selective_scan', C.byref(d))
    _advanced(state)
    del keep
    return y
