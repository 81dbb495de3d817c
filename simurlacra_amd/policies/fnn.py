"""
FNN and FNNPolicy (Pyrado/pyrado/policies/fnn.py:14-203): Linear -> nonlinearity ... -> Linear (-> output nonlinearity).
"""
from typing import Callable, Sequence

import torch as to
import torch.nn as nn
from torch.nn.utils import convert_parameters as cp

from .. import operators as ops
from ..specs import PolicySpec
from ..utils.data_types import EnvSpec
from ..utils.exceptions import ShapeErr
from .base import Policy
from .initialization import init_param

_FUSABLE_NL = {None: None, to.tanh: 'tanh', to.relu: 'relu', to.sigmoid: 'sigmoid'}
try:
    import torch.nn.functional as F
    _FUSABLE_NL.update({F.relu: 'relu', F.tanh: 'tanh', F.sigmoid: 'sigmoid'})
except Exception:
    pass


class FNN(nn.Module):
    def __init__(self, input_size: int, output_size: int, hidden_sizes: Sequence[int], hidden_nonlin, dropout: float = 0.,
                 output_nonlin: Callable = None, init_param_kwargs: dict = None, use_cuda: bool = False):
        self._device = 'cuda' if use_cuda and to.cuda.is_available() else 'cpu'
        super().__init__()
        hidden_sizes = list(hidden_sizes)
        self._hidden_nonlin = (list(hidden_nonlin) if isinstance(hidden_nonlin, (list, tuple))
                               else len(hidden_sizes)*[hidden_nonlin])
        self._dropout, self._output_nonlin = dropout, output_nonlin
        self.hidden_layers = nn.ModuleList()
        last = input_size
        for hs in hidden_sizes:
            self.hidden_layers.append(nn.Linear(last, hs))
            last = hs
            if dropout > 0:
                self.hidden_layers.append(nn.Dropout(p=dropout))
        self.output_layer = nn.Linear(last, output_size)
        self.double()
        self.init_param(None, **(init_param_kwargs or dict()))
        self.to(self.device)

    @property
    def device(self) -> str:
        return self._device

    @property
    def dropout(self):
        return self._dropout

    @property
    def hidden_nonlin(self):
        return self._hidden_nonlin

    @property
    def output_nonlin(self):
        return self._output_nonlin

    @property
    def param_values(self) -> to.Tensor:
        return cp.parameters_to_vector(self.parameters())

    @param_values.setter
    def param_values(self, param):
        cp.vector_to_parameters(param, self.parameters())

    def init_param(self, init_values: to.Tensor = None, **kwargs):
        if init_values is None:
            for layer in self.hidden_layers:
                init_param(layer, **kwargs)
            init_param(self.output_layer, **kwargs)
        else:
            self.param_values = init_values

    def forward(self, input: to.Tensor) -> to.Tensor:
        x = input.to(self.device)
        lin = 0
        for layer in self.hidden_layers:
            x = layer(x)
            if isinstance(layer, nn.Linear):
                nl = self._hidden_nonlin[lin]
                lin += 1
                if nl is not None:
                    x = nl(x)
        x = self.output_layer(x)
        return x if self._output_nonlin is None else self._output_nonlin(x)


class FNNPolicy(Policy):
    name: str = 'fnn'

    def __init__(self, spec: EnvSpec, hidden_sizes: Sequence[int], hidden_nonlin, dropout: float = 0.,
                 output_nonlin: Callable = None, init_param_kwargs: dict = None, use_cuda: bool = False):
        super().__init__(spec, use_cuda)
        self.net = FNN(spec.obs_space.flat_dim, spec.act_space.flat_dim, hidden_sizes, hidden_nonlin, dropout,
                       output_nonlin, init_param_kwargs, use_cuda)

    def init_param(self, init_values: to.Tensor = None, **kwargs):
        if init_values is None:
            self.net.init_param(None, **kwargs)
        else:
            self.param_values = init_values

    def forward(self, obs: to.Tensor) -> to.Tensor:
        return self.net(obs)

    def fused_spec(self):
        net = self.net
        hidden = [l.out_features for l in net.hidden_layers if isinstance(l, nn.Linear)]
        if net.dropout > 0 or not 1 <= len(hidden) <= 4 or max(hidden) > 64:
            return None
        try:
            nls = [_FUSABLE_NL[nl] for nl in net.hidden_nonlin]
            out_nl = _FUSABLE_NL[net.output_nonlin]
        except (KeyError, TypeError):
            return None
        return PolicySpec('fnn', self.env_spec.obs_space.flat_dim, self.env_spec.act_space.flat_dim, hidden=hidden,
                          hidden_nonlin=nls, out_nonlin=out_nl)

    # ---- populations of networks of any width and depth (those that the rollout kernels do not take), layer by layer
    @property
    def supports_population(self) -> bool:
        """ Whether the nonlinearities are among those of operators.grouped_linear, and none is random. """
        try:
            return self.net.dropout == 0 and all(nl in _FUSABLE_NL for nl in [*self.net.hidden_nonlin, self.net.output_nonlin])
        except TypeError:
            return False

    def population_forward(self, params: to.Tensor, obs: to.Tensor, rows: to.Tensor) -> to.Tensor:
        """ Policy p, with the parameters params[p], acts on obs[rows[p]:rows[p + 1]] (GPU tensors, float64). """
        if not self.supports_population:
            raise NotImplementedError('a population needs networks without dropout whose nonlinearities are tanh, relu, sigmoid or none')
        if params.dim() != 2 or params.shape[1] != self.num_param:
            raise ShapeErr(msg=f'params must have the shape [policies, {self.num_param}], but has {list(params.shape)}!')
        layers = [l for l in self.net.hidden_layers if isinstance(l, nn.Linear)] + [self.net.output_layer]
        x, at, P = obs, 0, params.shape[0]
        for l, nl in zip(layers, [*self.net.hidden_nonlin, self.net.output_nonlin]):
            mid, end = at + l.weight.numel(), at + l.weight.numel() + l.bias.numel()
            x = ops.grouped_linear(x, params[:, at:mid].view(P, *l.weight.shape), params[:, mid:end], rows, _FUSABLE_NL[nl])
            at = end
        return x

    def population_evaluate(self, params: to.Tensor, obs: to.Tensor, offsets: to.Tensor, groups: to.Tensor) -> to.Tensor:
        """ The actions for whole episodes obs[offsets[s]:offsets[s + 1]], of which groups[p] .. groups[p + 1] - 1 are policy p's. """
        return self.population_forward(params.to(obs.device, obs.dtype), obs, offsets[groups.long()])
