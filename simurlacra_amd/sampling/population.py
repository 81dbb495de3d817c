"""
Evaluation of a population of policies on recorded rollouts, each member on its own: what Policy.evaluate
(Pyrado/pyrado/policies/base.py:131-156) does for one policy and rollout, for all of them at once, with gradients with respect to every
member's parameters (the particles of an ensemble that are trained by policy gradients, Pyrado/pyrado/algorithms/svpg.py).
"""
import torch as to

from ..utils.exceptions import ShapeErr, ValueErr


def pack_observations(batch):
    """ The observations of a RolloutBatch (all but the last of each rollout), rollout after rollout: (rows [R, O], offsets [n + 1]
    int32), on the GPU that holds the trajectories. """
    out = batch.device_results
    if 'obs' not in out:
        raise ValueErr(msg='The trajectories of this batch were not recorded!')
    first, n = batch._offset, len(batch)
    lengths = to.as_tensor(batch.lengths.copy(), dtype=to.long)
    obs = out['obs'][:, :, first:first + n]                        # [T + 1, O, n]
    offsets = to.zeros(n + 1, dtype=to.int32)
    offsets[1:] = lengths.cumsum(0)
    env = to.repeat_interleave(to.arange(n), lengths)
    step = to.arange(int(lengths.sum())) - offsets[:-1].long()[env]
    return obs[step.to(obs.device), :, env.to(obs.device)], offsets.to(obs.device)


def evaluate_population(policy, param_sets, batch, rollouts_per_param: int = None):
    """ The actions of every parameter set on the recorded observations of its own rollouts: (actions [R, A], offsets [n + 1]) with
    the rows of rollout i at offsets[i] .. offsets[i + 1] - 1, differentiable with respect to param_sets [P, num_param].

    `batch`: the n = P x rollouts_per_param rollouts of a population, the sets one after the other, as
    ParameterExplorationSampler.sample() records them (ParameterSamplingResult.batch). """
    if not hasattr(policy, 'population_evaluate'):
        raise NotImplementedError(f'{type(policy).__name__} cannot be evaluated as a population')
    n, P = len(batch), param_sets.shape[0]
    per = n//P if rollouts_per_param is None else int(rollouts_per_param)
    if P < 1 or per*P != n:
        raise ShapeErr(msg=f'{n} rollouts are not the same number for each of {P} parameter sets!')
    obs, offsets = pack_observations(batch)
    groups = to.arange(P + 1, dtype=to.int32, device=obs.device)*per
    return policy.population_evaluate(param_sets.to(obs.device), obs, offsets, groups), offsets
