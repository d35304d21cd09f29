"""AdamW: one step over all tensors of a model in few launches, with states in 32 bits or in 8."""
from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from . import _native

BLOCK = 256          # elements that share a scale


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence, exp_avg_sqs: Sequence, *, step, lr, betas: tuple[float, float] = (0.9, 0.999),
               eps: float = 1e-8, weight_decay: float = 1e-2, masters: Sequence[Tensor | None] | None = None, grad_scale: Tensor | None = None, seed: int = 0) -> None:
    """One step of AdamW in place: ``params`` (bfloat16, float16 or float32), their states, and where given the float32 ``masters`` whose roundings the parameters are.

    States are float32 tensors laid out like their parameter, or in 8 bits pairs ``(values, scales)``: float8_e4m3fn values in the parameter's storage order and one
    float32 scale per 256 of them.  ``exp_avg_sqs`` in 8 bits hold the roots of the second moments.  8-bit states are rounded stochastically, by a hash of ``seed``, ``step``,
    the parameter's place in the list and the element: the same call gives the same bits.  :func:`state_8bit` makes empty ones.

    ``step`` counts from 1, this step included.  ``step`` (int64) and ``lr`` (float32) may be tensors of one number on the GPU, which a recorded and
    replayed call reads anew; ``grad_scale`` is one that gradients are multiplied by (a clipping coefficient).  Parameters that share memory, or one that is given twice, are refused.
    """
    _call(params, grads, exp_avgs, exp_avg_sqs, masters, step=step, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, grad_scale=grad_scale, seed=seed)


def _call(params, grads, exp_avgs, exp_avg_sqs, masters, *, step, lr, betas, eps, weight_decay, grad_scale, seed, launch=True):
    # (without a launch: the checks alone)
    _native.torch_ext().adamw_step(params, grads, exp_avgs, exp_avg_sqs, masters, step, lr, float(betas[0]), float(betas[1]), float(eps), float(weight_decay), grad_scale,
                                   int(seed) & 0xffffffff, launch)


def state_8bit(param: Tensor) -> tuple[Tensor, Tensor]:
    """A state of zeros in 8 bits for a parameter: its values and their scales."""
    return (torch.zeros(param.numel(), dtype=torch.float8_e4m3fn, device=param.device),
            torch.zeros(-(-param.numel() // BLOCK), dtype=torch.float32, device=param.device))


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on :func:`adamw_step` (no amsgrad, no maximize).

    ``state_bits``: 32, or 8 for parameters of at least ``min_8bit_size`` elements (the states of smaller ones cost nothing and stay in 32).  ``masters``: bfloat16 and float16 parameters are
    the roundings of float32 copies that the optimizer keeps, so that steps smaller than half a place of theirs are not lost; a parameter that is set from outside between steps has to be
    set in ``state[param]['master']`` too, or the next step takes it back.  Parameters without a gradient are left out of a step and
    count their own steps.

    ``capturable``: the step count of each group is on the GPU, and ``lr`` may be a float32 tensor there, so that a recorded :meth:`step` can be replayed; all parameters of a group
    need gradients then, in every step, and the first one is not recorded (a replay would make the states anew).  The parameters of a group are on one GPU.  The option may be
    changed between steps (``group['capturable'] = True`` behind a checkpoint that was saved without it): the count goes on where it was, which has to be one for all parameters.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits: int = 32, masters: bool = True, min_8bit_size: int = 4096,
                 capturable: bool = False, seed: int = 0):
        if not isinstance(lr, Tensor) and not 0 <= lr < float('inf'):
            raise ValueError(f'lr must be finite and not negative, got {lr}')
        if isinstance(lr, Tensor) and not capturable:
            raise ValueError('lr as a tensor needs capturable=True')
        if not all(0 <= b < 1 for b in betas) or not 0 <= eps < float('inf') or not 0 <= weight_decay < float('inf'):
            raise ValueError(f'betas in [0, 1), eps and weight_decay not negative: got {betas}, {eps}, {weight_decay}')
        if state_bits not in (8, 32):
            raise ValueError(f'states of 8 or 32 bits, got {state_bits}')
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits, masters=masters, min_8bit_size=min_8bit_size,
                                      capturable=capturable, seed=seed))

    def _state_of(self, param, group):
        state = self.state[param]
        state['step'] = 0
        for name in ('exp_avg', 'exp_avg_sq'):
            if group['state_bits'] == 8 and param.numel() >= group['min_8bit_size']:
                state[name], state[name + '_scales'] = state_8bit(param)
            else:
                state[name] = torch.zeros_like(param, dtype=torch.float32, memory_format=torch.preserve_format)
        if group['masters'] and param.dtype is not torch.float32:
            state['master'] = param.detach().to(torch.float32, copy=True, memory_format=torch.preserve_format)
        return state

    @torch.no_grad()
    def step(self, closure=None, *, grad_scale: Tensor | None = None):
        """One step.  ``grad_scale``: a float32 tensor of one number on the GPU that gradients are multiplied by."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        recording = torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()
        # (all groups are looked at before the first is changed: a step that is refused leaves the optimizer as it was)
        calls, made, begun = [], {}, []
        try:
            for index, group in enumerate(self.param_groups):
                for count, lists in self._lists(group, recording, made, begun).items():
                    calls.append((group, count, lists, dict(lr=group['lr'], betas=group['betas'], eps=group['eps'], weight_decay=group['weight_decay'], grad_scale=grad_scale,
                                                            seed=group['seed'] + 0x10000 * index)))
            if len(calls) > 1:                     # (one call is refused as a whole)
                for group, count, (_, *lists), more in calls:
                    _call(*lists, step=group['step_at'] if group['capturable'] else count + 1, launch=False, **more)
            for group, count, (states, *lists), more in calls:
                if group['capturable']:
                    group['step_at'] += 1
                    try:
                        _call(*lists, step=group['step_at'], **more)
                    except BaseException:
                        group['step_at'] -= 1
                        raise
                else:
                    _call(*lists, step=count + 1, **more)
                    for state in states:
                        state['step'] = count + 1
                for param in lists[0] if made else ():
                    made.pop(param, None)
                begun = [other for other in begun if other is not group]
        except BaseException:
            for param in made:
                del self.state[param]
            for group in begun:
                del group['step_at']
            raise
        return loss

    def _lists(self, group, recording, made, begun):
        """What a step of a group works on, by the steps that its parameters have made: lists of states, parameters, gradients, both averages, masters.  New states go to ``made``, a
        group whose count moves to the GPU to ``begun``."""
        capturable, by_count = group['capturable'], {}
        if recording and not capturable:
            raise RuntimeError('a step that is recorded needs capturable=True: every replay would be the same step')
        if not capturable and 'step_at' in group:
            # (the option has been taken back: the parameters count on from there)
            count = int(group.pop('step_at'))
            for param in group['params']:
                if self.state.get(param):
                    self.state[param]['step'] = count
        for param in group['params']:
            grad = param.grad
            if grad is None:
                if capturable:
                    raise RuntimeError('a group that can be captured needs gradients of all its parameters')
                continue
            state = self.state.get(param)
            if not state:
                if recording:
                    raise RuntimeError('the first step of a parameter cannot be recorded: a replay would make its states anew')
                if capturable and 'step_at' in group:
                    raise RuntimeError('a group that can be captured has one count of steps: parameters that come later need a group of their own')
                made[param] = True
                state = self._state_of(param, group)
            lists = by_count.get(state['step'])
            if lists is None:
                lists = by_count[state['step']] = ([], [], [], [], [], [])
            lists[0].append(state)
            lists[1].append(param)
            lists[2].append(grad)
            if 'exp_avg_scales' in state:
                lists[3].append((state['exp_avg'], state['exp_avg_scales']))
                lists[4].append((state['exp_avg_sq'], state['exp_avg_sq_scales']))
            else:
                lists[3].append(state['exp_avg'])
                lists[4].append(state['exp_avg_sq'])
            lists[5].append(state.get('master'))
        if capturable and by_count and 'step_at' not in group:
            if recording:
                raise RuntimeError('the first step of a group that can be captured cannot be recorded: a replay would begin its count anew')
            if len(by_count) > 1:
                raise RuntimeError('a group that can be captured has one count of steps: its parameters have made different numbers of them')
            begun.append(group)
            group['step_at'] = torch.full((1,), next(iter(by_count)), dtype=torch.int64, device=group['params'][0].device)
        return by_count

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        if not all('state_bits' in group for group in state_dict['param_groups']):
            raise ValueError('these are the states of another optimizer')
        super().load_state_dict(state_dict)
        # (torch casts states to their parameter's dtype: these have dtypes of their own)
        saved = [index for group in state_dict['param_groups'] for index in group['params']]
        params = [param for group in self.param_groups for param in group['params']]
        for index, param in zip(saved, params):
            for name, value in state_dict['state'].get(index, {}).items():
                if isinstance(value, Tensor):
                    self.state[param][name] = value.detach().to(param.device, copy=True)
        for mine, given in zip(self.param_groups, state_dict['param_groups']):
            for name in ('step_at', 'lr'):
                if isinstance(given.get(name), Tensor):
                    mine[name] = given[name].detach().to(mine['params'][0].device, copy=True)
