"""AdamW (decoupled weight decay) over many tensors at once, beside the reference's FusedAdam (adam.py).

FusedAdamW updates every parameter of every group in one kernel launch per 384 tensors (csrc/adamw.cu): float32,
bfloat16 or float16 parameters, moments in float32 or in 8 bits, an optional float32 copy of half-precision parameters,
and clipping by the global gradient norm without a host round trip.
"""
import copy
import sys

import torch

from ._lib import host

BLOCK = 256  # elements of a tensor that share one exponent byte where the moments are held in 8 bits


class FusedAdamW(torch.optim.Optimizer):
    """AdamW whose step() updates all parameters that have a gradient, of any number of tensors and groups, in one launch
    per 384 tensors of a type.

    Per element, in float32, with t the parameter's own step count and c the clip factor:
      g <- c g; m <- b1 m + (1 - b1) g; v <- b2 v + (1 - b2) g^2;
      p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    Options of a group: `lr` (a number, or up to 7 numbers cycled over a tensor's elements as in FusedAdam), `betas`,
    `eps`, `weight_decay`, and
      state_bits=32: float32 moments; state_bits=8: one byte per element and moment plus one exponent byte for each 256
        elements (three mantissa bits, rounded with thresholds that are spread evenly over the steps, so that slow
        changes are kept; the same inputs give the same codes). Updates differ from those of float32 moments by some 11 %
        rms with noisy gradients, 14 % for a while after these have shrunk a lot. read_moments() gives the moments' values.
      master_weights=True: half-precision parameters keep a float32 copy in the state ('master'), which is updated; the
        parameter is its rounding. Float32 parameters need none.
    `max_grad_norm` (for all groups together; inf only measures): gradients are scaled by min(1, max_grad_norm /
    (norm + 1e-6)) as they are read, p.grad stays as it is, and `grad_norm` then holds the norm (a 0-dim device tensor, a
    new one at each step; None after a step without clipping or gradients). An infinite or NaN gradient makes the norm
    infinite or NaN: the step is then not skipped, what it scales by 0 or NaN becomes so. With 8-bit moments an infinite or
    NaN moment makes those of its block of 256 elements NaN.

    Parameters, gradients and state must be contiguous CUDA tensors on one device, and no two parameters may share
    memory. The step count is a host value, so a step cannot be captured into a CUDA graph, nor recorded by a tracer
    (RuntimeError); torch.compile runs it between its graphs. Options of other AdamWs that a step does not follow (maximize,
    amsgrad, differentiable, weight decay that is not decoupled) are refused. Anything refused is refused before state is
    made or a kernel launched, and leaves parameters, state and step counts as they were. For autograd a step is a change
    in place.
    """

    grad_norm = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, master_weights=False,
                 max_grad_norm=None) -> None:
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError('max_grad_norm must be positive (or None for no clipping)')
        super().__init__(params, {'lr': lr, 'betas': betas, 'eps': eps, 'weight_decay': weight_decay, 'state_bits': state_bits,
                                  'master_weights': master_weights})
        self.max_grad_norm = max_grad_norm

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), 'max_grad_norm': self.max_grad_norm}

    @staticmethod
    def _check_options(options: dict) -> None:
        """Raises ValueError for options of a group that a step cannot follow, those of other AdamWs among them."""
        lrs = options['lr'] if isinstance(options['lr'], (list, tuple)) else [options['lr']]
        if not 1 <= len(lrs) <= 7:
            raise ValueError('between 1 and 7 learning rates are supported')
        if any(not float(v) >= 0.0 for v in lrs):
            raise ValueError('learning rates must not be negative')
        if len(options['betas']) != 2 or any(not 0.0 <= float(b) < 1.0 for b in options['betas']):
            raise ValueError('betas must be two numbers in [0, 1)')
        if not float(options['eps']) >= 0.0 or not float(options['weight_decay']) >= 0.0:
            raise ValueError('eps and weight_decay must not be negative')
        if 0.0 < float(options['eps']) < 1.2e-38:
            raise ValueError('eps must be zero or a normal float32 (at least 1.2e-38)')
        if options['state_bits'] not in (8, 32):
            raise ValueError('state_bits must be 8 or 32')
        for name in ('maximize', 'amsgrad', 'differentiable'):
            if options.get(name, False):
                raise ValueError(f'{name} is not supported')
        if not options.get('decoupled_weight_decay', True) and float(options['weight_decay']) != 0.0:
            raise ValueError('weight decay is always decoupled: that of Adam (decoupled_weight_decay=False) is not supported')

    def add_param_group(self, param_group: dict) -> None:
        self._check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    @staticmethod
    def _new_state(p: torch.Tensor, bits: int, master: bool) -> dict:
        kind = torch.uint8 if bits == 8 else torch.float32
        state = {'step': 0}
        # names as literals: interned strings are found by identity, made ones by their letters (5 us of a step over 300 tensors)
        for name, exponent in (('exp_avg', 'exp_avg_exponent'), ('exp_avg_sq', 'exp_avg_sq_exponent')):
            state[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
            if bits == 8:
                state[exponent] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, dtype=torch.uint8, device=p.device)
        if master:
            state['master'] = p.detach().float()
        return state

    def step(self, closure=None):
        """One update of every parameter that has a gradient. `closure` (optional) recomputes the loss, which is returned."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        host().adamw_step(self.state, self.param_groups, self._new_state, self.max_grad_norm, self)
        return loss

    def read_moments(self, exp_avgs: list | None = None, exp_avg_sqs: list | None = None, dtype: torch.dtype = torch.float32) -> tuple[list, list]:
        """The first and second moments of all parameters (in the order of the groups) as values: written into the given
        lists of contiguous tensors (float32 or bfloat16, which hold 8-bit moments exactly; one type for all), or into
        new tensors of `dtype`. Parameters that were never updated have zero moments."""
        groups = self.param_groups
        params = groups[0]['params'] if len(groups) == 1 else [p for group in groups for p in group['params']]
        if (exp_avgs is None) != (exp_avg_sqs is None):
            raise ValueError('give both lists or neither')
        if exp_avgs is None:
            exp_avgs, exp_avg_sqs = ([torch.empty(p.shape, dtype=dtype, device=p.device) for p in params] for _ in range(2))
        if len(exp_avgs) != len(params) or len(exp_avg_sqs) != len(params):
            raise ValueError('one tensor per parameter is needed')
        host().read_moments(self.state, params, list(exp_avgs), list(exp_avg_sqs))
        return exp_avgs, exp_avg_sqs

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but the state keeps its own types (torch's casts it to the parameters' type). Groups saved by another
        AdamW take this one's options where they lack them (its moments become float32: state_bits=32); what this one cannot
        follow (maximize, amsgrad, differentiable, weight decay that is not decoupled) is refused, and nothing is changed. Hooks
        around the loading see the whole state."""
        loaded = {}

        def take(_, state_dict: dict) -> dict:  # behind all other pre-hooks; torch's loading sees no state of a parameter
            for group in state_dict['param_groups']:
                self._check_options({**self.defaults, **group})
            rest = dict(state_dict['state'])
            for group, mine in zip(state_dict['param_groups'], self.param_groups):
                for key, p in zip(group['params'], mine['params']):
                    if key in rest:
                        loaded[p] = self._loaded_state(p, rest.pop(key))
            return {**state_dict, 'state': rest}

        def put(_) -> None:  # before all other post-hooks
            for group in self.param_groups:
                for name, value in self.defaults.items():
                    group.setdefault(name, value)
            self.state.update(loaded)

        hooks = [self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(put, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    @staticmethod
    def _loaded_state(p: torch.Tensor, saved: dict) -> dict:
        state = {}
        for name, value in saved.items():
            if name == 'step':
                value = int(value)
            elif torch.is_tensor(value):
                floats = name in ('exp_avg', 'exp_avg_sq') and value.is_floating_point()  # those of half-precision AdamWs, exactly
                value = value.detach().to(p.device, torch.float32 if floats else None, copy=True).contiguous()
            else:
                value = copy.deepcopy(value)
            state[sys.intern(name)] = value
        return state
