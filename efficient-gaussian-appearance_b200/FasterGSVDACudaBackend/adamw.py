"""AdamW (decoupled weight decay) over many tensors at once, beside the reference's FusedAdam (adam.py).

FusedAdamW updates every parameter of every group in one kernel launch per 384 tensors (csrc/adamw.cu): float32,
bfloat16 or float16 parameters, moments in float32 or in 8 bits, an optional float32 copy of half-precision parameters,
and clipping by the global gradient norm without a host round trip.
"""
import ctypes
import importlib.util
from array import array

import torch

from . import _lib
from ._lib import lib, check

_HOST_PATH = _lib._LIB_PATH.with_name('_fgs_host.so')
if not _HOST_PATH.exists():
    raise ImportError(f'{_HOST_PATH} not found; build it with `python efficient-gaussian-appearance_b200/build.py` (or __graft_entry__.build())')
_spec = importlib.util.spec_from_file_location('_fgs_host', _HOST_PATH)
_host = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(_host)

BLOCK = 256  # elements of a tensor that share one exponent byte where the moments are held in 8 bits
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_F32, _U8 = 0, 3
_COLUMNS = 8  # param, grad, exp_avg, exp_avg_sq, their exponents, master, element counts


def _hyper(group: dict, step: int) -> _lib.AdamwHyper:
    lr = group['lr']
    lrs = [float(v) for v in lr] if isinstance(lr, (list, tuple)) else [float(lr)]
    if not 1 <= len(lrs) <= 7:
        raise RuntimeError('between 1 and 7 learning rates are supported')
    h = _lib.AdamwHyper()
    h.learning_rates[:len(lrs)] = lrs
    h.n_learning_rates = len(lrs)
    h.beta1, h.beta2 = float(group['betas'][0]), float(group['betas'][1])
    h.eps, h.weight_decay, h.step = float(group['eps']), float(group['weight_decay']), step
    return h


class _Job:
    """Tensors of one call of the kernel (one type, one kind of state): the columns that fgs_adamw_step reads."""

    def __init__(self, code: int, bits: int, master: bool) -> None:
        self.code, self.bits, self.master = code, bits, master
        self.params, self.grads, self.states, self.hyper = [], [], [], []

    def pack(self, device: int) -> int:
        n = len(self.params)
        self.columns = array('q', bytes(8 * _COLUMNS * n))
        at = self.columns.buffer_info()[0]
        self.at = [at + 8 * n * k for k in range(_COLUMNS)]
        counts = self.at[7]
        device = _host.pack(self.params, 'parameters', self.code, device, counts, 0, self.at[0])
        _host.pack(self.grads, 'gradients', self.code, device, counts, 1, self.at[1])
        kind = _U8 if self.bits == 8 else _F32
        for k, name, code, per in ((2, 'exp_avg', kind, 1), (3, 'exp_avg_sq', kind, 1), (4, 'exp_avg_exponent', _U8, BLOCK),
                                   (5, 'exp_avg_sq_exponent', _U8, BLOCK), (6, 'master', _F32, 1)):
            if (k in (4, 5) and self.bits != 8) or (k == 6 and not self.master):
                continue
            _host.pack([s[name] for s in self.states], name, code, device, counts, per, self.at[k])
        return device

    def launch(self, hypers, n_hypers: int, partials, n_partials: int, max_norm: float, norm, stream: int) -> None:
        index = array('i', self.hyper)
        a = self.at
        t = _lib.AdamwTensors(len(self.params), a[0], a[1], a[2], a[3], a[4] if self.bits == 8 else None, a[5] if self.bits == 8 else None,
                              a[6] if self.master else None, a[7], index.buffer_info()[0])
        check(lib.fgs_adamw_step(ctypes.byref(t), hypers, n_hypers, self.code, self.bits, partials, n_partials, max_norm, norm, stream))


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
        changes are kept; the same inputs give the same codes). read_moments() gives their values.
      master_weights=True: half-precision parameters keep a float32 copy in the state ('master'), which is updated; the
        parameter is its rounding. Float32 parameters need none.
    `max_grad_norm` (for all groups together): gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) as they are
    read, p.grad stays as it is, and `grad_norm` then holds the norm (a 0-dim device tensor, a new one at each step). An
    infinite or NaN gradient makes the norm infinite or NaN: the step is then not skipped, what it scales by 0 or NaN
    becomes so.

    Parameters, gradients and state must be contiguous CUDA tensors on one device. The step count is a host value, so a
    step cannot be captured into a CUDA graph (RuntimeError). Anything refused is refused before a kernel is launched
    and leaves parameters, state and step counts as they were.
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

    def add_param_group(self, param_group: dict) -> None:
        options = {**self.defaults, **param_group}
        lrs = options['lr'] if isinstance(options['lr'], (list, tuple)) else [options['lr']]
        if not 1 <= len(lrs) <= 7:
            raise ValueError('between 1 and 7 learning rates are supported')
        if any(not float(v) >= 0.0 for v in lrs):
            raise ValueError('learning rates must not be negative')
        if len(options['betas']) != 2 or any(not 0.0 <= float(b) < 1.0 for b in options['betas']):
            raise ValueError('betas must be two numbers in [0, 1)')
        if not float(options['eps']) >= 0.0 or not float(options['weight_decay']) >= 0.0:
            raise ValueError('eps and weight_decay must not be negative')
        if options['state_bits'] not in (8, 32):
            raise ValueError('state_bits must be 8 or 32')
        super().add_param_group(param_group)

    def _new_state(self, p: torch.Tensor, bits: int, master: bool) -> dict:
        kind = torch.uint8 if bits == 8 else torch.float32
        state = {'step': 0}
        for name in ('exp_avg', 'exp_avg_sq'):
            state[name] = torch.zeros(p.shape, dtype=kind, device=p.device)
            if bits == 8:
                state[name + '_exponent'] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, dtype=torch.uint8, device=p.device)
        if master:
            state['master'] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient. `closure` (optional) recomputes the loss, which is returned."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        jobs: dict[tuple, _Job] = {}
        hypers, index, counted, fresh = [], {}, [], []
        for i, group in enumerate(self.param_groups):
            bits = group['state_bits']
            for code, params, grads in _host.live(group['params']):
                master = bool(group['master_weights']) and code != _F32
                job = jobs.setdefault((code, bits, master), _Job(code, bits, master))
                for p in params:
                    state = self.state.get(p)
                    if not state:
                        if not p.is_cuda or not p.is_contiguous():
                            raise RuntimeError('parameters must be contiguous CUDA tensors')
                        state = self._new_state(p, bits, master)
                        fresh.append((p, state))
                    t = int(state['step']) + 1
                    k = index.get((i, t))
                    if k is None:
                        k = index[(i, t)] = len(hypers)
                        hypers.append(_hyper(group, t))
                    job.hyper.append(k)
                    job.states.append(state)
                    counted.append((state, t))
                job.params += params
                job.grads += grads
        if not jobs:
            return loss
        device = -1
        try:
            for job in jobs.values():
                device = job.pack(device)
        except KeyError as e:
            raise RuntimeError(f'the optimizer state has no {e}: it was made with other state_bits or master_weights') from None
        if device != torch.cuda.current_device():
            with torch.cuda.device(device):
                self._run(jobs, hypers, device)
        else:
            self._run(jobs, hypers, device)
        for p, state in fresh:
            self.state[p] = state
        for state, t in counted:
            state['step'] = t
        return loss

    def _run(self, jobs: dict, hypers: list, device: int) -> None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('FusedAdamW.step cannot be captured into a CUDA graph: its step count is a host value')
        stream = torch.cuda.current_stream().cuda_stream
        c_hypers = (_lib.AdamwHyper * len(hypers))(*hypers)
        partials, n_partials, limit, norm = None, 0, 0.0, None
        if self.max_grad_norm is not None:
            limit = float(self.max_grad_norm)
            room, used = ctypes.c_int(0), ctypes.c_int(0)
            need = []
            for job in jobs.values():
                check(lib.fgs_grad_squares_capacity(len(job.params), ctypes.byref(room)))
                need.append(room.value)
            buffer = torch.empty(sum(need), dtype=torch.float64, device=f'cuda:{device}')
            self.grad_norm = torch.empty((), dtype=torch.float32, device=buffer.device)
            partials, norm = buffer.data_ptr(), self.grad_norm.data_ptr()
            for job in jobs.values():
                check(lib.fgs_grad_squares(job.at[1], job.at[7], bytes([job.code]) * len(job.params), len(job.params), partials + 8 * n_partials,
                                           sum(need) - n_partials, ctypes.byref(used), stream))
                n_partials += used.value
            if n_partials == 0:  # only empty gradients: no kernel writes the norm
                self.grad_norm.zero_()
        for job in jobs.values():
            job.launch(c_hypers, len(hypers), partials, n_partials, limit, norm, stream)

    @torch.no_grad()
    def read_moments(self, exp_avgs: list | None = None, exp_avg_sqs: list | None = None, dtype: torch.dtype = torch.float32) -> tuple[list, list]:
        """The first and second moments of all parameters (in the order of the groups) as values: written into the given
        lists of contiguous tensors (float32 or bfloat16, which hold 8-bit moments exactly; one type for all), or into
        new tensors of `dtype`. Parameters that were never updated have zero moments."""
        params = [p for group in self.param_groups for p in group['params']]
        if (exp_avgs is None) != (exp_avg_sqs is None):
            raise ValueError('give both lists or neither')
        if exp_avgs is None:
            exp_avgs, exp_avg_sqs = ([torch.empty(p.shape, dtype=dtype, device=p.device) for p in params] for _ in range(2))
        if len(exp_avgs) != len(params) or len(exp_avg_sqs) != len(params):
            raise ValueError('one tensor per parameter is needed')
        codes, exponents, outs = [], [], []
        for p, *to in zip(params, exp_avgs, exp_avg_sqs):
            state = self.state.get(p)
            for name, out in zip(('exp_avg', 'exp_avg_sq'), to):
                if out.numel() != p.numel():
                    raise ValueError('moments must be read into tensors of the size of their parameter')
                if not state:
                    out.zero_()
                elif state[name].dtype == torch.uint8:
                    codes.append(state[name])
                    exponents.append(state[name + '_exponent'])
                    outs.append(out)
                else:
                    out.copy_(state[name].view(out.shape))
        if outs:
            kind = outs[0].dtype
            if kind not in (torch.float32, torch.bfloat16):
                raise RuntimeError('moments are read as float32 or bfloat16')
            n = len(outs)
            columns = array('q', bytes(8 * 4 * n))
            at = [columns.buffer_info()[0] + 8 * n * k for k in range(4)]
            device = _host.pack(codes, 'moments', _U8, -1, at[3], 0, at[0])
            _host.pack(exponents, 'exponents', _U8, device, at[3], BLOCK, at[1])
            _host.pack(outs, 'outputs', _TYPES[kind], device, at[3], 1, at[2])
            with torch.cuda.device(device):
                check(lib.fgs_adamw_read_moments(at[0], at[1], b'\x01\x00' * (n // 2), at[3], n, at[2], _TYPES[kind],
                                                 torch.cuda.current_stream().cuda_stream))
        return exp_avgs, exp_avg_sqs

    def load_state_dict(self, state_dict: dict) -> None:
        """As torch's, but the state keeps its own types (torch's casts it to the parameters' type)."""
        saved = state_dict['state']
        super().load_state_dict({**state_dict, 'state': {}})
        self.state.clear()
        for group, mine in zip(state_dict['param_groups'], self.param_groups):
            for key, p in zip(group['params'], mine['params']):
                if key in saved:
                    self.state[p] = {k: v.detach().to(p.device, copy=True).contiguous() if torch.is_tensor(v) and k != 'step' else int(v)
                                     for k, v in saved[key].items()}
