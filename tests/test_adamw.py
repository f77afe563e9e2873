"""FusedAdamW without a GPU: what it refuses, its state handling, and the 8-bit format of its moments."""
import copy
import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw as O


def _param(n=5, dtype=torch.float32, grad=True):
    p = torch.nn.Parameter(torch.ones(n, dtype=dtype))
    if grad:
        p.grad = torch.ones(n, dtype=dtype)
    return p


@pytest.mark.parametrize('options,match', [
    ({'lr': -1.0}, 'learning rates'), ({'lr': [1e-3] * 8}, 'learning rates'), ({'lr': []}, 'learning rates'), ({'betas': (0.9, 1.0)}, 'betas'),
    ({'betas': (0.9,)}, 'betas'), ({'eps': -1e-8}, 'eps'), ({'eps': 1e-39}, 'eps'), ({'weight_decay': -0.1}, 'weight_decay'), ({'state_bits': 16}, 'state_bits'),
    ({'max_grad_norm': 0.0}, 'max_grad_norm'), ({'max_grad_norm': float('nan')}, 'max_grad_norm'), ({'lr': float('nan')}, 'learning rates')])
def test_options_refused(options, match):
    import FasterGSVDACudaBackend as F
    with pytest.raises(ValueError, match=match):
        F.FusedAdamW([_param()], **options)


def test_group_options_refused():
    import FasterGSVDACudaBackend as F
    with pytest.raises(ValueError, match='state_bits'):
        F.FusedAdamW([{'params': [_param()], 'state_bits': 4}])


def test_cpu_tensors_refused_and_left_alone():
    import FasterGSVDACudaBackend as F
    p = _param()
    opt = F.FusedAdamW([p])
    with pytest.raises(RuntimeError, match='CUDA'):
        opt.step()
    assert not opt.state and torch.equal(p.detach(), torch.ones(5))


def test_types_refused():
    import FasterGSVDACudaBackend as F
    with pytest.raises(RuntimeError, match='float32, bfloat16 or float16'):
        F.FusedAdamW([_param(dtype=torch.float64)]).step()


def test_step_without_gradients_does_nothing():
    import FasterGSVDACudaBackend as F
    p = _param(grad=False)
    opt = F.FusedAdamW([p])
    assert opt.step() is None and not opt.state and opt.grad_norm is None
    assert opt.step(lambda: 3.0) == 3.0


def test_layouts_refused():
    """Strides, sparse gradients and gradients of another type are refused before anything is looked at on a device."""
    import FasterGSVDACudaBackend as F
    p = torch.nn.Parameter(torch.zeros(4, 6).t())
    p.grad = torch.zeros(6, 4)
    with pytest.raises(RuntimeError, match='parameter must be a contiguous float32'):
        F.FusedAdamW([p]).step()
    q = torch.nn.Parameter(torch.ones(4, 4, dtype=torch.bfloat16).expand(2, 4, 4))
    q.grad = torch.ones(2, 4, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='contiguous bfloat16'):
        F.FusedAdamW([q]).step()


def test_entries_of_the_host_module_refuse():
    import FasterGSVDACudaBackend as F
    host = F._lib.host()
    with pytest.raises(TypeError):
        host.adamw_step([], [], None, None)
    for groups, match in (([3], 'dicts'), ([{}], 'params'), ([{'params': ()}], 'list'), ([{'params': [3], 'state_bits': 8, 'master_weights': 0}], 'tensor'),
                          ([{'params': [], 'state_bits': 5, 'master_weights': 0}], 'state_bits')):
        with pytest.raises(RuntimeError, match=match):
            host.adamw_step({}, groups, None, None)
    with pytest.raises(RuntimeError, match='max_grad_norm'):
        host.adamw_step({}, [], None, -1.0)
    with pytest.raises(TypeError):
        host.adamw_step({}, [], None, 'x')
    with pytest.raises(RuntimeError, match='one tensor'):
        host.read_moments({}, [_param()], [], [])
    with pytest.raises(RuntimeError, match='CUDA'):
        host.read_moments({}, [_param()], [torch.zeros(5)], [torch.zeros(5)])
    with pytest.raises(RuntimeError, match='float32 or bfloat16'):
        host.read_moments({}, [_param()], [torch.zeros(5).half()], [torch.zeros(5).half()])


def _abi_call(**change):
    from FasterGSVDACudaBackend import _lib
    one = lambda v: (ctypes.c_uint64 * 1)(v)  # noqa: E731
    keep = {'param': one(64), 'grad': one(64), 'exp_avg': one(64), 'exp_avg_sq': one(64), 'n_elements': (ctypes.c_int64 * 1)(4),
            'hyper': (ctypes.c_int32 * 1)(0)}
    keep.update(change.get('tensors', {}))
    t = _lib.AdamwTensors(1, **{k: ctypes.addressof(v) for k, v in keep.items()})
    h = _lib.AdamwHyper()
    h.learning_rates[0], h.n_learning_rates, h.beta1, h.beta2, h.eps, h.weight_decay, h.step = 1e-3, 1, 0.9, 0.999, 1e-8, 0.0, 1
    for k, v in change.get('hyper', {}).items():
        setattr(h, k, v)
    return _lib.check(_lib.lib.fgs_adamw_step(ctypes.byref(t), ctypes.byref(h), change.get('n_hypers', 1), change.get('dtype', 0),
                                              change.get('bits', 32), change.get('partials'), change.get('n_partials', 0), change.get('max_norm', 0.0),
                                              change.get('norm'), None))


@pytest.mark.parametrize('change,match', [
    ({'dtype': 3}, 'dtype'), ({'bits': 4}, 'state_bits'), ({'bits': 8}, 'exponents'), ({'n_hypers': 0}, 'NULL'),
    ({'hyper': {'step': 0}}, 'step'), ({'hyper': {'n_learning_rates': 8}}, 'learning rates'), ({'hyper': {'beta1': 1.0}}, 'betas'),
    ({'hyper': {'beta2': float('nan')}}, 'betas'), ({'hyper': {'eps': -1.0}}, 'eps'), ({'hyper': {'eps': 1e-40}}, 'eps'), ({'partials': 64, 'max_norm': 1.0}, 'grad_norm'),
    ({'partials': 64, 'norm': 64}, 'max_norm'), ({'tensors': {'hyper': (ctypes.c_int32 * 1)(1)}}, 'index'),
    ({'tensors': {'grad': (ctypes.c_uint64 * 1)(0)}}, 'NULL'), ({'tensors': {'master': (ctypes.c_uint64 * 1)(64)}}, 'master')])
def test_c_entry_refuses(change, match):
    """Bad arguments come back as an error status with a message, before any launch."""
    with pytest.raises(RuntimeError, match=match):
        _abi_call(**change)


def test_c_entries_of_the_norm_and_the_moments_refuse():
    from FasterGSVDACudaBackend import _lib
    lib, check = _lib.lib, _lib.check
    room, used = ctypes.c_int(0), ctypes.c_int(0)
    check(lib.fgs_grad_squares_capacity(1025, ctypes.byref(room)))
    room_of_two = room.value
    check(lib.fgs_grad_squares_capacity(1024, ctypes.byref(room)))
    assert room_of_two - 1 == 2 * (room.value - 1) > 0  # 1024 tensors per launch, and one value for the clip factor
    ptr, n, kind = (ctypes.c_uint64 * 1)(64), (ctypes.c_int64 * 1)(4), (ctypes.c_uint8 * 1)(3)
    a = ctypes.addressof
    with pytest.raises(RuntimeError, match='dtype'):
        check(lib.fgs_grad_squares(a(ptr), a(n), a(kind), 1, 64, room.value, ctypes.byref(used), None))
    kind[0] = 0
    with pytest.raises(RuntimeError, match='partial sums'):
        check(lib.fgs_grad_squares(a(ptr), a(n), a(kind), 1, 64, room.value - 1, ctypes.byref(used), None))
    with pytest.raises(RuntimeError, match='bad argument'):
        check(lib.fgs_grad_squares(a(ptr), a(n), a(kind), -1, 64, room.value, ctypes.byref(used), None))
    with pytest.raises(RuntimeError, match='fp32 or bf16'):
        check(lib.fgs_adamw_read_moments(a(ptr), a(ptr), a(kind), a(n), 1, a(ptr), 2, None))


def test_state_keeps_its_types_over_save_and_load():
    """torch's own load_state_dict would cast codes and float32 copies to the parameters' type."""
    import FasterGSVDACudaBackend as F
    p = _param(300, torch.bfloat16)
    opt = F.FusedAdamW([p], state_bits=8, master_weights=True, max_grad_norm=1.0)
    state = opt._new_state(p, 8, True)
    state['exp_avg'].random_(0, 256)
    opt.state[p] = {**state, 'step': 7}
    other = F.FusedAdamW([_param(300, torch.bfloat16)], state_bits=8, master_weights=True)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    got = next(iter(other.state.values()))
    assert got['step'] == 7 and got['exp_avg'].dtype == torch.uint8 and got['exp_avg_exponent'].numel() == 2
    assert got['master'].dtype == torch.float32 and torch.equal(got['exp_avg'], state['exp_avg'])
    again = copy.deepcopy(opt)
    assert again.max_grad_norm == 1.0 and next(iter(again.state.values()))['exp_avg'].dtype == torch.uint8


def test_state_of_another_adamw_loads():
    """A checkpoint of torch's AdamW: its step counts are tensors and its groups lack this optimizer's options."""
    import FasterGSVDACudaBackend as F
    p = _param(6)
    ref = torch.optim.AdamW([p], lr=0.02, betas=(0.8, 0.95))
    for _ in range(3):
        ref.step()
    opt = F.FusedAdamW([p], state_bits=32, master_weights=True)
    opt.load_state_dict(ref.state_dict())
    group, state = opt.param_groups[0], opt.state[p]
    assert group['lr'] == 0.02 and tuple(group['betas']) == (0.8, 0.95) and group['state_bits'] == 32 and group['master_weights'] is True
    assert state['step'] == 3 and isinstance(state['step'], int) and torch.equal(state['exp_avg'], ref.state[p]['exp_avg'])
    assert state['exp_avg'].data_ptr() != ref.state[p]['exp_avg'].data_ptr()


def test_code_values():
    """Every code's value survives coding in a block of its own exponent, whatever the threshold: it needs no rounding."""
    for signed in (True, False):
        top = O.top_of(signed)
        for e in (0, 1, 14, 15, 16, 31, 32, 127, 200, 253):
            codes = np.zeros(256, np.uint8)
            q = np.arange(1, top - 7)  # codes whose exponent is at most e
            codes[:q.size] = q
            if signed:
                codes[q.size:2 * q.size] = q | 128
            x = O.decode(codes, np.array([e], np.uint8), signed)
            for step in (1, 2, 1000):
                got, exp = O.encode(x, step, signed)
                if not (x != 0).any():
                    continue
                if exp[0] == e:
                    np.testing.assert_array_equal(O.decode(got, exp, signed), x)


def test_thresholds_spread_evenly():
    """Over 4096 steps the average of an element's coded value is the value: the counts of the two neighbouring codes
    follow the value's place between them within half a percent of a code step (an independent threshold per step would
    be off by 0.8 % rms)."""
    rng = np.random.default_rng(0)
    for signed in (True, False):
        x = np.exp2(rng.uniform(-6, 0, 256)).astype(np.float32)
        x[0] = 1.0
        total = np.zeros(256)
        for t in range(1, 4097):
            q, e = O.encode(x, t, signed)
            total += O.decode(q, e, signed)
        unit = np.exp2(np.floor(np.log2(x)) - 3)
        assert np.abs(total / 4096 - x).max() <= (0.005 * unit).max() and (np.abs(total / 4096 - x) <= 0.005 * unit).all()


def test_small_values_are_kept():
    """Below the smallest code the first moment is kept on average, and a nonzero second moment never becomes zero."""
    x = np.full(256, 1e-6, np.float32)
    x[0] = 1.0
    total = np.zeros(256)
    for t in range(1, 4097):
        q, e = O.encode(x, t, True)
        total += O.decode(q, e, True)
    least = 1.25 * 2.0 ** -15
    assert np.abs(total[1:] / 4096 - 1e-6).max() <= 0.005 * least
    x = np.full(256, 1e-30, np.float32)
    x[0], x[1] = 1.0, 0.0
    v = O.decode(*O.encode(x, 5, False), False)
    assert v[1] == 0.0 and (v[2:] == np.float32(1.25 * 2.0 ** -31)).all()


@pytest.mark.parametrize('kind', ['jit.trace', 'real', 'fake', 'symbolic'])
def test_tracers_refused(kind):
    """A tracer would record none of the kernel's writes."""
    import FasterGSVDACudaBackend as F
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    p = _param()
    opt = F.FusedAdamW([p])

    def step(x):
        opt.step()
        return x + p.detach()

    def read(x):
        opt.read_moments([torch.zeros(5)], [torch.zeros(5)])
        return x + 1.0

    for f in (step, read):
        with pytest.raises(RuntimeError, match='cannot be traced'):
            if kind == 'jit.trace':
                torch.jit.trace(f, (torch.zeros(5),))
            elif kind == 'fake':
                with FakeTensorMode(allow_non_fake_inputs=True):
                    f(torch.zeros(5))
            else:
                make_fx(f, tracing_mode=kind)(torch.zeros(5))
    assert not opt.state


def test_tensors_without_memory_refused():
    import FasterGSVDACudaBackend as F
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        p = torch.nn.Parameter(mode.from_tensor(torch.ones(5)))
        p.grad = mode.from_tensor(torch.ones(5))
    with pytest.raises(RuntimeError, match='plain tensor'):
        F.FusedAdamW([p]).step()


def test_lazily_negated_tensors_refused():
    """Their memory holds the negative of their values (the imaginary part of a conjugate, for one)."""
    import FasterGSVDACudaBackend as F
    p = torch.nn.Parameter(torch.complex(torch.ones(1), torch.ones(1)).conj().imag)
    p.grad = torch.ones(1)
    with pytest.raises(RuntimeError, match='parameter must not be a lazily negated view'):
        F.FusedAdamW([p]).step()


@pytest.mark.parametrize('options,match', [({'maximize': True}, 'maximize'), ({'amsgrad': True}, 'amsgrad'), ({'differentiable': True}, 'differentiable'),
                                           ({'decoupled_weight_decay': False, 'weight_decay': 0.1}, 'decoupled')])
def test_options_of_other_optimizers_refused(options, match):
    """A step that went on without them would turn around, or decay otherwise."""
    import FasterGSVDACudaBackend as F
    with pytest.raises(ValueError, match=match):
        F.FusedAdamW([{'params': [_param()], **options}])
    p = _param()
    opt = F.FusedAdamW([p], lr=0.5)
    opt.state[p] = {**opt._new_state(p, 32, False), 'step': 7}
    state = copy.deepcopy(opt.state_dict())
    state['param_groups'][0].update({'lr': 0.25, **options})
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(state)
    assert opt.param_groups[0]['lr'] == 0.5 and opt.state[p]['step'] == 7
    plain = {k: (False if v is True else v) for k, v in options.items()}
    if match == 'decoupled':
        plain['weight_decay'] = 0.0  # without a decay there is no difference
    state['param_groups'][0].update(plain)
    opt.load_state_dict(state)
    assert opt.param_groups[0]['lr'] == 0.25


@pytest.mark.parametrize('options', [{'maximize': True}, {'amsgrad': True}, {'decoupled_weight_decay': False, 'weight_decay': 0.1}])
def test_checkpoints_that_cannot_be_followed_are_refused(options):
    import FasterGSVDACudaBackend as F
    p = _param(6)
    make = torch.optim.Adam if 'decoupled_weight_decay' in options else torch.optim.AdamW
    ref = make([p], **{k: v for k, v in options.items() if k != 'decoupled_weight_decay'})
    ref.step()
    with pytest.raises(ValueError):
        F.FusedAdamW([p]).load_state_dict(ref.state_dict())


@pytest.mark.parametrize('options,match', [({'maximize': True}, 'maximize'), ({'amsgrad': 1}, 'amsgrad'), ({'differentiable': True}, 'differentiable'),
                                           ({'decoupled_weight_decay': False, 'weight_decay': 0.1}, 'decoupled')])
def test_options_set_on_a_group_are_refused_by_the_step(options, match):
    import FasterGSVDACudaBackend as F
    opt = F.FusedAdamW([_param()])
    opt.param_groups[0].update(options)
    with pytest.raises(RuntimeError, match=match):
        opt.step()
    assert not opt.state


def _stepped(n=300, step=7):
    import FasterGSVDACudaBackend as F
    p = _param(n, torch.bfloat16)
    opt = F.FusedAdamW([p], state_bits=8, master_weights=True)
    opt.state[p] = {**opt._new_state(p, 8, True), 'step': step}
    opt.state[p]['exp_avg'].random_(0, 256)
    opt.state[p]['master'] += 1e-4  # no bfloat16
    return p, opt


def test_hooks_around_loading():
    """Pre-hooks see the saved state and may change it, post-hooks see the loaded one; both before and after the call of
    this class's own."""
    _, saved = _stepped()
    p, opt = _stepped(step=3)
    seen = []

    def before(o, state_dict):
        assert o is opt
        seen.append((opt.state[p]['step'], state_dict['state'][0]['step']))
        state = {k: {**v, 'step': 99} for k, v in state_dict['state'].items()}
        return {**state_dict, 'state': state}

    def after(o):
        seen.append((opt.state[p]['step'], opt.state[p]['exp_avg'].dtype, dict(opt.param_groups[0])['state_bits']))

    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(after, prepend=True)
    source = saved.state_dict()
    kept = copy.deepcopy(source)
    opt.load_state_dict(source)
    assert seen == [(3, 7), (99, torch.uint8, 8)] and opt.state[p]['step'] == 99
    for name in ('exp_avg', 'master'):
        assert torch.equal(opt.state[p][name], kept['state'][0][name]) and opt.state[p][name].dtype == kept['state'][0][name].dtype
    assert source['state'][0]['step'] == 7  # the caller's dict is as it was
    opt.load_state_dict(source)
    assert len(seen) == 4


def test_post_hooks_see_the_options_of_this_class():
    import FasterGSVDACudaBackend as F
    p = _param(6)
    ref = torch.optim.AdamW([p])
    ref.step()
    opt = F.FusedAdamW([p])
    seen = []
    opt.register_load_state_dict_post_hook(lambda o: seen.append((o.param_groups[0]['state_bits'], o.state[p]['step'])))
    opt.load_state_dict(ref.state_dict())
    assert seen == [(32, 1)]


@pytest.mark.parametrize('spoil', [lambda s: s['state'][0].update(step=None), lambda s: s['state'][0].update(step='x'),
                                   lambda s: s['param_groups'].append(copy.deepcopy(s['param_groups'][0])),
                                   lambda s: s['param_groups'][0]['params'].append(1), lambda s: s.pop('state')])
def test_a_checkpoint_that_does_not_load_changes_nothing(spoil):
    p, opt = _stepped(step=3)
    opt.param_groups[0]['lr'] = 0.5
    before = copy.deepcopy(opt.state[p])
    _, saved = _stepped()
    bad = copy.deepcopy(saved.state_dict())
    spoil(bad)
    with pytest.raises((TypeError, ValueError, KeyError)):
        opt.load_state_dict(bad)
    assert opt.param_groups[0]['lr'] == 0.5 and list(opt.state) == [p] and opt.state[p].keys() == before.keys()
    assert all(torch.equal(opt.state[p][k], v) if torch.is_tensor(v) else opt.state[p][k] == v for k, v in before.items())
    opt.load_state_dict(saved.state_dict())  # and no hook is left behind
    assert opt.state[p]['step'] == 7 and opt.param_groups[0]['lr'] == 1e-3


def test_state_beside_the_moments_is_kept():
    """Entries of a user's own, of a parameter and of none, come back as they were."""
    p, saved = _stepped()
    saved.state[p]['note'] = {'a': [1, 2]}
    state = copy.deepcopy(saved.state_dict())
    state['state']['epoch'] = {'n': 5}
    q, opt = _stepped(step=3)
    opt.load_state_dict(state)
    assert opt.state[q]['note'] == {'a': [1, 2]} and opt.state['epoch'] == {'n': 5} and opt.state[q]['step'] == 7


@pytest.mark.parametrize('signed', [True, False], ids=['first moment', 'second moment'])
@pytest.mark.parametrize('e', [0, 1, 14, 15, 16, 30, 31, 32, 127, 200, 253, 254])
def test_every_code_keeps_its_value(e, signed):
    """All codes of a block whose largest exponent is e: values need no rounding, whatever the threshold. Codes below the
    smallest subnormal that the format holds (low exponents) stand for zero."""
    top = O.top_of(signed)
    q = np.arange(1, top)  # the code `top` has the next exponent
    codes = np.zeros(256, np.uint8)
    codes[:q.size] = q
    if signed:
        codes[q.size:2 * q.size] = q | 128
    x = O.decode(codes, np.array([e], np.uint8), signed)
    assert np.isfinite(x).all() and (x[q.size - 7:q.size] > 0).all() and np.unique(x[:q.size][x[:q.size] > 0]).size >= 7
    for step in (1, 2, 1000, 2 ** 31):
        got, exponents = O.encode(x, step, signed)
        assert exponents.tolist() == [e]
        np.testing.assert_array_equal(O.decode(got, exponents, signed), x)
    if e < 254:
        above = O.decode(np.array([top, top - 1], np.uint8), np.array([e], np.uint8), signed)
        got, exponents = O.encode(above, 5, signed)
        assert exponents.tolist() == [e + 1]
        np.testing.assert_array_equal(O.decode(got, exponents, signed), above)


def _run_coded(steps, n=4096, b1=0.9, b2=0.999):
    """Noisy gradients of many sizes, a tenth as large after step 1500, with the moments coded after every step and with
    moments in 64 bits: the mean relative difference of the second moments, and the updates' relative difference."""
    size = np.exp(np.random.default_rng(3).normal(0.0, 1.5, n))
    noise = np.random.default_rng(4)
    m, v = np.zeros(n), np.zeros(n)
    coded = [(np.zeros(n, np.uint8), np.zeros(n // O.BLOCK, np.uint8))] * 2
    for t in range(1, steps + 1):
        g = (noise.normal(0.3, 1.0, n) * size * (1.0 if t <= 1500 else 0.1)).astype(np.float32)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.astype(np.float64) ** 2
        m8, v8 = O.moments32(O.decode(*coded[0], True), O.decode(*coded[1], False), g, (b1, b2))
        coded = [O.encode(m8, t, True), O.encode(v8, t, False)]
    u, u8 = m / np.sqrt(v), m8 / np.sqrt(v8.astype(np.float64))
    return float((O.decode(*coded[1], False) / v).mean() - 1.0), float(np.linalg.norm(u8 - u) / np.linalg.norm(u))


def test_moments_in_8_bits_follow_those_in_64(monkeypatch):
    """Coding a value once is off by up to half a code step, 2^-4 of it. After 1000 steps the mean of the second moments is
    within that, and the updates are within a code step (2^-3); 1500 steps behind a drop of the gradients to a tenth the
    mean is within a code step, the updates within one and a half. With a fixed threshold, which is rounding to nearest,
    b2 = 0.999 leaves the second moment behind by more than half."""
    bias, off = _run_coded(1000)
    assert abs(bias) <= 2.0 ** -4 and off <= 2.0 ** -3, (bias, off)
    bias, off = _run_coded(3000)
    assert abs(bias) <= 2.0 ** -3 and off <= 1.5 * 2.0 ** -3, (bias, off)
    monkeypatch.setattr(O, 'thresholds', lambda count, step, signed: np.full(count, 2 ** 31, np.int64))
    assert _run_coded(1000)[0] < -0.5


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_step_within_a_compiled_function(backend):
    """torch.compile runs the step between its graphs."""
    import FasterGSVDACudaBackend as F
    p = _param(grad=False)
    opt = F.FusedAdamW([p], max_grad_norm=1.0)
    opt.grad_norm = 'old'
    torch._dynamo.reset()

    @torch.compile(backend=backend)
    def step(x):
        y = x * 2.0
        opt.step()
        return y + 1.0

    assert torch.equal(step(torch.ones(2)), torch.full((2,), 3.0)) and opt.grad_norm is None
    p.grad = torch.ones(5)
    with pytest.raises(RuntimeError, match='CUDA'):
        step(torch.ones(2))


def test_freed_storages_refused():
    """Storages that were resized beneath their tensors: views within them keep an address."""
    import FasterGSVDACudaBackend as F
    flat = torch.ones(20)
    p = torch.nn.Parameter(flat[10:15])
    p.grad = torch.ones(5)
    flat.untyped_storage().resize_(14 * 4)
    with pytest.raises(RuntimeError, match='a parameter has less memory'):
        F.FusedAdamW([p]).step()
    with pytest.raises(RuntimeError, match='an output has less memory'):
        F.FusedAdamW([_param()]).read_moments([p.detach()], [torch.zeros(5)])


@pytest.mark.parametrize('change', [
    {'tensors': {'param': (ctypes.c_uint64 * 1)(66)}}, {'tensors': {'grad': (ctypes.c_uint64 * 1)(65)}}, {'tensors': {'exp_avg': (ctypes.c_uint64 * 1)(66)}},
    {'tensors': {'exp_avg_sq': (ctypes.c_uint64 * 1)(67)}}, {'dtype': 1, 'tensors': {'param': (ctypes.c_uint64 * 1)(65)}},
    {'dtype': 1, 'tensors': {'master': (ctypes.c_uint64 * 1)(66)}}, {'partials': 68, 'norm': 64, 'max_norm': 1.0}, {'partials': 64, 'norm': 66, 'max_norm': 1.0}])
def test_c_entry_refuses_misaligned_pointers(change):
    """A kernel would fault on an address that is no multiple of its elements' size."""
    with pytest.raises(RuntimeError, match='aligned'):
        _abi_call(**change)


def test_c_entries_of_the_norm_and_the_moments_refuse_misaligned_pointers():
    from FasterGSVDACudaBackend import _lib
    lib, check = _lib.lib, _lib.check
    room, used = ctypes.c_int(0), ctypes.c_int(0)
    check(lib.fgs_grad_squares_capacity(1, ctypes.byref(room)))
    ptr, odd, n, kind, a = (ctypes.c_uint64 * 1)(64), (ctypes.c_uint64 * 1)(66), (ctypes.c_int64 * 1)(4), (ctypes.c_uint8 * 1)(0), ctypes.addressof
    with pytest.raises(RuntimeError, match='gradient pointer is not aligned'):
        check(lib.fgs_grad_squares(a(odd), a(n), a(kind), 1, 64, room.value, ctypes.byref(used), None))
    with pytest.raises(RuntimeError, match='partials is not aligned'):
        check(lib.fgs_grad_squares(a(ptr), a(n), a(kind), 1, 68, room.value, ctypes.byref(used), None))
    with pytest.raises(RuntimeError, match='output pointer is not aligned'):
        check(lib.fgs_adamw_read_moments(a(ptr), a(ptr), a(kind), a(n), 1, a(odd), 0, None))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_half_precision_moments_of_another_adamw_load(dtype):
    """torch's AdamW keeps its moments in the parameters' type; here they are float32, with the same values."""
    import FasterGSVDACudaBackend as F
    p = _param(6, dtype)
    ref = torch.optim.AdamW([p])
    ref.step()
    opt = F.FusedAdamW([p])
    opt.load_state_dict(ref.state_dict())
    for name in ('exp_avg', 'exp_avg_sq'):
        assert opt.state[p][name].dtype == torch.float32 and torch.equal(opt.state[p][name], ref.state[p][name].float())
        assert ref.state[p][name].dtype == dtype
