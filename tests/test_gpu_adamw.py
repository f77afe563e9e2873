"""FusedAdamW on the GPU against its formula in 64 bits (tolerances counted in roundings: oracle/adamw.py bounds) and, for
8-bit moments, bit for bit against the restatement of the block format."""
import copy
import warnings

import numpy as np
import pytest
import torch

from oracle import adamw as O

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half the subnormals' spacing


def _np(t):
    return t.detach().float().cpu().numpy().reshape(-1)


def _snapshot(opt):
    """Everything a step reads, as arrays: per parameter (p, m, v, codes, exponents, step)."""
    m, v = opt.read_moments()
    out = []
    for p, a, b in zip([p for g in opt.param_groups for p in g['params']], m, v):
        s = opt.state.get(p) or {}
        out.append({'p': _np(s['master']) if 'master' in s else _np(p), 'm': _np(a), 'v': _np(b), 'step': s.get('step', 0),
                    'param': _np(p)})
    return out


def _check(opt, before, clip=1.0, clipped=False):
    """Compares the optimizer after a step with the formula applied to the snapshot taken before it."""
    m, v = opt.read_moments()
    i = 0
    for group in opt.param_groups:
        for p in group['params']:
            b, mi, vi = before[i], _np(m[i]), _np(v[i])
            i += 1
            if p.grad is None:
                np.testing.assert_array_equal(_np(p), b['param'])
                continue
            s = opt.state[p]
            g = _np(p.grad)
            args = (b['p'], b['m'], b['v'], clip * g.astype(np.float64) if clipped else g, b['step'] + 1, group['lr'], group['betas'], group['eps'],
                    group['weight_decay'])
            assert s['step'] == b['step'] + 1
            wp, wm, wv = O.step64(*args)
            dp, dm, dv = O.bounds(*args, clipped)
            if 'master' in s:
                assert (np.abs(_np(s['master']) - wp) <= dp).all()
                np.testing.assert_array_equal(_np(p), _np(s['master'].to(p.dtype)))
            else:
                err = np.abs(_np(p) - wp)
                assert (err <= dp + HALF_STEP[p.dtype] * (np.abs(wp) + dp) + SMALLEST[p.dtype]).all(), float((err - dp).max())
            if group['state_bits'] == 32:
                assert (np.abs(mi - wm) <= dm).all() and (np.abs(vi - wv) <= dv).all()
            elif not clipped:
                m32, v32 = O.moments32(b['m'], b['v'], g, group['betas'])
                for name, x, signed in (('exp_avg', m32, True), ('exp_avg_sq', v32, False)):
                    q, e = O.encode(x, b['step'] + 1, signed)
                    np.testing.assert_array_equal(s[name + '_exponent'].cpu().numpy(), e, err_msg=name)
                    np.testing.assert_array_equal(s[name].cpu().numpy().reshape(-1), q, err_msg=name)
            else:  # the clip factor itself carries a few roundings: codes within one step of the value's, 2^-3 of it
                for x, w, top, spread in ((mi, wm, 127, 16), (vi, wv, 255, 32)):
                    high = np.abs(np.pad(w, (0, -w.size % 256))).reshape(-1, 256).max(1).repeat(256)[:w.size]
                    assert (np.abs(x - w) <= 0.1251 * np.abs(w) + 2.0 ** (2 - spread) * high).all()


SHAPES = [(1000, 3), (5000, 15, 3), (1,), (255,), (256,), (257,), (64, 80), (0,), (7, 1, 3)]


def _params(shapes, dtype, device, seed=0, misalign=False):
    g = torch.Generator().manual_seed(seed)
    out = []
    for s in shapes:
        n = int(np.prod(s))
        x = torch.randn(n + 3, generator=g).to(dtype).to(device)
        out.append(torch.nn.Parameter(x[3:].view(s) if misalign else x[3:].clone().view(s)))
    return out


def _grads(params, step, seed=0):
    g = torch.Generator().manual_seed(1000 * step + seed)
    for i, p in enumerate(params):
        size = torch.exp(torch.randn(p.shape, generator=g) * 2.0)  # several orders of magnitude within a block
        p.grad = (torch.randn(p.shape, generator=g) * size * 10.0 ** (i % 4 - 2)).to(p.dtype).to(p.device)


@pytest.mark.parametrize('misalign', [False, True], ids=['aligned', 'odd addresses'])
@pytest.mark.parametrize('clip', [False, True], ids=['plain', 'clipped'])
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype,master', [(torch.float32, False), (torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False),
                                          (torch.float16, True)], ids=['fp32', 'bf16', 'bf16 master', 'fp16', 'fp16 master'])
def test_steps_against_the_formula(cuda, dtype, master, bits, clip, misalign):
    import FasterGSVDACudaBackend as F
    params = _params(SHAPES, dtype, cuda, misalign=misalign)
    opt = F.FusedAdamW(params, lr=3e-3, weight_decay=0.1, state_bits=bits, master_weights=master, max_grad_norm=0.7 if clip else None)
    for step in range(1, 5):
        _grads(params, step)
        before = _snapshot(opt)
        if master and step == 1:
            for b in before:
                b['p'] = b['param']
        grads = [p.grad.clone() for p in params]
        opt.step()
        factor = 1.0
        if clip:
            norm = np.sqrt(sum((_np(p.grad).astype(np.float64) ** 2).sum() for p in params))
            # squares summed 32 at a time in float32 (33 roundings), half of that on the root, and the conversion
            assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
            factor = min(1.0, 0.7 / (norm + 1e-6))
            assert factor < 1.0
        _check(opt, before, factor, clip)
        for p, g in zip(params, grads):
            assert torch.equal(p.grad, g)


def test_norm_below_the_limit_changes_nothing(cuda):
    import FasterGSVDACudaBackend as F
    a, b, c = (_params(SHAPES, torch.float32, cuda) for _ in range(3))
    one, two, three = F.FusedAdamW(a), F.FusedAdamW(b, max_grad_norm=1e9), F.FusedAdamW(c, max_grad_norm=float('inf'))
    for params, opt in ((a, one), (b, two), (c, three)):
        _grads(params, 1)
        opt.step()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)
    assert torch.equal(two.grad_norm, three.grad_norm)
    assert one.grad_norm is None and two.grad_norm.shape == ()


@pytest.mark.parametrize('bits', [32, 8])
def test_more_tensors_than_one_launch_takes(cuda, bits):
    """1100 tensors: three update launches, two launches of the norm, and sizes that leave most chunks short."""
    import FasterGSVDACudaBackend as F
    params = _params([(1 + (37 * i) % 900,) for i in range(1100)], torch.float32, cuda)
    opt = F.FusedAdamW(params, state_bits=bits, max_grad_norm=1.0)
    for step in (1, 2):
        _grads(params, step)
        before = _snapshot(opt)
        opt.step()
        norm = np.sqrt(sum((_np(p.grad).astype(np.float64) ** 2).sum() for p in params))
        assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
        _check(opt, before, 1.0 / (norm + 1e-6), True)


def test_long_tensor(cuda):
    """More chunks than CTAs, several rounds per chunk, and a last block that is cut."""
    import FasterGSVDACudaBackend as F
    n = 12_000_000 + 77
    p = torch.nn.Parameter(torch.randn(n, device=cuda, generator=torch.Generator(cuda).manual_seed(0)))
    opt = F.FusedAdamW([p], state_bits=8)
    for step in (1, 2):
        p.grad = torch.randn(n, device=cuda, generator=torch.Generator(cuda).manual_seed(step))
        before = _snapshot(opt)
        opt.step()
        _check(opt, before)


def test_groups_types_and_step_counts(cuda):
    """Nine groups with their own hyperparameters (more than one launch's table of them), learning rates per column,
    mixed types and kinds of state, and parameters that miss steps."""
    import FasterGSVDACudaBackend as F
    groups, params = [], []
    for i in range(9):
        dtype = (torch.float32, torch.bfloat16, torch.float16)[i % 3]
        ps = _params([(40, 7), (513,)], dtype, cuda, seed=i)
        params += ps
        lr = [1e-3 * (k + 1) for k in range(7)] if i == 3 else 1e-3 * (i + 1)
        groups.append({'params': ps, 'lr': lr, 'betas': (0.8 + 0.01 * i, 0.99), 'eps': 10.0 ** -(4 + i), 'weight_decay': 0.01 * i,
                       'state_bits': 8 if i % 2 else 32, 'master_weights': i % 4 == 1})
    opt = F.FusedAdamW(groups)
    for step in range(1, 5):
        _grads(params, step)
        for i, p in enumerate(params):
            if (i + step) % 3 == 0:
                p.grad = None
        before = _snapshot(opt)
        for b, p in zip(before, params):
            if 'master' not in (opt.state.get(p) or {}):
                b['p'] = b['param']
        opt.step()
        _check(opt, before)
    assert len({s['step'] for s in opt.state.values()}) > 1


@pytest.mark.parametrize('bits', [32, 8])
def test_infinite_and_nan_gradients_stay_where_they_are(cuda, bits):
    """Without clipping an infinity or NaN reaches its own element (32 bits) or its own block of 256 moments (8 bits)."""
    import FasterGSVDACudaBackend as F
    params = _params([(1024,)], torch.float32, cuda)
    p = params[0]
    opt = F.FusedAdamW(params, state_bits=bits)
    p.grad = torch.ones_like(p)
    p.grad[300], p.grad[700] = float('inf'), float('nan')
    opt.step()
    bad = ~torch.isfinite(p.detach())
    assert bad[[300, 700]].all() and bad.sum() == 2
    m, v = opt.read_moments()
    for x in (m[0], v[0]):
        bad = ~torch.isfinite(x)
        if bits == 32:
            assert bad.sum() == 2
        else:
            assert torch.isnan(x[256:512]).all() and torch.isnan(x[512:768]).all() and bad.sum() == 512


def test_clipping_with_nan_reaches_everything(cuda):
    import FasterGSVDACudaBackend as F
    params = _params([(1024,), (3,)], torch.float32, cuda)
    opt = F.FusedAdamW(params, max_grad_norm=1.0)
    _grads(params, 1)
    params[0].grad[5] = float('nan')
    opt.step()
    assert torch.isnan(opt.grad_norm) and all(torch.isnan(p).all() for p in params)


def test_extremes_of_the_8_bit_range(cuda):
    """Blocks of subnormal values only, of zeros, next to the largest float, and over 40 octaves."""
    import FasterGSVDACudaBackend as F
    p = torch.nn.Parameter(torch.zeros(5 * 256 + 9, device=cuda))
    opt = F.FusedAdamW([p], state_bits=8, betas=(0.0, 0.0), eps=1.0)
    g = torch.zeros(p.numel())
    r = torch.Generator().manual_seed(0)
    g[:256] = torch.rand(256, generator=r) * 1e-39
    g[512:768] = torch.rand(256, generator=r) * 3.4e38
    g[768:1024] = torch.exp2(-torch.arange(256) * 0.2)
    g[1024:1280] = torch.rand(256, generator=r) * 1.7e19
    for step in (1, 2, 3):
        p.grad = g.to(cuda)
        before = _snapshot(opt)
        opt.step()
        m32, v32 = O.moments32(before[0]['m'], before[0]['v'], g.numpy(), (0.0, 0.0))
        m32 = np.where(np.isnan(m32), g.numpy(), m32)  # 0 * NaN of a block that overflowed before
        s = opt.state[p]
        q, e = O.encode(m32, step, True)
        ok = np.repeat(np.isfinite(np.pad(before[0]['m'], (0, -p.numel() % 256)).reshape(-1, 256)).all(1), 256)[:p.numel()]
        np.testing.assert_array_equal(s['exp_avg'].cpu().numpy()[ok], q[ok])
        fine = np.isfinite(v32) & ok
        fine &= np.repeat(np.pad(fine, (0, -p.numel() % 256), constant_values=True).reshape(-1, 256).all(1), 256)[:p.numel()]
        q, e = O.encode(np.where(fine, v32, 0), step, False)
        np.testing.assert_array_equal(s['exp_avg_sq'].cpu().numpy()[fine], q[fine])
        m, v = opt.read_moments()
        assert torch.isfinite(m[0]).all()


def test_save_load_continue(cuda):
    """A loaded optimizer goes on bit for bit as the saved one would have."""
    import FasterGSVDACudaBackend as F
    a = _params(SHAPES, torch.bfloat16, cuda)
    one = F.FusedAdamW(a, state_bits=8, master_weights=True)
    _grads(a, 1)
    one.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    two = F.FusedAdamW(b, state_bits=8, master_weights=True)
    two.load_state_dict(copy.deepcopy(one.state_dict()))
    for params, opt in ((a, one), (b, two)):
        for step in (2, 3):
            _grads(params, step)
            opt.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k, x in one.state[p].items():
            assert torch.equal(x, two.state[q][k]) if torch.is_tensor(x) else x == two.state[q][k]


def test_other_stream_and_repeat(cuda):
    """The kernels run on the current stream, and the same inputs give the same bits."""
    import FasterGSVDACudaBackend as F
    results = []
    for k in range(3):
        params = _params([(70_000,), (33,)], torch.float32, cuda)
        opt = F.FusedAdamW(params, state_bits=8, max_grad_norm=0.1)
        stream = torch.cuda.Stream() if k else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for step in (1, 2):
                _grads(params, step)
                opt.step()
        torch.cuda.current_stream().wait_stream(stream)
        results.append([x.clone() for p in params for x in (p.detach(), opt.state[p]['exp_avg'], opt.state[p]['exp_avg_sq'])] + [opt.grad_norm])
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))


def test_refusals_leave_everything_as_it_was(cuda):
    import FasterGSVDACudaBackend as F
    p, q = _params([(40, 6), (8, 4)], torch.float32, cuda)
    opt = F.FusedAdamW([p, q])
    _grads([p, q], 1)
    opt.step()
    keep = [p.detach().clone(), q.detach().clone()]
    q.grad = torch.ones(4, 8, device=cuda).t()
    with pytest.raises(RuntimeError, match='contiguous'):
        opt.step()
    q.grad = torch.ones(8, 4, device=cuda)
    state = opt.state[q]
    good = state['exp_avg']
    for bad, match in ((good[:4], 'elements'), (good.half(), 'float32'), (good.cpu(), 'CUDA')):
        state['exp_avg'] = bad.contiguous()
        with pytest.raises(RuntimeError, match=match):
            opt.step()
    state['exp_avg'] = good
    opt.param_groups[0]['state_bits'] = 8
    with pytest.raises(RuntimeError):
        opt.step()
    opt.param_groups[0]['state_bits'] = 32
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='captured'):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach(), keep[0]) and torch.equal(q.detach(), keep[1]) and opt.state[p]['step'] == opt.state[q]['step'] == 1
    opt.step()
    assert opt.state[p]['step'] == 2


def test_moments_into_given_tensors(cuda):
    """bfloat16 holds the 8-bit moments' values exactly; parameters without state read as zero."""
    import FasterGSVDACudaBackend as F
    params = _params([(1000,), (3, 5)], torch.float32, cuda)
    opt = F.FusedAdamW(params, state_bits=8)
    _grads(params, 1)
    params[1].grad = None
    opt.step()
    m, v = opt.read_moments()
    to = [[torch.full(p.shape, 7.0, dtype=torch.bfloat16, device=cuda) for p in params] for _ in range(2)]
    opt.read_moments(*to)
    for a, b in zip(m + v, to[0] + to[1]):
        assert torch.equal(a, b.float())
    assert not m[1].any() and not v[1].any()
    with pytest.raises(ValueError):
        opt.read_moments(to[0], None)
    with pytest.raises(ValueError):
        opt.read_moments(to[0][:1], to[1])
    with pytest.raises(ValueError):
        opt.read_moments([to[0][0][:5], to[0][1]], to[1])
    with pytest.raises(RuntimeError):
        opt.read_moments([x.half() for x in to[0]], [x.half() for x in to[1]])


def test_closure_hooks_and_schedulers(cuda):
    """What torch's optimizers offer around a step: a closure with gradients enabled, hooks, and learning-rate schedulers."""
    import FasterGSVDACudaBackend as F
    p = torch.nn.Parameter(torch.ones(300, device=cuda))
    opt = F.FusedAdamW([p], lr=0.1, max_grad_norm=2.0)
    schedule = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)
    seen = []
    opt.register_step_post_hook(lambda *a: seen.append('after'))

    def closure():
        opt.zero_grad()
        loss = (p ** 2).sum()
        loss.backward()
        return loss

    with torch.no_grad():
        before = _snapshot(opt)
        loss = opt.step(closure)
    assert float(loss.detach()) == 300.0 and seen == ['after']
    norm = 2.0 * np.sqrt(300.0)
    assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
    _check(opt, before, 2.0 / (norm + 1e-6), True)
    schedule.step()
    assert opt.param_groups[0]['lr'] == 0.05
    opt.max_grad_norm = None
    before = _snapshot(opt)
    opt.step()
    assert opt.grad_norm is None
    _check(opt, before)


def test_two_optimizers_at_once(cuda):
    """Steps of two optimizers on two streams do not share anything: the bits of each by itself."""
    import FasterGSVDACudaBackend as F

    def make(seed):
        params = _params([(400_000,), (9,)], torch.float32, cuda, seed=seed)
        _grads(params, 1, seed)
        return params, F.FusedAdamW(params, state_bits=8, max_grad_norm=0.5)

    alone = []
    for seed in (0, 1):
        params, opt = make(seed)
        for _ in range(4):
            opt.step()
        alone.append(([p.detach().clone() for p in params], opt.grad_norm.clone()))
    both = [make(0), make(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for (params, opt), s in zip(both, streams):
            with torch.cuda.stream(s):
                opt.step()
    torch.cuda.synchronize()
    for (params, opt), (ref, norm) in zip(both, alone):
        assert all(torch.equal(p, q) for p, q in zip(params, ref)) and torch.equal(opt.grad_norm, norm)


def test_more_than_2_31_elements(cuda):
    """One tensor whose offsets pass 32 bits, looked at around its begin, 2^31 and its end."""
    import FasterGSVDACudaBackend as F
    n = 2 ** 31 + 1000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=cuda))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    places = [slice(0, 512), slice(2 ** 31 - 512, 2 ** 31 + 256), slice(n - 1000, n)]
    r = torch.Generator().manual_seed(0)
    for k in places:
        p.grad[k] = torch.randn(k.stop - k.start, generator=r).bfloat16().to(cuda)
    opt = F.FusedAdamW([p], lr=0.5, state_bits=8, weight_decay=0.0)
    opt.step()
    s = opt.state[p]
    for k in places:
        g = _np(p.grad[k])
        w, _, _ = O.step64(np.zeros_like(g), np.zeros_like(g), np.zeros_like(g), g, 1, 0.5, (0.9, 0.999), 1e-8, 0.0)
        assert (np.abs(_np(p[k]) - w) <= (2.0 ** -8 + 2.0 ** -19) * np.abs(w) + 2.0 ** -134).all()
        m32, v32 = O.moments32(np.zeros_like(g), np.zeros_like(g), g, (0.9, 0.999))
        first = k.start  # a multiple of 256, but for the thresholds' element numbers, which are the tensor's
        assert first % 256 == 0 or k.stop == n
        first = first // 256 * 256
        lead = k.start - first
        for name, x, signed in (('exp_avg', m32, True), ('exp_avg_sq', v32, False)):
            full = np.zeros(k.stop - first, np.float32)
            full[lead:] = x
            turn = first * O.TURN
            shift = O.thresholds(full.size, 1, signed)
            wrapped = (shift + turn) & 0xFFFFFFFF
            keep = O.thresholds
            O.thresholds = lambda *a: wrapped
            try:
                q, e = O.encode(full, 1, signed)
            finally:
                O.thresholds = keep
            np.testing.assert_array_equal(s[name][first:k.stop].cpu().numpy(), q)
            np.testing.assert_array_equal(s[name + '_exponent'][first // 256:first // 256 + e.size].cpu().numpy(), e)


def test_parameters_of_one_memory_are_refused(cuda):
    """The same parameter twice, or two that overlap, would be updated by two threads at once; neighbours are not touched."""
    import FasterGSVDACudaBackend as F
    flat = torch.ones(1024, device=cuda)
    a, b = (torch.nn.Parameter(flat[s]) for s in (slice(0, 512), slice(512, 1024)))
    c = torch.nn.Parameter(flat[500:600])
    half = torch.nn.Parameter(flat[508:512].view(torch.bfloat16))
    empty = torch.nn.Parameter(flat[100:100])
    for p in (a, b, c, half, empty):
        p.grad = torch.ones_like(p)
    with warnings.catch_warnings():
        warnings.simplefilter('ignore')
        twice = F.FusedAdamW([b, a, b])
    for opt in (twice, F.FusedAdamW([a, c]), F.FusedAdamW([c, b]), F.FusedAdamW([half, b, a])):
        with pytest.raises(RuntimeError, match='share memory'):
            opt.step()
        assert all(not opt.state[p] for p in (a, b, c, half))
    torch.cuda.synchronize()
    assert (flat == 1).all()
    F.FusedAdamW([b, empty, a]).step()
    assert (flat < 1).all()


@pytest.mark.parametrize('clip', [None, 1.0])
def test_a_step_is_a_change_in_place_for_autograd(cuda, clip):
    """A graph that saved a parameter before the step must not go on with the new values; read moments neither."""
    import FasterGSVDACudaBackend as F
    p, idle = _params([(40, 6), (8,)], torch.float32, cuda)
    opt = F.FusedAdamW([p, idle], max_grad_norm=clip)
    loss, other = (p * p).sum(), (idle * idle).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    other.backward()  # not updated: as it was
    outs = [[torch.zeros(40, 6, device=cuda), torch.zeros(8, device=cuda)] for _ in range(2)]
    x = torch.ones(40, 6, device=cuda, requires_grad=True)
    loss = (x * outs[0][0]).sum()
    opt.read_moments(*outs)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


@pytest.mark.parametrize('bits', [32, 8])
def test_moments_into_shared_memory_are_refused(cuda, bits):
    import FasterGSVDACudaBackend as F
    p, = _params([(40, 6)], torch.float32, cuda)
    p.grad = torch.ones_like(p)
    opt = F.FusedAdamW([p], state_bits=bits)
    opt.step()
    flat = torch.full((480,), 7.0, device=cuda)
    whole, apart = flat[:240].view(40, 6), flat[240:].view(40, 6)
    for a, b in ((whole, whole), (whole, flat[239:479].view(40, 6))):
        with pytest.raises(RuntimeError, match='share memory'):
            opt.read_moments([a], [b])
    torch.cuda.synchronize()
    assert (flat == 7).all()
    opt.read_moments([whole], [apart])
    assert (flat != 7).all()


def test_lazily_negated_gradients_are_refused(cuda):
    import FasterGSVDACudaBackend as F
    p = torch.nn.Parameter(torch.ones(300, device=cuda))
    p.grad = torch._neg_view(torch.ones(300, device=cuda))
    opt = F.FusedAdamW([p])
    with pytest.raises(RuntimeError, match='a gradient must not be a lazily negated view'):
        opt.step()
    assert (p == 1).all()
    p.grad = p.grad.resolve_neg()
    opt.step()
    assert (p > 1 - 1e-2).all() and not (p == 1).any()
    with pytest.raises(RuntimeError, match='an output must not be a lazily negated view'):
        opt.read_moments([torch._neg_view(torch.empty(300, device=cuda))], [torch.empty(300, device=cuda)])


def test_a_refused_first_step_makes_no_state(cuda, monkeypatch):
    """Refusals come before the state of new parameters is made and filled: on the device, or into a graph under capture."""
    import FasterGSVDACudaBackend as F
    made = []
    new_state = F.FusedAdamW._new_state
    monkeypatch.setattr(F.FusedAdamW, '_new_state', staticmethod(lambda *a: made.append(1) or new_state(*a)))
    p, q = _params([(40, 6), (8, 4)], torch.bfloat16, cuda)
    flat = torch.ones(600, device=cuda)
    a, b = torch.nn.Parameter(flat[:400]), torch.nn.Parameter(flat[200:])
    good = [torch.ones_like(x) for x in (p, q, a, b)]

    def refused(params, match, grads=good, **options):
        for x, g in zip((p, q, a, b), grads):
            x.grad = g
        opt = F.FusedAdamW(params, state_bits=8, master_weights=True)
        opt.param_groups[-1].update(options)
        opt.max_grad_norm = 1.0
        with pytest.raises((RuntimeError, TypeError), match=match):
            opt.step()
        assert not opt.state and not made
        return opt

    refused([p, q], 'contiguous', [good[0], torch.ones(4, 8, dtype=torch.bfloat16, device=cuda).t()] + good[2:])
    refused([p, a, b], 'share memory')
    refused([{'params': [p]}, {'params': [q]}], 'betas', betas=(0.9, 1.0))
    refused([{'params': [p]}, {'params': [q]}], 'betas', betas=(float('nan'), 0.9))
    refused([{'params': [p]}, {'params': [q]}], 'eps', eps=-1.0)
    refused([{'params': [p]}, {'params': [q]}], 'eps', eps=1e-40)
    refused([{'params': [p]}, {'params': [q]}], 'learning rates', lr=[])
    refused([{'params': [p]}, {'params': [q]}], 'real number', lr='x')
    opt = F.FusedAdamW([p, q], state_bits=8)
    graph = torch.cuda.CUDAGraph()
    x = torch.ones(3, device=cuda)
    with pytest.raises(RuntimeError, match='captured'):
        with torch.cuda.graph(graph):
            x += 1
            opt.step()
    torch.cuda.synchronize()
    assert not opt.state and not made
    opt.step()
    assert len(made) == 2 and opt.state[p]['step'] == opt.state[q]['step'] == 1


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('limit', [0.7, 1e9], ids=['clipped', 'below the limit'])
@pytest.mark.parametrize('shapes,dtypes', [
    ([(10_500_000 + 77,)], (torch.float32,)),                                        # one launch of many CTAs: the factor is made once
    ([(26_000 + i % 5,) for i in range(770)], (torch.float32,)),                     # two such launches and a short one behind them
    ([(10_100_000,), (9_900_000 + 3,), (300,), (7, 5)], (torch.bfloat16, torch.float32)),  # two types, one norm
    ([(1 + (977 * i) % 5000,) for i in range(60)], (torch.float32, torch.float16)),  # tables of the middle size
], ids=['long', 'many', 'two types', '60 tensors'])
def test_long_clipped_steps(cuda, shapes, dtypes, limit, bits):
    import FasterGSVDACudaBackend as F
    params = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.randn(s, device=cuda, generator=torch.Generator(cuda).manual_seed(i)).to(dtypes[i % len(dtypes)]))
        p.grad = (torch.randn(s, device=cuda, generator=torch.Generator(cuda).manual_seed(10_000 + i)) * 10.0 ** (i % 3 - 1)).to(p.dtype)
        params.append(p)
    opt = F.FusedAdamW(params, state_bits=bits, master_weights=True, max_grad_norm=limit)
    norm = np.sqrt(sum((_np(p.grad).astype(np.float64) ** 2).sum() for p in params))
    for _ in range(2):
        before = _snapshot(opt)
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
        _check(opt, before, min(1.0, limit / (norm + 1e-6)), True)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_clipping_of_gradients_whose_squares_overflow(cuda, dtype, bits):
    """Finite gradients up to 1e30, whose squares are no float32 but whose norm is: clipped like others. In whole accesses,
    in the rest behind them, and in tensors at odd addresses."""
    import FasterGSVDACudaBackend as F
    for misalign in (False, True):
        params = _params([(5000,), (7, 3), (8192 * 3 + 5,)], dtype, cuda, misalign=misalign)
        opt = F.FusedAdamW(params, state_bits=bits, max_grad_norm=1.0)
        _grads(params, 1)
        params[0].grad[17], params[0].grad[4999], params[1].grad[6, 2], params[2].grad[8192 * 3 + 1] = 1e30, 3e29, -1e25, 2e19
        norm = np.sqrt(sum((_np(p.grad).astype(np.float64) ** 2).sum() for p in params))
        before = _snapshot(opt)
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 18 * 2.0 ** -24 * norm
        assert all(torch.isfinite(p).all() for p in params)
        if bits == 32:
            _check(opt, before, 1.0 / (norm + 1e-6), True)
    params[0].grad[18] = float('inf')
    opt.step()
    assert torch.isinf(opt.grad_norm)


def test_goes_on_from_a_checkpoint_of_another_adamw(cuda):
    import FasterGSVDACudaBackend as F
    params = _params([(300,), (8, 5)], torch.bfloat16, cuda)
    ref = torch.optim.AdamW(params, lr=0.02, weight_decay=0.1)
    for step in (1, 2):
        _grads(params, step)
        ref.step()
    opt = F.FusedAdamW(params)
    opt.load_state_dict(ref.state_dict())
    _grads(params, 3)
    before = _snapshot(opt)
    assert all(b['step'] == 2 and b['m'].any() for b in before)
    opt.step()
    _check(opt, before)
