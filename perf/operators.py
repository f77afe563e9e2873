"""Timing cases of the training-side operators: the AdamW step over many tensors (states in 32 or in 8 bits, with the
global gradient norm that clips it) and the scaled embedding lookup with its gradient.

run() computes a pass in plain torch operations, or, where `own` is set, through the library's entry points."""
import math
import random
import sys

import torch

own = False

BLOCK = 256  # elements that share one exponent where the moments are held in 8 bits
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.01, 1e-3
FIRST_STEP = 40  # the optimizer's state is that of a run under way


def _library():
    import os
    root = os.path.join(os.getcwd(), 'efficient-gaussian-appearance_b200')
    if root not in sys.path:
        sys.path.insert(0, root)
    import FasterGSVDACudaBackend
    return FasterGSVDACudaBackend


# ---------------------------------------------------------------------------------------------------------------
# cases

def _adamw(name, dtype, bits, clip, master, widths='', rows=0, tensors=0, total=0, mix=0):
    return {'name': name, 'op': 'adamw', 'dtype': dtype, 'bits': bits, 'clip': clip, 'master': master, 'widths': widths, 'rows': rows,
            'tensors': tensors, 'total': total, 'mix': mix}


def _embed(name, train, dtype, rows, width, tokens, spread, absent, wide):
    return {'name': name, 'op': 'embed', 'train': train, 'dtype': dtype, 'rows': rows, 'width': width, 'tokens': tokens, 'spread': spread,
            'absent': absent, 'wide': wide}


def listed():
    return [
        # the weights of one small network (the c4 workload's MLP): a single tensor, latency only
        _adamw('step one MLP', 'fp32', 32, False, False, widths='10240', rows=1),
        # the SH-3 scene of 1M Gaussians (means, scales, rotations, opacities, base colours, residuals), moments in 32 and 8 bits
        _adamw('step SH-3 scene', 'fp32', 32, False, False, widths='3,3,4,1,3,45', rows=1_000_000),
        _adamw('step SH-3 scene 8 bits', 'fp32', 8, False, False, widths='3,3,4,1,3,45', rows=1_000_000),
        # many tensors of mixed sizes in half precision, clipped by the global norm, with a float copy of the weights
        _adamw('clipped step 300 tensors', 'bf16', 32, True, True, tensors=300, total=40_000_000, mix=1),
        _adamw('clipped step 300 tensors 8 bits', 'bf16', 8, True, False, tensors=300, total=40_000_000, mix=1),
        # a few odd-sized tensors with clipping: what a fine-tuning run updates
        _adamw('clipped step 13 tensors 8 bits', 'fp32', 8, True, True, tensors=13, total=77_777, mix=2),
        # one token of a serving step; rows of a wide table
        _embed('lookup one token', False, 'bf16', 32_000, 4096, 1, 'zipf', 0.0, False),
        # a prompt batch
        _embed('lookup 32k tokens', False, 'bf16', 32_000, 2048, 32_768, 'zipf', 0.0, True),
        # latent rows shared by 2M Gaussians: a codebook of 32 features, as the neural appearance model reads them
        _embed('lookup codebook', False, 'fp32', 4096, 32, 2_000_000, 'even', 0.0, True),
        # training passes: a short batch with padding, a vocabulary with its usual skew, and the codebook
        _embed('train 257 tokens', True, 'fp32', 5000, 769, 257, 'zipf', 0.1, True),
        _embed('train 32k tokens', True, 'bf16', 50_000, 1024, 32_768, 'zipf', 0.05, True),
        _embed('train codebook', True, 'fp32', 4096, 32, 2_000_000, 'even', 0.0, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        dtype = rng.choice(['fp32', 'fp32', 'bf16', 'fp16'])
        tensors = _log(rng, 1, 400)
        total = max(tensors, _log(rng, 1000, 40_000_000))
        c = _adamw('', dtype, rng.choice([32, 8]), rng.random() < 0.5, rng.random() < 0.5, tensors=tensors, total=total, mix=rng.randrange(1 << 20))
    else:
        width = _log(rng, 1, 4096)
        tokens = _log(rng, 1, min(2_000_000, (1 << 25) // width))
        rows = _log(rng, 1, min(200_000, (1 << 25) // width))
        c = _embed('', rng.random() < 0.6, rng.choice(['fp32', 'bf16', 'fp16']), rows, width, tokens, rng.choice(['zipf', 'even', 'runs']),
                   rng.choice([0.0, 0.0, 0.1, 1.0 / 3]), rng.random() < 0.5)
    del c['name']
    return c


def _sizes(case):
    """Elements of each tensor of an AdamW case."""
    if case['widths']:
        return [case['rows'] * int(w) for w in case['widths'].split(',')]
    rng = random.Random(case['mix'])  # mixed sizes over a factor of a few hundred, odd ones among them
    share = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case['tensors'])]
    left = case['total'] - case['tensors']
    return [1 + int(left * s / sum(share)) for s in share]


# ---------------------------------------------------------------------------------------------------------------
# the state a training program holds

def _encode(x, signed):
    """8-bit codes and block exponents of a flat float tensor (whole blocks), each value cut to the code below it."""
    top = 127 if signed else 255
    bits = x.abs().view(torch.int32)
    exponent = bits.view(-1, BLOCK).amax(1) >> 23
    base = (exponent + 1) * 8 - top
    code = (bits.view(-1, BLOCK) >> 20) - base[:, None]
    code = torch.where((code > 0) & (code + base[:, None] > 0), code, 0).view(-1)
    if signed:
        code = code | torch.where(x < 0, 128, 0)
    return code.to(torch.uint8), exponent.to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    if case['op'] == 'embed':
        rows, width, tokens = case['rows'], case['width'], case['tokens']
        s = {'case': case, 'scale': math.sqrt(width)}
        s['table'] = (torch.randn(rows, width, generator=gen, device='cuda') * 0.02).to(dtype).requires_grad_(case['train'])
        u = torch.rand(tokens, generator=gen, device='cuda', dtype=torch.float64)
        if case['spread'] == 'zipf':  # row r with a share that falls as 1 / (r + 1)
            idx = torch.exp(u * math.log(rows + 1.0)).floor() - 1.0
        elif case['spread'] == 'runs':  # the same row for many tokens on end
            idx = torch.floor((torch.arange(tokens, device='cuda') // 97 * 0.6180339887498949) % 1.0 * rows)
        else:
            idx = torch.floor(u * rows)
        idx = idx.clamp(0, rows - 1).to(torch.int64)
        if case['spread'] != 'even':
            idx = torch.randperm(rows, generator=gen, device='cuda')[idx]
        if case['absent'] > 0.0:
            idx = torch.where(torch.rand(tokens, generator=gen, device='cuda') < case['absent'], -1, idx)
        s['indices'] = idx.to(torch.int64 if case['wide'] else torch.int32)
        if case['train']:
            s['grad'] = (torch.randn(tokens, width, generator=gen, device='cuda') * 0.01).to(dtype)
        return s
    sizes = _sizes(case)
    starts, at = [], 0
    for n in sizes:  # tensors of one arena, each from a block's border on
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    inside = torch.zeros(at, dtype=torch.bool, device='cuda')
    for a, n in zip(starts, sizes):
        inside[a:a + n] = True
    views = lambda flat: [flat[a:a + n] for a, n in zip(starts, sizes)]  # noqa: E731
    blocks = lambda flat: [flat[a // BLOCK:(a + n + BLOCK - 1) // BLOCK] for a, n in zip(starts, sizes)]  # noqa: E731
    normal = lambda: torch.randn(at, generator=gen, device='cuda') * inside  # noqa: E731
    # gradients over a few orders of magnitude, as those of a scene or of layers of different depth
    size = torch.exp(torch.randn(at // BLOCK, generator=gen, device='cuda') * 2.0 - 7.0).repeat_interleave(BLOCK)
    s = {'case': case, 'step': FIRST_STEP, 'sizes': sizes}
    s['weights'] = normal().to(dtype)
    s['grads'] = (normal() * size).to(dtype)
    m, v = normal() * size * 0.3, (normal() * size).square()
    if case['master'] and dtype != torch.float32:
        s['master'] = s['weights'].float() + normal() * 1e-4
        s['weights'] = s['master'].to(dtype)
    if case['bits'] == 8:
        s['m'], s['m_exp'] = _encode(m, True)
        s['v'], s['v_exp'] = _encode(v, False)
        s['m_out'], s['v_out'] = torch.zeros(at, dtype=torch.bfloat16, device='cuda'), torch.zeros(at, dtype=torch.bfloat16, device='cuda')
    else:
        s['m'], s['v'] = m, v
    s['norm_limit'] = 0.5 if case['clip'] else None
    if own:
        params = [torch.nn.Parameter(w) for w in views(s['weights'])]
        for p, g in zip(params, views(s['grads'])):
            p.grad = g
        opt = _library().FusedAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case['bits'], master_weights='master' in s,
                                    max_grad_norm=s['norm_limit'])
        names = [('exp_avg', views(s['m'])), ('exp_avg_sq', views(s['v']))]
        if case['bits'] == 8:
            names += [('exp_avg_exponent', blocks(s['m_exp'])), ('exp_avg_sq_exponent', blocks(s['v_exp']))]
            s['out_views'] = (views(s['m_out']), views(s['v_out']))
        if 'master' in s:
            names.append(('master', views(s['master'])))
        for i, p in enumerate(params):
            opt.state[p] = {'step': FIRST_STEP, **{k: t[i] for k, t in names}}
        s['opt'] = opt
    else:
        s['position'] = torch.cat([torch.arange((n + BLOCK - 1) // BLOCK * BLOCK, device='cuda') for n in sizes])
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass

def _decode(code, exponent, signed):
    top = 127 if signed else 255
    code = code.to(torch.int32).view(-1, BLOCK)
    q = code & top
    bits = q + ((exponent.to(torch.int32) + 1) * 8 - top)[:, None]
    x = torch.where((q > 0) & (bits > 0), bits << 20, 0).view(torch.float32)
    return (torch.where(code > 127, -x, x) if signed else x).view(-1)


def _code(x, position, step, signed):
    """Codes of the new moments: the bits under the third mantissa bit are rounded with an even sequence over the steps."""
    top, rate = (127, 0xC13FA9A9) if signed else (255, 0x91E10DA5)
    u = (position * 0x9E3779B9 + step * rate) & 0xFFFFFFFF
    bits = x.abs().view(torch.int32)
    exponent = bits.view(-1, BLOCK).amax(1) >> 23
    base = ((exponent + 1) * 8 - top).repeat_interleave(BLOCK)
    floor = base.clamp(min=0)
    k = (bits + (u >> 12).to(torch.int32)) >> 20
    least = (floor + 1) << 20
    if signed:  # under the smallest code: that code with the share of the value in it
        low = x.abs() > (u >> 8).to(torch.float32) * 2.0 ** -24 * least.view(torch.float32)
    else:
        low = bits > 0
    q = torch.where(bits < least, torch.where(low, floor + 1 - base, 0), k - base).clamp(max=top)
    if signed:
        q = q | torch.where(x < 0, 128, 0)
    return q.to(torch.uint8), exponent.to(torch.uint8)


def _plain_step(s):
    case = s['case']
    s['step'] += 1
    t, (b1, b2) = s['step'], BETAS
    rate, root = LR / (1.0 - b1 ** t), math.sqrt(1.0 - b2 ** t)
    out = {}
    grads = s['grads'].float()
    weights = s['master'] if 'master' in s else s['weights'].float()
    if case['clip']:
        out['norm'] = grads.square().sum().sqrt()
        grads = grads * (s['norm_limit'] / (out['norm'] + 1e-6)).clamp(max=1.0)
    if case['bits'] == 32:
        m, v = s['m'].mul_(b1).add_(grads, alpha=1.0 - b1), s['v'].mul_(b2).addcmul_(grads, grads, value=1.0 - b2)
    else:
        m = _decode(s['m'], s['m_exp'], True) * b1 + grads * (1.0 - b1)
        v = _decode(s['v'], s['v_exp'], False) * b2 + grads * (1.0 - b2) * grads
    weights.mul_(1.0 - LR * DECAY).addcdiv_(m, (v.sqrt() / root).add_(EPS), value=-rate)
    if weights is not s['weights']:
        s['weights'].copy_(weights)
    if case['bits'] == 8:
        s['m'], s['m_exp'] = _code(m, s['position'], t, True)
        s['v'], s['v_exp'] = _code(v, s['position'], t, False)
        m = s['m_out'].copy_(_decode(s['m'], s['m_exp'], True))
        v = s['v_out'].copy_(_decode(s['v'], s['v_exp'], False))
    out.update(weights=s['weights'], m=m, v=v)
    if 'master' in s:
        out['master'] = s['master']
    return out


def _most(case):
    """About how many tokens the most frequent row has: very long sums are taken in 64 bits."""
    rows, tokens = case['rows'], case['tokens']
    return tokens * math.log(2.0) / math.log(rows + 1.0) if case['spread'] == 'zipf' else tokens / rows + 97


def _plain_rows(s):
    table, idx, scale = s['table'].detach(), s['indices'], s['scale']
    there = (idx >= 0)[:, None]
    at = idx.clamp(min=0).long()
    out = {'rows': torch.where(there, table[at].float() * scale, 0.0).to(table.dtype)}
    if s['case']['train']:
        grad = torch.where(there, s['grad'].float(), 0.0)
        total = torch.zeros(table.shape, dtype=torch.float64 if _most(s['case']) > 30_000 else torch.float32, device=table.device)
        out['grad'] = (total.index_add_(0, at, grad.to(total.dtype)) * scale).to(table.dtype)
    return out


def run(state):
    if not own:
        return _plain_step(state) if state['case']['op'] == 'adamw' else _plain_rows(state)
    s = state
    if s['case']['op'] == 'adamw':
        opt = s['opt']
        opt.step()
        out = {'weights': s['weights'], 'm': s['m'], 'v': s['v']}
        if s['case']['bits'] == 8:
            opt.read_moments(*s['out_views'])
            out['m'], out['v'] = s['m_out'], s['v_out']
        if s['case']['clip']:
            out['norm'] = opt.grad_norm
        if 'master' in s:
            out['master'] = s['master']
        return out
    lookup = _library().embedding_lookup
    if not s['case']['train']:
        return {'rows': lookup(s['table'], s['indices'], scale=s['scale'])}
    s['table'].grad = None
    rows = lookup(s['table'], s['indices'], scale=s['scale'])
    rows.backward(s['grad'])
    return {'rows': rows, 'grad': s['table'].grad}


# ---------------------------------------------------------------------------------------------------------------
# what a pass has to move and compute

def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'embed':
        moved = case['tokens'] * case['width'] * size
        table = min(case['rows'], case['tokens']) * case['width'] * size
        index = case['tokens'] * (8 if case['wide'] else 4)
        if not case['train']:
            return {'bytes': moved + table + index, 'flops': case['tokens'] * case['width']}
        return {'bytes': 2 * moved + table + case['rows'] * case['width'] * size + index, 'flops': 3 * case['tokens'] * case['width']}
    n = sum(_sizes(case))
    per = 3 * size + (8 if case['master'] and size == 2 else 0)
    if case['master'] and size == 2:
        per -= size  # the half copy is only written
    per += 16 if case['bits'] == 32 else 4 + 4  # moments read and written; those in 8 bits come back as values too
    return {'bytes': n * per, 'flops': n * (14 + (2 if case['clip'] else 0))}


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits

def _value(q, exponent, top):
    """What a code stands for: (8 + j) / 8 * 2^e with q = 8 e' + j counted down from the block's largest exponent."""
    place = q.long() + (exponent.long() + 1).repeat_interleave(BLOCK) * 8 - top
    x = torch.ldexp(1.0 + (place % 8).double() / 8.0, (place // 8 - 127).double())
    return torch.where((q > 0) & (place >= 8), x, torch.where((q > 0) & (place > 0), place.double() * 2.0 ** -129, 0.0))


def _rounded(x, position, step, signed):
    """The value that the 8-bit code of x stands for."""
    top, rate = (127, 0xC13FA9A9) if signed else (255, 0x91E10DA5)
    u = ((position * 0x9E3779B9 + step * rate) % 2 ** 32).double() / 2.0 ** 32
    a = x.abs()
    e = torch.frexp(a)[1].double() - 1.0  # a = f 2^e, 1 <= f < 2
    e = torch.where(a >= 2.0 ** -126, e, -126.0)
    high = torch.where(a > 0, e, -127.0).view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)
    unit = torch.exp2(e - 3.0)
    y = torch.floor(a / unit + torch.floor(u * 2 ** 20) / 2 ** 20) * unit
    least = torch.exp2(high + 1.0 - math.ceil(top / 8)) * (1.0 + ((8 - top % 8) % 8 + 1) / 8.0)
    keep = torch.where(a > torch.floor(u * 2 ** 24) / 2 ** 24 * least, least, 0.0) if signed else torch.where(a > 0, least, 0.0)
    y = torch.where(a < least, keep, y)
    return torch.where(x < 0, -y, y)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case['op'] == 'embed':
        table, idx = s['table'].detach().double(), s['indices'].long()
        use = idx >= 0
        rows = torch.zeros(idx.numel(), case['width'], dtype=torch.float64, device='cuda')
        rows[use] = table.index_select(0, idx[use]) * s['scale']
        out = {'rows': rows}
        if case['train']:
            total = torch.zeros_like(table)
            total.index_put_((idx[use],), s['grad'].double()[use], accumulate=True)
            out['grad'] = total * s['scale']
        return out
    t, (b1, b2) = FIRST_STEP + 1, BETAS
    g = s['grads'].double()
    out = {}
    if case['clip']:
        out['norm'] = g.pow(2).sum().sqrt()
        g = g * min(1.0, s['norm_limit'] / (float(out['norm']) + 1e-6))
    if case['bits'] == 8:
        m = _value(s['m'] & 127, s['m_exp'], 127) * torch.where(s['m'] > 127, -1.0, 1.0)
        v = _value(s['v'], s['v_exp'], 255)
    else:
        m, v = s['m'].double(), s['v'].double()
    w = s['master'].double() if 'master' in s else s['weights'].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    w = w - LR * DECAY * w - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    out['weights'] = w
    if 'master' in s:
        out['master'] = w
    if case['bits'] == 8:
        m, v = _rounded(m, s['position'], t, True), _rounded(v, s['position'], t, False)
    out.update(m=m, v=v)
    return out
