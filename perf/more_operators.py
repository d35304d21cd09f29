"""Measured cases of the operators of a training step, and of the norm that serving shares with it.

A case is one pass through one operator, as a program that trains (or serves) a language model calls it:

* ``kind='ce'``     ``linear_cross_entropy``: loss of a read-out layer and its gradients for hidden rows and weight, without keeping the logits,
* ``kind='norm'``   ``add_rms_norm``: the residual's addition and the norm behind it; with ``grad`` also the backward pass,
* ``kind='norm8'``  ``add_rms_norm_8bit``: the same with its output in e4m3 and scales (inference),
* ``kind='adamw'``  ``adamw_step``: one step of AdamW over all tensors of a model, states in 32 or 8 bits.

Ranges that the listed cases stand for (``draw`` samples them): losses of 1 .. 16384 rows of 64 .. 4096 channels over 256 .. 131072 tokens, up to a third of the
rows ignored, bfloat16 (mostly) and float16, channel counts off the multiples of 8 too; norms of 1 .. 65536 rows of 16 .. 16384 channels in bfloat16, float16 and
float32, the residual stream in float32 or not there; steps over 1 .. 16 layers' tensors of 64 .. 2048 channels.
"""
import math

import torch

own = False

_DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
_SIZES = {'bf16': 2, 'fp16': 2, 'fp32': 4}
_TINY = torch.finfo(torch.float32).tiny
_BETAS, _EPS, _LR, _DECAY = (0.9, 0.999), 1e-8, 1e-3, 0.01


def _ce(name, rows, dim, vocab, dtype='bf16', ignored=0., reduction='mean'):
    return {'name': name, 'kind': 'ce', 'rows': rows, 'dim': dim, 'vocab': vocab, 'dtype': dtype, 'ignored': ignored, 'reduction': reduction}


def _norm(name, rows, dim, dtype='bf16', residual='same', grad=True):
    return {'name': name, 'kind': 'norm', 'rows': rows, 'dim': dim, 'dtype': dtype, 'residual': residual, 'grad': grad}


def _norm8(name, rows, dim, dtype='bf16', residual='same', group=0):
    return {'name': name, 'kind': 'norm8', 'rows': rows, 'dim': dim, 'dtype': dtype, 'residual': residual, 'group': group}


def _adamw(name, layers, dim, vocab, dtype, bits, masters):
    return {'name': name, 'kind': 'adamw', 'layers': layers, 'dim': dim, 'vocab': vocab, 'dtype': dtype, 'bits': bits, 'masters': masters}


def listed():
    return [
        # fine-tuning on one short text, the byte-level vocabulary (latency and launches)
        _ce('ce_smallest', 60, 128, 256),
        # the training step of the byte-level model: 8 x 2048 tokens
        _ce('ce_bytes_8x2048_d512', 16384, 512, 256),
        # padded batch, a vocabulary and channels off every tile, per-token losses that the program weighs itself
        _ce('ce_ragged_fp16', 1237, 328, 10007, 'fp16', 0.3, 'none'),
        # a large vocabulary under wide rows: products and nothing else
        _ce('ce_8192_d2048_v131072', 8192, 2048, 131072),
        # a decode step of one sequence: no gradients, one row (latency)
        _norm('norm_one_token', 1, 512, grad=False),
        # the training step of the byte-level model
        _norm('norm_8x2048_d512', 16384, 512),
        # mixed precision with the residual stream in 32 bits, a batch and channels off the powers of two
        _norm('norm_stream32_d1000', 5003, 1000, 'bf16', 'fp32'),
        # prefill of wide rows, 8-bit operands in groups of 128 channels for the product behind it
        _norm8('norm8_8192_d4096_g128', 8192, 4096, group=128),
        # a decode step of 32 sequences, one scale a row
        _norm8('norm8_32_d1024', 32, 1024),
        # a small model in 32 bits: many tensors, most of them tiny (latency and launches)
        _adamw('adamw_small_fp32', 2, 64, 256, 'fp32', 32, False),
        # the 12-layer byte-level model in bfloat16 with 32-bit master weights and states
        _adamw('adamw_12x512_masters', 12, 512, 256, 'bf16', 32, True),
        # wide layers and a large embedding, states in 8 bits
        _adamw('adamw8_4x2048', 4, 2048, 32000, 'bf16', 8, True),
    ]


# ---- geometry

def _shapes(c):
    """Parameters of a decoder: embedding, and per layer two norms, three projections and a feed-forward with biases."""
    d = c['dim']
    layer = [(d,), (d, d), (d, d), (d, d), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return [(c['vocab'], d)] + layer * c['layers']


def _starts(sizes):
    """Where each tensor begins in a flat buffer, and where the buffer ends: whole blocks of 256 elements."""
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // 256) * 256)
    return starts[:-1], starts[-1]


def work(case):
    """Inputs read once, outputs written once; the three products of a loss and its two gradients."""
    c = case
    size = _SIZES.get(c['dtype'])
    if c['kind'] == 'ce':
        rows, n, d, v = c['rows'] * (1 - c['ignored']), c['rows'], c['dim'], c['vocab']
        return {'bytes': size * (rows * d + n * d + 2 * v * d) + 8 * n, 'flops': 6 * rows * d * v}
    if c['kind'] == 'adamw':
        n = sum(math.prod(s) for s in _shapes(c))
        return {'bytes': n * (3 * size + (8 if c['masters'] else 0) + (16 if c['bits'] == 32 else 4 + 16 / 256)), 'flops': 0}
    n = c['rows'] * c['dim']
    wide = 4 if c['residual'] == 'fp32' else size
    has = c['residual'] != 'none'
    if c['kind'] == 'norm8':
        scales = c['rows'] * (-(-c['dim'] // c['group']) if c['group'] else 1)
        return {'bytes': n * (size + 2 * wide * has + 1) + 4 * scales, 'flops': 0}
    forward = n * (2 * size + 2 * wide * has) + c['dim'] * size
    # (the backward reads the rows that were normalised, both outputs' gradients, and writes the inputs' gradients: with one type these are one tensor)
    backward = n * (size + (wide if has else size) + wide * has + size + (wide if c['residual'] == 'fp32' else 0)) + 2 * c['dim'] * size
    return {'bytes': forward + (backward if c['grad'] else 0), 'flops': 0}


# ---- inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    dtype = _DTYPES[c['dtype']]
    randn = lambda *shape: torch.randn(*shape, generator=g, device='cuda')
    if c['kind'] == 'ce':
        n, d, v = c['rows'], c['dim'], c['vocab']
        weight = randn(v, d) * (1.5 * d ** -0.5)
        targets = torch.randint(0, v, (n,), generator=g, device='cuda')
        # rows of a final norm, half of which point at their token as those of a trained model do
        hint = weight[targets]
        hidden = randn(n, d) + hint * (6 * torch.rand(n, 1, generator=g, device='cuda') * (torch.rand(n, 1, generator=g, device='cuda') < 0.5) / hint.norm(dim=1, keepdim=True))
        # (the ends of the texts of a padded batch)
        padding = torch.arange(n, device='cuda') % 64 >= 64 * (1 - c['ignored'])
        targets = torch.where(padding, -100, targets)
        return {'case': c, 'hidden': hidden.to(dtype).requires_grad_(), 'weight': weight.to(dtype).requires_grad_(), 'targets': targets,
                'up': torch.rand(n, generator=g, device='cuda') / n if c['reduction'] == 'none' else torch.ones((), device='cuda')}
    if c['kind'] == 'adamw':
        shapes = _shapes(c)
        starts, total = _starts([math.prod(s) for s in shapes])
        state = {'case': c, 'step': 100}
        real = torch.zeros(total, dtype=torch.bool, device='cuda')
        for at, s in zip(starts, shapes):
            real[at:at + math.prod(s)] = True
        flat = lambda scale: torch.where(real, randn(total) * scale, 0.)
        value = flat(0.02)
        # (gradients of very different sizes within a tensor, as they are)
        size = lambda: (2 * randn(total)).exp()
        grad = flat(1e-3) * size()
        average, square = flat(3e-4) * size(), flat(1e-3).mul_(size()).square_()
        buffers = {'params': value.to(dtype), 'grads': grad.to(dtype)}
        if c['masters']:
            buffers['masters'] = value
        if c['bits'] == 32:
            buffers |= {'averages': average, 'squares': square}
        else:
            for name, x in (('averages', average), ('roots', square.sqrt())):
                scale = (x.view(-1, 256).abs().amax(1) * (1 / 448)).clamp(min=_TINY)
                buffers[name], buffers[name + '_scales'] = (x.view(-1, 256) / scale[:, None]).to(torch.float8_e4m3fn).view(-1), scale
        state['flat'] = buffers
        cut = lambda b, per=1: [b[at // per:at // per + -(-math.prod(s) // per)] for at, s in zip(starts, shapes)]
        whole = lambda b: [t.view(s) for t, s in zip(cut(b), shapes)]
        state['params'], state['grads'] = whole(buffers['params']), whole(buffers['grads'])
        state['masters'] = whole(value) if c['masters'] else None
        if c['bits'] == 32:
            state['averages'], state['squares'] = whole(average), whole(square)
        else:
            state['averages'], state['squares'] = (list(zip(whole(buffers[name]), cut(buffers[name + '_scales'], 256))) for name in ('averages', 'roots'))
        return state
    n, d = c['rows'], c['dim']
    wide = torch.float32 if c['residual'] == 'fp32' else dtype
    # (a residual stream has grown over the layers, some channels much more than others)
    stream = randn(n, d) * (1 + 4 * torch.rand(d, generator=g, device='cuda') ** 4)
    state = {'case': c, 'x': randn(n, d).to(dtype), 'residual': None if c['residual'] == 'none' else stream.to(wide), 'weight': (1 + 0.2 * randn(d)).to(dtype)}
    if c['kind'] == 'norm' and c['grad']:
        for name in ('x', 'residual', 'weight'):
            if state[name] is not None:
                state[name].requires_grad_()
        state['up'] = randn(n, d).to(dtype)
        state['up_total'] = None if c['residual'] == 'none' else randn(n, d).to(wide)
    return state


# ---- the operators as elementary operations, in 32 bits

def _plain_ce(s):
    hidden, weight, targets = s['hidden'].detach().float(), s['weight'].detach().float(), s['targets']
    valid = targets != -100
    index = targets.clamp(min=0)[:, None]
    logits = torch.matmul(hidden, weight.t())
    top = logits.amax(1, keepdim=True)
    p = (logits - top).exp()
    total = p.sum(1, keepdim=True)
    losses = torch.where(valid, (total.log() + top - logits.gather(1, index))[:, 0], 0.)
    del logits
    if s['case']['reduction'] == 'none':
        loss, each = losses, s['up']
    else:
        count = valid.sum().float() if s['case']['reduction'] == 'mean' else 1.
        loss, each = losses.sum() / count, s['up'] / count
    each = torch.where(valid, each, 0.)[:, None]
    p *= each / total
    p.scatter_add_(1, index, -each)
    return loss, torch.matmul(p, weight).to(s['hidden'].dtype), torch.matmul(p.t(), hidden).to(s['weight'].dtype)


def _plain_total(s):
    x = s['x'].detach()
    return x if s['residual'] is None else (x.float() + s['residual'].detach().float()).to(s['residual'].dtype)


def _plain_norm(s):
    total, weight, dtype = _plain_total(s), s['weight'].detach().float(), s['x'].dtype
    t = total.float()
    scale = (t.square().mean(1, keepdim=True) + torch.finfo(torch.float32).eps).rsqrt()
    normed = (t * scale * weight).to(dtype)
    kept = [] if s['residual'] is None else [total]
    if not s['case']['grad']:
        return [normed, *kept]
    up = s['up'].float()
    flat = t * scale
    inner = up * weight
    back = scale * (inner - flat * (inner * flat).mean(1, keepdim=True))
    if kept:
        back = back + s['up_total'].float()
    grads = [back.to(dtype)] + ([back.to(s['residual'].dtype)] if kept else [])
    return [normed, *kept, *grads, (up * flat).sum(0).to(s['weight'].dtype)]


def _groups(y, group):
    """(rows, dim) in groups of channels, the last one filled with zeros"""
    group = group or y.shape[1]
    return torch.nn.functional.pad(y, (0, -y.shape[1] % group)).unflatten(1, (-1, group))


def _plain_norm8(s):
    total = _plain_total(s)
    t = total.float()
    y = t * (t.square().mean(1, keepdim=True) + torch.finfo(torch.float32).eps).rsqrt() * s['weight'].float()
    parts = _groups(y, s['case']['group'])
    scales = (parts.abs().amax(2) * (1 / 448)).clamp(min=_TINY)
    values = (parts * (1 / scales)[:, :, None]).flatten(1)[:, :y.shape[1]].to(torch.float8_e4m3fn)
    return [values, scales, *([] if s['residual'] is None else [total])]


def _mixed(x):
    """32 well mixed bits of 32 bits (the finalizer of MurmurHash3, A. Appleby)"""
    x = ((x ^ (x >> 16)) * 0x85ebca6b) & 0xffffffff
    x = ((x ^ (x >> 13)) * 0xc2b2ae35) & 0xffffffff
    return x ^ (x >> 16)


def _to_8bit(x, u):
    """x (blocks, 256) in e4m3 by stochastic rounding with 16 random bits u: what is below the largest value's 448th part is kept in steps of a 512th of that"""
    scale = (x.abs().amax(1) * (1 / 448)).clamp(min=_TINY)
    t = x.abs() * (1 / scale)[:, None]
    normal = ((t.view(torch.int32).long() + (u << 4)) >> 20) - 960
    small = (t * 512 + u.float() * 2. ** -16).floor().nan_to_num(0., 0., 0.).clamp(max=64).long()
    code = torch.where(t < 2. ** -6, small, normal).clamp(0, 126)
    return code, scale


def _plain_adamw(s):
    c, b = s['case'], s['flat']
    s['step'] += 1
    t = s['step']
    b1, b2 = _BETAS
    value = b['masters'] if c['masters'] else b['params'].float()
    grad = b['grads'].float()
    eight = c['bits'] == 8
    if eight:
        wide = lambda name: (b[name].float().view(-1, 256) * b[name + '_scales'][:, None]).view(-1)
        average, square = wide('averages'), wide('roots').square()
    else:
        average, square = b['averages'], b['squares']
    average = average * b1 + grad * (1 - b1)
    square = square * b2 + grad * grad * (1 - b2)
    root = square.sqrt()
    away = average / (root * (1 / math.sqrt(1 - b2 ** t)) + _EPS)
    value = value * (1 - _LR * _DECAY) - away * (_LR / (1 - b1 ** t))
    b['params'].copy_(value)
    if c['masters']:
        b['masters'].copy_(value)
    if not eight:
        b['averages'].copy_(average)
        b['squares'].copy_(square)
    else:
        sizes = [math.prod(x) for x in _shapes(c)]
        starts, total = _starts(sizes)
        step = _mixed(torch.tensor([(t + 0x9e3779b9 * (i + 1)) & 0xffffffff for i in range(len(sizes))], device='cuda'))
        padded = torch.tensor(starts[1:] + [total], device='cuda') - torch.tensor(starts, device='cuda')
        at = torch.arange(total, device='cuda') - torch.tensor(starts, device='cuda').repeat_interleave(padded)
        random = _mixed(at ^ _mixed(step).repeat_interleave(padded)).view(-1, 256)
        signed, unsigned = average.view(-1, 256), root.view(-1, 256)
        code, b['averages_scales'][:] = _to_8bit(signed, random & 0xffff)
        b['averages'].copy_((code | (torch.signbit(signed) * 128)).to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
        code, b['roots_scales'][:] = _to_8bit(unsigned, random >> 16)
        b['roots'].copy_(torch.where(unsigned > 0, code.clamp(min=1), code).to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    return {name: t for name, t in b.items() if name != 'grads'}


def run(state):
    c, s = state['case'], state
    if not own:
        return {'ce': _plain_ce, 'norm': _plain_norm, 'norm8': _plain_norm8, 'adamw': _plain_adamw}[c['kind']](s)
    import simplicial_attention_amd as sa
    if c['kind'] == 'ce':
        loss = sa.linear_cross_entropy(s['hidden'], s['weight'], s['targets'], reduction=c['reduction'])
        return (loss.detach(), *torch.autograd.grad(loss, (s['hidden'], s['weight']), s['up']))
    if c['kind'] == 'norm8':
        values, scales, total = sa.add_rms_norm_8bit(s['x'], s['residual'], s['weight'], group=c['group'] or None)
        return [values, scales, *([] if s['residual'] is None else [total])]
    if c['kind'] == 'norm':
        normed, total = sa.add_rms_norm(s['x'], s['residual'], s['weight'])
        kept = [] if s['residual'] is None else [total]
        if not c['grad']:
            return [normed, *kept]
        leaves = [s['x'], *([s['residual']] if kept else []), s['weight']]
        grads = torch.autograd.grad([normed, *kept], leaves, [s['up'], *([s['up_total']] if kept else [])])
        return [normed.detach(), *(t.detach() for t in kept), *grads]
    s['step'] += 1
    sa.adamw_step(s['params'], s['grads'], s['averages'], s['squares'], masters=s['masters'], step=s['step'], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY)
    return {name: t for name, t in s['flat'].items() if name != 'grads'}


# ---- the same from the definitions, in 64 bits

def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c['kind'] == 'ce':
        return _exact_ce(s)
    if c['kind'] == 'adamw':
        b = s['flat']
        n = s['step'] + 1
        g = b['grads'].double()
        if c['bits'] == 8:
            m = b['averages'].double().unflatten(0, (-1, 256)).mul(b['averages_scales'].double()[:, None]).flatten()
            v = b['roots'].double().unflatten(0, (-1, 256)).mul(b['roots_scales'].double()[:, None]).flatten() ** 2
        else:
            m, v = b['averages'].double(), b['squares'].double()
        m = torch.lerp(g, m, _BETAS[0])
        v = torch.lerp(g ** 2, v, _BETAS[1])
        x = (b['masters'] if c['masters'] else b['params']).double()
        x = x - _LR * (_DECAY * x + m / (1 - _BETAS[0] ** n) / (torch.sqrt(v / (1 - _BETAS[1] ** n)) + _EPS))
        out = {name: None for name in b if name != 'grads'}
        out['params'] = x
        if c['masters']:
            out['masters'] = x
        if c['bits'] == 32:
            out['averages'], out['squares'] = m, v
        return out
    x, r, w = s['x'].detach(), s['residual'], s['weight'].detach().double()
    # (what is normalised is the rounded sum)
    total = x if r is None else (x.double() + r.detach().double()).to(r.dtype)
    t = total.double()
    length = torch.sqrt((t ** 2).sum(1) / c['dim'] + torch.finfo(torch.float32).eps)[:, None]
    y = t / length * w
    kept = [] if r is None else [t]
    if c['kind'] == 'norm8':
        parts = _groups(y, c['group'])
        scales = torch.clamp(parts.abs().max(2).values / 448, min=_TINY)
        return [(parts / scales[:, :, None]).flatten(1)[:, :c['dim']].to(torch.float8_e4m3fn).double(), scales, *kept]
    if not c['grad']:
        return [y, *kept]
    up = s['up'].double()
    dt = up * w / length - t * ((up * w * t).sum(1) / c['dim'])[:, None] / length ** 3
    if r is not None:
        dt = dt + s['up_total'].double()
    return [y, *kept, dt, *([] if r is None else [dt]), (up * t / length).sum(0)]


def _exact_ce(s):
    targets = s['targets']
    keep = (targets >= 0).nonzero()[:, 0]
    h, w = s['hidden'].detach().double(), s['weight'].detach().double()
    n, kind = len(targets), s['case']['reduction']
    losses = torch.zeros(n, dtype=torch.float64, device='cuda')
    weigh = torch.zeros(n, dtype=torch.float64, device='cuda')
    weigh[keep] = s['up'].double()[keep] if kind == 'none' else s['up'].double() / (len(keep) if kind == 'mean' else 1)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for rows in keep.split(2048):
        z = h[rows] @ w.T
        losses[rows] = torch.logsumexp(z, 1) - z[torch.arange(len(rows), device='cuda'), targets[rows]]
        dz = torch.softmax(z, 1)
        dz[torch.arange(len(rows), device='cuda'), targets[rows]] -= 1
        dz *= weigh[rows][:, None]
        dh[rows] = dz @ w
        dw += dz.T @ h[rows]
    loss = losses if kind == 'none' else losses.sum() / (len(keep) if kind == 'mean' else 1)
    return loss, dh, dw


# ---- more cases of the same ranges

# a drawn case costs at most what the largest listed one of its kind does
_MOST_FLOPS = work(listed()[3])['flops']
_MOST_BYTES = {'norm': work(listed()[5])['bytes'] * 4, 'norm8': work(listed()[7])['bytes'], 'adamw': work(listed()[11])['bytes']}


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fits(c):
    w = work(c)
    if c['kind'] == 'ce':
        return w['flops'] <= _MOST_FLOPS and c['rows'] * c['vocab'] <= 8192 * 131072 and c['vocab'] * c['dim'] <= 1 << 28
    return w['bytes'] <= _MOST_BYTES[c['kind']]


def draw(rng):
    while True:
        kind = rng.choice(['ce', 'ce', 'ce', 'norm', 'norm', 'norm8', 'adamw', 'adamw'])
        dtype = rng.choice(['bf16', 'bf16', 'fp16'])
        if kind == 'ce':
            dim = _log_uniform(rng, 64, 4096)
            dim = rng.choice([dim, -(-dim // 8) * 8, -(-dim // 64) * 64])
            case = _ce('', _log_uniform(rng, 1, 16384), dim, _log_uniform(rng, 256, 131072), dtype, rng.choice([0., 0., rng.random() / 3]), rng.choice(['mean', 'mean', 'sum', 'none']))
        elif kind == 'adamw':
            bits = rng.choice([32, 8])
            case = _adamw('', rng.randint(1, 16), _log_uniform(rng, 64, 2048), _log_uniform(rng, 256, 32000), rng.choice(['bf16', 'fp16', 'fp32']), bits, False)
            case['masters'] = case['dtype'] != 'fp32' and rng.random() < 0.7
        else:
            dim = _log_uniform(rng, 16, 16384)
            dim = rng.choice([dim, -(-dim // 8) * 8, -(-dim // 64) * 64])
            dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
            residual = rng.choice(['same', 'same', 'none'] + ['fp32'] * (dtype != 'fp32'))
            rows = _log_uniform(rng, 1, 65536)
            if kind == 'norm':
                case = _norm('', rows, dim, dtype, residual, rng.random() < 0.7)
            else:
                case = _norm8('', rows, dim, dtype, residual, rng.choice([0, 32, 64, 128]))
        del case['name']
        if _fits(case):
            return case
