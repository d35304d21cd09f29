"""adamw_step and the AdamW optimizer against the formulas in 64 bits, and 8-bit states bit by bit."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
U = 2. ** -24
HYPER = dict(betas=(.9, .99), eps=1e-8, weight_decay=.1)


def tensors(shapes, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    randn = lambda s: torch.randn(s, generator=g, device='cuda')
    params = [(.1 * randn(s)).to(dtype) for s in shapes]
    grads = [(randn(s) * torch.exp(2 * randn(s)) * 1e-2).to(dtype) for s in shapes]
    m = [1e-2 * randn(s) for s in shapes]
    v = [(1e-2 * randn(s)).square() for s in shapes]
    return params, grads, m, v


def formula(p, g, m, v, step, lr, scale=1.):
    b1, b2 = HYPER['betas']
    g, m, v, p = g.double() * scale, m.double(), v.double(), p.double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    away = m / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + HYPER['eps'])
    return p * (1 - lr * HYPER['weight_decay']) - lr * away, m, v, lr * away


SHAPES = [(1,), (7,), (8,), (255,), (256,), (257,), (2047,), (2048,), (3, 683), (5000,), (70001,), (0,), (64, 64)]


@pytest.mark.parametrize('masters', [False, True])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('step', [1, 2, 1000])
def test_states_in_32_bits(dtype, masters, step):
    from simplicial_attention_amd import adamw_step
    params, grads, m, v = tensors(SHAPES, TYPES[dtype])
    wide = [p.float() + 1e-4 * torch.randn_like(p, dtype=torch.float32) for p in params] if masters else None
    before = [t.clone() for t in (wide or params)]
    want = [formula(*x, step, .01) for x in zip(before, grads, m, v)]
    adamw_step(params, grads, m, v, masters=wide, step=step, lr=.01, **HYPER)
    for i, (x, wm, wv, away) in enumerate(want):
        # three roundings each in 32 bits, of terms of which the two parts of m may cancel
        size = wm.abs() + .1 * grads[i].double().abs() + .9 * m[i].double().abs()
        assert bool(((m[i].double() - wm).abs() <= 4 * U * size).all()) and bool(((v[i].double() - wv).abs() <= 6 * U * wv).all())
        got = wide[i] if masters else params[i]
        half = torch.finfo(got.dtype).eps / 2
        # the quotient: m's error by its parts (size / |m| times), root, corrections, eps, quotient and product a few roundings each
        off = 16 * U * (away.abs() + .01 * size / (wv / (1 - .99 ** step)).sqrt().clamp(min=1e-30) / (1 - .9 ** step)) + 4 * U * before[i].double().abs()
        low = torch.finfo(got.dtype).smallest_normal * half
        assert bool(((got.double() - x).abs() <= off + x.abs() * half * 1.01 + low).all())
        if masters:
            assert torch.equal(params[i], got.to(params[i].dtype))


# ---- 8-bit states: what the header says, in numpy's 32 bits

def mixed(x):
    x = x.astype(np.uint32)
    x = (x ^ (x >> np.uint32(16))) * np.uint32(0x85ebca6b)
    x = (x ^ (x >> np.uint32(13))) * np.uint32(0xc2b2ae35)
    return x ^ (x >> np.uint32(16))


def codes(x, u):
    """x (blocks, 256) fp32 -> codes, scales"""
    scale = np.maximum(np.abs(x).max(1) * np.float32(1 / 448), np.float32(2. ** -126))
    t = np.abs(x) * (np.float32(1) / scale)[:, None]
    normal = ((t.view(np.uint32) + (u << np.uint32(4))) >> np.uint32(20)).astype(np.int64) - 960
    small = np.floor(t * np.float32(512) + u.astype(np.float32) * np.float32(2. ** -16)).astype(np.int64)
    return np.minimum(np.where(t < np.float32(2. ** -6), small, normal), 126), scale


def random_state(n, seed, positive):
    g = torch.Generator(device='cuda').manual_seed(seed)
    values = (torch.randn(n, generator=g, device='cuda') * 60).clamp(-448, 448)
    values = (values.abs() if positive else values).to(torch.float8_e4m3fn)
    return values, torch.rand(-(-n // 256), generator=g, device='cuda') * 1e-4 + 1e-5


def emulate(p, g, m, v, step, lr, index, seed):
    """numpy's fp32, every operation rounded once; p as fp32"""
    f = np.float32
    n = p.size
    wide = lambda s: np.pad(s[0].float().cpu().numpy(), (0, -n % 256)).reshape(-1, 256) * s[1].cpu().numpy()[:, None]
    b1, b2 = HYPER['betas']
    pad = lambda a: np.pad(a, (0, -n % 256)).reshape(-1, 256)
    p, g = pad(p), pad(g)
    am, r = wide(m), wide(v)
    am = am * f(b1) + g * f(1 - b1)
    av = r * r * f(b2) + g * g * f(1 - b2)
    root = np.sqrt(av)
    p = p * f(1 - lr * HYPER['weight_decay']) - am / (root * f(1 / math.sqrt(1 - b2 ** step)) + f(HYPER['eps'])) * f(lr / (1 - b1 ** step))
    with np.errstate(over='ignore'):
        key = mixed(mixed(np.array([(step + 0x9e3779b9 * (index + 1)) & 0xffffffff])) ^ np.uint32(seed))
        random = mixed(np.arange(p.size, dtype=np.uint32) ^ key).reshape(-1, 256)
    mc, ms = codes(am, random & np.uint32(0xffff))
    vc, vs = codes(root, random >> np.uint32(16))
    vc = np.where(root > 0, np.maximum(vc, 1), vc)
    return p.reshape(-1)[:n], (mc | (np.signbit(am) * 128)).astype(np.uint8).reshape(-1)[:n], ms, vc.astype(np.uint8).reshape(-1)[:n], vs


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('step,seed', [(1, 0), (7, 0xfedcba98)])
def test_states_in_8_bits_bit_by_bit(dtype, step, seed):
    from simplicial_attention_amd import adamw_step
    sizes = [1, 5, 8, 255, 256, 257, 511, 2048, 2049, 6000, 70001]
    params, grads, _, _ = tensors([(n,) for n in sizes], TYPES[dtype], seed=step)
    grads[3].zero_()                                       # a block of zeros beside others
    grads[4][100:] = 0
    m, v = [random_state(n, n, False) for n in sizes], [random_state(n, n + 1, True) for n in sizes]
    m[3][0].zero_()
    v[3][0].zero_()
    masters = [p.float().clone() for p in params]
    want = [emulate(x.cpu().numpy(), g.float().cpu().numpy(), a, b, step, .01, i, seed) for i, (x, g, a, b) in enumerate(zip(masters, grads, m, v))]
    adamw_step(params, grads, m, v, masters=masters, step=step, lr=.01, seed=seed, **HYPER)
    for i, (x, mc, ms, vc, vs) in enumerate(want):
        assert np.array_equal(masters[i].cpu().numpy(), x), i
        assert torch.equal(params[i], masters[i].to(params[i].dtype))
        assert np.array_equal(m[i][1].cpu().numpy(), ms) and np.array_equal(v[i][1].cpu().numpy(), vs), i
        assert np.array_equal(m[i][0].view(torch.uint8).cpu().numpy(), mc), i
        assert np.array_equal(v[i][0].view(torch.uint8).cpu().numpy(), vc), i


def test_rounding_keeps_the_expectation():
    from simplicial_attention_amd import adamw_step, state_8bit
    n, tries = 1024, 400
    g = torch.Generator(device='cuda').manual_seed(0)
    grad = torch.randn(n, generator=g, device='cuda') * torch.exp(2 * torch.randn(n, generator=g, device='cuda'))
    total = torch.zeros(n, device='cuda', dtype=torch.float64)
    scale = None
    for seed in range(tries):
        p = torch.zeros(n, device='cuda')
        m, v = state_8bit(p), state_8bit(p)
        adamw_step([p], [grad], [m], [v], step=1, lr=0., seed=seed, **HYPER)
        scale = m[1].repeat_interleave(256).double()
        total += m[0].double() * scale
    exact = grad.double() * .1
    # a rounding is below one step (2^-3 of the value, or 2^-9 of the scale), its deviation at most half of one; six deviations of the mean of 400
    step = torch.maximum(exact.abs() * 2. ** -3, scale * 2. ** -9)
    assert bool(((total / tries - exact).abs() <= 6 * .5 * step / math.sqrt(tries)).all())


def test_values_that_are_not_numbers_stay_in_their_block():
    from simplicial_attention_amd import adamw_step, state_8bit
    p, grad = torch.ones(1000, device='cuda'), torch.ones(1000, device='cuda')
    grad[300], grad[999] = float('nan'), float('inf')
    m, v = state_8bit(p), state_8bit(p)
    adamw_step([p], [grad], [m], [v], step=1, lr=.1, weight_decay=0.)
    wide = lambda s: s[0].float() * s[1].repeat_interleave(256)[:1000]
    bad = torch.zeros(1000, dtype=torch.bool, device='cuda')
    bad[256:512] = True
    bad[768:] = True
    # (an infinity is itself: 448 times an infinite scale)
    assert not bool(wide(m)[bad].isfinite().any()) and bool(wide(m)[bad][:-1].isnan().all()) and bool(wide(m)[~bad].isfinite().all()) and bool((wide(v)[~bad] > 0).all())
    assert bool(p[300].isnan()) and int(p.isnan().sum()) == 2
    q, m, v = torch.ones(10, device='cuda'), torch.zeros(10, device='cuda'), torch.zeros(10, device='cuda')
    adamw_step([q], [grad[295:305]], [m], [v], step=1, lr=.1)
    assert int(q.isnan().sum()) == 1


def test_alignment_layout_and_many_tensors():
    from simplicial_attention_amd import adamw_step
    # (odd offsets of every tensor, more tensors than one launch takes, several dtypes among them)
    base = {t: torch.randn(40000, device='cuda').to(t) for t in TYPES.values()}
    kinds = list(TYPES.values())
    params, grads = [], []
    for i in range(130):
        t = kinds[i % 3]
        at = 1 + 131 * (i // 3)
        params.append(base[t][at:at + 100 + i % 31])
        grads.append(torch.randn(300, device='cuda').to(t)[3:3 + 100 + i % 31])
    m = [torch.randn(200, device='cuda')[1:1 + p.numel()] for p in params]
    v = [torch.rand(200, device='cuda')[3:3 + p.numel()] for p in params]
    kept = {t: b.clone() for t, b in base.items()}
    want = [formula(*x, 3, .01) for x in zip(params, grads, m, v)]
    adamw_step(params, grads, m, v, step=3, lr=.01, **HYPER)
    touched = {t: torch.zeros(40000, dtype=torch.bool, device='cuda') for t in kinds}
    for i, (x, wm, wv, away) in enumerate(want):
        assert bool(((m[i].double() - wm).abs() <= 1e-6).all())
        assert bool(((params[i].double() - x).abs() <= 1e-5 + x.abs() * torch.finfo(params[i].dtype).eps / 2 * 1.01).all())
        at = 1 + 131 * (i // 3)
        touched[kinds[i % 3]][at:at + params[i].numel()] = True
    for t in kinds:
        assert torch.equal(base[t][~touched[t]], kept[t][~touched[t]])      # nothing between the tensors is written
    # a transposed parameter with states like it, and a gradient that is not
    p = torch.randn(30, 20, device='cuda').t()
    g, a, b = torch.randn(20, 30, device='cuda'), torch.zeros_like(p), torch.zeros_like(p)
    want = formula(p.clone(), g, a, b, 1, .01)
    adamw_step([p], [g], [a], [b], step=1, lr=.01, **HYPER)
    assert bool(((p.double() - want[0]).abs() <= 1e-6).all()) and bool(((a.double() - want[1]).abs() <= 1e-6).all())
    one = torch.ones(20, 30, device='cuda')
    want = formula(p.clone(), one, a.clone(), b.clone(), 2, .01)
    adamw_step([p], [torch.ones((), device='cuda').expand(20, 30)], [a], [b], step=2, lr=.01, **HYPER)
    assert bool(((p.double() - want[0]).abs() <= 1e-6).all())


def test_numbers_on_the_device_and_replays():
    from simplicial_attention_amd import adamw_step, state_8bit
    params, grads, m, v = tensors([(300,), (5000,)], torch.float32)
    eight = [state_8bit(p) for p in params], [state_8bit(p) for p in params]
    other = [p.clone() for p in params]
    step, lr, scale = torch.zeros(1, dtype=torch.int64, device='cuda'), torch.tensor(.01, device='cuda'), torch.tensor(.5, device='cuda')
    keep = [[t.clone() for t in x] for x in (params, m, v)]
    keep8 = [[(a.clone(), b.clone()) for a, b in x] for x in eight]
    start = [p.clone() for p in other]

    def both():
        step.add_(1)
        adamw_step(params, grads, m, v, step=step, lr=lr, grad_scale=scale, **HYPER)
        adamw_step(other, grads, *eight, step=step, lr=lr, grad_scale=scale, seed=3, **HYPER)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for n in range(1, 5):
        lr.fill_(.01 * n)
        graph.replay()
        torch.cuda.synchronize()
        # the same steps from numbers; lr has been rounded to 32 bits
        rate = float(lr)
        adamw_step(keep[0], grads, keep[1], keep[2], step=n, lr=rate, grad_scale=scale, **HYPER)
        adamw_step(start, grads, *keep8, step=n, lr=rate, grad_scale=scale, seed=3, **HYPER)
        for a, b in zip((*params, *m, *v, *other), (*keep[0], *keep[1], *keep[2], *start)):
            # (corrections are formed by another pow: a rounding of each step)
            assert bool(((a - b).abs() <= n * 8 * U * (b.abs() + .1)).all())
        for x, y in zip(eight, keep8):
            for (a, s), (b, z) in zip(x, y):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(s, z)


def test_another_stream_gives_the_same():
    from simplicial_attention_amd import adamw_step
    a, b = tensors([(4097,), (12,)], torch.bfloat16), tensors([(4097,), (12,)], torch.bfloat16)
    adamw_step(*a, step=1, lr=.1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        adamw_step(*b, step=1, lr=.1)
    stream.synchronize()
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_refusals():
    from simplicial_attention_amd import AdamW, adamw_step, state_8bit
    p, g, m, v = (x[0] for x in tensors([(600,)], torch.float32))
    call = lambda p=p, g=g, m=m, v=v, n=1, **k: adamw_step([p] * n, [g] * n, [m] * n, [v] * n, **{'step': 1, 'lr': .1, **k})
    kept = p.clone()
    for change, error in ((dict(p=p.double()), TypeError), (dict(g=g.bfloat16()), TypeError), (dict(g=g[:5]), ValueError), (dict(m=m.bfloat16()), TypeError), (dict(m=m[:5]), ValueError),
                          (dict(step=0), ValueError), (dict(p=p.cpu()), AssertionError), (dict(m=state_8bit(p)), TypeError), (dict(m=state_8bit(p[:300]), v=state_8bit(p[:300])), ValueError),
                          (dict(p=p[::2], g=g[::2], m=m[::2], v=v[::2]), ValueError), (dict(masters=[p[:1]]), ValueError), (dict(masters=[]), ValueError), (dict(step=torch.ones(1, device='cuda')), TypeError),
                          (dict(lr=torch.ones(1, device='cuda').double()), TypeError), (dict(grad_scale=torch.ones(2, device='cuda')), TypeError)):
        with pytest.raises(error):
            call(**change)
    # the same parameter twice, a state for two, a parameter inside another one
    for change in (dict(n=2), dict(lr=-1.), dict(eps=float('nan')), dict(betas=(1., .9)), dict(weight_decay=-1.), dict(m=v), dict(m=p)):
        with pytest.raises(Exception, match='.'):
            call(**change)
    with pytest.raises(Exception, match='share memory'):
        adamw_step([p[:400], p[300:]], [g[:400], g[300:]], [m[:400].clone(), m[300:].clone()], [v[:400].clone(), v[300:].clone()], step=1, lr=.1)
    assert torch.equal(p, kept)
    for bad in (dict(lr=-1.), dict(state_bits=4), dict(betas=(.9, 1.)), dict(eps=-1.), dict(lr=torch.tensor(.1))):
        with pytest.raises(ValueError):
            AdamW([p.clone().requires_grad_()], **bad)


def run(optimizer, params, steps, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    for _ in range(steps):
        for p in params:
            p.grad = torch.randn(p.shape, generator=g, device='cuda').to(p.dtype)
        optimizer.step()


@pytest.mark.parametrize('bits', [32, 8])
def test_optimizer_steps_as_the_formula_and_resumes(bits):
    from simplicial_attention_amd import AdamW
    shapes = [(100, 60), (60,), (9000,)]
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator(device='cuda').manual_seed(4), device='cuda').bfloat16()) for s in shapes]
    params = make()
    opt = AdamW(params, lr=.01, state_bits=bits, **HYPER)
    run(opt, params, 4)
    assert (opt.state[params[1]]['exp_avg'].dtype is torch.float32) and (opt.state[params[2]]['exp_avg'].dtype is (torch.float8_e4m3fn if bits == 8 else torch.float32))
    if bits == 32:
        ref = [p.detach().float().double() for p in make()]
        m, v = [torch.zeros_like(p) for p in ref], [torch.zeros_like(p) for p in ref]
        g = torch.Generator(device='cuda').manual_seed(0)
        for n in range(1, 5):
            for i, p in enumerate(ref):
                ref[i], m[i], v[i], _ = formula(p, torch.randn(p.shape, generator=g, device='cuda').bfloat16(), m[i], v[i], n, .01)
        for p, x in zip(params, ref):
            assert bool(((opt.state[p]['master'].double() - x).abs() <= 1e-5).all())
    # the state goes through a checkpoint and the steps go on as if nothing had been
    twin = make()
    again = AdamW(twin, lr=.01, state_bits=bits, **HYPER)
    with torch.no_grad():
        for a, b in zip(twin, params):
            a.copy_(b)
    again.load_state_dict(opt.state_dict())
    run(opt, params, 3, seed=9)
    run(again, twin, 3, seed=9)
    for a, b in zip(params, twin):
        assert torch.equal(a, b)
        for name, value in opt.state[a].items():
            other = again.state[b][name]
            assert torch.equal(value.view(torch.uint8), other.view(torch.uint8)) if isinstance(value, torch.Tensor) else value == other
    # a parameter that had no gradient counts its own steps
    params[0].grad = None
    opt.step()
    assert opt.state[params[0]]['step'] == 7 and opt.state[params[1]]['step'] == 8


def test_optimizer_recorded_and_replayed():
    from simplicial_attention_amd import AdamW
    make = lambda: [torch.nn.Parameter(torch.randn(3000, generator=torch.Generator(device='cuda').manual_seed(i), device='cuda')) for i in range(3)]
    params, twin = make(), make()
    opt = AdamW(params, lr=torch.tensor(.01, device='cuda'), capturable=True, **HYPER)
    ref = AdamW(twin, lr=float(torch.tensor(.01)), **HYPER)
    for a, b in zip(params, twin):
        a.grad, b.grad = torch.randn_like(a), None
        b.grad = a.grad.clone()
    opt.step()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for n in range(3):
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        for a, b in zip(params, twin):
            assert bool(((a - b).abs() <= (n + 2) * 8 * U * (b.abs() + .1)).all())
    params[0].grad = None
    with pytest.raises(RuntimeError):
        opt.step()


def test_a_stale_graph_is_noticed():
    from simplicial_attention_amd import adamw_step
    p = torch.ones(16, device='cuda', requires_grad=True)
    y = (p * p).sum()
    adamw_step([p], [torch.ones(16, device='cuda')], [torch.zeros(16, device='cuda')], [torch.zeros(16, device='cuda')], step=1, lr=.1)
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.backward()
