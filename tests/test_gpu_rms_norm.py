"""add_rms_norm and its 8-bit form against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
U = 2. ** -24                  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):           # half of the smallest step there is
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def inputs(rows, dim, x_type, r_type, w_type, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed + rows * 7 + dim)
    randn = lambda *s: torch.randn(*s, generator=g, device='cuda')
    x = randn(rows, dim).to(x_type)
    r = None if r_type is None else (3 * randn(rows, dim)).to(r_type)
    w = None if w_type is None else (1 + .3 * randn(dim)).to(w_type)
    return x, r, w


def total_of(x, r):
    return x if r is None else (x.float() + r.float()).to(r.dtype)


def formula(t, w, eps):
    t = t.double()
    rstd = (t.square().mean(-1, keepdim=True) + eps).rsqrt()
    return t * rstd * (1. if w is None else w.double()), rstd


# a sum of n fp32 terms in lanes of 64 (or workgroups) is off by at most this many half steps of the sum of magnitudes: terms of a lane one after
# another (8 to 64), a tree of 6 and up to 16 waves behind it; with the few roundings of the quotient around it
C = 100

SHAPES = [(1, 1), (3, 7), (1, 16), (5, 32), (4, 33), (17, 40), (2, 128), (7, 129), (1, 512), (65, 512), (3, 513), (33, 1000), (2, 1024), (5, 1025), (2, 2048), (3, 2056),
          (3, 4096), (2, 5003), (2, 8192), (2, 8200), (1, 16384), (4500, 72), (1100, 512)]
MIXES = [('bf16', 'bf16', 'bf16'), ('bf16', 'fp32', 'fp32'), ('fp16', 'fp16', 'fp16'), ('fp16', 'fp32', 'fp16'), ('fp32', 'fp32', 'fp32'), ('bf16', None, 'bf16'), ('fp32', None, None),
         ('fp16', None, 'fp32')]


@pytest.mark.parametrize('mix', MIXES, ids=lambda m: '-'.join(str(x) for x in m))
@pytest.mark.parametrize('rows,dim', SHAPES)
def test_forward_and_backward(rows, dim, mix):
    from simplicial_attention_amd import add_rms_norm
    x, r, w = inputs(rows, dim, *(TYPES.get(m) for m in mix))
    eps = 1e-5
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    normed, total = add_rms_norm(x, r, w, eps)
    assert torch.equal(total, total_of(x.detach(), None if r is None else r.detach()))
    t = total.detach()
    want, rstd = formula(t, w if w is None else w.detach(), eps)
    assert bool(((normed.double() - want).abs() <= want.abs() * (half_step(x.dtype) * 1.01 + C * U) + floor_of(x.dtype)).all())

    g = torch.Generator(device='cuda').manual_seed(5)
    up = torch.randn(rows, dim, generator=g, device='cuda').to(x.dtype)
    up_total = torch.randn(rows, dim, generator=g, device='cuda').to(t.dtype) if r is not None else None
    grads = torch.autograd.grad([normed] + ([total] if r is not None else []), leaves, [up] + ([up_total] if r is not None else []))
    flat = t.double() * rstd
    inner = up.double() * (1. if w is None else w.detach().double())
    mean = (inner * flat).mean(1, keepdim=True)
    dt = rstd * (inner - flat * mean) + (0. if up_total is None else up_total.double())
    size = rstd * (inner.abs() + flat.abs() * (inner * flat).abs().mean(1, keepdim=True)) + (0. if up_total is None else up_total.double().abs())
    for got in grads[:1 if r is None else 2]:
        assert bool(((got.double() - dt).abs() <= dt.abs() * half_step(got.dtype) * 1.01 + 2 * C * U * size + floor_of(got.dtype)).all())
    if w is not None:
        terms = up.double() * flat
        dw, got = terms.sum(0), grads[-1]
        # (rows one after another in a workgroup, 1024 of which there are at most; then their parts)
        assert bool(((got.double() - dw).abs() <= dw.abs() * half_step(got.dtype) * 1.01 + (2 * C + rows / 1024) * U * terms.abs().sum(0) + floor_of(got.dtype)).all())


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
def test_same_bits_as_the_separate_calls_where_sums_are_exact(dtype):
    """Rows of small powers of two: sums are exact in any order, so nothing but the roundings is left."""
    from simplicial_attention_amd import add_rms_norm
    dtype = TYPES[dtype]
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randint(-2, 3, (64, 256), generator=g, device='cuda').to(dtype)
    r = torch.randint(-2, 3, (64, 256), generator=g, device='cuda').to(dtype)
    normed, total = add_rms_norm(x, r)
    want = (r + x).double()
    assert torch.equal(total, r + x)
    y = want * (want.square().mean(1, keepdim=True) + torch.finfo(torch.float32).eps).rsqrt()
    assert bool(((normed.double() - y).abs() <= y.abs() * (half_step(dtype) * 1.001 + 4 * U)).all())


def test_gradients_match_differences():
    from simplicial_attention_amd import add_rms_norm
    x, r, w = (t.requires_grad_() for t in inputs(3, 24, torch.float32, torch.float32, torch.float32))
    g = torch.Generator(device='cuda').manual_seed(2)
    a, b = (torch.randn(3, 24, generator=g, device='cuda') for _ in range(2))

    def value(x, r, w):
        y, rstd = formula(x.double() + r.double(), w, 1e-3)
        return (y * a).sum() + ((x.double() + r.double()) * b).sum()
    normed, total = add_rms_norm(x, r, w, 1e-3)
    grads = torch.autograd.grad([normed, total], [x, r, w], [a, b])
    # central differences in 64 bits, h^2 and the cancellation below 1e-7
    for which, got in enumerate(grads):
        flat = got.flatten()
        for at in range(0, flat.numel(), 5):
            ends = []
            for h in (1e-5, -1e-5):
                args = [t.detach().double().clone() for t in (x, r, w)]
                args[which].view(-1)[at] += h
                ends.append(float(value(*args)))
            want = (ends[0] - ends[1]) / 2e-5
            assert abs(float(flat[at]) - want) <= 1e-5 * (1 + abs(want)), (which, at)


def test_strides_alignment_and_broadcast_gradients():
    from simplicial_attention_amd import add_rms_norm
    g = torch.Generator(device='cuda').manual_seed(3)
    base = torch.randn(4, 9, 3 + 200, generator=g, device='cuda').bfloat16()
    x = base[:, 1:8, 3:]                                  # rows 2 bytes off any alignment, batches apart
    r = torch.randn(200, 7, 4, generator=g, device='cuda').bfloat16().permute(2, 1, 0)
    w = torch.randn(400, generator=g, device='cuda').bfloat16()[::2]
    for a, b in ((x, r), (x[:, :1], r[:, :1]), (x[:0], r[:0]), (x[0, 0], r[0, 0])):
        normed, total = add_rms_norm(a, b, w)
        assert torch.equal(total, a + b) and normed.shape == a.shape
        want, _ = formula(total, w, torch.finfo(torch.float32).eps)
        assert bool(((normed.double() - want).abs() <= want.abs() * (half_step(torch.bfloat16) * 1.01 + C * U)).all())
    # gradients that are one number spread out
    xl, rl, wl = x.detach().clone().requires_grad_(), r.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    normed, total = add_rms_norm(xl, rl, wl)
    got = torch.autograd.grad(normed.sum() + total.sum(), [xl, rl, wl])
    ones = torch.ones_like(normed)
    normed, total = add_rms_norm(xl, rl, wl)
    want = torch.autograd.grad([normed, total], [xl, rl, wl], [ones, ones])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # rows that are one row spread out
    row = torch.randn(200, device='cuda').bfloat16()
    normed, total = add_rms_norm(row.expand(5, 200), x[0, :5])
    assert torch.equal(total, row + x[0, :5])


def test_parts_of_the_gradient():
    from simplicial_attention_amd import add_rms_norm
    x, r, w = inputs(6, 96, torch.bfloat16, torch.float32, torch.bfloat16)
    full = lambda: [t.clone().requires_grad_() for t in (x, r, w)]
    up, up_total = torch.randn(6, 96, device='cuda').bfloat16(), torch.randn(6, 96, device='cuda')
    leaves = full()
    n, t = add_rms_norm(*leaves)
    want = torch.autograd.grad([n, t], leaves, [up, up_total])
    for which in range(3):                                # one leaf at a time
        leaves = [a.clone().requires_grad_(i == which) for i, a in enumerate((x, r, w))]
        n, t = add_rms_norm(*leaves)
        got, = torch.autograd.grad([n, t], [leaves[which]], [up, up_total])
        assert torch.equal(got, want[which])
    leaves = full()
    n, t = add_rms_norm(*leaves)                          # the sum alone is used
    got = torch.autograd.grad(t, leaves, up_total, allow_unused=True)
    assert torch.equal(got[0], up_total.bfloat16()) and torch.equal(got[1], up_total) and got[2] is None
    leaves = full()
    n, t = add_rms_norm(*leaves)                          # the norm alone
    got = torch.autograd.grad(n, leaves, up)
    leaves = full()
    n, t = add_rms_norm(*leaves)
    want = torch.autograd.grad([n, t], leaves, [up, torch.zeros_like(t)])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    empty = [a.requires_grad_() for a in (x[:0].detach(), r[:0].detach(), w.detach().clone())]
    n, t = add_rms_norm(*empty)
    got = torch.autograd.grad(n.sum(), empty)
    assert got[0].shape == (0, 96) and bool((got[2] == 0).all())


def test_rows_that_are_not_numbers_stay_their_own():
    from simplicial_attention_amd import add_rms_norm, add_rms_norm_8bit
    x, r, w = inputs(9, 300, torch.float32, torch.float32, torch.float32)
    clean = add_rms_norm(x, r, w)[0]
    x[2, 17], x[5, 299], x[7, 0] = float('nan'), float('inf'), -float('inf')
    normed, total = add_rms_norm(x, r, w)
    keep = torch.tensor([i for i in range(9) if i not in (2, 5, 7)], device='cuda')
    assert torch.equal(normed[keep], clean[keep]) and bool(normed[2].isnan().all()) and bool(normed[5, 299].isnan()) and bool((normed[5, :299] == 0).all())
    values, scales, _ = add_rms_norm_8bit(x, r, w, group=128)
    assert bool(scales[2].isnan().all()) and bool(values[2].float().isnan().all()) and bool(scales[keep].isfinite().all())
    assert bool(scales[5, 2].isnan()) and bool((scales[5, :2] == 2. ** -126).all()) and bool((values[5, :256].float() == 0).all())
    # rows of zeros, and without eps
    zeros = torch.zeros(2, 64, device='cuda')
    assert bool((add_rms_norm(zeros)[0] == 0).all()) and bool(add_rms_norm(zeros, eps=0.)[0].isnan().all())


@pytest.mark.parametrize('group', [None, 32, 64, 128])
@pytest.mark.parametrize('rows,dim', [(1, 1), (3, 17), (5, 32), (4, 33), (2, 100), (9, 128), (3, 129), (7, 500), (2, 1000), (32, 1024), (3, 2050), (2, 4096), (1, 16384), (300, 96)])
@pytest.mark.parametrize('mix', [MIXES[0], MIXES[1], MIXES[4], MIXES[5]], ids=lambda m: '-'.join(str(x) for x in m))
def test_8_bits(rows, dim, group, mix):
    from simplicial_attention_amd import add_rms_norm_8bit
    x, r, w = inputs(rows, dim, *(TYPES.get(m) for m in mix), seed=11)
    x[0] *= 1e-3
    if r is not None:
        r[0] *= 1e-3
    values, scales, total = add_rms_norm_8bit(x, r, w, 1e-6, group=group)
    assert values.dtype is torch.float8_e4m3fn and torch.equal(total, total_of(x, r))
    y, _ = formula(total, w, 1e-6)
    g = group or dim
    parts = torch.nn.functional.pad(y, (0, -dim % g)).unflatten(1, (-1, g))
    want = (parts.abs().amax(2) / 448).clamp(min=2. ** -126)
    assert scales.shape == want.shape and bool(((scales.double() - want).abs() <= want * C * U).all())
    # the nearest e4m3: off by half a step, 2^-4 of the value or 2^-10 where steps are 2^-9
    t = torch.nn.functional.pad(values.double(), (0, -dim % g)).unflatten(1, (-1, g))
    exact = parts / scales.double()[:, :, None]
    assert bool(((t - exact).abs() <= torch.maximum(exact.abs() * 2. ** -4, torch.tensor(2. ** -10, device='cuda').double()) * (1 + 1e-4)).all())


def test_streams_graphs_and_devices():
    from simplicial_attention_amd import add_rms_norm, add_rms_norm_8bit
    x, r, w = inputs(300, 512, torch.bfloat16, torch.bfloat16, torch.bfloat16)
    for t in (x, r, w):
        t.requires_grad_()
    up = torch.randn(300, 512, device='cuda').bfloat16()

    def both():
        n, t = add_rms_norm(x, r, w)
        # (without their graph: one that lives on while a backward of its leaves is recorded ends the process, whatever its nodes are)
        return n.detach(), t.detach(), *torch.autograd.grad([n, t], [x, r, w], [up, up])
    want = both()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = both()
        with torch.no_grad():
            eight = add_rms_norm_8bit(x, r, w)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = both()
        with torch.no_grad():
            recorded8 = add_rms_norm_8bit(x, r, w)
    for _ in range(3):
        for t in (*recorded, recorded8[1]):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(recorded, both()):
            assert torch.equal(a, b)
        assert torch.equal(recorded8[0].view(torch.uint8), eight[0].view(torch.uint8)) and torch.equal(recorded8[1], eight[1])


def test_refusals():
    from simplicial_attention_amd import add_rms_norm, add_rms_norm_8bit
    x = torch.randn(4, 64, device='cuda')
    for bad, error in (((x.double(),), TypeError), ((x.cpu(),), AssertionError), ((x, x[:3]), ValueError), ((x, x.bfloat16()), TypeError), ((x, None, x[0, :32]), ValueError),
                       ((x, None, None, -1.), ValueError), ((x[0, 0],), ValueError), ((x, None, x[0].cpu()), AssertionError), ((x[:, :0],), ValueError)):
        with pytest.raises(error):
            add_rms_norm(*bad)
    with pytest.raises(Exception, match='16384'):
        add_rms_norm(torch.zeros(1, 16385, device='cuda'))
    with pytest.raises(ValueError):
        add_rms_norm_8bit(x, group=48)
    with pytest.raises(RuntimeError):
        add_rms_norm_8bit(x.clone().requires_grad_())
    leaf = x.clone().requires_grad_()
    y, _ = add_rms_norm(leaf)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: add_rms_norm(t)[0])(x)
