"""linear_cross_entropy and its gradients against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2. ** -24
SCALE = {torch.bfloat16: 1., torch.float16: 1024.}


def inputs(rows, dim, vocab, dtype, seed=0, ignored=.25):
    g = torch.Generator(device='cuda').manual_seed(seed + rows * 31 + dim * 7 + vocab)
    weight = torch.randn(vocab, dim, generator=g, device='cuda') * 2 * dim ** -.5
    targets = torch.randint(0, vocab, (rows,), generator=g, device='cuda')
    hidden = torch.randn(rows, dim, generator=g, device='cuda') + 2 * torch.nn.functional.normalize(weight[targets], dim=1)
    if ignored and rows > 1:
        targets = torch.where(torch.rand(rows, generator=g, device='cuda') < ignored, -100, targets)
    return hidden.to(dtype), weight.to(dtype), targets


def reference(hidden, weight, targets, reduction, up):
    """losses and gradients in 64 bits, and how far a computation in 32 bits with dz rounded to the operands' dtype may be from them"""
    dtype, half = hidden.dtype, torch.finfo(hidden.dtype).eps / 2
    h, w = hidden.double(), weight.double()
    n, dim, vocab = len(h), h.shape[1], len(w)
    counts = targets != -100
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    index = targets.clamp(min=0)[:, None]
    losses = torch.where(counts, lse - z.gather(1, index)[:, 0], 0.)
    # a logit: dim exact products summed in 32 bits; its exponent in base 2: two more roundings of it and of lse; the sum of a tile's terms and of the tiles': fewer than
    # 400 one behind another
    off_z = dim * U * (h.abs() @ w.abs().t())
    off_lse = off_z.amax(1) + 4 * U * (z.abs().amax(1) + lse.abs()) + 400 * U
    off_losses = torch.where(counts, off_lse + off_z.gather(1, index)[:, 0] + 2 * U * (lse.abs() + z.gather(1, index)[:, 0].abs()), 0.)
    number = int(counts.sum())
    if reduction == 'none':
        each, loss, off_loss = up.double(), losses, off_losses
    else:
        by = max(number, 1) if reduction == 'mean' else 1
        each, loss, off_loss = up.double().expand(n) / by, losses.sum() / by, (off_losses.sum() + 200 * U * losses.abs().sum()) / by
    each = torch.where(counts, each, 0.)[:, None]
    p = (z - lse[:, None]).exp()
    dz = p.clone()
    dz.scatter_add_(1, index, -torch.ones_like(each))
    # rounded to the dtype (times a power of two), of p with its own error; the least steps of the dtype
    largest = float(each.abs().max())
    off_dz = each.abs() * (p * (off_z + off_lse[:, None] + 8 * U * (z.abs() + lse.abs()[:, None] + 1)) * 1.1 + dz.abs() * half * 1.05 + 4 * U) + largest * torch.finfo(dtype).smallest_normal * half / SCALE[dtype]
    off_dz = torch.where(counts[:, None], off_dz, 0.)
    dz *= each
    dh, dw = dz @ w, dz.t() @ h
    floor = torch.finfo(dtype).smallest_normal * half
    off_dh = off_dz @ w.abs() + (vocab + 8) * U * (dz.abs() @ w.abs()) + 1.02 * half * dh.abs() + floor
    off_dw = off_dz.t() @ h.abs() + (n + 8) * U * (dz.abs().t() @ h.abs()) + 1.02 * half * dw.abs() + floor
    return (loss, dh, dw), (off_loss, off_dh * (1 + 1e-6), off_dw * (1 + 1e-6))


def check(hidden, weight, targets, reduction, up, got):
    want, off = reference(hidden.detach(), weight.detach(), targets, reduction, up)
    for name, a, b, o in zip(('loss', 'dhidden', 'dweight'), got, want, off):
        assert bool(((a.double() - b).abs() <= o).all()), (name, float(((a.double() - b).abs() / o.clamp(min=1e-30)).max()))


def run(hidden, weight, targets, reduction, up, **more):
    from simplicial_attention_amd import linear_cross_entropy
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = linear_cross_entropy(h, w, targets, reduction=reduction, **more)
    return (loss.detach(), *torch.autograd.grad(loss, (h, w), up))


def up_of(reduction, rows):
    return torch.rand(rows, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda') + .01 if reduction == 'none' else torch.tensor(1.7, device='cuda')


SHAPES = [(1, 8, 1), (1, 64, 256), (2, 8, 2), (3, 100, 7), (31, 16, 33), (32, 32, 32), (33, 33, 129), (60, 128, 256), (129, 72, 300), (257, 328, 1007), (300, 64, 4096),
          (33, 1000, 2049), (1000, 96, 513),
          (4096, 40, 3300),            # large tiles of logits
          (6200, 2048, 40),            # large tiles of the rows' gradients
          (70, 2048, 6300),            # ... of the weight's
          (3000, 8, 100),              # shares over the rows
          (5, 24, 70001)]              # shares over the vocabulary


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('rows,dim,vocab', SHAPES)
def test_loss_and_gradients(rows, dim, vocab, dtype, reduction):
    hidden, weight, targets = inputs(rows, dim, vocab, dtype)
    up = up_of(reduction, rows)
    check(hidden, weight, targets, reduction, up, run(hidden, weight, targets, reduction, up))


# few tiles of logits over many channels, which are computed in shares
FEW = [(1, 4096, 900), (5, 3992, 1148), (33, 4088, 2049), (40, 3993, 777), (172, 3816, 745), (6, 3160, 5506), (129, 4096, 129)]


@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('rows,dim,vocab', FEW)
def test_few_tiles_over_many_channels(rows, dim, vocab, dtype, reduction):
    hidden, weight, targets = inputs(rows, dim, vocab, dtype)
    up = up_of(reduction, rows)
    got = run(hidden, weight, targets, reduction, up)
    check(hidden, weight, targets, reduction, up, got)
    for a, b in zip(got, run(hidden, weight, targets, reduction, up)):
        assert torch.equal(a, b)


def test_few_tiles_with_rows_that_do_not_count():
    hidden, weight, targets = inputs(60, 4096, 700, torch.bfloat16)
    targets[3], targets[4], targets[59] = -100, 699, 0
    up = up_of('none', 60)
    want = run(hidden, weight, targets, 'none', up)
    dirty = hidden.clone()
    dirty[targets == -100] = float('nan')
    dirty[3] = float('inf')
    for a, b in zip(run(dirty, weight, targets, 'none', torch.where(targets == -100, float('nan'), up)), want):
        assert torch.equal(a, b)
    for bad in (700, 703, 1 << 40, -1):
        other = targets.clone()
        other[4] = bad
        loss, dh, dw = run(hidden, weight, other, 'none', up)
        keep = torch.arange(60, device='cuda') != 4
        assert bool(loss[4].isnan()) and bool(dh[4].isnan().all()) and bool(dw.isnan().all())
        assert torch.equal(loss[keep], want[0][keep]) and torch.equal(dh[keep], want[1][keep])
    # logits far beyond what their exponentials hold: the largest alone is left
    big = (hidden.float() * 2 ** 60).to(torch.bfloat16)
    z = big.double() @ weight.double().t()
    top = z.argmax(1)
    loss, dh, dw = run(big, weight, torch.where(targets == -100, -100, top), 'sum', up_of('sum', 0))
    assert float(loss) == 0 and not dh.any() and not dw.any()


def test_pieces_of_the_vocabulary():
    """16384 rows over 17000 tokens: three pieces, the last one ragged"""
    hidden, weight, targets = inputs(16384, 16, 17000, torch.bfloat16)
    up = up_of('mean', 0)
    got = run(hidden, weight, targets, 'mean', up)
    check(hidden, weight, targets, 'mean', up, got)
    for a, b in zip(got, run(hidden, weight, targets, 'mean', up)):
        assert torch.equal(a, b)


def test_masked_rows_may_hold_anything():
    from simplicial_attention_amd import linear_cross_entropy
    hidden, weight, targets = inputs(200, 64, 300, torch.bfloat16)
    targets[40:120] = -100                                  # (whole blocks of 32 rows among them)
    for reduction in ('mean', 'sum', 'none'):
        up = up_of(reduction, 200)
        want = run(hidden, weight, targets, reduction, up)
        dirty = hidden.clone()
        dirty[targets == -100] = float('nan')
        dirty[41], dirty[42] = float('inf'), 3e38
        if reduction == 'none':
            up = torch.where(targets == -100, float('nan'), up)
        got = run(dirty, weight, targets, reduction, up)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert bool((got[1][targets == -100] == 0).all())
    # an index of their own, within the vocabulary too
    want = run(hidden, weight, targets, 'mean', up_of('mean', 0))
    other = torch.where(targets == -100, 7, torch.where(targets == 7, 8, targets))
    same = torch.where(other == 7, -100, other)
    for a, b in zip(run(hidden, weight, other, 'mean', up_of('mean', 0), ignore_index=7), run(hidden, weight, same, 'mean', up_of('mean', 0))):
        assert torch.equal(a, b)
    none = torch.full_like(targets, -100)
    loss, dh, dw = run(hidden, weight, none, 'mean', up_of('mean', 0))
    assert bool(loss.isnan()) and bool((dh == 0).all()) and bool((dw == 0).all())
    loss, dh, dw = run(hidden, weight, none, 'sum', up_of('mean', 0))
    assert float(loss) == 0 and bool((dh == 0).all()) and bool((dw == 0).all())
    assert bool((linear_cross_entropy(hidden, weight, none, reduction='none') == 0).all())


def test_targets_that_are_no_tokens_are_loud():
    hidden, weight, targets = inputs(100, 64, 300, torch.bfloat16, ignored=0)
    for bad in (300, -1, 1 << 40, -(1 << 40), 511):
        t = targets.clone()
        t[17] = bad
        losses, dh, dw = run(hidden, weight, t, 'none', up_of('none', 100))
        assert bool(losses[17].isnan()) and int(losses.isnan().sum()) == 1
        assert bool(dh[17].isnan().all()) and int(dh.isnan().any(1).sum()) == 1 and bool(dw.isnan().any())


def test_weights_of_the_losses_that_are_not_numbers_stay_with_their_rows():
    from simplicial_attention_amd import linear_cross_entropy
    for dtype in (torch.bfloat16, torch.float16):
        hidden, weight, targets = inputs(70, 64, 300, dtype)
        targets[0], targets[1] = 5, -100
        up = torch.linspace(.5, 1, 70, device='cuda')
        # (the largest counts, so that the rows are scaled alike with and without the first ones)
        targets[-1] = 7
        hidden.requires_grad_()
        loss = linear_cross_entropy(hidden, weight, targets, reduction='none')
        want = torch.autograd.grad(loss, hidden, up, retain_graph=True)[0]
        for bad in (float('nan'), float('inf'), -float('inf')):
            for rows in ([0], [0, 1]):
                given = up.clone()
                given[rows] = bad
                got = torch.autograd.grad(loss, hidden, given, retain_graph=True)[0]
                assert not got[0].isfinite().any() and not got[1].any() and torch.equal(got[2:], want[2:])
        # weights of zero and one that is no number
        given = torch.zeros_like(up)
        given[0] = float('nan')
        got = torch.autograd.grad(loss, hidden, given, retain_graph=True)[0]
        assert got[0].isnan().all() and not got[1:].any()


def test_logits_without_bound():
    hidden, weight, targets = inputs(70, 64, 500, torch.bfloat16)
    for scale in (30., 1e4, 1e15):                          # probabilities of 0 and 1
        up = up_of('mean', 0)
        got = run(hidden * scale, weight, targets, 'mean', up)
        assert all(bool(t.isfinite().all()) for t in got)
        check(hidden * scale, weight, targets, 'mean', up, got)
    weight[33] = float('-inf')                              # tokens that cannot be: logits of -inf or inf by the sign of the row
    loss, dh, dw = run(hidden.abs(), weight, torch.where(targets == 33, 5, targets), 'mean', up)
    assert bool(loss.isfinite())
    hidden[3] = float('nan')
    targets[3] = 4
    losses, _, _ = run(hidden, weight.nan_to_num(0., 0., 0.), targets, 'none', up_of('none', 70))
    assert bool(losses[3].isnan()) and int(losses.isnan().sum()) == 1


def test_gradients_match_differences():
    from simplicial_attention_amd import linear_cross_entropy
    hidden, weight, targets = inputs(9, 16, 21, torch.float16)
    up = up_of('none', 9)
    _, dh, dw = run(hidden, weight, targets, 'none', up)

    def value(h, w):
        z = h @ w.t()
        each = torch.logsumexp(z, 1) - z.gather(1, targets.clamp(min=0)[:, None])[:, 0]
        return float((torch.where(targets == -100, 0., each) * up.double()).sum())
    for which, got in enumerate((dh, dw)):
        for at in range(0, got.numel(), 7):
            ends = []
            for d in (1e-5, -1e-5):
                args = [hidden.double(), weight.double()]
                args[which].view(-1)[at] += d
                ends.append(value(*args))
            # half a step of fp16 for dz (whose terms sum up to less than 4 here) and for the result
            assert abs(float(got.flatten()[at]) - (ends[0] - ends[1]) / 2e-5) <= 2. ** -11 * 8 + 1e-6


def test_strides_types_and_shapes():
    from simplicial_attention_amd import linear_cross_entropy
    g = torch.Generator(device='cuda').manual_seed(2)
    base = torch.randn(3, 21, 77, generator=g, device='cuda').bfloat16()
    weight = torch.randn(70, 300, generator=g, device='cuda').bfloat16().t()                      # columns apart
    targets = torch.randint(0, 300, (21, 3), generator=g, device='cuda').t()
    for hidden, w, t in ((base[:, :, 5:75], weight, targets), (base[:, 1:, :70], weight, targets[:, 1:]), (base[:, 3, 2:72], weight, targets[:, 3]), (base[0, 0, :70], weight, targets[0, 0]),
                         (base[:, :, :64], weight[:, 6:], targets.int()), (base[:, :1, :70].expand(3, 21, 70), weight, targets)):
        h, ww = hidden.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(h, ww, t)
        dh, dw = torch.autograd.grad(loss, (h, ww))
        assert dh.shape == h.shape and dw.shape == ww.shape
        flat = hidden.reshape(-1, hidden.shape[-1]).contiguous()
        check(flat, w.contiguous(), t.reshape(-1).long(), 'mean', torch.ones((), device='cuda'), (loss.detach(), dh.reshape(flat.shape), dw))
        losses = linear_cross_entropy(hidden, w, t, reduction='none')
        assert losses.shape == t.shape
        # a gradient that is one number spread out
        each = linear_cross_entropy(h, ww, t, reduction='none')
        a = torch.autograd.grad(each.sum(), (h, ww))
        for x, y in zip(a, torch.autograd.grad(linear_cross_entropy(h, ww, t, reduction='sum'), (h, ww))):
            assert torch.equal(x, y)
    empty = base[:0, :, :70].detach().requires_grad_()
    w = weight.detach().requires_grad_()
    for reduction in ('mean', 'sum', 'none'):
        loss = linear_cross_entropy(empty, w, targets[:0], reduction=reduction)
        dh, dw = torch.autograd.grad(loss.sum(), (empty, w))
        assert dh.shape == empty.shape and bool((dw == 0).all())
        assert loss.numel() == 0 if reduction == 'none' else (bool(loss.isnan()) if reduction == 'mean' else float(loss) == 0)


def test_one_gradient_alone_and_none():
    from simplicial_attention_amd import linear_cross_entropy
    hidden, weight, targets = inputs(300, 136, 700, torch.bfloat16)
    up = torch.ones((), device='cuda')
    loss, dh, dw = run(hidden, weight, targets, 'mean', up)
    h, w = hidden.clone().requires_grad_(), weight.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, weight, targets), h)[0], dh)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(hidden, w, targets), w)[0], dw)
    with torch.no_grad():
        plain = linear_cross_entropy(h, w, targets)
    assert not plain.requires_grad and torch.equal(plain, loss)
    # a weight of zero for the whole loss, and weights some of which are zero or negative
    assert all(bool((t == 0).all()) for t in run(hidden, weight, targets, 'mean', up * 0)[1:])
    mixed = torch.linspace(-1, 1, 300, device='cuda') * (torch.arange(300, device='cuda') % 3 > 0)
    check(hidden, weight, targets, 'none', mixed, run(hidden, weight, targets, 'none', mixed))
    assert all(bool((t == 0).all()) for t in run(hidden, weight, targets, 'none', mixed * 0)[1:])


def test_streams_and_graphs():
    hidden, weight, targets = inputs(500, 64, 1000, torch.bfloat16)
    other = inputs(130, 64, 300, torch.bfloat16)
    up, up2 = torch.ones((), device='cuda'), up_of('none', 130)
    want, want2 = run(hidden, weight, targets, 'mean', up), run(*other, 'none', up2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(hidden, weight, targets, 'mean', up)
        got2 = run(*other, 'none', up2)
    stream.synchronize()
    for a, b in zip((*got, *got2), (*want, *want2)):
        assert torch.equal(a, b)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        rec = run(hidden, weight, targets, 'mean', up)
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        rec2 = run(*other, 'none', up2)
    new = inputs(500, 64, 1000, torch.bfloat16, seed=9)
    for _ in range(2):
        graphs[0].replay()
        graphs[1].replay()
        eager = run(hidden, weight, targets, 'mean', up)
        torch.cuda.synchronize()
        for a, b in zip(rec2, want2):
            assert torch.equal(a, b)
        graphs[0].replay()
        torch.cuda.synchronize()
        for a, b in zip(rec, eager):
            assert torch.equal(a, b)
        for a, b in zip((hidden, weight, targets), new):
            a.copy_(b)


def test_refusals():
    from simplicial_attention_amd import linear_cross_entropy
    h, w, t = inputs(4, 64, 10, torch.bfloat16)
    for bad, error in (((h.float(), w.float(), t), TypeError), ((h, w.half(), t), TypeError), ((h, w, t.float()), TypeError), ((h, w[:, :32], t), ValueError), ((h, w, t[:3]), ValueError),
                       ((h, w[0], t), ValueError), ((h, w[:0], t), ValueError), ((h.cpu(), w, t), AssertionError), ((h, w, t.cpu()), AssertionError)):
        with pytest.raises(error):
            linear_cross_entropy(*bad)
    with pytest.raises(ValueError):
        linear_cross_entropy(h, w, t, reduction='max')
    # (more rows than the count holds, in no memory; nothing is copied in front of the refusal)
    from simplicial_attention_amd._native import Sa2Error
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for rows in (2 ** 24 + 1, 2 ** 32 + 4):
        with pytest.raises(Sa2Error, match='rows='):
            linear_cross_entropy(h[0, :3].expand(rows, 3), w[:, :3], t[0].expand(rows))
    with pytest.raises(Sa2Error, match='too large'):
        linear_cross_entropy(h[0].expand(2 ** 24, 64), w[0].expand(2 ** 24, 64), t[0].expand(2 ** 24))
    assert torch.cuda.max_memory_allocated() - before < 2 ** 24
    leaf = h.clone().requires_grad_()
    loss = linear_cross_entropy(leaf, w, t)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: linear_cross_entropy(x, w, t))(h.expand(2, 4, 64))
