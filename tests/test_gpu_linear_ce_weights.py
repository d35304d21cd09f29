"""linear_cross_entropy with weights of the rows' losses that are far apart: a row's gradient does not depend on what other rows weigh."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2. ** -24
SCALE = {torch.bfloat16: 1., torch.float16: 1024.}


def inputs(rows, dim, vocab, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed + rows * 31 + dim * 7 + vocab)
    weight = torch.randn(vocab, dim, generator=g, device='cuda') * 2 * dim ** -.5
    targets = torch.randint(0, vocab, (rows,), generator=g, device='cuda')
    hidden = torch.randn(rows, dim, generator=g, device='cuda') + 2 * torch.nn.functional.normalize(weight[targets], dim=1)
    targets = torch.where(torch.rand(rows, generator=g, device='cuda') < .25, -100, targets)
    targets[0], targets[1] = 1, 0
    return hidden.to(dtype), weight.to(dtype), targets


def bounds(hidden, weight, targets, up):
    """Gradients in 64 bits and how far they may be off where dz is rounded by itself for the rows' gradients and, for the weight's, in proportion to the largest weight"""
    dtype, half = hidden.dtype, torch.finfo(hidden.dtype).eps / 2
    h, w = hidden.double(), weight.double()
    counts = (targets != -100)[:, None]
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    p = (z - lse[:, None]).exp()
    index = targets.clamp(min=0)[:, None]
    dz = p.clone().scatter_add_(1, index, -torch.ones_like(index, dtype=p.dtype)) * counts
    each = torch.where(counts, up.double()[:, None], 0.)
    # a logit and lse: sums in 32 bits, two roundings of the exponent; dz: half a place of its own, and the least step of the dtype
    off_z = h.shape[1] * U * (h.abs() @ w.abs().t())
    off_lse = off_z.amax(1) + 4 * U * (z.abs().amax(1) + lse.abs()) + 400 * U
    rounded = (p * (off_z + off_lse[:, None] + 8 * U * (z.abs() + lse.abs()[:, None] + 1)) * 1.1 + dz.abs() * half * 1.05 + 4 * U) * counts
    least = torch.finfo(dtype).smallest_normal * half / SCALE[dtype]
    floor = torch.finfo(dtype).smallest_normal * half
    dh = each * (dz @ w)
    off_dh = each.abs() * ((rounded + least * counts) @ w.abs() + (len(w) + 8) * U * (dz.abs() @ w.abs())) + 1.02 * half * dh.abs() + floor
    dw = (each * dz).t() @ h
    off_dw = (each.abs() * rounded + float(each.abs().max()) * least * counts).t() @ h.abs() + (len(h) + 8) * U * ((each * dz).abs().t() @ h.abs()) + 1.02 * half * dw.abs() + floor
    return (dh, dw), (off_dh * (1 + 1e-6), off_dw * (1 + 1e-6))


# (one launch for both gradients and two; logits in shares; several pieces of the vocabulary)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('rows,dim,vocab', [(60, 64, 32000), (300, 100, 5000), (172, 3816, 745), (2500, 2048, 3000), (6000, 16, 20000), (33, 8, 2)])
def test_rows_beside_one_that_weighs_a_million_times_more(rows, dim, vocab, dtype):
    from simplicial_attention_amd import linear_cross_entropy
    hidden, weight, targets = inputs(rows, dim, vocab, dtype)
    up = torch.rand(rows, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda') * 4e-3 + 2e-3
    up[3] = 0
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = linear_cross_entropy(h, w, targets, reduction='none')
    alone = torch.autograd.grad(loss, (h, w), up, retain_graph=True)
    up[0] = 6e3
    got = torch.autograd.grad(loss, (h, w), up, retain_graph=True)
    want, off = bounds(hidden.detach(), weight.detach(), targets, up)
    for a, b, o in zip(got, want, off):
        assert bool(((a.double() - b).abs() <= o).all()), float(((a.double() - b).abs() / o).max())
    if dtype is torch.float16:
        assert torch.equal(got[0][1:], alone[0][1:])
    # each gradient alone, and the same again
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, weight.detach(), targets, reduction='none'), h, up)[0], got[0])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(hidden.detach(), w, targets, reduction='none'), w, up)[0], got[1])
    for a, b in zip(torch.autograd.grad(loss, (h, w), up), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize('bad', [float('inf'), float('nan')])
def test_weights_that_are_not_numbers_beside_targets_that_are_no_tokens(bad):
    from simplicial_attention_amd import linear_cross_entropy
    for rows, dim, vocab in ((70, 64, 300), (60, 4096, 700)):
        hidden, weight, targets = inputs(rows, dim, vocab, torch.float16)
        h, up = hidden.requires_grad_(), torch.linspace(.5, 1, rows, device='cuda')
        targets[2], targets[4] = vocab, -100
        want, = torch.autograd.grad(linear_cross_entropy(h, weight, targets, reduction='none'), h, up)
        assert bool(want[2].isnan().all()) and not want[4].any()
        up[0] = up[4] = bad
        got, = torch.autograd.grad(linear_cross_entropy(h, weight, targets, reduction='none'), h, up)
        assert not got[0].isfinite().any() and bool(got[2].isnan().all()) and not got[4].any()
        rest = [1, 3, *range(5, rows)]
        assert torch.equal(got[rest], want[rest]) and bool(want[rest].isfinite().all())
