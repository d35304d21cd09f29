"""What the kernels of a fused model do not cover goes through torch: transforms, tangents, subclasses, more rows than a launch takes."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch import nn

pytestmark = pytest.mark.gpu


class Named(torch.Tensor):
    pass


def models(dtype=torch.float32):
    from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialLM
    for fused in (False, True):
        torch.manual_seed(0)
        yield TwoSimplicialLM(num_tokens=50, dim=64, depth=2, heads=2, dim_head=32, two_simplicial_attn_every=4, transformer_kwargs=dict(key_value_heads=2), fused=fused).cuda().to(dtype)


def rows(*shape, dtype=torch.float32, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to('cuda', dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['fp32', 'bf16'])
def test_transforms_of_a_fused_stack(dtype):
    separate, fused = (m.transformer for m in models(dtype))
    x = rows(3, 2, 5, 64, dtype=dtype)
    assert torch.equal(torch.func.vmap(fused)(x), torch.func.vmap(separate)(x))
    gradient = lambda m: torch.func.grad(lambda x: m(x).square().sum())(x[0])
    assert torch.equal(gradient(fused), gradient(separate))
    seen = lambda m: torch.func.functionalize(m)(x[0])
    assert torch.equal(seen(fused), seen(separate))


def test_transforms_of_a_fused_loss():
    separate, fused = models(torch.bfloat16)
    tokens = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(2)).cuda()
    names = dict(separate.named_parameters())
    loss = lambda m: torch.func.grad(lambda params: torch.func.functional_call(m, params, (tokens,), dict(return_loss=True)))({k: v.detach() for k, v in names.items()})
    for a, b in zip(loss(fused).values(), loss(separate).values()):
        assert torch.equal(a, b)


@pytest.mark.parametrize('has_residual', [False, True])
def test_norms_of_tensors_that_carry_more(has_residual):
    from simplicial_attention_amd.rms_norm import norm_behind
    norm, x, r = nn.RMSNorm(64).cuda(), rows(7, 64), rows(7, 64, seed=2) if has_residual else None
    tangent = rows(7, 64, seed=3)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, tangent)
        want = fwAD.unpack_dual(norm(dual if r is None else r + dual)).tangent
        got = fwAD.unpack_dual(norm_behind(norm, dual, r)[0]).tangent
    assert torch.equal(got, want)
    for given in ((x.as_subclass(Named), r), (x, r.as_subclass(Named)) if has_residual else (x.as_subclass(Named), None)):
        normed, total = norm_behind(norm, *given)
        assert type(normed) is Named and type(total) is Named
    norm.weight = nn.Parameter(norm.weight.detach().as_subclass(Named))
    assert type(norm.weight) is Named and type(norm_behind(norm, x, r)[0]) is Named


def test_what_the_kernels_cover():
    from simplicial_attention_amd import _native
    ext = _native.torch_ext()
    x, w = rows(4, 1032, dtype=torch.bfloat16), rows(1032, dtype=torch.bfloat16)
    assert ext.norm_covers(x, None, w) and ext.norm_covers(x, x, w) and ext.norm_covers(x[:0], None, w) and ext.norm_covers(x[0], None, w)
    assert ext.norm_covers(x, x.float(), w) and not ext.norm_covers(x, x[:2], w) and not ext.norm_covers(x, None, w[:4]) and not ext.norm_covers(x, None, w.cpu())
    assert not ext.norm_covers(x.double(), None, w.double()) and not ext.norm_covers(x.to_sparse(), None, w) and not ext.norm_covers(x[0, 0], None, w)
    wide = rows(1, 16385)
    assert not ext.norm_covers(wide, None, wide[0]) and ext.norm_covers(wide[:, 1:], None, wide[0, 1:])
    # (rows of one line of memory)
    assert ext.norm_covers(x[:1].expand(4194303, 1032), None, w) and not ext.norm_covers(x[:1].expand(4194304, 1032), None, w)
    t = torch.zeros(4, dtype=torch.int64, device='cuda')
    assert ext.loss_covers(x, x, t) and ext.loss_covers(x, x, t.int()) and not ext.loss_covers(x, x, t.cpu()) and not ext.loss_covers(x, x, t.float())
    assert ext.loss_covers(x, x[:1].expand(1 << 24, 1032), t) and not ext.loss_covers(x, x[:1].expand((1 << 24) + 1, 1032), t) and not ext.loss_covers(x, x, t[:1].expand((1 << 24) + 1))


def test_second_derivatives_and_batched_gradients_are_refused():
    _, fused = models(torch.bfloat16)
    tokens = torch.arange(12, device='cuda').view(2, 6)
    weight = fused.transformer.norm.weight
    loss = fused(tokens, return_loss=True)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(loss, weight, create_graph=True)
    with pytest.raises(RuntimeError, match='plain tensors'):
        torch.autograd.grad(loss, weight, torch.ones(3, device='cuda'), is_grads_batched=True)
