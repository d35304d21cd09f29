"""Attention and the norms in front of it refuse recorders that would keep a result's allocation without the kernel that fills it (torch.jit.trace sees their Python Functions)."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from simplicial_attention_amd import SlidingWindowTwoSimplicialMHA, sliding_two_simplicial_attn


def attend(q):
    return sliding_two_simplicial_attn(q, (q, q), (q, q), w1=8, w2=4)


def test_attention_in_a_graph_of_operators_is_refused():
    # (a host tensor, which is refused too: the recorder has to be noticed first)
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(attend)(torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize('grad', [False, True])
def test_module_in_a_graph_of_operators_is_refused(grad):
    module = SlidingWindowTwoSimplicialMHA(64, dim_head=64, heads=2, key_value_heads=1, w1=40, w2=9).cuda().bfloat16()
    x = torch.randn(1, 96, 64, device='cuda').bfloat16()
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(module)(x)


@pytest.mark.gpu
def test_backward_is_not_recorded():
    q = torch.randn(1, 32, 1, 64, device='cuda').bfloat16().requires_grad_()
    out = attend(q)
    up = torch.ones_like(out)
    want, = torch.autograd.grad(out, q, up, retain_graph=True)
    with pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(lambda up: torch.autograd.grad(out, q, up, retain_graph=True)[0])(up)
    assert torch.equal(torch.autograd.grad(out, q, up)[0], want)
