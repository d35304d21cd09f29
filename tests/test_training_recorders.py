"""The training step's functions refuse recorders, which would keep a result's allocation without the kernel that fills it."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from simplicial_attention_amd import adamw_step, add_rms_norm, add_rms_norm_8bit, linear_cross_entropy

W = torch.zeros(5, 8, dtype=torch.bfloat16)
T = torch.zeros(2, dtype=torch.int64)


def stepped(x):
    adamw_step([x], [x.clone()], [x.clone()], [x.clone()], step=1, lr=.1)
    return x


CALLS = {
    'add_rms_norm': lambda x: add_rms_norm(x)[0],
    'add_rms_norm_residual': lambda x: add_rms_norm(x, x.clone())[1],
    'add_rms_norm_8bit': lambda x: add_rms_norm_8bit(x)[1],
    'linear_cross_entropy': lambda x: linear_cross_entropy(x.bfloat16(), W, T),
    'adamw_step': stepped,
}


# (on host tensors, which each call refuses too: the recorder has to be noticed first)
@pytest.mark.parametrize('name', CALLS)
@pytest.mark.parametrize('grad', [False, True])
def test_traced_calls_are_refused(name, grad):
    x = torch.zeros(2, 8)
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match='cannot be traced'):
        torch.jit.trace(CALLS[name], x.requires_grad_(grad and name not in ('add_rms_norm_8bit', 'adamw_step')), check_trace=False)


@pytest.mark.parametrize('name', CALLS)
@pytest.mark.parametrize('mode', ['real', 'fake'])
def test_calls_in_a_graph_of_operators_are_refused(name, mode):
    with torch.no_grad(), pytest.raises(RuntimeError, match='cannot be traced'):
        make_fx(CALLS[name], tracing_mode=mode)(torch.zeros(2, 8))


@pytest.mark.parametrize('name', CALLS)
def test_calls_among_fake_tensors_are_refused(name):
    x = torch.zeros(2, 8)
    with torch.no_grad(), FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(RuntimeError, match='cannot be traced'):
        CALLS[name](x)


@pytest.mark.gpu
def test_backward_is_not_recorded():
    """A graph that was built before the recorder came."""
    x = torch.ones(2, 8, device='cuda', requires_grad=True)
    h = torch.ones(2, 8, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    for out, leaf in ((add_rms_norm(x)[0].sum(), x), (linear_cross_entropy(h, W.cuda(), T.cuda()), h)):
        want, = torch.autograd.grad(out, leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match='cannot be traced'):
            make_fx(lambda up: torch.autograd.grad(out, leaf, up, retain_graph=True)[0])(torch.ones_like(out))
        assert torch.equal(torch.autograd.grad(out, leaf)[0], want)
