"""Which step an AdamW optimizer takes: counts that move between the parameters and the GPU, and calls that are refused."""
import pytest
import torch

from simplicial_attention_amd import AdamW, adamw

HYPER = dict(betas=(.9, .99), eps=1e-8, weight_decay=.1)


@pytest.fixture
def taken(monkeypatch):
    """The steps of the calls that reach the native function, which is left out."""
    steps = []
    monkeypatch.setattr(adamw, 'adamw_step', lambda params, *args, step, **more: steps.append((len(params), int(step))))
    return steps


def leaves(n=2, device='cpu'):
    g = torch.Generator().manual_seed(7)
    params = [torch.nn.Parameter(torch.randn(40 + i, generator=g).to(device)) for i in range(n)]
    for p in params:
        p.grad = torch.randn(p.shape, generator=g).to(device)
    return params


def test_a_group_that_becomes_capturable_goes_on_counting(taken):
    opt = AdamW(leaves())
    for _ in range(3):
        opt.step()
    again = AdamW(leaves(), capturable=True)
    again.load_state_dict(opt.state_dict())
    assert not again.param_groups[0]['capturable']          # (options are the checkpoint's)
    again.param_groups[0]['capturable'] = True
    again.step()
    again.step()
    again.param_groups[0]['capturable'] = False
    again.step()
    assert taken == [(2, 1), (2, 2), (2, 3), (2, 4), (2, 5), (2, 6)]
    again.param_groups[0]['capturable'] = True
    again.step()
    third = AdamW(leaves(), capturable=True)
    third.load_state_dict(again.state_dict())
    third.step()
    assert taken[6:] == [(2, 7), (2, 8)]


def test_parameters_with_counts_of_their_own_are_not_captured_together(taken):
    params = leaves()
    opt = AdamW(params)
    opt.step()
    grad, params[0].grad = params[0].grad, None
    opt.step()
    params[0].grad = grad
    opt.step()
    assert taken == [(2, 1), (1, 2), (1, 2), (1, 3)]
    opt.param_groups[0]['capturable'] = True
    with pytest.raises(RuntimeError, match='different numbers'):
        opt.step()
    opt.param_groups[0]['capturable'] = False
    late, = leaves(1)
    other = AdamW(leaves(), capturable=True)
    other.step()
    other.param_groups[0]['params'].append(late)
    with pytest.raises(RuntimeError, match='come later'):
        other.step()
    assert len(taken) == 5


def test_a_count_is_not_begun_while_a_step_is_recorded(taken, monkeypatch):
    params = leaves()
    opt = AdamW(params)
    opt.step()
    opt.param_groups[0]['capturable'] = True
    with monkeypatch.context() as patch:
        patch.setattr(torch.cuda, 'is_initialized', lambda: True)
        patch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
        with pytest.raises(RuntimeError, match='first step of a group'):
            opt.step()
    opt.step()
    assert taken == [(2, 1), (2, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize('bits', [32, 8])
def test_a_checkpoint_resumed_as_capturable_takes_the_next_step(bits):
    kw = dict(lr=.01, state_bits=bits, min_8bit_size=1, **HYPER)
    params, twin = leaves(device='cuda'), leaves(device='cuda')
    opt = AdamW(params, **kw)
    for _ in range(3):
        opt.step()
    again = AdamW(twin, **kw)
    with torch.no_grad():
        for a, b in zip(twin, params):
            a.copy_(b)
    again.load_state_dict(opt.state_dict())
    again.param_groups[0]['capturable'] = True
    again.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again.step()
    for replay in range(2):
        graph.replay()
    torch.cuda.synchronize()
    again.param_groups[0]['capturable'] = False
    again.step()
    for _ in range(4):
        opt.step()
    for a, b in zip(params, twin):
        # (corrections of a step on the GPU come of another pow: a rounding of 2^-24 of an update of at most .01 (here below .1 of the values' size) in three of the four steps)
        assert bool(((a - b).abs() <= 8 * 3 * 2. ** -24 * (a.abs() + .1)).all())
        assert opt.state[a]['step'] == again.state[b]['step'] == 7
        if bits == 8:
            assert torch.equal(opt.state[a]['exp_avg'].view(torch.uint8), again.state[b]['exp_avg'].view(torch.uint8))
