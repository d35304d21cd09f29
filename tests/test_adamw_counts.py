"""Which step an AdamW optimizer takes: counts that move between the parameters and the GPU, and calls that are refused."""
import pytest
import torch

from simplicial_attention_amd import AdamW, _native

HYPER = dict(betas=(.9, .99), eps=1e-8, weight_decay=.1)


class Native:
    """The calls that reach the native function: parameters and step of each; ``refuse``: for a call with that many parameters."""

    def __init__(self):
        self.steps, self.checked, self.refuse = [], [], None

    def adamw_step(self, params, grads, exp_avgs, exp_avg_sqs, masters, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed, launch):
        (self.steps if launch else self.checked).append((len(params), int(step)))
        if len(params) == self.refuse:
            (self.steps if launch else self.checked).pop()
            raise ValueError('refused')


@pytest.fixture
def native(monkeypatch):
    native = Native()
    monkeypatch.setattr(_native, 'torch_ext', lambda: native)
    return native


@pytest.fixture
def taken(native):
    return native.steps


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


def snapshot(opt):
    counts = [{name: value for name, value in state.items() if name == 'step'} for state in opt.state.values()]
    return counts, [int(group['step_at']) if 'step_at' in group else None for group in opt.param_groups]


@pytest.mark.parametrize('capturable', [False, True])
@pytest.mark.parametrize('groups', [1, 2])
def test_a_refused_step_leaves_the_counts(native, capturable, groups):
    params = leaves(3)
    opt = AdamW([dict(params=params[:2]), dict(params=params[2:])][:groups], capturable=capturable)
    native.refuse = 1 if groups == 2 else 2                          # (the last group)
    with pytest.raises(ValueError, match='refused'):
        opt.step()
    assert native.steps == [] and not opt.state and snapshot(opt)[1] == [None] * groups
    native.refuse = None
    opt.step()
    before, native.refuse = snapshot(opt), 1 if groups == 2 else 2
    with pytest.raises(ValueError, match='refused'):
        opt.step()
    assert snapshot(opt) == before
    native.refuse = None
    opt.step()
    assert native.steps == [(2, 1), (1, 1), (2, 2), (1, 2)][::3 - groups]


def test_groups_are_looked_at_before_the_first_is_changed(native):
    params = leaves(3)
    opt = AdamW([dict(params=params[:2]), dict(params=params[2:], capturable=True)])
    opt.step()
    grad, params[2].grad = params[2].grad, None
    before = snapshot(opt)
    with pytest.raises(RuntimeError, match='gradients of all'):
        opt.step()
    assert snapshot(opt) == before and len(native.steps) == 2
    params[2].grad = grad
    opt.step()
    assert native.steps == [(2, 1), (1, 1), (2, 2), (1, 2)] and [n for n, _ in native.checked] == [2, 1, 2, 1]


@pytest.mark.gpu
def test_a_refused_group_leaves_all_parameters():
    a, b = leaves(2, 'cuda')
    kept = [a.detach().clone(), b.detach().clone()]
    for bits in (32, 8):
        for share in (False, True):
            opt = AdamW([dict(params=[a]), dict(params=[b])], state_bits=bits, min_8bit_size=1)
            opt.step()
            with torch.no_grad():
                a.copy_(kept[0])
                b.copy_(kept[1])
            state = {name: value.clone() for name, value in opt.state[a].items() if isinstance(value, torch.Tensor)}
            if share:                                                # (noticed below the tensors' checks: a state that is the parameter)
                opt.state[b]['exp_avg' if bits == 32 else 'exp_avg_scales'] = b.detach() if bits == 32 else b.detach()[:1]
            else:
                opt.param_groups[1]['eps'] = -1.
            with pytest.raises(RuntimeError, match='share memory' if share else 'eps=-1'):
                opt.step()
            torch.cuda.synchronize()
            assert torch.equal(a, kept[0]) and torch.equal(b, kept[1]) and opt.state[a]['step'] == opt.state[b]['step'] == 1
            for name, value in state.items():
                assert torch.equal(opt.state[a][name].view(torch.uint8), value.view(torch.uint8))


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


def test_the_checks_alone_are_those_of_the_call():
    import ctypes
    lib = _native.load()
    item = _native.AdamwTensor(param=0x10000, grad=0x11000, exp_avg=0x12000, exp_avg_sq=0x13000, n=100, type=2, bits=32)
    step = lambda **k: _native.AdamwStep(**{**dict(beta1=.9, beta2=.999, eps=1e-8, weight_decay=.01, lr=1e-3, step=1), **k})
    two = (_native.AdamwTensor * 2)(item, item)
    assert lib.sa2_adamw_check(ctypes.byref(item), 1, step()) == 0
    for items, n, s, code in ((two, 2, step(), 2), (two, 1, step(lr=-1.), 2), (two, 1, step(step=0), 2), (two, -1, step(), 2), (None, 1, step(), 1), (two, 1, None, 1)):
        assert lib.sa2_adamw_check(items, n, s) == code == lib.sa2_adamw(items, n, s, None)
