"""adamw_step refuses what its kernels would get wrong, each for its reason, before anything is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CASES = {
    'parameter twice': (dict(n=2), 'share memory'),
    'state used twice': (dict(m='v'), 'share memory'),
    'state is the parameter': (dict(m='p'), 'share memory'),
    'master is a state': (dict(masters=['v']), 'share memory'),
    'rate': (dict(lr=-1.), 'lr=-1 '),
    'rate no number': (dict(lr=float('nan')), 'lr=.?nan '),
    'eps': (dict(eps=float('nan')), 'eps=.?nan '),
    'beta1': (dict(betas=(1., .9)), 'betas=1, 0.9 '),
    'beta2': (dict(betas=(.9, -.5)), 'betas=0.9, -0.5 '),
    'decay': (dict(weight_decay=-1.), 'weight_decay=-1$'),
}


@pytest.mark.parametrize('name', CASES)
def test_refused_for_its_reason(name):
    from simplicial_attention_amd import adamw_step
    from simplicial_attention_amd._native import Sa2Error
    change, text = CASES[name]
    tensors = dict(p=torch.ones(600, device='cuda'), g=torch.ones(600, device='cuda'), m=torch.zeros(600, device='cuda'), v=torch.zeros(600, device='cuda'))
    change = dict(change)
    n, m = change.pop('n', 1), tensors[change.pop('m', 'm')]
    if 'masters' in change:
        change['masters'] = [tensors[x] for x in change['masters']]
    with pytest.raises(Sa2Error, match=text):
        adamw_step([tensors['p']] * n, [tensors['g']] * n, [m] * n, [tensors['v']] * n, **{'step': 1, 'lr': .1, **change})
    torch.cuda.synchronize()
    assert all(bool((tensors[x] == value).all()) for x, value in (('p', 1), ('m', 0), ('v', 0)))
    adamw_step([tensors['p']], [tensors['g']], [tensors['m']], [tensors['v']], step=1, lr=.1)          # (the same without the mistake)
    assert bool((tensors['p'] < 1).all())
