"""adamw_step and tensors that were made in inference mode, whose versions nobody counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('which', ['param', 'exp_avg', 'master', 'scales'])
def test_inference_tensors_are_refused_before_anything_is_written(which):
    from simplicial_attention_amd import adamw_step, state_8bit
    p, g = torch.ones(300, device='cuda'), torch.ones(300, device='cuda')
    m, v = [state_8bit(p) if which == 'scales' else torch.zeros_like(p) for _ in range(2)]
    master = p.clone()
    with torch.inference_mode():
        if which == 'param':
            p = p.clone()
        elif which == 'exp_avg':
            m = m.clone()
        elif which == 'master':
            master = master.clone()
        else:
            v = (v[0], v[1].clone())
    call = lambda: adamw_step([p], [g], [m], [v], masters=[master], step=1, lr=.1)
    with pytest.raises(RuntimeError, match='inference'):
        call()
    torch.cuda.synchronize()
    moments = [t for s in (m, v) for t in (s if isinstance(s, tuple) else (s,))]
    assert bool((p == 1).all()) and bool((master == 1).all()) and not any(bool(t.float().any()) for t in moments)
    with torch.inference_mode():
        call()
    assert bool((p < 1).all()) and bool((master == p).all())
