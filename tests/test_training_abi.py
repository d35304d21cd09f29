"""The training step's functions of the C ABI refuse, before any launch, what their kernels do not cover, and say how much workspace they want."""
import ctypes
import os

import pytest
import torch

from simplicial_attention_amd import _native


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_native.LIB_PATH):
        _native.build()
    return _native.load()


def text(lib):
    return lib.sa2_last_error().decode()


def norm(**changes):
    return _native.NormProblem(**{**dict(rows=4, dim=64, x_type=0, residual_type=0, weight_type=0, eps=1e-6), **changes})


BAD_NORMS = [('rows', 0, 2), ('rows', 1 << 40, 2), ('dim', 0, 2), ('dim', 16385, 3), ('x_type', 3, 3), ('residual_type', 1, 3), ('weight_type', -1, 3), ('eps', -1., 2), ('eps', float('nan'), 2),
             ('eps', float('inf'), 2)]


@pytest.mark.parametrize('field,value,code', BAD_NORMS)
def test_norm_refuses_problems(lib, field, value, code):
    p = norm(**{field: value})
    assert lib.sa2_add_rms_norm(p, 0x1000, 64, 0x2000, 64, None, 0x3000, 0x4000, None, None) == code and text(lib) != ''
    assert lib.sa2_add_rms_norm_8bit(p, 0x1000, 64, 0x2000, 64, None, 0, 0x3000, 0x5000, 0x4000, None) == code
    assert lib.sa2_add_rms_norm_bwd_workspace_bytes(p) == -1
    assert lib.sa2_add_rms_norm_bwd(p, 0x1000, 64, None, 0x2000, 0x3000, 64, None, 0, 0x4000, None, None, None, 0, None) == code


def test_norm_refuses_pointers_and_groups(lib):
    p = norm()
    call = lambda x=0x1000, r=0x2000, w=None, y=0x3000, t=0x4000: lib.sa2_add_rms_norm(p, x, 64, r, 64, w, y, t, None, None)
    assert call(x=None) == 1 and call(y=None) == 1 and call(t=None) == 1
    assert call(x=0x1001) == 4 and call(r=0x2001) == 4 and call(w=0x5001) == 4 and call(y=0x3001) == 4 and call(t=0x4001) == 4
    eight = lambda group=0, scales=0x5000: lib.sa2_add_rms_norm_8bit(p, 0x1000, 64, None, 0, None, group, 0x3000, scales, None, None)
    assert eight(scales=None) == 1 and eight(group=16) == 3 and eight(group=-32) == 3 and eight(group=256) == 3
    need = lib.sa2_add_rms_norm_bwd_workspace_bytes(p)
    assert need > 0 and need % (64 * 4) == 0
    back = lambda t=0x1000, rstd=0x2000, up=0x3000, dw=0x6000, ws=0x7000, size=need: lib.sa2_add_rms_norm_bwd(p, t, 64, None, rstd, up, 64, None, 0, 0x4000, None, dw, ws, size, None)
    assert back(t=None) == 1 and back(rstd=None) == 1 and back(up=None) == 1 and back(ws=None) == 2 and back(size=need - 1) == 2 and back(ws=0x7004) == 4 and back(dw=0x6001) == 4
    # (the workspace does not grow with the rows beyond what fills the chip)
    assert lib.sa2_add_rms_norm_bwd_workspace_bytes(norm(rows=1 << 20)) == lib.sa2_add_rms_norm_bwd_workspace_bytes(norm(rows=1 << 22))


def test_norm_refuses_outputs_within_its_inputs(lib):
    # (a row's last piece may be read by two lanes, so nothing may be written over it)
    p = norm()                         # 4 rows of 128 bytes
    call = lambda x=0x1000, xs=64, r=0x2000, rs=64, y=0x3000, t=0x4000: lib.sa2_add_rms_norm(p, x, xs, r, rs, None, y, t, None, None)
    assert call(y=0x1000) == 2 and 'share memory' in text(lib)
    assert call(t=0x2000) == 2 and call(t=0x11fe) == 2 and call(y=0x0e02) == 2 and call(x=0x1000, xs=128, y=0x107e) == 2 and call(rs=0, r=0x3002) == 2
    assert lib.sa2_add_rms_norm_8bit(p, 0x1000, 64, None, 0, None, 0, 0x11ff, 0x5000, None, None) == 2
    back = lambda dx=0x5000, dr=None, dt=0x4000: lib.sa2_add_rms_norm_bwd(p, 0x1000, 64, None, 0x2000, 0x3000, 64, dt, 64, dx, dr, None, None, 0, None)
    assert back(dx=0x1000) == 2 and back(dx=0x3000) == 2 and back(dr=0x4000) == 2 and back(dx=None, dr=0x3180) == 2


def ce(**changes):
    return _native.LinearCeProblem(**{**dict(rows=100, dim=64, vocab=300, dtype=0, reduction=1, ignore_index=-100), **changes})


@pytest.mark.parametrize('field,value,code', [('rows', 0, 2), ('rows', (1 << 24) + 1, 2), ('dim', 60, 2), ('dim', 0, 2), ('dim', 65544, 2), ('vocab', 0, 2), ('vocab', (1 << 24) + 1, 2), ('dtype', 2, 3),
                                              ('reduction', 3, 2), ('reduction', -1, 2),
                                              ('channels', 65, 2), ('channels', -1, 2)])
def test_loss_refuses_problems(lib, field, value, code):
    p = ce(**{field: value})
    assert lib.sa2_linear_ce(p, 0x1000, 64, 0x2000, 64, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 1 << 30, None) == code and text(lib) != ''
    assert lib.sa2_linear_ce_bwd(p, 0x1000, 64, 0x2000, 64, 0x3000, 0x4000, 0x5000, 0x6000, 0x7000, 0x8000, 0x9000, 0xa000, 1 << 30, None) == code
    assert lib.sa2_linear_ce_workspace_bytes(p) == -1 and lib.sa2_linear_ce_bwd_workspace_bytes(p) == -1


def test_loss_refuses_pointers_strides_and_workspaces(lib):
    p = ce()
    need, back = lib.sa2_linear_ce_workspace_bytes(p), lib.sa2_linear_ce_bwd_workspace_bytes(p)
    assert need > 0 and back > 0
    call = lambda h=0x1000, hs=64, w=0x2000, ws=64, t=0x3000, loss=0x4000, lse=0x5000, count=0x6000, mask=0x7000, space=0x8000, size=need: lib.sa2_linear_ce(
        p, h, hs, w, ws, t, loss, lse, count, mask, space, size, None)
    for name in ('h', 'w', 't', 'loss', 'lse', 'count', 'mask'):
        assert call(**{name: None}) == 1, name
    assert call(h=0x1008) == 4 and call(w=0x2004) == 4 and call(hs=65) == 4 and call(ws=68) == 4
    assert call(hs=-64) == 3 and call(ws=(1 << 23) + 8) == 3
    assert call(space=None) == 2 and call(size=need - 1) == 2 and str(need) in text(lib) and call(space=0x8004) == 4
    grad = lambda h=0x1000, t=0x3000, lse=0x4000, up=0x7000, dh=0x8000, dw=0x9000, space=0xa000, size=back: lib.sa2_linear_ce_bwd(
        p, h, 64, 0x2000, 64, t, lse, 0x5000, 0x6000, up, dh, dw, space, size, None)
    assert grad(h=None) == 1 and grad(t=None) == 1 and grad(lse=None) == 1 and grad(up=None) == 1
    assert grad(dh=0x8008) == 4 and grad(dw=0x9004) == 4 and grad(size=back - 1) == 2 and grad(space=0xa001) == 4
    assert grad(dh=None, dw=None) == 0


def test_loss_workspace_is_a_piece_of_the_vocabulary(lib):
    for rows, vocab in ((8192, 131072), (16384, 100000), (1 << 20, 50000), (1, 1 << 24)):
        size = lib.sa2_linear_ce_bwd_workspace_bytes(ce(rows=rows, vocab=vocab, dim=64))
        # dz of 256 MiB, or of 256 tokens, its rows padded by 256 bytes; and the results' shares
        assert 0 < size <= max(256 << 20, rows * 512) + rows * 256 + 64 * 4 * 64 * (rows + 1 + (1 << 25) // max(rows, 1)) + 4096, (rows, vocab, size)
    assert lib.sa2_linear_ce_workspace_bytes(ce(rows=1 << 24, vocab=1 << 24)) == -1                 # (more tiles than a launch)


def step(**changes):
    return _native.AdamwStep(**{**dict(beta1=.9, beta2=.999, eps=1e-8, weight_decay=.01, lr=1e-3, step=1, step_at=None, lr_at=None, grad_scale=None, seed=0), **changes})


def adam(at=0x10000, **changes):
    return _native.AdamwTensor(**{**dict(param=at, grad=at + 0x1000, exp_avg=at + 0x2000, exp_avg_sq=at + 0x3000, exp_avg_scales=None, exp_avg_sq_scales=None, master=None, n=100, type=2, bits=32),
                                  **changes})


def call(lib, items, s=None):
    return lib.sa2_adamw((_native.AdamwTensor * max(len(items), 1))(*items), len(items), s or step(), None)


def test_adamw_refuses(lib):
    assert call(lib, [adam()], step(step=0)) == 2 and call(lib, [adam()], step(beta1=1.)) == 2 and call(lib, [adam()], step(beta2=-.1)) == 2 and call(lib, [adam()], step(eps=float('nan'))) == 2
    assert call(lib, [adam()], step(lr=-1.)) == 2 and call(lib, [adam()], step(weight_decay=float('inf'))) == 2
    assert lib.sa2_adamw(None, 1, step(), None) == 1 and lib.sa2_adamw(None, 0, None, None) == 1 and lib.sa2_adamw(None, -1, step(), None) in (1, 2)
    for name in ('param', 'grad', 'exp_avg', 'exp_avg_sq'):
        assert call(lib, [adam(**{name: None})]) == 1, name
    assert call(lib, [adam(bits=8)]) == 1 and call(lib, [adam(bits=4)]) == 3 and call(lib, [adam(type=3)]) == 3 and call(lib, [adam(n=-1)]) == 2
    assert call(lib, [adam(param=0x10002)]) == 4 and call(lib, [adam(exp_avg=0x12001)]) == 4 and call(lib, [adam(master=0x20002)]) == 4
    # what is written twice: a parameter given again, one that begins inside another, a state that two share, a master that is a state
    for items in ([adam(), adam()], [adam(), adam(0x20000, param=0x10000 + 396)], [adam(), adam(0x20000, exp_avg=0x12000)], [adam(master=0x13000)], [adam(exp_avg_sq=0x10000)]):
        assert call(lib, items) == 2 and 'share memory' in text(lib)
    assert call(lib, []) == 0 and call(lib, [adam(n=0, param=None)]) == 0


def test_functions_refuse_host_tensors():
    from simplicial_attention_amd import adamw_step, add_rms_norm, add_rms_norm_8bit, linear_cross_entropy
    x = torch.zeros(2, 8)
    for f in (lambda: add_rms_norm(x), lambda: add_rms_norm_8bit(x), lambda: adamw_step([x], [x], [x], [x], step=1, lr=.1),
              lambda: linear_cross_entropy(x.bfloat16(), x.bfloat16(), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(AssertionError):
            f()
    adamw_step([], [], [], [], step=1, lr=.1)


def test_optimizer_checks_its_arguments():
    from simplicial_attention_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(lr=float('nan')), dict(betas=(0., 1.)), dict(weight_decay=-1.), dict(state_bits=16), dict(lr=torch.tensor(.1))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    AdamW([p]).step()                       # (no gradients: nothing to do)
    with pytest.raises(RuntimeError):
        AdamW([p], capturable=True).step()


def test_optimizer_refuses_what_a_replay_would_get_wrong(monkeypatch):
    from simplicial_attention_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    monkeypatch.setattr(torch.cuda, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='capturable'):
        AdamW([p]).step()
    with pytest.raises(RuntimeError, match='first step'):
        AdamW([p], capturable=True).step()


def test_optimizer_refuses_states_of_another():
    from simplicial_attention_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    other = torch.optim.AdamW([p])
    other.step()
    with pytest.raises(ValueError, match='another optimizer'):
        AdamW([p]).load_state_dict(other.state_dict())


def test_stacks_without_the_option_still_run():
    """Models pickled before there was one have no such attribute."""
    from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialTransformer
    stack = TwoSimplicialTransformer(16, depth=1, heads=1, key_value_heads=1, dim_head=16, two_simplicial_attn_every=2)
    x = torch.randn(1, 4, 16)
    want = stack(x)
    del stack.__dict__['fused']
    assert not stack.fused and torch.equal(stack(x), want)
