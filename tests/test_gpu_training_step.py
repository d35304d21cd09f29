"""Norms, loss and optimizer together: the fused stack and loss of the language model, its training step, and a recorded step."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

KW = dict(num_tokens=300, dim=128, depth=4, max_seq_len=96, dim_head=64, heads=4, two_simplicial_attn_every=2,
          transformer_kwargs=dict(key_value_heads=2, two_simplicial_attn_kwargs=dict(w1=48, w2=8, qk_rmsnorm=True)))


def model(fused, dtype=torch.bfloat16, seed=3):
    from simplicial_attention_amd.two_simplicial_transformer import TwoSimplicialLM
    torch.manual_seed(seed)
    return TwoSimplicialLM(**KW, fused=fused).to(dtype).cuda()


def tokens(seed=5):
    return torch.randint(0, 300, (3, 91), generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda')


def exact_of(lm):
    """The same model in float32 whose simplicial layers attend in float32 too."""
    from functools import partial
    from oracle import reference_attend as R
    from simplicial_attention_amd.two_simplicial_attention import SlidingWindowTwoSimplicialMHA
    ref = model(False, torch.float32)
    ref.load_state_dict({k: v.float() for k, v in lm.state_dict().items()})
    for attn, _ in ref.transformer.layers:
        if isinstance(attn, SlidingWindowTwoSimplicialMHA):
            attn.attend = partial(R.sliding_two_simplicial_attn, w1=48, w2=8)
    return ref


def loss_and_grads(lm, x):
    loss = lm(x, return_loss=True)
    return loss.detach(), torch.autograd.grad(loss, list(lm.parameters()))


def test_fused_model_is_no_further_from_the_exact_one_than_the_separate_calls():
    fused, separate, x = model(True), model(False), tokens()
    assert all(torch.equal(a, b) for a, b in zip(fused.parameters(), separate.parameters()))
    want_loss, want = loss_and_grads(exact_of(separate), x)
    norm = torch.stack([g.double().norm() for g in want]).norm()

    def off(lm):
        loss, grads = loss_and_grads(lm, x)
        return float((loss - want_loss).abs()), float(torch.stack([(a.double() - b.double()).norm() for a, b in zip(grads, want)]).norm() / norm)
    (loss, grads), (loss_separate, grads_separate) = off(fused), off(separate)
    # both round every layer's rows to bfloat16 at the same places; the separate loss rounds the logits too
    assert loss <= 1.5 * loss_separate + 2. ** -9 and grads <= 1.25 * grads_separate, (loss, loss_separate, grads, grads_separate)


def test_fused_stack_runs_as_the_separate_calls_where_it_cannot_be_seen():
    fused, separate, x = model(True), model(False), tokens()
    with torch.no_grad():
        a, b = fused(x), separate(x)
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2. ** -6         # (norms' sums in another order: a last place of bfloat16 here and there)
    seen = []
    handle = fused.transformer.layers[1][0].register_forward_hook(lambda *a: seen.append(1))
    with torch.no_grad():
        assert torch.equal(fused.transformer(fused.token_emb(x)), separate.transformer(separate.token_emb(x))) and seen == [1]
    handle.remove()
    fused.transformer.fused = False
    with torch.no_grad():
        assert torch.equal(fused(x), separate(x))
    cpu_fused, cpu_separate = model(True, torch.float32).transformer.cpu(), model(False, torch.float32).transformer.cpu()
    for t in (cpu_fused, cpu_separate):
        t.layers = t.layers[:1]                                                               # (the simplicial layers run on the GPU only)
    y = torch.randn(2, 7, 128)
    assert torch.equal(cpu_fused(y), cpu_separate(y))


def test_fused_cache_answers_as_the_whole_text():
    lm, x = model(True), tokens()[:, :70]
    with torch.no_grad():
        whole = lm(x)
        cache = lm.transformer.cache(pages=64, page_size=8)
        names = [cache.new() for _ in range(len(x))]
        parts = [lm.logits_cached(x[:, i:i + n], cache, cache.extend(names, n)) for i, n in ((0, 33), (33, 1), (34, 36))]
        off = (torch.cat(parts, 1).double() - whole.double()).norm() / whole.double().norm()
        assert float(off) < 2. ** -6
        out, logprobs = lm.generate(x[:, :20], 5, temperature=0.)
        assert out.shape == (3, 1, 5) and bool((logprobs <= 0).all())


@pytest.mark.parametrize('bits', [32, 8])
def test_training_step(bits):
    from simplicial_attention_amd import AdamW
    lm, x = model(True), tokens()
    params = list(lm.parameters())
    opt = AdamW(params, lr=1e-3, weight_decay=.01, state_bits=bits, min_8bit_size=1000)
    masters = [p.detach().float().clone() for p in params]
    before = [p.detach().clone() for p in params]
    for step in range(2):
        opt.zero_grad(set_to_none=True)
        loss = lm(x, return_loss=True)
        loss.backward()
        del loss
        grads = [p.grad.clone() for p in params]
        opt.step()
        if step == 0:
            for p, g, m in zip(params, grads, masters):
                # the first step: m / sqrt(v) is the sign, but for eps
                want = m.double() * (1 - 1e-5) - 1e-3 * g.double() / (g.double().abs() + 1e-8)
                assert bool(((opt.state[p]['master'].double() - want).abs() <= 1e-7 + 2. ** -20 * want.abs()).all())
                assert torch.equal(p, opt.state[p]['master'].to(p.dtype))
    assert all(bool(p.isfinite().all()) for p in params) and any(not torch.equal(p, b) for p, b in zip(params, before))


def test_recorded_step_of_the_three():
    """A norm, a read-out with its loss, and the optimizer in one graph, replayed while eager work goes on between."""
    from simplicial_attention_amd import AdamW, add_rms_norm, linear_cross_entropy
    g = torch.Generator(device='cuda').manual_seed(1)
    x, r = (torch.randn(200, 72, generator=g, device='cuda').bfloat16() for _ in range(2))
    targets = torch.randint(0, 500, (200,), generator=g, device='cuda')
    start = [torch.ones(72, device='cuda').bfloat16(), (torch.randn(500, 72, generator=g, device='cuda') * .1).bfloat16()]

    class Run:
        def __init__(self):
            self.params = [torch.nn.Parameter(p.clone()) for p in start]
            self.opt = AdamW(self.params, lr=torch.tensor(.01, device='cuda'), capturable=True, state_bits=8, seed=7)

        def step(self):
            normed, _ = add_rms_norm(x, r, self.params[0])
            loss = linear_cross_entropy(normed, self.params[1], targets)
            for p, grad in zip(self.params, torch.autograd.grad(loss, self.params)):
                p.grad = grad
            self.opt.step()
            return loss.detach()
    eager, recorded = Run(), Run()
    eager.step()
    recorded.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = recorded.step()
    for n in range(4):
        graph.replay()
        want = eager.step()
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        for a, b in zip(recorded.params, eager.params):
            assert torch.equal(a, b)
            assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(recorded.opt.state[a].values(), eager.opt.state[b].values()) if isinstance(u, torch.Tensor))
        x.copy_(torch.randn(200, 72, generator=g, device='cuda'))
    assert int(recorded.opt.param_groups[0]['step_at']) == 5


def test_loss_of_a_padded_batch_is_that_of_its_texts():
    from simplicial_attention_amd import linear_cross_entropy
    lm = model(True)
    x = tokens()
    with torch.no_grad():
        hidden = lm.transformer(lm.token_emb(x[:, :-1]) + lm.pos_emb(torch.arange(90, device='cuda')))
        target = x[:, 1:].clone()
        target[1, 40:] = -100
        loss = linear_cross_entropy(hidden, lm.to_logits.weight, target)
        want = F.cross_entropy((hidden.double() @ lm.to_logits.weight.double().t()).flatten(0, 1), target.flatten(), ignore_index=-100)
    assert abs(float(loss) - float(want)) <= 1e-5
