"""One round as a program runs it: a prompt forked into a group of samples, each served with an adapter; the samples scored and the adapters
trained on them with the policy loss; the trained adapters served."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _models(n_adapters=3):
    from treeattn_b200.adapters import AdapterSet
    from treeattn_b200.config import Config
    from treeattn_b200.engine import weights_from_ours
    from treeattn_b200.model import GPT
    from treeattn_b200.speculative import PagedDecoder
    torch.manual_seed(0)
    # a window of all positions: the trained model attends to every key, as the served one does
    cfg = Config(attn='seg', vocab_size=96, seq_len=64, n_layer=2, n_head=2, n_embd=64, neighbors=False, chunk=64, local=64)
    model = GPT(cfg).to('cuda', torch.bfloat16).requires_grad_(False)
    adapters = AdapterSet(n_adapters, 2, 64, rank=8, alpha=16)
    with torch.no_grad():
        for b in adapters.b:
            b.copy_(torch.randn_like(b) * 0.05)
    dec = PagedDecoder(weights_from_ours(model.state_dict(), cfg), 2, 2, 64, batch=6, page=16, adapters=adapters)
    return model, adapters, dec


def test_round():
    from treeattn_b200.losses import policy_loss, token_logp
    model, adapters, dec = _models()
    prompt, steps = 21, 30
    tok = torch.randint(0, 96, (6, prompt), device='cuda')
    dec.set_adapter(0, 1)
    dec.set_adapter(3, 0)
    logits = dec.forward(tok)[:, -1]
    held = len(dec.pool.free)
    dec.fork([0, 0, 3, 3], [1, 2, 4, 5])
    assert dec.which.tolist() == [1, 1, 1, 0, 0, 0] and len(dec.pool.free) > held  # the group's prompts are one page each
    tok, logits = tok[[0, 0, 0, 3, 3, 3]], logits[[0, 0, 0, 3, 3, 3]]
    seen, served = [tok], []
    for _ in range(steps):  # a group's samples part ways
        p = logits.float().log_softmax(-1)
        new = torch.multinomial(p.exp(), 1)
        served.append(p.gather(1, new))
        seen.append(new)
        logits = dec.forward(new)[:, 0]
    seen, served = torch.cat(seen, 1), torch.cat(served, 1)
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[4], seen[5])

    # the training side sees the same tokens: the sampled tokens' log-probabilities agree to the 8-bit cache's and bf16's steps
    idx = torch.zeros(6, 64, device='cuda', dtype=torch.int64)
    idx[:, :prompt + steps] = seen
    handle = adapters.attach(model)
    adapters.use(dec.which)
    weight = torch.zeros(6, 63, device='cuda')
    weight[:, prompt - 1:prompt + steps - 1] = 1 / (6 * steps)
    on = weight > 0
    with torch.no_grad():
        old = token_logp(model(idx)[0][:, :-1], idx[:, 1:])
        adapters.use(None)
        ref = token_logp(model(idx)[0][:, :-1], idx[:, 1:])
        adapters.use(dec.which)
    assert (old[on].view(6, steps) - served).abs().mean() < 0.05 and (old - ref)[on].abs().mean() > 0.01

    adv = torch.tensor([1.0, -1.0, 0.5, 0.7, -0.2, -0.9], device='cuda')[:, None].expand(6, 63)

    def own(logits):
        return policy_loss(logits[:, :-1], idx[:, 1:], old, adv, ref_logp=ref, weight=weight, kl=0.1)[0]

    def plain(logits):
        lp = logits[:, :-1].float().log_softmax(-1).gather(-1, idx[:, 1:, None])[..., 0]
        rho, d = (lp - old).exp(), ref - lp
        return (weight * (-torch.minimum(rho * adv, rho.clamp(0.8, 1.2) * adv) + 0.1 * (d.exp() - d - 1))).sum()

    grads = []
    for loss in (own, plain):
        adapters.zero_grad()
        loss(model(idx)[0]).backward()
        grads.append([p.grad.clone() for p in adapters.parameters()])
    for g, w in zip(*grads):
        assert g[:2].abs().sum() > 0 and not g[2].any()
        # the same formula; logits' gradients rounded to bf16 once each way, and summed in no fixed order by the attention's backward pass
        assert (g.float() - w.float()).norm() <= 0.03 * w.float().norm()

    # a step of training, and the decoder serves what was trained
    dec.reset()
    dec.which[:] = torch.tensor([1, 0, 2, -1, 1, 0], device='cuda')
    before = dec.forward(tok)
    with torch.no_grad():
        for p, g in zip(adapters.parameters(), grads[0]):
            p -= 0.5 * g / g.float().abs().max().to(g.dtype) * 0.1
    dec.reset()
    after = dec.forward(tok)
    changed = [not torch.equal(before[b], after[b]) for b in range(6)]
    assert changed == [True, True, False, False, True, True]
    handle.remove()
    from treeattn_b200 import _ops
    assert _ops.device_error()[0] == 0


def test_two_adapters_train_apart():
    """A batch that trains two adapters gives each the gradient of a batch with its own sequences alone."""
    from treeattn_b200.losses import policy_loss
    model, adapters, _ = _models()
    idx = torch.randint(0, 96, (4, 64), device='cuda')
    old, adv = torch.full((4, 63), -4.5, device='cuda'), torch.randn(4, 63, device='cuda')
    weight = torch.full((4, 63), 1 / 252, device='cuda')
    handle = adapters.attach(model)

    def grads(rows, which):
        adapters.zero_grad()
        adapters.use(which)
        policy_loss(model(idx[rows])[0][:, :-1], idx[rows, 1:], old[rows], adv[rows], weight=weight[rows])[0].backward()
        return [p.grad.clone() for p in adapters.parameters()]

    both = grads([0, 1, 2, 3], [0, 2, 2, 0])
    first, second = grads([0, 3], [0, 0]), grads([1, 2], [2, 2])
    handle.remove()
    for b, f, s in zip(both, first, second):
        for a, alone in ((0, f), (2, s)):
            assert (b[a].float() - alone[a].float()).norm() <= 0.03 * alone[a].float().norm()
        assert not b[1].any()
