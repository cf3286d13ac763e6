"""The losses over a vocabulary's logits against the formulas in 64 bits (torch's autograd in float64) and against differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def _inputs(B, T, V, dtype, seed=0, spread=2.5):
    g = torch.Generator(device='cuda').manual_seed(seed)
    logits = (torch.randn(B, T, V, device='cuda', generator=g) * spread).to(DT[dtype])
    tokens = torch.randint(0, V, (B, T), device='cuda', generator=g)
    lp = logits.double().log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    old = lp + torch.randn(B, T, device='cuda', generator=g) * 0.2
    ref = lp + torch.randn(B, T, device='cuda', generator=g) * 0.4
    adv = torch.randn(B, T, device='cuda', generator=g)
    weight = torch.rand(B, T, device='cuda', generator=g) / (B * T) * (torch.rand(B, T, device='cuda', generator=g) > 0.2)
    return logits, tokens, old, adv, ref, weight


def _reference(logits, tokens, old, adv, ref, weight, lo, hi, kl, tau):
    """Loss, logp and gradient in float64; rows of weight 0 are taken out before anything else."""
    z = logits.double().masked_fill((weight == 0)[..., None], 0).requires_grad_()
    on = weight != 0
    lp = (z / tau).log_softmax(-1).gather(-1, tokens.masked_fill(~on, 0)[..., None])[..., 0]
    rho = (lp - old.double()).exp()
    term = -torch.minimum(rho * adv.double(), rho.clamp(1 - lo, 1 + hi) * adv.double())
    if kl:
        d = ref.double() - lp
        term = term + kl * (d.exp() - d - 1)
    loss = (weight.double() * term)[on].sum()
    grad, = torch.autograd.grad(loss, z)
    return loss.detach(), lp.detach().masked_fill(~on, 0), grad


def _logp_error(logits, tau):
    """A bound on logp's error, in steps of 2^-24: the exponents are a difference and a product, each rounded (two times |z - max| / tau
    steps at most, taken at the row's spread), exp2 is within 4, a thread adds up to V / 512 + 8 numbers of a share and 15 more across the
    CTA and the cluster, and the final difference, product and logarithm add three of its own size."""
    x = logits.double() / tau
    x = x.masked_fill(~x.isfinite(), 0)
    spread = (x.amax(-1) - x.amin(-1)).amax().item()
    return (2 * spread + 4 + logits.shape[-1] / 512 + 23 + 3 * (spread + math.log(logits.shape[-1]) + 1)) * 2.0 ** -24


def _check(logits, tokens, old, adv, ref, weight, clip, kl, tau, up=None):
    from treeattn_b200.losses import policy_loss
    lo, hi = clip
    x = logits.detach().requires_grad_()
    loss, logp = policy_loss(x, tokens, old, adv, ref_logp=ref if kl else None, weight=weight, clip=clip, kl=kl, temperature=tau)
    grad, = torch.autograd.grad(loss, x, None if up is None else torch.tensor(up, device='cuda'))
    rl, rp, rg = _reference(logits, tokens, old, adv, ref, weight, lo, hi, kl, tau)
    e = _logp_error(logits, tau)
    assert (logp.double() - rp).abs().max() <= e
    # what a row's logp is off by moves its term and its slope by at most these
    on = weight != 0
    rho = (rp - old.double()).exp()
    size = weight.double().abs() * (adv.double().abs() * rho + (kl * (1 + (ref.double() - rp).exp()) if kl else 0))
    size = size.masked_fill(~on, 0)
    assert (loss.double() - rl).abs() <= 2 * (e + 8 * 2.0 ** -24) * size.sum()
    # rows whose ratio is within e of a border may fall on either side
    edge = ((rho - (1 - lo)).abs() < 4 * e) | ((rho - (1 + hi)).abs() < 4 * e)
    assert edge.float().mean() < 0.02
    scale = 1.0 if up is None else up
    p = (logits.double() / tau).softmax(-1).masked_fill(~on[..., None], 0)
    hot = torch.nn.functional.one_hot(tokens.masked_fill(~on, 0), logits.shape[-1]).double()
    rg = rg * scale
    # half a step of the output's type, the row's factor's error and that of p (twice e: through the sum and through its own exponent)
    least = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[logits.dtype]
    tol = (rg.abs() * torch.finfo(logits.dtype).eps / 2 * 1.01 + scale / tau * size[..., None] * 4 * (e + 8 * 2.0 ** -24) * (p + hot) +
           scale * 2.0 ** -126 + least)
    assert grad.dtype is logits.dtype and grad.shape == logits.shape
    bad = ((grad.double() - rg).abs() > tol) & ~edge[..., None]
    assert not bad.any(), (bad.nonzero()[:4].tolist(), grad[bad][:4], rg[bad][:4], tol[bad][:4])
    return loss, logp, grad


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,T,V', [(1, 1, 1), (2, 3, 2), (1, 5, 7), (3, 2, 8), (2, 2, 9), (1, 37, 1000), (5, 7, 4099), (2, 9, 16384),
                                   (3, 3, 50257), (1, 2, 131072), (2, 200, 2051), (1, 3, 262143)])
def test_policy_loss(B, T, V, dtype):
    args = _inputs(B, T, V, dtype, seed=V)
    _check(*args, clip=(0.2, 0.28), kl=0.05, tau=1.0)


@pytest.mark.parametrize('kl,tau,up', [(0.0, 1.0, None), (0.1, 0.7, None), (0.02, 1.4, 3.0), (0.05, 1.0, 1024.0), (0.05, 1.0, 0.1)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_terms_temperatures_and_factors(dtype, kl, tau, up):
    args = _inputs(4, 60, 5003, dtype, seed=3)
    _check(*args, clip=(0.1, 0.3), kl=kl, tau=tau, up=up)


def test_many_rows():
    """More rows than the GPU holds at a time, two CTAs a row."""
    _check(*_inputs(3, 700, 60001, 'f32', seed=5), clip=(0.2, 0.2), kl=0.05, tau=1.0)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_views(dtype):
    """Logits without their last position, with a part of the vocabulary, every second row, one shared by the batch; by-row tensors
    expanded and transposed; a flat batch."""
    full, tokens, old, adv, ref, weight = _inputs(4, 9, 1237, dtype, seed=11)
    cut = lambda v: v[:, :-1]
    _check(full[:, :-1], *[cut(v) for v in (tokens, old, adv, ref, weight)], clip=(0.2, 0.2), kl=0.1, tau=1.0)
    part = full[..., 5:1000]
    _check(part, tokens % 995, old, adv, ref, weight, clip=(0.2, 0.2), kl=0.1, tau=1.0)
    _check(full[:, ::2], *[v[:, ::2] for v in (tokens, old, adv, ref, weight)], clip=(0.2, 0.2), kl=0.1, tau=1.0)
    turned = [v.t().contiguous().t() for v in (tokens, old, adv, ref, weight)]
    a = _check(full, *turned, clip=(0.2, 0.2), kl=0.1, tau=1.0)
    b = _check(full.view(36, -1), *[v.reshape(36) for v in (tokens, old, adv, ref, weight)], clip=(0.2, 0.2), kl=0.1, tau=1.0)
    assert a[0] == b[0] and torch.equal(a[2].view(36, -1), b[2])
    _check(full, tokens, old, adv[:, :1].expand(4, 9), ref, weight[:1, :1].expand(4, 9), clip=(0.2, 0.2), kl=0.1, tau=1.0)


def test_default_weight():
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, _ = _inputs(3, 5, 100, 'f32')
    loss, _ = policy_loss(logits, tokens, old, adv)
    even, _ = policy_loss(logits, tokens, old, adv, weight=torch.full_like(old, 1 / 15))
    assert loss == even


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', [77, 4099, 50304])
def test_uncounted_rows(dtype, V):
    """What rows of weight 0 hold does not matter: NaN, infinities, tokens out of range; all rows of weight 0 give 0."""
    from treeattn_b200 import _ops
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(2, 6, V, dtype, seed=2)
    weight[0, 2] = weight[1, 5] = 0
    clean = _check(logits, tokens, old, adv, ref, weight, clip=(0.2, 0.2), kl=0.1, tau=1.0)
    for t in (logits, old, adv, ref):
        t[0, 2], t[1, 5] = math.nan, -math.inf
    tokens[0, 2], tokens[1, 5] = -100, 1 << 40
    x = logits.requires_grad_()
    loss, logp = policy_loss(x, tokens, old, adv, ref_logp=ref, weight=weight, kl=0.1)
    grad, = torch.autograd.grad(loss, x)
    assert loss == clean[0] and torch.equal(logp, clean[1]) and torch.equal(grad, clean[2])
    assert logp[0, 2] == 0 and (grad[0, 2] == 0).all() and (grad[1, 5] == 0).all()
    loss, logp = policy_loss(x, tokens, old, adv, ref_logp=ref, weight=torch.zeros_like(weight), kl=0.1)
    grad, = torch.autograd.grad(loss, x)
    assert loss == 0 and (logp == 0).all() and (grad == 0).all()
    assert _ops.device_error()[0] == 0


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('V', [50, 40000, 200003])
def test_values_at_the_ends(dtype, V):
    """Words banned by -inf (whole shares of a row among them), large logits, and rows that are NaN by the formula: all -inf, +inf, NaN,
    a token outside the vocabulary. The other rows keep their values."""
    from treeattn_b200 import _ops
    from treeattn_b200.losses import policy_loss, token_logp
    big = 3e38 if dtype != 'f16' else 6e4
    logits, tokens, old, adv, ref, weight = _inputs(1, 8, V, dtype, seed=4)
    weight[:] = 0.1
    logits[0, 0, : V // 2] = -math.inf
    tokens[0, 0] = V - 1
    logits[0, 1] = -math.inf
    logits[0, 1, 3] = 1.5  # one word left: probability 1
    tokens[0, 1] = 3
    logits[0, 2, 5] = big
    tokens[0, 2] = 5
    logits[0, 3] = -math.inf
    logits[0, 4, 7] = math.inf
    logits[0, 5, V - 1] = math.nan
    tokens[0, 6] = V
    lp = logits.double().log_softmax(-1).gather(-1, tokens.clamp(max=V - 1)[..., None])[..., 0]
    old[:] = torch.where(lp.isfinite(), lp, 0).float()
    x = logits.clone().requires_grad_()
    loss, logp = policy_loss(x, tokens, old, adv, weight=weight)
    grad, = torch.autograd.grad(loss, x)
    assert loss.isnan()
    bad = [3, 4, 5, 6]
    for t in bad:
        assert logp[0, t].isnan() and grad[0, t].isnan().all()
    assert _ops.device_error() == (3, 19, 6, V)
    good = [0, 1, 2, 7]
    assert (logp[0, good].double() - lp[0, good]).abs().max() <= 4 * _logp_error(logits[:, [0, 7]], 1.0)
    p = logits[0, good].double().softmax(-1)
    hot = torch.nn.functional.one_hot(tokens[0, good], V)
    want = (-0.1 * adv[0, good, None].double()) * (hot - p)  # the ratio is 1
    tol = want.abs() * torch.finfo(DT[dtype]).eps / 2 * 1.01 + 0.1 * adv.abs().max() * 1e-4 * (p + hot) + 2.0 ** -24
    assert ((grad[0, good].double() - want).abs() <= tol).all()
    assert torch.equal(torch.isnan(token_logp(logits, tokens)), torch.isnan(logp))
    assert _ops.device_error()[0] == 3


def test_borders_of_the_clip():
    """Where the ratio is the same on both sides of a minimum the free side's gradient flows: inside, and where clipping helps."""
    from treeattn_b200.losses import policy_loss
    logits = torch.zeros(1, 6, 2, device='cuda', requires_grad=True)
    tokens = torch.zeros(1, 6, device='cuda', dtype=torch.int64)
    lp = math.log(0.5)
    ratio = torch.tensor([[0.5, 0.5, 1.0, 1.0, 1.5, 1.5]], device='cuda')
    adv = torch.tensor([[1.0, -1.0, 1.0, -1.0, 1.0, -1.0]], device='cuda')
    loss, _ = policy_loss(logits, tokens, lp - ratio.log(), adv, weight=torch.ones(1, 6, device='cuda'))
    grad, = torch.autograd.grad(loss, logits)
    want = -(adv * ratio * torch.tensor([1, 0, 1, 1, 0, 1.0], device='cuda')) * 0.5
    assert (grad[0, :, 0] - want[0]).abs().max() < 1e-6 and (grad[0, :, 1] + want[0]).abs().max() < 1e-6
    assert abs(float(loss.detach()) - float((-torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)).sum())) < 1e-5


def test_gradient_against_differences():
    """Central differences of the loss itself: steps of 2^-6, whose third-order term is below 2^-12 / 6 times a few slopes, over a loss
    held to about 2^-22."""
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(2, 3, 11, 'f32', seed=9, spread=1.0)
    weight[:] = 1.0
    old = old + 0.05 * adv.sign()  # (away from the borders: the largest step moves a ratio by 2^-6)
    f = lambda z: policy_loss(z, tokens, old, adv, ref_logp=ref, weight=weight, kl=0.3, clip=(0.9, 9.0))[0]
    x = logits.clone().requires_grad_()
    grad, = torch.autograd.grad(f(x), x)
    h = 2.0 ** -6
    for i in range(66):
        step = torch.zeros(66, device='cuda')
        step[i] = h
        step = step.view(2, 3, 11)
        diff = (f(logits + step).double() - f(logits - step).double()) / (2 * h)
        size = 1 + float(adv.abs().max()) * 3
        assert abs(float(diff) - float(grad.view(-1)[i])) <= (h * h + 2.0 ** -21 / h) * size


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,T,V', [(1, 1, 1), (2, 3, 9), (1, 40, 1001), (3, 2, 50257), (1, 1, 262144)])
def test_token_logp(B, T, V, dtype):
    from treeattn_b200.losses import token_logp
    logits, tokens, *_ = _inputs(B, T, V, dtype, seed=V + 1)
    up = torch.randn(T, B, device='cuda').t() * 0.3
    up[0, 0] = 0
    for tau in (1.0, 0.6):
        x, z = logits.clone().requires_grad_(), logits.double().requires_grad_()
        logp = token_logp(x, tokens, temperature=tau)
        assert torch.equal(logp, token_logp(logits, tokens, temperature=tau))
        want = (z / tau).log_softmax(-1).gather(-1, tokens[..., None])[..., 0]
        e = _logp_error(logits, tau)
        assert (logp.double() - want).abs().max() <= e
        grad, = torch.autograd.grad(logp, x, up)
        rg, = torch.autograd.grad(want, z, up.double())
        p = (logits.double() / tau).softmax(-1)
        hot = torch.nn.functional.one_hot(tokens, V)
        tol = rg.abs() * torch.finfo(DT[dtype]).eps / 2 * 1.01 + up.abs()[..., None] / tau * 4 * (e + 8 * 2.0 ** -24) * (p + hot) + 2.0 ** -24 * (
            dtype == 'f16') + 2.0 ** -126
        assert ((grad.double() - rg).abs() <= tol).all()
        assert (grad[0, 0] == 0).all()


def test_backward_twice_and_after_changes():
    """A second backward pass gives the same gradient whatever was done to the first one; logits changed in between are refused."""
    from treeattn_b200.losses import policy_loss, token_logp
    for dtype in ('f32', 'bf16', 'f16'):
        logits, tokens, old, adv, ref, weight = _inputs(2, 5, 3001, dtype, seed=6)
        x = logits.clone().requires_grad_()
        loss, _ = policy_loss(x, tokens, old, adv, ref_logp=ref, weight=weight, kl=0.1)
        g1, = torch.autograd.grad(loss, x, retain_graph=True)
        keep = g1.clone()
        g1.mul_(7)
        g2, = torch.autograd.grad(loss, x, retain_graph=True)
        # formed from the saved sums: one row's exponentials about another maximum differ by a few steps of 2^-24 before rounding
        assert (g2.double() - keep.double()).abs().max() <= (torch.finfo(DT[dtype]).eps + 2.0 ** -20) * keep.abs().max().double()
        g3, = torch.autograd.grad(loss, x, torch.tensor(2.0, device='cuda'), retain_graph=True)
        assert torch.equal(g3, g2 * 2) or dtype == 'f16'
        assert torch.equal(torch.autograd.grad(loss, x, retain_graph=True)[0], g2)
        y = x * 1
        loss, _ = policy_loss(y, tokens, old, adv, weight=weight)
        lp = token_logp(y, tokens)
        y.data  # (not an in-place change)
        with torch.no_grad():
            y.add_(1)
        for out in (loss, lp.sum()):
            with pytest.raises(RuntimeError, match='inplace'):
                torch.autograd.grad(out, x, retain_graph=True)


def test_saved_elsewhere():
    """Saved tensors that come back from host memory, at other addresses."""
    from treeattn_b200.losses import policy_loss, token_logp
    logits, tokens, old, adv, ref, weight = _inputs(2, 5, 3001, 'f16', seed=6)
    up = torch.rand(2, 5, device='cuda')
    grads = []
    for elsewhere in (False, True):
        x = logits.clone().requires_grad_()
        with torch.autograd.graph.save_on_cpu() if elsewhere else torch.enable_grad():
            y = x * 1
            loss, lp = policy_loss(y, tokens, old, adv, weight=weight)[0], token_logp(y, tokens)
        del y
        torch.randn(1 << 20, device='cuda')
        grads.append(torch.autograd.grad([loss, lp], x, [torch.tensor(1.0, device='cuda'), up])[0])
    assert torch.equal(*grads)


def test_no_gradient_asked():
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(2, 5, 301, 'bf16')
    with torch.no_grad():
        a, la = policy_loss(logits.requires_grad_(), tokens, old, adv, weight=weight)
    b, lb = policy_loss(logits, tokens, old, adv, weight=weight)
    assert not a.requires_grad and b.requires_grad and not lb.requires_grad and a == b and torch.equal(la, lb)
    with pytest.raises(ValueError, match='no gradient of old_logp'):
        policy_loss(logits, tokens, old.clone().requires_grad_(), adv)
    empty = policy_loss(logits[:0], tokens[:0], old[:0], adv[:0])
    assert empty[0] == 0 and empty[1].shape == (0, 5)


def test_captured():
    """Forward and backward in one captured graph: replays follow the inputs; another stream's calls run beside them."""
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(2, 8, 2003, 'bf16', seed=8)
    x = logits.clone().requires_grad_()

    def step():
        loss, logp = policy_loss(x, tokens, old, adv, ref_logp=ref, weight=weight, kl=0.1)
        return loss, logp, torch.autograd.grad(loss, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    graph.replay()
    for got, want in zip(outs, first):
        assert torch.equal(got, want)
    other = _inputs(2, 8, 2003, 'bf16', seed=9)
    with torch.no_grad():
        x.copy_(other[0])
        tokens.copy_(other[1])
        old.copy_(other[2])
    graph.replay()
    for got, want in zip(outs, step()):
        assert torch.equal(got, want)


def test_training_a_model_on_its_answers():
    """GPT's logits through the loss: the model's gradients are those of the same loss built from torch's own operations."""
    from treeattn_b200.config import Config
    from treeattn_b200.losses import policy_loss, token_logp
    from treeattn_b200.model import GPT
    torch.manual_seed(0)
    cfg = Config(attn='seg', vocab_size=211, seq_len=64, n_layer=2, n_head=2, n_embd=64, neighbors=False, chunk=64)
    model = GPT(cfg).cuda()
    idx = torch.randint(0, 211, (4, 64), device='cuda')
    weight = torch.zeros(4, 63, device='cuda')
    weight[:, 20:] = 1 / (4 * 43)
    adv = torch.tensor([1.0, -0.5, 0.3, -0.8], device='cuda')[:, None].expand(4, 63)
    with torch.no_grad():
        old = token_logp(model(idx)[0][:, :-1], idx[:, 1:])
        ref = old + 0.1 * torch.randn_like(old)
    logits = model(idx)[0]
    loss, logp = policy_loss(logits[:, :-1], idx[:, 1:], old, adv, ref_logp=ref, weight=weight, kl=0.1)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    logits = model(idx)[0]
    lp = logits[:, :-1].log_softmax(-1).gather(-1, idx[:, 1:, None])[..., 0]
    rho = (lp - old).exp()
    d = ref - lp
    want = (weight * (-torch.minimum(rho * adv, rho.clamp(0.8, 1.2) * adv) + 0.1 * (d.exp() - d - 1))).sum()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
    for n, p in model.named_parameters():
        assert (got[n] - p.grad).abs().max() <= 1e-4 * max(float(p.grad.abs().max()), 1e-3), n


def _banned(B, T, V, dtype, value, seed):
    """Rows whose words are banned by a finite value but for a few, in different places of the row; the tokens are among those."""
    logits, tokens, old, adv, ref, weight = _inputs(B, T, V, dtype, seed=seed)
    free = torch.zeros(B, T, V, device='cuda', dtype=torch.bool)
    for i in range(B * T):
        at = (i * 7919 * 13) % (V - 40)
        free.view(B * T, V)[i, at:at + 40] = True
        tokens.view(-1)[i] = at + i % 40
    z = logits.double()
    lp = z.masked_fill(~free, -math.inf).log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    shift = lp - z.log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    return logits.masked_fill(~free, value), free, tokens, old + shift, adv, ref + shift, weight.clamp(min=1e-3)


@pytest.mark.parametrize('value', [-1e4, -1e9, -1e10, -1e12, -1e20, -1e29, -1e30, -3e38])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('B,T,V', [(1, 2, 50304), (2, 200, 4099), (1, 1, 200003)])
def test_words_banned_by_a_finite_value(B, T, V, dtype, value):
    """Whole pieces, threads' and CTAs' shares of a row hold one large negative number: its words weigh nothing, the others what they
    weigh among themselves. A banned word lies so far off that its probability is 0 in 64 bits too."""
    from treeattn_b200.losses import policy_loss, token_logp
    if dtype == 'f16' and value < -6e4:
        value = -6e4
    logits, free, tokens, old, adv, ref, weight = _banned(B, T, V, dtype, value, seed=V + 3)
    # (the spread is the free words')
    e = _logp_error(torch.where(free, logits, 0), 1.0)
    rl, rp, rg = _reference(logits, tokens, old, adv, ref, weight, 0.2, 0.28, 0.05, 1.0)
    rho = (rp - old.double()).exp()
    size = weight.double() * (adv.double().abs() * rho + 0.05 * (1 + (ref.double() - rp).exp()))
    edge = ((rho - 0.8).abs() < 4 * e) | ((rho - 1.28).abs() < 4 * e)
    p = logits.double().softmax(-1)
    hot = torch.nn.functional.one_hot(tokens, V).double()
    least = {'f32': 2.0 ** -126, 'bf16': 2.0 ** -126, 'f16': 2.0 ** -24}[dtype]
    tol = rg.abs() * torch.finfo(logits.dtype).eps / 2 * 1.01 + size[..., None] * 4 * (e + 8 * 2.0 ** -24) * (p + hot) + least
    x = logits.clone().requires_grad_()
    kw = dict(ref_logp=ref, weight=weight, clip=(0.2, 0.28), kl=0.05)
    loss, logp = policy_loss(x, tokens, old, adv, **kw)
    grad, = torch.autograd.grad(loss, x, retain_graph=True)
    again, = torch.autograd.grad(loss, x)  # formed from the saved sums
    bare, blogp = policy_loss(logits, tokens, old, adv, **kw)
    for lp in (logp, blogp, token_logp(logits, tokens)):
        assert (lp.double() - rp).abs().max() <= e
    for l in (loss, bare):
        assert (l.detach().double() - rl).abs() <= 2 * (e + 8 * 2.0 ** -24) * size.sum()
    for g in (grad, again):
        assert (((g.double() - rg).abs() <= tol) | edge[..., None]).all()
    up = torch.rand(B, T, device='cuda') + 0.5
    g, = torch.autograd.grad(token_logp(x, tokens), x, up)
    want = up.double()[..., None] * (hot - p)
    assert ((g.double() - want).abs() <= want.abs() * torch.finfo(logits.dtype).eps / 2 * 1.01 + up[..., None] * 4 * (e + 8 * 2.0 ** -24) * (p + hot) +
            least).all()


def test_references_beside_the_border():
    """Rows whose products with log2(e) lie on both sides of 2^20, where an exponent's reference changes its form: sums about one and
    about the other meet in one row."""
    from treeattn_b200.losses import token_logp
    g = torch.Generator(device='cuda').manual_seed(1)
    for border in (2.0 ** 20 * math.log(2), -2.0 ** 20 * math.log(2)):
        z = (torch.randint(-128, 129, (64, 9001), device='cuda', generator=g) / 16 + round(border)).float()
        x = z.clone().requires_grad_()
        tokens = torch.randint(0, 9001, (64,), device='cuda', generator=g)
        logp = token_logp(x, tokens)
        want = z.double().log_softmax(-1).gather(1, tokens[:, None])[:, 0]
        assert (logp.double() - want).abs().max() <= _logp_error(z, 1.0)


@pytest.mark.parametrize('c', [0.0, 100.0, 1e4, -1e4, 2.0 ** 19, 1e6, -1e6])
@pytest.mark.parametrize('tau', [1.0, 0.125])
def test_rows_far_from_zero(c, tau):
    """A constant added to a row changes nothing (the sums are exact: words in steps of 1/16): logp, loss and the fp32 gradient keep the
    accuracy that the row's spread allows, and the gradient is the same whether the forward pass formed it or the backward pass did."""
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(2, 8, 3001, 'f32', seed=12)
    logits = (logits * 16).round() / 16
    lp = (logits.double() / tau).log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    args = (logits + c, tokens, lp + (old - lp).clamp(-0.3, 0.3), adv, lp + 0.2, weight)
    assert torch.equal(args[0].double() - c, logits.double())
    _, _, grad = _check(*args, clip=(0.2, 0.28), kl=0.05, tau=tau)
    _, _, twice = _check(*args, clip=(0.2, 0.28), kl=0.05, tau=tau, up=2.0)
    # p by the same exponentials: products in another order, 4 steps of 2^-24, and what the token's sum cancels
    p = (logits.double() / tau).softmax(-1)
    hot = torch.nn.functional.one_hot(tokens, 3001)
    slope = grad.double().abs().sum(-1, keepdim=True)
    assert ((twice.double() / 2 - grad.double()).abs() <= 4 * 2.0 ** -24 * slope * (p + hot) + 2.0 ** -126).all()


@pytest.mark.parametrize('c', [0.0, 100.0, 250.0, 512.0])
def test_bf16_rows_far_from_zero(c):
    """The same in bf16, on both sides of where the factor leaves the exponent."""
    logits, tokens, old, adv, ref, weight = _inputs(2, 8, 3001, 'bf16', seed=12)
    logits = logits.float().round()
    lp = logits.double().log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    logits = (logits + c).to(torch.bfloat16)
    moved = logits.double().log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    _check(logits, tokens, moved + (old - lp).clamp(-0.3, 0.3), adv, moved + 0.2, weight, clip=(0.2, 0.28), kl=0.05, tau=1.0)


@pytest.mark.parametrize('V', [8192, 8200])
def test_logits_written_by_the_launch_before(V):
    """Logits that a kernel of this library writes, which lets the next launch begin before it ends: the losses wait for them."""
    from treeattn_b200.adapters import adapter_add
    from treeattn_b200.losses import policy_loss, token_logp
    g = torch.Generator(device='cuda').manual_seed(7)
    rand = lambda *s: torch.randn(*s, device='cuda', generator=g).to(torch.bfloat16)
    n, ys = 300, [rand(300, V) for _ in range(4)]
    x, a, b = rand(n, 64), rand(1, 8, 64), rand(1, V, 8)
    start, which = torch.tensor([0, n], device='cuda', dtype=torch.int32), torch.zeros(1, device='cuda', dtype=torch.int32)
    tokens = torch.randint(0, V, (n,), device='cuda', generator=g)
    old, adv = torch.full((n,), -9.0, device='cuda'), torch.randn(n, device='cuda', generator=g)
    up = torch.ones(n, device='cuda')
    outs = []

    def losses(logits):
        z = logits.detach().requires_grad_()
        lp = token_logp(z, tokens)
        loss, lp2 = policy_loss(logits, tokens, old, adv, clip=100.0)
        return [token_logp(logits, tokens), lp.detach(), loss, lp2, torch.autograd.grad(lp, z, up)[0]]

    want = []
    for y in ys:
        logits = adapter_add(y, x, a, b, start, which, n)
        torch.cuda.synchronize()
        want.append(losses(logits))
    logits = torch.empty_like(ys[0])
    for i in range(200):
        adapter_add(ys[i % 4], x, a, b, start, which, n, out=logits)
        outs.append(losses(logits) if i % 10 == 0 else [token_logp(logits, tokens)])
    for i, got in enumerate(outs):
        for o, w in zip(got, want[i % 4]):
            assert torch.equal(o, w)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_an_advantage_that_is_nan(dtype):
    """A counted row whose advantage is NaN has a NaN gradient beside its NaN loss, whichever side of the clip its ratio lies on; the
    other rows keep theirs."""
    from treeattn_b200.losses import policy_loss
    logits, tokens, old, adv, ref, weight = _inputs(1, 6, 1003, dtype, seed=21)
    lp = logits.double().log_softmax(-1).gather(-1, tokens[..., None])[..., 0].float()
    old = lp - torch.tensor([[-0.5, 0.0, 0.5, 0.0, -0.5, 0.5]], device='cuda')
    weight[:] = 0.2
    x = logits.requires_grad_()
    want, = torch.autograd.grad(policy_loss(x, tokens, old, adv, weight=weight)[0], x)
    adv[0, :3] = math.nan
    loss, _ = policy_loss(x, tokens, old, adv, weight=weight)
    got, = torch.autograd.grad(loss, x)
    assert loss.isnan() and got[0, :3].isnan().all() and torch.equal(got[0, 3:], want[0, 3:])
