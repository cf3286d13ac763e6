"""The paged decoder and speculative decoding against plain torch forwards of the same model."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _model(seed=0, n_layer=2, n_head=4, n_embd=256, vocab=512, seq_len=512):
    from treeattn_b200.config import Config
    from treeattn_b200.engine import weights_from_ours
    from treeattn_b200.model import GPT
    torch.manual_seed(seed)
    cfg = Config(attn='seg', vocab_size=vocab, seq_len=seq_len, n_layer=n_layer, n_head=n_head, n_embd=n_embd, wmax=8, beam=8,
                 local=32, neighbors=False, leaf=16)
    sd = {k: v.detach() * (4.0 if v.dim() == 2 else 1.0) for k, v in GPT(cfg).state_dict().items()}
    return cfg, weights_from_ours(sd, cfg)


def _dense(W, cfg, idx, dtype):
    """Causal dense forward in 64 bits on the weights as `dtype` holds them."""
    d = lambda t: t.to(DEV, dtype).double()
    n = lambda t: t.to(DEV, torch.float32).double()
    B, T = idx.shape
    H, C = cfg.n_head, cfg.n_embd
    x = d(W['wte'])[idx] + d(W['wpe'])[:T]
    mask = torch.ones(T, T, device=DEV, dtype=torch.bool).tril()
    for L in W['layers']:
        q, k, v = [t.view(B, T, H, C // H).transpose(1, 2) for t in
                   (F.layer_norm(x, (C,), n(L['ln1'])) @ d(L['c_attn']).t()).split(C, 2)]
        s = (q @ k.transpose(2, 3) / (C // H) ** 0.5).masked_fill(~mask, -float('inf')).softmax(-1)
        x = x + (s @ v).transpose(1, 2).reshape(B, T, C) @ d(L['c_proj']).t()
        x = x + F.gelu(F.layer_norm(x, (C,), n(L['ln2'])) @ d(L['c_fc']).t()) @ d(L['c_mlp']).t()
    return F.layer_norm(x, (C,), n(W['ln_f'])) @ d(W['wte']).t()


# e4m3 keys and values (half a step 2^-4 of the value) and 16-bit activations through two layers: logits within a tenth of their
# spread, root mean square within a twentieth
def _close(got, want):
    spread = want.std()
    d = got.double() - want
    return d.abs().max() < 0.5 * spread and d.square().mean().sqrt() < 0.05 * spread


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
def test_chunks_drafts_and_single_tokens_agree(dt):
    """The same tokens as one prompt, as chunks, and as runs of a few and single tokens: logits of the 64-bit dense forward."""
    from treeattn_b200.speculative import PagedDecoder
    cfg, W = _model()
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(cfg.vocab_size, (3, 200), generator=g).to(DEV)
    want = _dense(W, cfg, idx, dt)
    for cuts in ([200], [70, 64, 66], [100] + [5] * 18 + [1] * 10):
        dec = PagedDecoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, batch=3, max_len=256, page=32, dtype=dt)
        got, at = [], 0
        for c in cuts:
            got.append(dec.forward(idx[:, at:at + c]))
            at += c
        assert _close(torch.cat(got, 1), want)
    from treeattn_b200 import _ops
    assert _ops.device_error()[0] == 0


def _restart(dec, idx, n):
    """The decoder, emptied and fed the first n tokens."""
    dec.pos, dec._floor = [0] * dec.batch, [0] * dec.batch
    dec.forward(idx[:, :81])
    dec.forward(idx[:, 81:n])
    return dec


def test_cut_back():
    """Drafts that are dropped leave no trace in the logits that follow; what is gone from the 16-bit pages is refused."""
    from treeattn_b200.speculative import PagedDecoder
    cfg, W = _model(1)
    g = torch.Generator().manual_seed(2)
    idx = torch.randint(cfg.vocab_size, (2, 150), generator=g).to(DEV)
    a = PagedDecoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, batch=2, max_len=256, page=16)
    b = PagedDecoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, batch=2, max_len=256, page=16)
    a.forward(idx[:, :93])
    b.forward(idx[:, :93])
    a.forward(torch.randint(cfg.vocab_size, (2, 7), generator=g).to(DEV))
    a.cut_back([93, 95])
    a.cut_back([93, 93])
    assert torch.equal(a.forward(idx[:, 93:98]), b.forward(idx[:, 93:98]))
    with pytest.raises(ValueError, match='cannot go'):
        a.cut_back([98, 60])
    # positions up to 100 (page 6) were written: page 4's place is gone even after going back to page 5 and on from there
    a.cut_back([81, 81])
    a.forward(idx[:, 81:82])
    with pytest.raises(ValueError, match='cannot go'):
        a.cut_back([79, 82])
    assert torch.equal(a.forward(idx[:, 82:98]), PagedDecoder.forward(_restart(b, idx, 82), idx[:, 82:98]))
    with pytest.raises(ValueError, match='cannot go'):
        a.cut_back([99, 98])
    with pytest.raises(ValueError, match='max_len'):
        a.forward(torch.zeros(2, 200, dtype=torch.long, device=DEV))


def _pair(cfg, W, B, dtype=torch.bfloat16):
    from treeattn_b200.engine import Decoder
    from treeattn_b200.speculative import PagedDecoder
    args = (W, cfg.n_layer, cfg.n_head, cfg.n_embd)
    return (Decoder(*args, cfg.seq_len, 'seg', cfg, DEV, batch=B, dtype=dtype),
            PagedDecoder(*args, batch=B, max_len=cfg.seq_len, page=32, dtype=dtype))


def test_greedy_speculation_is_the_dense_models():
    """Greedy: every token that comes out is the dense model's best one (its 64-bit logit within the cache's and the
    activations' error of the largest), drafts stand, and the positions add up."""
    from treeattn_b200.speculative import SpeculativeDecoder
    cfg, W = _model(3)
    B, T = 4, 120
    draft, target = _pair(cfg, W, B)
    dec = SpeculativeDecoder(draft, target, 4, temperature=0)
    prompt = torch.randint(cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(4))
    out = [[int(t)] for t in dec.prefill(prompt)]
    for _ in range(12):
        new = dec.step()
        assert all(1 <= len(x) <= 5 for x in new)
        for o, x in zip(out, new):
            o.extend(x)
        assert target.pos == [T + len(o) - 1 for o in out]
    assert dec.accepted > 0 and sum(map(len, out)) == B + 12 * B + dec.accepted
    for b in range(B):
        idx = torch.cat([prompt[b], torch.tensor(out[b])])[None].to(DEV)
        logits = _dense(W, cfg, idx[:, :-1], torch.bfloat16)[0, T - 1:]
        best = logits.max(-1).values
        chosen = logits.gather(1, idx[0, T:, None])[:, 0]
        assert (best - chosen <= 0.5 * logits.std()).all()
        assert (chosen == best).double().mean() > 0.8
    from treeattn_b200 import _ops
    assert _ops.device_error()[0] == 0


def test_sampled_speculation_runs_and_repeats():
    """Sampling: the same generator seed gives the same tokens; the cache after the rounds gives the logits of a fresh one."""
    from treeattn_b200.speculative import PagedDecoder, SpeculativeDecoder
    cfg, W = _model(5)
    B, T = 3, 77
    prompt = torch.randint(cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(6))
    runs = []
    for _ in range(2):
        draft, target = _pair(cfg, W, B)
        dec = SpeculativeDecoder(draft, target, 3, temperature=0.8, generator=torch.Generator(DEV).manual_seed(7))
        out = [[int(t)] for t in dec.prefill(prompt)]
        for _ in range(10):
            for o, x in zip(out, dec.step()):
                o.extend(x)
        runs.append(out)
    assert runs[0] == runs[1]
    got = target.forward(torch.tensor([[o[-1]] for o in out], device=DEV))[:, 0]  # each at its own position
    for b in range(B):
        fresh = PagedDecoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, batch=1, max_len=cfg.seq_len, page=32)
        want = fresh.forward(torch.cat([prompt[b], torch.tensor(out[b])])[None].to(DEV))[0, -1]
        assert fresh.pos[0] == target.pos[b] and _close(got[b], want.double())


def test_refusals():
    from treeattn_b200.config import Config
    from treeattn_b200.speculative import PagedDecoder, SpeculativeDecoder
    cfg, W = _model()
    draft, target = _pair(cfg, W, 2)
    with pytest.raises(ValueError, match='n_draft'):
        SpeculativeDecoder(draft, target, 32)
    with pytest.raises(ValueError, match='batch'):
        SpeculativeDecoder(draft, _pair(cfg, W, 3)[1])
    with pytest.raises(TypeError, match='float16'):
        PagedDecoder(W, 2, 4, 256, dtype=torch.float32)
    with pytest.raises(ValueError, match='position table'):
        PagedDecoder(W, 2, 4, 256, max_len=4096)
    draft.cfg = Config(**dict(cfg.to_dict(), beam_mode='pred', global_pool=True))
    with pytest.raises(ValueError, match='taken? back|take drafts back'):
        SpeculativeDecoder(draft, target)
    small = PagedDecoder(W, 2, 4, 256, batch=2, max_len=256, page=16, n_pages=5)
    with pytest.raises(MemoryError, match='pages wanted'):
        small.forward(torch.zeros(2, 60, dtype=torch.long, device=DEV))
    assert small.pos == [0, 0]


def test_example_runs():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, 'examples', 'speculative_decode.py'), '--batch', '2', '--prompt',
                        '100', '--tokens', '12'], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert 'tokens/s' in r.stdout


@pytest.mark.parametrize('neighbors', [False, True])
def test_a_context_is_used_to_its_last_position(neighbors):
    """Rounds up to the last position of the caches, with the fused draft kernel and with a draft that borrows neighbours' leaves
    (its stored leaves are indexed by position): every position is generated, nothing is fed beyond, then a round is refused. The
    tokens are the dense model's (greedy)."""
    from treeattn_b200.config import Config
    from treeattn_b200.speculative import SpeculativeDecoder
    cfg, W = _model(3, seq_len=128)
    cfg = Config(**dict(cfg.to_dict(), neighbors=neighbors))
    B, T = 2, 90
    draft, target = _pair(cfg, W, B)
    dec = SpeculativeDecoder(draft, target, 4, temperature=0)
    prompt = torch.randint(cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(4))
    out = [[int(t)] for t in dec.prefill(prompt)]
    while max(target.pos) < 128:
        for o, x in zip(out, dec.step()):
            o.extend(x)
    with pytest.raises(ValueError, match='all 128 positions'):
        dec.step()
    from treeattn_b200 import _ops
    assert _ops.device_error()[0] == 0
    assert target.pos == [T + len(o) - 1 for o in out]
    for b in range(B):
        idx = torch.cat([prompt[b], torch.tensor(out[b])])[None].to(DEV)
        logits = _dense(W, cfg, idx[:, :-1], torch.bfloat16)[0, T - 1:]
        chosen = logits.gather(1, idx[0, T:, None])[:, 0]
        assert (logits.max(-1).values - chosen <= 0.5 * logits.std()).all()


@pytest.mark.parametrize('neighbors', [False, True])
def test_sampled_rounds_follow_the_target(neighbors):
    """The first token of a round and the one before it: over many sequences and rounds of one prompt each pair's count within 5
    standard deviations of what the target's probabilities give, whatever the draft proposes (its weights are another model's)."""
    from treeattn_b200.config import Config
    from treeattn_b200.engine import Decoder
    from treeattn_b200.speculative import PagedDecoder, SpeculativeDecoder
    V, B, T, rounds = 8, 1024, 24, 6
    cfg, W = _model(7, n_layer=1, n_head=2, n_embd=128, vocab=V, seq_len=64)
    cfg = Config(**dict(cfg.to_dict(), neighbors=neighbors))
    _, other = _model(8, n_layer=1, n_head=2, n_embd=128, vocab=V, seq_len=64)
    args = (cfg.n_layer, cfg.n_head, cfg.n_embd)
    draft = Decoder(other, *args, cfg.seq_len, 'seg', cfg, DEV, batch=B, dtype=torch.bfloat16)
    target = PagedDecoder(W, *args, batch=B, max_len=64, page=16)
    dec = SpeculativeDecoder(draft, target, 3, generator=torch.Generator(DEV).manual_seed(1))
    prompt = torch.randint(V, (1, T), generator=torch.Generator().manual_seed(9))
    counts = torch.zeros(V, V, device=DEV, dtype=torch.float64)
    for _ in range(rounds):
        first = dec.prefill(prompt.expand(B, T)).clone()
        second = torch.tensor([x[0] for x in dec.step()], device=DEV)
        counts += torch.bincount(first * V + second, minlength=V * V).view(V, V)
    one = PagedDecoder(W, *args, batch=V, max_len=64, page=16)
    p0 = dec._probs(one.forward(prompt.expand(V, T))[:1, -1])[0].double()
    p1 = dec._probs(one.forward(torch.arange(V)[:, None])[:, -1]).double()
    p = p0[:, None] * p1
    n = B * rounds
    assert 0.02 < dec.accepted / dec.drafted < 0.98  # some drafts stand, some fall
    # (the 16-bit logits of batches of other sizes differ by 2^-8 of them at most: a few per cent of a probability)
    sd = (n * p * (1 - p)).sqrt()
    assert ((counts - n * p).abs() <= 5 * sd + 0.02 * n * p + 1).all(), (counts / n, p)
