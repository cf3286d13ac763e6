"""Cases of three sets of operators around sampling from one model, training it on the samples, and serving what was trained:

copy, fork   records of the 8-bit paged cache moved inside their pools (compaction) and the 16-bit open pages of sequences copied to
             other slots of the batch (a prompt forked into a group of samples, beams reordered), over all layers at once
adapter      low-rank adapters of many requests beside a shared projection: out = y + scale_a (x A_a^T) B_a^T on the rows of each
             sequence, a = which[sequence]; serving, and training with the gradients of y, x, A and B
policy, logp the clipped policy loss with its KL term over a vocabulary's logits, with the gradient; the tokens' log-probabilities

A pool keeps one record of 2 * page * dh + 16 bytes per (page, kv head), the open pages are (batch, kv head, 2, 2, page * dh) in
16 bits (see perf/operators.py)."""
import math

import torch

own = False

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    def copy(name, layers, pages, moves, Hkv, dh, page):
        return dict(name=name, op='copy', layers=layers, pages=pages, moves=moves, Hkv=Hkv, dh=dh, page=page, dtype='bf16')

    def fork(name, layers, B, moves, Hkv, dh, page, dtype, beams):
        return dict(name=name, op='fork', layers=layers, B=B, moves=moves, Hkv=Hkv, dh=dh, page=page, dtype=dtype, beams=beams)

    def adapter(name, B, n, K, N, rank, adapters, dtype, ragged, train=False):
        return dict(name=name, op='adapter', B=B, n=n, K=K, N=N, rank=rank, adapters=adapters, dtype=dtype, ragged=ragged,
                    train=train)

    def policy(name, B, T, V, dtype, ragged, kl, temperature):
        return dict(name=name, op='policy', B=B, T=T, V=V, dtype=dtype, ragged=ragged, kl=kl, temperature=temperature)

    def logp(name, B, T, V, dtype, temperature, train):
        return dict(name=name, op='logp', B=B, T=T, V=V, dtype=dtype, temperature=temperature, train=train)

    return [
        # a step of beam search over eight slots, which take over one another's sequences, chains and cycles among them: latency
        fork('reorder_beams_8', 12, 8, 6, 12, 64, 64, 'f16', True),
        # one prompt into a group of 64 samples, all layers of the serving configuration
        fork('fork_group_64', 12, 64, 63, 12, 64, 64, 'bf16', False),
        # a pool shrunk by a third: the pages at its end move into the holes
        copy('compact_pool', 12, 2048, 683, 12, 64, 64),
        # a lone user's token
        adapter('adapter_one', 1, 1, 2048, 2048, 8, 4, 'f16', False),
        # a decode batch, each request with an adapter of its own choice
        adapter('adapter_decode_64', 64, 1, 768, 2304, 16, 24, 'bf16', True),
        # prompts of uneven lengths through a wide projection
        adapter('adapter_prompt_ragged', 8, 1001, 2048, 6144, 32, 8, 'bf16', True),
        # adapters in training: the forward and the backward pass of one projection
        adapter('adapter_train', 8, 2048, 768, 2304, 16, 2, 'bf16', False, True),
        # one short answer
        policy('policy_short', 1, 33, 50304, 'f32', False, 0.05, 1.0),
        # answers of uneven lengths, a vocabulary whose rows are not aligned, sampled below temperature 1
        policy('policy_ragged', 5, 411, 50257, 'f16', True, 0.02, 0.8),
        # a training step: eight answers of 1024 tokens
        policy('policy_train', 8, 1024, 50304, 'bf16', True, 0.04, 1.0),
        # the reference model's log-probabilities of sampled tokens
        logp('logp_score', 16, 512, 50304, 'bf16', 1.0, False),
        # log-probabilities that a loss of the program's own is built on, and their gradient
        logp('logp_train', 4, 300, 32003, 'bf16', 1.0, True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(['copy', 'fork', 'adapter', 'adapter', 'train', 'policy', 'policy', 'logp'])
    if op in ('copy', 'fork'):
        dh, page, Hkv = rng.choice([16, 32, 64, 64, 128]), rng.choice([16, 32, 64]), rng.choice([1, 2, 3, 4, 8, 12, 16])
        layers = rng.choice([1, 2, 6, 12, 24, 30])
        base = dict(op=op, layers=layers, Hkv=Hkv, dh=dh, page=page, dtype=rng.choice(['bf16', 'f16']))
        if op == 'copy':
            room = 12 * 683 * 12 * 64 * 64 // (layers * Hkv * dh * page)
            moves = max(1, min(_log(rng, 1, 6000), room))
            return dict(base, moves=moves, pages=moves * 2 + rng.randint(1, 200))
        B = rng.randint(2, 64)
        room = 12 * 63 * 12 * 64 * 64 // (layers * Hkv * dh * page)
        return dict(base, B=B, moves=max(1, min(rng.randint(1, B - 1), room)), beams=rng.random() < 0.5)
    if op in ('adapter', 'train'):
        K, N = 8 * _log(rng, 8, 800), 8 * _log(rng, 8, 800)
        rank = 8 * _log(rng, 1, 16)
        n = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, 2048)]) if op == 'adapter' else _log(rng, 17, 2048)
        room = 8 * 2048 * 7000 * 16
        B = max(1, min(_log(rng, 1, 64), room // (n * (K + N) * max(16, rank))))
        return dict(op='adapter', B=B, n=n, K=K, N=N, rank=rank, adapters=rng.choice([1, 2, 3, 8, 16, 33]),
                    dtype='bf16' if op == 'train' else rng.choice(['bf16', 'f16']), ragged=rng.random() < 0.7,
                    train=op == 'train')
    dtype = rng.choice(['bf16', 'bf16', 'f32', 'f16'])
    V = _log(rng, 1000, 131000)
    room = 8 * 1024 * 50304 // (2 if dtype == 'f32' else 1)
    T = _log(rng, 1, 2048)
    B = max(1, min(_log(rng, 1, 32), room // (T * V)))
    base = dict(op=op, B=B, T=min(T, room // V), V=V, dtype=dtype, temperature=rng.choice([1.0, 1.0, 0.7, 1.3]))
    if op == 'logp':
        return dict(base, train=rng.random() < 0.5)
    return dict(base, ragged=rng.random() < 0.7, kl=rng.choice([0.0, round(rng.uniform(0.01, 0.2), 3)]))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    make = dict(copy=prepare_records, fork=prepare_records, adapter=prepare_adapter, policy=prepare_policy,
                logp=prepare_policy)[case['op']]
    return make(dict(case), g)


def prepare_records(c, g):
    """All layers' pools or open pages, and which record goes where: lists, as the host's bookkeeping gives them."""
    P, dh, Hkv, dev = c['page'], c['dh'], c['Hkv'], 'cuda'
    s = dict(op=c['op'], page=P, dh=dh)
    B, n_pages = (1, c['pages']) if c['op'] == 'copy' else (c['B'], 1)
    s['pool'] = [torch.randint(0, 256, (n_pages, Hkv, 2 * P * dh + 16), device=dev, generator=g, dtype=torch.uint8)
                 for _ in range(c['layers'])]
    s['tail'] = [torch.randn(B, Hkv, 2, 2, P * dh, device=dev, generator=g, dtype=DT[c['dtype']]) for _ in range(c['layers'])]
    s['table'] = torch.zeros(B, 4, device=dev, dtype=torch.int32)
    m = c['moves']
    if c['op'] == 'copy':  # pages at the pool's end into holes before them
        keep = c['pages'] - m
        s['src'] = (keep + torch.randperm(m, device=dev, generator=g)).tolist()
        s['dst'] = torch.randperm(keep, device=dev, generator=g)[:m].tolist()
    elif c['beams']:  # any slot from any other
        s['dst'] = torch.randperm(B, device=dev, generator=g)[:m].tolist()
        s['src'] = torch.randint(0, B, (m,), device=dev, generator=g).tolist()
    else:  # a prompt's slot into others
        slots = torch.randperm(B, device=dev, generator=g).tolist()
        s['dst'], s['src'] = slots[1:m + 1], [slots[0]] * m
    return s


def prepare_adapter(c, g):
    dev, dt, B, n = 'cuda', DT[c['dtype']], c['B'], c['n']
    K, N, r, na = c['K'], c['N'], c['rank'], c['adapters']
    which = torch.randint(0, na, (B,), device=dev, generator=g)
    count = torch.full((B,), n, device=dev)
    if c['ragged']:  # uneven lengths; in a larger batch one sequence has nothing new, one has no adapter
        count = n - torch.arange(B, device=dev) * 7919 % (n // 2 + 1) if n > 1 else count
        if B >= 4:
            count[1] = 0
            which[2] = -1
    start = torch.zeros(B + 1, device=dev, dtype=torch.int32)
    start[1:] = count.cumsum(0)
    rows = int(start[-1])

    def rand(*shape, by=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * by).to(dt)

    s = dict(op='adapter', train=c['train'], n=n, start=start, which=which.int(), x=rand(rows, K), y=rand(rows, N),
             a=rand(na, r, K, by=1 / math.sqrt(K)), b=rand(na, N, r, by=0.3 / math.sqrt(r)),
             scale=torch.rand(na, device=dev, generator=g) + 0.5)
    if c['train']:
        s['dy'] = rand(rows, N, by=1e-3)
        s['leaves'] = [s[k].detach().requires_grad_() for k in ('y', 'x', 'a', 'b')]
    return s


def prepare_policy(c, g):
    dev, B, T, V, tau = 'cuda', c['B'], c['T'], c['V'], c['temperature']
    logits = torch.empty(B, T, V, device=dev, dtype=DT[c['dtype']])
    tokens = torch.empty(B, T, device=dev, dtype=torch.int64)
    logp = torch.empty(B, T, device=dev)
    for i in range(B):  # tokens drawn from the policy that the logits give
        z = (torch.randn(T, V, device=dev, generator=g) * 2.5).to(logits.dtype)
        logits[i] = z
        z = z.float() / tau
        tokens[i] = (z - torch.empty_like(z).exponential_(generator=g).log_()).argmax(-1)
        logp[i] = z.log_softmax(-1).gather(1, tokens[i][:, None])[:, 0]
    s = dict(op=c['op'], logits=logits, tokens=tokens, tau=tau)
    if c['op'] == 'logp':
        s['train'] = c['train']
        if c['train']:
            s.update(leaf=logits.detach().requires_grad_(), dlogp=torch.randn(B, T, device=dev, generator=g) * 0.1)
        return s
    lo, hi = 0.2, 0.28
    far = torch.randn(B, T, device=dev, generator=g) * 0.2  # log of the ratio to the policy that sampled
    for edge in (math.log1p(-lo), math.log1p(hi)):  # but not at a border, where the gradient jumps
        far = torch.where((far - edge).abs() < 1e-4, edge + 2e-4, far)
    length = torch.full((B,), T, device=dev)
    if c['ragged']:
        length -= torch.arange(B, device=dev) * 7919 % (T // 2 + 1)
    valid = torch.arange(T, device=dev) < length[:, None]
    s['tokens'] = tokens.masked_fill_(~valid, -100)
    s.update(old=logp - far, ref=logp + torch.randn(B, T, device=dev, generator=g) * 0.3 if c['kl'] else None, kl=c['kl'],
             adv=torch.randn(B, 1, device=dev, generator=g).expand(B, T), clip=(lo, hi),
             weight=valid / valid.sum(1, keepdim=True) / B, leaf=logits.detach().requires_grad_(),
             up=torch.tensor(4096.0, device=dev) if c['dtype'] == 'f16' else None)  # f16 trains with a scaled loss
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return dict(copy=run_records, fork=run_records, adapter=run_adapter, policy=run_policy, logp=run_logp)[state['op']](state)


def run_records(s):
    if own:
        from treeattn_b200.paged import PagedKV, paged_copy, paged_fork
        if 'caches' not in s:  # a program's caches, made once
            s['caches'] = [PagedKV(p, t, s['table'], s['page'], s['dh']) for p, t in zip(s['pool'], s['tail'])]
        if s['op'] == 'copy':
            paged_copy(s['caches'], s['src'], s['dst'])
            return s['pool']
        paged_fork(s['caches'], s['src'], s['dst'])
        return s['tail']
    held = s['pool'] if s['op'] == 'copy' else s['tail']
    src, dst = torch.tensor([s['src'], s['dst']], device='cuda')
    return [t.index_copy_(0, dst, t.index_select(0, src)) for t in held]


def run_adapter(s):
    if own:
        from treeattn_b200.adapters import adapter_add
        if not s['train']:
            return adapter_add(s['y'], s['x'], s['a'], s['b'], s['start'], s['which'], s['n'], scale=s['scale'])
        y, x, a, b = s['leaves']
        out = adapter_add(y, x, a, b, s['start'], s['which'], s['n'], scale=s['scale'])
        dy, dx, da, db = torch.autograd.grad(out, (y, x, a, b), s['dy'])
        return dict(out=out.detach(), dy=dy, dx=dx, da=da, db=db)
    # the sequences' rows side by side, padded to the longest; a sequence without an adapter takes one of scale 0
    start, n, B = s['start'].long(), s['n'], s['which'].shape[0]
    r = torch.arange(s['x'].shape[0], device='cuda')
    seq = torch.searchsorted(start[1:], r, right=True)
    at = r - start[seq]
    which = s['which'].long().clamp(min=0)
    by = torch.where(s['which'] < 0, 0.0, s['scale'][which])[:, None, None]
    A, Bm = s['a'][which].float(), s['b'][which].float()

    def side(t):
        z = torch.zeros(B, n, t.shape[1], device='cuda')
        z[seq, at] = t.float()
        return z

    x = side(s['x'])
    t = x @ A.transpose(1, 2)
    dt = s['y'].dtype
    out = (s['y'].float() + (by * (t @ Bm.transpose(1, 2)))[seq, at]).to(dt)
    if not s['train']:
        return out
    dy = side(s['dy'])
    u = by * (dy @ Bm)
    da, db = torch.zeros(s['a'].shape, device='cuda'), torch.zeros(s['b'].shape, device='cuda')
    da.index_add_(0, which, u.transpose(1, 2) @ x)
    db.index_add_(0, which, by * (dy.transpose(1, 2) @ t))
    return dict(out=out, dy=s['dy'], dx=(u @ A)[seq, at].to(dt), da=da.to(dt), db=db.to(dt))


def run_policy(s):
    if own:
        from treeattn_b200.losses import policy_loss
        loss, logp = policy_loss(s['leaf'], s['tokens'], s['old'], s['adv'], ref_logp=s['ref'], weight=s['weight'],
                                 clip=s['clip'], kl=s['kl'], temperature=s['tau'])
        grad, = torch.autograd.grad(loss, s['leaf'], s['up'])
        return dict(loss=loss.detach(), logp=logp, grad=grad)
    z = s['logits'].float() / s['tau']
    w, adv, (lo, hi) = s['weight'], s['adv'], s['clip']
    y = s['tokens'].clamp(min=0)[..., None]
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    tot = e.sum(-1, keepdim=True)
    logp = torch.where(w > 0, (z.gather(-1, y) - top - tot.log())[..., 0], 0.0)
    ratio = torch.exp(logp - s['old'])
    gain = torch.minimum(ratio * adv, ratio.clamp(1 - lo, 1 + hi) * adv)
    live = torch.where(adv > 0, ratio <= 1 + hi, ratio >= 1 - lo)
    term, slope = -gain, torch.where(live, -adv * ratio, 0.0)
    if s['kl']:
        d = s['ref'] - logp
        term = term + s['kl'] * (torch.exp(d) - d - 1)
        slope = slope + s['kl'] * (1 - torch.exp(d))
    loss = torch.where(w > 0, w * term, 0.0).double().sum().float()
    slope = (torch.where(w > 0, w * slope, 0.0) / s['tau'])[..., None]
    if s['up'] is not None:
        slope = slope * s['up']
    grad = -slope * (e / tot)
    grad.scatter_add_(-1, y, slope)
    return dict(loss=loss, logp=logp, grad=grad.to(s['logits'].dtype))


def run_logp(s):
    if own:
        from treeattn_b200.losses import token_logp
        if not s['train']:
            return token_logp(s['logits'], s['tokens'], temperature=s['tau'])
        logp = token_logp(s['leaf'], s['tokens'], temperature=s['tau'])
        grad, = torch.autograd.grad(logp, s['leaf'], s['dlogp'])
        return dict(logp=logp.detach(), grad=grad)
    z, y = s['logits'].float() / s['tau'], s['tokens'][..., None]
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    tot = e.sum(-1, keepdim=True)
    logp = (z.gather(-1, y) - top - tot.log())[..., 0]
    if not s['train']:
        return logp
    slope = (s['dlogp'] / s['tau'])[..., None]
    grad = (-slope * (e / tot)).scatter_add_(-1, y, slope)
    return dict(logp=logp, grad=grad.to(s['logits'].dtype))


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case['op'] == 'copy':
        return None
    s = prepare(case, seed)
    if case['op'] == 'fork':
        return exact_fork(s)
    return exact_adapter(s) if case['op'] == 'adapter' else exact_policy(s)


def exact_fork(s):
    """Slot by slot, from what all slots held before."""
    out = []
    for held in s['tail']:
        new = held.double()
        for i, j in zip(s['src'], s['dst']):
            new[j] = held[i]
        out.append(new)
    return out


def exact_adapter(s):
    """Sequence by sequence, in 64 bits."""
    start, which = s['start'].tolist(), s['which'].tolist()
    x, out = s['x'].double(), s['y'].double()
    back = s['train']
    if back:
        dy, dx = s['dy'].double(), torch.zeros_like(x)
        da, db = torch.zeros_like(s['a'], dtype=torch.float64), torch.zeros_like(s['b'], dtype=torch.float64)
    for i, a in enumerate(which):
        r = slice(start[i], start[i + 1])
        if a < 0:
            continue
        A, Bm, by = s['a'][a].double(), s['b'][a].double(), float(s['scale'][a])
        out[r] += by * torch.einsum('nr,mr->nm', torch.einsum('nk,rk->nr', x[r], A), Bm)
        if back:
            u = by * torch.einsum('nm,mr->nr', dy[r], Bm)
            dx[r] = torch.einsum('nr,rk->nk', u, A)
            da[a] += torch.einsum('nr,nk->rk', u, x[r])
            db[a] += by * torch.einsum('nm,nr->mr', dy[r], torch.einsum('nk,rk->nr', x[r], A))
    return dict(out=out, dy=dy, dx=dx, da=da, db=db) if back else out


def exact_policy(s):
    """Row by row of the batch, in 64 bits."""
    tau, logits, tokens, train = s['tau'], s['logits'], s['tokens'], s['op'] == 'policy' or s['train']
    logp = torch.zeros(tokens.shape, device='cuda', dtype=torch.float64)
    grad = torch.empty(logits.shape, device='cuda', dtype=torch.float64) if train else None
    loss = torch.zeros((), device='cuda', dtype=torch.float64)
    for i in range(tokens.shape[0]):
        full = (logits[i].double() / tau).log_softmax(-1)
        y = tokens[i].clamp(min=0)[:, None]
        lp = full.gather(1, y)[:, 0]
        logp[i] = lp
        if not train:
            continue
        if s['op'] == 'logp':
            slope = s['dlogp'][i].double()
        else:
            w, adv, old = s['weight'][i].double(), s['adv'][i].double(), s['old'][i].double()
            on = w > 0
            logp[i] = lp.masked_fill(~on, 0)
            lo, hi = 1 - s['clip'][0], 1 + s['clip'][1]
            ratio = (lp - old).exp()
            held = ratio.clip(lo, hi)
            free = ratio * adv <= held * adv
            term = -torch.where(free, ratio, held) * adv
            slope = -adv * ratio * free
            if s['kl']:
                d = s['ref'][i].double() - lp
                term = term + s['kl'] * (d.expm1() - d)
                slope = slope - s['kl'] * d.expm1()
            loss += (w * term)[on].sum()
            slope = (w * slope).masked_fill(~on, 0) * (1.0 if s['up'] is None else float(s['up']))
        slope = slope[:, None] / tau
        hot = torch.zeros_like(full).scatter_(1, y, 1.0)
        grad[i] = slope * (hot - full.exp())
    if s['op'] == 'logp':
        return dict(logp=logp, grad=grad) if train else logp
    return dict(loss=loss, logp=logp, grad=grad)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c['op'] == 'copy':
        return dict(bytes=2.0 * c['layers'] * c['moves'] * c['Hkv'] * (2 * c['page'] * c['dh'] + 16), flops=0.0)
    if c['op'] == 'fork':  # a source that several slots continue is read once
        record = c['layers'] * c['Hkv'] * 4 * c['page'] * c['dh'] * 2.0
        return dict(bytes=record * (c['moves'] + (c['moves'] * 0.7 if c['beams'] else 1)), flops=0.0)
    B = c['B']
    if c['op'] == 'adapter':
        n, K, N, r = c['n'], c['K'], c['N'], c['rank']
        rows = B * n * (0.75 if c['ragged'] and n > 1 else 1.0)
        used = c['adapters'] * (1 - (1 - 1 / c['adapters']) ** B)
        size = used * r * (K + N) * 2.0
        if not c['train']:
            return dict(bytes=rows * (K + 2 * N) * 2 + size, flops=2 * rows * r * (K + N))
        return dict(bytes=rows * (2 * K + 3 * N) * 2 + size + c['adapters'] * r * (K + N) * 2.0, flops=6 * rows * r * (K + N))
    size = 4 if c['dtype'] == 'f32' else 2
    if c['op'] == 'logp':
        rows = B * c['T']
        return dict(bytes=rows * c['V'] * size * (1 + c['train']) + rows * 16.0, flops=4.0 * rows * c['V'] * (1 + c['train']))
    rows = B * c['T'] * (0.75 if c['ragged'] else 1.0)
    return dict(bytes=(rows + B * c['T']) * c['V'] * size + rows * 32.0, flops=8.0 * rows * c['V'])
