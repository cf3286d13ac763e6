"""Cases of the serving operators over the 8-bit paged cache: appending keys and values to it (with the position
rotation), attention over it, and the verification of drafted tokens.

A page holds P tokens. The pool keeps one record of 2 * P * dh + 16 bytes per (page, kv head): the e4m3 codes of the
keys, those of the values, and the two fp32 scales (value = code * scale, scale = largest magnitude / 448, taken once, when
the page's last token arrives). The open page and the one before it are held in 16 bits in `tail` (batch, kv head, page
parity, key / value, P * dh). Both keep their elements in the order in which the tensor-core fragments take them;
k_view and v_view give the token-major view."""
import math

import torch

own = False

DT = {'bf16': torch.bfloat16, 'f16': torch.float16, 'f32': torch.float32}
WS_BYTES = 64 << 20  # scratch for the joined parts of long contexts, zeroed once (it is left zeroed where it counts)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    def app(name, B, n, ctx, Hq, Hkv, dh, page, rot, dtype, ragged):
        return dict(name=name, op='append', B=B, n=n, ctx=ctx, Hq=Hq, Hkv=Hkv, dh=dh, page=page, rot=rot, dtype=dtype,
                    ragged=ragged)

    def att(name, B, n, ctx, Hq, Hkv, dh, page, window, dtype, ragged):
        return dict(name=name, op='attn', B=B, n=n, ctx=ctx, Hq=Hq, Hkv=Hkv, dh=dh, page=page, window=window,
                    dtype=dtype, ragged=ragged)

    def ver(name, B, G, V, dtype, ragged):
        return dict(name=name, op='verify', B=B, G=G, V=V, dtype=dtype, ragged=ragged)

    return [
        # one new token of a few sequences: the append of a small decode batch, launch-bound
        app('append_decode_8', 8, 1, 4096, 12, 12, 64, 64, 64, 'bf16', True),
        # four drafts and a token for each of 64 sequences of uneven lengths
        app('append_drafts_64', 64, 5, 4096, 12, 12, 64, 32, 64, 'f16', True),
        # prompts of uneven lengths, shared key heads, half of the dimensions rotated
        app('append_prompt_ragged', 8, 2011, 300, 16, 4, 128, 16, 64, 'bf16', True),
        # whole prompts of 8192 tokens into an empty cache, positions learned (no rotation)
        app('append_prompt_8192', 4, 8192, 0, 12, 12, 64, 64, 0, 'bf16', False),
        # one sequence, one token: the latency of a lone user's step
        att('attn_one_4096', 1, 1, 4096, 12, 12, 64, 64, 0, 'bf16', False),
        # the decode batch of the serving configuration: 64 sequences of uneven lengths
        att('attn_decode_64', 64, 1, 4351, 12, 12, 64, 64, 0, 'bf16', True),
        # long contexts at head dimension 128
        att('attn_decode_32768', 8, 1, 32768, 16, 16, 128, 64, 0, 'bf16', True),
        # four drafts and a token against shared key heads, sliding window
        att('attn_drafts_window', 24, 5, 9001, 16, 4, 128, 32, 4096, 'f16', True),
        # a prompt's next chunk over what the cache already holds
        att('attn_chunk_512', 2, 512, 4000, 12, 12, 64, 64, 0, 'bf16', True),
        # drafts of one sequence, of a serving batch, and of a large one with a smaller vocabulary
        ver('verify_1', 1, 4, 50304, 'f32', False),
        ver('verify_64', 64, 4, 50304, 'f32', True),
        ver('verify_256', 256, 8, 32000, 'bf16', True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(['append', 'attn', 'verify'])
    if op == 'verify':
        V = _log(rng, 2000, 51000)
        return dict(op=op, B=max(1, min(_log(rng, 1, 256), 8000000 // V)), G=rng.randint(1, 8), V=V,
                    dtype=rng.choice(['f32', 'f32', 'bf16', 'f16']), ragged=rng.random() < 0.7)
    dh = rng.choice([16, 32, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8, 12, 16])
    group = rng.choice([1, 1, 2, 4, 8])
    group = group if group * Hkv <= 32 else 1
    page = rng.choice([16, 32, 64])
    dtype = rng.choice(['bf16', 'bf16', 'f16'])
    ragged = rng.random() < 0.8
    B = _log(rng, 1, 64)
    base = dict(op=op, Hq=Hkv * group, Hkv=Hkv, dh=dh, page=page, dtype=dtype, ragged=ragged)
    if op == 'append':
        n = _log(rng, 1, 8001) | 1
        ctx = rng.choice([0, _log(rng, 1, 20000)])
        room = 32768 * 12 * 64 * 3 // ((group + 2) * Hkv * dh)  # tokens in all, so that no draw exceeds the largest
        n = max(1, min(n, room))
        B = max(1, min(B, room // n, 2000000000 // (Hkv * dh * 2 * (n + ctx + 64))))
        return dict(base, B=B, n=n, ctx=ctx, rot=rng.choice([0, dh // 2, dh, dh]))
    n = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 500)])
    ctx = _log(rng, 1, 32000) | 1
    room = 8 * 16 * 32768 * 128
    ctx = min(ctx, max(1, 12000000000 // (group * Hkv * dh * n * 2)))
    B = max(1, min(B, room // (Hkv * dh * (ctx + n)), 24000000000 // (group * Hkv * dh * n * (ctx + n) * 2)))
    return dict(base, B=B, n=n, ctx=ctx, window=rng.choice([0, 0, _log(rng, 1, 8000)]))


# ------------------------------------------------------------------------------------------------ layout
def k_view(x, P, dh):
    """(..., P * dh) of a page's keys as stored -> the view (..., P/16, 2, 8 | dims): tokens, then head dimensions."""
    E = min(16, dh // 4)
    G = dh // (4 * E)
    d = x.dim() - 1
    return x.unflatten(-1, (P // 16, G, 2, 8, 4, E)).permute(*range(d), d, d + 2, d + 3, d + 1, d + 4, d + 5)


def v_view(x, P, dh):
    """The same of a page's values: (..., P/16, 2, 4, 2 | dims)."""
    M = min(2, dh // 16)
    d = x.dim() - 1
    return x.unflatten(-1, (P // 16, dh // (16 * M), 8, 4, M, 2, 2, 2)).permute(
        *range(d), d, d + 6, d + 3, d + 7, d + 1, d + 4, d + 5, d + 2)


def views(s):
    """The pool's codes and scales and the 16-bit pages, by token and dimension, as views."""
    P, dh, pool, tail = s['page'], s['dh'], s['pool'], s['tail']
    codes = pool[..., :2 * P * dh].view(torch.float8_e4m3fn)
    return dict(k=k_view(codes[..., :P * dh], P, dh), v=v_view(codes[..., P * dh:], P, dh),
                scale=pool.view(torch.float32)[..., -4:-2], tail_k=k_view(tail[:, :, :, 0], P, dh),
                tail_v=v_view(tail[:, :, :, 1], P, dh))


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dev = 'cuda'
    c = dict(case)
    B, dt = c['B'], DT[c['dtype']]
    if c['op'] == 'verify':
        G, V = c['G'], c['V']
        target = torch.randn(B, G + 1, V, device=dev, generator=g) * 2.5
        p = target.softmax(-1)
        q = (target[:, :G] + 0.7 * torch.randn(B, G, V, device=dev, generator=g)).softmax(-1)
        drafts = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, G)
        u = torch.rand(B, G + 1, device=dev, generator=g)
        n = torch.randint(0 if c['ragged'] else G, G + 1, (B,), device=dev, generator=g).int()
        return dict(op='verify', p=p.to(dt), q=q.to(dt), drafts=drafts, u=u, n=n)
    n, ctx, Hq, Hkv, dh, P = c['n'], c['ctx'], c['Hq'], c['Hkv'], c['dh'], c['page']
    if c['ragged']:  # uneven lengths; in a larger batch one sequence has nothing new, one is still empty
        count = n - torch.arange(B, device=dev) * 7919 % (n // 2 + 1) if n > 1 else torch.ones(B, device=dev).long()
        pos = torch.randint(ctx // 2, ctx + 1, (B,), device=dev, generator=g)
        if B >= 4:
            count[1] = 0
            pos[2] = 0
    else:
        count = torch.full((B,), n, device=dev)
        pos = torch.full((B,), ctx, device=dev)
    start = torch.zeros(B + 1, device=dev, dtype=torch.int32)
    start[1:] = count.cumsum(0)
    N = int(start[-1])
    W = -(-(ctx + n) // P)  # pages a sequence can come to hold
    pool = torch.empty(B * W, Hkv, 2 * P * dh + 16, device=dev, dtype=torch.uint8)
    pool[..., :2 * P * dh] = (torch.randn(pool[..., :2 * P * dh].shape, device=dev, generator=g, dtype=dt) * 110).clamp(
        -448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    sc = pool.view(torch.float32)
    sc[..., -4:] = 0
    sc[..., -4:-2] = torch.rand(B * W, Hkv, 2, device=dev, generator=g) * 0.008 + 0.006
    table = torch.randperm(B * W, device=dev, generator=g).int().view(B, W)
    tail = torch.randn(B, Hkv, 2, 2, P * dh, device=dev, generator=g).to(dt)
    qkv = torch.randn(N, (Hq + 2 * Hkv) * dh, device=dev, generator=g).to(dt)  # the projection's rows
    s = dict(op=c['op'], page=P, dh=dh, Hq=Hq, Hkv=Hkv, n=n, pool=pool, table=table, tail=tail, start=start,
             pos=pos.int(), q=qkv[:, :Hq * dh].view(N, Hq, dh), k=qkv[:, Hq * dh:(Hq + Hkv) * dh].view(N, Hkv, dh),
             v=qkv[:, (Hq + Hkv) * dh:].view(N, Hkv, dh))
    if c['op'] == 'attn':
        s.update(window=c['window'], ws=torch.zeros(WS_BYTES, device=dev, dtype=torch.uint8))
        return s
    s.update(rot=c['rot'])
    if c['rot']:
        f = 10000.0 ** (-torch.arange(0, c['rot'], 2, device=dev, dtype=torch.float64) / c['rot'])
        a = torch.arange(ctx + n, device=dev, dtype=torch.float64)[:, None] * f
        s.update(cos=a.cos().float(), sin=a.sin().float())
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if state['op'] == 'verify':
        return run_verify(state)
    return run_append(state) if state['op'] == 'append' else run_attn(state)


def rows_of(s):
    """Each row's sequence and position."""
    r = torch.arange(s['q'].shape[0], device=s['q'].device)
    b = torch.searchsorted(s['start'][1:].long(), r, right=True)
    return r, b, s['pos'][b].long() + r - s['start'][b]


def rotated(x, t, s, ft):
    h = s['rot'] // 2
    x = x.to(ft)
    if not h:
        return x
    c, n = s['cos'].to(ft)[t].unsqueeze(1), s['sin'].to(ft)[t].unsqueeze(1)
    x1, x2 = x[..., :h], x[..., h:2 * h]
    return torch.cat([x1 * c - x2 * n, x2 * c + x1 * n, x[..., 2 * h:]], -1)


def run_append(s):
    if own:
        from treeattn_b200.paged import PagedKV, paged_append
        cache = PagedKV(s['pool'], s['tail'], s['table'], s['page'], s['dh'])
        q = paged_append(cache, s['k'], s['v'], s['start'], s['pos'], s['n'], q=s['q'],
                         rotation=(s['cos'], s['sin']) if s['rot'] else None)
        return dict(views(s), q=q)
    P, dh, Hkv, dt = s['page'], s['dh'], s['Hkv'], s['q'].dtype
    V = views(s)
    start, pos = s['start'].long(), s['pos'].long()
    end = pos + start[1:] - start[:-1]
    r, b, t = rows_of(s)
    q = rotated(s['q'], t, s, torch.float32).to(dt)
    new = torch.stack([rotated(s['k'], t, s, torch.float32).to(dt), s['v']])  # (2, N, Hkv, dh)
    # pages that a sequence's new tokens reach, each token from the new rows or from the open page
    j = pos[:, None] // P + torch.arange((s['n'] - 1) // P + 2, device=q.device)
    at = j[:, :, None] * P + torch.arange(P, device=q.device)
    fresh = (at >= pos[:, None, None]) & (at < end[:, None, None])
    src = torch.where(fresh, start[:-1, None, None] + at - pos[:, None, None], 0)
    full = ((j + 1) * P <= end[:, None]).nonzero()
    fb, fj = full[:, 0], full[:, 1]
    par = j[fb, fj] % 2
    held = torch.stack([V['tail_k'][fb, :, par].reshape(-1, Hkv, P, dh), V['tail_v'][fb, :, par].reshape(-1, Hkv, P, dh)])
    page = torch.where(fresh[fb, fj][None, :, None, :, None], new[:, src[fb, fj]].transpose(2, 3), held).float()
    top = page.abs().amax((-1, -2), keepdim=True)  # (2, pages, Hkv, 1, 1)
    tiny, odd = top < 2.0 ** -100, ~top.isfinite()
    lim = torch.full_like(top, 448.0)
    code = (page * (lim / torch.where(tiny | odd, lim, top))).masked_fill(tiny | odd, 0).to(torch.float8_e4m3fn)
    scale = (top / lim).masked_fill(tiny, 1.0).masked_fill(odd, math.nan)[..., 0, 0]
    phys = s['table'][fb, j[fb, fj]].long()
    u8 = s['pool'][..., :2 * P * dh]
    kv, vv = k_view(u8[..., :P * dh], P, dh), v_view(u8[..., P * dh:], P, dh)
    kv[phys] = code[0].view(torch.uint8).reshape(-1, *kv.shape[1:])
    vv[phys] = code[1].view(torch.uint8).reshape(-1, *vv.shape[1:])
    V['scale'][phys] = scale.permute(1, 2, 0)
    # the last two pages stay in 16 bits
    keep = (t // P >= (end[b] - 1) // P - 1).nonzero()[:, 0]
    kb, kt = b[keep], t[keep]
    i, par = kt % P, kt // P % 2
    V['tail_k'][kb, :, par, i // 16, i // 8 % 2, i % 8] = new[0, keep].reshape(-1, Hkv, *V['tail_k'].shape[-3:])
    V['tail_v'][kb, :, par, i // 16, i // 8 % 2, i // 2 % 4, i % 2] = new[1, keep].reshape(-1, Hkv, *V['tail_v'].shape[-4:])
    return dict(V, q=q)


def gathered(s, ft):
    """Keys and values (B, Hkv, tokens, dh) of every position that the cache holds, in type ft, and the lengths."""
    P, dh, B = s['page'], s['dh'], s['pos'].shape[0]
    V = views(s)
    end = s['pos'].long() + (s['start'][1:] - s['start'][:-1]).long()
    nf = end // P
    W = s['table'].shape[1]
    tab = s['table'].long()
    bi = torch.arange(B, device=tab.device)
    past = torch.arange((W + 1) * P, device=tab.device) >= end[:, None]
    got = []
    for kv, name in enumerate('kv'):
        x = V[name].reshape(-1, s['Hkv'], P, dh)[tab].to(ft) * V['scale'][tab][..., kv, None, None].to(ft)
        x = torch.cat([x, torch.zeros_like(x[:, :1])], 1)
        x[bi, nf] = V['tail_' + name][bi, :, nf % 2].reshape(B, -1, P, dh).to(ft)
        got.append(x.transpose(1, 2).reshape(B, -1, (W + 1) * P, dh).masked_fill_(past[:, None, :, None], 0))
    return got[0], got[1], end


def attended(s, ft):
    K, Vv, end = gathered(s, ft)
    B, n, Hq, Hkv, dh = K.shape[0], s['n'], s['Hq'], s['Hkv'], s['dh']
    r, b, t = rows_of(s)
    i = r - s['start'][b]
    q = torch.zeros(B, n, Hq, dh, device=K.device, dtype=ft)
    q[b, i] = s['q'].to(ft)
    q = q.view(B, n, Hkv, Hq // Hkv, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, dh)
    sc = (q @ K.transpose(2, 3)).view(B, Hkv, Hq // Hkv, n, -1) * (1.0 / math.sqrt(dh))
    at = torch.arange(K.shape[2], device=K.device)
    tq = (s['pos'].long()[:, None] + torch.arange(n, device=K.device))[:, :, None]
    seen = (at <= tq) & (at < end[:, None, None])
    if s['window']:
        seen = seen & (at > tq - s['window'])
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    w = torch.exp(sc - torch.where(top == -math.inf, 0, top))
    tot = w.sum(-1, keepdim=True)
    o = (w.view(B, Hkv, -1, w.shape[-1]) @ Vv).view(B, Hkv, Hq // Hkv, n, dh) / torch.where(tot == 0, 1, tot)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, dh)[b, i]


def run_attn(s):
    if own:
        from treeattn_b200.paged import PagedKV, paged_attn
        cache = PagedKV(s['pool'], s['tail'], s['table'], s['page'], s['dh'])
        return paged_attn(cache, s['q'], s['start'], s['pos'], s['n'], window=s['window'], ws=s['ws'])
    return attended(s, torch.float32).to(s['q'].dtype)


def run_verify(s):
    if own:
        from treeattn_b200.paged import verify_drafts
        tokens, accepted = verify_drafts(s['p'], s['q'], s['drafts'], s['u'], s['n'])
        return dict(tokens=tokens, accepted=accepted)
    p, q, d, u, n = s['p'].float(), s['q'].float(), s['drafts'], s['u'], s['n'].long()
    B, G, V = q.shape
    ok = u[:, :G] * q.gather(2, d[..., None])[..., 0] < p[:, :G].gather(2, d[..., None])[..., 0]
    ok &= torch.arange(G, device=p.device) < n[:, None]
    a = ok.long().cumprod(1).sum(1)
    bi = torch.arange(B, device=p.device)
    pr = p[bi, a]
    qr = torch.where((a < n)[:, None], q[bi, a.clamp(max=G - 1)], 0.0)
    # fixed point in steps of 2^-38, so that the sums do not depend on their order
    left = torch.where(pr > qr, pr - qr, 0.0).clamp(max=1.0)
    left = (left * 2.0 ** 38).long()
    whole = (torch.where(pr > 0, pr, 0.0).clamp(max=1.0) * 2.0 ** 38).long()
    left = torch.where(left.sum(1, keepdim=True) > 0, left, whole)
    cum = left.cumsum(1)
    ui = (u[:, G] * 2.0 ** 24).long().clamp(0, (1 << 24) - 1)
    tot = cum[:, -1]
    mark = (tot >> 24) * ui + (((tot & 0xffffff) * ui) >> 24)
    tok = (cum <= mark[:, None]).sum(1).clamp(max=V - 1)
    i = torch.arange(G + 1, device=p.device)
    dd = torch.cat([d, d.new_zeros(B, 1)], 1)
    tokens = torch.where(i < a[:, None], dd, torch.where(i == a[:, None], tok[:, None], -1))
    return dict(tokens=tokens, accepted=a.int())


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case['op'] == 'verify':
        return None
    s = prepare(case, seed)
    if case['op'] == 'attn':
        return exact_attn(s)
    return exact_append(s)


def exact_attn(s):
    """Token by token positions, one sequence at a time, in 64 bits."""
    P, dh, Hkv, grp = s['page'], s['dh'], s['Hkv'], s['Hq'] // s['Hkv']
    V = views(s)
    start, pos = s['start'].tolist(), s['pos'].tolist()
    out = torch.zeros(s['q'].shape, device='cuda', dtype=torch.float64)
    for b in range(len(pos)):
        n = start[b + 1] - start[b]
        L = pos[b] + n
        if not n:
            continue
        pages = s['table'][b, :L // P].long()
        K, U = [(V[x][pages].reshape(-1, Hkv, P, dh).double() * V['scale'][pages][:, :, i, None, None].double())
                .transpose(0, 1).reshape(Hkv, -1, dh) for i, x in enumerate('kv')]
        rest = L % P
        tk, tv = [V[x][b, :, (L // P) % 2].reshape(Hkv, P, dh)[:, :rest].double() for x in ('tail_k', 'tail_v')]
        K, U = torch.cat([K, tk], 1), torch.cat([U, tv], 1)
        q = s['q'][start[b]:start[b + 1]].double().view(n, Hkv, grp, dh).permute(1, 2, 0, 3)
        sc = torch.einsum('hgnd,htd->hgnt', q, K) / math.sqrt(dh)
        at = torch.arange(L, device='cuda')
        tq = pos[b] + torch.arange(n, device='cuda')[:, None]
        hide = at > tq
        if s['window']:
            hide |= at <= tq - s['window']
        w = sc.masked_fill(hide, -math.inf).softmax(-1)
        out[start[b]:start[b + 1]] = torch.einsum('hgnt,htd->nhgd', w, U).reshape(n, -1, dh)
    return out


def exact_append(s):
    """The 16-bit pages unrounded but as the type holds them where they are quantised; codes and scales of full pages."""
    P, dh, Hkv, dt = s['page'], s['dh'], s['Hkv'], s['q'].dtype
    start, pos = s['start'].tolist(), s['pos'].tolist()
    V = {x: y.double().contiguous() for x, y in views(s).items()}  # copies, filled in below
    q = torch.zeros(s['q'].shape, device='cuda', dtype=torch.float64)
    h = s['rot'] // 2
    if h:
        f = 10000.0 ** (-torch.arange(h, device='cuda', dtype=torch.float64) / h)

    def turned(x, t):
        x = x.double()
        if not h:
            return x
        z = torch.complex(x[..., :h], x[..., h:2 * h]) * torch.complex((t[:, None] * f).cos(), (t[:, None] * f).sin())[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * h:]], -1)

    for b in range(len(pos)):
        n = start[b + 1] - start[b]
        if not n:
            continue
        t = torch.arange(pos[b], pos[b] + n, device='cuda')
        rows = slice(start[b], start[b + 1])
        q[rows] = turned(s['q'][rows], t)
        L, f0 = pos[b] + n, pos[b] // P
        last = (L - 1) // P
        for i, (x, new) in enumerate((('k', turned(s['k'][rows], t)), ('v', s['v'][rows].double()))):
            name = 'tail_' + x
            flat = V[name][b].reshape(Hkv, 2, P, dh).clone()  # by token
            all_ = torch.cat([flat[:, f0 % 2, :pos[b] % P], new.transpose(0, 1)], 1)  # from the open page's start
            full = L // P - f0
            if full:
                held = all_[:, :full * P].to(dt).double().view(Hkv, full, P, dh).transpose(0, 1)
                top = held.abs().amax((-1, -2))
                pages = s['table'][b, f0:f0 + full].long()
                V[x][pages] = (held * (448 / top)[..., None, None]).to(torch.float8_e4m3fn).double().reshape(V[x][pages].shape)
                V['scale'][pages, :, i] = top / 448
            for j in range(max(f0, last - 1), last + 1):
                a, e = max(j * P, pos[b]), min((j + 1) * P, L)
                flat[:, j % 2, a - j * P:e - j * P] = new[a - pos[b]:e - pos[b]].transpose(0, 1)
            V[name][b] = flat.reshape(V[name][b].shape)
    return dict(V, q=q)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    B = c['B']
    size = 4 if c['dtype'] == 'f32' else 2
    share = 0.75 if c['ragged'] else 1.0  # of the largest length, on average
    if c['op'] == 'verify':
        # the target's row that the token comes from, and the draft's unless all drafts stood (about a quarter)
        return dict(bytes=1.75 * B * c['V'] * size + B * c['G'] * 24, flops=4.0 * B * c['V'])
    Hq, Hkv, dh, P, n = c['Hq'], c['Hkv'], c['dh'], c['page'], c['n']
    N = max(1.0, B * n * (share if n > 1 else 1.0))
    if c['op'] == 'append':
        kept = min(N, B * 1.5 * P)
        return dict(bytes=N * (2 * Hq + 2 * Hkv) * dh * 2 + N * c['rot'] * 4 + N * Hkv * 2 * dh + kept * Hkv * dh * 4,
                    flops=N * (3.0 * c['rot'] * (Hq + Hkv) + 4.0 * Hkv * dh))
    span = c['ctx'] * share + n * share
    read = min(span, c['window'] + n) if c['window'] else span
    seen = min(span - n * share / 2, c['window']) if c['window'] else span - n * share / 2
    return dict(bytes=B * Hkv * max(1.0, read) * (2 * dh + 16.0 / P) + 2 * N * Hq * dh * 2,
                flops=4.0 * N * Hq * dh * max(1.0, seen))
