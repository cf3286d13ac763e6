"""Low-rank adapters on the GPU against the formulas in 64 bits and against differences; sets of adapters in training and serving."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

LENGTHS = [[1], [0, 1, 0], [5, 16, 17, 3], [64, 1, 65, 0, 130], [200], [1] * 33, [63, 64, 15]]


def _inputs(lengths, K, N, r, dtype, na=3, before=0, after=0, seed=0, scale=True):
    g = torch.Generator(device='cuda').manual_seed(seed)
    B, n = len(lengths), before + sum(lengths) + after
    rand = lambda *s, by=1.0: (torch.randn(*s, device='cuda', generator=g) * by).to(dtype)
    start = [before]
    for l in lengths:
        start.append(start[-1] + l)
    which = torch.randint(-1, na, (B,), device='cuda', generator=g).int()
    which[-1] = na - 1
    return dict(y=rand(n, N), x=rand(n, K), a=rand(na, r, K, by=K ** -0.5), b=rand(na, N, r, by=r ** -0.5),
                start=torch.tensor(start, device='cuda', dtype=torch.int32), which=which,
                max_new=max(lengths), scale=(torch.rand(na, device='cuda', generator=g) + 0.5) if scale else None)


def _formula(y, x, a, b, start, which, max_new, scale, dy=None):
    """Outputs in 64 bits, each with the sum of its terms' magnitudes."""
    y, x, a, b = [t.double() for t in (y, x, a, b)]
    out, size = y.clone(), torch.zeros_like(y)
    res = dict(out=(out, size))
    if dy is not None:
        dy = dy.double()
        dx, dxs, da, das, db, dbs = [torch.zeros_like(t) for t in (x, x, a, a, b, b)]
        res.update(dx=(dx, dxs), da=(da, das), db=(db, dbs))
    for i, w in enumerate(which.tolist()):
        if w < 0:
            continue
        r = slice(int(start[i]), int(start[i + 1]))
        s = 1.0 if scale is None else float(scale[w])
        t, ta = s * x[r] @ a[w].T, s * x[r].abs() @ a[w].abs().T
        out[r] += t @ b[w].T
        size[r] = ta @ b[w].abs().T
        if dy is not None:
            u, ua = s * dy[r] @ b[w], s * dy[r].abs() @ b[w].abs()
            dx[r], dxs[r] = u @ a[w], ua @ a[w].abs()
            da[w] += u.T @ x[r]
            das[w] += ua.T @ x[r].abs()
            db[w] += dy[r].T @ t
            dbs[w] += dy[r].abs().T @ ta
    return res


def _near(got, want, terms, what):
    """Half a step of the output's type; t as two 16-bit numbers (2^-16 of it at most); fp32 sums, each of whose `terms` additions is off by a
    step of 2^-23 of the magnitudes' sum."""
    w, size = want
    tol = w.abs() * torch.finfo(got.dtype).eps / 2 * 1.01 + (2.0 ** -16 + terms * 2.0 ** -23) * size + 2.0 ** -24 * (got.dtype is torch.float16) + 2.0 ** -126
    bad = ~((got.double() - w).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4], w[bad][:4], tol[bad][:4])


def _forward(s, **kw):
    from treeattn_b200.adapters import adapter_add
    out = adapter_add(**s, **kw)
    K, r = s['x'].shape[1], s['a'].shape[1]
    _near(out, _formula(**s)['out'], K + r, 'out')
    return out


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('K,N,r', [(8, 8, 8), (64, 72, 16), (72, 64, 24), (768, 2304, 16), (1000, 136, 32), (136, 1000, 48), (512, 384, 64),
                                   (200, 264, 96), (2048, 256, 128)])
@pytest.mark.parametrize('lengths', LENGTHS, ids=str)
def test_forward(lengths, K, N, r, dtype):
    _forward(_inputs(lengths, K, N, r, dtype, seed=K + r))


@pytest.mark.parametrize('K,N,r', [(8, 8, 8), (64, 72, 16), (768, 2304, 16), (1000, 136, 32), (136, 1000, 48), (512, 384, 64), (200, 264, 128)])
@pytest.mark.parametrize('lengths', LENGTHS + [[700, 3, 1500]], ids=str)
def test_gradients(lengths, K, N, r):
    from treeattn_b200.adapters import adapter_add
    s = _inputs(lengths, K, N, r, torch.bfloat16, before=3, after=5, seed=K + r)
    leaves = {k: s[k].clone().requires_grad_() for k in ('y', 'x', 'a', 'b')}
    out = adapter_add(**dict(s, **leaves))
    dy = torch.randn(out.shape, device='cuda').to(out.dtype)
    got = dict(zip(('y', 'x', 'a', 'b'), torch.autograd.grad(out, list(leaves.values()), dy, retain_graph=True)))
    want = _formula(**s, dy=dy)
    n = sum(lengths)
    _near(out.detach(), want['out'], K + r, 'out')
    assert torch.equal(got['y'], dy)
    _near(got['x'], want['dx'], N + r, 'dx')
    _near(got['a'], want['da'], N + n, 'da')
    _near(got['b'], want['db'], K + n, 'db')
    again = torch.autograd.grad(out, list(leaves.values()), dy)
    for g, h in zip(got.values(), again):
        assert torch.equal(g, h)  # one order of additions


@pytest.mark.parametrize('asked', ['x', 'a', 'b', 'y', 'ab', 'xb', 'ya'])
def test_some_gradients(asked):
    """Each gradient by itself is what it is among the others."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([30, 0, 90], 128, 192, 16, torch.bfloat16, seed=5)
    dy = torch.randn(s['y'].shape, device='cuda').to(torch.bfloat16)
    full = {k: s[k].clone().requires_grad_() for k in 'yxab'}
    part = {k: s[k].clone().requires_grad_(k in asked) for k in 'yxab'}
    want = dict(zip('yxab', torch.autograd.grad(adapter_add(**dict(s, **full)), list(full.values()), dy)))
    for k, g in zip(asked, torch.autograd.grad(adapter_add(**dict(s, **part)), [part[k] for k in asked], dy)):
        assert torch.equal(g, want[k])


def test_gradients_against_differences():
    """out is linear in each factor: differences of any length are its gradient, up to the outputs' and gradients' roundings. The
    factors and steps are numbers that bf16 holds with their sums."""
    from treeattn_b200.adapters import adapter_add
    g = torch.Generator(device='cuda').manual_seed(2)
    s = _inputs([7, 40, 20], 64, 72, 16, torch.bfloat16, seed=6, scale=False)
    for k in ('x', 'a', 'b'):
        s[k] = (torch.randint(-32, 33, s[k].shape, device='cuda', generator=g) / 64).to(torch.bfloat16)
    s['y'] = torch.zeros_like(s['y'])
    dy = (torch.randint(-8, 9, s['y'].shape, device='cuda', generator=g) / 8).to(torch.bfloat16)
    leaves = {k: s[k].clone().requires_grad_() for k in 'yxab'}
    grads = dict(zip('yxab', torch.autograd.grad(adapter_add(**dict(s, **leaves)), list(leaves.values()), dy)))
    for k in 'xab':
        step = (torch.randint(-1, 2, s[k].shape, device='cuda', generator=g) / 2).to(torch.bfloat16)
        up, down = [adapter_add(**dict(s, **{k: s[k] + sign * step})).double() for sign in (1, -1)]
        diff = float((dy.double() * (up - down)).sum() / 2)
        slope = float((grads[k].double() * step.double()).sum())
        tol = float((dy.double().abs() * (up.abs() + down.abs())).sum() / 2 + (grads[k].double() * step.double()).abs().sum()) * (2.0 ** -8 * 0.51 * 2)
        assert abs(diff - slope) <= tol
    wrong = float((grads['x'].double().abs()).sum())
    assert wrong > 0


def test_places():
    """Rows of no sequence, rows with strides, parts of a wider row, in place, a given output."""
    from treeattn_b200.adapters import adapter_add
    for dtype in (torch.bfloat16, torch.float16):
        s = _inputs([9, 0, 70], 128, 192, 16, dtype, before=4, after=11, seed=3)
        want = _forward(s)
        assert torch.equal(want[:4], s['y'][:4]) and torch.equal(want[-11:], s['y'][-11:])
        wide = torch.zeros(94, 704, device='cuda', dtype=dtype)
        wide[:, 8:136], wide[:, 144:336] = s['x'], s['y']
        t = dict(s, x=wide[:, 8:136], y=wide[:, 144:336])
        assert torch.equal(adapter_add(**t), want)
        keep = wide.clone()
        out = adapter_add(**t, out=wide[:, 400:592])
        assert torch.equal(out, want) and torch.equal(wide[:, :400], keep[:, :400]) and torch.equal(wide[:, 592:], keep[:, 592:])
        out = adapter_add(**t, out=t['y'])
        assert out is t['y'] and torch.equal(out, want)
        keep[:, 144:336] = want
        keep[:, 400:592] = want
        assert torch.equal(wide, keep)
        s['which'][:] = -1
        assert torch.equal(adapter_add(**s), s['y'])
        empty = dict(s, x=s['x'][:0], y=s['y'][:0], start=s['start'] * 0)
        assert adapter_add(**empty).shape == (0, 192)
        if dtype is torch.bfloat16:
            leaves = {k: empty[k].clone().requires_grad_() for k in 'yxab'}
            got = torch.autograd.grad(adapter_add(**dict(empty, **leaves)), list(leaves.values()), s['y'][:0])
            assert got[1].shape == (0, 128) and not got[2].any() and not got[3].any()
        none = dict(s, start=s['start'][:1] * 0, which=s['which'][:0], max_new=0)
        assert torch.equal(adapter_add(**none), s['y'])


def test_max_new_is_only_a_size():
    from treeattn_b200.adapters import adapter_add
    s = _inputs([150, 20, 333], 256, 136, 32, torch.bfloat16, seed=8)
    for new in (0, 1, 16, 17, 100, 5000):
        _forward(dict(s, max_new=new))
    leaves = {k: s[k].clone().requires_grad_() for k in 'yxab'}
    dy = torch.randn(s['y'].shape, device='cuda').to(torch.bfloat16)
    want = _formula(**s, dy=dy)
    for new in (1, 1000):
        got = torch.autograd.grad(adapter_add(**dict(s, **leaves, max_new=new)), list(leaves.values()), dy)
        _near(got[1], want['dx'], 136 + 32, 'dx')
        _near(got[2], want['da'], 136 + 503, 'da')
        _near(got[3], want['db'], 256 + 503, 'db')


def test_what_does_not_concern_a_row():
    """NaN and infinities in other rows, in unused adapters, in rows of no sequence; an adapter outside the set."""
    from treeattn_b200 import _ops
    from treeattn_b200.adapters import adapter_add
    for new in (16, 40):
        s = _inputs([12, 16, 9, 40], 128, 72, 16, torch.bfloat16, na=4, before=2, after=2, seed=4)
        s['which'][:] = torch.tensor([0, 2, -1, 0], device='cuda')
        s['max_new'] = new
        want = adapter_add(**s)
        dy = torch.randn(s['y'].shape, device='cuda').to(torch.bfloat16)
        leaves = {k: s[k].clone().requires_grad_() for k in 'yxab'}
        grads = torch.autograd.grad(adapter_add(**dict(s, **leaves)), list(leaves.values()), dy)
        t = {k: v.clone() if torch.is_tensor(v) else v for k, v in s.items()}
        t['x'][5] = math.nan
        t['x'][:2] = t['x'][-2:] = math.inf
        t['x'][30:39] = math.nan  # the sequence without an adapter
        t['a'][1] = t['b'][3] = math.nan
        got = adapter_add(**t)
        assert got[5].isnan().all()
        ok = torch.arange(len(got), device='cuda') != 5
        assert torch.equal(got[ok], want[ok])
        t['x'][5] = s['x'][5]
        dirty = dy.clone()
        dirty[:2] = dirty[30:39] = math.nan
        leaves = {k: t[k].clone().requires_grad_() for k in 'yxab'}
        g2 = torch.autograd.grad(adapter_add(**dict(t, **leaves)), list(leaves.values()), dirty)
        for g, h in zip(grads[1:], g2[1:]):
            assert torch.equal(g, h)
        assert (g2[2][[1, 3]] == 0).all() and (g2[3][[1, 3]] == 0).all() and (g2[1][30:39] == 0).all()
        assert _ops.device_error()[0] == 0
        for bad in (4, -2, 2 ** 30):
            s['which'][1] = bad
            got = adapter_add(**s)
            rows = slice(14, 30)
            assert got[rows].isnan().all() and torch.equal(got[:14], want[:14]) and torch.equal(got[30:], want[30:])
            assert _ops.device_error() == (3, 20, 1, bad)


def test_values_at_the_ends():
    """f16: t beyond the type's range with a small B, and t so small that its low part would vanish; bf16: infinities as the formula has them."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([20], 512, 64, 16, torch.float16, na=1, seed=1)
    for up in (2.0 ** 7, 2.0 ** -9):
        t = dict(s, a=s['a'] * 8 * up, b=s['b'] * (2.0 ** -12 / up), y=s['y'] * 0, x=s['x'] * 64)
        assert (up < 1) or float((t['x'].double() @ t['a'][0].double().T).abs().max()) > 2 ** 16
        _forward(t)
    s = _inputs([20], 64, 64, 16, torch.bfloat16, na=1, seed=1)
    s['x'][3, 7] = math.inf
    out = adapter_add(**s)
    want = _formula(**s)['out'][0]
    assert not want[3].isfinite().any() and not out[3].isfinite().any()
    assert out[:3].isfinite().all() and out[4:].isfinite().all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rank', [8, 24, 56, 72, 128])
@pytest.mark.parametrize('rows', [7, 40])
def test_infinite_rows(dtype, rank, rows):
    """Where every term of a sum has one sign an infinity in x gives infinities, not NaN: at ranks that are filled up too."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([rows], 64, 72, rank, dtype, na=1, scale=False, seed=2)
    s = dict(s, a=s['a'].abs() + 0.125, b=s['b'].abs() + 0.125)
    s['which'][:] = 0
    s['x'][3, 7] = math.inf
    out = adapter_add(**s)
    assert (out[3] == math.inf).all()
    assert out[:3].isfinite().all() and out[4:].isfinite().all()


def test_long_offsets():
    """Rows beyond 2^31 elements from the first."""
    from treeattn_b200.adapters import adapter_add
    n, K, N = 270000, 8200, 64
    s = _inputs([40], K, N, 8, torch.bfloat16, na=1)
    x = torch.empty(n, K, device='cuda', dtype=torch.bfloat16)
    x[-40:] = s['x']
    y = torch.zeros(n, N, device='cuda', dtype=torch.bfloat16)
    y[-40:] = s['y']
    start = torch.tensor([n - 40, n], device='cuda', dtype=torch.int32)
    assert (n - 40) * K > 2 ** 31
    leaves = [t.requires_grad_() for t in (y, x, s['a'].clone(), s['b'].clone())]
    out = adapter_add(*leaves, start, s['which'], 40, scale=s['scale'])
    dy = torch.randn(40, N, device='cuda').to(torch.bfloat16)
    got = torch.autograd.grad(out[-40:], leaves, dy)
    want = _formula(**s, dy=dy)
    _near(out[-40:].detach(), want['out'], K + 8, 'out')
    _near(got[1][-40:], want['dx'], N + 8, 'dx')
    _near(got[2], want['da'], N + 40, 'da')
    _near(got[3], want['db'], K + 40, 'db')
    assert (out[:n - 40] == 0).all() and (got[1][:1000] == 0).all()


def test_captured_and_on_another_stream():
    from treeattn_b200.adapters import adapter_add
    s = _inputs([30, 1, 80], 256, 136, 16, torch.bfloat16, seed=7)
    leaves = {k: s[k].clone().requires_grad_() for k in 'yxab'}
    dy = torch.randn(s['y'].shape, device='cuda').to(torch.bfloat16)

    def step():
        out = adapter_add(**dict(s, **leaves))
        return [out, *torch.autograd.grad(out, list(leaves.values()), dy)]

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
    with torch.no_grad():
        leaves['x'].mul_(2)
        s['which'].copy_(torch.tensor([1, 0, -1], device='cuda'))
        s['start'].copy_(torch.tensor([5, 50, 51, 111], device='cuda'))
    graph.replay()
    for got, want in zip(outs, step()):
        assert torch.equal(got, want)


def test_refused():
    from treeattn_b200.adapters import adapter_add
    s = _inputs([5], 64, 64, 8, torch.float16)
    x = s['x'].clone().requires_grad_()
    with pytest.raises(TypeError, match='bfloat16 only'):
        adapter_add(**dict(s, x=x))
    s = _inputs([5], 64, 64, 8, torch.bfloat16)
    x = s['x'].clone().requires_grad_()
    with pytest.raises(ValueError, match='given output'):
        adapter_add(**dict(s, x=x), out=torch.empty_like(s['y']))
    with pytest.raises(ValueError, match='gradient of scale'):
        adapter_add(**dict(s, scale=s['scale'].clone().requires_grad_()))
    with pytest.raises(ValueError, match='CUDA'):
        adapter_add(**s, out=torch.empty(5, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='shape'):
        adapter_add(**s, out=torch.empty(6, 64, dtype=torch.bfloat16, device='cuda'))
    with pytest.raises(ValueError, match='x.s place'):
        adapter_add(**dict(s, y=s['x']), out=s['x'])
    y = torch.zeros(5, 68, device='cuda', dtype=torch.bfloat16)[:, 4:]
    from treeattn_b200._lib import TreeAttnError
    with pytest.raises(TreeAttnError, match='aligned'):
        adapter_add(**dict(s, y=y))


def test_gradients_from_any_place():
    """A gradient that comes in transposed, expanded, or off the 16-byte boundaries is taken as its values."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([40, 9], 64, 72, 8, torch.bfloat16, seed=3)
    leaves = {k: s[k].clone().requires_grad_() for k in 'yxab'}
    base = torch.randn(49, 72, device='cuda').to(torch.bfloat16)
    off = torch.empty(49 * 72 + 1, device='cuda', dtype=torch.bfloat16)[1:].view(49, 72).copy_(base)
    turned = base.t().contiguous().t()
    wide = torch.zeros(49, 75, device='cuda', dtype=torch.bfloat16)[:, 1:73].copy_(base)
    out = adapter_add(**dict(s, **leaves))
    want = torch.autograd.grad(out, list(leaves.values()), base, retain_graph=True)
    for dy in (off, turned, wide):
        for g, w in zip(torch.autograd.grad(out, list(leaves.values()), dy, retain_graph=True), want):
            assert torch.equal(g, w)
    one = base[:1, :1].expand(49, 72)
    got = torch.autograd.grad(out, list(leaves.values()), one, retain_graph=True)
    for g, w in zip(got, torch.autograd.grad(out, list(leaves.values()), one.contiguous())):
        assert torch.equal(g, w)


def test_cast_sets():
    """A set that is cast whole keeps working: its scale is taken in float32 all the same."""
    model, cfg = _gpt(local=64)
    model.requires_grad_(False)
    s = _trained()
    idx = torch.randint(0, 96, (2, 64), device='cuda')
    handle = s.attach(model)
    s.use([0, 1])
    want = model(idx)[0]
    s.to(torch.bfloat16)
    assert s.scale.dtype is torch.bfloat16 and torch.equal(model(idx)[0], want)  # (alpha / rank is 2, which bf16 holds)
    which = torch.tensor([0, 1], device='cuda', dtype=torch.int32)
    s.use(which)
    which[:] = 2  # the caller's tensor is the caller's
    assert torch.equal(model(idx)[0], want)
    handle.remove()


def test_in_place_in_autograd():
    """In place on a projection's output: the gradients are those of the sum."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([30, 33], 64, 72, 8, torch.bfloat16, seed=9)
    w = (torch.randn(72, 64, device='cuda') / 8).to(torch.bfloat16)
    res = []
    for into in (False, True):
        leaves = [t.clone().requires_grad_() for t in (w, s['x'], s['a'], s['b'])]
        y = leaves[1] @ leaves[0].t()
        out = adapter_add(y, *leaves[1:], s['start'], s['which'], 33, scale=s['scale'], out=y if into else None)
        res.append([out.detach(), *torch.autograd.grad((out.float() ** 2).sum(), leaves)])
    for a, b in zip(*res):
        assert torch.equal(a, b)


def _gpt(dtype=torch.bfloat16, **kw):
    from treeattn_b200.config import Config
    from treeattn_b200.model import GPT
    torch.manual_seed(0)
    cfg = Config(**dict(dict(attn='seg', vocab_size=96, seq_len=64, n_layer=2, n_head=2, n_embd=64, neighbors=False, chunk=64), **kw))
    return GPT(cfg).to('cuda', dtype), cfg


def _trained(n_adapters=3, rank=8, **kw):
    from treeattn_b200.adapters import AdapterSet
    torch.manual_seed(1)
    s = AdapterSet(n_adapters, 2, 64, rank=rank, alpha=2 * rank, **kw)
    with torch.no_grad():
        for b in s.b:
            b.copy_(torch.randn_like(b) * 0.05)
    return s


def _step(model, idx, tgt, s):
    logits, loss, _ = model(idx, tgt)
    loss.backward()
    grads = [p.grad.clone() for p in s.parameters()]
    s.zero_grad()
    return logits.detach(), grads


def _hooked(model, s, hook):
    return [block.get_submodule(s.MODULES[name]).register_forward_hook(hook(*s.factors(i, name)))
            for i, block in enumerate(model.blocks) for name in s.projections]


def test_captured_set():
    """A captured pass keeps the adapters and row offsets that it was captured with, and what it works with stays in place, whatever
    the set is used for afterwards; offsets first needed in a capture are none that a later call may find unwritten."""
    model, cfg = _gpt()
    model.requires_grad_(False)
    s = _trained()
    s.attach(model)
    x = torch.randn(4, 64, 64, device='cuda').to(torch.bfloat16)

    def blocks(x):
        for block in model.blocks:
            x = block(x)
        return x

    with torch.no_grad():
        s.use([0, 1, -1, 2])
        want = blocks(x).clone()
        s.use([1, 1])
        two = blocks(x[:2]).clone()
        s._start.clear()
        for warm in (False, True):  # the offsets of 2 rows of 64 are first needed in the capture, then kept from before
            s.use([1, 1])
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = blocks(x[:2])
            assert torch.equal(blocks(x[:2]), two)  # before any replay
            s.use([0, 1, -1, 2])
            for n in range(1, 20):  # other shapes take the kept ones' places
                s._starts(n, n)
            held = [torch.full((m,), 7, device='cuda', dtype=torch.int32) for m in (1, 2, 3, 4, 5) for _ in range(64)]
            assert torch.equal(blocks(x), want)
            graph.replay()
            assert torch.equal(captured, two)
            assert all((h == 7).all() for h in held)


def test_outputs_that_overlap_are_refused():
    from treeattn_b200.adapters import adapter_add
    s = _inputs([5], 64, 64, 8, torch.bfloat16)
    wide = torch.zeros(5 * 64, device='cuda', dtype=torch.bfloat16)
    for strides in ((0, 1), (32, 1)):
        out = wide.as_strided((5, 64), strides)
        with pytest.raises(ValueError, match='overlap'):
            adapter_add(**s, out=out)
        with pytest.raises(ValueError, match='overlap'):
            adapter_add(**dict(s, y=out), out=out)
        with pytest.raises(ValueError, match='overlap'):
            adapter_add(**dict(s, y=out, x=s['x'].clone().requires_grad_()), out=out)
        _near(adapter_add(**dict(s, y=out)), _formula(**dict(s, y=out))['out'], 72, 'expanded y')  # as an input it may
    one = _inputs([1], 64, 64, 8, torch.bfloat16)
    out = wide.as_strided((1, 64), (0, 1))
    _near(adapter_add(**one, out=out), _formula(**one)['out'], 72, 'one row')


@pytest.mark.parametrize('attn', ['seg', 'dyn', 'block'])
def test_set_on_every_model(attn):
    """The set's hooks are adapter_add on each projection's rows with that projection's factors; the frozen model's weights get no
    gradient, an adapter that no sequence takes none either; None and remove() take the adapters off."""
    from treeattn_b200.adapters import adapter_add
    model, cfg = _gpt(attn=attn)
    model.requires_grad_(False)
    s = _trained()
    idx, tgt = torch.randint(0, 96, (2, 4, 64), device='cuda')
    plain = model(idx)[0]
    which = torch.tensor([2, -1, 0, 2], device='cuda', dtype=torch.int32)
    handle = s.attach(model)
    s.use(which.tolist())
    logits, grads = _step(model, idx, tgt, s)
    assert not torch.equal(logits, plain) and all(g.any() for g in grads) and not any(g[1].any() for g in grads)
    s.use(None)
    assert torch.equal(model(idx)[0], plain)
    s.use([0])
    with pytest.raises(ValueError, match='1 sequences'):
        model(idx)
    handle.remove()
    assert torch.equal(model(idx)[0], plain)
    start = torch.tensor([0, 64, 128, 192, 256], device='cuda', dtype=torch.int32)
    hooks = _hooked(model, s, lambda a, b: lambda m, args, y: adapter_add(
        y.view(256, -1), args[0].reshape(256, -1), a, b, start, which, 64, scale=s.scale).view(y.shape))
    want, wg = _step(model, idx, tgt, s)
    for h in hooks:
        h.remove()
    assert torch.equal(logits, want)
    for g, w in zip(grads, wg):  # the attention's backward pass adds in no fixed order, so that bf16 numbers may fall on the next step
        assert (g.float() - w.float()).norm() <= 2.0 ** -7 * w.float().norm()
    assert all(p.grad is None for p in model.parameters())


def test_set_in_training():
    """A model whose attention window holds every position (its output is then continuous: no keys are chosen): logits and gradients are
    those with the adapters' products added by torch's own operations."""
    model, cfg = _gpt(local=64)
    model.requires_grad_(False)
    s = _trained()
    idx, tgt = torch.randint(0, 96, (2, 4, 64), device='cuda')
    which = [2, -1, 0, 2]
    handle = s.attach(model)
    s.use(which)
    logits, grads = _step(model, idx, tgt, s)
    handle.remove()

    def hook(a, b):
        def add(module, args, y):
            rows = []
            for i, w in enumerate(which):
                t = args[0][i].float() @ a[w].float().t() * s.scale[w] if w >= 0 else None
                rows.append(y[i] if t is None else (y[i].float() + t @ b[w].float().t()).to(y.dtype))
            return torch.stack(rows)
        return add

    hooks = _hooked(model, s, hook)
    want, wg = _step(model, idx, tgt, s)
    for h in hooks:
        h.remove()
    # the same operations but for t's last bits, through two blocks of bf16: a few of its steps
    assert (logits.float() - want.float()).abs().max() <= 0.05 * want.float().abs().max()
    for g, w in zip(grads, wg):
        assert (g.float() - w.float()).norm() <= 0.1 * w.float().norm()


def test_set_in_serving():
    """PagedDecoder: each sequence's logits are those of a decoder whose weights have its adapter added, in prompts and token by token,
    and a fork takes its source's adapter."""
    from treeattn_b200.engine import weights_from_ours
    from treeattn_b200.speculative import PagedDecoder
    model, cfg = _gpt(torch.float32)
    W = weights_from_ours(model.state_dict(), cfg)
    s = _trained()
    dec = PagedDecoder(W, 2, 2, 64, batch=3, page=16, adapters=s)
    merged = []
    for w in (0, 1, 2):
        layers = []
        for i, L in enumerate(W['layers']):
            L = dict(L)
            for name in s.projections:
                a, b = s.factors(i, name)
                L[name] = L[name].double() + float(s.scale[w]) * b[w].double() @ a[w].double()
            layers.append(L)
        merged.append(PagedDecoder(dict(W, layers=layers), 2, 2, 64, batch=3, page=16))
    base = PagedDecoder(W, 2, 2, 64, batch=3, page=16)
    tok = torch.randint(0, 96, (3, 20), device='cuda')
    assert torch.equal(dec.forward(tok), base.forward(tok))  # no adapters yet
    dec.reset()
    base.reset()
    dec.set_adapter(0, 2)
    dec.set_adapter(2, 0)
    seen = {0: merged[2], 1: base, 2: merged[0]}
    for chunk in (tok, *torch.randint(0, 96, (3, 3, 1), device='cuda')):
        got = dec.forward(chunk)
        refs = {b: d.forward(chunk) for b, d in seen.items()}
        for b, ref in refs.items():
            # the product added in fp32 to a rounded row, against weights rounded after their sum: a few steps of bf16 through two blocks
            assert (got[b].float() - ref[b].float()).abs().max() <= 0.05 * ref[b].float().abs().max()
    dec.fork([0], [1])
    assert dec.which.tolist() == [2, 2, 0]
    new = torch.randint(0, 96, (1, 1), device='cuda').expand(3, 1)
    got = dec.forward(new)
    assert torch.equal(got[0], got[1])
    with pytest.raises(ValueError, match='adapter'):
        dec.set_adapter(0, 3)
    with pytest.raises(TypeError, match='adapters for'):
        PagedDecoder(W, 2, 2, 64, adapters=s, dtype=torch.float16)
    with pytest.raises(ValueError, match='adapters of'):
        PagedDecoder(W, 2, 4, 128, adapters=s)


def _one_signed(lengths, dtype, exact, rank=16):
    """Positive factors and rows; exact: t and u are numbers that the type holds, so that nothing is left for their low parts."""
    s = _inputs(lengths, 64, 72, rank, dtype, na=1, scale=False, seed=2)
    for k in 'xab':
        s[k] = torch.full_like(s[k], 0.25) if exact else s[k].abs() + 0.125
    s['which'][:] = 0
    return s


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('rows', [7, 40])
@pytest.mark.parametrize('exact', [False, True])
@pytest.mark.parametrize('sign', [1, -1])
def test_infinite_factors(dtype, rows, exact, sign):
    """An infinity in A or B gives the formula's infinities, whatever t's low part is: 0, or of the other sign than its high part."""
    from treeattn_b200.adapters import adapter_add
    s = _one_signed([rows], dtype, exact)
    b = s['b'].clone()
    b[0, 5, 3] = sign * math.inf
    out = adapter_add(**dict(s, b=b))
    assert (out[:, 5] == sign * math.inf).all()
    rest = [i for i in range(72) if i != 5]
    assert out[:, rest].isfinite().all()
    a = s['a'].clone()
    a[0, 3, 7] = sign * math.inf
    assert (adapter_add(**dict(s, a=a)) == sign * math.inf).all()
    assert (adapter_add(**dict(s, a=a, b=s['b'] * -1)) == sign * -math.inf).all()


@pytest.mark.parametrize('rows', [7, 40, 300])
@pytest.mark.parametrize('exact', [False, True])
def test_infinities_in_gradients(rows, exact):
    """Infinities in A reach dx, those of x reach dA, those of dy reach dB: as infinities."""
    from treeattn_b200.adapters import adapter_add
    s = _one_signed([rows], torch.bfloat16, exact)
    dy = torch.full_like(s['y'], 0.25) if exact else torch.rand_like(s['y']) + 0.125

    def grads(dy, **kw):
        leaves = {k: dict(s, **kw)[k].clone().requires_grad_() for k in 'yxab'}
        return dict(zip('yxab', torch.autograd.grad(adapter_add(**dict(s, **leaves)), list(leaves.values()), dy)))

    a = s['a'].clone()
    a[0, 3, 7] = -math.inf
    dx = grads(dy, a=a)['x']
    assert (dx[:, 7] == -math.inf).all() and dx[:, [i for i in range(64) if i != 7]].isfinite().all()
    x = s['x'].clone()
    x[2, 9] = math.inf
    da = grads(dy, x=x)['a']
    assert (da[0, :, 9] == math.inf).all() and da[0, :, [i for i in range(64) if i != 9]].isfinite().all()
    d = dy.clone()
    d[4, 11] = -math.inf
    db = grads(d)['b']
    assert (db[0, 11] == -math.inf).all() and db[0, [i for i in range(72) if i != 11]].isfinite().all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_small_parts_of_t(dtype):
    """Elements of t that are far below their row's largest, powers of two and subnormal numbers among them, weigh what they are."""
    s = _inputs([20], 64, 64, 16, dtype, na=1, scale=False, seed=1)
    s['which'][:] = 0
    s['a'] = torch.zeros_like(s['a'])
    s['a'][0, range(16), range(16)] = 1  # t is x's first columns
    for by in (1.0, 3.0):
        s['x'] = (torch.tensor([2.0 ** -i for i in range(16)] + [0.0] * 48, device='cuda') * by).to(dtype).expand(20, 64).contiguous()
        s['y'] = torch.zeros_like(s['y'])
        _forward(s)


def test_outputs_that_autograd_has_saved():
    """A given output that a backward pass still needs is found to have changed, as with torch's own in-place operations."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([5, 40], 64, 72, 8, torch.bfloat16, seed=3)
    for new in (5, 40):
        for into_y in (True, False):
            out = s['y'].clone()
            w = torch.ones_like(out, requires_grad=True)
            loss = (w * out).sum()  # keeps `out` for w's gradient
            before = out._version
            with torch.no_grad():
                adapter_add(**dict(s, y=out if into_y else s['y'], max_new=new), out=out)
            assert out._version > before
            with pytest.raises(RuntimeError, match='inplace'):
                loss.backward()
    with torch.inference_mode():
        out = s['y'].clone()
        assert torch.equal(adapter_add(**s, out=out), adapter_add(**s))


def test_outputs_that_want_gradients_are_refused():
    """Neither a leaf nor a result of autograd is written without a word to its graph."""
    from treeattn_b200.adapters import adapter_add
    for dtype in (torch.bfloat16, torch.float16):
        s = _inputs([5], 64, 64, 8, dtype)
        leaf = torch.zeros_like(s['y']).requires_grad_()
        for out in (leaf, leaf * 1):
            with pytest.raises((ValueError, TypeError), match='given output|bfloat16 only'):
                adapter_add(**s, out=out)
        with torch.no_grad():
            assert torch.equal(adapter_add(**s, out=leaf), adapter_add(**s))


def test_captured_tensors_are_let_go():
    """What captured passes read is kept until release_captured: captures of many shapes do not add up for the set's life."""
    model, cfg = _gpt()
    model.requires_grad_(False)
    s = _trained()
    s.attach(model)
    x = torch.randn(2, 64, 64, device='cuda').to(torch.bfloat16)
    with torch.no_grad():
        s.use([0, 2])
        want = model.blocks[0](x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model.blocks[0](x)
        s.use([1, 1])
        graph.replay()
        assert torch.equal(out, want) and len(s._captured) > 0
        del graph, out
        s.release_captured()
        assert len(s._captured) == 0
        s.use([0, 2])
        assert torch.equal(model.blocks[0](x), want)


@pytest.mark.parametrize('rows', [7, 40])
def test_f16_rows_without_a_power_of_two(rows):
    """Rows of t that cannot be brought near 1: all below 2^-126, which weigh nothing, and rows with an infinity beside numbers above
    f16's range, which stay the infinity that they are."""
    from treeattn_b200.adapters import adapter_add
    s = _inputs([rows], 64, 64, 16, torch.float16, na=1, seed=1)
    s['which'][:] = 0
    s['scale'][:] = 2.0 ** -140
    s['y'] = torch.zeros_like(s['y'])
    assert not _forward(s).any()
    # t is infinite in the first rank and 64 x 60000 in the others, whose part of the sum is finite
    s['scale'][:] = 1
    s['x'], s['a'] = torch.ones_like(s['x']), torch.full_like(s['a'], 60000.0)
    s['a'][0, 0, 3] = math.inf
    s['b'] = torch.full_like(s['b'], -2.0 ** -10)
    s['b'][0, :, 0] = 1.0
    assert (adapter_add(**s) == math.inf).all()
