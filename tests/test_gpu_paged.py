"""The 8-bit paged cache and its operators (paged_append, paged_attn, verify_drafts) against plain 64-bit forms.

Tolerances, from the formats: u(bf16) = 2^-8, u(f16) = 2^-11 half a step relative to the value; e4m3 half a step 2^-4 relative,
2^-10 of the scale below its normal range. Attention: the output's rounding u |o|; the weights' rounding before the product
(f16 for pages in codes, the 16-bit type for the open page), u relative, times sum p |v|; the scores' fp32 sums, an
absolute error d = 2 dh 2^-24 scale sum |q k| in the exponent, which moves p by 2 d relative."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, HF = torch.bfloat16, torch.float16


def _mod():
    from treeattn_b200 import paged
    return paged


def _no_device_error():
    from treeattn_b200 import _ops
    code = _ops.device_error()
    assert code[0] == 0, code


def _device_error():
    from treeattn_b200 import _ops
    torch.cuda.synchronize()
    return _ops.device_error()


def _starts(counts):
    s = torch.zeros(len(counts) + 1, dtype=torch.int32)
    s[1:] = torch.tensor(counts).cumsum(0)
    return s.to(DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Rig:
    """A cache with shuffled pages (those of no sequence, and the table beyond each sequence, hold garbage) and the tokens
    put into it, kept in 64 bits as the 16-bit type has them."""

    def __init__(self, B, Hkv, dh, page, dtype, cap, seed=0):
        P = _mod()
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.B, self.Hkv, self.dh, self.page, self.dt = B, Hkv, dh, page, dtype
        W = -(-cap // page)
        n = B * W + 3
        self.perm = torch.randperm(n, generator=self.g, device=DEV)[:B * W].int().view(B, W)
        self.cache = P.PagedKV.empty(n, Hkv, dh, torch.full((B, W), -7, device=DEV, dtype=torch.int32), page, dtype)
        self.cache.pool.fill_(0x7f)   # e4m3 NaN codes and NaN-like scales wherever nothing is written
        self.cache.tail.fill_(math.nan)
        self.K = torch.zeros(B, Hkv, cap, dh, device=DEV, dtype=dtype)
        self.V = torch.zeros_like(self.K)
        self.len = [0] * B

    def randn(self, *shape, spread=1.0):
        return (torch.randn(*shape, device=DEV, generator=self.g) * spread).to(self.dt)

    def append(self, counts, k=None, v=None, pos=None, **kw):
        N = sum(counts)
        pos = list(self.len) if pos is None else pos
        k = self.randn(N, self.Hkv, self.dh) if k is None else k
        v = self.randn(N, self.Hkv, self.dh) if v is None else v
        r = 0
        for b, c in enumerate(counts):
            full = (pos[b] + c) // self.page
            self.cache.table[b, :full] = self.perm[b, :full]  # only pages that are read or written have an entry
            if kw.get('rotation') is None:
                self.K[b, :, pos[b]:pos[b] + c] = k[r:r + c].transpose(0, 1)
                self.V[b, :, pos[b]:pos[b] + c] = v[r:r + c].transpose(0, 1)
            r += c
            self.len[b] = pos[b] + c
        return _mod().paged_append(self.cache, k, v, _starts(counts), _i32(pos), max(counts + [0]), **kw)

    def check_reads(self):
        """cache.read against the tokens: exact in the open page, within e4m3's half step of the page's scale elsewhere."""
        for b in range(self.B):
            n = self.len[b]
            full = n // self.page * self.page
            for got, want in zip(self.cache.read(b, n), (self.K[b, :, :n], self.V[b, :, :n])):
                want = want.double()
                assert got.shape == want.shape
                assert torch.equal(got[:, full:].double(), want[:, full:])
                w = want[:, :full].reshape(self.Hkv, -1, self.page, self.dh)
                x = got[:, :full].double().reshape(w.shape)
                scale = w.abs().amax((-1, -2), keepdim=True) / 448
                # half a step, and the fp32 rounding of the scale and the product that is rounded (3 x 2^-24)
                assert ((x - w).abs() <= w.abs() * (2.0 ** -4 + 2.0 ** -20) + scale * 2.0 ** -10 * 1.001).all()


SHAPES = [(64, 64, BF), (64, 16, HF), (128, 64, BF), (128, 32, HF), (32, 32, BF), (16, 16, BF), (16, 64, HF), (32, 16, HF)]


@pytest.mark.parametrize('dh,page,dt', SHAPES)
def test_append_reads_back(dh, page, dt):
    """Ragged appends: lengths of zero and one, page ends inside a call, several pages at once, an odd number of heads."""
    r = Rig(5, 3, dh, page, dt, 6 * page, seed=dh + page)
    r.append([page - 1, 0, 1, 3 * page + 5, page])
    r.check_reads()
    r.append([1, 1, page - 2, 2 * page, page + 1])
    r.append([1, 2 * page - 1, 1, 0, 1])
    r.append([1, 1, 1, 1, 1])
    r.check_reads()
    _no_device_error()


@pytest.mark.parametrize('dh,page,dt', SHAPES[:4])
def test_codes_do_not_depend_on_how_tokens_arrive(dh, page, dt):
    """The same tokens in one call, in uneven calls and one by one: the same records, bit for bit."""
    n = 2 * page + 3
    got = []
    for cuts in ([n], [1, page - 1, 2, page + 1], [1] * n, [page + 7, n - page - 7]):
        r = Rig(1, 2, dh, page, dt, n, seed=5)
        k, v = r.randn(n, 2, dh), r.randn(n, 2, dh)
        at = 0
        for c in cuts:
            r.append([c], k[at:at + c], v[at:at + c])
            at += c
        assert r.len == [n]
        got.append(r.cache.pool[r.perm[0, :2].long()][..., :2 * page * dh + 8].clone())
        r.check_reads()
    for x in got[1:]:
        assert torch.equal(x, got[0])
    _no_device_error()


@pytest.mark.parametrize('rot', [8, 32, 64])
@pytest.mark.parametrize('dt', [BF, HF])
def test_rotation(rot, dt):
    """Rotated queries and open-page keys within half a step of the 64-bit rotation (and 4 x 2^-24 of the terms for the fp32
    products and the tables); dims beyond rot are copied; q and k strided as a projection's output has them."""
    P = _mod()
    dh, Hq, Hkv, counts, pos = 64, 6, 2, [3, 0, 17], [40, 5, 0]
    r = Rig(3, Hkv, dh, 64, dt, 128, seed=rot)
    qkv = r.randn(20, (Hq + 2 * Hkv) * dh)
    q = qkv[:, :Hq * dh].view(20, Hq, dh)
    k = qkv[:, Hq * dh:(Hq + Hkv) * dh].view(20, Hkv, dh)
    v = qkv[:, (Hq + Hkv) * dh:].view(20, Hkv, dh)
    cos, sin = P.rotation_table(64, rot)
    out = r.append(counts, k, v, pos, q=q, rotation=(cos, sin))
    t = torch.tensor([40, 41, 42] + list(range(17)), device=DEV, dtype=torch.float64)
    a = t[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    h = rot // 2

    def ref(x):
        x = x.double()
        c, s = a.cos()[:, None], a.sin()[:, None]
        y = torch.cat([x[..., :h] * c - x[..., h:rot] * s, x[..., h:rot] * c + x[..., :h] * s, x[..., rot:]], -1)
        m = torch.cat([x[..., :h].abs() + x[..., h:rot].abs()] * 2 + [torch.zeros_like(x[..., rot:])], -1)
        return y, m

    def near(got, x):
        y, m = ref(x)
        assert ((got.double() - y).abs() <= U[dt] * y.abs() + 4 * 2.0 ** -24 * m + 2.0 ** -25).all()

    near(out, q)
    assert torch.equal(out[..., rot:], q[..., rot:])
    kr = torch.cat([r.cache.read(0, 43)[0][:, 40:].transpose(0, 1), r.cache.read(2, 17)[0].transpose(0, 1)])
    near(kr, k)
    assert torch.equal(r.cache.read(2, 17)[1].transpose(0, 1), v[3:].float())
    _no_device_error()


def test_cut_back_and_append_again():
    """Rejected drafts: a sequence cut back across a page end and continued with other tokens holds what one that never saw
    the drafts holds."""
    page, dh = 16, 64
    for n0, draft in ((14, 5), (16, 1), (31, 16), (33, 15), (47, 17)):
        a, b = (Rig(1, 2, dh, page, BF, 96, seed=3) for _ in range(2))
        k, v = a.randn(96, 2, dh), a.randn(96, 2, dh)
        for r in (a, b):
            r.append([n0], k[:n0], v[:n0])
        a.append([draft], a.randn(draft, 2, dh, spread=9.0), a.randn(draft, 2, dh, spread=9.0))
        keep = max(n0 - 1, ((n0 + draft - 1) // page - 1) * page)  # the last kept token is replaced as well
        for r in (a, b):
            r.append([40], k[40:80], v[40:80], pos=[keep])
        full = (keep + 40) // page
        assert torch.equal(a.cache.pool[a.perm[0, keep // page:full].long()][..., :2 * page * dh + 8],
                           b.cache.pool[b.perm[0, keep // page:full].long()][..., :2 * page * dh + 8])
        a.check_reads()
    _no_device_error()


@pytest.mark.parametrize('page', [16, 32, 64])
def test_every_offset_keeps_the_last_two_pages(page):
    """Calls that begin at every offset of a page and of the 64 positions around it, of lengths around a page, two pages and
    64: full pages read back, and after cutting back the last page but one comes from the 16-bit copy, token for token."""
    B = 128
    for n in (1, page - 1, page, page + 1, 2 * page - 1, 2 * page, 2 * page + 5, 65, 3 * page + 2, 150):
        r = Rig(B, 1, 16, page, BF, 128 + 200, seed=n)
        pos = list(range(B))
        r.append(pos)
        r.append([n] * B)
        r.check_reads()
        r.len = [max(0, (p + n - 1) // page * page - 1) for p in pos]  # all but one token of the page before the last
        r.check_reads()
    _no_device_error()


def test_odd_pages():
    """Pages of zeros, of values below 2^-100, of the type's largest values, with an infinity, with a NaN."""
    page, dh = 16, 32
    r = Rig(6, 1, dh, page, BF, page)
    k = r.randn(6 * page, 1, dh)
    v = r.randn(6 * page, 1, dh)
    k[:page] = 0
    k[page:2 * page] *= 2.0 ** -110
    k[2 * page:3 * page] = 3.3e38
    v[3 * page + 3, 0, 5] = math.inf
    k[4 * page + 7, 0, 1] = math.nan
    r.append([page] * 6, k, v)
    got = [r.cache.read(b, page) for b in range(6)]
    assert (got[0][0] == 0).all() and (got[1][0] == 0).all()
    assert torch.isfinite(got[2][0]).all() and (got[2][0] - 3.3e38).abs().max() < 3.3e38 * 2.0 ** -4
    assert torch.isnan(got[3][1]).all() and torch.isfinite(got[3][0]).all()
    assert torch.isnan(got[4][0]).all() and torch.isfinite(got[4][1]).all()
    assert torch.isfinite(got[5][0]).all()
    _no_device_error()


# ------------------------------------------------------------------------------------------------ attention
def _attend_ref(r, q, counts, pos, scale, window):
    """64-bit attention over what the cache reads back: out, the tolerance's parts, lse."""
    Hq, dh = q.shape[1:]
    grp = Hq // r.Hkv
    outs, tols, lses = [], [], []
    row = 0
    for b, n in enumerate(counts):
        L = pos[b] + n
        K, V = [x.double() for x in r.cache.read(b, L)]
        qb = q[row:row + n].double().view(n, r.Hkv, grp, dh).permute(1, 2, 0, 3)
        s = torch.einsum('hgnd,htd->hgnt', qb, K) * scale
        mag = torch.einsum('hgnd,htd->hgnt', qb.abs(), K.abs()).amax(-1) * scale if L else s.sum(-1)
        at = torch.arange(L, device=DEV)
        tq = pos[b] + torch.arange(n, device=DEV)[:, None]
        hide = at > tq
        if window:
            hide |= at <= tq - window
        s = s.masked_fill(hide, -math.inf)
        p = s.softmax(-1)
        o = torch.einsum('hgnt,htd->nhgd', p, V).reshape(n, Hq, dh)
        # weights' rounding: f16 for codes, the type for the open page
        full = L // r.page * r.page
        u = torch.full((L,), 2.0 ** -11, device=DEV, dtype=torch.float64)
        u[full:] = U[r.dt]
        pv = torch.einsum('hgnt,htd->nhgd', p * u, V.abs()).reshape(n, Hq, dh)
        d = 2 * dh * 2.0 ** -24 * mag
        move = torch.einsum('hgnt,htd->nhgd', p * (2 * d)[..., None], V.abs()).reshape(n, Hq, dh)
        outs.append(o)
        tols.append(U[r.dt] * o.abs() + pv + move + 1e-5 * torch.einsum('hgnt,htd->nhgd', p, V.abs()).reshape(n, Hq, dh)
                    + 2.0 ** -25)
        lses.append((s.logsumexp(-1), 2 * d + 1e-5))
        row += n
    lse = torch.cat([x.permute(2, 0, 1).reshape(-1, Hq) for x, _ in lses])
    ltol = torch.cat([x.permute(2, 0, 1).reshape(-1, Hq) for _, x in lses])
    return torch.cat(outs), torch.cat(tols), lse, ltol


ATTN = [
    # dh, page, dtype, Hq, Hkv, earlier lengths, new rows, window
    (64, 64, BF, 12, 12, [0, 63, 64, 65, 1000, 4096], [1] * 6, 0),
    (64, 64, BF, 12, 12, [0, 63, 64, 65, 1000, 4096], [1, 1, 0, 5, 4, 8], 0),
    (64, 32, HF, 4, 1, [0, 31, 500], [3, 2, 5], 0),
    (128, 64, BF, 16, 16, [3000, 17], [1, 1], 0),
    (128, 32, HF, 16, 4, [700, 0, 33], [5, 1, 64], 0),
    (128, 16, BF, 8, 1, [100, 250], [3, 1], 0),
    (32, 16, BF, 6, 3, [5, 90, 15, 16], [1, 7, 1, 33], 0),
    (16, 16, HF, 2, 2, [0, 200], [40, 1], 0),
    (16, 64, BF, 8, 2, [64, 1], [1, 1], 0),
    (64, 64, BF, 4, 2, [0, 130], [257, 100], 0),
    (128, 64, BF, 4, 4, [0, 61], [150, 70], 0),
    # windows: of one token, inside a page, across pages, longer than the sequence
    (64, 64, BF, 4, 4, [200, 64, 5], [1, 2, 1], 1),
    (64, 32, HF, 4, 2, [300, 64, 5], [9, 1, 3], 7),
    (128, 16, BF, 8, 2, [300, 90], [5, 40], 50),
    (64, 64, BF, 4, 4, [1000, 700], [130, 1], 300),
    (32, 32, BF, 4, 4, [40], [3], 5000),
]


@pytest.mark.parametrize('dh,page,dt,Hq,Hkv,before,new,window', ATTN)
def test_attention(dh, page, dt, Hq, Hkv, before, new, window):
    P = _mod()
    r = Rig(len(new), Hkv, dh, page, dt, max(a + b for a, b in zip(before, new)), seed=dh + page + Hq)
    if any(before):
        r.append(before)
    pos = list(r.len)
    r.append(new)
    N = sum(new)
    qkv = r.randn(N, (Hq + 3) * dh, spread=1.5)
    q = qkv[:, dh:dh + Hq * dh].view(N, Hq, dh)      # strided rows
    hold = torch.full((N, Hq + 1, dh), 7.0, device=DEV, dtype=dt)
    out = hold[:, :Hq]                               # strided output
    lse = torch.empty(N, Hq, device=DEV)
    ws = P.paged_attn_workspace(len(new), Hq, Hkv, dh, max(new))
    P.paged_attn(r.cache, q, _starts(new), _i32(pos), max(new), window=window, out=out, lse=lse, ws=ws)
    want, tol, wl, ltol = _attend_ref(r, q, new, pos, 1 / math.sqrt(dh), window)
    d = (out.double() - want).abs()
    assert (d <= tol).all(), float((d / tol).max())
    assert ((lse.double() - wl).abs() <= ltol).all()
    assert (hold[:, Hq] == 7.0).all()
    # again on the same workspace, and on one of its own: the same bits
    again = P.paged_attn(r.cache, q, _starts(new), _i32(pos), max(new), window=window, ws=ws)
    assert torch.equal(again, out)
    assert torch.equal(P.paged_attn(r.cache, q, _starts(new), _i32(pos), max(new), window=window), out)
    _no_device_error()


@pytest.mark.parametrize('dt', [BF, HF])
def test_attention_spread_scales(dt):
    """Pages whose key and value scales differ by orders of magnitude, large scores, and rows of large and tiny queries: the
    weights' reference follows score and value scale together."""
    P = _mod()
    page, dh = 16, 64
    r = Rig(2, 2, dh, page, dt, 200, seed=1)
    n = [150, 199]
    N = sum(n)
    k, v = r.randn(N, 2, dh), r.randn(N, 2, dh)
    f = torch.exp2(torch.randint(-9, 9, (N // page + 1,), device=DEV, generator=r.g).float()).repeat_interleave(page)[:N]
    v = (v.float() * f[:, None, None]).to(dt)
    k = (k.float() * f.flip(0).clamp(max=8)[:, None, None]).to(dt)
    r.append(n, k, v)
    r.append([1, 1])
    q = r.randn(2, 4, dh)
    q[0, 0] *= 30
    q[1, 2] *= 2.0 ** -12
    q[1, 3] = 0
    got = P.paged_attn(r.cache, q, _starts([1, 1]), _i32(n), 1)
    want, tol, _, _ = _attend_ref(r, q, [1, 1], n, 0.125, 0)
    assert ((got.double() - want).abs() <= tol).all()
    _no_device_error()


def test_attention_bad_page_stays_with_its_sequence():
    """A page that reads back as NaN gives NaN to the rows that see it and to no others; a query before it is not touched."""
    P = _mod()
    page, dh = 16, 64
    r = Rig(2, 1, dh, page, BF, 64)
    k, v = r.randn(64, 1, dh), r.randn(64, 1, dh)
    v[20, 0, 0] = math.inf                              # sequence 0, page 1
    r.append([32, 32], k, v)
    q = r.randn(64, 1, dh)
    out = P.paged_attn(r.cache, q, _starts([32, 32]), _i32([0, 0]), 32)
    assert torch.isfinite(out[:16]).all() and torch.isfinite(out[32:]).all()
    assert torch.isnan(out[16:32]).all()
    _no_device_error()


def test_long_table_and_many_sequences():
    """A pool of more than 2^32 bytes is addressed in 64 bits; more sequences than a grid dimension of warps."""
    P = _mod()
    page, dh, H = 64, 128, 16
    n_pages = 2 ** 32 // (H * (2 * page * dh + 16)) + 40
    table = torch.full((1, 8), 0, device=DEV, dtype=torch.int32)
    cache = P.PagedKV.empty(n_pages, H, dh, table, page, BF)
    table[0, :3] = _i32([n_pages - 1, 0, n_pages - 2])
    g = torch.Generator(device=DEV).manual_seed(0)
    k = torch.randn(200, H, dh, device=DEV, generator=g).to(BF)
    v = torch.randn(200, H, dh, device=DEV, generator=g).to(BF)
    P.paged_append(cache, k, v, _starts([200]), _i32([0]), 200)
    q = torch.randn(200, H, dh, device=DEV, generator=g).to(BF)
    r = Rig.__new__(Rig)
    r.cache, r.Hkv, r.page, r.dt = cache, H, page, BF
    got = P.paged_attn(cache, q, _starts([200]), _i32([0]), 200)
    want, tol, _, _ = _attend_ref(r, q, [200], [0], 1 / math.sqrt(dh), 0)
    assert ((got.double() - want).abs() <= tol).all()
    _no_device_error()
    del cache, r
    B = 600
    r = Rig(B, 1, 16, 16, BF, 80, seed=2)
    before = [(7 * b) % 70 for b in range(B)]
    r.append(before)
    r.append([1] * B)
    q = r.randn(B, 2, 16)
    got = P.paged_attn(r.cache, q, _starts([1] * B), _i32(before), 1)
    want, tol, _, _ = _attend_ref(r, q, [1] * B, before, 0.25, 0)
    assert ((got.double() - want).abs() <= tol).all()
    _no_device_error()


@pytest.mark.parametrize('dh,Hq,Hkv,before,new,room', [
    (64, 8, 1, [20000], [1], 0),              # every part of the one item: more than a hundred for each of a few heads
    (128, 6, 2, [9000], [1], 0),
    (64, 4, 2, [15000], [7], 0),              # two groups of rows
    (32, 2, 1, [40000], [1], 0),
    (64, 12, 12, [0], [1], 30000),            # a long table that holds little: no parts, one, a few
    (64, 2, 1, [63, 0, 700], [1, 1, 1], 60000),
    (128, 4, 2, [9000, 5, 127], [2, 0, 1], 9000),
])
def test_attention_of_many_parts(dh, Hq, Hkv, before, new, room):
    """Few items over long tables: their states come from many warps of many CTAs."""
    P = _mod()
    r = Rig(len(new), Hkv, dh, 64, BF, max(max(a + b for a, b in zip(before, new)), room), seed=dh + Hq)
    if any(before):
        r.append(before)
    r.append(new)
    q = r.randn(sum(new), Hq, dh)
    ws = P.paged_attn_workspace(len(new), Hq, Hkv, dh, max(new))
    lse = torch.empty(sum(new), Hq, device=DEV)
    got = P.paged_attn(r.cache, q, _starts(new), _i32(before), max(new), ws=ws, lse=lse)
    want, tol, wl, ltol = _attend_ref(r, q, new, before, 1 / math.sqrt(dh), 0)
    assert ((got.double() - want).abs() <= tol).all()
    assert ((lse.double() - wl).abs() <= ltol).all()
    for _ in range(3):
        assert torch.equal(P.paged_attn(r.cache, q, _starts(new), _i32(before), max(new), ws=ws), got)
    _no_device_error()


def test_one_workspace_for_many_shapes():
    """A workspace large enough for every call serves calls of other shapes in turn: few rows, other batches and heads, tiles."""
    P = _mod()
    calls = []
    for B, H, Hq, dh, n, before, seed in ((1, 2, 2, 64, 1, 3000, 1), (40, 4, 8, 64, 2, 200, 2), (2, 2, 4, 64, 300, 900, 3),
                                          (3, 8, 8, 128, 1, 2000, 4), (2, 1, 8, 128, 3, 2500, 5), (64, 12, 12, 16, 1, 40, 6)):
        r = Rig(B, H, dh, 32, BF, before + n, seed=seed)
        r.append([before] * B)
        r.append([n] * B)
        q = r.randn(B * n, Hq, dh)
        calls.append((r, q, n, [before] * B, Hq))
    ws = torch.zeros(64 << 20, device=DEV, dtype=torch.uint8)
    want = [_attend_ref(r, q, [n] * r.B, pos, 1 / math.sqrt(r.dh), 0)[:2] for r, q, n, pos, _ in calls]
    for _ in range(2):
        for (r, q, n, pos, _), (w, tol) in zip(calls, want):
            got = P.paged_attn(r.cache, q, _starts([n] * r.B), _i32(pos), n, ws=ws)
            assert ((got.double() - w).abs() <= tol).all()
    with pytest.raises(RuntimeError, match='workspace'):
        r, q, n, pos, _ = calls[0]
        P.paged_attn(r.cache, q, _starts([n]), _i32(pos), n, ws=ws[:4096])
    _no_device_error()


def test_more_sequences_than_one_plan_holds():
    """2100 sequences, some with nothing new."""
    P = _mod()
    B = 2100
    r = Rig(B, 1, 16, 16, HF, 48, seed=9)
    before, new = [b % 40 for b in range(B)], [(b % 3 != 0) * 1 for b in range(B)]
    r.append(before)
    r.append(new)
    q = r.randn(sum(new), 2, 16)
    got = P.paged_attn(r.cache, q, _starts(new), _i32(before), 1)
    want, tol, _, _ = _attend_ref(r, q, new, before, 0.25, 0)
    assert ((got.double() - want).abs() <= tol).all()
    _no_device_error()


@pytest.mark.parametrize('n', [1, 60])
def test_scales_and_windows_at_their_ends(n):
    """A negative scale, scale 0 (the mean of the values), a window of the largest integer (the whole prefix)."""
    P = _mod()
    r = Rig(2, 2, 64, 16, BF, 200, seed=8)
    r.append([100, 30])
    r.append([n, n])
    q = r.randn(2 * n, 2, 64)
    for scale, window in ((-0.3, 0), (0.0, 0), (0.125, 2 ** 31 - 1), (-0.2, 33)):
        got = P.paged_attn(r.cache, q, _starts([n, n]), _i32([100, 30]), n, scale=scale, window=window)
        want, tol, _, _ = _attend_ref(r, q, [n, n], [100, 30], scale, 0 if window > 1000 else window)
        assert ((got.double() - want).abs() <= tol.abs() + 1e-5).all(), (scale, window)
    _no_device_error()


def test_run_time_faults_are_recorded():
    """Pages outside the pool, positions beyond the table, more rows than max_new: recorded, the others computed."""
    P = _mod()
    r = Rig(2, 1, 64, 16, BF, 64, seed=4)
    r.append([20, 20])
    before = r.cache.pool.clone()
    r.cache.table[0, 1] = 10 ** 6
    r.cache.table[1, 1] = r.perm[1, 1]
    P.paged_append(r.cache, r.randn(24, 1, 64), r.randn(24, 1, 64), _starts([12, 12]), _i32([20, 20]), 12)
    assert _device_error()[:3] == (3, 16, 0)
    changed = (r.cache.pool != before).any(-1).any(-1).nonzero()[:, 0].tolist()
    assert changed == [int(r.perm[1, 1])]
    P.paged_append(r.cache, r.randn(2, 1, 64), r.randn(2, 1, 64), _starts([1, 1]), _i32([16 * 4 + 15, 20]), 1)
    assert _device_error()[:2] == (2, 16)
    q = r.randn(2, 1, 64)
    out = torch.full((2, 1, 64), 3.0, device=DEV, dtype=BF)
    P.paged_attn(r.cache, q, _starts([1, 1]), _i32([-1, 18]), 1, out=out)
    assert _device_error()[:2] == (2, 17)
    assert (out[0] == 3).all() and torch.isfinite(out[1]).all() and (out[1] != 3).any()
    out.fill_(3)
    P.paged_attn(r.cache, r.randn(4, 1, 64), _starts([3, 1]), _i32([15, 18]), 1, out=torch.empty(4, 1, 64, device=DEV, dtype=BF))
    assert _device_error()[:2] == (3, 17)


def test_other_stream_and_graph():
    """The calls run on the current stream, and a captured graph of append and attention replays on changed contents."""
    P = _mod()
    r = Rig(3, 2, 64, 16, BF, 64, seed=6)
    r.append([10, 15, 31])
    pos = _i32([10, 15, 31])
    start = _starts([1, 1, 1])
    r.cache.table[:, :3] = r.perm[:, :3]
    k, v, q = r.randn(3, 2, 64), r.randn(3, 2, 64), r.randn(3, 4, 64)
    ws = P.paged_attn_workspace(3, 4, 2, 64, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        P.paged_append(r.cache, k, v, start, pos, 1)
        P.paged_attn(r.cache, q, start, pos, 1, out=out, ws=ws)
        with torch.cuda.graph(g, stream=s):
            P.paged_append(r.cache, k, v, start, pos, 1)
            P.paged_attn(r.cache, q, start, pos, 1, out=out, ws=ws)
    torch.cuda.current_stream().wait_stream(s)
    for step in range(4):
        for t in (k, v, q):
            t.copy_(r.randn(*t.shape))
        g.replay()
        at = [10 + step, 15 + step, 31 + step]
        for b in range(3):
            r.K[b, :, at[b]], r.V[b, :, at[b]] = k[b], v[b]
        r.len = [x + 1 for x in at]
        want, tol, _, _ = _attend_ref(r, q, [1, 1, 1], at, 0.125, 0)
        assert ((out.double() - want).abs() <= tol).all()
        pos += 1
    r.check_reads()
    _no_device_error()


def test_refusals():
    P = _mod()
    r = Rig(2, 2, 64, 16, BF, 64)
    k, q, s, p = r.randn(2, 2, 64), r.randn(2, 4, 64), _starts([1, 1]), _i32([0, 0])
    with pytest.raises(ValueError, match='16, 32 or 64'):
        P.PagedKV(r.cache.pool, r.cache.tail, r.cache.table, 48, 64)
    with pytest.raises(ValueError, match='pool must be'):
        P.PagedKV(r.cache.pool, r.cache.tail, r.cache.table, 32, 64)
    with pytest.raises(ValueError, match='tail must be'):
        P.PagedKV(r.cache.pool, r.cache.tail[:, :1], r.cache.table, 16, 64)
    with pytest.raises(TypeError, match='bfloat16 or float16'):
        P.PagedKV(r.cache.pool, r.cache.tail.float(), r.cache.table, 16, 64)
    with pytest.raises(ValueError, match='table'):
        P.PagedKV(r.cache.pool, r.cache.tail, r.cache.table.long(), 16, 64)
    with pytest.raises(TypeError, match='tail'):
        P.paged_append(r.cache, k.half(), k.half(), s, p, 1)
    with pytest.raises(ValueError, match='k and v'):
        P.paged_append(r.cache, k[:, :1], k[:, :1], s, p, 1)
    with pytest.raises(TypeError, match='int32'):
        P.paged_append(r.cache, k, k, s.long(), p, 1)
    with pytest.raises(ValueError, match='batch'):
        P.paged_append(r.cache, k, k, s[:2], p[:1], 1)
    with pytest.raises(ValueError, match='contiguous'):
        P.paged_append(r.cache, k.transpose(1, 2).contiguous().transpose(1, 2), k, s, p, 1)
    with pytest.raises(ValueError, match='rotation'):
        P.paged_append(r.cache, k, k, s, p, 1, rotation=(torch.zeros(4, 8, device=DEV), torch.zeros(4, 4, device=DEV)))
    with pytest.raises(ValueError, match='even'):
        P.rotation_table(8, 7)
    with pytest.raises(ValueError, match='CUDA'):
        P.paged_attn(r.cache, q.cpu(), s, p, 1)
    with pytest.raises(RuntimeError, match='multiple of Hkv'):
        P.paged_attn(r.cache, r.randn(2, 3, 64), s, p, 1)
    with pytest.raises(RuntimeError, match='window'):
        P.paged_attn(r.cache, q, s, p, 1, window=-1)
    with pytest.raises(ValueError, match='lse'):
        P.paged_attn(r.cache, q, s, p, 1, lse=torch.empty(2, 2, device=DEV))
    with pytest.raises(RuntimeError, match='aligned'):
        P.paged_attn(r.cache, r.randn(2 * 4 * 64 + 4)[4:].view(2, 4, 64), s, p, 1)
    a = torch.rand(2, 3, 10, device=DEV)
    d, u = torch.zeros(2, 2, device=DEV, dtype=torch.int64), torch.rand(2, 3, device=DEV)
    for bad in ((a, a, d, u), (a, a[:, :2].half(), d, u), (a, a[:, :2], d.int(), u), (a, a[:, :2], d, u[:, :2])):
        with pytest.raises((ValueError, TypeError), match='verify_drafts'):
            P.verify_drafts(*bad)
    # nothing to do: accepted, nothing written
    assert P.paged_attn(r.cache, q[:0], _starts([0, 0]), p, 0).shape == (0, 4, 64)
    _no_device_error()


# ------------------------------------------------------------------------------------------------ verification
def _verify_ref(p, q, d, u, n):
    """The definition in whole numbers, word by word."""
    f = np.float32
    p, q, u = [x.float().cpu().numpy() for x in (p, q, u)]
    B, G, V = q.shape
    tokens = np.full((B, G + 1), -1, np.int64)
    acc = np.zeros(B, np.int32)
    with np.errstate(invalid='ignore'):
        for b in range(B):
            a = 0
            while a < n[b] and f(u[b, a] * q[b, a, d[b, a]]) < p[b, a, d[b, a]]:
                a += 1

            def units(x, y):
                z = np.where(x > y, np.minimum(x - y, f(1)), f(0))
                return [int(w * f(2.0 ** 38)) for w in z]

            w = units(p[b, a], q[b, a] if a < n[b] else np.zeros(V, f))
            if sum(w) == 0:
                w = units(p[b, a], np.zeros(V, f))
            mark = sum(w) * min(int(u[b, G] * f(2 ** 24)), 2 ** 24 - 1) >> 24
            c, tok = 0, V - 1
            for i, x in enumerate(w):
                c += x
                if c > mark:
                    tok = i
                    break
            acc[b] = a
            tokens[b, :a] = d[b, :a]
            tokens[b, a] = tok
    return tokens, acc


def _verify_case(B, G, V, dt, seed, noise=0.7, sharp=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, G + 1, V, device=DEV, generator=g) * sharp
    p = x.softmax(-1)
    q = (x[:, :G] + noise * torch.randn(B, G, V, device=DEV, generator=g)).softmax(-1)
    d = torch.multinomial(q.reshape(-1, V), 1, generator=g).view(B, G) if G else torch.zeros(B, 0, device=DEV).long()
    u = torch.rand(B, G + 1, device=DEV, generator=g)
    n = torch.randint(0, G + 1, (B,), device=DEV, generator=g).int()
    return p.to(dt), q.to(dt), d, u, n


@pytest.mark.parametrize('B,G,V,dt', [(7, 4, 1000, torch.float32), (3, 1, 33, BF), (5, 8, 4096, HF), (2, 3, 50304, torch.float32),
                                      (4, 2, 1, torch.float32), (3, 0, 257, torch.float32), (2, 5, 8191, BF),
                                      (40, 16, 31, torch.float32), (1, 2, 131071, BF)])
def test_verify(B, G, V, dt):
    P = _mod()
    p, q, d, u, n = _verify_case(B, G, V, dt, B * V + G)
    for nd in (n, None):
        tok, acc = P.verify_drafts(p, q, d, u, nd)
        wt, wa = _verify_ref(p, q, d.cpu().numpy(), u, n.tolist() if nd is not None else [G] * B)
        assert np.array_equal(acc.cpu().numpy(), wa)
        assert np.array_equal(tok.cpu().numpy(), wt)
    _no_device_error()


def test_verify_edges():
    """u at 0 and just below 1; a row whose residual is empty; zeros, NaN and infinities in the rows; strided rows; a drafted
    word outside the vocabulary."""
    P = _mod()
    p, q, d, u, n = _verify_case(6, 3, 300, torch.float32, 9)
    u[0] = 0
    u[1] = 1 - 2.0 ** -24
    q[2] = p[2, :3] * 2          # every draft fails at u above 1/2, and nothing is left over
    u[2] = 0.75
    p[3, :, 100:] = 0
    p[4, 1, 5] = math.nan
    p[4, 0, 7] = math.inf
    wide = torch.zeros(6, 8, 320, device=DEV)
    wide[:, 1:5, 7:307] = p
    for pp in (p, wide[:, 1:5, 7:307]):
        tok, acc = P.verify_drafts(pp, q, d, u)
        wt, wa = _verify_ref(p, q, d.cpu().numpy(), u, [3] * 6)
        assert np.array_equal(acc.cpu().numpy(), wa) and np.array_equal(tok.cpu().numpy(), wt)
    assert int(acc[2]) == 0
    _no_device_error()
    d[5, 0] = 300
    tok, acc = P.verify_drafts(p, q, d, u)
    assert _device_error()[:3] == (3, 18, 5) and int(acc[5]) == 0
    # no positive weight at all
    tok, acc = P.verify_drafts(torch.zeros_like(p), q, torch.zeros_like(d), u)
    assert (acc == 0).all() and (tok[:, 0] == 299).all()
    _no_device_error()


def test_verify_distribution():
    """Over many draws the first emitted token follows p[0] whatever q is: each word's count within 5 standard deviations."""
    P = _mod()
    B, V = 200000, 7
    g = torch.Generator(device=DEV).manual_seed(11)
    p = torch.tensor([0.4, 0.05, 0.2, 0.0, 0.25, 0.09, 0.01], device=DEV)
    q = torch.tensor([0.1, 0.3, 0.1, 0.2, 0.1, 0.1, 0.1], device=DEV)
    d = torch.multinomial(q.expand(B, V), 1, generator=g)
    u = torch.rand(B, 2, device=DEV, generator=g)
    tok, acc = P.verify_drafts(p.expand(B, 2, V), q.expand(B, 1, V), d, u)
    first = torch.bincount(tok[:, 0], minlength=V).double()
    assert first.sum() == B
    sd = (B * p.double() * (1 - p.double())).sqrt()
    assert ((first - B * p.double()).abs() <= 5 * sd + 1e-9).all(), first / B


# ------------------------------------------------------------------------------------------------ sizes of the values
def _value_units(r, b, L):
    """What one code of each token's value stands for (an upper bound), in 64 bits: the page's scale; in the open page the power of
    two that takes a 16-token group's largest value into [2^8, 2^9) (at least 1 for f16, which is not scaled down); 2^-64 where
    all values are 0."""
    V = r.cache.read(b, L)[1].double().abs()                       # (Hkv, L, dh)
    u = torch.empty(r.Hkv, L, device=DEV, dtype=torch.float64)
    full = L // r.page * r.page
    for a in range(0, L, 16):
        top = V[:, a:a + 16].amax((-1, -2))
        if a < full:
            page = a // r.page * r.page
            unit = V[:, page:page + r.page].amax((-1, -2)) * 2 / 448  # (a page whose largest value is no multiple of a code)
        else:
            unit = top * 2.0 ** -8
            if r.dt == HF:
                unit = unit.clamp(min=2.0 ** -30)
        u[:, a:a + 16] = torch.where(top > 0, unit, 2.0 ** -64)[:, None]
    return u


def _attend_tight(r, q, counts, pos, scale):
    """As _attend_ref, but a tolerance that scales with the values: no absolute term but the output's last place (f16) and, for
    every token, half of f16's smallest step (2^-25) of a weight where the largest weight of the row is at least 2^6."""
    Hq, dh = q.shape[1:]
    grp = Hq // r.Hkv
    outs, tols = [], []
    row = 0
    for b, n in enumerate(counts):
        L = pos[b] + n
        K, V = [x.double() for x in r.cache.read(b, L)]
        qb = q[row:row + n].double().view(n, r.Hkv, grp, dh).permute(1, 2, 0, 3)
        s = torch.einsum('hgnd,htd->hgnt', qb, K) * scale
        mag = torch.einsum('hgnd,htd->hgnt', qb.abs(), K.abs()).amax(-1) * abs(scale)
        hide = torch.arange(L, device=DEV) > pos[b] + torch.arange(n, device=DEV)[:, None]
        p = s.masked_fill(hide, -math.inf).softmax(-1)
        unit = _value_units(r, b, L)
        u = torch.full((L,), 2.0 ** -11, device=DEV, dtype=torch.float64)
        u[L // r.page * r.page:] = U[r.dt]
        d = 2 * dh * 2.0 ** -24 * mag
        step = 2.0 ** -31 * (p * unit[:, None, None]).amax(-1, keepdim=True) / unit[:, None, None]  # of a token's p
        part = p * u + p * (2 * d + 1e-5)[..., None] + step.masked_fill(hide, 0)
        o = torch.einsum('hgnt,htd->nhgd', p, V).reshape(n, Hq, dh)
        outs.append(o)
        tols.append(U[r.dt] * o.abs() + torch.einsum('hgnt,htd->nhgd', part, V.abs()).reshape(n, Hq, dh)
                    + (2.0 ** -25 if r.dt == HF else 2.0 ** -133))
        row += n
    return torch.cat(outs), torch.cat(tols)


SIZES = [(64, 64, BF, 1, -20), (64, 64, BF, 1, -30), (64, 64, BF, 40, -20), (64, 64, BF, 40, -30), (128, 32, BF, 1, -30),
         (128, 32, BF, 48, -30), (64, 16, HF, 1, -12), (64, 16, HF, 1, -20), (64, 64, HF, 40, -12), (128, 64, HF, 40, -20),
         (32, 32, BF, 1, -30), (32, 32, BF, 40, -30), (16, 64, HF, 36, -12), (64, 64, BF, 1, 40), (64, 32, BF, 40, 40),
         (64, 64, HF, 1, 10), (128, 64, HF, 40, 10), (64, 64, BF, 20, -30), (128, 64, HF, 20, -20)]


def _many(n):
    """Sequences: so many items of 160 kv heads that a warp, or a CTA, holds whole ones (the parts of an item that several share
    meet in fp32)."""
    return 8 if n <= 32 else 2


@pytest.mark.parametrize('dh,page,dt,n,shift', SIZES)
def test_attention_of_small_and_large_values(dh, page, dt, n, shift):
    """Values scaled by a power of two, in full pages and in the open one: the output's error scales with them."""
    P = _mod()
    B, H = _many(n), 160
    r = Rig(B, H, dh, page, dt, 400 + n, seed=dh + n - shift)
    before = [256 + (i % 2) * (page // 2 + 3) for i in range(B)]
    N = sum(before)
    r.append(before, r.randn(N, H, dh), (r.randn(N, H, dh).float() * 2.0 ** shift).to(dt))
    r.append([n] * B, r.randn(n * B, H, dh), (r.randn(n * B, H, dh).float() * 2.0 ** shift).to(dt))
    q = r.randn(B * n, H, dh)
    got = P.paged_attn(r.cache, q, _starts([n] * B), _i32(before), n)
    want, tol = _attend_tight(r, q, [n] * B, before, 1 / math.sqrt(dh))
    d = (got.double() - want).abs()
    assert (d <= tol).all(), float((d / tol).max())
    _no_device_error()


@pytest.mark.parametrize('dh,page,dt,n,shift', SIZES)
def test_attention_beside_zero_values(dh, page, dt, n, shift):
    """Pages of zeros (which store scale 1) before and between pages of scaled values, 16 tokens of zeros inside another, and, in
    every second sequence, an open page of zeros: they weigh what their scores say and the others keep their precision."""
    P = _mod()
    B, H = _many(n), 160
    r = Rig(B, H, dh, page, dt, 400 + n, seed=dh + n + shift)
    before = [256 + (i % 2) * (page // 2 + 3) for i in range(B)]
    N = sum(before)
    k, v = r.randn(N, H, dh, spread=2.0), (r.randn(N, H, dh).float() * 2.0 ** shift).to(dt)
    new = (r.randn(n * B, H, dh).float() * 2.0 ** shift).to(dt)
    row = 0
    for b in range(B):
        for a in (0, 128):
            v[row + a:row + a + 64] = 0
        v[row + 80:row + 96] = 0
        if b % 2:
            v[row + 256:row + before[b]] = 0
            new[b * n:(b + 1) * n] = 0
        row += before[b]
    r.append(before, k, v)
    r.append([n] * B, r.randn(n * B, H, dh), new)
    q = r.randn(B * n, H, dh)
    lse = torch.empty(B * n, H, device=DEV)
    got = P.paged_attn(r.cache, q, _starts([n] * B), _i32(before), n, lse=lse)
    want, tol = _attend_tight(r, q, [n] * B, before, 1 / math.sqrt(dh))
    d = (got.double() - want).abs()
    assert (d <= tol).all(), float((d / tol).max())
    _, _, wl, ltol = _attend_ref(r, q, [n] * B, before, 1 / math.sqrt(dh), 0)
    assert ((lse.double() - wl).abs() <= ltol).all()
    _no_device_error()


@pytest.mark.parametrize('page,dh,dt', [(16, 64, BF), (64, 128, HF), (32, 16, BF)])
def test_pages_of_zero_values_are_marked(page, dh, dt):
    """The record's third word is 1 for pages whose values are all 0 (or below 2^-100), whatever the keys hold, and 0 for every other
    page, one that is quantised again with values among them."""
    r = Rig(5, 1, dh, page, dt, 2 * page)
    k, v = r.randn(5 * page, 1, dh), r.randn(5 * page, 1, dh)
    v[:page] = 0
    v[page:2 * page] = -0.0
    k[2 * page:3 * page] = 0
    v[3 * page + 1, 0, 2] = math.nan
    v[4 * page:] = 448.0 if dt == BF else 1.0
    if dt == BF:
        v[page + 3] = 2.0 ** -104

    def marks():
        return [float(r.cache.pool[int(r.perm[b, 0])].view(torch.float32)[0, -2]) for b in range(5)]

    r.append([page] * 5, k, v)
    assert marks() == [1, 1, 0, 0, 0]
    r.append([1] * 5, r.randn(5, 1, dh), r.randn(5, 1, dh), pos=[page - 1] * 5)  # the last token of each page replaced
    assert marks() == [0, 0, 0, 0, 0]
    _no_device_error()


@pytest.mark.parametrize('dh,page,dt,grp,n', [(64, 64, BF, 1, 30), (64, 64, HF, 1, 30), (64, 64, BF, 2, 30), (128, 64, HF, 2, 30),
                                               (32, 32, BF, 1, 20), (32, 64, HF, 2, 30), (16, 16, BF, 4, 8), (128, 64, BF, 1, 9)])
@pytest.mark.parametrize('window', [0, 4])
def test_odd_values_in_the_open_page_stay_with_their_rows(dh, page, dt, grp, n, window):
    """An infinity or NaN in a value of the open page reaches the rows that see its token, in its dim, and nothing else: neither
    earlier queries of the call (some of them of the page before), nor those whose window has passed it."""
    P = _mod()
    r = Rig(2, 1, dh, page, dt, 4 * page, seed=dh + n)
    before = [2 * page - 5, 7]                        # the first call's queries begin in the page before the open one
    r.append(before)
    k, v = r.randn(2 * n, 1, dh), r.randn(2 * n, 1, dh)
    odd = v.clone()
    at = [5 + (n - 5) // 3, 5 + (n - 5) // 2]         # rows of sequence 0 that stand in its open page
    odd[at[0], 0, 3], odd[at[1], 0, 5], odd[at[1], 0, dh - 1] = math.nan, math.inf, -math.inf
    odd[n, 0, 0] = -math.inf                          # sequence 1: its first new token
    v = torch.where(torch.isfinite(odd), odd, 0)
    q = r.randn(2 * n, grp, dh)
    pos = list(r.len)
    assert (pos[0] + n) // page == 2 and (pos[1] + n) < page or page < 64
    r.append([n, n], k, v)
    want, tol, wl, ltol = _attend_ref(r, q, [n, n], pos, 1 / math.sqrt(dh), window)
    r.append([n, n], k, odd, pos=pos)
    for b in range(2):  # only tokens that are still in 16 bits are asked about
        assert torch.isfinite(r.cache.read(b, r.len[b] // page * page)[1]).all()
    for i in range(2 * n):
        b, j = divmod(i, n)
        for row, dim in ((at[0], 3), (at[1], 5), (at[1], dh - 1), (n, 0)):
            if row // n == b and row % n <= j and (not window or row % n > j - window):
                want[i, :, dim] += float(odd[row, 0, dim])
    lse = torch.empty(2 * n, grp, device=DEV)
    got = P.paged_attn(r.cache, q, _starts([n, n]), _i32(pos), n, window=window, lse=lse).double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert ((got - want).abs() <= tol)[fin].all()
    assert ((lse.double() - wl).abs() <= ltol).all()
    _no_device_error()


@pytest.mark.parametrize('dh,Hq,Hkv,n,room', [(64, 2, 2, 2, 0), (64, 8, 1, 1, 30000), (128, 4, 1, 4, 20000), (128, 2, 2, 2, 0),
                                               (64, 4, 1, 40, 0), (128, 4, 1, 50, 0), (32, 4, 2, 2, 40000)])
def test_odd_values_of_items_in_parts(dh, Hq, Hkv, n, room):
    """The same where an item's pages are shared by many warps or CTAs, joined on the spot or late: the open page's part tells the one
    that writes the output."""
    P = _mod()
    r = Rig(2, Hkv, dh, 64, BF, max(6000 + n, room), seed=dh + n)
    r.append([5000, 5504])                            # open pages of 8 and 0 tokens before the call
    k, v = r.randn(2 * n, Hkv, dh), r.randn(2 * n, Hkv, dh)
    q = r.randn(2 * n, Hq, dh)
    pos = list(r.len)
    odd = v.clone()
    odd[n - 1, 0, 7], odd[n, Hkv - 1, dh - 2] = math.inf, math.nan  # sequence 0's last token, sequence 1's first
    v = torch.where(torch.isfinite(odd), odd, 0)
    r.append([n, n], k, v)
    want, tol, wl, ltol = _attend_ref(r, q, [n, n], pos, 1 / math.sqrt(dh), 0)
    r.append([n, n], k, odd, pos=pos)
    want[n - 1, :Hq // Hkv, 7] += math.inf
    want[n:, Hq - Hq // Hkv:, dh - 2] += math.nan
    lse = torch.empty(2 * n, Hq, device=DEV)
    ws = P.paged_attn_workspace(2, Hq, Hkv, dh, n)
    for _ in range(2):
        got = P.paged_attn(r.cache, q, _starts([n, n]), _i32(pos), n, lse=lse, ws=ws).double()
        fin = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
        assert ((got - want).abs() <= tol)[fin].all()
        assert ((lse.double() - wl).abs() <= ltol).all()
    _no_device_error()


@pytest.mark.parametrize('dh,n', [(64, 1), (64, 40), (128, 3), (32, 40), (128, 50)])
def test_large_keys_and_small_queries(dh, n):
    """bf16 keys of 2^112 against queries of 2^-106: scores far below the type's end, from codes and from the open page alike."""
    P = _mod()
    r = Rig(2, 1, dh, 64, BF, 256, seed=dh + n)
    before = [3, 150]
    N = sum(before) + 2 * n
    k = (r.randn(N, 1, dh).float() * 2.0 ** 112).to(BF)
    r.append(before, k[2 * n:], r.randn(sum(before), 1, dh))
    r.append([n, n], k[:2 * n], r.randn(2 * n, 1, dh))
    q = (r.randn(2 * n, 2, dh).float() * 2.0 ** -106).to(BF)
    got = P.paged_attn(r.cache, q, _starts([n, n]), _i32(before), n)
    want, tol, _, _ = _attend_ref(r, q, [n, n], before, 1 / math.sqrt(dh), 0)
    assert ((got.double() - want).abs() <= tol).all()
    _no_device_error()


@pytest.mark.parametrize('dh,page,grp,n', [(64, 64, 1, 1), (64, 16, 2, 3), (128, 64, 1, 1), (128, 16, 4, 2), (64, 32, 2, 40),
                                            (128, 64, 1, 70), (32, 16, 1, 40), (16, 32, 2, 1)])
@pytest.mark.parametrize('entry', [-3, 10 ** 6])
def test_pages_outside_the_pool_read_as_nan(dh, page, grp, n, entry):
    """A table entry outside the pool is recorded, and rows that see its page are NaN, not what another page holds; rows that do
    not see it (a window past it, another sequence) are as they would be."""
    P = _mod()
    r = Rig(2, 1, dh, page, BF, 4 * page + 2 * n + 16, seed=dh + n)
    r.cache.pool[0] = 0                              # what a page outside must not be taken for
    before = [4 * page + 5, 3 * page + 2]
    r.append(before)
    r.append([n, n])
    q = r.randn(2 * n, grp, dh)
    start, pos = _starts([n, n]), _i32(before)
    for window in (0, 2 * page):
        want, tol, _, _ = _attend_ref(r, q, [n, n], before, 1 / math.sqrt(dh), window)
        r.cache.table[0, 1] = entry
        got = P.paged_attn(r.cache, q, start, pos, n, window=window).double()
        r.cache.table[0, 1] = r.perm[0, 1]
        sees = torch.zeros(2 * n, dtype=torch.bool, device=DEV)
        for i in range(n):
            sees[i] = not window or before[0] + i - window + 1 < 2 * page
        assert torch.isnan(got[sees]).all()
        assert ((got - want).abs() <= tol)[~sees].all()
        code = _device_error()
        assert code[:3] == (3, 17, 0) if bool(sees.any()) else code[0] in (0, 3)
    again = P.paged_attn(r.cache, q, start, pos, n)
    want, tol, _, _ = _attend_ref(r, q, [n, n], before, 1 / math.sqrt(dh), 0)
    assert ((again.double() - want).abs() <= tol).all()
    _no_device_error()


def test_errors_of_both_kinds_are_reported():
    """A wait that gave up in one kernel and a position out of range in a serving kernel: one after the other, none lost."""
    from treeattn_b200 import _lib, _ops
    P = _mod()
    r = Rig(1, 1, 64, 16, BF, 64)
    r.append([3])
    _no_device_error()
    _lib.call('ta_wait_probe', 1000 * 1000, _ops._stream(r.cache.pool))
    P.paged_append(r.cache, r.randn(1, 1, 64), r.randn(1, 1, 64), _starts([1]), _i32([-4]), 1)
    seen = [_device_error()[:2] for _ in range(3)]
    assert sorted(seen) == [(0, 0), (1, 13), (2, 16)] and seen[2] == (0, 0)


@pytest.mark.parametrize('rot', [0, 32])
def test_a_given_query_output_is_written(rot):
    """q_out receives the queries, rotated or as they are, of the rows that belong to a sequence."""
    P = _mod()
    r = Rig(2, 2, 64, 16, BF, 64, seed=rot)
    qkv = r.randn(5, 8 * 64)
    q = qkv[:, :4 * 64].view(5, 4, 64)
    k, v = r.randn(5, 2, 64), r.randn(5, 2, 64)
    rotation = P.rotation_table(64, rot) if rot else None
    out = torch.full((5, 4, 64), 9.0, device=DEV, dtype=BF)
    got = P.paged_append(r.cache, k, v, _starts([3, 2]), _i32([4, 0]), 3, q=q, rotation=rotation, q_out=out)
    assert got is out
    want = q if not rot else P.paged_append(r.cache, k, v, _starts([3, 2]), _i32([4, 0]), 3, q=q, rotation=rotation)
    assert torch.equal(out, want)
    with pytest.raises(ValueError, match='q_out'):
        P.paged_append(r.cache, k, v, _starts([3, 2]), _i32([4, 0]), 3, q=q, rotation=rotation, q_out=out[:4])
    _no_device_error()


@pytest.mark.parametrize('Hkv,grp,n,before,room,worker', [(4, 1, 1, [3000, 700], 0, 1), (4, 1, 1, [3000, 700], 0, 9), (1, 8, 1, [9000, 300], 30000, 3),
                                                           (2, 1, 4, [9000, 40], 30000, 1), (2, 1, 60, [3000, 40], 0, 0),
                                                           (2, 1, 60, [3000, 40], 0, 2), (160, 1, 40, [100, 90], 0, 0)])
def test_a_wait_that_gives_up_leaves_the_workspace_ready(Hkv, grp, n, before, room, worker):
    """One worker's copies never come: its wait runs out after 2 s and is recorded, the rows of the items it took part in are NaN, all
    others are as ever, and the next call on the same workspace gives what it gave before."""
    from treeattn_b200 import _lib
    P = _mod()
    B, dh = len(before), 64
    r = Rig(B, Hkv, dh, 64, BF, max(max(before) + n, room), seed=Hkv + n)
    r.append(before)
    r.append([n] * B)
    q = r.randn(B * n, Hkv * grp, dh)
    start, pos = _starts([n] * B), _i32(before)
    ws = P.paged_attn_workspace(B, Hkv * grp, Hkv, dh, n)
    want = P.paged_attn(r.cache, q, start, pos, n, ws=ws)
    got, lse = torch.zeros_like(want), torch.zeros(B * n, Hkv * grp, device=DEV)
    c = r.cache
    _no_device_error()
    _lib.call('ta_paged_attn_probe', worker, c.pool.data_ptr(), c.tail.data_ptr(), c.table.data_ptr(), c.table.stride(0),
              c.pool.shape[0], c.table.shape[1], 64, 1, B, Hkv * grp, Hkv, dh, q.data_ptr(), q.stride(0), q.stride(1), B * n,
              start.data_ptr(), pos.data_ptr(), n, 0.125, 0, got.data_ptr(), got.stride(0), got.stride(1), lse.data_ptr(),
              ws.data_ptr(), ws.nbytes, P._stream(q))
    code = _device_error()
    assert code[0] == 1 and code[1] in (17, 19), code
    bad = torch.isnan(lse)
    assert bad.any() and not bad.all()
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])
    heads = bad.view(B, n, Hkv, grp)
    if n * grp <= 8:  # an item is NaN as a whole (a tile: 128 of its rows)
        assert torch.equal(heads, heads[:, :1, :, :1].expand_as(heads))
    for _ in range(2):
        assert torch.equal(P.paged_attn(r.cache, q, start, pos, n, ws=ws), want)
    _no_device_error()
