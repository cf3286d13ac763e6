"""Copies of the paged cache's records on the GPU, against indexing: bytes are equal."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _caches(layers, n_pages, B, H, dh, page, dtype, seed=0):
    from treeattn_b200.paged import PagedKV
    g = torch.Generator(device='cuda').manual_seed(seed)
    table = torch.zeros(B, 4, device='cuda', dtype=torch.int32)
    return [PagedKV(torch.randint(0, 256, (n_pages, H, 2 * page * dh + 16), device='cuda', generator=g, dtype=torch.uint8),
                    torch.randn(B, H, 2, 2, page * dh, device='cuda', generator=g).to(dtype), table, page, dh)
            for _ in range(layers)]


def _check(fn, caches, of, src, dst):
    want = []
    for c in caches:
        t = of(c).clone()
        if len(src):
            t[torch.tensor(dst, device='cuda')] = of(c)[torch.tensor(src, device='cuda')]
        want.append(t)
    fn(caches, src, dst)
    for c, w in zip(caches, want):
        assert torch.equal(of(c).view(torch.uint8), w.view(torch.uint8))


SHAPES = [(1, 1, 16, 16, torch.bfloat16), (3, 4, 128, 16, torch.float16), (2, 3, 32, 32, torch.bfloat16),
          (70, 1, 16, 16, torch.float16), (12, 12, 64, 64, torch.bfloat16)]


@pytest.mark.parametrize('layers,H,dh,page,dtype', SHAPES)
def test_moves(layers, H, dh, page, dtype):
    """One move, one source into many, chains, cycles, trees that end in a cycle, records onto themselves, none."""
    from treeattn_b200.paged import paged_copy, paged_fork
    caches = _caches(layers, 40, 13, H, dh, page, dtype)
    pool, tail = (lambda c: c.pool), (lambda c: c.tail)
    cases = [([0], [12]), ([5] * 12, [0, 1, 2, 3, 4, 6, 7, 8, 9, 10, 11, 12]), (list(range(12)), list(range(1, 13))),
             (list(range(13)), list(range(1, 13)) + [0]), ([1, 0, 1, 2, 7, 7], [0, 1, 2, 3, 7, 8]), ([], []), ([4, 5, 6], [4, 5, 6]),
             ([1, 2, 0, 4, 3, 2, 11], [0, 1, 2, 3, 4, 11, 12])]
    for src, dst in cases:
        _check(paged_fork, caches, tail, src, dst)
        _check(paged_copy, caches, pool, [s + 20 for s in src], [d + 20 for d in dst])


@pytest.mark.parametrize('n_pages,moves', [(5000, 4999), (5000, 2500), (70000, 700), (30, 30)])
def test_many_moves(n_pages, moves):
    """Lists longer than one launch holds, and pools above the size whose records are looked up in a table."""
    from treeattn_b200.paged import paged_copy
    rng = random.Random(n_pages + moves)
    caches = _caches(2, n_pages, 1, 1, 16, 16, torch.bfloat16)
    dst = rng.sample(range(n_pages), moves)
    _check(paged_copy, caches, lambda c: c.pool, [rng.randrange(n_pages) for _ in dst], dst)
    _check(paged_copy, caches, lambda c: c.pool, dst[::-1], dst)  # cycles of two
    chain = list(range(n_pages - 1))
    _check(paged_copy, caches, lambda c: c.pool, chain, [i + 1 for i in chain])  # one chain, over several launches


def test_offsets_beyond_32_bits():
    """Records at both ends of a pool of more than 2^32 bytes."""
    from treeattn_b200.paged import PagedKV, paged_copy
    page, dh, H = 64, 128, 16
    n = 2 ** 32 // (H * (2 * page * dh + 16)) + 40
    pool = torch.empty(n, H, 2 * page * dh + 16, device='cuda', dtype=torch.uint8)
    pool[:8].random_(0, 256)
    pool[-8:].random_(0, 256)
    c = PagedKV(pool, torch.zeros(1, H, 2, 2, page * dh, device='cuda', dtype=torch.bfloat16),
                torch.zeros(1, 1, device='cuda', dtype=torch.int32), page, dh)
    head, end = pool[:8].clone(), pool[-8:].clone()
    paged_copy([c], [0, n - 1, 3], [n - 1, 0, n - 4])
    head[0], end[7], end[4] = end[7].clone(), head[0].clone(), head[3]
    assert torch.equal(pool[:8], head) and torch.equal(pool[-8:], end)


def test_captured_and_on_another_stream():
    """A captured call repeats its moves, whatever the lists hold later; a call on a side stream follows that stream's work."""
    from treeattn_b200.paged import paged_fork
    caches = _caches(3, 2, 5, 2, 64, 32, torch.bfloat16)
    src, dst = [0, 1, 2], [1, 2, 0]
    before = [c.tail.clone() for c in caches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged_fork(caches, src, dst)
    torch.cuda.current_stream().wait_stream(side)
    for c, b in zip(caches, before):
        assert torch.equal(c.tail[[1, 2, 0]], b[[0, 1, 2]])
        c.tail.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged_fork(caches, src, dst)
    src[:], dst[:] = [3, 3, 3], [0, 1, 2]
    for _ in range(3):
        graph.replay()
    for c, b in zip(caches, before):
        assert torch.equal(c.tail, b)  # a cycle of three, three times


def _rows(rng, n, H, dh, dtype):
    return [torch.randn(n, H, dh, device='cuda', generator=rng).to(dtype) for _ in range(3)]


def test_forked_sequences_go_on_apart():
    """A prompt, forked, cut back into a shared page, appended to, compacted: attention over each sequence is what it is over a
    cache that was filled with the same rows sequence by sequence."""
    from treeattn_b200.paged import PagedKV, PagePool, paged_append, paged_attn, paged_copy, paged_fork
    B, H, dh, page, dt = 4, 2, 64, 16, torch.bfloat16
    g = torch.Generator(device='cuda').manual_seed(1)
    pool = PagePool(40, B, 8, page)
    caches = [PagedKV.empty(pool.n_pages, H, dh, pool.table, page, dt)]
    history = [[] for _ in range(B)]  # the rows (q, k, v) that each sequence holds
    pos = [0] * B

    def feed(counts):
        nonlocal pos
        pool.reserve([p + c for p, c in zip(pos, counts)], pos)
        q, k, v = _rows(g, sum(counts), H, dh, dt)
        start = torch.tensor([sum(counts[:i]) for i in range(B + 1)], device='cuda', dtype=torch.int32)
        at = torch.tensor(pos, device='cuda', dtype=torch.int32)
        paged_append(caches[0], k, v, start, at, max(counts))
        out = paged_attn(caches[0], q, start, at, max(counts))
        for b in range(B):
            rows = slice(int(start[b]), int(start[b + 1]))
            history[b] += list(zip(q[rows], k[rows], v[rows]))
        pos = [p + c for p, c in zip(pos, counts)]
        return out, start

    def alone():
        """The last row of each sequence over caches of their own."""
        want = []
        for b in range(B):
            n = len(history[b])
            if not n:
                want.append(None)
                continue
            table = torch.arange(8, device='cuda', dtype=torch.int32)[None]
            c = PagedKV.empty(8, H, dh, table, page, dt)
            q, k, v = [torch.stack(x) for x in zip(*history[b])]
            start, at = torch.tensor([0, n], device='cuda', dtype=torch.int32), torch.zeros(1, device='cuda', dtype=torch.int32)
            paged_append(c, k, v, start, at, n)
            want.append(paged_attn(c, q, start, at, n)[-1])
        return want

    def check(out, start):
        for b, w in enumerate(alone()):
            if start[b + 1] > start[b]:
                # the same codes and rows, taken by another split of the work: a few roundings of the output's type
                assert (out[int(start[b + 1]) - 1].float() - w.float()).abs().max() <= 4 * 2 ** -9 * w.float().abs().max()

    check(*feed([41, 0, 0, 5]))
    src, dst = [0, 0, 3], [1, 2, 0]  # and sequence 0 goes on from 3
    pool.fork(src, dst, [pos[s] for s in src])
    paged_fork(caches, src, dst)
    was = [list(h) for h in history], list(pos)
    for s, d in zip(src, dst):
        history[d], pos[d] = list(was[0][s]), was[1][s]
    check(*feed([3, 9, 2, 1]))
    # 2 goes back into a page that it shares with 1, and writes it again
    pos[2] = 30
    history[2] = history[2][:30]
    check(*feed([2, 1, 20, 12]))
    pool.release(3)
    history[3], pos[3] = [], 0
    n = pool.n_pages - len(pool.free) + 3
    paged_copy(caches, *pool.compact(n))
    c = caches[0]
    caches[0] = PagedKV(c.pool[:n].clone(), c.tail, c.table, page, dh)
    check(*feed([1, 3, 1, 0]))
    from treeattn_b200 import _ops
    assert _ops.device_error()[0] == 0


def test_decoder_forks():
    """PagedDecoder: forked sequences give the logits of sequences that were fed the same tokens, before and after compaction."""
    from treeattn_b200.config import Config
    from treeattn_b200.engine import weights_from_ours
    from treeattn_b200.model import GPT
    from treeattn_b200.speculative import PagedDecoder
    torch.manual_seed(0)
    cfg = Config(attn='seg', vocab_size=96, seq_len=128, n_layer=2, n_head=2, n_embd=64, neighbors=False, chunk=64)
    W = weights_from_ours(GPT(cfg).state_dict(), cfg)
    made = lambda: PagedDecoder(W, 2, 2, 64, batch=3, page=16)
    dec, ref = made(), made()
    tok = torch.randint(0, 96, (3, 37), device='cuda')
    dec.forward(tok)
    dec.fork([0, 0, 1], [1, 2, 0])
    seen = tok[[1, 0, 0]]
    for step in range(3):
        new = torch.randint(0, 96, (3, 7), device='cuda')
        seen = torch.cat([seen, new], 1)
        got = dec.forward(new)
        ref.reset()
        want = ref.forward(seen)[:, -7:]
        # another split of the attention's work: a few roundings of 16 bits through two layers
        assert (got.float() - want.float()).abs().max() <= 0.02 * want.float().abs().max()
        if step == 0:
            dec.cut_back([dec.pos[0], dec.pos[1] - 7, dec.pos[2]])  # 1 drops its new tokens; the others keep theirs
            assert dec.pos == [44, 37, 44]
            dec.fork([0], [1])
            seen[1] = seen[0]
        if step == 1:
            held = dec.pool.n_pages
            dec.compact(held - 5)
            assert dec.caches[0].pool.shape[0] == held - 5
    dec.release(2)
    assert dec.pos[2] == 0
    with pytest.raises(ValueError, match='sequences'):
        dec.fork([0], [3])
