"""CPU checks of the serving operators: rejected arguments, the page allocator, the order of a page's elements."""
import ctypes

import pytest
import torch


def test_rejected_arguments_without_gpu():
    """The entry points refuse bad arguments with a message before any CUDA call."""
    from treeattn_b200 import _lib
    lib = _lib.load()
    a = 1 << 20  # an aligned address that is never dereferenced
    f = ctypes.c_float(0.125)

    def attn(page=64, dtype=1, B=2, Hq=4, Hkv=4, dh=64, q=a, window=0, pool=a, n_pages=9, max_pages=3, sb=3):
        return lib.ta_paged_attn(pool, a, a, sb, n_pages, max_pages, page, dtype, B, Hq, Hkv, dh, q, 256, 64, 2, a, a, 1, f,
                                 window, a, 256, 64, None, a, 1 << 30, None)

    for kw, what in ((dict(page=48), 'pages of 48'), (dict(dtype=0), 'dtype'), (dict(dh=48), 'head dim'),
                     (dict(Hq=6), 'multiple of Hkv'), (dict(window=-2), 'window'), (dict(q=a + 2), 'aligned'),
                     (dict(pool=None), 'null'), (dict(n_pages=0), 'page counts'), (dict(sb=2), 'page counts'),
                     (dict(pool=a + 4), 'aligned'), (dict(B=-1), 'bad sizes'), (dict(q=None), 'null')):
        assert attn(**kw) == _lib.TA_ERR_ARG
        assert 'ta_paged_attn' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())
    assert attn(B=0) == _lib.TA_OK

    def append(k=a, rot=64, cos=a, q=a, qo=a, dtype=2, max_new=1):
        return lib.ta_paged_append(a, a, a, 3, 9, 3, 16, dtype, 2, 4, 64, k, a, 256, 64, 256, 64, 2, a, a, max_new, cos, a,
                                   100, rot, q, 8, 512, 64, qo, None)

    for kw, what in ((dict(rot=63), 'rotated dims'), (dict(rot=128), 'rotated dims'), (dict(cos=None), 'null'),
                     (dict(q=None), 'null'), (dict(k=a + 8), 'aligned'), (dict(dtype=0), 'dtype'), (dict(max_new=-1), 'bad sizes')):
        assert append(**kw) == _lib.TA_ERR_ARG
        assert 'ta_paged_append' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())

    def verify(p=a, dtype=0, G=4, V=100):
        return lib.ta_verify_drafts(p, 500, 100, a, 400, 100, dtype, 2, G, V, a, a, None, a, a, None)

    for kw, what in ((dict(p=None), 'null'), (dict(dtype=7), 'dtype'), (dict(G=-1), 'bad sizes'), (dict(V=0), 'bad sizes'),
                     (dict(G=5000), 'bad sizes')):
        assert verify(**kw) == _lib.TA_ERR_ARG
        assert 'ta_verify_drafts' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())


def test_cpu_tensors_are_refused():
    from treeattn_b200 import paged
    with pytest.raises(ValueError, match='CUDA'):
        paged.PagedKV.empty(4, 2, 64, torch.zeros(1, 2, dtype=torch.int32), 16)
    p = torch.rand(2, 3, 8)
    with pytest.raises(ValueError, match='CUDA'):
        paged.verify_drafts(p, p[:, :2], torch.zeros(2, 2, dtype=torch.int64), torch.rand(2, 3))


def test_page_pool():
    """Pages are handed out once, come back, and a request that cannot be met changes nothing."""
    from treeattn_b200.paged import PagePool
    pool = PagePool(10, 3, 6, 16, device='cpu')
    pool.reserve([17, 0, 64])
    assert [len(o) for o in pool.owned] == [2, 0, 4]
    seen = [pg for o in pool.owned for pg in o]
    assert len(set(seen)) == 6 and set(seen) | set(pool.free) == set(range(10))
    for b, o in enumerate(pool.owned):
        assert pool.table[b, :len(o)].tolist() == o
    pool.reserve([1, 1, 1])
    assert [len(o) for o in pool.owned] == [2, 1, 4]
    before = ([list(o) for o in pool.owned], list(pool.free), pool.table.clone())
    with pytest.raises(MemoryError):
        pool.reserve([96, 17, 64])
    with pytest.raises(ValueError, match='above'):
        pool.reserve([97, 0, 0])
    assert before[0] == pool.owned and before[1] == pool.free and torch.equal(before[2], pool.table)
    pool.release(2)
    pool.reserve([96, 17, 0])
    assert [len(o) for o in pool.owned] == [6, 2, 0]
    assert sorted(pg for o in pool.owned for pg in o) + sorted(pool.free) != [] and len(pool.free) == 2


@pytest.mark.parametrize('dh', [16, 32, 64, 128])
def test_page_order(dh):
    """The element order of a page, spelled out from the layout's definition."""
    from treeattn_b200.paged import PagedKV
    P = 32
    c = PagedKV.__new__(PagedKV)
    c.page, c.head_dim = P, dh
    x = torch.arange(P * dh)
    K, V = c._keys(x), c._values(x)
    E, M = min(16, dh // 4), min(2, dh // 16)
    at = 0
    for s in range(P // 16):
        for h in range(dh // (4 * E)):
            for r in range(2):
                for g in range(8):
                    for t in range(4):
                        for e in range(E):
                            assert K[16 * s + 8 * r + g, h * 4 * E + t * E + e] == at
                            at += 1
    at = 0
    for s in range(P // 16):
        for cc in range(dh // (16 * M)):
            for g in range(8):
                for t in range(4):
                    for m in range(M):
                        for r in range(2):
                            for kh in range(2):
                                for lo in range(2):
                                    assert V[16 * s + 8 * kh + 2 * t + lo, (cc * M + m) * 16 + 8 * r + g] == at
                                    at += 1


def test_rotation_table():
    from treeattn_b200.paged import rotation_table
    cos, sin = rotation_table(50, 8, device='cpu')
    assert cos.shape == sin.shape == (50, 4) and cos.dtype == torch.float32
    assert torch.allclose(cos.double() ** 2 + sin.double() ** 2, torch.ones(50, 4).double(), atol=1e-6)
    assert cos[0].eq(1).all() and abs(float(sin[7, 0]) - 0.6569865987187891) < 1e-7


def test_append_refuses_unaligned_queries_and_tables():
    """Where queries and rotation tables are read in 16-byte pieces (rotations by multiples of 16 dims, none included), a row or
    a table off that boundary is refused before any launch; k and v always."""
    from treeattn_b200 import _lib
    lib = _lib.load()
    a = 1 << 20  # an aligned address that is never dereferenced

    def append(rot=64, q=a, q_sr=512, q_sh=64, qo=a, cos=a, sin=a, k=a, k_sr=256):
        return lib.ta_paged_append(a, a, a, 3, 9, 3, 16, 2, 2, 4, 64, k, a, k_sr, 64, 256, 64, 2, a, a, 1, cos, sin, 100, rot,
                                   q, 8, q_sr, q_sh, qo, None)

    for kw, what in ((dict(q=a + 2), 'q and q_out'), (dict(q_sr=513), 'q and q_out'), (dict(q_sh=68), 'q and q_out'),
                     (dict(qo=a + 2), 'q and q_out'), (dict(cos=a + 4), 'tables'), (dict(sin=a + 8), 'tables'),
                     (dict(rot=0, q=a + 2, cos=None, sin=None), 'q and q_out'), (dict(rot=32, qo=a + 8), 'q and q_out'),
                     (dict(rot=24, k=a + 2), 'k and v'), (dict(k_sr=260), 'k and v')):
        assert append(**kw) == _lib.TA_ERR_ARG, kw
        assert 'ta_paged_append' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())


class _Gpu(torch.Tensor):
    """A host tensor that says it is on a GPU: what the checks of a call let through, with no call made."""
    is_cuda = property(lambda self: True)


def _gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


def _stub_cache(monkeypatch):
    """A cache of 2 sequences (2 kv heads of 64, 16-token pages) whose calls end at the C entry point, which is recorded."""
    from treeattn_b200 import paged
    calls = []
    monkeypatch.setattr(paged, '_call', lambda name, *args: calls.append(name))
    monkeypatch.setattr(paged, '_stream', lambda t: 0)
    cache = paged.PagedKV(_gpu(5, 2, 2 * 16 * 64 + 16, dtype=torch.uint8), _gpu(2, 2, 2, 2, 16 * 64),
                          _gpu(2, 4, dtype=torch.int32), 16, 64)
    return paged, cache, calls


def test_host_buffers_are_refused_before_the_call(monkeypatch):
    """Outputs and scratch in host memory, and a workspace with gaps, never reach a kernel."""
    paged, cache, calls = _stub_cache(monkeypatch)
    start, pos = _gpu(3, dtype=torch.int32), _gpu(2, dtype=torch.int32)
    k, q = _gpu(2, 2, 64), _gpu(2, 4, 64)
    rot = (_gpu(8, 32, dtype=torch.float32), _gpu(8, 32, dtype=torch.float32))
    ws = _gpu(1 << 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match='paged_append.*CUDA'):
        paged.paged_append(cache, k, k, start, pos, 1, q=q, rotation=rot, q_out=torch.zeros(2, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='paged_attn.*CUDA'):
        paged.paged_attn(cache, q, start, pos, 1, ws=ws, lse=torch.zeros(2, 4))
    with pytest.raises(ValueError, match='paged_attn.*CUDA'):
        paged.paged_attn(cache, q, start, pos, 1, ws=torch.zeros(1 << 16, dtype=torch.uint8))
    with pytest.raises(ValueError, match='ws must be contiguous'):
        paged.paged_attn(cache, q, start, pos, 1, ws=ws[::2])
    assert calls == []
    paged.paged_append(cache, k, k, start, pos, 1, q=q, rotation=rot, q_out=_gpu(2, 4, 64))
    paged.paged_attn(cache, q, start, pos, 1, ws=ws, lse=_gpu(2, 4, dtype=torch.float32))
    assert calls == ['ta_paged_append', 'ta_paged_attn']
