"""Serving over an 8-bit paged key / value cache: the cache, appending to it with the position rotation, attention over
it for one or several new tokens of each sequence, copies of its pages and sequences, and the verification of drafted tokens.

The reference's engine keeps one fp32 tensor per sequence and decodes one token at a time (engine.py:74-81, 149-177); these
operators are the dense model's side of speculative decoding: the segment-tree Decoder drafts, the dense model verifies
(speculative.py runs the two together). Like every entry point of this package they take CUDA tensors, check them, and
enqueue on the current stream without synchronising."""
import array
import ctypes
import math

import torch

from . import _lib
from ._ops import _DT, _need_cuda, _p

PAGE_SIZES = (16, 32, 64)


class PagedKV:
    """The cache of one layer: the tensors that the kernels read and write (include/treeattn_b200.h has the layout).

    pool (n_pages, n_kv_head, 2 * page * head_dim + 16) uint8: a record per (page, kv head): e4m3 codes of the keys, of the
    values, their two fp32 scales, the mark of a page of zeros. tail (batch, n_kv_head, 2, 2, page * head_dim) bf16 or f16:
    the open page of each sequence and the one before it. table (batch, max_pages) int32: the pool page of each page of a
    sequence (several layers may share one). PagedKV.empty allocates pool and tail."""
    __slots__ = ('pool', 'tail', 'table', 'page', 'head_dim')

    def __init__(self, pool, tail, table, page, head_dim):
        self.pool, self.tail, self.table, self.page, self.head_dim = pool, tail, table, int(page), int(head_dim)
        n = self.page * self.head_dim
        if self.page not in PAGE_SIZES:
            raise ValueError('PagedKV: pages of 16, 32 or 64 tokens (got %d)' % self.page)
        shape = pool.shape
        if pool.dtype is not torch.uint8 or len(shape) != 3 or shape[2] != 2 * n + 16:
            raise ValueError('PagedKV: pool must be (n_pages, n_kv_head, 2 * page * head_dim + 16) uint8')
        tshape = tail.shape
        if len(tshape) != 5 or tshape[1:] != (shape[1], 2, 2, n):
            raise ValueError('PagedKV: tail must be (batch, n_kv_head, 2, 2, page * head_dim)')
        if tail.dtype is not torch.bfloat16 and tail.dtype is not torch.float16:
            raise TypeError('PagedKV: the tail holds bfloat16 or float16 (got %s)' % tail.dtype)
        if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != tshape[0] or (
                table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError('PagedKV: table must be (batch, max_pages) int32 with unit inner stride')
        if not (pool.is_contiguous() and tail.is_contiguous()):
            raise ValueError('PagedKV: pool and tail must be contiguous')
        if not (pool.is_cuda and tail.is_cuda and table.is_cuda):
            _need_cuda('PagedKV', pool, tail, table)

    @classmethod
    def empty(cls, n_pages, n_kv_head, head_dim, table, page=64, dtype=torch.bfloat16):
        dev = table.device
        return cls(torch.zeros(n_pages, n_kv_head, 2 * page * head_dim + 16, device=dev, dtype=torch.uint8),
                   torch.zeros(table.shape[0], n_kv_head, 2, 2, page * head_dim, device=dev, dtype=dtype), table, page,
                   head_dim)

    @property
    def n_kv_head(self):
        return self.pool.shape[1]

    def _keys(self, x):
        P, dh = self.page, self.head_dim
        E = min(16, dh // 4)
        d = x.dim() - 1
        return x.unflatten(-1, (P // 16, dh // (4 * E), 2, 8, 4, E)).permute(
            *range(d), d, d + 2, d + 3, d + 1, d + 4, d + 5).reshape(*x.shape[:-1], P, dh)

    def _values(self, x):
        P, dh = self.page, self.head_dim
        M = min(2, dh // 16)
        d = x.dim() - 1
        return x.unflatten(-1, (P // 16, dh // (16 * M), 8, 4, M, 2, 2, 2)).permute(
            *range(d), d, d + 6, d + 3, d + 7, d + 1, d + 4, d + 5, d + 2).reshape(*x.shape[:-1], P, dh)

    def read(self, b, length):
        """Keys and values (n_kv_head, length, head_dim) fp32 of sequence b's first `length` positions, as attention sees
        them: full pages from the codes, the rest from the tail."""
        P, n = self.page, self.page * self.head_dim
        full = length // P
        rec = self.pool[self.table[b, :full].long()]
        codes = rec[..., :2 * n].view(torch.float8_e4m3fn)
        scale = rec[..., 2 * n:2 * n + 8].contiguous().view(torch.float32)
        out = []
        for i, order in enumerate((self._keys, self._values)):
            x = order(codes[..., i * n:(i + 1) * n]).float() * scale[..., i, None, None]
            x = x.transpose(0, 1).reshape(self.n_kv_head, full * P, self.head_dim)
            rest = order(self.tail[b, :, full % 2, i])[:, :length - full * P].float()
            out.append(torch.cat([x, rest], 1))
        return out


class PagePool:
    """Which pages of a pool are free, and the table of those that are not: host bookkeeping for a batch of sequences. The
    device table is updated by one small copy when a sequence's pages change.

    Full pages may be shared: fork lets a sequence go on from another's positions. refs[p] counts the sequences that hold page p."""

    def __init__(self, n_pages, batch, max_pages, page, device='cuda'):
        self.page, self.n_pages, self.max_pages = int(page), int(n_pages), int(max_pages)
        self.free = list(range(n_pages - 1, -1, -1))
        self.refs = [0] * self.n_pages
        self.extra = 0  # holders beyond each page's first: 0 where nothing is shared
        self.owned = [[] for _ in range(batch)]
        self.host = torch.zeros(batch, max_pages, dtype=torch.int32)
        self.table = torch.zeros(batch, max_pages, device=device, dtype=torch.int32)

    def _take(self, b, at):
        page = self.free.pop()
        self.refs[page] = 1
        self.host[b, at] = page
        return page

    def _drop(self, pages):
        for p in reversed(pages):
            self.refs[p] -= 1
            if self.refs[p]:
                self.extra -= 1
            else:
                self.free.append(p)

    def reserve(self, lengths, pos=None):
        """Makes room for lengths[b] positions of each sequence b (a list; shorter ones keep what they have). pos: the position
        that each sequence will write next. From its page on the sequence gets pages of its own where it shares them (what a page
        that is not full holds is in the tail, so nothing is copied); needed where sequences are forked and cut back. Raises
        MemoryError, with nothing changed, when the pool has too few free pages."""
        need = [max(0, -(-int(n) // self.page) - len(o)) for n, o in zip(lengths, self.owned)]
        for n, k in zip(lengths, need):
            if -(-int(n) // self.page) > self.max_pages:
                raise ValueError('PagePool: %d positions above the %d of a sequence' % (n, self.max_pages * self.page))
        shared, left = [], {}
        for b, at in enumerate(() if pos is None or not self.extra else pos):
            own = self.owned[b]
            for j in range(int(at) // self.page, len(own)):
                n = left.get(own[j], self.refs[own[j]])
                if n > 1:  # the last holder of a page keeps it
                    left[own[j]] = n - 1
                    shared.append((b, j))
        if sum(need) + len(shared) > len(self.free):
            raise MemoryError('PagePool: %d pages wanted, %d free' % (sum(need) + len(shared), len(self.free)))
        self.extra -= len(shared)
        for b, j in shared:
            self.refs[self.owned[b][j]] -= 1
            self.owned[b][j] = self._take(b, j)
        for b, k in enumerate(need):
            for _ in range(k):
                self.owned[b].append(self._take(b, len(self.owned[b])))
        if shared or any(need):
            self.table.copy_(self.host)

    def release(self, b):
        """Gives sequence b's pages back (those that no other sequence holds become free)."""
        self._drop(self.owned[b])
        self.owned[b] = []

    def _forked(self, src, dst, lengths):
        """Checks a fork's lists; the pages that each destination is to hold."""
        B = len(self.owned)
        src, dst, lengths = [[int(i) for i in x] for x in (src, dst, lengths)]
        if not len(src) == len(dst) == len(lengths):
            raise ValueError('PagePool.fork: %d sources, %d destinations, %d lengths' % (len(src), len(dst), len(lengths)))
        if any(not 0 <= b < B for b in (*src, *dst)) or len(set(dst)) != len(dst):
            raise ValueError('PagePool.fork: sequences in [0, %d), each a destination once' % B)
        new = {}
        for s, d, n in zip(src, dst, lengths):
            full = n // self.page
            if n < 0 or full > len(self.owned[s]):
                raise ValueError('PagePool.fork: sequence %d does not hold %d positions' % (s, n))
            if s != d:
                new[d] = self.owned[s][:full]
        return new

    def fork(self, src, dst, lengths):
        """Sequence dst[i] goes on from the first lengths[i] positions of sequence src[i], for all i at once (a sequence may be a
        source and a destination): it shares the full pages among them, and what dst[i] held is given back. The open pages, which
        live in the caches' tails, are paged_fork's to copy."""
        self._share(self._forked(src, dst, lengths))

    def _share(self, new):
        for pages in new.values():
            self.extra += len(pages)
            for p in pages:
                self.refs[p] += 1
        for d, pages in new.items():
            self._drop(self.owned[d])
            self.owned[d] = pages
            self.host[d, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        if new:
            self.table.copy_(self.host)

    def compact(self, n_pages=None):
        """Shrinks the pool to its first n_pages pages (default: as many as are held): returns (src, dst), the pages to move, for
        paged_copy on every cache of the pool before anything else touches them. Raises MemoryError, with nothing changed, when
        more pages than that are held."""
        held = self.n_pages - len(self.free)
        n_pages = max(held, 1) if n_pages is None else int(n_pages)
        if not max(held, 1) <= n_pages <= self.n_pages:
            raise MemoryError('PagePool: %d pages held, of %d, cannot become %d' % (held, self.n_pages, n_pages))
        src = [p for p in range(n_pages, self.n_pages) if self.refs[p]]
        free = sorted((p for p in self.free if p < n_pages), reverse=True)
        dst = [free.pop() for _ in src]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d] = self.refs[s]
        for b, own in enumerate(self.owned):
            own[:] = [to.get(p, p) for p in own]
            self.host[b] = 0  # (a row's places beyond its pages may name pages that are gone)
            self.host[b, :len(own)] = torch.tensor(own, dtype=torch.int32)
        self.refs, self.free, self.n_pages = self.refs[:n_pages], free, n_pages
        self.table.copy_(self.host)
        return src, dst


def rotation_table(n_pos, rot, base=10000.0, device='cuda'):
    """(cos, sin) (n_pos, rot / 2) fp32 of the angles pos * base^(-2 i / rot), formed in 64 bits."""
    if rot < 2 or rot % 2:
        raise ValueError('rotation_table: rot must be even and positive (got %d)' % rot)
    f = base ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    a = torch.arange(n_pos, device=device, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


# A decode step's calls take a few microseconds on the GPU: the checks below ask each tensor once, the entry points are looked
# up once, the current stream is read without building a torch Stream object (2.3 -> 0.2 us), and outputs are allocated like
# an input (2.4 -> 1.4 us).
_entry = {}


def _call(name, *args):
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    if fn(*args) != _lib.TA_OK:
        raise _lib.TreeAttnError('%s: %s' % (name, _lib.last_error()))


def _stream(t):
    return torch._C._cuda_getCurrentRawStream(t.get_device())


class _Here:
    """Nothing to do: the tensors' device is the current one."""

    def __enter__(self):
        pass

    def __exit__(self, *e):
        pass


_here = _Here()


def _on(t):
    """Makes t's device the current one for a call, where it is not."""
    return _here if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _rows(name, cache, start, pos):
    if start.dtype is not torch.int32 or pos.dtype is not torch.int32 or not (start.is_contiguous() and pos.is_contiguous()):
        raise TypeError('%s: start and pos must be contiguous int32' % name)
    B = cache.table.shape[0]
    if start.shape != (B + 1,) or pos.shape != (B,):
        raise ValueError('%s: start (batch + 1,) and pos (batch,) for the cache\'s %d sequences' % (name, B))
    if not (start.is_cuda and pos.is_cuda):
        _need_cuda(name, start, pos)
    return B


def _heads(name, cache, x, dtype):
    """Checks rows (n, heads, head_dim) and returns their shape and strides."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != cache.head_dim:
        raise ValueError('%s: rows must be (n, heads, %d)' % (name, cache.head_dim))
    if x.dtype is not dtype:
        raise TypeError('%s: %s rows for a cache with a %s tail' % (name, x.dtype, dtype))
    if stride[2] != 1:
        raise ValueError('%s: the innermost (head) dimension must be contiguous' % name)
    if not x.is_cuda:
        _need_cuda(name, x)
    return shape, stride


def paged_append(cache, k, v, start, pos, max_new, q=None, rotation=None, q_out=None):
    """Puts new rows into the cache: sequence b's rows [start[b], start[b + 1]) of k and v (n, n_kv_head, head_dim) (any row
    and head strides that keep rows 16-byte aligned; q and the tables too where they rotate by multiples of 16 dims) go to
    positions pos[b], pos[b] + 1, .... `max_new` bounds the rows of one sequence. rotation = (cos, sin)
    (rotation_table) turns the first dims of k, and of q (n, n_head, head_dim) into q_out (allocated here when not given).
    Without a rotation q is returned as it is (a given q_out gets a copy). A page is quantised when its last token arrives;
    afterwards a sequence may be cut back to any length whose page is the last or last but one that was ever written."""
    pool, tail, table = cache.pool, cache.tail, cache.table
    dt = tail.dtype
    B = _rows('paged_append', cache, start, pos)
    kshape, ks = _heads('paged_append', cache, k, dt)
    vshape, vs = _heads('paged_append', cache, v, dt)
    n, H, dh = kshape
    n_pages, n_kv, _ = pool.shape
    if H != n_kv or vshape != kshape:
        raise ValueError('paged_append: k and v must be (n, %d, %d)' % (n_kv, dh))
    cos = sin = qp = qo = None
    rot = n_pos = Hq = qr = qh = 0
    if rotation is not None:
        cos, sin = rotation
        if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.shape != sin.shape or cos.dim() != 2 or
                not (cos.is_contiguous() and sin.is_contiguous())):
            raise ValueError('paged_append: rotation must be two contiguous fp32 tables (positions, rot / 2)')
        if not (cos.is_cuda and sin.is_cuda):
            _need_cuda('paged_append', cos, sin)
        n_pos, rot = cos.shape
        rot *= 2
        cos, sin = cos.data_ptr(), sin.data_ptr()
    if q is not None:
        qshape, qs = _heads('paged_append', cache, q, dt)
        if qshape[0] != n:
            raise ValueError('paged_append: q has %d rows, k %d' % (qshape[0], n))
        if rot or q_out is not None:
            Hq, qr, qh = qshape[1], qs[0], qs[1]
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            elif q_out.shape != qshape or q_out.dtype is not dt or not q_out.is_contiguous():
                raise ValueError('paged_append: q_out must be contiguous, of q\'s shape and type')
            elif not q_out.is_cuda:
                _need_cuda('paged_append', q_out)
            qp, qo = q.data_ptr(), q_out.data_ptr()
        else:
            q_out = q
    _call('ta_paged_append', pool.data_ptr(), tail.data_ptr(), table.data_ptr(), table.stride(0), n_pages, table.shape[1],
          cache.page, _DT[dt], B, H, dh, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], n, start.data_ptr(),
          pos.data_ptr(), max_new, cos, sin, n_pos, rot, qp, Hq, qr, qh, qo, _stream(k))
    return q_out


def _records(name, caches, src, dst, of, per_record):
    """One ta_record_copy over the caches' buffers; src and dst are whole numbers on the host."""
    bufs = [of(c) for c in caches]
    if not bufs:
        raise ValueError('%s: no caches' % name)
    first = bufs[0]
    shape, dt, dev = first.shape, first.dtype, first.get_device()
    for b in bufs:
        if b.shape != shape or b.dtype is not dt or b.get_device() != dev:
            raise ValueError('%s: the caches must be alike, and on one device' % name)
    src, dst = [x.tolist() if torch.is_tensor(x) or hasattr(x, 'tolist') else x for x in (src, dst)]
    if len(src) != len(dst):
        raise ValueError('%s: %d sources, %d destinations' % (name, len(src), len(dst)))
    if not len(src):
        return
    try:
        moves = array.array('i', src), array.array('i', dst)
    except (TypeError, OverflowError):
        raise ValueError('%s: sources and destinations must be whole numbers of 32 bits' % name) from None
    _need_cuda(name, first)
    ptrs = (ctypes.c_void_p * len(bufs))(*[b.data_ptr() for b in bufs])
    with _on(first):
        _call('ta_record_copy', ptrs, len(bufs), per_record(first), first.shape[0], moves[0].buffer_info()[0],
              moves[1].buffer_info()[0], len(src), _stream(first))


def paged_copy(caches, src, dst):
    """Copies page src[i] of the pool to page dst[i], for all i at once (every page is read before any is written: chains and cycles
    of pages are fine; no page is written twice), in all caches (PagedKV of one shape, one per layer) by one launch. src and dst
    are whole numbers on the host (lists, PagePool.compact's): a captured call repeats the same moves."""
    _records('paged_copy', caches, src, dst, lambda c: c.pool, lambda t: t.shape[1] * t.shape[2])


def paged_fork(caches, src, dst):
    """Copies what sequence src[i] holds in 16 bits, its open page and the one before it, to sequence dst[i], for all i at once, in all
    caches: what PagePool.fork leaves to do when a sequence goes on in another's slot (samples of one prompt, beams). src and
    dst as paged_copy's."""
    _records('paged_fork', caches, src, dst, lambda c: c.tail, lambda t: t.shape[1] * t.shape[2] * t.shape[3] * t.shape[4] * 2)


def _workspace_bytes(batch, n_head, n_kv_head, head_dim, max_new):
    return max(_lib.load().ta_paged_attn_workspace(int(batch), int(n_head), int(n_kv_head), int(head_dim), int(max_new)), 16)


def paged_attn_workspace(batch, n_head, n_kv_head, head_dim, max_new, device='cuda'):
    """A zeroed workspace for paged_attn at these sizes: one per stream of calls, kept by the caller. Calls of other sizes
    may share it when it is large enough for each."""
    return torch.zeros(_workspace_bytes(batch, n_head, n_kv_head, head_dim, max_new), device=device, dtype=torch.uint8)


def paged_attn(cache, q, start, pos, max_new, scale=None, window=0, out=None, lse=None, ws=None):
    """Attention of new rows q (n, n_head, head_dim) over the cache, after paged_append has put the same rows into it: query
    i of sequence b sees the positions up to pos[b] + i (its last `window` ones when window > 0). n_head is a multiple of the
    cache's kv heads. Returns out (n, n_head, head_dim) in q's type; rows of no sequence are left as they are. lse (n, n_head)
    fp32, when given, receives the natural logarithm of each row's sum of exponentials. ws: a workspace of
    paged_attn_workspace that the caller keeps (allocated for the call when not given)."""
    pool, tail, table = cache.pool, cache.tail, cache.table
    dt = tail.dtype
    B = _rows('paged_attn', cache, start, pos)
    qshape, qs = _heads('paged_attn', cache, q, dt)
    n, Hq, dh = qshape
    n_pages, H, _ = pool.shape
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        os = (Hq * dh, dh)
    else:
        oshape, os = _heads('paged_attn', cache, out, dt)
        if oshape != qshape:
            raise ValueError('paged_attn: out must have q\'s shape')
    if lse is not None and (lse.shape != (n, Hq) or lse.dtype is not torch.float32 or not lse.is_contiguous()):
        raise ValueError('paged_attn: lse must be (n, n_head) fp32, contiguous')
    if ws is None:
        ws = paged_attn_workspace(B, Hq, H, dh, max_new, q.device)
    elif not ws.is_contiguous():
        raise ValueError('paged_attn: ws must be contiguous')
    if not (ws.is_cuda and (lse is None or lse.is_cuda)):
        _need_cuda('paged_attn', ws, lse)
    _call('ta_paged_attn', pool.data_ptr(), tail.data_ptr(), table.data_ptr(), table.stride(0), n_pages, table.shape[1],
          cache.page, _DT[dt], B, Hq, H, dh, q.data_ptr(), qs[0], qs[1], n, start.data_ptr(), pos.data_ptr(), max_new,
          1.0 / math.sqrt(dh) if scale is None else scale, window, out.data_ptr(), os[0], os[1], _p(lse), ws.data_ptr(),
          ws.nbytes, _stream(q))
    return out


def verify_drafts(p, q, drafts, u, n_draft=None):
    """Which drafted tokens stand, and the token that follows them. p (B, G + 1, V) the target's probabilities after each
    prefix, q (B, G, V) those the drafts were drawn from (fp32, bf16 or f16; any outer strides), drafts (B, G) int64, u
    (B, G + 1) fp32 uniform in [0, 1) (one for each draft, the last for the draw), n_draft (B,) int32 the drafts of each sequence (all G when None). Returns tokens
    (B, G + 1) int64 - the drafts that stand, the token drawn after them, then -1 - and accepted (B,) int32. The output is
    distributed as sampling from p, whatever q is."""
    pshape, qshape, ps, qs, dt = p.shape, q.shape, p.stride(), q.stride(), p.dtype
    if len(qshape) != 3 or pshape != (qshape[0], qshape[1] + 1, qshape[2]):
        raise ValueError('verify_drafts: p (B, G + 1, V) and q (B, G, V)')
    B, G, V = qshape
    if dt is not q.dtype or dt not in _DT:
        raise TypeError('verify_drafts: p and q must share float32, bfloat16 or float16')
    if ps[2] != 1 or (G and qs[2] != 1):
        raise ValueError('verify_drafts: the innermost (vocabulary) dimension must be contiguous')
    if drafts.shape != (B, G) or drafts.dtype is not torch.int64 or not drafts.is_contiguous():
        raise ValueError('verify_drafts: drafts must be (B, G) int64, contiguous')
    if u.shape != (B, G + 1) or u.dtype is not torch.float32 or not u.is_contiguous():
        raise ValueError('verify_drafts: u must be (B, G + 1) fp32, contiguous')
    if n_draft is not None and (n_draft.shape != (B,) or n_draft.dtype is not torch.int32 or not n_draft.is_contiguous()):
        raise ValueError('verify_drafts: n_draft must be (B,) int32, contiguous')
    if not (p.is_cuda and q.is_cuda and drafts.is_cuda and u.is_cuda and (n_draft is None or n_draft.is_cuda)):
        _need_cuda('verify_drafts', p, q, drafts, u, n_draft)
    tokens = torch.empty_like(u, dtype=torch.int64)
    accepted = u.new_empty((B,), dtype=torch.int32) if n_draft is None else torch.empty_like(n_draft)
    _call('ta_verify_drafts', p.data_ptr(), ps[0], ps[1], q.data_ptr(), qs[0], qs[1], _DT[dt], B, G, V, drafts.data_ptr(),
          u.data_ptr(), _p(n_draft), tokens.data_ptr(), accepted.data_ptr(), _stream(p))
    return tokens, accepted
