"""Low-rank adapters of many requests beside one model's projections: the operator, with its gradients, and the sets of adapters that a
model is trained with (GPT) and served with (speculative.PagedDecoder).

The reference has one set of weights. Here a batch's sequences may each name an adapter: a projection W x of its rows then gets
scale (x A^T) B^T added, A (rank, inputs) and B (outputs, rank) of that adapter. The shared projection stays one library product
over all rows; adapter_add adds the rest in one kernel, reading each row of x and of the projection once."""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from ._ops import _DT, _need_cuda, _no_tangents, _p
from .paged import _call, _on, _stream


def _rows(name, what, t, dtype=None):
    """Checks rows (n, columns) that the kernels read in 16-byte pieces."""
    if t.dim() != 2 or t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError('%s: %s must be (rows, columns) with contiguous columns' % (name, what))
    if dtype is not None and t.dtype is not dtype:
        raise TypeError('%s: %s is %s, not %s' % (name, what, t.dtype, dtype))


def _check(name, y, x, a, b, start, which, scale):
    """Checks a call's tensors; returns (adapters, rank, inputs, outputs, rows, batch)."""
    dt, dev = x.dtype, x.get_device()
    (n, K), (m, N), (na, r, ka), bs, (B,), (s,) = _dims(name, y, x, a, b, start, which)
    if (dt is torch.bfloat16 or dt is torch.float16) and y.dtype is dt and a.dtype is dt and b.dtype is dt and m == n and ka == K and (
            bs == (na, N, r)) and s == B + 1 and start.dtype is torch.int32 and which.dtype is torch.int32 and x.stride(1) == 1 and (
            y.stride(1) == 1) and a.is_contiguous() and b.is_contiguous() and start.is_contiguous() and which.is_contiguous() and dev >= 0 and (
            y.get_device() == dev and a.get_device() == dev and b.get_device() == dev and start.get_device() == dev and
            which.get_device() == dev) and (scale is None or scale.dtype is torch.float32 and scale.shape == (na,) and
                                            scale.is_contiguous() and scale.get_device() == dev):
        return na, r, K, N, n, B
    # something does not fit: what
    if dt is not torch.bfloat16 and dt is not torch.float16:
        raise TypeError('%s: bfloat16 or float16 (got %s)' % (name, dt))
    for what, t in (('x', x), ('y', y)):
        _rows(name, what, t, dt)
    if a.dtype is not dt or b.dtype is not dt:
        raise ValueError('%s: a (adapters, rank, inputs) and b (adapters, outputs, rank) of x\'s type' % name)
    if ka != K or bs != (na, N, r) or m != n:
        raise ValueError('%s: x %s, y %s, a %s, b %s do not fit' % (name, tuple(x.shape), tuple(y.shape), tuple(a.shape),
                                                                   tuple(b.shape)))
    if not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError('%s: a and b must be contiguous' % name)
    if start.dtype is not torch.int32 or which.dtype is not torch.int32 or not (start.is_contiguous() and which.is_contiguous()):
        raise TypeError('%s: start and which must be contiguous int32' % name)
    if s != B + 1:
        raise ValueError('%s: which (batch,) and start (batch + 1,)' % name)
    if scale is not None and (scale.dtype is not torch.float32 or scale.shape != (na,) or not scale.is_contiguous()):
        raise ValueError('%s: scale must be (adapters,) float32, contiguous' % name)
    _need_cuda(name, x, y, a, b, start, which, scale)
    for t in (y, a, b, start, which, scale):
        if t is not None and t.get_device() != dev:
            raise ValueError('%s: tensors on one device (got %s and %s)' % (name, x.device, t.device))
    return na, r, K, N, n, B  # (a single column's stride does not matter)


def _dims(name, y, x, a, b, start, which):
    shapes = x.shape, y.shape, a.shape, b.shape, which.shape, start.shape
    if tuple(len(s) for s in shapes) != (2, 2, 3, 3, 1, 1):
        for what, t in (('x', x), ('y', y)):
            _rows(name, what, t)
        if a.dim() != 3 or b.dim() != 3:
            raise ValueError('%s: a (adapters, rank, inputs) and b (adapters, outputs, rank)' % name)
        raise ValueError('%s: which (batch,) and start (batch + 1,)' % name)
    return shapes


def _add(y, x, a, b, start, which, dims, max_new, scale, out, t=None):
    na, r, K, N, n, B = dims
    if t is None and max_new > 16:  # many rows: t goes by way of memory (f16's rows with a factor each)
        t = torch.empty(2 * n * r + (2 * n if x.dtype is torch.float16 else 0), device=x.device, dtype=x.dtype)
    with _on(x):
        _call('ta_adapter_add', y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), a.data_ptr(), b.data_ptr(),
              None if scale is None else scale.data_ptr(), _DT[x.dtype], na, K, N, r, n, start.data_ptr(), which.data_ptr(), B, max_new,
              out.data_ptr(), out.stride(0), None if t is None else t.data_ptr(), _stream(x))
    return out


class _AdapterAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, start, which, dims, max_new, scale, into):
        need = ctx.needs_input_grad
        t = torch.empty(2, x.shape[0], a.shape[1], device=x.device, dtype=x.dtype) if need[3] else None  # what dB needs of x
        if into:
            out = y
            ctx.mark_dirty(y)
        else:
            out = torch.empty_like(y, memory_format=torch.contiguous_format)
        _add(y, x, a, b, start, which, dims, max_new, scale, out, t)
        ctx.save_for_backward(x, a, b, start, which, scale, t)
        ctx.max_new = max_new
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, a, b, start, which, scale, t = ctx.saved_tensors
        need = ctx.needs_input_grad
        n, (na, r, K), N = x.shape[0], a.shape, b.shape[1]
        d = dy
        if d.stride(1) != 1 or d.stride(0) % 8 or d.data_ptr() % 16:
            d = d.clone(memory_format=torch.contiguous_format)
        dx = torch.empty(n, K, device=x.device, dtype=x.dtype) if need[1] else None
        da, db = torch.empty_like(a) if need[2] else None, torch.empty_like(b) if need[3] else None
        u = torch.empty(2, n, r, device=x.device, dtype=x.dtype) if need[1] or need[2] else None
        if need[1] or need[2] or need[3]:
            with _on(x):
                _call('ta_adapter_bwd', d.data_ptr(), d.stride(0), x.data_ptr(), x.stride(0), a.data_ptr(), b.data_ptr(), _p(scale), na,
                      K, N, r, n, start.data_ptr(), which.data_ptr(), which.shape[0], ctx.max_new, _p(t), _p(u), _p(dx),
                      K if dx is None else dx.stride(0), _p(da), _p(db), _stream(x))
        return (dy if need[0] else None, dx, da, db) + (None,) * 6


def adapter_add(y, x, a, b, start, which, max_new, scale=None, out=None):
    """y + scale (x A^T) B^T on the rows of each sequence: sequence i owns rows [start[i], start[i + 1]) of x (n, inputs) and y (n, outputs)
    and takes adapter which[i] of a (adapters, rank, inputs), b (adapters, outputs, rank) and scale (adapters,) float32 (1 when None);
    which[i] = -1: none. bfloat16 or float16; ranks a multiple of 8 up to 128 (adapters of smaller ranks are filled up with zeros);
    inputs and outputs multiples of 8, rows of any stride that keeps them 16-byte aligned. start (batch + 1,) and which (batch,) int32;
    max_new is about the rows of the longest sequence (it sizes the grid; more are done all the same). Rows of no sequence, and of
    sequences without an adapter, are y's. Returns a new tensor, or `out` (y itself: in place; it overlaps nothing else). An adapter outside the
    set gives NaN rows and is recorded (device_error).
    Differentiable in y, x, a and b in bfloat16 (not with an `out` other than y); sequences that share an adapter add to one gradient, in
    one order. t = x A^T is summed in fp32 and multiplied with B as two 16-bit numbers; the sum with y is rounded once."""
    _no_tangents('adapter_add', y, x, a, b, scale)
    dims = _check('adapter_add', y, x, a, b, start, which, scale)
    max_new = int(max_new)
    if out is not None:
        if out.data_ptr() == x.data_ptr() and x.numel():
            raise ValueError('adapter_add: the output in x\'s place')
        if out.dim() == 2 and out.shape[0] > 1 and out.stride(0) < out.shape[1]:
            raise ValueError('adapter_add: rows of the output overlap')
    if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad or
                                    scale is not None and scale.requires_grad or out is not None and out.requires_grad):
        if scale is not None and scale.requires_grad:
            raise ValueError('adapter_add: no gradient of scale')
        if x.dtype is not torch.bfloat16:
            raise TypeError('adapter_add: gradients in bfloat16 only (got %s)' % x.dtype)
        if out is not None and out is not y:
            raise ValueError('adapter_add: no gradient through a given output (other than y itself)')
        return _AdapterAdd.apply(y, x, a, b, start, which, dims, max_new, scale, out is y)
    if out is None:
        return _add(y, x, a, b, start, which, dims, max_new, scale, torch.empty_like(y, memory_format=torch.contiguous_format))
    if out is not y:
        _rows('adapter_add', 'out', out, y.dtype)
        if out.shape != y.shape:
            raise ValueError('adapter_add: out must have y\'s shape')
        _need_cuda('adapter_add', out)
        if out.get_device() != x.get_device():
            raise ValueError('adapter_add: tensors on one device (got %s and %s)' % (x.device, out.device))
    _add(y, x, a, b, start, which, dims, max_new, scale, out)
    torch.autograd.graph.increment_version(out)  # (written through its address: what autograd saved of it before is gone)
    return out


class AdapterSet(nn.Module):
    """Adapters for every block of a model of n_layer blocks of width n_embd: on c_attn, c_proj, c_fc and c_mlp (a subset by
    `projections`). A starts at random, B at 0, so that a fresh adapter changes nothing; scale (adapters,) is alpha / rank.

    Training: attach(model) adds them to a GPT's projections (the model's own weights need no gradient); use(which) says which adapter
    each sequence of the next batches takes. Serving: PagedDecoder(..., adapters=set) and its `which`."""
    SHAPES = dict(c_attn=(1, 3), c_proj=(1, 1), c_fc=(1, 4), c_mlp=(4, 1))  # inputs and outputs, in widths
    MODULES = dict(c_attn='attn.c_attn', c_proj='attn.c_proj', c_fc='mlp.c_fc', c_mlp='mlp.c_proj')

    def __init__(self, n_adapters, n_layer, n_embd, rank=16, alpha=None, projections=('c_attn', 'c_proj', 'c_fc', 'c_mlp'),
                 device='cuda', dtype=torch.bfloat16):
        super().__init__()
        if n_adapters < 1 or rank < 8 or rank > 128 or rank % 8:
            raise ValueError('AdapterSet: %d adapters of rank %d (at least 1, of a multiple of 8 up to 128)' % (n_adapters, rank))
        if n_embd % 8:
            raise ValueError('AdapterSet: width %d (a multiple of 8)' % n_embd)
        unknown = [p for p in projections if p not in self.SHAPES]
        if unknown:
            raise ValueError('AdapterSet: no projection %s' % unknown[0])
        self.n_adapters, self.n_layer, self.n_embd, self.projections = n_adapters, n_layer, n_embd, tuple(projections)
        self.a, self.b = nn.ParameterList(), nn.ParameterList()
        for _ in range(n_layer):
            for p in self.projections:
                i, o = [w * n_embd for w in self.SHAPES[p]]
                self.a.append(nn.Parameter((torch.randn(n_adapters, rank, i, device=device) * i ** -0.5).to(dtype)))
                self.b.append(nn.Parameter(torch.zeros(n_adapters, o, rank, device=device, dtype=dtype)))
        self.register_buffer('scale', torch.full((n_adapters,), (rank if alpha is None else alpha) / rank, device=device))
        self._which, self._start, self._captured = None, {}, {}

    def factors(self, layer, projection):
        """(a, b) of a block's projection, or None where there are none."""
        if projection not in self.projections:
            return None
        i = layer * len(self.projections) + self.projections.index(projection)
        return self.a[i], self.b[i]

    def _starts(self, B, n):
        """Row offsets of n rows a sequence (kept for the lengths that come up most; copied from the host, so that they are there for
        every stream). A graph that is being captured forms its own where there are none."""
        dev = self.scale.device
        key = B, n, dev
        if key not in self._start:
            if dev.type == 'cuda' and torch.cuda.is_current_stream_capturing():
                return torch.arange(B + 1, device=dev, dtype=torch.int32) * n
            if len(self._start) >= 16:
                self._start.clear()
            self._start[key] = self._held((torch.arange(B + 1, dtype=torch.int32) * n).to(dev), made=True)
        return self._held(self._start[key])

    def _held(self, t, made=False):
        """t, which this set may let go while the current stream (another one than it was made on), or a graph that is being captured, still
        reads it."""
        if t.is_cuda:
            if made:
                t.made_on = _stream(t)
            if torch.cuda.is_current_stream_capturing():
                self._captured[t.data_ptr()] = t
            elif getattr(t, 'made_on', None) != _stream(t):
                t.record_stream(torch.cuda.current_stream(t.device))
        return t

    def release_captured(self):
        """Lets go of the adapters and row offsets that captured passes read: once their graphs are no longer replayed. (They are kept
        for the set's life otherwise.)"""
        self._captured.clear()

    def use(self, which):
        """The adapters of the next batches of the attached model: whole numbers, -1 for none (None: no adapters at all). A captured pass
        keeps those that it was captured with."""
        if which is None:
            self._which = None
            return
        which = torch.as_tensor(which)
        if which.dim() != 1 or which.is_floating_point():
            raise ValueError('AdapterSet: which must be whole numbers, one a sequence')
        self._which = self._held(which.to(self.scale.device, torch.int32, copy=True), made=True)

    def _scale(self):
        return self.scale if self.scale.dtype is torch.float32 else self.scale.float()  # (a cast of the whole set casts it too)

    def apply_to(self, y, x, layer, projection, start, which, max_new):
        """Adds a projection's adapters to its rows y, in place."""
        f = self.factors(layer, projection)
        return y if f is None or which is None else adapter_add(y, x, *f, start, which, max_new, scale=self._scale(), out=y)

    def attach(self, model):
        """Adds the adapters to the projections of a GPT (16-bit, on the set's device). Returns a handle whose remove() takes them
        off again."""
        if len(model.blocks) != self.n_layer or model.cfg.n_embd != self.n_embd:
            raise ValueError('AdapterSet: %d blocks of width %d for a model of %d of %d' % (
                self.n_layer, self.n_embd, len(model.blocks), model.cfg.n_embd))
        hooks = []
        for i, block in enumerate(model.blocks):
            for p in self.projections:
                hooks.append(block.get_submodule(self.MODULES[p]).register_forward_hook(self._hook(i, p)))
        return _Attached(hooks)

    def _hook(self, layer, projection):
        def add(module, args, y):
            if self._which is None:
                return None
            x = args[0]
            B, n = x.shape[0], x.shape[1]
            if self._which.shape[0] != B:
                raise ValueError('AdapterSet: adapters for %d sequences, a batch of %d' % (self._which.shape[0], B))
            a, b = self.factors(layer, projection)
            rows = adapter_add(y.reshape(B * n, -1), x.reshape(B * n, -1), a, b, self._starts(B, n), self._held(self._which), n,
                               scale=self._scale())
            return rows.view(y.shape)
        return add


class _Attached:
    def __init__(self, hooks):
        self._hooks = hooks

    def remove(self):
        for h in self._hooks:
            h.remove()
        self._hooks = []
