"""CPU checks of the adapters: what the entry points and their Python refuse before any CUDA call."""
import pytest
import torch


def test_rejected_arguments_without_gpu():
    from treeattn_b200 import _lib
    lib = _lib.load()
    p = 1 << 20

    def add(y=p, ysr=64, x=p, xsr=128, a=p, b=p, dtype=1, na=3, K=128, N=64, r=16, n=9, start=p, which=p, B=2, new=4, out=p + 4096,
            osr=64, t=None):
        return lib.ta_adapter_add(y, ysr, x, xsr, a, b, None, dtype, na, K, N, r, n, start, which, B, new, out, osr, t, None)

    for kw, what in ((dict(dtype=0), 'dtype'), (dict(r=4), 'rank'), (dict(r=20), 'rank'), (dict(r=136), 'rank'), (dict(K=12), 'multiples of 8'),
                     (dict(N=0), 'multiples of 8'), (dict(na=0), 'bad sizes'), (dict(n=-1), 'bad sizes'), (dict(B=-1), 'bad sizes'),
                     (dict(B=65535), 'bad sizes'), (dict(new=-1), 'bad sizes'), (dict(start=None), 'null'), (dict(which=None), 'null'),
                     (dict(x=None), 'null'), (dict(y=None), 'null'), (dict(a=None), 'null'), (dict(out=None), 'null'),
                     (dict(x=p + 8), 'aligned'), (dict(xsr=132), 'aligned'), (dict(ysr=68), 'aligned'), (dict(osr=1), 'aligned'),
                     (dict(b=p + 2), 'aligned'), (dict(new=17), 't is needed'), (dict(new=17, t=p + 8), 't is needed'), (dict(out=p, osr=72), 'strides')):
        assert add(**kw) == _lib.TA_ERR_ARG
        assert 'ta_adapter_add' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())
    assert add(n=0) == _lib.TA_OK

    def bwd(dy=p, x=p, a=p, t=p, u=p, dx=p, da=p, db=p, r=16, xsr=128):
        return lib.ta_adapter_bwd(dy, 64, x, xsr, a, p, None, 3, 128, 64, r, 9, p, p, 2, 4, t, u, dx, 128, da, db, None)

    for kw, what in ((dict(dy=None), 'null'), (dict(x=None), 'null'), (dict(t=None), 'null'), (dict(u=None), 'null'), (dict(a=None), 'null'),
                     (dict(dx=p + 8), 'aligned'), (dict(da=p + 8), 'aligned'), (dict(db=p + 2), 'aligned'), (dict(xsr=4), 'aligned'), (dict(u=p + 8), 'aligned'), (dict(r=7), 'rank')):
        assert bwd(**kw) == _lib.TA_ERR_ARG
        assert 'ta_adapter_bwd' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())
    assert bwd(dx=None, da=None, db=None) == _lib.TA_OK


def test_refused_tensors():
    from treeattn_b200.adapters import adapter_add
    h = torch.bfloat16
    base = dict(y=torch.zeros(5, 64, dtype=h), x=torch.zeros(5, 32, dtype=h), a=torch.zeros(2, 8, 32, dtype=h),
                b=torch.zeros(2, 64, 8, dtype=h), start=torch.tensor([0, 5], dtype=torch.int32),
                which=torch.zeros(1, dtype=torch.int32), max_new=5, scale=torch.ones(2))
    for kw, kind, what in ((dict(x=base['x'].float()), TypeError, 'float16'), (dict(y=base['y'].half()), TypeError, 'y is'),
                           (dict(x=base['x'].t()), ValueError, 'contiguous columns'), (dict(y=torch.zeros(5, 56, dtype=h)), ValueError, 'fit'),
                           (dict(x=base['x'][:4]), ValueError, 'fit'), (dict(b=torch.zeros(3, 64, 8, dtype=h)), ValueError, 'fit'),
                           (dict(a=base['a'].float()), ValueError, 'type'), (dict(a=base['a'].transpose(1, 2)), ValueError, 'fit'),
                           (dict(b=torch.zeros(2, 8, 64, dtype=h).transpose(1, 2)), ValueError, 'contiguous'),
                           (dict(start=base['start'].long()), TypeError, 'int32'), (dict(which=torch.zeros(2, dtype=torch.int32)), ValueError, 'batch'),
                           (dict(scale=torch.ones(3)), ValueError, 'scale'), (dict(scale=torch.ones(2).half()), ValueError, 'scale'),
                           (dict(), ValueError, 'CUDA')):
        with pytest.raises(kind, match='adapter_add.*' + what):
            adapter_add(**dict(base, **kw))


def test_adapter_set_shapes_and_refusals():
    from treeattn_b200.adapters import AdapterSet
    from treeattn_b200.config import Config
    from treeattn_b200.model import GPT
    s = AdapterSet(3, 2, 64, rank=8, alpha=16, projections=('c_mlp', 'c_attn'), device='cpu')
    assert s.factors(1, 'c_attn')[0].shape == (3, 8, 64) and s.factors(1, 'c_attn')[1].shape == (3, 192, 8)
    assert s.factors(0, 'c_mlp')[0].shape == (3, 8, 256) and s.factors(0, 'c_fc') is None
    assert s.scale.tolist() == [2.0] * 3 and all(not b.any() for b in s.b)
    assert len(list(s.parameters())) == 8
    for kw in (dict(n_adapters=0), dict(rank=12), dict(rank=136), dict(n_embd=60), dict(projections=('c_out',))):
        with pytest.raises(ValueError, match='AdapterSet'):
            AdapterSet(**dict(dict(n_adapters=2, n_layer=1, n_embd=64, device='cpu'), **kw))
    model = GPT(Config(attn='seg', vocab_size=32, seq_len=64, n_layer=1, n_head=2, n_embd=64, chunk=64))
    with pytest.raises(ValueError, match='2 blocks'):
        s.attach(model)
    with pytest.raises(ValueError, match='whole numbers'):
        s.use([0.5])
    s.use([0, -1, 2])
    s.use(None)
    attached = AdapterSet(1, 1, 64, device='cpu').attach(model)
    assert sum(len(m._forward_hooks) for m in model.modules()) == 4
    attached.remove()
    assert sum(len(m._forward_hooks) for m in model.modules()) == 0


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    from treeattn_b200.adapters import adapter_add
    x, y, a, b = [torch.randn(s).to(torch.bfloat16) for s in ((5, 16), (5, 24), (2, 8, 16), (2, 24, 8))]
    start, which = torch.tensor([0, 5], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with forward_ad.dual_level():
        for i in range(4):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate((y, x, a, b))]
            with pytest.raises(NotImplementedError, match='adapter_add.*forward-mode'):
                adapter_add(*args, start, which, 5)
