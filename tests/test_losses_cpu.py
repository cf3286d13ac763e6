"""CPU checks of the losses: what the entry points and their Python refuse before any CUDA call."""
import ctypes

import pytest
import torch


def test_rejected_arguments_without_gpu():
    from treeattn_b200 import _lib
    lib = _lib.load()
    a = 1 << 20
    f = ctypes.c_float

    def logp(z=a, dtype=1, B=2, T=3, V=100, tokens=a, tau=1.0, out=a, stats=a):
        return lib.ta_token_logp(z, dtype, 300, 100, B, T, V, tokens, 3, 1, f(tau), out, stats, None)

    for kw, what in ((dict(z=None), 'null'), (dict(tokens=None), 'null'), (dict(dtype=5), 'dtype'), (dict(V=0), 'bad sizes'),
                     (dict(V=524289), 'bad sizes'), (dict(B=-1), 'bad sizes'), (dict(B=1 << 20, T=1 << 8), 'bad sizes'),
                     (dict(tau=0.0), 'temperature'), (dict(tau=-1.0), 'temperature'), (dict(tau=float('nan')), 'temperature'),
                     (dict(tau=float('inf')), 'temperature'), (dict(tau=1e-42), 'temperature'), (dict(tau=4e-39), 'temperature'), (dict(out=None), 'null'),
                     (dict(stats=None), 'null')):
        assert logp(**kw) == _lib.TA_ERR_ARG
        assert 'ta_token_logp' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())
    assert logp(B=0) == _lib.TA_OK

    def loss(rows=(a, a, a, a), kl=0.1, lo=0.8, hi=1.2, out=a, by=True, stats=a, V=100):
        ptr = (ctypes.c_void_p * 4)(*rows) if by else None
        st = (ctypes.c_int64 * 8)(*[1] * 8)
        return lib.ta_policy_loss(a, 1, 300, 100, 2, 3, V, a, 3, 1, ptr, st, f(1 / 6), f(lo), f(hi), f(kl), f(1.0), out, a, stats,
                                  None, 0, 0, None)

    for kw, what in ((dict(rows=(None, a, a, a)), 'null'), (dict(rows=(a, None, a, a)), 'null'), (dict(rows=(a, a, None, a)), 'null'),
                     (dict(by=False), 'null'), (dict(out=None), 'null'), (dict(stats=None), 'null'), (dict(lo=1.1), 'clipped'),
                     (dict(hi=0.9), 'clipped'), (dict(lo=float('nan')), 'clipped'), (dict(kl=float('inf')), 'KL'),
                     (dict(V=1 << 20), 'bad sizes')):
        assert loss(**kw) == _lib.TA_ERR_ARG
        assert 'ta_policy_loss' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())

    def grad(stats=a, slope=a, out=a, tau=1.0):
        return lib.ta_logits_grad(a, 1, 300, 100, 2, 3, 100, a, 3, 1, stats, slope, 3, 1, f(1.0), f(tau), None, 0, out, 300, 100, None)

    for kw, what in ((dict(stats=None), 'null'), (dict(slope=None), 'null'), (dict(out=None), 'null'), (dict(tau=0.0), 'temperature')):
        assert grad(**kw) == _lib.TA_ERR_ARG
        assert 'ta_logits_grad' in _lib.last_error() and what in _lib.last_error(), (kw, _lib.last_error())


def test_refused_tensors():
    from treeattn_b200.losses import policy_loss, token_logp
    z, y, r = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for kw, kind, what in ((dict(logits=z.double()), TypeError, 'float32'), (dict(logits=z[0, 0]), ValueError, 'rows'),
                           (dict(logits=z.transpose(1, 2)), ValueError, 'contiguous'), (dict(tokens=y.int()), ValueError, 'int64'),
                           (dict(tokens=y[:1]), ValueError, 'int64'), (dict(), ValueError, 'CUDA')):
        args = dict(dict(logits=z, tokens=y), **kw)
        with pytest.raises(kind, match='token_logp.*' + what):
            token_logp(**args)
        with pytest.raises(kind, match='policy_loss.*' + what):
            policy_loss(old_logp=r, advantages=r, **args)
    with pytest.raises(ValueError, match='ref_logp'):
        policy_loss(z, y, r, r, kl=0.1)
    with pytest.raises(ValueError, match='clip'):
        policy_loss(z, y, r, r, clip=(-0.1, 0.2))
    with pytest.raises(ValueError, match='clip'):
        policy_loss(z, y, r, r, clip=float('nan'))


def test_forward_mode_is_refused():
    """A tangent would be lost without a word: a dual tensor does not ask for gradients."""
    from torch.autograd import forward_ad
    from treeattn_b200.losses import policy_loss, token_logp
    z, y, r = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    with forward_ad.dual_level():
        dz, dr = forward_ad.make_dual(z, torch.ones_like(z)), forward_ad.make_dual(r, torch.ones_like(r))
        for call in (lambda: token_logp(dz, y), lambda: policy_loss(dz, y, r, r), lambda: policy_loss(z, y, dr, r),
                     lambda: policy_loss(z, y, r, r, ref_logp=dr, kl=0.1), lambda: policy_loss(z, y, r, r, weight=dr)):
            with pytest.raises(NotImplementedError, match='(token_logp|policy_loss).*forward-mode'):
                call()
        with pytest.raises(ValueError, match='CUDA'):  # tensors without a tangent are what they are elsewhere
            token_logp(z, y)
