"""Losses of training on sampled answers, over a vocabulary's logits: the clipped policy loss with its KL term, and the tokens'
log-probabilities, each with the gradient of the logits.

The reference trains on cross entropy alone (model.py:79-93). Here a group of answers is sampled (PagedDecoder.fork, Decoder),
scored, and the model that GPT.forward runs is trained on them: policy_loss takes its logits. Rows are read once; what a loss needs of a row
beside its softmax are a few scalars, so the gradient is formed in the same pass. CUDA tensors only, on the current stream."""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._ops import _DT, _need_cuda, _no_tangents
from .paged import _call, _on, _stream

_V4 = ctypes.c_void_p * 4
_L8 = ctypes.c_int64 * 8


def _logits(name, logits, tokens):
    """Checks logits (..., V) and tokens (...); returns what the entry points ask about them, one or two leading dims as two: (address,
    type, strides (2), b, t, V, the tokens' address and strides (2))."""
    code = _DT.get(logits.dtype)
    if code is None:
        raise TypeError('%s: logits must be float32, bfloat16 or float16 (got %s)' % (name, logits.dtype))
    shape, s, t = logits.shape, logits.stride(), tokens.stride()
    if len(shape) not in (2, 3):
        raise ValueError('%s: logits must be (rows, vocabulary) or (batch, rows, vocabulary)' % name)
    if shape[-1] < 1 or s[-1] != 1:
        raise ValueError('%s: the innermost (vocabulary) dimension must be contiguous' % name)
    if tokens.dtype is not torch.int64 or tokens.shape != shape[:-1]:
        raise ValueError('%s: tokens must be %s int64' % (name, tuple(shape[:-1])))
    dev = logits.get_device()
    if dev < 0 or tokens.get_device() != dev:
        _need_cuda(name, logits, tokens)
        raise ValueError('%s: tensors on one device (got %s and %s)' % (name, logits.device, tokens.device))
    if len(shape) == 3:
        return (logits.data_ptr(), code, s[0], s[1], shape[0], shape[1], shape[2], tokens.data_ptr(), t[0], t[1])
    return (logits.data_ptr(), code, 0, s[0], 1, shape[0], shape[1], tokens.data_ptr(), 0, t[0])


def _by_row(name, what, v, like):
    """Checks a float32 tensor by row and returns its strides."""
    if v.dtype is not torch.float32 or v.shape != like.shape:
        raise ValueError('%s: %s must be %s float32' % (name, what, tuple(like.shape)))
    if v.get_device() != like.get_device():
        _need_cuda(name, v)
        raise ValueError('%s: tensors on one device (got %s and %s)' % (name, like.device, v.device))
    s = v.stride()
    return s if len(s) == 2 else (0, s[0])


def _grad_like(logits):
    """An output that lies in memory as the logits do (their rows then meet 16-byte boundaries alike), without their overlaps."""
    s = logits.stride()
    V = logits.shape[-1]
    dense = s[-2] >= V and (logits.dim() == 2 or s[0] >= s[1] * logits.shape[1])
    # (room between the rows that the logits do not have themselves is not allocated: a slice of a wider tensor is made compact)
    if dense and s[-2] == V and (logits.dim() == 2 or s[0] <= s[1] * (logits.shape[1] + 1)):
        return torch.empty_strided(logits.shape, s, device=logits.device, dtype=logits.dtype)
    return torch.empty_like(logits, memory_format=torch.contiguous_format)


def _grad_strides(g):
    s = g.stride()
    return (s[0], s[1]) if g.dim() == 3 else (0, s[0])


def _logits_grad(logits, of, stats, slope, ss, by, temperature, up, unit_done, grad):
    gs = _grad_strides(grad)
    with _on(logits):
        _call('ta_logits_grad', *of, stats.data_ptr(), slope, ss[0], ss[1], by, temperature, None if up is None else up.data_ptr(),
              int(unit_done), grad.data_ptr(), gs[0], gs[1], _stream(logits))


# ------------------------------------------------------------------------------------------------ log-probabilities
def _token_logp(logits, tokens, temperature):
    of = _logits('token_logp', logits, tokens)
    logp = torch.empty(tokens.shape, device=logits.device, dtype=torch.float32)
    stats = torch.empty(2, of[4] * of[5], device=logits.device, dtype=torch.float32)  # the rows' references and sums
    with _on(logits):
        _call('ta_token_logp', *of, temperature, logp.data_ptr(), stats.data_ptr(), _stream(logits))
    return logp, stats


class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature):
        logp, stats = _token_logp(logits, tokens, temperature)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.temperature = temperature
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp):
        logits, tokens, stats = ctx.saved_tensors
        grad = _grad_like(logits)
        s = dlogp.stride()
        _logits_grad(logits, _logits('token_logp', logits, tokens), stats, dlogp.data_ptr(), s if len(s) == 2 else (0, s[0]),
                     1.0 / ctx.temperature, ctx.temperature, None, False, grad)
        return grad, None, None


def token_logp(logits, tokens, temperature=1.0):
    """log softmax(logits / temperature) at tokens: logits (rows, V) or (batch, rows, V) in float32, bfloat16 or float16 (any outer
    strides), tokens their leading shape, int64. Returns that shape in float32; differentiable in logits (rows whose gradient is 0 get
    zeros, whatever the logits hold). A token outside [0, V) gives NaN and is recorded (device_error)."""
    temperature = float(temperature)
    _no_tangents('token_logp', logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _TokenLogp.apply(logits, tokens, temperature)
    return _token_logp(logits, tokens, temperature)[0]


# ------------------------------------------------------------------------------------------------ policy loss
def _policy(logits, tokens, old_logp, advantages, ref_logp, weight, clip, kl, temperature, with_grad):
    name = 'policy_loss'
    of = _logits(name, logits, tokens)
    o, a = _by_row(name, 'old_logp', old_logp, tokens), _by_row(name, 'advantages', advantages, tokens)
    r = w = (0, 0)
    ref = wp = None
    if ref_logp is not None:
        r, ref = _by_row(name, 'ref_logp', ref_logp, tokens), ref_logp.data_ptr()
    if weight is not None:
        w, wp = _by_row(name, 'weight', weight, tokens), weight.data_ptr()
    dev, n = logits.device, of[4] * of[5]
    loss = torch.empty((), device=dev, dtype=torch.float32)
    logp = torch.empty(tokens.shape, device=dev, dtype=torch.float32)
    stats = torch.empty(4, n, device=dev, dtype=torch.float32)  # the rows' references, sums, slopes and terms
    grad, gp, gs = None, None, (0, 0)
    if with_grad:
        grad = _grad_like(logits)
        gp, gs = grad.data_ptr(), _grad_strides(grad)
    with _on(logits):
        _call('ta_policy_loss', *of, _V4(old_logp.data_ptr(), advantages.data_ptr(), ref, wp),
              _L8(o[0], o[1], a[0], a[1], r[0], r[1], w[0], w[1]), 1.0 / max(n, 1), clip[0], clip[1], kl, temperature, loss.data_ptr(),
              logp.data_ptr(), stats.data_ptr(), gp, gs[0], gs[1], _stream(logits))
    return loss, logp, stats, grad


class _PolicyLoss(torch.autograd.Function):
    """The forward pass also forms the gradient for a factor of 1, and the first backward pass hands it out (formed again, by a
    kernel that asks for the factor on the device, where it is another). float16 waits for the factor, a loss scale, which keeps
    its small gradients from being rounded to 0."""

    @staticmethod
    def forward(ctx, logits, tokens, old_logp, advantages, ref_logp, weight, clip, kl, temperature):
        loss, logp, stats, ctx.grad = _policy(logits, tokens, old_logp, advantages, ref_logp, weight, clip, kl, temperature,
                                                      logits.dtype is not torch.float16)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(logp)
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        if dloss is None:
            return (None,) * 9
        logits, tokens, stats = ctx.saved_tensors
        grad, ctx.grad = ctx.grad, None
        formed = grad is not None
        if not formed:
            grad = _grad_like(logits)
        of = _logits('policy_loss', logits, tokens)
        b, t = of[4], of[5]
        _logits_grad(logits, of, stats, stats.data_ptr() + 8 * b * t, (t, 1), 1.0, ctx.temperature, dloss, formed, grad)
        return (grad,) + (None,) * 8


def policy_loss(logits, tokens, old_logp, advantages, ref_logp=None, weight=None, clip=0.2, kl=0.0, temperature=1.0):
    """The clipped policy loss over sampled tokens, with a KL term towards a reference model:
      rho = exp(logp - old_logp), loss = sum of weight (-min(rho A, clip(rho, 1 - lo, 1 + hi) A) + kl (exp(d) - d - 1)), d = ref_logp - logp
    logits (rows, V) or (batch, rows, V) (float32, bfloat16 or float16; any outer strides: logits[:, :-1] is taken as it is), tokens
    their leading shape, int64; old_logp, advantages, ref_logp (only with kl) and weight of that shape, float32 (expanded ones are
    fine), and without gradients of their own. weight: each token's share (1 / tokens when None). A token of weight 0 does not count: its row gets
    zeros in the gradient and 0 as logp, whatever the logits and the other tensors hold there. clip: lo = hi, or (lo, hi).
    temperature: the one that the tokens were sampled at. Returns loss (scalar float32, differentiable in logits) and logp (the tokens'
    log-probabilities, float32, without gradient). A counted token outside [0, V) makes the loss NaN and is recorded (device_error)."""
    lo, hi = (clip, clip) if not isinstance(clip, (tuple, list)) else clip
    lo, hi, kl, temperature = float(lo), float(hi), float(kl), float(temperature)
    if not (lo >= 0 and hi >= 0):
        raise ValueError('policy_loss: clip %s (not negative)' % (clip,))
    if kl and ref_logp is None:
        raise ValueError('policy_loss: a KL term needs ref_logp')
    _no_tangents('policy_loss', logits, old_logp, advantages, ref_logp, weight)
    if torch.is_grad_enabled():
        for what, v in (('old_logp', old_logp), ('advantages', advantages), ('ref_logp', ref_logp), ('weight', weight)):
            if v is not None and v.requires_grad:
                raise ValueError('policy_loss: no gradient of %s (detach it)' % what)
    args = (logits, tokens, old_logp, advantages, ref_logp if kl else None, weight, (1.0 - lo, 1.0 + hi), kl, temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        return _PolicyLoss.apply(*args)
    return _policy(*args, False)[:2]
