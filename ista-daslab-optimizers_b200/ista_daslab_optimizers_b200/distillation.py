"""Distillation of a frozen teacher into the model that the optimizer trains.

The teacher's weights and activations are 8-bit integers with a scale per channel and token (`quantize_rows`, `int8_matmul`); of its logits only
the largest are kept, with the mass of the rest (`topk_logits`); the student's loss and its gradient come from those (`distill_loss` through
autograd, `distill_step` as one call).

    codes, scales = quantize_rows(weight)                        # once per frozen layer
    x, x_scales = quantize_rows(hidden)                          # per batch
    teacher = int8_matmul(x, codes, x_scales, scales)
    values, indices, rest = topk_logits(teacher, 64, temperature=2.0)
    loss, grad = distill_step(student, indices, values, rest, weights, temperature=2.0)
    student.backward(grad)                                       # or: distill_loss(...).sum().backward()
    optimizer.step()

Every tensor is a CUDA tensor of one device; the work is enqueued on that device's current stream.  Matrices are two-dimensional, their rows
contiguous; the rows themselves may lie any distance apart (a slice of columns, every second row).  What the kernels cannot take raises
NativeError before anything is launched; there is no other implementation behind them.  Outputs that are given (`codes`, `scales`, `out`, `grad`) share no
memory with inputs (but `grad` with the logits that it replaces).  A wait inside a kernel that runs out (a device in trouble)
cannot raise where it happens: what the kernel should have written is NaN, and `_native.device_error()`, which waits for the device, returns 1.
"""
from __future__ import annotations

import operator

import torch
from torch.autograd import forward_ad

from . import _native as N

__all__ = ['quantize_rows', 'int8_matmul', 'topk_logits', 'distill_loss', 'distill_step']


def _rows(t, what, dtypes=(torch.float32, torch.bfloat16)):
    """Raises unless t is a CUDA matrix of one of these types whose rows are contiguous and do not overlap."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise N.NativeError(f'{what} must be a two-dimensional tensor')
    if not t.is_cuda:
        raise N.NativeError(f'{what} must be a CUDA tensor (got {t.device}); there is no CPU implementation')
    if t.dtype not in dtypes:
        raise N.NativeError(f'{what} has element type {t.dtype}; it takes {" or ".join(str(d) for d in dtypes)}')
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise N.NativeError(f'the rows of {what} must be contiguous')
    if rows > 1 and t.stride(0) < cols:
        raise N.NativeError(f'the rows of {what} overlap')


def _tensors(optional=(), **given):
    for what, t in given.items():
        if not isinstance(t, torch.Tensor) and not (t is None and what in optional):
            raise N.NativeError(f'{what} must be a tensor (got {t!r})')
        if t is not None and t.is_neg():
            raise N.NativeError(f'{what} has a negation that is not resolved yet: hand over {what}.resolve_neg()')


def _vector(t, n, what, device, optional=False):
    if optional and t is None:
        return
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        got = f'{tuple(t.shape)}, {t.dtype}, {t.device}' if isinstance(t, torch.Tensor) else f'{t!r}'
        raise N.NativeError(f'{what} must be {n} contiguous float32 values on {device} (got {got})')


def _same_device(device, **tensors):
    for what, t in tensors.items():
        if t.device != device:
            raise N.NativeError(f'{what} is on {t.device}, not on {device}')


def _no_tangent_for(call, **tensors):
    for what, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise N.NativeError(f'{call} has no forward-mode derivative: the tangent of {what} would be lost')


def _no_grad_for(call, **tensors):
    _no_tangent_for(call, **tensors)
    for what, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise N.NativeError(f'{call} has no gradient for {what}: what belongs to a frozen teacher is handed over detached, or under torch.no_grad()')


_native_calls = None


def _calls():
    global _native_calls
    _native_calls = N.load_distill_calls()
    return _native_calls


def _fail(result, what, explain, *args):
    """What the native side answered instead of tensors: a status of the library, or None where an argument is not as it should be."""
    if result is None:
        explain(*args)
        raise N.NativeError(f'{what} cannot take these arguments')
    N.check(result, what)


def quantize_rows(x, codes=None, scales=None):
    """8-bit codes and one float32 scale per row of x (float32 or bfloat16 [rows, cols]): scale = max |x| / 127, code = the integer nearest
    x / scale, half to even.  A row with a NaN or an infinity gets the scale NaN and zeros.  Returns (codes, scales); codes made here
    lie a multiple of 16 bytes apart, as `int8_matmul` wants them.  Not differentiable."""
    result = (_native_calls or _calls()).quantize_rows(x, codes, scales)
    return result if type(result) is tuple else _fail(result, 'quantize_rows', _explain_quantize, x, codes, scales)


def _explain_quantize(x, codes, scales):
    _tensors(x=x, codes=codes, scales=scales, optional=('codes', 'scales'))
    _rows(x, 'x')
    _no_grad_for('quantize_rows', x=x, scales=scales)
    if codes is not None:
        _rows(codes, 'codes', (torch.int8,))
        if codes.shape != x.shape:
            raise N.NativeError(f'codes must have the shape of x, {tuple(x.shape)} (got {tuple(codes.shape)})')
        _same_device(x.device, codes=codes)
    _vector(scales, x.shape[0], 'scales', x.device, optional=True)


def int8_matmul(a, b, a_scales, b_scales, bias=None, out=None, dtype=torch.bfloat16):
    """out[i, j] = (sum_c a[i, c] b[j, c]) a_scales[i] b_scales[j] + bias[j] for int8 a [tokens, inner] and b [channels, inner]: the sum exact in
    32-bit integers, then fp32, rounded once to `dtype` (float32 or bfloat16; that of `out` where it is given).  The codes start on 16 bytes and
    their rows lie a multiple of 16 bytes apart (`quantize_rows` makes them so); the inner size is at most 131071.  Not differentiable."""
    if out is None and dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise N.NativeError(f'unsupported element type {dtype}: the kernels write float32 and bfloat16')
    result = (_native_calls or _calls()).int8_matmul(a, b, a_scales, b_scales, bias, out, dtype is torch.bfloat16)
    return result[0] if type(result) is tuple else _fail(result, 'int8_matmul', _explain_matmul, a, b, a_scales, b_scales, bias, out)


def _explain_matmul(a, b, a_scales, b_scales, bias, out):
    _tensors(a=a, b=b, a_scales=a_scales, b_scales=b_scales, bias=bias, out=out, optional=('bias', 'out'))
    _rows(a, 'a', (torch.int8,))
    _rows(b, 'b', (torch.int8,))
    if a.shape[1] != b.shape[1]:
        raise N.NativeError(f'a and b have inner sizes {a.shape[1]} and {b.shape[1]}')
    _same_device(a.device, b=b)
    m, n = a.shape[0], b.shape[0]
    _vector(a_scales, m, 'a_scales', a.device)
    _vector(b_scales, n, 'b_scales', a.device)
    _vector(bias, n, 'bias', a.device, optional=True)
    _no_grad_for('int8_matmul', a_scales=a_scales, b_scales=b_scales, bias=bias, out=out)
    if out is not None:
        _rows(out, 'out')
        if out.shape != (m, n):
            raise N.NativeError(f'out must have the shape {(m, n)} (got {tuple(out.shape)})')
        _same_device(a.device, out=out)


def topk_logits(logits, k, temperature=1.0):
    """(values, indices, rest): the k largest logits of every row (float32 or bfloat16 [rows, vocab], k at most 1024) in descending order,
    ties to the lower index, in the logits' type; their int32 indices; and the float32 logarithm of sum exp(logit / temperature) over all others, -inf
    where there is nothing else.  NaN ranks below -inf and makes `rest` NaN.  Not differentiable."""
    k = operator.index(k)
    result = (_native_calls or _calls()).topk_logits(logits, k, float(temperature))
    return result if type(result) is tuple else _fail(result, 'topk_logits', _explain_topk, logits, k)


def _explain_topk(logits, k):
    _tensors(logits=logits)
    _rows(logits, 'logits')
    _no_grad_for('topk_logits', logits=logits)
    if not 1 <= k <= logits.shape[1]:
        raise N.NativeError(f'k={k} is not between 1 and the {logits.shape[1]} logits of a row')


def _explain_lists(what, logits, indices, values, rest, weights, temperature):
    _tensors(logits=logits, indices=indices, values=values, rest=rest, weights=weights, optional=('rest', 'weights'))
    _no_grad_for(what, values=values, rest=rest, weights=weights)
    _no_tangent_for(what, logits=logits)
    _rows(logits, 'logits')
    rows, vocab = logits.shape
    if indices.dim() != 2 or indices.shape[0] != rows or values.shape != indices.shape:
        raise N.NativeError(f'indices and values must be [{rows}, k] (got {tuple(indices.shape)} and {tuple(values.shape)})')
    if indices.dtype != torch.int32 or values.dtype not in (torch.float32, torch.bfloat16):
        raise N.NativeError(f'indices must be int32, values float32 or bfloat16 (got {indices.dtype} and {values.dtype})')
    _same_device(logits.device, indices=indices, values=values)
    N.dev_ptr(indices, 'indices')
    N.dev_ptr(values, 'values')
    _vector(rest, rows, 'rest', logits.device, optional=True)
    _vector(weights, rows, 'weights', logits.device, optional=True)
    if not 1 <= indices.shape[1] <= N.MAB_MAX_LIST or not 1 <= vocab <= N.MAB_MAX_VOCAB or not 1e-6 < temperature < 1e6:
        raise N.NativeError(f'lists of {indices.shape[1]} entries (at most {N.MAB_MAX_LIST}), rows of {vocab} logits (at most {N.MAB_MAX_VOCAB}), '
                            f'temperature {temperature} (between 1e-6 and 1e6)')


def distill_loss(logits, indices, values, rest=None, weights=None, temperature=1.0):
    """Loss of every row, float32 [rows]: weights * KL(teacher || student), both at `temperature`, over the teacher's listed tokens and one class
    for all others.

    logits          the student's, float32 or bfloat16 [rows, vocab]; the only input with a gradient
    indices, values the teacher's list, int32 and float32 or bfloat16 [rows, k], as `topk_logits` gives it (k at most 1024).  An index outside
                    [0, vocab) is an entry that is not there (lists of different lengths); one that occurs again is a term p log(p / q) for
                    each of its entries: the gradient is that of the sum of their shares, and the loss lies below the divergence of the merged entries by the
                    entropy of the split among them times their share, which does not depend on the student (two equal entries with all of the mass: by log 2, so
                    it can be negative)
    rest            float32 [rows]: the logarithm of the teacher's mass outside its list at this temperature, as `topk_logits` gives it; None: the
                    teacher's distribution is the one over its list
    weights         float32 [rows] or None: a row with weight 0 is not read, whatever it holds, and has loss and gradient 0.  (Multiply by
                    temperature ** 2 here for gradients that do not shrink with the temperature.)

    The gradient comes from a second pass over the logits; `distill_step` gives both in one call.  Differentiable once, backward only (a tangent of
    forward-mode differentiation is refused)."""
    temperature = float(temperature)
    result = (_native_calls or _calls()).distill_loss(logits, indices, values, rest, weights, temperature)
    return result if result is not None else _fail(result, 'distill_loss', _explain_lists, 'distill_loss', logits, indices, values, rest, weights, temperature)


def distill_step(logits, indices, values, rest=None, weights=None, temperature=1.0, grad=None):
    """(loss, grad): the losses of `distill_loss` and the gradient of their sum with respect to the logits, in the logits' type, in one call.  Nothing is
    recorded for autograd: hand the gradient on with `logits.backward(grad)`.  `grad` can be given, and can be the logits' own memory
    (`grad=logits.detach()`): the gradient then replaces them."""
    temperature = float(temperature)
    result = (_native_calls or _calls()).distill_step(logits, indices, values, rest, weights, temperature, grad)
    return result if type(result) is tuple else _fail(result, 'distill_step', _explain_step, logits, indices, values, rest, weights, temperature, grad)


def _explain_step(logits, indices, values, rest, weights, temperature, grad):
    _explain_lists('distill_step', logits, indices, values, rest, weights, temperature)
    _tensors(grad=grad, optional=('grad',))
    _no_tangent_for('distill_step', grad=grad)
    if grad is not None:
        if grad.shape != logits.shape or grad.dtype != logits.dtype or grad.requires_grad:
            raise N.NativeError(f'grad must be like the logits, {tuple(logits.shape)} of {logits.dtype}, and require no gradient itself')
        _rows(grad, 'grad')
        _same_device(logits.device, grad=grad)
