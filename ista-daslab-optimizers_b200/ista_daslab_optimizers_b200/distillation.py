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
NativeError before anything is launched; there is no other implementation behind them.
"""
from __future__ import annotations

import torch

from . import _native as N

__all__ = ['quantize_rows', 'int8_matmul', 'topk_logits', 'distill_loss', 'distill_step']


def _rows(t, what, dtypes=(torch.float32, torch.bfloat16)):
    """(pointer, distance of the rows) of a matrix whose rows are contiguous."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise N.NativeError(f'{what} must be a two-dimensional tensor')
    if not t.is_cuda:
        raise N.NativeError(f'{what} must be a CUDA tensor (got {t.device}); there is no CPU implementation')
    if t.dtype not in dtypes:
        raise N.NativeError(f'{what} has element type {t.dtype}; it takes {" or ".join(str(d) for d in dtypes)}')
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise N.NativeError(f'the rows of {what} must be contiguous')
    pitch = t.stride(0) if rows > 1 else max(cols, 1)
    if pitch < cols:
        raise N.NativeError(f'the rows of {what} overlap')
    return t.data_ptr(), pitch


def _vector(t, n, what, device):
    """Pointer of n contiguous float32 values, or None."""
    if t is None:
        return None
    if t.dtype != torch.float32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise N.NativeError(f'{what} must be {n} contiguous float32 values on {device} (got {tuple(t.shape)}, {t.dtype}, {t.device})')
    return t.data_ptr()


def _same_device(device, **tensors):
    for what, t in tensors.items():
        if t.device != device:
            raise N.NativeError(f'{what} is on {t.device}, not on {device}')


def _no_grad_for(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise N.NativeError(f'{what} has no gradient: its inputs belong to a frozen teacher (call it under torch.no_grad())')


def quantize_rows(x, codes=None, scales=None):
    """8-bit codes and one float32 scale per row of x (float32 or bfloat16 [rows, cols]): scale = max |x| / 127, code = the integer nearest
    x / scale, half to even.  A row with a NaN or an infinity gets the scale NaN and zeros.  Returns (codes, scales); codes made here
    lie a multiple of 16 bytes apart, as `int8_matmul` wants them.  Not differentiable."""
    p, pitch = _rows(x, 'x')
    _no_grad_for('quantize_rows', x)
    rows, cols = x.shape
    if codes is None:
        codes = torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=x.device)[:, :cols]
    cp, codes_pitch = _rows(codes, 'codes', (torch.int8,))
    if codes.shape != x.shape:
        raise N.NativeError(f'codes must have the shape of x, {tuple(x.shape)} (got {tuple(codes.shape)})')
    if scales is None:
        scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    _same_device(x.device, codes=codes)
    sp = _vector(scales, rows, 'scales', x.device)
    N._run(x, 'quantize_rows', N.load().mab_quantize_rows, rows, cols, p, N.dtype_code(x), pitch, cp, codes_pitch, sp)
    return codes, scales


def int8_matmul(a, b, a_scales, b_scales, bias=None, out=None, dtype=torch.bfloat16):
    """out[i, j] = (sum_c a[i, c] b[j, c]) a_scales[i] b_scales[j] + bias[j] for int8 a [tokens, inner] and b [channels, inner]: the sum exact in
    32-bit integers, then fp32, rounded once to `dtype` (float32 or bfloat16; that of `out` where it is given).  The codes start on 16 bytes and
    their rows lie a multiple of 16 bytes apart (`quantize_rows` makes them so); the inner size is at most 131071.  Not differentiable."""
    ap, a_pitch = _rows(a, 'a', (torch.int8,))
    bp, b_pitch = _rows(b, 'b', (torch.int8,))
    (m, k), (n, kb) = a.shape, b.shape
    if k != kb:
        raise N.NativeError(f'a and b have inner sizes {k} and {kb}')
    _no_grad_for('int8_matmul', a_scales, b_scales, bias)
    if out is None:
        out = torch.empty(m, n, dtype=dtype, device=a.device)
    op, out_pitch = _rows(out, 'out')
    if out.shape != (m, n):
        raise N.NativeError(f'out must have the shape {(m, n)} (got {tuple(out.shape)})')
    _same_device(a.device, b=b, out=out)
    if m == 1:
        a_pitch = (a_pitch + 15) // 16 * 16             # one row: no distance
    if n == 1:
        b_pitch = (b_pitch + 15) // 16 * 16
    N._run(a, 'int8_matmul', N.load().mab_int8_matmul, m, n, k, ap, a_pitch, bp, b_pitch, _vector(a_scales, m, 'a_scales', a.device),
           _vector(b_scales, n, 'b_scales', a.device), _vector(bias, n, 'bias', a.device), op, N.dtype_code(out), out_pitch)
    return out


def topk_logits(logits, k, temperature=1.0):
    """(values, indices, rest): the k largest logits of every row (float32 or bfloat16 [rows, vocab], k at most 1024) in descending order,
    ties to the lower index, in the logits' type; their int32 indices; and the float32 logarithm of sum exp(logit / temperature) over all others, -inf
    where there is nothing else.  NaN ranks below -inf and makes `rest` NaN.  Not differentiable."""
    p, pitch = _rows(logits, 'logits')
    _no_grad_for('topk_logits', logits)
    rows, vocab = logits.shape
    values = torch.empty(rows, k, dtype=logits.dtype, device=logits.device)
    indices = torch.empty(rows, k, dtype=torch.int32, device=logits.device)
    rest = torch.empty(rows, dtype=torch.float32, device=logits.device)
    N._run(logits, 'topk_logits', N.load().mab_topk_logits, rows, vocab, k, p, N.dtype_code(logits), pitch, float(temperature), values.data_ptr(),
           indices.data_ptr(), rest.data_ptr())
    return values, indices, rest


def _teacher(logits, indices, values, rest, weights):
    """The arguments that the loss and the step share, checked: (rows, vocab, k) and the pointers."""
    p, pitch = _rows(logits, 'logits')
    rows, vocab = logits.shape
    device = logits.device
    if indices.dim() != 2 or indices.shape[0] != rows or values.shape != indices.shape:
        raise N.NativeError(f'indices and values must be [{rows}, k] (got {tuple(indices.shape)} and {tuple(values.shape)})')
    if indices.dtype != torch.int32:
        raise N.NativeError(f'indices must be int32 (got {indices.dtype})')
    _same_device(device, indices=indices, values=values)
    return (rows, vocab, indices.shape[1]), (p, N.dtype_code(logits), pitch, N.dev_ptr(indices, 'indices'), N.dev_ptr(values, 'values'),
                                             N.dtype_code(values), _vector(rest, rows, 'rest', device), _vector(weights, rows, 'weights', device))


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, indices, values, rest, weights, temperature):
        (rows, vocab, k), args = _teacher(logits, indices, values, rest, weights)
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        stats = torch.empty(rows, 2, dtype=torch.float32, device=logits.device)
        list_grad = torch.empty(rows, k, dtype=torch.float32, device=logits.device)
        N._run(logits, 'distill_loss', N.load().mab_distill_loss, rows, vocab, k, *args, temperature, loss.data_ptr(), stats.data_ptr(),
               list_grad.data_ptr())
        ctx.save_for_backward(logits, indices, weights, stats, list_grad)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, indices, weights, stats, list_grad = ctx.saved_tensors
        p, pitch = _rows(logits, 'logits')
        rows, vocab = logits.shape
        if grad_loss.dtype != torch.float32:
            grad_loss = grad_loss.float()
        grad = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
        N._run(logits, 'distill_loss backward', N.load().mab_distill_grad, rows, vocab, indices.shape[1], p, N.dtype_code(logits), pitch,
               indices.data_ptr(), None if weights is None else weights.data_ptr(), ctx.temperature, stats.data_ptr(), list_grad.data_ptr(),
               grad_loss.data_ptr(), grad_loss.stride(0), grad.data_ptr(), vocab)
        return grad, None, None, None, None, None


def distill_loss(logits, indices, values, rest=None, weights=None, temperature=1.0):
    """Loss of every row, float32 [rows]: weights * KL(teacher || student), both at `temperature`, over the teacher's listed tokens and one class
    for all others.

    logits          the student's, float32 or bfloat16 [rows, vocab]; the only input with a gradient
    indices, values the teacher's list, int32 and float32 or bfloat16 [rows, k], as `topk_logits` gives it (k at most 1024).  An index outside
                    [0, vocab) is an entry that is not there (lists of different lengths); one that occurs again counts with the sum of its entries
    rest            float32 [rows]: the logarithm of the teacher's mass outside its list at this temperature, as `topk_logits` gives it; None: the
                    teacher's distribution is the one over its list
    weights         float32 [rows] or None: a row with weight 0 is not read, whatever it holds, and has loss and gradient 0.  (Multiply by
                    temperature ** 2 here for gradients that do not shrink with the temperature.)

    The gradient comes from a second pass over the logits; `distill_step` reads them once."""
    for what, t in (('values', values), ('rest', rest), ('weights', weights)):
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise N.NativeError(f'distill_loss has no gradient for {what}')
    return _DistillLoss.apply(logits, indices, values, rest, weights, float(temperature))


def distill_step(logits, indices, values, rest=None, weights=None, temperature=1.0, grad=None):
    """(loss, grad): the losses of `distill_loss` and the gradient of their sum with respect to the logits, in the logits' type, in one call.  Nothing is
    recorded for autograd: hand the gradient on with `logits.backward(grad)`.  `grad` can be given, and can be the logits' own memory
    (`grad=logits.detach()`): the gradient then replaces them."""
    (rows, vocab, k), args = _teacher(logits, indices, values, rest, weights)
    if grad is None:
        grad = torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
    elif grad.shape != logits.shape or grad.dtype != logits.dtype or grad.requires_grad:
        raise N.NativeError(f'grad must be like the logits, {tuple(logits.shape)} of {logits.dtype}, and require no gradient itself')
    gp, grad_pitch = _rows(grad, 'grad')
    _same_device(logits.device, grad=grad)
    loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
    N._run(logits, 'distill_step', N.load().mab_distill_step, rows, vocab, k, *args, float(temperature), loss.data_ptr(), gp, grad_pitch)
    return loss, grad
