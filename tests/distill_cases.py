"""Plain 64-bit forms of the distillation operators, and how far a kernel may be from them.

u = 2^-24 is half a step of fp32, relative to the value; h = eps / 2 of the output type.

* A thread sums every 512th vector of a row, at most V / 512 + 64 terms one after another, then 21 more additions join the threads: (V / 512 + 85) u.
* A term exp2((z - ref) scale): 2^-22 = 4 u of the instruction; the difference, the product and the rounded scale err by u each relative to
  the exponent, an absolute error of the exponent x of 3 u x, so 3 ln 2 u x relative to the term.  Terms below 2^-30 of the largest cannot
  matter for rows of 2^20: x <= 30 gives 63 u.
So `sum_error(V)` = (V / 512 + 152) u bounds the relative error of a sum of exponentials and the absolute one of its logarithm.
"""
import math

import torch

U = 2.0 ** -24


def sum_error(vocab):
    return (vocab / 512 + 152) * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def quantize(x):
    x = x.double()
    top = x.abs().amax(1)
    scales = (top / 127.0).float()
    scales = torch.where(scales < 2.0 ** -126, 0.0, scales)
    bad = ~torch.isfinite(x).all(1)
    scales = torch.where(bad, math.nan, scales)
    fine = (~bad & (scales > 0))[:, None]
    codes = torch.where(fine, x / scales.double()[:, None], 0.0).round()
    return torch.where(fine, codes, 0.0).to(torch.int8), scales


def matmul(a, b, a_scales, b_scales, bias):
    """(value, tolerance in fp32): the sum is rounded once, then two products and a fused addition."""
    v = (a.double() @ b.double().T) * a_scales.double()[:, None] * b_scales.double()
    size = v.abs() + (0 if bias is None else bias.double().abs())
    return v + (0 if bias is None else bias.double()), 4 * U * size + 2.0 ** -148


def topk(z, k, tau):
    x = z.double() + 0.0
    x = torch.where(x.isnan(), -math.inf, x)
    # NaN behind -inf: by a second key, stable sorts in turn
    order = torch.sort(z.isnan().int(), dim=1, stable=True).indices
    by_value = torch.sort(x.gather(1, order), dim=1, descending=True, stable=True).indices
    order = order.gather(1, by_value)
    # (-inf and NaN have one value above: the first sort put the NaN behind)
    idx = order[:, :k]
    others = z.double().scatter(1, idx, -math.inf) / tau
    rest = torch.logsumexp(others, 1)
    rest = torch.where(z.isnan().any(1), math.nan, rest)
    return z.gather(1, idx), idx.int(), rest


def distill(z, idx, val, rest, weights, tau):
    """(loss, grad, what the gradient's error is relative to)."""
    rows, vocab = z.shape
    y = z.double() / tau
    there = (idx >= 0) & (idx < vocab)
    to = torch.where(there, idx.long(), vocab)
    t = torch.where(there, val.double() / tau, -math.inf)
    r = torch.full((rows,), -math.inf, dtype=torch.float64, device=z.device) if rest is None else rest.double()
    # everything relative to the rows' largest: where those are 1e16, or the type's lowest value, nothing else would be left of 64 bits either
    m = torch.cat([t, r[:, None]], 1).amax(1)
    none = m == -math.inf
    m = torch.where(none, 0.0, m)
    t, r = t - m[:, None], r - m
    lp = torch.where(none, 0.0, torch.logsumexp(torch.cat([t, r[:, None]], 1), 1))
    p = torch.zeros(rows, vocab + 1, dtype=torch.float64, device=z.device).scatter_add_(1, to, torch.where(there, (t - lp[:, None]).exp(), 0.0))
    in_list = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=z.device).scatter_(1, to, True)
    p, in_list = p[:, :vocab], in_list[:, :vocab]
    pt = (r - lp).exp()
    y = y - y.amax(1, keepdim=True)
    total = torch.logsumexp(y, 1)
    outside = y.masked_fill(in_list, -math.inf)
    o = outside.amax(1)
    o = torch.where(o == -math.inf, 0.0, o)
    mass = torch.logsumexp(outside - o[:, None], 1)
    log_q = y - total[:, None]
    lg = torch.cat([log_q, torch.zeros_like(log_q[:, :1])], 1).gather(1, to)
    pj = torch.where(there, (t - lp[:, None]).exp(), 0.0)
    loss = torch.where(pj > 0, pj * (t - lp[:, None] - lg), 0.0).sum(1)
    loss = loss + torch.where(pt > 0, pt * (r - lp - (mass + (o - total))), 0.0)
    share = torch.where(in_list | (mass == -math.inf)[:, None], 0.0, pt[:, None] * (outside - o[:, None] - mass[:, None]).exp())
    q = log_q.exp()
    grad = torch.where(none[:, None], 0.0, (q - p - share) / tau)
    size = (q + p + share) / tau
    loss = torch.where(none, 0.0, loss)
    w = torch.ones(rows, dtype=torch.float64, device=z.device) if weights is None else weights.double()
    loss, grad, size = loss * w, grad * w[:, None], size * w.abs()[:, None]
    skip = w == 0
    return torch.where(skip, 0.0, loss), torch.where(skip[:, None], 0.0, grad), torch.where(skip[:, None], 0.0, size)


def assert_near(got, want, tol, what):
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        at = bad.nonzero()[0].tolist()
        i = tuple(at)
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {got[i]!r}, want {want[i]!r}, tolerance {tol[i]!r}')


def assert_distill(loss, grad, want, vocab, what=''):
    """The loss enters with an error of the sum over the rest times a difference of probabilities (at most 1), and its own rounding; the gradient with
    the errors of its terms (another exponent, as above, and four roundings) and the rounding to its type."""
    w_loss, w_grad, size = want
    assert_near(loss, w_loss, sum_error(vocab) + 2 * U * w_loss.abs(), f'loss {what}')
    assert_near(grad, w_grad, (sum_error(vocab) + 72 * U) * size + (half_step(grad.dtype) * 1.001) * w_grad.abs() + 2.0 ** -126, f'grad {what}')
