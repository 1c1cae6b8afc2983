"""The operators that bring a frozen teacher's answer into the model that the optimizer trains, as cases that can be timed.

* 'quantize': rows of activations or weights into 8-bit integers with a scale for each row;
* 'matmul':   product of two such operands, scaled for each token and channel;
* 'topk':     the top logits of every row, in order, and the logarithm of the mass of the rest;
* 'loss':     the distillation loss from such rows and its gradient, forward and backward as autograd calls them;
* 'step':     loss and gradient in one call.

With `own` false `run` computes the plain form, with `own` true it makes the calls of this package.  `listed()` are fixed
cases, `draw()` makes further ones of the same ranges, `exact()` gives the definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}
_BYTES = {'f32': 4, 'bf16': 2}
_NEG = -math.inf


def _package():
    # the package's folder lies in the repository's root, which is the working folder
    at = os.path.join(os.getcwd(), 'ista-daslab-optimizers_b200')
    if at not in sys.path:
        sys.path.insert(0, at)
    import ista_daslab_optimizers_b200
    return ista_daslab_optimizers_b200


def _quantize(name, rows, width, dtype):
    return dict(name=name, op='quantize', rows=rows, width=width, dtype=dtype)


def _matmul(name, rows, cols, width, dtype, bias=False):
    return dict(name=name, op='matmul', rows=rows, cols=cols, width=width, dtype=dtype, bias=bias)


def _topk(name, rows, vocab, k, dtype, tau=1.0, padded=0):
    return dict(name=name, op='topk', rows=rows, vocab=vocab, k=k, dtype=dtype, tau=tau, padded=padded)


def _distill(name, op, rows, vocab, k, dtype, values, tau=1.0, rest=True, masked=0, ragged=False, padded=0):
    return dict(name=name, op=op, rows=rows, vocab=vocab, k=k, dtype=dtype, values=values, tau=tau, rest=rest, masked=masked, ragged=ragged,
                padded=padded)


def listed():
    return [
        # the activations of eight tokens that a teacher of width 4096 is decoding: all latency
        _quantize('quantize_decode', 8, 4096, 'bf16'),
        # the activations behind the wide half of a layer, an odd number of tokens in fp32
        _quantize('quantize_tokens_fp32', 2047, 14336, 'f32'),
        # one token through a square projection of width 4096
        _matmul('matmul_one_token', 1, 4096, 4096, 'bf16'),
        # a ragged batch of tokens through the wide half of a layer, the weights' bytes dominate
        _matmul('matmul_batch', 41, 14336, 4096, 'bf16', bias=True),
        # a ragged product with an odd inner size and an odd vocabulary, fp32 logits
        _matmul('matmul_odd_fp32', 777, 50257, 767, 'f32'),
        # a training batch through the head of the 128256-token vocabulary: the largest product
        _matmul('matmul_head', 2048, 128256, 4096, 'bf16'),
        # few rows of an odd vocabulary in fp32, as an interactive teacher gives them; the table is padded
        _topk('topk_few_rows_fp32', 5, 50257, 20, 'f32', padded=17),
        # a training batch of teacher logits, 64 kept of 128256
        _topk('topk_batch', 2048, 128256, 64, 'bf16', tau=2.0),
        # few sequences of a small student: forward and backward of 60 rows, fp32, no mass outside the list, lists of different lengths
        _distill('loss_few_rows_fp32', 'loss', 60, 50257, 32, 'f32', 'f32', rest=False, ragged=True),
        # a training batch through autograd, a quarter of its tokens belongs to the prompt and has no loss
        _distill('loss_batch', 'loss', 2048, 128256, 64, 'bf16', 'bf16', tau=2.0, masked=512),
        # odd rows of an odd, padded vocabulary, fp32, long lists
        _distill('step_odd_fp32', 'step', 333, 50257, 257, 'f32', 'bf16', tau=1.5, padded=17),
        # the same training batch, twice as many rows, loss and gradient in one call
        _distill('step_batch', 'step', 4096, 128256, 64, 'bf16', 'bf16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(['quantize', 'matmul', 'matmul', 'topk', 'loss', 'step'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    if op == 'quantize':
        rows = _log_int(rng, 1, 4096)
        c = _quantize('', rows, min(_log_int(rng, 64, 16384), (1 << 25) // rows), dtype)
    elif op == 'matmul':
        width, cols = _log_int(rng, 64, 8192), _log_int(rng, 64, 50257)
        if rng.random() < 0.5:                           # (what models have is a multiple of 64 more often than not)
            width, cols = (width + 63) // 64 * 64, (cols + 63) // 64 * 64
        rows = _log_int(rng, 1, min(4096, (1 << 39) // (width * cols)))
        c = _matmul('', rows, cols, width, dtype, bias=rng.random() < 0.3)
    else:
        vocab = _log_int(rng, 1000, 151936)
        if rng.random() < 0.5:
            vocab = (vocab + 63) // 64 * 64
        rows = _log_int(rng, 1, min(4096, (1 << 27) // vocab))
        k, tau, padded = _log_int(rng, 1, 512), rng.choice([1.0, 1.0, 2.0, 0.7]), rng.choice([0, 0, 17, 100])
        if op == 'topk':
            c = _topk('', rows, vocab, min(k, vocab // 2), dtype, tau, padded)
        else:
            c = _distill('', op, rows, vocab, min(k, vocab // 2), dtype, rng.choice(['bf16', 'f32']), tau, rng.random() < 0.7,
                         rng.choice([0, 0, rows // 4]), rng.random() < 0.3, padded)
    del c['name']
    return c


def work(c):
    if c['op'] == 'quantize':
        n = c['rows'] * c['width']
        return dict(bytes=n * (_BYTES[c['dtype']] + 1) + 4 * c['rows'], flops=2 * n)
    if c['op'] == 'matmul':
        m, n, k = c['rows'], c['cols'], c['width']
        return dict(bytes=m * k + n * k + m * n * _BYTES[c['dtype']] + 4 * (m + n + (n if c['bias'] else 0)), flops=2 * m * n * k)
    e, row = _BYTES[c['dtype']], c['vocab'] * _BYTES[c['dtype']]
    if c['op'] == 'topk':
        return dict(bytes=c['rows'] * (row + c['k'] * (e + 4) + 4), flops=3 * c['rows'] * c['vocab'])
    rows = c['rows'] - c['masked']                       # a row without a weight is not read, its gradient is written
    lists = rows * c['k'] * (4 + _BYTES[c['values']]) + c['rows'] * 12
    reads = 2 if c['op'] == 'loss' else 1                # the backward pass comes later, when nothing of the forward pass is on chip
    return dict(bytes=rows * row * reads + c['rows'] * row + lists, flops=rows * c['vocab'] * 8)


# ---------------------------------------------------------------------------------------------------- inputs

def _logits(gen, rows, vocab, padded):
    """Rows as language models give them: a common slope over the vocabulary, a spread for each token, a few likely tokens; the last
    `padded` columns belong to no token."""
    z = torch.randn(rows, vocab, generator=gen, device='cuda')
    z *= 1.0 + torch.rand(rows, 1, generator=gen, device='cuda')
    z -= torch.log1p(torch.arange(vocab, device='cuda') * (50.0 / vocab))
    part = (vocab - padded) // 6                         # one in each sixth: no column twice
    at = torch.randint(0, part, (rows, 6), generator=gen, device='cuda') + torch.arange(6, device='cuda') * part
    z.scatter_add_(1, at, 4.0 + 6.0 * torch.rand(rows, 6, generator=gen, device='cuda'))
    if padded:
        z[:, vocab - padded:] = _NEG
    return z


def _codes(gen, rows, width):
    """8-bit codes of normal rows, and their scales, in rows that lie a multiple of 16 bytes apart, as `quantize_rows` leaves them."""
    x = torch.randn(rows, width, generator=gen, device='cuda')
    scales = x.abs().amax(1) / 127.0
    codes = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device='cuda')[:, :width]
    codes.copy_((x / scales[:, None]).round_())
    return codes, scales * 0.02


def prepare(c, seed):
    gen = torch.Generator('cuda')
    gen.manual_seed(seed)
    s = dict(case=c, pkg=_package() if own else None)
    if c['op'] == 'quantize':
        x = torch.randn(c['rows'], c['width'], generator=gen, device='cuda')
        x *= 0.1 + 3.0 * torch.rand(c['rows'], 1, generator=gen, device='cuda')
        x[:, :: 97] *= 8.0                               # the few large channels of a trained model's activations
        s['x'] = x.to(_DTYPES[c['dtype']])
    elif c['op'] == 'matmul':
        s['a'], s['a_scales'] = _codes(gen, c['rows'], c['width'])
        s['b'], s['b_scales'] = _codes(gen, c['cols'], c['width'])
        s['bias'] = torch.randn(c['cols'], generator=gen, device='cuda') if c['bias'] else None
    elif c['op'] == 'topk':
        s['logits'] = _logits(gen, c['rows'], c['vocab'], c['padded']).to(_DTYPES[c['dtype']])
    else:
        rows, vocab, k = c['rows'], c['vocab'], c['k']
        teacher = _logits(gen, rows, vocab, c['padded'])
        z = torch.randn(rows, vocab, generator=gen, device='cuda').add_(teacher, alpha=0.7)
        s['logits'] = z.to(_DTYPES[c['dtype']]).requires_grad_(c['op'] == 'loss')
        del z
        values, indices = torch.topk(teacher, k)
        s['values'], s['indices'] = values.to(_DTYPES[c['values']]), indices.to(torch.int32)
        s['rest'] = torch.logsumexp(teacher.scatter_(1, indices, _NEG) / c['tau'], 1) if c['rest'] else None
        if c['ragged']:                                  # lists that end where the teacher was sure enough
            n = torch.randint(1, k + 1, (rows, 1), generator=gen, device='cuda')
            s['indices'][torch.arange(k, device='cuda') >= n] = -1
        s['weights'] = None
        if c['masked']:
            s['weights'] = torch.full((rows,), 1.0 / (rows - c['masked']), device='cuda')
            s['weights'][:c['masked']] = 0.0
        if c['op'] == 'loss':
            s['grad_loss'] = torch.ones(rows, device='cuda')
    return s


# ---------------------------------------------------------------------------------------------------- plain forms

def _lse(z):
    """log sum exp along the rows, the long sum and the logarithm in 64 bits; -inf where a row has nothing."""
    m = z.amax(1, keepdim=True)
    m = torch.where(m == _NEG, torch.zeros_like(m), m)
    return m[:, 0].double() + (z - m).exp().sum(1, dtype=torch.float64).log()


def _plain_quantize(x):
    # quotients in 64 bits: the scale is the fp32 number nearest to its own, and a code next to a half decides by its exact one
    x = x.double()
    scales = (x.abs().amax(1) / 127.0).float()
    return (x / scales.double()[:, None]).round().to(torch.int8), scales


def _plain_matmul(a, b, a_scales, b_scales, bias, dtype):
    out = (a.float() @ b.float().T) * a_scales[:, None] * b_scales
    return (out if bias is None else out + bias).to(dtype)


def _plain_topk(logits, k, tau):
    z = logits.float()
    bits = (z + 0.0).view(torch.int32)                   # order of floats as an order of integers (+ 0.0: the two zeros are equal)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key += torch.arange(z.shape[1] - 1, -1, -1, device=z.device)
    indices = torch.topk(key, k).indices                 # distinct keys: ties went to the lower index
    rest = _lse(z.scatter(1, indices, _NEG) / tau).float()
    return logits.gather(1, indices), indices.int(), rest


def _plain_distill(logits, indices, values, rest, weights, tau, grad_loss):
    z = logits.detach().float() / tau
    # the lists and the logarithms in 64 bits: the loss is what is left of a difference of distributions that are alike
    t = values.double() / tau
    there = indices >= 0
    at = indices.clamp(min=0).long()
    t = torch.where(there, t, _NEG)
    lp = _lse(t) if rest is None else _lse(torch.cat([t, rest.double()[:, None]], 1))
    log_p = t - lp[:, None]
    p = log_p.exp()
    log_q_all = _lse(z)
    # absent entries point at column 0, which must not leave the rest on their account: they are sent to a column of their own
    wide = torch.cat([z, torch.zeros_like(z[:, :1])], 1)
    to = torch.where(there, at, z.shape[1])
    others = wide.scatter(1, to, _NEG)[:, :-1]
    log_q_rest = _lse(others)
    log_q = logits.detach().gather(1, at).double() / tau - log_q_all[:, None]
    loss = torch.where(there, p * (log_p - log_q), 0.0).sum(1)
    q = (z - log_q_all.float()[:, None]).exp()
    grad = torch.cat([q, torch.zeros_like(q[:, :1])], 1)
    if rest is not None:
        log_pt = rest.double() - lp
        pt = log_pt.exp()
        loss = loss + torch.where(pt > 0, pt * (log_pt - (log_q_rest - log_q_all)), 0.0)
        grad[:, :-1] -= pt.float()[:, None] * (others - log_q_rest.float()[:, None]).exp()
    grad = grad.scatter_add(1, to, torch.where(there, -p, 0.0).float())[:, :-1]
    w = torch.ones_like(loss) if weights is None else weights.double()
    back = w / tau if grad_loss is None else w * grad_loss / tau
    return (loss * w).float(), (grad * back.float()[:, None]).to(logits.dtype)


def run(s):
    c = s['case']
    if c['op'] == 'quantize':
        return s['pkg'].quantize_rows(s['x']) if own else _plain_quantize(s['x'])
    if c['op'] == 'matmul':
        operands = (s['a'], s['b'], s['a_scales'], s['b_scales'], s['bias'])
        return s['pkg'].int8_matmul(*operands, dtype=_DTYPES[c['dtype']]) if own else _plain_matmul(*operands, _DTYPES[c['dtype']])
    if c['op'] == 'topk':
        return s['pkg'].topk_logits(s['logits'], c['k'], c['tau']) if own else _plain_topk(s['logits'], c['k'], c['tau'])
    given = (s['logits'], s['indices'], s['values'], s['rest'], s['weights'], c['tau'])
    if c['op'] == 'step':
        return s['pkg'].distill_step(*given) if own else _plain_distill(*given, None)
    if not own:
        return _plain_distill(*given, s['grad_loss'])
    loss = s['pkg'].distill_loss(*given)
    return loss.detach(), torch.autograd.grad(loss, s['logits'], s['grad_loss'])[0]


# ---------------------------------------------------------------------------------------------------- definitions in 64 bits

def _exact_distill(s, tau):
    z = s['logits'].detach().double().div_(tau)
    rows, vocab = z.shape
    teacher = torch.full((rows, vocab + 1), _NEG, dtype=torch.float64, device='cuda')      # the last column takes absent entries
    where = torch.where(s['indices'] >= 0, s['indices'].long(), vocab)
    teacher.scatter_(1, where, s['values'].double() / tau)
    teacher = teacher[:, :vocab]
    kept = teacher > _NEG
    total = torch.logsumexp(teacher, 1, keepdim=True)
    if s['rest'] is not None:
        total = torch.logaddexp(total, s['rest'].double()[:, None])
    teacher -= total
    z -= torch.logsumexp(z, 1, keepdim=True)
    loss = torch.where(kept, teacher.exp() * (teacher - z), 0.0).sum(1)
    target = teacher.exp()
    if s['rest'] is not None:
        share = s['rest'].double()[:, None] - total
        outside = z.masked_fill(kept, _NEG)
        mass = torch.logsumexp(outside, 1, keepdim=True)
        term = share.exp() * (share - mass)
        loss += torch.where(share > _NEG, term, 0.0)[:, 0]
        target += (outside - mass + share).exp()
    grad = z.exp().sub_(target)
    scale = torch.ones(rows, dtype=torch.float64, device='cuda') if s['weights'] is None else s['weights'].double()
    return loss * scale, grad.mul_(scale[:, None] / tau)


def exact(c, seed):
    s = prepare(c, seed)
    if c['op'] == 'quantize':
        return None, s['x'].double().abs().max(1).values / 127
    if c['op'] == 'matmul':
        out = torch.matmul(s['a'].double(), s['b'].double().t())
        out.mul_(s['a_scales'].double().unsqueeze(1)).mul_(s['b_scales'].double().unsqueeze(0))
        return out if s['bias'] is None else out.add_(s['bias'].double())
    if c['op'] == 'topk':
        z = s['logits'].double()
        ordered = torch.sort(z, dim=1, descending=True, stable=True).values
        return ordered[:, :c['k']], None, torch.logsumexp(ordered[:, c['k']:] / c['tau'], 1)
    return _exact_distill(s, c['tau'])
