"""What the distillation operators refuse, without a device: every refusal comes before any CUDA call."""
import math
import os
import sys

import pytest
import torch

import distill_cases as D

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, BAD, UNSUPPORTED, LIMIT = 0, -1, -2, -4


@pytest.fixture(scope='module')
def lib():
    sys.path.insert(0, os.path.join(ROOT, 'ista-daslab-optimizers_b200'))
    import build
    build.build()
    from ista_daslab_optimizers_b200 import _native
    return _native.load()


P = 1 << 20                                              # an aligned address; nothing is dereferenced on these paths


def quant(lib, rows=4, cols=64, x=P, dtype=0, xp=64, c=P, cp=64, s=P):
    return lib.mab_quantize_rows(rows, cols, x, dtype, xp, c, cp, s, None)


def matmul(lib, m=4, n=8, k=64, a=P, ap=64, b=P, bp=64, sa=P, sb=P, bias=None, out=P, dtype=0, op=8):
    return lib.mab_int8_matmul(m, n, k, a, ap, b, bp, sa, sb, bias, out, dtype, op, None)


def topk(lib, rows=4, vocab=64, k=8, z=P, dtype=0, pitch=64, tau=1.0, v=P, i=P, r=P):
    return lib.mab_topk_logits(rows, vocab, k, z, dtype, pitch, tau, v, i, r, None)


def loss(lib, rows=4, vocab=64, k=8, z=P, dtype=0, pitch=64, i=P, v=P, vd=0, r=None, w=None, tau=1.0, out=P, st=P, lg=P):
    return lib.mab_distill_loss(rows, vocab, k, z, dtype, pitch, i, v, vd, r, w, tau, out, st, lg, None)


def grad(lib, rows=4, vocab=64, k=8, z=P, dtype=0, pitch=64, i=P, w=None, tau=1.0, st=P, lg=P, up=P, stride=1, g=P + 4096, gp=64):
    return lib.mab_distill_grad(rows, vocab, k, z, dtype, pitch, i, w, tau, st, lg, up, stride, g, gp, None)


def step(lib, rows=4, vocab=64, k=8, z=P, dtype=0, pitch=64, i=P, v=P, vd=0, r=None, w=None, tau=1.0, out=P, g=P + 4096, gp=64):
    return lib.mab_distill_step(rows, vocab, k, z, dtype, pitch, i, v, vd, r, w, tau, out, g, gp, None)


@pytest.mark.parametrize('call,wrong,status', [
    (quant, dict(rows=-1), BAD), (quant, dict(cols=0), BAD), (quant, dict(x=None), BAD), (quant, dict(c=None), BAD), (quant, dict(s=None), BAD),
    (quant, dict(xp=63), BAD), (quant, dict(cp=63), BAD), (quant, dict(dtype=2), UNSUPPORTED), (quant, dict(x=P + 2), BAD), (quant, dict(x=P + 1, dtype=1), BAD),
    (quant, dict(s=P + 2), BAD), (quant, dict(cols=1 << 31, xp=1 << 31, cp=1 << 31), LIMIT), (quant, dict(rows=0, x=None), OK),
    (matmul, dict(k=0), BAD), (matmul, dict(m=-1), BAD), (matmul, dict(k=131072, ap=131072, bp=131072), LIMIT), (matmul, dict(dtype=3), UNSUPPORTED),
    (matmul, dict(a=None), BAD), (matmul, dict(b=None), BAD), (matmul, dict(sa=None), BAD), (matmul, dict(sb=None), BAD), (matmul, dict(out=None), BAD),
    (matmul, dict(ap=48), BAD), (matmul, dict(ap=72), BAD), (matmul, dict(bp=72), BAD), (matmul, dict(a=P + 8), BAD), (matmul, dict(b=P + 8), BAD),
    (matmul, dict(op=7), BAD), (matmul, dict(bias=P + 1), BAD), (matmul, dict(out=P + 2), BAD), (matmul, dict(m=1 << 30), LIMIT), (matmul, dict(m=0), OK),
    (matmul, dict(n=0), OK),
    (topk, dict(k=0), BAD), (topk, dict(k=65), BAD), (topk, dict(vocab=2000, pitch=2000, k=1025), LIMIT), (topk, dict(vocab=(1 << 20) + 1, pitch=1 << 21), LIMIT),
    (topk, dict(pitch=63), BAD), (topk, dict(tau=0.0), BAD), (topk, dict(tau=-1.0), BAD), (topk, dict(tau=math.nan), BAD), (topk, dict(tau=math.inf), BAD),
    (topk, dict(z=None), BAD), (topk, dict(v=None), BAD), (topk, dict(i=None), BAD), (topk, dict(r=None), BAD), (topk, dict(dtype=7), UNSUPPORTED),
    (topk, dict(z=P + 2), BAD), (topk, dict(rows=1 << 28), LIMIT), (topk, dict(rows=0, z=None), OK),
    (loss, dict(k=0), BAD), (loss, dict(k=1025), LIMIT), (loss, dict(vocab=0), BAD), (loss, dict(pitch=63), BAD), (loss, dict(tau=0.0), BAD),
    (loss, dict(dtype=2), UNSUPPORTED), (loss, dict(vd=2), UNSUPPORTED), (loss, dict(i=None), BAD), (loss, dict(v=None), BAD), (loss, dict(st=None), BAD),
    (loss, dict(lg=None), BAD), (loss, dict(out=None), BAD), (loss, dict(r=P + 2), BAD), (loss, dict(w=P + 2), BAD), (loss, dict(st=P + 4), BAD),
    (loss, dict(rows=0, z=None), OK),
    (grad, dict(up=None), BAD), (grad, dict(g=None), BAD), (grad, dict(gp=63), BAD), (grad, dict(stride=-1), BAD), (grad, dict(g=P + 2), BAD), (grad, dict(rows=0), OK),
    (grad, dict(g=P + 16), BAD), (grad, dict(g=P, gp=65), BAD),
    (step, dict(out=None), BAD), (step, dict(g=None), BAD), (step, dict(gp=63), BAD), (step, dict(g=P + 2), BAD), (step, dict(rows=0), OK), (step, dict(g=P - 64), BAD),
    (step, dict(g=P, gp=65), BAD)])
def test_calls_refused_before_any_launch(lib, call, wrong, status):
    assert call(lib, **wrong) == status
    if status != OK:
        assert len(lib.mab_last_error()) > 10


def test_cpu_tensors_and_shapes_are_refused(lib):
    import ista_daslab_optimizers_b200 as pkg
    from ista_daslab_optimizers_b200._native import NativeError
    x, i, v = torch.zeros(4, 64), torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 8)
    codes = torch.zeros(4, 64, dtype=torch.int8)
    for call in (lambda: pkg.quantize_rows(x), lambda: pkg.topk_logits(x, 3), lambda: pkg.distill_step(x, i, v), lambda: pkg.distill_loss(x, i, v),
                 lambda: pkg.int8_matmul(codes, codes, x[:, 0], x[:, 0])):
        with pytest.raises(NativeError, match='no CPU implementation'):
            call()
    with pytest.raises(NativeError, match='two-dimensional'):
        pkg.quantize_rows(x[0])
    with pytest.raises(NativeError, match='no gradient for rest'):
        pkg.distill_loss(x, i, v, torch.zeros(4, requires_grad=True))


def test_plain_form_of_the_loss_is_the_gradient_it_says():
    """The 64-bit form the kernels are held to, against autograd on the definition."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(3, 50, generator=g, dtype=torch.float64, requires_grad=True)
    idx = torch.tensor([[4, 9, -1, 7], [1, 1, 30, 49], [0, 2, 50, 3]], dtype=torch.int32)
    val, rest, w = torch.randn(3, 4, generator=g).double(), torch.randn(3, generator=g).double(), torch.tensor([0.5, 2.0, 1.0], dtype=torch.float64)
    tau = 1.7
    total = 0.0
    for r in range(3):
        q = torch.softmax(z[r] / tau, 0)
        entries = [(int(i), float(v) / tau) for i, v in zip(idx[r], val[r]) if 0 <= i < 50]
        lp = torch.logsumexp(torch.tensor([t for _, t in entries] + [float(rest[r])], dtype=torch.float64), 0)
        others = [c for c in range(50) if c not in {i for i, _ in entries}]
        l = sum(math.exp(t - lp) * (t - lp - q[i].log()) for i, t in entries)
        l = l + math.exp(rest[r] - lp) * (rest[r] - lp - q[others].sum().log())
        total = total + w[r] * l
    want, = torch.autograd.grad(total, z)
    loss, grad, _ = D.distill(z.detach(), idx, val, rest, w, tau)
    assert abs(float(loss.sum() - total)) < 1e-12
    assert (grad - want).abs().max() < 1e-12


@pytest.mark.parametrize('call,wrong', [
    (quant, dict(c=P)), (quant, dict(c=P + 4 * 64 * 4 - 1)), (quant, dict(c=P - 255)), (quant, dict(c=P + 4096, s=P + 1020)), (quant, dict(c=P + 4096, s=P + 4096 + 252)),
    (quant, dict(xp=128, c=P + 255, cp=512)), (quant, dict(xp=128, c=P + 449, cp=512)), (quant, dict(xp=128, c=P + 256, cp=500)),
    (matmul, dict(a=P, b=P + 4096, sa=P + 8192, sb=P + 8256, out=P + 128)), (matmul, dict(a=P, b=P + 4096, sa=P + 8192, sb=P + 8256, out=P + 4096 - 4)),
    (matmul, dict(a=P, b=P + 4096, sa=P + 8192, sb=P + 8256, out=P + 8192 + 12)), (matmul, dict(a=P, b=P + 4096, sa=P + 8192, sb=P + 8256, out=P + 8256 - 124)),
    (matmul, dict(a=P, b=P + 4096, sa=P + 8192, sb=P + 8256, bias=P + 16384, out=P + 16384 + 28)),
    (topk, dict(v=P + 1020, i=P + 8192, r=P + 12288)), (topk, dict(v=P + 4096, i=P + 4096 + 124, r=P + 12288)), (topk, dict(v=P + 4096, i=P + 8192, r=P + 8192 + 124)),
    (topk, dict(v=P + 4096, i=P + 8192, r=P)),
    (grad, dict(z=P, i=P + 4096 + 1020)), (grad, dict(lg=P + 4096 - 124)), (grad, dict(st=P + 4096)), (grad, dict(w=P + 4096 + 1020)), (grad, dict(up=P + 4096 - 48, stride=4)),
    (step, dict(i=P + 4096 + 1020)), (step, dict(v=P + 4096 - 124)), (step, dict(v=P + 4096 - 60, vd=1)), (step, dict(r=P + 4096)), (step, dict(w=P + 4096 + 1020)), (step, dict(out=P + 4096))])
def test_overlapping_memory_is_refused(lib, call, wrong):
    """What a call writes lies over what it reads, or over what else it writes, by as little as a byte."""
    assert call(lib, **wrong) == BAD
    assert b'overlap' in lib.mab_last_error()


def test_arguments_that_are_no_tensors_are_refused(lib):
    import ista_daslab_optimizers_b200 as pkg
    from ista_daslab_optimizers_b200._native import NativeError
    x, i, v, r, c = torch.zeros(4, 64), torch.zeros(4, 8, dtype=torch.int32), torch.zeros(4, 8), torch.zeros(4), torch.zeros(4, 64, dtype=torch.int8)
    for other in ([1.0], 3, 'x'):
        for name, call in (('x', lambda o: pkg.quantize_rows(o)), ('codes', lambda o: pkg.quantize_rows(x, o)), ('scales', lambda o: pkg.quantize_rows(x, None, o)),
                           ('a', lambda o: pkg.int8_matmul(o, c, r, r)), ('b', lambda o: pkg.int8_matmul(c, o, r, r)), ('a_scales', lambda o: pkg.int8_matmul(c, c, o, r)),
                           ('b_scales', lambda o: pkg.int8_matmul(c, c, r, o)), ('bias', lambda o: pkg.int8_matmul(c, c, r, r, o)), ('out', lambda o: pkg.int8_matmul(c, c, r, r, None, o)),
                           ('logits', lambda o: pkg.topk_logits(o, 3)), ('logits', lambda o: pkg.distill_loss(o, i, v)), ('indices', lambda o: pkg.distill_loss(x, o, v)),
                           ('values', lambda o: pkg.distill_loss(x, i, o)), ('rest', lambda o: pkg.distill_loss(x, i, v, o)), ('weights', lambda o: pkg.distill_loss(x, i, v, r, o)),
                           ('indices', lambda o: pkg.distill_step(x, o, v)), ('values', lambda o: pkg.distill_step(x, i, o))):
            with pytest.raises(NativeError, match=name + ' must be a tensor'):
                call(other)
    for call in (lambda: pkg.distill_step(x, None, v), lambda: pkg.distill_loss(x, i, None), lambda: pkg.int8_matmul(c, c, None, r)):
        with pytest.raises(NativeError, match='must be a tensor'):
            call()


def split_entropy(p, idx):
    """Sum over the indices of a list of p H(p_j / p), p the sum of their entries' p_j: by how much terms of their own lie below those of merged entries."""
    h = 0.0
    for i in set(idx):
        parts = [x for x, j in zip(p, idx) if j == i]
        h -= sum(x * math.log(x / sum(parts)) for x in parts)
    return h


def test_repeated_indices_against_merged_entries():
    """A list with repeated indices has the gradient of the list in which they are one entry each, and its loss less the entropy of the split."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(1, 30, generator=g, dtype=torch.float64) * 2
    idx, val, rest = [4, 9, 4, 7, 9, 4], torch.randn(1, 6, generator=g).double(), torch.randn(1, generator=g).double()
    merged = sorted(set(idx))
    sums = torch.stack([torch.logsumexp(val[0, [n for n, j in enumerate(idx) if j == i]], 0) for i in merged])[None]
    one = D.distill(z, torch.tensor([idx], dtype=torch.int32), val, rest, None, 1.0)
    two = D.distill(z, torch.tensor([merged], dtype=torch.int32), sums, rest, None, 1.0)
    p = torch.softmax(torch.cat([val, rest[:, None]], 1), 1)[0, :6].tolist()
    assert abs(float(two[0] - one[0]) - split_entropy(p, idx)) < 1e-12
    assert (one[1] - two[1]).abs().max() < 1e-12
    # two equal entries on a token that the student is sure of
    z = torch.full((1, 5), -100.0, dtype=torch.float64)
    z[0, 2] = 100.0
    loss = D.distill(z, torch.tensor([[2, 2]], dtype=torch.int32), torch.zeros(1, 2), None, None, 1.0)[0]
    assert abs(float(loss) + math.log(2)) < 1e-12
