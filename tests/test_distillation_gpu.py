"""The distillation operators against plain forms in 64 bits (distill_cases.py, which derives the tolerances): types, odd sizes, offsets, distances of
rows, masks, ties, infinities and NaN, and a run of them together in front of the optimizer's step."""
import math

import pytest
import torch

import distill_cases as D

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
INF = math.inf


def _gen(seed):
    return torch.Generator('cuda').manual_seed(seed)


def _normal(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device='cuda') * scale


def _placed(x, dtype, skip=0, gap=0):
    """x in rows `gap` further apart than they are long, starting `skip` elements into a buffer; what lies between is NaN (or 77)."""
    rows, cols = x.shape
    buf = torch.full((skip + rows * (cols + gap) + 16,), 77 if dtype == torch.int8 else math.nan, dtype=dtype, device='cuda')
    out = buf[skip:skip + rows * (cols + gap)].view(rows, cols + gap)[:, :cols]
    out.copy_(x)
    return out


# ------------------------------------------------------------------------------------------------ quantize_rows

@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,cols,skip,gap', [(1, 1, 0, 0), (3, 5, 1, 0), (1, 4096, 0, 0), (7, 257, 3, 2), (130, 64, 0, 8), (5, 767, 0, 0), (33, 8191, 0, 0),
                                                (2, 16384, 0, 0), (2, 40001, 1, 3), (3, 70000, 0, 0)])
def test_quantize_rows(dtype, rows, cols, skip, gap):
    from ista_daslab_optimizers_b200 import quantize_rows
    g = _gen(rows * 1000 + cols)
    x = _normal(g, rows, cols) * (0.01 + 100 * torch.rand(rows, 1, generator=g, device='cuda'))
    x = _placed(x.to(dtype), dtype, skip, gap)
    codes, scales = quantize_rows(x)
    want, want_scales = D.quantize(x)
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes, want)
    assert codes.stride(0) % 16 == 0 or rows == 1


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_quantize_rows_values_next_to_a_half(dtype):
    """Rows whose scale is a power of two times 1 or an odd mantissa, with every half-integer multiple of it and its neighbours."""
    from ista_daslab_optimizers_b200 import quantize_rows
    rows = []
    for s in (1.0, 2.0 ** -20, 0.7, 1.9999999, 3.0e-38, 1.1754944e-38, 1e36, 0.33333334):
        s = torch.tensor(s, dtype=F32)
        half = (torch.arange(-127, 127).float() + 0.5) * s
        near = torch.cat([half, torch.nextafter(half, half * 2), torch.nextafter(half, half * 0), torch.arange(-126, 127).float() * s])
        near = near.clamp(-127 * s, 127 * s)
        rows.append(torch.cat([127 * s[None], near]))
    x = torch.stack(rows).cuda().to(dtype)
    x = torch.cat([x, torch.zeros_like(x[:1]), torch.full_like(x[:1], 1e-40)])
    codes, scales = quantize_rows(x)
    want, want_scales = D.quantize(x)
    assert torch.equal(scales, want_scales)
    assert torch.equal(codes, want)


def test_quantize_rows_non_finite_and_given_outputs():
    from ista_daslab_optimizers_b200 import quantize_rows
    x = _normal(_gen(5), 6, 300)
    x[1, 7], x[2, 299], x[3, 0], x[4, :] = INF, math.nan, -INF, 0.0
    buf = torch.full((8, 304), 55, dtype=torch.int8, device='cuda')
    scales = torch.full((8,), 5.0, device='cuda')
    quantize_rows(x, buf[1:7, 2:302], scales[1:7])
    want, want_scales = D.quantize(x)
    assert torch.equal(scales[1:7].nan_to_num(9.0), want_scales.nan_to_num(9.0)) and torch.equal(buf[1:7, 2:302], want)
    assert (buf[0] == 55).all() and (buf[7] == 55).all() and (buf[:, :2] == 55).all() and (buf[:, 302:] == 55).all()
    assert scales[0] == 5.0 and scales[7] == 5.0


# ------------------------------------------------------------------------------------------------ int8_matmul

def _codes(g, rows, cols, extreme=False):
    c = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device='cuda')[:, :cols]
    c.copy_(torch.full((rows, cols), -128, device='cuda') if extreme else torch.randint(-128, 128, (rows, cols), generator=g, device='cuda'))
    return c


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('m,n,k,bias', [
    (1, 1, 1, False), (1, 130, 16, True), (2, 77, 767, False), (3, 1000, 129, True), (4, 4096, 4096, False), (5, 128, 128, True), (5, 130, 100, False),
    (16, 300, 1000, False), (17, 129, 31, True), (31, 1024, 4096, False), (41, 257, 2049, True), (64, 128, 8192, False), (65, 300, 640, True), (65, 300, 6400, True), (100, 1001, 8190, False), (128, 513, 6145, True),
    (128, 256, 255, False), (129, 511, 513, True), (256, 384, 1024, False), (257, 1025, 767, True), (300, 2048, 512, False), (777, 515, 129, False),
    (70, 9500, 300, True), (129, 9729, 1025, False), (300, 5000, 1, False), (777, 5003, 767, True), (2048, 1300, 257, False), (1025, 2305, 2048, True)])
def test_int8_matmul(dtype, m, n, k, bias):
    from ista_daslab_optimizers_b200 import int8_matmul
    g = _gen(m * 7 + n * 3 + k)
    a, b = _codes(g, m, k), _codes(g, n, k)
    sa, sb = torch.rand(m, generator=g, device='cuda') + 0.01, torch.rand(n, generator=g, device='cuda') * 0.01
    bs = _normal(g, n, scale=50.0) if bias else None
    buf = torch.full((m + 2, n + 3), 7.0, dtype=dtype, device='cuda')
    out = int8_matmul(a, b, sa, sb, bs, out=buf[1:m + 1, 1:n + 1])
    want, tol = D.matmul(a, b, sa, sb, bs)
    D.assert_near(out, want, tol + (0 if dtype == F32 else D.half_step(dtype) * want.abs()), 'product')
    assert (buf[0] == 7).all() and (buf[m + 1] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, n + 1:] == 7).all()
    assert torch.equal(int8_matmul(a, b, sa, sb, bs, dtype=dtype), out)


@pytest.mark.parametrize('m', [1, 7, 200])
def test_int8_matmul_longest_sum_and_special_scales(m):
    from ista_daslab_optimizers_b200 import int8_matmul, _native as N
    k = N.MAB_MAX_INNER
    a, b = _codes(None, m, k, extreme=True), _codes(None, 150, k, extreme=True)
    sa, sb = torch.ones(m, device='cuda'), torch.ones(150, device='cuda')
    sb[3], sb[4] = math.nan, 0.0
    out = int8_matmul(a, b, sa, sb, dtype=F32)
    want = torch.full((m, 150), float(k * 16384), device='cuda')
    want[:, 4] = 0.0
    assert out[:, 3].isnan().all()
    keep = [i for i in range(150) if i != 3]
    assert torch.equal(out[:, keep], want[:, keep])          # 131071 * 2^14 is exact in fp32


# ------------------------------------------------------------------------------------------------ topk_logits

def _check_topk(z, k, tau):
    from ista_daslab_optimizers_b200 import topk_logits
    values, indices, rest = topk_logits(z, k, tau)
    w_values, w_indices, w_rest = D.topk(z, k, tau)
    assert torch.equal(indices, w_indices)
    assert torch.equal(values.nan_to_num(123.0), w_values.nan_to_num(123.0)) and torch.equal(values.isnan(), w_values.isnan())
    assert values.dtype == z.dtype
    D.assert_near(rest, w_rest, D.sum_error(z.shape[1]) + 2 * D.U * w_rest.abs().nan_to_num(0.0, posinf=0.0, neginf=0.0), 'rest')


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,vocab,k,tau,skip,gap', [
    (1, 1, 1, 1.0, 0, 0), (3, 2, 1, 1.0, 1, 0), (2, 7, 7, 2.0, 1, 2), (4, 1000, 1, 0.7, 0, 0), (5, 50257, 20, 1.0, 0, 0), (3, 50257, 257, 2.0, 1, 6),
    (1, 128256, 64, 1.0, 0, 0), (2, 151936, 1000, 1.0, 3, 0), (150, 4097, 33, 1.0, 0, 0), (300, 2048, 1024, 1.0, 0, 0), (300, 30000, 512, 1.3, 1, 1),
    (160, 128256, 64, 2.0, 0, 0), (2, 1 << 20, 1024, 1.0, 0, 0), (200, 1024, 1024, 1.0, 0, 0), (149, 16384, 100, 1.0, 0, 0), (149, 16391, 1024, 1.0, 5, 0)])
def test_topk_logits(dtype, rows, vocab, k, tau, skip, gap):
    g = _gen(rows + vocab + k)
    z = _normal(g, rows, vocab, scale=3.0)
    _check_topk(_placed(z.to(dtype), dtype, skip, gap), k, tau)


@pytest.mark.parametrize('rows', [1, 3, 40, 70])
@pytest.mark.parametrize('step', [0.015625, 1.0, 50.0])
def test_topk_logits_of_slopes(rows, step):
    """Few rows are shared by several blocks, whose lists are merged; on a slope they lie far from one another."""
    for k in (7, 20, 33, 48, 65, 100, 128, 200, 300, 513, 1000):
        z = (torch.arange(40001, device='cuda').float() * step).expand(rows, 40001).clone()
        _check_topk(z, k, 1.0)
        _check_topk(z.flip(1).contiguous(), k, 3.0)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows', [2, 301])
@pytest.mark.parametrize('kind', ['equal', 'zeros', 'two', 'ascending', 'descending', 'late', 'masked', 'lowest', 'few', 'none', 'inf', 'many_inf', 'nan',
                                  'all_nan', 'gap', 'large', 'blocks'])
def test_topk_logits_kinds(dtype, rows, kind):
    vocab, k = 40001, 65
    g = _gen(rows)
    z = _normal(g, rows, vocab, scale=2.0)
    low = torch.finfo(dtype).min
    if kind == 'equal':
        z[:] = 1.5
    elif kind == 'zeros':
        z = torch.where(z > 0, 0.0, -0.0)
    elif kind == 'two':
        z = torch.where(z > 2.0, 1.0, 0.5)
    elif kind == 'ascending':
        z = torch.arange(vocab, device='cuda').float().div(64.0).expand(rows, vocab).clone()
    elif kind == 'descending':
        z = torch.arange(vocab, 0, -1, device='cuda').float().div(64.0).expand(rows, vocab).clone()
    elif kind == 'late':                             # the first half is masked
        z[:, :vocab // 2] = -1e4
    elif kind == 'masked':
        z[torch.rand(rows, vocab, generator=g, device='cuda') < 0.7] = -INF
    elif kind == 'lowest':                           # fewer numbers than k, the rest the type's lowest
        z[:, 40:] = low
    elif kind == 'few':
        z[:, 40:] = -INF
    elif kind == 'none':
        z[:] = -INF
    elif kind == 'inf':
        z[:, 17::5000] = INF
    elif kind == 'many_inf':
        z[:, 17::100] = INF
    elif kind == 'nan':
        z[0, 5::1000] = math.nan
        z[-1, 39000] = math.nan
    elif kind == 'all_nan':
        z[:, 30:] = math.nan
    elif kind == 'gap':                              # the rest is far below the list
        z[:, 500::600] += 400.0
        z[:, 500 + 600 * k:] = -7.0
    elif kind == 'large':
        z *= 1e30
    elif kind == 'blocks':                           # one value per stretch, rising late
        z = (torch.arange(vocab, device='cuda') // 9000).float().expand(rows, vocab).clone()
    _check_topk(z.to(dtype), k, 1.0)


# ------------------------------------------------------------------------------------------------ distillation

def _problem(rows, vocab, k, dtype, v_dtype, tau, rest, masked, ragged, skip=0, gap=0, seed=0):
    g = _gen(seed + rows + vocab + k)
    teacher = _normal(g, rows, vocab, scale=2.0)
    z = _placed((teacher * 0.7 + _normal(g, rows, vocab)).to(dtype), dtype, skip, gap)
    val, idx = torch.topk(teacher, k)
    idx = idx.int()
    r = torch.logsumexp(teacher.scatter(1, idx.long(), -INF) / tau, 1) if rest else None
    if ragged:
        idx[torch.rand(rows, k, generator=g, device='cuda') < 0.4] = -1
    w = None
    if masked:
        w = torch.rand(rows, generator=g, device='cuda') * 3 - 1
        w[::3] = 0.0
    return z, idx, val.to(v_dtype), r, w


def _check_distill(z, idx, val, rest, w, tau, what=''):
    from ista_daslab_optimizers_b200 import distill_loss, distill_step
    want = D.distill(z, idx, val, rest, w, tau)
    loss, grad = distill_step(z, idx, val, rest, w, tau)
    D.assert_distill(loss, grad, want, z.shape[1], 'step ' + what)
    leaf = z.detach().clone().requires_grad_() if z.is_contiguous() else z.detach().requires_grad_()
    out = distill_loss(leaf, idx, val, rest, w, tau)
    g, = torch.autograd.grad(out.sum(), leaf)
    D.assert_distill(out.detach(), g, want, z.shape[1], 'loss ' + what)
    z.requires_grad_(False)
    return loss, grad


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,vocab', [(2, 40001), (60, 700), (500, 3001)])
@pytest.mark.parametrize('kind', ['lowest_list', 'huge_list', 'huge_rest', 'lowest_logits', 'lowest_list_and_logits', 'far_below', 'no_logits', 'nan_and_no_teacher', 'nan_in_list', 'nan_in_list_alone'])
def test_distill_far_from_zero(dtype, rows, vocab, kind):
    """Masks of the type's lowest value that leave a row of the teacher or the student nothing, and logits so large that sums with ordinary ones lose those."""
    g = _gen(rows + vocab)
    k, low = 37, torch.finfo(dtype).min
    z = _normal(g, rows, vocab, scale=3.0)
    idx = torch.randint(0, vocab, (rows, k), generator=g, device='cuda', dtype=torch.int32)
    val = _normal(g, rows, k)
    rest = _normal(g, rows)
    if kind in ('lowest_list', 'lowest_list_and_logits'):
        val[:], rest[:] = low, -INF
    if kind == 'huge_list':
        val = val * 2.0 ** 55
    if kind == 'huge_rest':
        rest = rest.abs() * 2.0 ** 60
    if kind in ('lowest_logits', 'lowest_list_and_logits'):
        z[:] = low
        z[::2, 5] = 0.75 * low
    if kind == 'far_below':                          # every logit of the list but a few is -inf, the others far below 0
        z -= 3000.0
        z.scatter_(1, idx[:, :30].long(), -INF)
        val[:, :30], rest = -INF, None
    if kind == 'nan_and_no_teacher':
        val[:], rest[:] = -INF, -INF
        z[::2, ::97] = math.nan
    if kind == 'nan_in_list':
        z.scatter_(1, idx.long(), -2000.0)
        z[0, idx[0, 3]] = math.nan
    if kind == 'nan_in_list_alone':
        z = torch.full_like(z, -INF).scatter_(1, idx.long(), 1.0)
        z[0, idx[0, 3]] = math.nan
    if kind == 'no_logits':
        z[::2] = -INF
    _check_distill(z.to(dtype), idx, val.to(dtype), rest, None, 1.0 if kind != 'huge_list' else 2.0)


@pytest.mark.parametrize('k', [1, 100])
def test_distill_around_the_default_shared_memory(k):
    """Rows that a block holds whole, from 44 to 49 KB with its list."""
    from ista_daslab_optimizers_b200 import distill_loss, distill_step
    g = _gen(k)
    for vocab in range(11200 - 3 * k, 12500 - 3 * k, 50):
        z = _normal(g, 500, vocab)
        idx = torch.randint(0, vocab, (500, k), generator=g, device='cuda', dtype=torch.int32)
        val = _normal(g, 500, k)
        loss, _ = distill_step(z, idx, val)
        assert torch.equal(distill_loss(z, idx, val), loss)
        if vocab % 500 == 0:
            _check_distill(z, idx, val, None, None, 1.0)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,vocab,k,v_dtype,tau,rest,masked,ragged,skip,gap', [
    (1, 1, 1, F32, 1.0, False, False, False, 0, 0), (2, 2, 1, F32, 1.0, True, False, False, 1, 0), (3, 9, 9, BF16, 2.0, False, False, False, 1, 3),
    (4, 1000, 5, F32, 0.7, True, True, False, 0, 0), (60, 50257, 32, F32, 1.0, False, False, True, 0, 0), (5, 50257, 257, BF16, 1.5, True, False, False, 1, 6),
    (1, 128256, 64, F32, 2.0, True, False, False, 0, 0), (2, 151936, 1000, F32, 1.0, True, False, True, 3, 0), (150, 4097, 33, BF16, 1.0, True, True, True, 0, 0),
    (300, 2048, 1024, F32, 1.0, True, False, False, 0, 0), (300, 30001, 512, F32, 1.3, False, True, True, 1, 1), (2, 1 << 20, 1024, F32, 1.0, True, False, False, 0, 0),
    (310, 5003, 7, F32, 4.0, True, True, False, 0, 5)])
def test_distill(dtype, rows, vocab, k, v_dtype, tau, rest, masked, ragged, skip, gap):
    _check_distill(*_problem(rows, vocab, k, dtype, v_dtype, tau, rest, masked, ragged, skip, gap), tau)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows', [3, 320])
def test_distill_masks_and_indices(dtype, rows):
    """Entries that are absent, out of range, repeated; a row without a teacher; vocabularies masked by -inf and by the type's lowest value."""
    vocab, k, tau = 20011, 40, 1.0
    z, idx, val, rest, _ = _problem(rows, vocab, k, dtype, F32, tau, True, False, False)
    idx[0] = -1
    idx[1, 3:] = vocab
    idx[1, 7], idx[1, 8] = 2 ** 31 - 1, -2 ** 31
    _check_distill(z, idx, val, rest, None, tau, 'absent')
    idx[2, 10:30] = idx[2, 5].item()
    idx[2, 39] = idx[2, 0].item()
    _check_distill(z, idx, val, rest, None, tau, 'repeated')
    loss, grad = _check_distill(z, idx, val, None, None, tau, 'no rest')
    assert loss[0] == 0 and (grad[0] == 0).all()
    r2 = rest.clone()
    r2[0] = -INF                                     # neither entries nor a rest
    loss, grad = _check_distill(z, idx, val, r2, None, tau, 'no teacher')
    assert loss[0] == 0 and (grad[0] == 0).all()
    for low in (-INF, torch.finfo(dtype).min):
        y = z.clone()
        y[:, vocab - 100:] = low
        keep = idx.clone()
        keep[keep >= vocab - 100] = -1
        _check_distill(y, keep, val, rest, None, tau, f'columns {low}')
        y[:] = low                                   # only the list is left
        y.scatter_(1, keep.clamp(0, vocab - 1).long(), 1.0)
        _check_distill(y, keep, val, None, None, tau, f'list only {low}')
    v2 = val.clone()
    v2[:, 20:] = -INF                                # listed, with nothing
    _check_distill(z, idx, v2, rest, None, tau, 'empty entries')


def test_distill_skipped_rows_are_not_looked_at():
    from ista_daslab_optimizers_b200 import distill_loss, distill_step
    z, idx, val, rest, w = _problem(9, 3001, 8, F32, F32, 1.0, True, True, False)
    z[::3] = math.nan
    loss, grad = distill_step(z, idx, val, rest, w)
    assert (loss[::3] == 0).all() and (grad[::3] == 0).all() and torch.isfinite(loss).all() and torch.isfinite(grad).all()
    leaf = z.clone().requires_grad_()
    out = distill_loss(leaf, idx, val, rest, w)
    out.backward(torch.full_like(out, INF).where(w == 0, torch.ones_like(out)))
    assert (leaf.grad[::3] == 0).all() and torch.isfinite(leaf.grad).all()
    bad, bad_grad = distill_step(z, idx, val, rest, None)
    assert bad[::3].isnan().all() and bad_grad[::3].isnan().all() and torch.isfinite(bad[1::3]).all()


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('skip,gap', [(0, 0), (1, 3)])
def test_distill_step_in_place_and_elsewhere(dtype, skip, gap):
    from ista_daslab_optimizers_b200 import distill_step
    z, idx, val, rest, w = _problem(20, 9001, 50, dtype, F32, 1.0, True, True, True, skip, gap)
    loss, grad = distill_step(z, idx, val, rest, w)
    other = _placed(torch.zeros_like(z), dtype, 2, 5)      # another offset than the logits'
    loss2, g2 = distill_step(z, idx, val, rest, w, grad=other)
    assert g2.data_ptr() == other.data_ptr() and torch.equal(g2, grad) and torch.equal(loss, loss2)
    loss3, g3 = distill_step(z, idx, val, rest, w, grad=z)
    assert torch.equal(z, grad) and torch.equal(loss3, loss)
    gaps = z.as_strided((20, 9001 + gap), (9001 + gap, 1), z.storage_offset())[:, 9001:]
    assert gap == 0 or gaps.isnan().all()


def test_distill_gradient_against_differences():
    """Central differences of the loss kernel itself: f(z + h) - f(z - h) = 2 h f' + O(h^3 f'''), with |f'''| <= 2 / tau^3 for a mixture of log-sum-exps, and the
    loss's own error on both sides."""
    from ista_daslab_optimizers_b200 import distill_loss
    tau, vocab, k, h = 1.5, 200, 10, 0.05
    z, idx, val, rest, _ = _problem(1, vocab, k, F32, F32, tau, True, False, False)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(distill_loss(leaf, idx, val, rest, None, tau).sum(), leaf)
    step = h * torch.eye(vocab, device='cuda')
    rows = lambda t: t.expand(vocab, *t.shape[1:]).contiguous()      # noqa: E731
    up, down = z + step, z - step
    wide = (up.diagonal() - down.diagonal()).double()
    f = [distill_loss(x, rows(idx), rows(val), rows(rest), None, tau).double() for x in (up, down)]
    slope = (f[0] - f[1]) / wide
    tol = h * h / 6 * 2 / tau ** 3 + 2 * (D.sum_error(vocab) + 2 * D.U * 5) / (2 * h)
    D.assert_near(grad[0], slope, tol, 'slope')


def test_distill_broadcast_upstream_gradient():
    from ista_daslab_optimizers_b200 import distill_loss
    z, idx, val, rest, _ = _problem(6, 3000, 16, F32, F32, 1.0, True, False, False)
    leaf = z.clone().requires_grad_()
    g = torch.autograd.grad(distill_loss(leaf, idx, val, rest).mean(), leaf)[0]          # a gradient of distance 0
    up = torch.arange(12, device='cuda').float()
    every, = torch.autograd.grad(distill_loss(leaf, idx, val, rest), leaf, up[::2])       # ... and of distance 2
    one = D.distill(z, idx, val, rest, None, 1.0)
    tol = (D.sum_error(3000) + 72 * D.U) * one[2] + 2 * D.U * one[1].abs() + 2.0 ** -126
    D.assert_near(g, one[1] / 6, tol / 6, 'mean')
    D.assert_near(every, one[1] * up[::2, None].double(), tol * up[::2, None], 'rows')


def test_distill_saved_logits_cannot_change_unnoticed():
    from ista_daslab_optimizers_b200 import distill_loss
    z, idx, val, rest, _ = _problem(2, 500, 4, F32, F32, 1.0, True, False, False)
    leaf = z.clone().requires_grad_()
    y = leaf * 1.0
    loss = distill_loss(y, idx, val, rest)
    y.detach().mul_(2.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.sum().backward()


def test_outputs_that_autograd_keeps_are_noticed():
    """A step whose gradient replaces logits that something has saved for its own backward pass: that pass refuses."""
    from ista_daslab_optimizers_b200 import distill_step
    z, idx, val, rest, _ = _problem(3, 500, 4, F32, F32, 1.0, True, False, False)
    logits = (z.clone().requires_grad_() * 1.0).exp()      # exp saves its result
    distill_step(logits.detach(), idx, val, rest, grad=logits.detach())
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        logits.sum().backward()


def test_distill_twice_differentiated_is_refused():
    from ista_daslab_optimizers_b200 import distill_loss
    z, idx, val, rest, _ = _problem(3, 500, 4, F32, F32, 1.0, True, False, False)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(distill_loss(leaf, idx, val, rest).sum(), leaf, create_graph=True)
    D.assert_distill(distill_loss(leaf, idx, val, rest).detach(), grad.detach(), D.distill(z, idx, val, rest, None, 1.0), 500, 'with a graph')
    with pytest.raises(RuntimeError, match='differentiable once'):
        grad.sum().backward()


def test_nothing_to_do():
    from ista_daslab_optimizers_b200 import distill_loss, distill_step, int8_matmul, quantize_rows, topk_logits
    e = lambda *s, dtype=F32: torch.empty(*s, dtype=dtype, device='cuda')      # noqa: E731
    codes, scales = quantize_rows(e(0, 64))
    assert codes.shape == (0, 64) and scales.shape == (0,)
    assert int8_matmul(codes, e(5, 64, dtype=torch.int8), scales, e(5)).shape == (0, 5)
    assert int8_matmul(e(5, 64, dtype=torch.int8), codes, e(5), scales).shape == (5, 0)
    assert [tuple(t.shape) for t in topk_logits(e(0, 100), 3)] == [(0, 3), (0, 3), (0,)]
    idx, val = e(0, 3, dtype=torch.int32), e(0, 3)
    assert [tuple(t.shape) for t in distill_step(e(0, 100), idx, val)] == [(0,), (0, 100)]
    leaf = e(0, 100).requires_grad_()
    distill_loss(leaf, idx, val).sum().backward()
    assert leaf.grad.shape == (0, 100)


@pytest.mark.parametrize('call,match', [
    (lambda P, z, i, v, r: P.quantize_rows(z.half()), 'element type'), (lambda P, z, i, v, r: P.quantize_rows(z.t()), 'contiguous'),
    (lambda P, z, i, v, r: P.quantize_rows(z[0].expand(6, -1)), 'overlap'), (lambda P, z, i, v, r: P.quantize_rows(z, z), 'element type'),
    (lambda P, z, i, v, r: P.quantize_rows(z, scales=r.double()), 'scales must be'), (lambda P, z, i, v, r: P.quantize_rows(z, scales=r[:5]), 'scales must be'),
    (lambda P, z, i, v, r: P.quantize_rows(z.clone().requires_grad_()), 'no gradient'),
    (lambda P, z, i, v, r: P.topk_logits(z, 65), 'between 1 and'), (lambda P, z, i, v, r: P.topk_logits(z, 0), 'between 1 and'),
    (lambda P, z, i, v, r: P.topk_logits(z, 3, 0.0), 'temperature'), (lambda P, z, i, v, r: P.topk_logits(z.clone().requires_grad_(), 3), 'no gradient'),
    (lambda P, z, i, v, r: P.topk_logits(torch.zeros(2, 2000, device='cuda'), 1025), '1024'),
    (lambda P, z, i, v, r: P.distill_step(z, i.long(), v, r), 'int32'), (lambda P, z, i, v, r: P.distill_step(z, i[:5], v, r), 'must be'),
    (lambda P, z, i, v, r: P.distill_step(z, i, v[:, :3], r), 'must be'), (lambda P, z, i, v, r: P.distill_step(z, i.t().contiguous().t(), v, r), 'contiguous'),
    (lambda P, z, i, v, r: P.distill_step(z, i, v, r.cpu()), 'rest must be'), (lambda P, z, i, v, r: P.distill_step(z, i, v, r, r.double()), 'weights must be'),
    (lambda P, z, i, v, r: P.distill_step(z, i, v, r, grad=z.bfloat16()), 'grad must be'), (lambda P, z, i, v, r: P.distill_step(z, i, v, r, temperature=-1.0), 'temperature'),
    (lambda P, z, i, v, r: P.distill_step(z[:5], i[:5], v[:5], r[:5], grad=z[1:]), 'overlaps'),
    (lambda P, z, i, v, r: P.distill_loss(z, i, v.clone().requires_grad_(), r), 'no gradient for values'),
    (lambda P, z, i, v, r: P.distill_loss(z, i, v, r, temperature=1e9), 'temperature'),
    (lambda P, z, i, v, r: P.int8_matmul(z, z, r, r), 'element type'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char(), z.char()[:, :60], r, r), 'inner sizes'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char()[:, :50].contiguous(), z.char()[:, :50].contiguous(), r, r), 'multiple of 16'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char()[:, 8:56], z.char()[:, 8:56], r, r), 'start on 16'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char(), z.char(), r[:3], r), 'a_scales must be'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char(), z.char(), r, r, dtype=torch.float16), 'unsupported'),
    (lambda P, z, i, v, r: P.int8_matmul(z.char(), z.char(), r, r, out=z), 'shape')])
def test_what_is_refused(call, match):
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    z, r = torch.randn(6, 64, device='cuda'), torch.ones(6, device='cuda')
    i, v = torch.zeros(6, 4, dtype=torch.int32, device='cuda'), torch.zeros(6, 4, device='cuda')
    before = N.kernel_launch_count()
    with pytest.raises(N.NativeError, match=match):
        call(P, z, i, v, r)
    assert N.kernel_launch_count() == before


# ------------------------------------------------------------------------------------------------ together

def test_teacher_to_optimizer_step():
    """A frozen linear teacher in 8 bits, its top logits, the student's loss and gradient, the optimizer's step: each against the 64-bit form on the inputs
    it had, and the same step by autograd."""
    from ista_daslab_optimizers_b200 import MicroAdam, distill_loss, distill_step, int8_matmul, quantize_rows, topk_logits
    g = _gen(1)
    tokens, width, vocab, k, tau = 130, 256, 5003, 16, 2.0
    hidden = _normal(g, tokens, width).to(BF16)
    codes, scales = quantize_rows(_normal(g, vocab, width, scale=0.2).to(BF16))
    x, x_scales = quantize_rows(hidden)
    teacher = int8_matmul(x, codes, x_scales, scales)
    want, tol = D.matmul(x, codes, x_scales, scales, None)
    D.assert_near(teacher, want, tol + D.half_step(BF16) * want.abs(), 'teacher')
    values, indices, rest = topk_logits(teacher, k, tau)
    assert torch.equal(indices, D.topk(teacher, k, tau)[1])
    steps = []
    for by_autograd in (False, True):
        weight = torch.nn.Parameter(_normal(_gen(2), vocab, width, scale=0.1).to(BF16))
        opt = MicroAdam([weight], m=4, lr=1e-3, quant_block_size=64)
        for _ in range(2):
            student = hidden @ weight.T
            if by_autograd:
                distill_loss(student, indices, values, rest, None, tau).sum().backward()
            else:
                loss, grad = distill_step(student.detach(), indices, values, rest, None, tau)
                D.assert_distill(loss, grad, D.distill(student.detach(), indices, values, rest, None, tau), vocab, 'student')
                student.backward(grad)
            opt.step()
            opt.zero_grad()
        assert torch.isfinite(weight).all()
        steps.append(weight.detach().clone())
    assert (steps[0].float() - steps[1].float()).abs().max() < 4e-3     # two steps of lr 1e-3 each differ by at most twice as much
    assert not torch.equal(steps[0], _normal(_gen(2), vocab, width, scale=0.1).to(BF16))


def test_captured_and_replayed_with_other_streams():
    """The chain captured into a graph and replayed on new inputs gives what eager calls on another stream give, bit for bit."""
    from ista_daslab_optimizers_b200 import distill_step, int8_matmul, quantize_rows, topk_logits, _native as N
    g = _gen(3)
    codes, scales = quantize_rows(_normal(g, 3001, 512, scale=0.2))
    hidden, student = _normal(g, 70, 512).to(BF16), _normal(g, 70, 3001).to(BF16)

    def chain(h, s):
        x, xs = quantize_rows(h)
        t = int8_matmul(x, codes, xs, scales)
        v, i, r = topk_logits(t, 20)
        return (t, v, i, r) + distill_step(s, i, v, r)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(hidden, student)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(hidden, student)
    for seed in (4, 5):
        h, s = _normal(_gen(seed), 70, 512).to(BF16), _normal(_gen(seed + 10), 70, 3001).to(BF16)
        hidden.copy_(h)
        student.copy_(s)
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = chain(h, s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b)
    assert N.device_error() == 0


def test_forward_and_backward_captured_and_replayed():
    from ista_daslab_optimizers_b200 import distill_loss
    z, idx, val, rest, w = _problem(20, 5001, 12, BF16, F32, 1.0, True, True, True)
    leaf = z.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        distill_loss(leaf, idx, val, rest, w).sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = distill_loss(leaf, idx, val, rest, w)
        loss.sum().backward()
    for seed in (6, 7):
        new = _normal(_gen(seed), 20, 5001).to(BF16)
        with torch.no_grad():
            leaf.copy_(new)
            leaf.grad.zero_()
        graph.replay()
        other = new.clone().requires_grad_()
        want = distill_loss(other, idx, val, rest, w)
        want.sum().backward()
        assert torch.equal(loss, want) and torch.equal(leaf.grad, other.grad)


def test_calls_of_two_threads():
    """Two threads on streams of their own, one call behind the other without a wait between them: each has its own results."""
    import threading
    from ista_daslab_optimizers_b200 import distill_step, int8_matmul, quantize_rows, topk_logits
    results, errors = {}, []

    def work(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                g = _gen(seed)
                x, w, s = _normal(g, 90, 640).to(BF16), _normal(g, 4003, 640, scale=0.1), _normal(g, 90, 4003)
                for _ in range(10):
                    a, sa = quantize_rows(x)
                    b, sb = quantize_rows(w)
                    v, i, r = topk_logits(int8_matmul(a, b, sa, sb), 30)
                    results.setdefault(seed, []).append(distill_step(s, i, v, r))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(seed,)) for seed in (11, 12, 11, 12)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for seed in (11, 12):
        assert len(results[seed]) == 20
        for loss, grad in results[seed][1:]:
            assert torch.equal(loss, results[seed][0][0]) and torch.equal(grad, results[seed][0][1])


def test_repeated_calls_give_the_same_bits():
    from ista_daslab_optimizers_b200 import distill_step, topk_logits
    for rows in (3, 400):
        z, idx, val, rest, w = _problem(rows, 30011, 100, BF16, F32, 1.0, True, True, True)
        first = distill_step(z, idx, val, rest, w) + topk_logits(z, 100)
        for _ in range(5):
            again = distill_step(z, idx, val, rest, w) + topk_logits(z, 100)
            for a, b in zip(first, again):
                assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ kernels that begin while the one before them ends

def test_products_of_both_forms_in_a_row():
    """Tiles of one CTA (with and without a split inner size) and of two, which take all of an SM's tensor memory, behind one another without a wait: every product is
    the one that it is alone."""
    from ista_daslab_optimizers_b200 import int8_matmul, _native as N
    g = _gen(21)
    problems = []
    for m, n, k in ((16, 200, 128), (300, 3000, 128), (41, 4096, 1024), (700, 2000, 256), (5, 19000, 64), (1025, 2305, 300), (128, 400, 6400)):
        a, b = _codes(g, m, k), _codes(g, n, k)
        sa, sb = torch.rand(m, generator=g, device='cuda') + 0.01, torch.rand(n, generator=g, device='cuda') * 0.01
        torch.cuda.synchronize()
        problems.append((a, b, sa, sb, int8_matmul(a, b, sa, sb, dtype=F32)))
        torch.cuda.synchronize()
        want, tol = D.matmul(a, b, sa, sb, None)
        D.assert_near(problems[-1][4], want, tol, f'{m} x {n} x {k}')
    for _ in range(20):
        outs = [(int8_matmul(*p[:4], dtype=F32), p[4]) for p in problems + problems[::-1]]
        for out, want in outs:
            assert torch.equal(out, want)
    assert N.device_error() == 0


@pytest.mark.parametrize('m', [1, 2, 3, 4])
def test_product_reads_what_the_kernel_before_it_wrote(m):
    """A few tokens quantised into one buffer again and again, each time with the product behind it and no wait between."""
    from ista_daslab_optimizers_b200 import int8_matmul, quantize_rows
    g = _gen(31 + m)
    width, channels, times = 4096, 1500, 40
    b, sb = quantize_rows(_normal(g, channels, width, scale=0.1))
    x = _normal(g, times, m, width)
    codes, scales = torch.empty(m, width, dtype=torch.int8, device='cuda'), torch.empty(m, device='cuda')
    for _ in range(3):
        outs = []
        for i in range(times):
            quantize_rows(x[i], codes, scales)
            outs.append(int8_matmul(codes, b, scales, sb, dtype=F32))
        for i in range(times):
            c, s = D.quantize(x[i])
            want, tol = D.matmul(c, b, s, sb, None)
            D.assert_near(outs[i], want, tol, f'call {i}')
        # the weights written again, too
        wide = _normal(g, channels, width, scale=0.1)
        quantize_rows(wide, b, sb)
        out = int8_matmul(codes, b, scales, sb, dtype=F32)
        want_b, want_sb = D.quantize(wide)
        want, tol = D.matmul(c, want_b, s, want_sb, None)
        D.assert_near(out, want, tol, 'weights')


# ------------------------------------------------------------------------------------------------ hooks for saved tensors

@pytest.mark.parametrize('dtype', [F32, BF16])
def test_saved_tensors_through_hooks(dtype):
    """What is saved for the backward pass can be moved to the host, copied, or laid out otherwise meanwhile; what comes back as something else is refused."""
    from ista_daslab_optimizers_b200 import distill_loss, _native as N
    hooks = torch.autograd.graph.saved_tensors_hooks
    z, idx, val, rest, w = _problem(5, 3001, 8, dtype, F32, 1.0, True, True, False, 1, 3)

    def gradient(leaf, context=None):
        if context is None:
            loss = distill_loss(leaf, idx, val, rest, w)
        else:
            with context:
                loss = distill_loss(leaf, idx, val, rest, w)
        return torch.autograd.grad(loss.sum(), leaf)[0]

    leaf = z.detach().requires_grad_()
    want = gradient(leaf)
    turned = lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()      # noqa: E731
    for context in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), hooks(lambda t: t, torch.clone), hooks(lambda t: t, turned)):
        assert torch.equal(gradient(leaf, context), want)
    for other in (lambda t: t.cpu(), lambda t: t.double(), lambda t: t.half(), lambda t: t.to_sparse(), lambda t: t[:-1], lambda t: t.flatten(), lambda t: t[..., :1]):
        before = N.kernel_launch_count()
        with pytest.raises(RuntimeError, match='came back'):
            gradient(leaf, hooks(lambda t: t, other))
        assert N.kernel_launch_count() <= before + 1          # the loss, no gradient

    def broken(t):
        raise KeyError('a hook of the user')

    for context in (hooks(broken, lambda t: t), hooks(lambda t: t, broken)):
        with pytest.raises(KeyError, match='a hook of the user'):
            gradient(leaf, context)
    assert torch.equal(gradient(leaf), want)


# ------------------------------------------------------------------------------------------------ calls of one kernel with different sizes

def test_threads_with_different_sizes():
    """Threads whose calls are the same kernels with other amounts of shared memory: rows of other lengths, products with other inner sizes, lists of other lengths."""
    import threading
    from ista_daslab_optimizers_b200 import distill_loss, distill_step, int8_matmul, topk_logits
    g = _gen(41)
    sizes = ((9000, 640, 20), (15000, 128, 64), (12000, 300, 1000), (10000, 1024, 700))
    problems = []
    for vocab, inner, k in sizes:
        z, val = _normal(g, 500, vocab), _normal(g, 500, 20)
        idx = torch.randint(0, vocab, (500, 20), generator=g, device='cuda', dtype=torch.int32)
        a, b = _codes(g, 40, inner), _codes(g, 4000, inner)
        sa, sb = torch.rand(40, generator=g, device='cuda'), torch.rand(4000, generator=g, device='cuda')
        few = z[:6].contiguous()
        problems.append((lambda z=z, idx=idx, val=val: distill_step(z, idx, val), lambda z=z, idx=idx, val=val: (distill_loss(z, idx, val),),
                         lambda a=a, b=b, sa=sa, sb=sb: (int8_matmul(a, b, sa, sb),), lambda few=few, k=k: topk_logits(few, k)))
    want = [[call() for call in calls] for calls in problems]
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(len(problems))

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(60):
                    got = [call() for call in problems[n]]
                for outs, ref in zip(got, want[n]):
                    for x, y in zip(outs, ref):
                        assert torch.equal(x, y)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(problems))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]


def test_one_graph_with_different_sizes_of_one_kernel():
    """A captured graph holds launches of the same kernels with other amounts of shared memory, and eager calls with others still come between capture and replay."""
    from ista_daslab_optimizers_b200 import distill_step, int8_matmul
    g = _gen(43)
    inputs = []
    for vocab, inner in ((15000, 1024), (9000, 128), (12000, 640)):
        idx = torch.randint(0, vocab, (400, 20), generator=g, device='cuda', dtype=torch.int32)
        inputs.append((_normal(g, 400, vocab), idx, _normal(g, 400, 20), _codes(g, 40, inner), _codes(g, 4000, inner), torch.rand(40, generator=g, device='cuda'),
                       torch.rand(4000, generator=g, device='cuda')))

    def chain():
        outs = []
        for z, idx, val, a, b, sa, sb in inputs:
            outs += [*distill_step(z, idx, val), int8_matmul(a, b, sa, sb)]
        return outs

    want = chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain()
    small = torch.zeros(300, 8300, device='cuda')
    distill_step(small, inputs[0][1][:300, :2].contiguous() % 8300, inputs[0][2][:300, :2].contiguous())
    for _ in range(2):
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ NaN of either sign in a list

@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,vocab', [(2, 40001), (60, 700), (500, 3001), (3, 9), (300, 200000)])
@pytest.mark.parametrize('bits', ['sign', 'sign_least', 'sign_all', 'plain'])
def test_distill_nan_in_list_whatever_its_bits(dtype, rows, vocab, bits):
    """A listed logit that is NaN, with and without its sign, makes its row NaN throughout, whether the teacher gives the entry mass or not; -inf and repeated entries stay what they are."""
    g = _gen(vocab)
    k = 5
    z = _normal(g, rows, vocab).to(dtype)
    nan = dict(sign=0xFFC0, sign_least=0xFF81, sign_all=0xFFFF, plain=0x7FC0)[bits]
    idx = torch.stack([torch.randperm(vocab, generator=g, device='cuda')[:k] for _ in range(rows)]).int()
    idx[:, 4] = idx[:, 3]
    z.scatter_(1, idx[:, 2:3].long(), -INF)
    word, n = (torch.int16, nan) if dtype == BF16 else (torch.int32, nan << 16 | (0xFFFF if bits == 'sign_all' else 0))
    z.view(word)[0, idx[0, 1].item()] = n - (1 << (16 if dtype == BF16 else 32)) if n >> (15 if dtype == BF16 else 31) else n
    val = _normal(g, rows, k)
    val[:, 2] = -INF                                     # nothing where the student has nothing
    assert z.isnan().sum() == 1
    loss, grad = _check_distill(z, idx, val, None, None, 1.0, 'with mass')
    assert loss[0].isnan() and grad[0].isnan().all() and torch.isfinite(loss[1:]).all() and torch.isfinite(grad[1:]).all()
    val[:, 1] = -INF
    _, grad = _check_distill(z, idx, val, None, None, 1.0, 'without')
    assert grad[0].isnan().all() and torch.isfinite(grad[1:]).all()


# ------------------------------------------------------------------------------------------------ large logits and lowest masks at other temperatures

@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows,vocab', [(2, 40001), (60, 700), (500, 3001)])
@pytest.mark.parametrize('tau', [0.7, 0.3, 1.3, 3.0])
@pytest.mark.parametrize('kind', ['lowest_list', 'lowest_logits', 'lowest_rows', 'lowest_list_and_logits', 'huge_list', 'huge_logits', 'huge_both', 'huge_below', 'large'])
def test_distill_far_from_zero_at_other_temperatures(dtype, rows, vocab, tau, kind):
    """Lowest values divided by a temperature below 1 are beyond fp32, and quotients of 1e16 are further from their nearest float than any exponential reaches.  The plain form is the same
    as elsewhere; equal logits are equal after the division, others of that size are apart by more than an exponential sees."""
    g = _gen(rows + vocab)
    k, low = 37, torch.finfo(dtype).min
    z = _normal(g, rows, vocab, scale=3.0)
    idx = torch.stack([torch.randperm(vocab, generator=g, device='cuda')[:k] for _ in range(rows)]).int()
    val, rest = _normal(g, rows, k), _normal(g, rows)
    if kind in ('lowest_list', 'lowest_list_and_logits'):
        val[:], rest[:] = low, -INF
    if kind in ('lowest_logits', 'lowest_list_and_logits'):
        z[:] = low
    if kind == 'lowest_rows':                            # every other row masked, and so is the teacher's
        z[::2] = low
        val[::2], rest[::2] = low, -INF
    if kind in ('huge_list', 'huge_both'):               # two entries share the teacher's mass
        val[:] = 1.1e16
        val[:, 2:] = -1.1e16
        rest[:] = -INF
    if kind in ('huge_logits', 'huge_both'):
        z[:] = -1.3e16
        z.scatter_(1, idx[:, :3].long(), 1.3e16)
        val[:, 3:], rest[:] = -1.1e16, -INF
    if kind == 'huge_below':                             # all of the list and the rest at one height far below zero
        z[:], val[:], rest[:] = -7.7e15, -7.7e15, -INF
    if kind == 'large':
        z, val, rest = z * 1e3, val * 1e3, rest * 1e3
    from ista_daslab_optimizers_b200 import distill_loss, distill_step
    z, val = z.to(dtype), val.to(dtype)
    w_loss, w_grad, size = D.distill(z, idx, val, rest, None, tau)
    loss, grad = distill_step(z, idx, val, rest, None, tau)
    leaf = z.clone().requires_grad_()
    loss2 = distill_loss(leaf, idx, val, rest, None, tau)
    grad2, = torch.autograd.grad(loss2.sum(), leaf)
    for l, g, what in ((loss, grad, 'step '), (loss2.detach(), grad2, 'loss ')):
        D.assert_near(l, w_loss, D.sum_error(vocab) + 2 * D.U * w_loss.abs(), what + kind)
        # as for temperature 1, but an exponential below 2^-126 is 0 before it is multiplied by 1 / tau: off by up to 2^-126 / tau, where tau is below 1 more than 2^-126
        D.assert_near(g, w_grad, (D.sum_error(vocab) + 72 * D.U) * size + (D.half_step(dtype) * 1.001) * w_grad.abs() + 2.0 ** -126 / min(tau, 1.0), what + kind)


# ------------------------------------------------------------------------------------------------ forward-mode differentiation

@pytest.mark.parametrize('which', ['quantize x', 'matmul a_scales', 'matmul b_scales', 'matmul bias', 'topk logits', 'loss logits', 'loss leaf', 'loss values', 'loss rest', 'loss weights',
                                   'step logits', 'step values', 'step weights'])
def test_tangents_are_refused_not_lost(which):
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    from torch.autograd import forward_ad
    call, name = which.split()
    g = _gen(51)
    t = dict(x=_normal(g, 6, 64), a_scales=torch.ones(6, device='cuda'), b_scales=torch.ones(6, device='cuda'), bias=torch.ones(6, device='cuda'), logits=_normal(g, 6, 64),
             values=_normal(g, 6, 4), rest=_normal(g, 6), weights=torch.ones(6, device='cuda'))
    idx, codes = torch.zeros(6, 4, dtype=torch.int32, device='cuda'), torch.zeros(6, 64, dtype=torch.int8, device='cuda')
    calls = dict(quantize=lambda: P.quantize_rows(t['x']), matmul=lambda: P.int8_matmul(codes, codes, t['a_scales'], t['b_scales'], t['bias']),
                 topk=lambda: P.topk_logits(t['logits'], 3), loss=lambda: P.distill_loss(t['logits'], idx, t['values'], t['rest'], t['weights']),
                 step=lambda: P.distill_step(t['logits'], idx, t['values'], t['rest'], t['weights']))
    calls[call]()
    if name == 'leaf':
        name = 'logits'
        t['logits'].requires_grad_()
    with forward_ad.dual_level():
        plain = t[name]
        t[name] = forward_ad.make_dual(plain, torch.ones_like(plain))
        before = N.kernel_launch_count()
        for context in (torch.enable_grad(), torch.no_grad()):
            with context, pytest.raises(N.NativeError, match='no forward-mode derivative'):
                calls[call]()
        assert N.kernel_launch_count() == before
        t[name] = plain
        calls[call]()
    calls[call]()


def test_gradients_that_a_function_transform_asks_for_are_not_lost():
    """torch.func's tensors have no memory of their own: the operators refuse them rather than compute beside the transform."""
    from ista_daslab_optimizers_b200 import distill_loss, topk_logits
    z, idx, val, rest, _ = _problem(3, 500, 4, F32, F32, 1.0, True, False, False)
    for call in (lambda: torch.func.grad(lambda y: distill_loss(y, idx, val, rest).sum())(z), lambda: torch.vmap(lambda y: topk_logits(y[None], 3)[0])(z),
                 lambda: torch.func.jvp(lambda y: distill_loss(y, idx, val, rest), (z,), (z,))):
        with pytest.raises(RuntimeError):
            call()


# ------------------------------------------------------------------------------------------------ waits that run out

@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('m,n,k', [(5, 300, 100), (41, 4096, 4096), (64, 200, 8192), (128, 400, 6400), (65, 300, 640), (300, 5000, 64), (777, 3000, 767), (1025, 9729, 1024)])
def test_product_whose_copies_do_not_come(m, n, k, dtype):
    """As if every wait had run out: no element keeps what its memory held before, the flag is set, and the next product is right.  Nothing faults: no copy is issued."""
    from ista_daslab_optimizers_b200 import int8_matmul, _native as N
    g = _gen(m + n)
    a, b = _codes(g, m, k), _codes(g, n, k)
    sa, sb = torch.rand(m, generator=g, device='cuda'), torch.rand(n, generator=g, device='cuda')
    buf = torch.full((m + 2, n + 3), 7.0, dtype=dtype, device='cuda')
    out = buf[1:m + 1, 1:n + 1]
    assert N.device_error() == 0
    N.check(N.load().mab_int8_matmul_selftest(m, n, k, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), sa.data_ptr(), sb.data_ptr(), None, out.data_ptr(),
                                              N.MAB_F32 if dtype == F32 else N.MAB_BF16, out.stride(0), torch.cuda.current_stream().cuda_stream), 'selftest')
    assert N.device_error() == 1
    assert out.isnan().all()
    assert (buf[0] == 7).all() and (buf[m + 1] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, n + 1:] == 7).all()
    N.device_error_clear()
    int8_matmul(a, b, sa, sb, out=out)
    want, tol = D.matmul(a, b, sa, sb, None)
    D.assert_near(out, want, tol + (0 if dtype == F32 else D.half_step(dtype) * want.abs()), 'product')
    assert N.device_error() == 0


# ------------------------------------------------------------------------------------------------ memory that is shared

def test_outputs_between_the_rows_of_inputs():
    """Records that hold a row of the input and one of the output: no byte is shared, so they are taken.  An output over an input is not, whatever its type."""
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    g = _gen(61)
    rows, cols = 37, 256
    record = torch.zeros(rows, cols * 4 + cols, dtype=torch.uint8, device='cuda')      # float32 row, then its codes
    x = record.view(F32)[:, :cols]
    x.copy_(_normal(g, rows, cols))
    codes = record.view(torch.int8)[:, cols * 4:]
    _, scales = P.quantize_rows(x, codes)
    want, want_scales = D.quantize(x)
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)
    b, sb = P.quantize_rows(_normal(g, 64, cols))
    wide = torch.zeros(rows, cols + 64 * 4, dtype=torch.uint8, device='cuda')            # codes, then the product's row
    a, out = wide.view(torch.int8)[:, :cols], wide.view(F32)[:, cols // 4:]
    a.copy_(codes)
    P.int8_matmul(a, b, scales, sb, out=out)
    want, tol = D.matmul(codes, b, scales, sb, None)
    D.assert_near(out, want, tol, 'product')
    z, idx, val, rest, w = _problem(6, 64, 4, F32, F32, 1.0, True, True, False)
    before = N.kernel_launch_count()
    for call in (lambda: P.quantize_rows(x, x.view(torch.int8)[:, :cols]), lambda: P.quantize_rows(x, scales=record.view(F32).flatten()[:rows]),
                 lambda: P.int8_matmul(a, b, scales, sb, out=wide.view(F32)[:, :64])):
        with pytest.raises(N.NativeError, match='overlap'):
            call()
    buf = torch.zeros(6 * 64, device='cuda')
    for shared in (dict(indices=buf.view(torch.int32)[8:32].view(6, 4)), dict(values=buf[100:124].view(6, 4)), dict(rest=buf[378:]), dict(weights=buf[:6])):
        given = {**dict(indices=idx, values=val, rest=rest, weights=w), **shared}
        with pytest.raises(N.NativeError, match='overlaps the lists'):
            P.distill_step(z, **given, grad=buf.view(6, 64))
    assert N.kernel_launch_count() == before


def test_given_outputs_that_ask_for_a_gradient_are_refused():
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    z, idx, val, rest, _ = _problem(6, 64, 4, F32, F32, 1.0, True, False, False)
    scales, codes = torch.zeros(6, device='cuda', requires_grad=True), torch.zeros(6, 64, dtype=torch.int8, device='cuda')
    before = N.kernel_launch_count()
    with pytest.raises(N.NativeError, match='no gradient for scales'):
        P.quantize_rows(z, codes, scales)
    with pytest.raises(N.NativeError, match='no gradient for out'):
        P.int8_matmul(codes, codes, rest, rest, out=torch.zeros(6, 6, device='cuda', requires_grad=True))
    with pytest.raises(N.NativeError, match='require no gradient itself'):
        P.distill_step(z, idx, val, rest, grad=z.clone().requires_grad_())
    with pytest.raises(N.NativeError, match='grad must be a tensor'):
        P.distill_step(z, idx, val, rest, grad=3.0)
    assert N.kernel_launch_count() == before
    with torch.no_grad():
        P.quantize_rows(z, codes, scales)
    assert torch.equal(scales, D.quantize(z)[1])


@pytest.mark.parametrize('rows', [3, 320])
def test_repeated_indices_against_merged_entries(rows):
    """The kernels' loss and gradient with repeated indices, from those of the list in which they are one entry each: the same gradient, and the loss less the entropy of the split."""
    from ista_daslab_optimizers_b200 import distill_step
    from test_distillation_cpu import split_entropy
    vocab, k = 20011, 12
    z, idx, val, rest, _ = _problem(rows, vocab, k, F32, F32, 1.0, True, False, False)
    idx[:, 5:8] = idx[:, 1:2]
    idx[:, 11] = idx[:, 0]
    loss, grad = distill_step(z, idx, val, rest)
    v = val.double()
    v[:, 1] = torch.logsumexp(v[:, [1, 5, 6, 7]], 1)
    v[:, 0] = torch.logsumexp(v[:, [0, 11]], 1)
    keep = idx.clone()
    keep[:, 5:8], keep[:, 11] = -1, -1
    w_loss, w_grad, size = D.distill(z, keep, v, rest, None, 1.0)
    p = torch.softmax(torch.cat([val.double(), rest.double()[:, None]], 1), 1)[:, :k].tolist()
    below = torch.tensor([split_entropy(a, b) for a, b in zip(p, idx.tolist())], dtype=torch.float64, device='cuda')
    D.assert_distill(loss, grad, (w_loss - below, w_grad, size), vocab, 'repeated')


# ------------------------------------------------------------------------------------------------ what memory holds, and how far it reaches

def test_tensors_with_a_negation_put_off():
    """The imaginary part of a conjugate is a view whose memory holds the opposite numbers: it is refused, or resolved where it is the gradient from above."""
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    g = _gen(71)
    column = torch.complex(_normal(g, 5, 1), _normal(g, 5, 1)).conj().imag
    one = torch.complex(_normal(g, 1), _normal(g, 1)).conj().imag
    assert column.is_neg() and one.is_neg()
    idx, val = torch.zeros(5, 1, dtype=torch.int32, device='cuda'), torch.ones(5, 1, device='cuda')
    codes = torch.ones(1, 16, dtype=torch.int8, device='cuda')
    for call in (lambda: P.quantize_rows(column), lambda: P.topk_logits(column, 1), lambda: P.distill_step(column, idx, val), lambda: P.distill_loss(column, idx, val),
                 lambda: P.int8_matmul(codes, codes, one, one.resolve_neg()), lambda: P.int8_matmul(codes, codes, one.resolve_neg(), one.resolve_neg(), one),
                 lambda: P.distill_step(val[:1], idx[:1], val[:1], one), lambda: P.distill_step(val[:1], idx[:1], val[:1], None, one)):
        with pytest.raises(N.NativeError, match='negation'):
            call()
    z, idx, val, rest, _ = _problem(5, 500, 4, F32, F32, 1.0, True, False, False)
    leaf = z.clone().requires_grad_()
    up = torch.complex(_normal(g, 5), _normal(g, 5)).conj().imag
    got, = torch.autograd.grad(P.distill_loss(leaf, idx, val, rest), leaf, up)
    want, = torch.autograd.grad(P.distill_loss(leaf, idx, val, rest), leaf, up.resolve_neg().clone())
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits():
    """Matrices of more than 2^31 elements, by many rows and by few that lie far apart: their last rows are what they are alone."""
    from ista_daslab_optimizers_b200 import distill_loss, distill_step, int8_matmul, quantize_rows, topk_logits
    g = _gen(73)
    rows, vocab, k = 17000, 128256, 8
    last = _normal(g, 5, vocab).to(BF16)
    z = torch.zeros(rows, vocab, dtype=BF16, device='cuda')
    z[-5:] = last
    idx = torch.randint(0, vocab, (rows, k), generator=g, device='cuda', dtype=torch.int32)
    val = _normal(g, rows, k)
    for whole, alone in zip(topk_logits(z, k), topk_logits(last, k)):
        assert torch.equal(whole[-5:], alone) or whole.dtype == F32
        D.assert_near(whole[-5:], alone, 2 * D.sum_error(vocab) + 4 * D.U * alone.abs().float(), 'top')          # (other numbers of blocks a row)
    want = D.distill(last, idx[-5:], val[-5:], None, None, 1.0)
    leaf = z.requires_grad_()
    loss = distill_loss(leaf, idx, val)
    grad, = torch.autograd.grad(loss.sum(), leaf)
    D.assert_distill(loss[-5:].detach(), grad[-5:], want, vocab, 'loss')
    z = z.detach()
    loss, _ = distill_step(z, idx, val, grad=z)
    D.assert_distill(loss[-5:], z[-5:], want, vocab, 'step')
    del grad, leaf
    # products: 17000 x 128256 outputs
    a, b = _codes(g, rows, 64), _codes(g, vocab, 64)
    sa, sb = torch.rand(rows, generator=g, device='cuda'), torch.rand(vocab, generator=g, device='cuda')
    out = int8_matmul(a, b, sa, sb, out=z)
    p, tol = D.matmul(a[-300:], b, sa[-300:], sb, None)
    D.assert_near(out[-300:], p, tol + D.half_step(BF16) * p.abs(), 'product')
    codes, scales = quantize_rows(z)
    want_codes, want_scales = D.quantize(z[-300:])
    assert torch.equal(codes[-300:], want_codes) and torch.equal(scales[-300:], want_scales)
    # three rows 2^30 + 8 elements apart
    buf = z.flatten()
    del z, out, codes
    far = torch.empty(2 * (2 ** 30 + 8) + 70000, dtype=BF16, device='cuda')
    del buf
    x = far.as_strided((3, 70000), (2 ** 30 + 8, 1))
    x.copy_(_normal(g, 3, 70000))
    near = x.clone()
    for p, q in zip(topk_logits(x, 100) + quantize_rows(x) + distill_step(x, idx[:3] % 70000, val[:3]),
                    topk_logits(near, 100) + quantize_rows(near) + distill_step(near, idx[:3] % 70000, val[:3])):
        assert torch.equal(p, q)
    want = distill_step(near, idx[:3] % 70000, val[:3])[1]
    assert torch.equal(distill_step(x, idx[:3] % 70000, val[:3], grad=x)[1], want)
    # ... and codes and products as far apart
    wide = torch.empty(2 * (2 ** 30 + 16) + 4096, dtype=torch.int8, device='cuda')
    c = wide.as_strided((3, 4096), (2 ** 30 + 16, 1))
    quantize_rows(x[:, :4096].float(), c)
    o = far.as_strided((3, 3), (2 ** 30 + 8, 1))
    s = torch.ones(3, device='cuda')
    for pad in (c, torch.cat([c, torch.zeros(6, 4096, dtype=torch.int8, device='cuda')])):
        assert torch.equal(int8_matmul(pad, c, torch.ones(len(pad), device='cuda'), s, dtype=F32)[:3], int8_matmul(pad.contiguous(), c.contiguous(), torch.ones(len(pad), device='cuda'), s, dtype=F32)[:3])
    assert torch.equal(int8_matmul(c, c, s, s, out=o), int8_matmul(c.contiguous(), c.contiguous(), s, s))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('m', [1, 2, 3, 4, 5])
@pytest.mark.parametrize('n,k', [(4097, 4095), (4097, 4097), (33000, 515), (1200, 16001)])
def test_int8_matmul_of_few_tokens_on_both_sides_of_the_border(m, n, k, dtype):
    from ista_daslab_optimizers_b200 import int8_matmul
    g = _gen(m * 7 + n * 3 + k)
    a, b = _codes(g, m, k), _codes(g, n, k)
    sa, sb, bias = torch.rand(m, generator=g, device='cuda') + 0.01, torch.rand(n, generator=g, device='cuda') * 0.01, _normal(g, n, scale=50.0)
    want, tol = D.matmul(a, b, sa, sb, bias)
    D.assert_near(int8_matmul(a, b, sa, sb, bias, dtype=dtype), want, tol + (0 if dtype == F32 else D.half_step(dtype) * want.abs()), 'product')


@pytest.mark.parametrize('use_reentrant', [False, True])
def test_loss_inside_a_checkpoint(use_reentrant):
    """The student's head and its loss computed again in the backward pass instead of being kept: the gradients are the same."""
    from ista_daslab_optimizers_b200 import distill_loss
    from torch.utils.checkpoint import checkpoint
    _, idx, val, rest, w = _problem(20, 3001, 8, F32, F32, 1.0, True, True, True)
    g = _gen(81)
    hidden, weight = _normal(g, 20, 64).requires_grad_(), _normal(g, 3001, 64, scale=0.2).requires_grad_()

    def loss(h, u):
        return distill_loss(h @ u.t(), idx, val, rest, w).sum()

    want = torch.autograd.grad(loss(hidden, weight), (hidden, weight))
    for _ in range(2):
        hidden.grad = weight.grad = None
        checkpoint(loss, hidden, weight, use_reentrant=use_reentrant).backward()
        assert torch.equal(hidden.grad, want[0]) and torch.equal(weight.grad, want[1])


def test_scales_behind_a_row():
    """A vector in the gap behind a row of the output shares no byte with it; one that reaches the next row does."""
    import ista_daslab_optimizers_b200 as P
    from ista_daslab_optimizers_b200 import _native as N
    g = _gen(91)
    x = _normal(g, 5, 256)
    record = torch.zeros(5, 256 + 32, dtype=torch.uint8, device='cuda')
    codes, scales = record.view(torch.int8)[:, :256], record.view(F32)[1, 64:69]
    P.quantize_rows(x, codes, scales)
    want, want_scales = D.quantize(x)
    assert torch.equal(codes, want) and torch.equal(scales, want_scales)
    with pytest.raises(N.NativeError, match='overlap'):
        P.quantize_rows(x, codes, record.view(F32).flatten()[72 + 68:72 + 73])
