"""-m gpu: the head losses and top_logits where sizes and values are at their ends, against their formulas in 64 bits.

Tolerances, from the unit roundoff of each step (u16: half a step of the type, u = 2^-24), where the logits z themselves are
exact (given, or sums of few small integers): exponents are differences of logits, R = max (z - z') / tau over the unmasked
ones, so du = 4 u R (difference, 1 / tau, product, the exponential's argument); a sum of exponentials 2^-20 (fast
exponentials 2^-21 relative, the sum itself), a logarithm 2^-22, together under 2^-18:
  row loss    tau^2 P (2 du + 2^-18) + 2 u |loss|
  gradients   of logits: u16 |dz| + (2 du + 2^-18) c q, q = P s + p
              of a head: dz rounded to u16 as well, c sum (u16 + 2 du + 2^-18 + K u) q |x| over a contraction of K, u16 |out|
  f16         2^-25 for subnormals of an output
"""
import math

import pytest
import torch

from tests.test_gpu_head_losses import TYPES, U, U16, _formula, _targets

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from neuron_interpolation_model_fusion_amd import ops
    return ops


def _check_logits(ops, z, values, indices, tau, reach, reduction='none'):
    """topk_distillation and its gradient; reach: the largest difference of two unmasked logits of a row."""
    n = z.shape[0]
    p, at, live = _targets(values=values, indices=indices, tau=tau)
    t = (values.double() / tau).masked_fill((indices < 0) | (values == -math.inf), -math.inf)
    p = torch.where(live[:, None], torch.softmax(t, 1), torch.zeros_like(p))  # log V is lost in a log-sum-exp of lowest values
    zg = z.cuda().requires_grad_()
    loss = ops.topk_distillation(zg, values.cuda(), indices.cuda(), temperature=tau, reduction=reduction)
    got, = torch.autograd.grad(loss.sum(), zg)
    want, rows, dz, q, coef = _formula(z.double(), p, at, live, tau, reduction, torch.ones(n))
    du = 4 * U * reach / tau
    tol = tau * tau * p.sum(1) * (2 * du + 2.0 ** -18) + 2 * U * rows.abs() + 1e-30
    tol = tol if reduction == 'none' else tol.sum() / (max(1, int(live.sum())) if reduction == 'mean' else 1) + U * want.abs()
    off = (loss.detach().cpu().double() - want).abs()
    assert torch.all(off <= tol), float((off / tol).max())
    bound = U16[z.dtype] * dz.abs() + (2 * du + 2.0 ** -18) * coef * q + (2.0 ** -25 if z.dtype == torch.float16 else 1e-37)
    off = (got.cpu().double() - dz).abs()
    assert torch.all(off <= bound), float((off / bound).max())


def _top(n, k, classes, g):
    return torch.randn(n, k, generator=g), torch.stack([torch.randperm(classes, generator=g)[:k] for _ in range(n)])


@pytest.mark.parametrize('tau', [1.0, 0.5, 2.0])
@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v', [(3, 40), (5, 1001), (3, 30001), (300, 3001), (3, 262147)])
def test_classes_masked_by_the_lowest_value(ops, dt, tau, n, v):
    """finfo.min in a stretch of classes as wide as many threads' first loads, in the odd elements at a row's ends, in every
    class but one."""
    g = torch.Generator().manual_seed(v)
    low = torch.finfo(dt).min
    z = (3 * torch.randn(n, v, generator=g)).to(dt)
    z[0, : v - v // 8 - 1] = low
    z[1, 0], z[1, v - 2:] = low, low
    z[2, : v - 2], z[2, v - 1] = low, low
    values, _ = _top(n, 4, v, g)
    indices = torch.stack([torch.tensor([v - 3, v - 4, v - 2, -1]) for _ in range(n)])
    indices[1], indices[2] = torch.tensor([1, 2, 3, 4]), torch.tensor([v - 2, -1, -1, -1])
    _check_logits(ops, z, values, indices, tau, 40.0)
    _check_logits(ops, z, values, indices, tau, 40.0, 'mean')
    k = min(30, v)
    got, at, lse = ops.top_logits(z.cuda(), k, temperature=tau)
    want = torch.logsumexp(z.double() / tau, 1)
    assert torch.all((lse.cpu().double() - want).abs() <= 2.0 ** -18 + 2 * U * want.abs() + 4 * U * 40 / tau)
    order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    assert torch.equal(got.cpu().float(), order.values[:, :k]) and torch.equal(at.cpu().long(), order.indices[:, :k])


@pytest.mark.parametrize('tau', [1.0, 0.5, 2.0])
@pytest.mark.parametrize('dt', TYPES)
def test_the_log_sum_exp_of_a_row_of_lowest_values(ops, dt, tau):
    """low / tau + log V, which low absorbs; beyond float32's range it is -inf."""
    for v in (1, 7, 1000, 140001):
        z = torch.full((2, v), torch.finfo(dt).min, dtype=dt)
        values, at, lse = ops.top_logits(z.cuda(), 1, temperature=tau)
        want = torch.logsumexp(z.double() / tau, 1).float()
        assert torch.equal(at.cpu(), torch.zeros(2, 1, dtype=torch.int32)) and torch.equal(values.cpu(), z[:, :1])
        assert torch.allclose(lse.cpu(), want, rtol=2.0 ** -22, atol=2.0 ** -18)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('v', [1, 9, 1001, 140001])
def test_top_logits_of_rows_that_hold_infinity(ops, dt, v):
    """The log-sum-exp of a row that holds +inf is +inf, wherever it stands and whatever else is there but NaN."""
    g = torch.Generator().manual_seed(v)
    z = (3 * torch.randn(9, v, generator=g)).to(dt)
    z[1:5], z[5] = (z[1:5].float() * 300).to(dt), -math.inf
    for row, c in enumerate((0, v - 1, v // 2, v // 3)):
        z[row, c] = math.inf
    z[4, v // 4:] = math.inf
    z[5, v // 2] = math.inf
    z[6, v // 2] = math.nan
    z[7, 0], z[7, v - 1] = math.inf, math.nan
    k = min(v, 5)
    values, at, lse = ops.top_logits(z.cuda(), k, temperature=2.0)
    lse = lse.cpu()
    assert torch.all(lse[:6] == math.inf) and lse[6].isnan() and lse[7].isnan() and torch.isfinite(lse[8])
    order = torch.sort(z[:6].float(), dim=1, descending=True, stable=True)
    assert torch.equal(values.cpu()[:6].float(), order.values[:, :k]) and torch.equal(at.cpu()[:6].long(), order.indices[:, :k])
    # nothing finite is left of a loss on such a row
    loss = ops.topk_distillation(z.cuda(), torch.zeros(9, 1).cuda(), torch.zeros(9, 1, dtype=torch.int64).cuda(), reduction='none')
    assert not torch.isfinite(loss[:8]).any() and torch.isfinite(loss[8])


@pytest.mark.parametrize('tau', [1.0, 0.7])
@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v', [(3, 5), (9, 1001), (200, 30001), (300, 3001)])
def test_distillation_of_large_logits(ops, dt, tau, n, v):
    """Logits near a thousand, either sign: what is computed from them depends on their differences alone."""
    g = torch.Generator().manual_seed(n + v)
    z = (3 * torch.randn(n, v, generator=g) + torch.where(torch.arange(n) % 2 == 0, 1000.0, -1000.0)[:, None]).to(dt)
    values, indices = _top(n, min(v, 6), v, g)
    reach = float((z.double().amax(1) - z.double().amin(1)).max())
    _check_logits(ops, z, values, indices, tau, reach)


@pytest.mark.parametrize('tau', [1.0, 0.5])
@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('low', ['lowest', 'a thousand'])
def test_distillation_of_rows_of_one_value(ops, dt, tau, low):
    """Every class alike, at the type's lowest value (a row whose mask leaves nothing) too: the softmax is 1 / V."""
    for n, v in ((2, 3), (3, 1001), (2, 140001)):
        z = torch.full((n, v), torch.finfo(dt).min if low == 'lowest' else 1000.0, dtype=dt)
        values, indices = _top(n, 3, v, torch.Generator().manual_seed(v))
        _check_logits(ops, z, values, indices, tau, 0.0)


HEADS = [(5, 64, 40), (300, 64, 600), (600, 64, 700), (5, 64, 20011), (40, 72, 9001), (40, 67, 9001), (1100, 72, 3001), (600, 67, 3001)]


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('k, tau', [(None, 1.0), (5, 2.0)])
@pytest.mark.parametrize('n, d, v', HEADS)
def test_heads_of_large_logits(ops, dt, k, tau, n, d, v):
    """Logits near a thousand that are exact in 32 bits -- sums of -1, 0 and 1 and a bias of 1024 -- in the small form, with
    and without kept logits, with odd rows: the row's sum, not its rounded log-sum-exp, is what the softmax is divided by."""
    g = torch.Generator().manual_seed(n + v)
    h, w = (torch.randint(-1, 2, (rows, d), generator=g).to(dt) for rows in (n, v))
    b = torch.full((v,), 1024.0).to(dt)
    if k is None:
        y = torch.randint(0, v, (n,), generator=g)
        p, at, live = _targets(labels=y)
    else:
        values, indices = _top(n, k, v, g)
        p, at, live = _targets(values=values, indices=indices, tau=tau)
    hg, wg, bg = (t.cuda().requires_grad_() for t in (h, w, b))
    if k is None:
        loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction='none')
    else:
        loss = ops.linear_topk_distillation(hg, wg, values.cuda(), indices.cuda(), bg, temperature=tau, reduction='none')
    got = torch.autograd.grad(loss.sum(), (hg, wg, bg))
    h, w = h.double(), w.double()
    z = h @ w.t() + 1024.0
    want, rows, dz, q, coef = _formula(z, p, at, live, tau, 'none', torch.ones(n))
    du = 4 * U * float((z.amax(1) - z.amin(1)).max()) / tau
    tol = tau * tau * p.sum(1) * (2 * du + 2.0 ** -18) + 2 * U * rows.abs()
    off = (loss.detach().cpu().double() - want).abs()
    assert torch.all(off <= tol), float((off / tol).max())
    cq, rel = coef * q, (U16[dt] if dt != torch.float32 else 2 * U) + 2 * du + 2.0 ** -18
    for x, ref, size, length in ((got[0], dz @ w, cq @ w.abs(), v), (got[1], dz.t() @ h, cq.t() @ h.abs(), n), (got[2], dz.sum(0), cq.sum(0), n)):
        bound = U16[dt] * ref.abs() + (rel + (length + 64) * U) * size + (2.0 ** -24 if dt == torch.float16 else 1e-37)
        off = (x.cpu().double() - ref).abs()
        assert torch.all(off <= bound), float((off / bound).max())


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v', HEADS)
def test_heads_whose_classes_are_all_masked_by_the_lowest_value(ops, dt, n, d, v):
    """z = low for every class: the softmax is 1 / V, the loss log V."""
    h, w = torch.ones(n, d, dtype=dt), torch.zeros(v, d, dtype=dt)
    b = torch.full((v,), torch.finfo(dt).min, dtype=dt)
    y = torch.arange(n) * 7 % v
    hg, wg, bg = (t.cuda().requires_grad_() for t in (h, w, b))
    loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction='none')
    db, = torch.autograd.grad(loss.sum(), bg)
    assert torch.all((loss.detach().cpu().double() - math.log(v)).abs() <= 2.0 ** -18 + 2 * U * math.log(v))
    want = n / v - torch.bincount(y, minlength=v).double()
    q = n / v + torch.bincount(y, minlength=v).double()
    assert torch.all((db.cpu().double() - want).abs() <= U16[dt] * want.abs() + (U16[dt] + 2.0 ** -18 + (n + 64) * U) * q)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n', [0, 5, 700])
@pytest.mark.parametrize('d, v', [(24, 40), (264, 9001)])
def test_no_row_that_counts_has_no_gradient_whatever_arrives(ops, dt, n, d, v):
    h, w, b = (torch.ones(*s, dtype=dt, device='cuda').requires_grad_() for s in ((n, d), (v, d), (v,)))
    y = torch.full((n,), -100, device='cuda')
    for reduction in ('mean', 'sum', 'none'):
        for up in (math.nan, math.inf):
            loss = ops.linear_cross_entropy(h, w, y, b, reduction=reduction)
            for x in torch.autograd.grad(loss, (h, w, b), grad_outputs=torch.full_like(loss, up)):
                assert torch.all(x == 0)


@pytest.mark.parametrize('reduction', [0, 1, 2])
@pytest.mark.parametrize('d, v', [(24, 40), (264, 9001)])
def test_no_rows_need_no_arriving_gradient(d, v, reduction):
    """Through the C ABI: zero rows, no gradient given, zeros in dweight and dbias."""
    import ctypes

    from neuron_interpolation_model_fusion_amd import _lib
    lib, st = _lib.lib, torch.cuda.current_stream().cuda_stream
    w, dw, db = torch.ones(v, d, device='cuda'), torch.full((v, d), 7.0, device='cuda'), torch.full((v,), 7.0, device='cuda')
    desc = _lib.HeadDesc(ldh=d, weight=w.data_ptr(), ldw=d, rows=0, features=d, classes=v, dtype=_lib.NIF_F32, reduction=reduction,
                         ignore_index=-100, temperature=1.0)
    at = ctypes.byref(desc)
    state, ws, ws_b = (torch.empty(f(at), dtype=torch.uint8, device='cuda') for f in (
        lib.nif_head_state_bytes, lib.nif_head_forward_workspace_bytes, lib.nif_head_backward_workspace_bytes))
    loss = torch.full((1,), 7.0, device='cuda')
    assert lib.nif_head_forward(at, loss.data_ptr(), state.data_ptr(), state.numel(), ws.data_ptr(), ws.numel(), st) == 0
    assert lib.nif_head_backward(at, None, state.data_ptr(), state.numel(), None, d, dw.data_ptr(), d, db.data_ptr(), ws_b.data_ptr(),
                                 ws_b.numel(), st) == 0
    torch.cuda.synchronize()
    assert torch.all(dw == 0) and torch.all(db == 0) and (reduction == 0 or float(loss) == 0)


MANY = (1 << 24) + 5  # 256 threads a row are more than 2^32 in one grid dimension


@pytest.mark.parametrize('dt', TYPES)
def test_more_rows_than_a_grid_dimension_holds(ops, dt):
    """Logits, top logits and their distillation of 2^24 + 5 rows: the same numbers as the rows' last and first alone."""
    n, v, k = MANY, 4, 2
    g = torch.Generator(device='cuda').manual_seed(3)
    z = torch.randn(n, v, generator=g, device='cuda').to(dt)
    z[12345:12400] = z[0]
    z.requires_grad_()
    values, indices, lse = ops.top_logits(z, k, temperature=2.0)
    assert torch.equal(values.float(), z.detach().float().topk(k, dim=1).values)
    assert torch.equal(z.detach().gather(1, indices.long()), values)
    loss = ops.topk_distillation(z, values, indices, temperature=2.0, top_lse=lse, reduction='none')
    dz, = torch.autograd.grad(loss, z, grad_outputs=torch.ones_like(loss))
    for part in (slice(0, 70), slice(n // 2, n // 2 + 70), slice(n - 70, n)):
        few = z.detach()[part].requires_grad_()
        top = ops.top_logits(few, k, temperature=2.0)
        assert torch.equal(top[0], values[part]) and torch.equal(top[1], indices[part]) and torch.equal(top[2], lse[part])
        alone = ops.topk_distillation(few, *top[:2], temperature=2.0, top_lse=top[2], reduction='none')
        assert torch.equal(alone, loss[part])
        assert torch.equal(torch.autograd.grad(alone, few, grad_outputs=torch.ones_like(alone))[0], dz[part])
    mean = ops.topk_distillation(z, values, indices, temperature=2.0, top_lse=lse)
    assert abs(float(mean.detach()) - float(loss.double().mean())) <= 2 * U * abs(float(mean.detach()))


@pytest.mark.parametrize('dt', TYPES)
def test_a_head_of_more_rows_than_a_grid_dimension_holds(ops, dt):
    n, d, v = MANY, 8, 5
    g = torch.Generator(device='cuda').manual_seed(4)
    h = torch.randint(-2, 3, (n, d), generator=g, device='cuda').to(dt).requires_grad_()
    w = torch.randint(-2, 3, (v, d), generator=g, device='cuda').to(dt).requires_grad_()
    b = torch.zeros(v, dtype=dt, device='cuda').requires_grad_()
    y = torch.randint(-1, v, (n,), generator=g, device='cuda')
    loss = ops.linear_cross_entropy(h, w, y, b, ignore_index=-1, reduction='sum')
    dh, dw, db = torch.autograd.grad(loss, (h, w, b), grad_outputs=torch.tensor(2.0 ** -12, device='cuda'))
    want, dz_all, size = 0.0, [], 0.0
    for lo in range(0, n, 1 << 22):  # the formula, a part of the rows at a time
        part = slice(lo, min(n, lo + (1 << 22)))
        x, live = h.detach()[part].double(), y[part] >= 0
        logs = torch.log_softmax(x @ w.detach().double().t(), 1)
        at = y[part].clamp(min=0)[:, None]
        want += float(-(logs.gather(1, at)[:, 0] * live).sum())
        dz = logs.exp().scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.float64)) * live[:, None] * 2.0 ** -12
        got = dh[part].double()
        ref = dz @ w.detach().double()
        # a row's |dz| sums to at most 2 . 2^-12, weights are at most 2: each rounding of dz, the sum's and the result's
        assert float((got - ref).abs().max()) <= 2.0 ** -12 * 4 * (2 * U16[dt] + 2.0 ** -17) + 2.0 ** -24
        dz_all.append((dz.t() @ x, dz.sum(0)))
        size = size + dz.abs().sum(0)
    assert abs(float(loss.detach()) - want) <= 2.0 ** -18 * n + 2 * U * want
    dw_ref, db_ref = sum(p[0] for p in dz_all), sum(p[1] for p in dz_all)
    # n additions of 32 bits in chains of at most 2^24 / 128, dz's rounding once
    slack = U16[dt] + 2.0 ** -17 + 2.0 ** 17 * U
    assert torch.all((dw.double() - dw_ref).abs() <= U16[dt] * dw_ref.abs() + 2 * slack * size[:, None])
    assert torch.all((db.double() - db_ref).abs() <= U16[dt] * db_ref.abs() + slack * size)


@pytest.mark.parametrize('dt', TYPES)
def test_more_tiles_of_a_product_than_one_launch_takes(ops, dt):
    """2^21 rows against 2^15 + 1 classes: over 2^20 tiles of the logits' product."""
    n, d, v = 1 << 21, 16, (1 << 15) + 1
    g = torch.Generator(device='cuda').manual_seed(5)
    h = torch.randint(-1, 2, (n, d), generator=g, device='cuda').to(dt)
    w = torch.randint(-1, 2, (v, d), generator=g, device='cuda').to(dt)
    y = torch.randint(0, v, (n,), generator=g, device='cuda')
    loss = ops.linear_cross_entropy(h, w, y, reduction='none')
    for part in (slice(0, 100), slice(n // 2 - 50, n // 2 + 50), slice(n - 100, n)):
        z = h[part].double() @ w.double().t()
        want = torch.logsumexp(z, 1) - z.gather(1, y[part][:, None])[:, 0]
        assert torch.all((loss[part].double() - want).abs() <= 2.0 ** -18 + 2 * U * want + 8 * U * 32)


@pytest.mark.parametrize('tau', [1.0, 0.5, 0.7])
@pytest.mark.parametrize('shift', [1000.0, -1000.0, 'lowest'])
def test_teachers_of_large_logits(ops, tau, shift):
    """A teacher's distribution over its entries is one of their differences; entries all at the lowest value are alike."""
    n, v, k = 40, 300, 70
    g = torch.Generator().manual_seed(17)
    values, indices = _top(n, k, v, g)
    values = torch.full((n, k), torch.finfo(torch.float32).min) if shift == 'lowest' else 3 * values + shift
    indices[3, 1:], indices[4, 60:] = -1, -1
    reach = 0.0 if shift == 'lowest' else float((values.amax(1) - values.amin(1)).max())
    for dt in TYPES:
        z = torch.randn(n, v, generator=g).to(dt)
        _check_logits(ops, z, values, indices, tau, max(10.0, reach))
    # through a head: the same targets, logits that are exact
    h, w = torch.randint(-1, 2, (n, 64), generator=g).float(), torch.randint(-1, 2, (v, 64), generator=g).float()
    z = h @ w.t()
    a = ops.linear_topk_distillation(h.cuda(), w.cuda(), values.cuda(), indices.cuda(), temperature=tau, reduction='none')
    b = ops.topk_distillation(z.cuda(), values.cuda(), indices.cuda(), temperature=tau, reduction='none')
    assert torch.isfinite(a).all() and torch.allclose(a, b, rtol=4 * U, atol=tau * tau * (2.0 ** -18 + 16 * U * 64 / tau))


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('k', [None, 1, 13])
@pytest.mark.parametrize('n, d, v', [(1, 64, 11021), (2, 72, 30011), (5, 67, 9001), (31, 264, 9001), (32, 64, 5003), (33, 40, 9001),
                                     (64, 520, 4099), (60, 131, 3001), (16, 8, 300011), (64, 16, 300001)])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_gradients_of_few_rows_are_rounded_once(ops, dt, k, n, d, v, reduction):
    """The roundings of a few rows' logit gradients would not average out: they are held in two 16-bit parts, together at
    least 2^-16 (2^-21) of them, with and without kept logits, in one piece and in several."""
    g = torch.Generator().manual_seed(n + d + v)
    h, w = torch.randn(n, d, generator=g).to(dt), (torch.randn(v, d, generator=g) * 2 / math.sqrt(d)).to(dt)
    b = torch.randn(v, generator=g).to(dt)
    if k is None:
        y = torch.randint(0, v, (n,), generator=g)
        if n > 3:
            y[1] = -100
        p, at, live = _targets(labels=y)
    else:
        values, indices = _top(n, k, v, g)
        if n > 3:
            indices[1] = -1
        p, at, live = _targets(values=values, indices=indices, tau=2.0)
    tau = 1.0 if k is None else 2.0
    up = torch.rand(n, generator=g) + 0.5 if reduction == 'none' else torch.ones(n)
    hg, wg, bg = (t.cuda().requires_grad_() for t in (h, w, b))
    if k is None:
        loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction=reduction)
    else:
        loss = ops.linear_topk_distillation(hg, wg, values.cuda(), indices.cuda(), bg, temperature=tau, reduction=reduction)
    got = torch.autograd.grad(loss, (hg, wg, bg), grad_outputs=up.cuda() if reduction == 'none' else torch.ones_like(loss))
    h, w = h.double(), w.double()
    z = h @ w.t() + b.double()
    _, _, dz, q, coef = _formula(z, p, at, live, tau, reduction, up)
    A = (h.abs() @ w.abs().t() + b.double().abs()).amax(1, keepdim=True)
    cq = coef * q * (2 * (d + 8) * U * A / tau + 2.0 ** -18 + U16[dt] ** 2)  # logits, exponentials, the two parts
    lost = coef.max() * 2.0 ** -37 if dt == torch.float16 else 0.0  # f16: subnormals of the scaled parts
    for x, ref, size, length, floor in ((got[0], dz @ w, (cq @ w.abs()), v, w.abs().sum(0)), (got[1], dz.t() @ h, cq.t() @ h.abs(), n, h.abs().sum(0)),
                                        (got[2], dz.sum(0), cq.sum(0), n, torch.tensor(float(n)))):
        terms = (coef * q) @ w.abs() if length == v else (coef * q).t() @ h.abs() if ref.dim() == 2 else (coef * q).sum(0)
        bound = U16[dt] * ref.abs() * (1 + 2.0 ** -8) + size + (length + 64) * U * terms + lost * floor + (2.0 ** -25 if dt == torch.float16 else 1e-37)
        off = (x.cpu().double() - ref).abs()
        assert torch.all(off <= bound), float((off / bound).max())


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
@pytest.mark.parametrize('n, d, v, k', [(65, 64, 9001, 13), (200, 72, 300, 8), (130, 40, 60001, 100), (700, 67, 3001, 2), (2100, 64, 520, None),
                                        (600, 64, 700, 9), (1500, 16, 500001, 5)])
def test_the_bias_gradient_keeps_what_its_targets_entries_round_off(ops, dt, reduction, n, d, v, k):
    """A class has few targets, so their entries' rounding does not average out in its column sum: it is added back.  What is
    left is that of the P s of every row, and the entries' own without it where a target falls."""
    g = torch.Generator(device='cuda').manual_seed(n + v)
    h = torch.randn(n, d, generator=g, device='cuda').to(dt)
    w = (torch.randn(v, d, generator=g, device='cuda') / math.sqrt(d)).to(dt)
    b = torch.zeros(v, dtype=dt, device='cuda').requires_grad_()
    tau = 1.0 if k is None else 2.0
    up = torch.rand(n, generator=g, device='cuda') + 0.5 if reduction == 'none' else None
    if k is None:
        y = torch.randint(0, v, (n,), generator=g, device='cuda')
        at, p = y[:, None], torch.ones(n, 1, device='cuda').double()
        loss = ops.linear_cross_entropy(h, w, y, b, reduction=reduction)
    else:
        values = 2 * torch.randn(n, k, generator=g, device='cuda')
        at = (torch.randint(0, v, (n, 1), generator=g, device='cuda') + torch.arange(k, device='cuda') * max(1, v // k)) % v
        p = torch.softmax(values.double() / tau, 1)
        loss = ops.linear_topk_distillation(h, w, values, at, b, temperature=tau, reduction=reduction)
    for _ in range(2):  # the second pass finds the buffers of the first
        got, = torch.autograd.grad(loss, b, grad_outputs=up if reduction == 'none' else torch.ones_like(loss), retain_graph=True)
    c = tau * (up.double() if reduction == 'none' else torch.full((n,), 1.0 / n, device='cuda').double())
    ref, left, q, terms = (torch.zeros(v, dtype=torch.float64, device='cuda') for _ in range(4))
    for lo in range(0, n, 100):
        part = slice(lo, min(n, lo + 100))
        z = (h[part].double() @ w.double().t()) / tau
        s = torch.softmax(z, 1) * c[part, None]
        A = (h[part].double().abs() @ w.double().abs().t()).amax(1, keepdim=True)
        cp = c[part, None] * p[part]
        q += (s * (2 * (d + 8) * U * A / tau + 2.0 ** -18)).sum(0) + 2.0 ** -18 * torch.zeros_like(ref).index_add_(0, at[part].reshape(-1), cp.reshape(-1))
        ref += s.sum(0).index_add_(0, at[part].reshape(-1), -cp.reshape(-1))
        left += s.scatter(1, at[part], 0.0).sum(0)
        terms += s.sum(0).index_add_(0, at[part].reshape(-1), cp.reshape(-1))
    bound = U16[dt] * (1 + 2.0 ** -8) * (ref.abs() + left) + q + (n + 64) * U * terms \
        + (2.0 ** -25 + n * c.max() * 2.0 ** -37 if dt == torch.float16 else 1e-37)
    off = (got.double() - ref).abs()
    assert torch.all(off <= bound), float((off / bound).max())


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v', [(5, 5003), (40, 20011), (96, 9001), (700, 600)])
def test_captured_steps_with_a_bias(ops, dt, n, v):
    """Replayed with new inputs, rows that are left out among them, eager steps of the same between: the buffers of one step
    are those of the next."""
    g = torch.Generator(device='cuda').manual_seed(n)
    d, k = 72, 7
    h, w, b = (torch.zeros(*s, dtype=dt, device='cuda', requires_grad=True) for s in ((n, d), (v, d), (v,)))
    values, indices = torch.zeros(n, k, device='cuda'), torch.zeros(n, k, dtype=torch.int32, device='cuda')

    def step():
        loss = ops.linear_topk_distillation(h, w, values, indices, b, temperature=2.0)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w, b)))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(4):
        with torch.no_grad():
            for t in (h, w, b):
                t.copy_(torch.randn(t.shape, generator=g, device='cuda') / 3)
            values.copy_(torch.randn(n, k, generator=g, device='cuda'))
            indices.copy_(torch.randint(0, v, (n, k), generator=g, device='cuda'))
            indices[turn::3] = -1
            if turn == 2:
                indices.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, c in zip(got, step()):
            assert torch.equal(a, c)
        torch.cuda.synchronize()
