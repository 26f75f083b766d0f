"""-m gpu: the head losses (linear_cross_entropy, linear_topk_distillation, topk_distillation) and top_logits against
their formulas in 64 bits.

Tolerances are elementwise bounds, from the unit roundoff of each step (u16: half a step of the 16-bit type, u = 2^-24):
  logits      |dz| <= (D + 8) u A / tau, A = max_nv (sum_d |h w| + |b|): a chain of D 32-bit additions of products that are
              exact; f32 operands as three bf16 parts drop three of nine products, each under 2^-24 |h w|: 4 u A more
  row loss    2 tau^2 |du| P for u and lse, and 2^-18 tau^2 P for exp / log / the sum over the classes (fast exponential
              2^-21 relative, sums of V positive terms 2^-24 log-depth, rounding of u near 32: 2^-20), + u |loss|
  gradients   q = P s + p bounds |dz| per row and class before cancellation; dz carries relative 2 |du| + 2^-18 + u16 (its
              rounding to 16 bits), so |d out| <= u16 |out| + (u16 + 2 |du| + 2^-18 + K u) c sum q |x|, K the length
              of the contraction; f16: absolute 2^-25 for subnormals of the output and c 2^-37 for those of the scaled dz
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
U16 = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope='module')
def ops():
    from neuron_interpolation_model_fusion_amd import ops
    return ops


def _targets(labels=None, ignore=-100, values=None, indices=None, lse=None, tau=1.0, classes=None):
    """(p [n, k] f64, at [n, k], live [n]) on the CPU."""
    if labels is not None:
        live = labels != ignore
        return live[:, None].double(), torch.where(live, labels, 0)[:, None].long(), live
    t = values.double() / tau
    some = (indices >= 0) & (values != -math.inf)
    live = some.any(1)
    t = torch.where(some, t, torch.tensor(-math.inf, dtype=torch.float64))
    L = torch.logsumexp(t, 1) if lse is None else lse.double()
    p = torch.where(some, torch.exp(t - L[:, None]), torch.tensor(0.0, dtype=torch.float64))
    p = torch.where(live[:, None], p, torch.zeros_like(p))
    return p, torch.where(some, indices.long(), 0), live


def _formula(z, p, at, live, tau, reduction, grad):
    """(loss, rows, dz, q, coef) in 64 bits; dz carries the incoming gradient, q the size of its terms."""
    z = torch.where(live[:, None], z, torch.zeros_like(z))
    logs = torch.log_softmax(z / tau, 1)
    terms = torch.where(p > 0, p * (torch.log(torch.where(p > 0, p, torch.ones_like(p))) - logs.gather(1, at)), torch.zeros_like(p))
    rows = tau * tau * terms.sum(1) * live
    P = p.sum(1, keepdim=True)
    target = torch.zeros_like(z).scatter_add_(1, at, p)
    count = max(1, int(live.sum())) if reduction == 'mean' else 1
    coef = (tau * live / count * grad.double())[:, None]
    s = logs.exp()
    loss = rows if reduction == 'none' else rows.sum() / count
    return loss, rows, coef * (P * s - target), P * s + target, coef.abs()


def _check_head(ops, dt, n, d, v, *, k=None, tau=1.0, bias=True, empty=0.0, reduction='mean', seed=0, lse=False, scale=2.0,
                layout=None):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g).to(dt)
    w = (torch.randn(v, d, generator=g) * scale / math.sqrt(d)).to(dt)
    b = torch.randn(v, generator=g).to(dt) if bias else None
    up = 512.0 if dt == torch.float16 else 1.0
    kw = {}
    out = torch.rand(n, generator=g) < empty
    if k is None:
        y = torch.randint(0, v, (n,), generator=g)
        y[out] = -100
        p, at, live = _targets(labels=y)
    else:
        values = 3 * torch.randn(n, k, generator=g)
        indices = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]).int() if n else torch.zeros(0, k).int()
        indices[out] = -1
        if k > 2 and n > 1:
            indices[-1, k // 2:] = -1  # a row of fewer entries
            values[0, 1] = -math.inf
        top_lse = (torch.logsumexp(values.nan_to_num(neginf=-30).double() / tau, 1) + 0.3).float() if lse else None
        p, at, live = _targets(values=values, indices=indices, lse=top_lse, tau=tau)
    grad = torch.rand(n, generator=g) * up if reduction == 'none' else torch.full((n,), up)
    h[~live] = math.nan  # whatever the rows that are left out hold

    hg, wg = h.cuda(), w.cuda()
    if layout is not None:
        hg, wg = layout(hg), layout(wg)
    hg, wg = hg.requires_grad_(), wg.requires_grad_()
    bg = b.cuda().requires_grad_() if bias else None
    if k is None:
        loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction=reduction)
    else:
        loss = ops.linear_topk_distillation(hg, wg, values.cuda(), indices.cuda(), bg, temperature=tau, reduction=reduction,
                                            top_lse=None if top_lse is None else top_lse.cuda())
    got = torch.autograd.grad(loss, [t for t in (hg, wg, bg) if t is not None],
                              grad_outputs=grad.cuda() if reduction == 'none' else torch.tensor(up, device='cuda'))

    h64, w64 = torch.where(live[:, None], h, torch.zeros_like(h)).double(), w.double()
    b64 = b.double() if bias else torch.zeros(v, dtype=torch.float64)
    z = h64 @ w64.t() + b64
    want, rows, dz, q, coef = _formula(z, p, at, live, tau, reduction, grad)
    A = float((h64.abs() @ w64.abs().t() + b64.abs()).max()) if n else 0.0
    du = (d + 8 + (4 if dt == torch.float32 else 0)) * U * A / tau
    P = p.sum(1)
    row_tol = tau * tau * (P * (2 * du + 2.0 ** -18)) + 2 * U * rows.abs() + 1e-30
    tol = row_tol if reduction == 'none' else row_tol.sum() / (max(1, int(live.sum())) if reduction == 'mean' else 1) + U * want.abs()
    assert torch.all((loss.detach().cpu().double() - want).abs() <= tol), ((loss.detach().cpu().double() - want).abs() / tol).max()

    u16 = U16[dt]
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    dz_rel = u16 + 2 * du + 2.0 ** -18
    cq = coef * q
    lost = coef.max() * max(1.0, float(P.max()) if n else 1.0) * 2.0 ** -37 if dt == torch.float16 and n else 0.0
    pairs = [(got[0], dz @ w64, cq @ w64.abs(), v, w64.abs().sum(0)), (got[1], dz.t() @ h64, cq.t() @ h64.abs(), n, h64.abs().sum(0))]
    if bias:
        pairs.append((got[2], dz.sum(0), cq.sum(0), n, torch.tensor(float(n))))
    for name, (x, ref, size, length, floor) in zip(('hidden', 'weight', 'bias'), pairs):
        assert x.dtype == dt and x.shape == ref.shape
        bound = u16 * ref.abs() + (dz_rel + (length + 64) * U) * size + sub + lost * floor + 1e-37
        off = (x.cpu().double() - ref).abs()
        assert torch.all(off <= bound), f'd{name}: {float((off / bound).max()):.3g} of the bound'
        if name == 'hidden':
            assert torch.all(x.cpu()[~live] == 0)


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 16, 10), (32, 512, 10), (33, 384, 200), (64, 64, 128), (65, 72, 129), (130, 100, 300), (257, 131, 515),
          (17, 1030, 1000), (300, 48, 2500)]


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v', SHAPES)
def test_cross_entropy_and_gradients(ops, dt, n, d, v):
    _check_head(ops, dt, n, d, v, bias=n % 2 == 1, empty=0.3 if n > 3 else 0.0, seed=n + d + v)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v, k', [(1, 8, 2, 1), (3, 16, 10, 10), (32, 384, 200, 8), (65, 72, 129, 70), (257, 131, 515, 33),
                                        (300, 48, 2500, 128)])
def test_distillation_of_a_head_and_gradients(ops, dt, n, d, v, k):
    _check_head(ops, dt, n, d, v, k=k, tau=2.0, bias=n % 2 == 0, empty=0.3 if n > 3 else 0.0, seed=n + d + v, lse=k % 2 == 0)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v, k', [(1030, 1048, 1300, None), (1290, 1025, 1543, 20), (1024, 1536, 2048, None)])
def test_sizes_of_the_large_tiles(ops, dt, n, d, v, k):
    _check_head(ops, dt, n, d, v, k=k, tau=2.0 if k else 1.0, bias=n % 4 == 2, empty=0.01, seed=n)


@pytest.mark.parametrize('dt', TYPES)
def test_large_tiles_are_the_same_every_time(ops, dt):
    """Waves that run ahead of each other: a stage overwritten too early showed as a few wrong elements, not every time."""
    g = torch.Generator(device='cuda').manual_seed(15)
    h = torch.randn(2048, 1048, generator=g, device='cuda').to(dt).requires_grad_()
    w = torch.randn(4096, 1048, generator=g, device='cuda').to(dt).requires_grad_()
    y = torch.randint(0, 4096, (2048,), generator=g, device='cuda')
    first = None
    for _ in range(6):
        loss = ops.linear_cross_entropy(h, w, y)
        out = (loss.detach(), *torch.autograd.grad(loss, (h, w)))
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
def test_reductions(ops, dt, reduction):
    _check_head(ops, dt, 70, 40, 90, reduction=reduction, empty=0.4, seed=1)
    _check_head(ops, dt, 70, 40, 90, k=5, tau=4.0, reduction=reduction, empty=0.4, seed=2)


@pytest.mark.parametrize('dt', TYPES)
def test_every_row_left_out_and_no_rows(ops, dt):
    for n in (5, 0):
        h, w, b = torch.full((n, 24), math.nan, dtype=dt), torch.randn(40, 24).to(dt), torch.randn(40).to(dt)
        h, w, b = (t.cuda().requires_grad_() for t in (h, w, b))
        y = torch.full((n,), 7).cuda()
        top = torch.zeros(n, 3).cuda(), torch.full((n, 3), -1, dtype=torch.int64).cuda()
        for reduction in ('mean', 'sum', 'none'):
            for loss in (ops.linear_cross_entropy(h, w, y, b, ignore_index=7, reduction=reduction),
                         ops.linear_topk_distillation(h, w, *top, b, reduction=reduction)):
                assert loss.shape == ((n,) if reduction == 'none' else ()) and torch.all(loss == 0)
                for x in torch.autograd.grad(loss.sum(), (h, w, b)):
                    assert torch.all(x == 0)
        z = torch.full((n, 11), math.nan, dtype=dt).cuda().requires_grad_()
        loss = ops.topk_distillation(z, *top)
        assert loss == 0 and torch.all(torch.autograd.grad(loss, z)[0] == 0)


@pytest.mark.parametrize('dt', TYPES)
def test_layouts(ops, dt):
    """Strided rows, a transposed matrix, an address that 16-byte loads cannot take."""
    def strided(t):
        x = torch.empty(t.shape[0], t.shape[1] + 24, dtype=dt, device='cuda')
        x.fill_(math.nan)
        x[:, 8:8 + t.shape[1]] = t
        return x[:, 8:8 + t.shape[1]].detach()

    def odd(t):
        x = torch.full((t.numel() + 3,), math.nan, dtype=dt, device='cuda')
        x[3:] = t.reshape(-1)
        return x[3:].view(t.shape).detach()
    for layout in (strided, odd, lambda t: t.t().contiguous().t()):
        _check_head(ops, dt, 40, 64, 300, layout=layout, seed=3)
        _check_head(ops, dt, 40, 56, 300, layout=layout, k=4, seed=4)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v, k', [(1, 1024, 9001, None), (5, 776, 20011, None), (100, 264, 10007, None), (64, 64, 5003, None),
                                        (129, 520, 4099, 3), (3, 40, 9000, 1024), (2, 2056, 4100, 70)])
def test_few_rows_over_many_classes(ops, dt, n, d, v, k):
    """Logits that are kept, their product split along the features."""
    _check_head(ops, dt, n, d, v, k=k, tau=2.0 if k else 1.0, bias=n % 2 == 1, empty=0.3 if n > 3 else 0.0, seed=n + v)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v', [(3, 16, 10), (5, 776, 20011), (300, 64, 2500), (700, 264, 5001)])
def test_a_loss_without_gradients(ops, dt, n, d, v):
    """Without a backward pass to come other variants may be faster; the loss is the formula's all the same."""
    g = torch.Generator().manual_seed(n)
    h, w, b = torch.randn(n, d, generator=g).to(dt), (torch.randn(v, d, generator=g) / math.sqrt(d)).to(dt), torch.randn(v, generator=g).to(dt)
    y = torch.randint(0, v, (n,), generator=g)
    y[-1] = -100
    args = [t.cuda() for t in (h, w, y, b)]
    got = ops.linear_cross_entropy(*args, reduction='none')
    with torch.no_grad():
        args[0].requires_grad_()
        assert torch.equal(ops.linear_cross_entropy(*args, reduction='none'), got)
    z = h.double() @ w.double().t() + b.double()
    want = torch.logsumexp(z, 1) - z.gather(1, y.clamp(min=0)[:, None])[:, 0]
    du = (d + 12) * U * float((h.double().abs() @ w.double().abs().t() + b.double().abs()).max())
    assert not got.requires_grad and got[-1] == 0
    assert torch.all((got.cpu().double() - want)[:-1].abs() <= (2 * du + 2.0 ** -18 + 2 * U * want.abs())[:-1])


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('k', [None, 5])
def test_rows_far_apart(ops, dt, k):
    """Rows over 2^20 elements apart."""
    def apart(t):
        x = torch.empty(t.shape[0], (1 << 20) + 8, dtype=dt, device='cuda')
        x[:, :t.shape[1]] = t
        return x[:, :t.shape[1]].detach()
    _check_head(ops, dt, 40, 72, 300, k=k, layout=apart, seed=6)
    _check_head(ops, dt, 300, 100, 500, k=k, layout=apart, seed=7)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n', [5, 63, 65, 300, 600])
def test_rows_off_16_byte_borders(ops, dt, n):
    """Few and many rows against a weight that direct loads cannot take, with and without kept logits."""
    for d, v, k in ((131, 1543, None), (77, 9001, 6)):
        _check_head(ops, dt, n, d, v, k=k, tau=2.0 if k else 1.0, empty=0.2, seed=n + d)


@pytest.mark.parametrize('dt', TYPES)
def test_many_targets_of_few_classes(ops, dt):
    _check_head(ops, dt, 1100, 962, 251, k=93, tau=4.0, empty=0.1, seed=9)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n', [5, 700])
def test_saved_tensors_that_come_back_elsewhere(ops, dt, n):
    """Saved tensors may return at another address, with other strides, than the forward pass saw."""
    g = torch.Generator(device='cuda').manual_seed(21)
    h = torch.randn(n, 776, generator=g, device='cuda').to(dt)
    w = torch.randn(5003, 776, generator=g, device='cuda').to(dt)
    y = torch.randint(0, 5003, (n,), generator=g, device='cuda')

    def grads(hook, weight):
        x, weight = h.clone().requires_grad_(), weight.detach().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(hook, lambda t: t):
            loss = ops.linear_cross_entropy(x, weight, y)
        return (loss.detach(), *torch.autograd.grad(loss, (x, weight)))

    def moved(t):
        if t.dim() != 2:
            return t
        out = torch.empty(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=t.device)[:, 1:-2]
        return out.copy_(t)
    far = moved(w)
    for hook, weight in ((moved, w), (lambda t: t.clone(), far)):
        want, got = grads(lambda t: t, weight), grads(hook, weight)
        assert torch.equal(got[0], want[0])
        # the same products by another kernel: each is off by its bound of the formula's, here in the large
        for a, b in zip(got[1:], want[1:]):
            assert float((a - b).float().norm()) <= 4 * max(U16[dt], 64 * U) * float(b.float().norm())


def test_kept_logits_of_a_weight_that_is_packed_in_pieces(ops):
    """Rows that 16-byte loads cannot take, more bytes of them than a piece holds."""
    _check_head(ops, torch.bfloat16, 4, 50001, 2700, seed=8)


@pytest.mark.parametrize('dt', TYPES)
def test_several_pieces_of_classes(ops, dt):
    """So many rows that the backward pass takes the classes in pieces, with a short last one."""
    from neuron_interpolation_model_fusion_amd import _lib
    n = 45000 if dt == torch.float32 else 131072
    d, v = 16, 1100
    g = torch.Generator(device='cuda').manual_seed(5)
    h = torch.randn(n, d, generator=g, device='cuda').to(dt)
    w = torch.randn(v, d, generator=g, device='cuda').to(dt)
    y = torch.randint(0, v, (n,), generator=g, device='cuda')
    h, w = h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, y)
    dh, dw = torch.autograd.grad(loss, (h, w), grad_outputs=torch.tensor(float(n), device='cuda'))
    z = h.detach().double() @ w.detach().double().t()
    dz = torch.softmax(z, 1)
    dz[torch.arange(n, device='cuda'), y] -= 1
    # norms: rounding of dz and of the result, independent for each element
    for x, ref in ((dh, dz @ w.detach().double()), (dw, dz.t() @ h.detach().double())):
        assert float((x.double() - ref).norm() / ref.norm()) < 2 * U16[dt] + 2e-6
    assert abs(float(loss) - float(torch.nn.functional.cross_entropy(z, y))) < 1e-5


@pytest.mark.parametrize('dt', TYPES)
def test_masked_classes_and_extreme_logits(ops, dt):
    n, d, v = 20, 32, 150
    g = torch.Generator().manual_seed(6)
    h, w = torch.randn(n, d, generator=g).to(dt), torch.randn(v, d, generator=g).to(dt)
    y = torch.randint(0, 100, (n,), generator=g)
    for low in (-math.inf, torch.finfo(dt).min):  # classes 100.. are masked by their bias
        b = torch.zeros(v, dtype=dt)
        b[100:] = low
        hg, wg, bg = (t.cuda().requires_grad_() for t in (h, w, b))
        loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg)
        dh, dw, db = torch.autograd.grad(loss, (hg, wg, bg))
        z = h.double() @ w.double()[:100].t()
        assert abs(float(loss) - float(torch.nn.functional.cross_entropy(z, y))) < 1e-4
        assert torch.all(dw[100:] == 0) and torch.all(db[100:] == 0) and torch.isfinite(dh).all() and torch.isfinite(dw).all()
    # a masked label: infinite loss, finite gradients
    y[0] = 120
    b[100:] = -math.inf
    hg, wg, bg = (t.cuda().requires_grad_() for t in (h, w, b))
    loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction='none')
    assert loss[0] == math.inf and torch.isfinite(loss[1:]).all()
    assert all(torch.isfinite(x).all() for x in torch.autograd.grad(loss, (hg, wg, bg), grad_outputs=torch.ones_like(loss)))
    # logits of a thousand: no overflow
    big = (100 * h.float()).to(dt)
    loss = ops.linear_cross_entropy(big.cuda(), w.cuda(), y.clamp(max=99).cuda())
    ref = torch.nn.functional.cross_entropy(big.double() @ w.double().t(), y.clamp(max=99))
    assert abs(float(loss) - float(ref)) < 1e-4 * float(ref)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, d, v', [(5, 776, 20011), (40, 131, 9001), (700, 72, 3001), (1100, 264, 1543)])
def test_masked_classes_of_large_heads(ops, dt, n, d, v):
    """Masked classes, a masked label, a row of +inf logits and one of NaN, with and without kept logits."""
    g = torch.Generator().manual_seed(n)
    live = v // 3
    h, w = torch.randn(n, d, generator=g).to(dt), (torch.randn(v, d, generator=g) / math.sqrt(d)).to(dt)
    y = torch.randint(0, live, (n,), generator=g)
    for low in (-math.inf, torch.finfo(dt).min):
        b = torch.zeros(v, dtype=dt)
        b[live:] = low
        y[0], y[1] = live + 1 if low == -math.inf else 0, -100
        x = h.clone()
        x[1], x[2, 0] = math.nan, math.nan
        hg, wg, bg = (t.cuda().requires_grad_() for t in (x, w, b))
        loss = ops.linear_cross_entropy(hg, wg, y.cuda(), bg, reduction='none')
        up = torch.ones(n, device='cuda')
        up[2] = 0.0
        z = h.double() @ w.double()[:live].t()
        want = torch.nn.functional.cross_entropy(z, y.clamp(0, live - 1), reduction='none')
        du = (d + 12) * U * float((h.double().abs() @ w.double().abs().t()).max())
        got = loss.detach().cpu().double()
        assert got[1] == 0 and torch.isnan(got[2]) and (got[0] == math.inf or low != -math.inf)
        assert torch.all((got - want)[3:].abs() <= 2 * du + 2.0 ** -18 + 2 * U * want[3:].abs())
        keep = torch.arange(n) != 2
        hg, wg, bg = (t.cuda().requires_grad_() for t in (x[keep], w, b))
        loss = ops.linear_cross_entropy(hg, wg, y[keep].cuda(), bg, reduction='sum')
        dh, dw, db = torch.autograd.grad(loss, (hg, wg, bg))
        assert all(torch.isfinite(t).all() for t in (dh, dw, db)) and torch.all(dh[1] == 0)
        masked = torch.arange(v) >= live
        masked[int(y[0])] = False
        assert torch.all(dw.cpu()[masked] == 0) and torch.all(db.cpu()[masked] == 0)


def test_targets_that_do_not_exist_make_their_row_nan(ops):
    h, w = torch.randn(6, 16).cuda().requires_grad_(), torch.randn(9, 16).cuda().requires_grad_()
    y = torch.tensor([0, 9, -1, 2 ** 40, 8, -100]).cuda()
    loss = ops.linear_cross_entropy(h, w, y, reduction='none')
    assert torch.equal(loss.isnan().cpu(), torch.tensor([False, True, True, True, False, False]))
    dh, = torch.autograd.grad(loss, h, grad_outputs=torch.ones_like(loss))
    assert torch.equal(dh.isnan().all(1).cpu(), torch.tensor([False, True, True, True, False, False]))
    assert torch.equal(dh.isnan().any(1).cpu(), torch.tensor([False, True, True, True, False, False]))
    z = torch.randn(3, 9).cuda().requires_grad_()
    idx = torch.tensor([[0, 1], [9, 0], [2 ** 33, 1]]).cuda()
    loss = ops.topk_distillation(z, torch.zeros(3, 2).cuda(), idx, reduction='none')
    assert torch.equal(loss.isnan().cpu(), torch.tensor([False, True, True]))
    dz, = torch.autograd.grad(loss, z, grad_outputs=torch.ones_like(loss))
    assert torch.equal(dz.isnan().all(1).cpu(), torch.tensor([False, True, True]))


@pytest.mark.parametrize('dt', TYPES)
def test_equal_indices_add_up(ops, dt):
    n, d, v = 5, 16, 12
    h, w = torch.randn(n, d).to(dt).cuda().requires_grad_(), torch.randn(v, d).to(dt).cuda().requires_grad_()
    twice = torch.tensor([3, 3, 7, -1]).repeat(n, 1).cuda(), torch.tensor([0.5, 0.25, 1.0, 9.0]).repeat(n, 1).cuda()
    once = torch.tensor([3, 7]).repeat(n, 1).cuda(), torch.tensor([math.log(math.exp(0.5) + math.exp(0.25)), 1.0]).repeat(n, 1).cuda()
    a = torch.autograd.grad(ops.linear_topk_distillation(h, w, twice[1], twice[0]), (h, w))
    b = torch.autograd.grad(ops.linear_topk_distillation(h, w, once[1], once[0]), (h, w))
    z = (h @ w.t()).detach().requires_grad_()
    a += torch.autograd.grad(ops.topk_distillation(z, twice[1], twice[0]), z)
    b += torch.autograd.grad(ops.topk_distillation(z, once[1], once[0]), z)
    for x, y in zip(a, b):
        assert torch.allclose(x.float(), y.float(), rtol=4 * U16[dt], atol=4 * U16[dt] * float(x.float().abs().max()))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v, k', [(1, 1, 1), (1, 5, 3), (32, 100, 10), (7, 1000, 40), (65, 257, 64), (3, 70001, 16), (130, 16385, 5),
                                     (40, 50, 50), (2, 2050, 1000)])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_distillation_of_logits(ops, dt, n, v, k, reduction):
    g = torch.Generator().manual_seed(n + v + k)
    tau = 2.0
    z = (3 * torch.randn(n, v, generator=g)).to(dt)
    if v > 40:
        z[:, 5] = -math.inf  # a masked class
    values = 2 * torch.randn(n, k, generator=g)
    indices = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]).int()
    indices[indices == 5] = -1
    if n > 3:
        indices[2] = -1
        values[3] = -math.inf
    lse = (torch.logsumexp(values.double() / tau, 1) + 0.2).float() if k % 2 == 0 and n <= 3 else None
    p, at, live = _targets(values=values, indices=indices, lse=lse, tau=tau)
    z[~live] = math.nan
    grad = torch.rand(n, generator=g) if reduction == 'none' else torch.ones(n)
    zg = z.cuda().requires_grad_()
    loss = ops.topk_distillation(zg, values.cuda(), indices.cuda(), temperature=tau, reduction=reduction,
                                 top_lse=None if lse is None else lse.cuda())
    got, = torch.autograd.grad(loss, zg, grad_outputs=grad.cuda() if reduction == 'none' else torch.ones_like(loss))
    want, rows, dz, q, coef = _formula(z.double(), p, at, live, tau, reduction, grad)
    du = 2 * U * float(z.nan_to_num(neginf=0.0).abs().max()) / tau
    row_tol = tau * tau * p.sum(1) * (2 * du + 2.0 ** -18) + 2 * U * rows.abs() + 1e-30
    tol = row_tol if reduction == 'none' else row_tol.sum() / max(1, int(live.sum())) + U * want.abs()
    assert torch.all((loss.detach().cpu().double() - want).abs() <= tol)
    bound = U16[dt] * dz.abs() + (2 * du + 2.0 ** -18) * coef * q + (2.0 ** -25 if dt == torch.float16 else 1e-37)
    off = (got.cpu().double() - dz).abs()
    assert got.dtype == dt and torch.all(off <= bound), float((off / bound).max())
    assert torch.all(got.cpu()[~live] == 0)


@pytest.mark.parametrize('dt', TYPES)
def test_distillation_of_strided_logits_and_leading_axes(ops, dt):
    g = torch.Generator().manual_seed(8)
    big = torch.randn(4, 6, 70, generator=g).to(dt).cuda()
    values, indices = torch.randn(4, 6, 3, generator=g).cuda(), torch.randint(0, 50, (4, 6, 3), generator=g).cuda()
    z = big[:, :, 7:57]
    plain = z.contiguous().requires_grad_()
    view = big.clone().requires_grad_()
    a = ops.topk_distillation(view[:, :, 7:57], values, indices, reduction='none')
    b = ops.topk_distillation(plain, values, indices, reduction='none')
    assert a.shape == (4, 6) and torch.allclose(a, b, rtol=1e-6)
    ga, = torch.autograd.grad(a.sum(), view)
    gb, = torch.autograd.grad(b.sum(), plain)
    assert torch.allclose(ga[:, :, 7:57].float(), gb.float(), rtol=2 * U16[dt], atol=1e-7)
    h = torch.randn(4, 6, 16, generator=g).to(dt).cuda()
    w = torch.randn(50, 16, generator=g).to(dt).cuda()
    y = torch.randint(0, 50, (4, 6), generator=g).cuda()
    per = ops.linear_cross_entropy(h, w, y, reduction='none')
    flat = ops.linear_cross_entropy(h.reshape(24, 16), w, y.reshape(24).int(), reduction='none')
    assert per.shape == (4, 6) and torch.equal(per.reshape(24), flat)
    v3, i3, l3 = ops.top_logits(z, 5)
    assert v3.shape == i3.shape == (4, 6, 5) and l3.shape == (4, 6)
    v2, i2, l2 = ops.top_logits(z.reshape(24, 50), 5)
    assert torch.equal(v3.reshape(24, 5), v2) and torch.equal(i3.reshape(24, 5), i2) and torch.equal(l3.reshape(24), l2)


def _top_reference(z, k, tau):
    x = z.double().cpu()
    x = torch.where(x.isnan(), torch.tensor(math.inf, dtype=torch.float64) , x)
    nan_first = torch.sort((~z.cpu().isnan()).int(), dim=1, stable=True).indices  # NaN, then the rest, each by class
    order = torch.sort(x.gather(1, nan_first), dim=1, descending=True, stable=True).indices
    idx = nan_first.gather(1, order)[:, :k]
    return z.cpu().gather(1, idx), idx.int(), torch.logsumexp(z.double().cpu() / tau, 1)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v, k', [(1, 1, 1), (5, 3, 3), (400, 1000, 10), (3, 257, 64), (70, 64, 64), (2, 131072, 64), (9, 50001, 200),
                                     (4, 4099, 1024), (1, 300000, 7)])
def test_top_logits(ops, dt, n, v, k):
    g = torch.Generator().manual_seed(n + v)
    z = (3 * torch.randn(n, v, generator=g)).to(dt)
    got = ops.top_logits(z.cuda(), k, temperature=2.0)
    want = _top_reference(z, k, 2.0)
    assert got[0].dtype == dt and got[1].dtype == torch.int32
    assert torch.equal(got[1].cpu(), want[1]) and torch.equal(got[0].cpu(), want[0])
    assert torch.allclose(got[2].cpu().double(), want[2], rtol=0, atol=2.0 ** -18)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n, v, k', [(3, 131072, 200), (5, 140001, 129), (2, 50001, 384), (2, 50001, 385), (3, 20011, 768), (2, 9000, 1000),
                                     (1100, 8200, 1000), (1030, 8200, 700), (600, 49153, 16)])
def test_top_logits_of_every_block_width(ops, dt, n, v, k):
    """Equal 16-bit logits abound: ties go to the lower class."""
    g = torch.Generator(device='cuda').manual_seed(v + k)
    z = (3 * torch.randn(n, v, generator=g, device='cuda')).to(dt)
    values, indices, lse = ops.top_logits(z, k, temperature=2.0)
    order = torch.sort(z.float(), dim=1, descending=True, stable=True)
    assert torch.equal(values.float(), order.values[:, :k]) and torch.equal(indices.long(), order.indices[:, :k])
    want = torch.logsumexp(z.double() / 2, 1)
    assert torch.all((lse.double() - want).abs() <= 2.0 ** -18 + 2 * U * want.abs())


@pytest.mark.parametrize('dt', TYPES)
def test_top_logits_of_ties_masks_and_nan(ops, dt):
    n, v, k = 8, 3000, 30
    g = torch.Generator().manual_seed(9)
    z = torch.randint(-2, 3, (n, v), generator=g).to(dt)  # thousands of equal values
    z[1] = 0.0
    z[1, ::2] = -0.0  # the two zeros are equal
    z[2] = -math.inf
    z[2, 17] = 1.0  # fewer finite values than k
    z[3, 100] = math.inf
    z[4, 2000:2003] = math.nan
    z[5] = math.nan
    z[6] = torch.finfo(dt).min
    z[7] = -math.inf
    got = ops.top_logits(z.cuda(), k)
    want = _top_reference(z, k, 1.0)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu().isnan(), want[0].isnan())
    assert torch.equal(got[0].cpu().nan_to_num(7.0), want[0].nan_to_num(7.0))
    assert got[2][7] == -math.inf and got[2][4].isnan() and got[2][5].isnan()


def test_gradients_against_differences(ops):
    g = torch.Generator().manual_seed(10)
    n, d, v, k = 9, 20, 31, 4
    h, w, b = torch.randn(n, d, generator=g), torch.randn(v, d, generator=g) / 3, torch.randn(v, generator=g)
    y = torch.randint(0, v, (n,), generator=g).cuda()
    values, indices = torch.randn(n, k, generator=g).cuda(), torch.randint(0, v, (n, k), generator=g).cuda()
    calls = [lambda h, w, b: ops.linear_cross_entropy(h, w, y, b),
             lambda h, w, b: ops.linear_topk_distillation(h, w, values, indices, b, temperature=2.0),
             lambda h, w, b: ops.topk_distillation(h @ w.t() + b, values, indices, temperature=2.0)]
    for call in calls:
        leaves = [t.cuda().requires_grad_() for t in (h, w, b)]
        grads = torch.autograd.grad(call(*leaves), leaves)
        for i in range(3):
            step = torch.randn(leaves[i].shape, generator=g).cuda()
            eps = 2.0 ** -6
            with torch.no_grad():
                args = [t.detach() for t in leaves]
                up, down = ([t + (s * eps * step if j == i else 0) for j, t in enumerate(args)] for s in (1, -1))
                slope = (call(*up).double() - call(*down).double()) / (2 * eps)
            # central difference: eps^2 / 6 of the third derivative (under |step|^3 of unit curvature), rounding 2^-20 / eps
            assert abs(float(slope) - float((grads[i] * step).sum())) < 2e-2 * max(1.0, abs(float(slope)))


def test_same_inputs_same_bits_and_second_backward_refused(ops):
    g = torch.Generator(device='cuda').manual_seed(11)
    for dt in TYPES:
        h = torch.randn(300, 96, generator=g, device='cuda').to(dt).requires_grad_()
        w = torch.randn(1000, 96, generator=g, device='cuda').to(dt).requires_grad_()
        z = torch.randn(300, 1000, generator=g, device='cuda').to(dt).requires_grad_()
        values, indices, _ = ops.top_logits(z, 20)
        first = None
        for _ in range(3):
            loss = ops.linear_topk_distillation(h, w, values, indices)
            kd = ops.topk_distillation(z, values, indices)
            out = [loss.detach(), kd.detach(), *torch.autograd.grad(loss, (h, w), retain_graph=True), *torch.autograd.grad(kd, z)]
            out += torch.autograd.grad(loss, (h, w))  # the saved state serves twice
            first = first or out
            assert all(torch.equal(a, b) for a, b in zip(first, out))
            assert torch.equal(out[2], out[5]) and torch.equal(out[3], out[6])
        dh, = torch.autograd.grad(ops.linear_topk_distillation(h, w, values, indices), h, create_graph=True)
        with pytest.raises(RuntimeError):
            dh.float().sum().backward()


def test_other_streams_and_partial_gradients(ops):
    g = torch.Generator(device='cuda').manual_seed(12)
    h = torch.randn(200, 64, generator=g, device='cuda').bfloat16().requires_grad_()
    w = torch.randn(500, 64, generator=g, device='cuda').bfloat16().requires_grad_()
    y = torch.randint(0, 500, (200,), generator=g, device='cuda')
    want = torch.autograd.grad(ops.linear_cross_entropy(h, w, y), (h, w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # three calls in flight at once, each with buffers of its own
        with torch.cuda.stream(s):
            outs.append(torch.autograd.grad(ops.linear_cross_entropy(h, w, y), (h, w)))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    dw, = torch.autograd.grad(ops.linear_cross_entropy(h.detach(), w, y), w)
    dh, = torch.autograd.grad(ops.linear_cross_entropy(h, w.detach(), y), h)
    assert torch.equal(dh, want[0]) and torch.equal(dw, want[1])


def test_captured_training_steps_replay(ops):
    """Two captured graphs (cross entropy, distillation from the teacher's top logits), replayed in turn with new inputs and
    eager work between the replays."""
    g = torch.Generator(device='cuda').manual_seed(13)
    n, d, v, k = 96, 64, 700, 12
    h = torch.zeros(n, d, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    w = torch.zeros(v, d, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    y = torch.zeros(n, dtype=torch.int64, device='cuda')
    t = torch.zeros(n, v, device='cuda')

    def ce():
        loss = ops.linear_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    def kd():
        values, indices, lse = ops.top_logits(t, k, temperature=2.0)
        loss = ops.linear_topk_distillation(h, w, values, indices, temperature=2.0, top_lse=lse)
        return (loss.detach(), values, indices, *torch.autograd.grad(loss, (h, w)))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ce(), kd()
    torch.cuda.synchronize()
    graphs = []
    for step in (ce, kd):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step))
    for _ in range(4):
        with torch.no_grad():
            h.copy_(torch.randn(n, d, generator=g, device='cuda'))
            w.copy_(torch.randn(v, d, generator=g, device='cuda') / 4)
            t.copy_(torch.randn(n, v, generator=g, device='cuda') * 2)
            y.copy_(torch.randint(0, v, (n,), generator=g, device='cuda'))
            y[::5] = -100
        for graph, out, step in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, step in graphs:
            for a, b in zip(out, step()):
                assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_capture_is_refused_while_an_eager_graph_of_the_same_leaves_lives(ops):
    """A leaf's accumulator stays on the stream of the pass that made it; captured, that stream would wait for the capture,
    which ends the process."""
    h, w = (torch.randn(n, 64, device='cuda').requires_grad_() for n in (40, 6000))
    z = torch.randn(20, 50, device='cuda').requires_grad_()
    y = torch.randint(0, 6000, (40,), device='cuda')
    top = torch.zeros(20, 3, device='cuda'), torch.arange(60, device='cuda').view(20, 3) % 50

    def head():
        return ops.linear_cross_entropy(h, w, y)

    def logits():
        return ops.topk_distillation(z, *top)

    def grads(loss, leaves):
        return [loss.detach().clone()] + [g.clone() for g in torch.autograd.grad(loss, leaves)]
    for call, leaves in ((head, (h, w)), (logits, (z,))):
        kept = call()  # its graph holds the leaves' accumulators
        want = grads(call(), leaves)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match='earlier pass'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                grads(call(), leaves)
        for grad_mode in (False, True):  # nothing to capture backwards
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph), torch.set_grad_enabled(grad_mode):
                alone = call().detach()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(alone, want[0])
        del kept
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = grads(call(), leaves)
        for _ in range(3):
            for t in got:
                t.fill_(7)
            graph.replay()
            grads(call(), leaves)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_teacher_and_a_student_head_together(ops):
    """As they are used: the teacher's top logits once, the student's steps from them -- through logits that are kept and
    through the head, which agree."""
    g = torch.Generator(device='cuda').manual_seed(14)
    n, d, v, k, tau = 150, 80, 900, 16, 2.0
    h = torch.randn(n, d, generator=g, device='cuda')
    teacher = torch.randn(v, d, generator=g, device='cuda') / 4
    w = torch.randn(v, d, generator=g, device='cuda') / 4
    b = torch.zeros(v, device='cuda')
    values, indices, lse = ops.top_logits(h @ teacher.t(), k, temperature=tau)
    w1, b1 = w.clone().requires_grad_(), b.clone().requires_grad_()
    w2, b2 = w.clone().requires_grad_(), b.clone().requires_grad_()
    for _ in range(3):
        la = ops.linear_topk_distillation(h, w1, values, indices, b1, temperature=tau, top_lse=lse)
        lb = ops.topk_distillation(torch.nn.functional.linear(h, w2, b2), values, indices, temperature=tau, top_lse=lse)
        ga, gb = torch.autograd.grad(la, (w1, b1)), torch.autograd.grad(lb, (w2, b2))
        assert abs(float(la) - float(lb)) < 1e-5 * abs(float(la)) + 1e-6
        for x, y2 in zip(ga, gb):
            assert float((x - y2).norm()) < 1e-5 * float(y2.norm())
        with torch.no_grad():
            for t, gr in ((w1, ga[0]), (b1, ga[1]), (w2, gb[0]), (b2, gb[1])):
                t -= 0.1 * gr


def test_errors_of_the_autograd_functions_are_the_librarys_own(ops):
    from neuron_interpolation_model_fusion_amd import _lib
    with pytest.raises(_lib.NifError, match='nif_top_logits failed with status -1'):
        _lib.nif_torch.top_logits(torch.zeros(2, 3, device='cuda'), 4, 1.0)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(torch.zeros(2, 3, device='cuda'), torch.zeros(4, 2, device='cuda'), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(_lib.NifError):  # one tensor on the host
        ops.linear_cross_entropy(torch.zeros(2, 3, device='cuda'), torch.zeros(4, 3, device='cuda'), torch.zeros(2, dtype=torch.int64))
