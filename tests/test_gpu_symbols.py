"""Symbol log probabilities, entropies, alternatives and their gradient against the definition in 64 bits.

Tolerances.  l - m is rounded once (2^-24 of its size, at most D = 104: below that a class adds nothing), an exponential
is good to 2^-22 plus the error of its argument, sums of positive terms keep the largest relative error of their terms
plus 2^-24 per addition (at most `chain` in a row: a thread's or a lane's share and the joins), a logarithm adds its own
2^-22.  So log p is off by at most (2 D + 16 + chain) 2^-23 and an entropy, the mean of |log p| under p, by that times
(2 + H) or less; a gradient, a product of these with probabilities at most one, by that times (|g_lp| + |g_H| (2 + 2 H))
plus half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.bfloat16, torch.float16)
NEG = float("-inf")


def definition(logits, symbols, top=0):
    """float64, any layout (N, C * V, h, w) / (N, V): log_prob, entropy, top lp, top classes, log p of all, p of all."""
    rows = logits.dim() == 2
    x = logits.double()
    x = x.view(x.size(0), 1, x.size(1), 1, 1) if rows else x.view(x.size(0), symbols.size(1), -1, *x.shape[2:])
    sym = symbols.view(-1, 1, 1, 1).long() if rows else symbols.long()
    v = x.size(2)
    bad = x.isnan().any(2, keepdim=True) | (x == float("inf")).any(2, keepdim=True)
    m = x.amax(2, keepdim=True)
    empty = m == NEG
    e = torch.exp(x - torch.where(empty, 0.0, m))
    total = e.sum(2, keepdim=True)
    lp = x - torch.where(empty, 0.0, m) - torch.where(empty, 0.0, total.log())
    lp = torch.where(bad, float("nan"), lp)
    p = torch.where(empty, 0.0, e / total)
    p = torch.where(bad, float("nan"), p)
    h = -torch.where(p == 0, 0.0, p * lp).sum(2)
    given = lp.gather(2, sym.clamp(0, v - 1)[:, :, None])[:, :, 0]
    given = torch.where(sym < 0, 0.0, torch.where(sym >= v, float("nan"), given))
    out = [given.view(symbols.shape), h.view(symbols.shape)]
    order = torch.sort(x, dim=2, descending=True, stable=True).indices[:, :, :top]
    shape = (x.size(0), top) if rows else (x.size(0), symbols.size(1) * top, *x.shape[3:])
    return out + [lp.gather(2, order).reshape(shape), order.to(torch.int32).reshape(shape), lp, p]


def step(classes, lp):
    fine = lp[torch.isfinite(lp)]
    d = min(104.0, float(fine.abs().max()) if fine.numel() else 0.0)
    return (2 * d + 16 + -(-classes // 64) + 64) * 2.0 ** -23


def same(got, want, tol):
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan())
    rest = ~fine & ~want.isnan()
    assert torch.equal(got[rest], want[rest])
    assert bool(((got - want).abs()[fine] <= (tol[fine] if torch.is_tensor(tol) else tol)).all()), float((got - want).abs()[fine].max())


CASES = [
    # groups (0: rows), classes, n, h, w
    (0, 1, 3, 0, 0), (0, 2, 130, 0, 0), (0, 37, 5, 0, 0), (0, 64, 64, 0, 0), (0, 257, 7, 0, 0), (0, 1000, 9, 0, 0), (0, 2049, 3, 0, 0),
    (0, 5003, 2, 0, 0), (0, 40001, 1, 0, 0), (0, 131072, 2, 0, 0),
    (1, 5, 1, 1, 1), (3, 7, 2, 1, 1), (1, 16, 2, 3, 5), (4, 64, 2, 16, 16), (7, 37, 1, 9, 13), (2, 300, 1, 8, 8), (1, 1000, 1, 2, 2), (2, 3, 1, 40, 70),
]


def inputs(groups, classes, n, h, w, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + classes + n + h)
    rows = groups == 0
    place = (n, classes) if rows else (n, groups * classes, h, w)
    site = (n,) if rows else (n, groups, h, w)
    logits = 4 * torch.randn(place, generator=g)
    logits = torch.where(torch.rand(place, generator=g) < 0.1, torch.full((), NEG), logits)
    logits = torch.where(torch.rand(place, generator=g) < 0.05, torch.full((), torch.finfo(dtype).min), logits)
    logits = logits.to(dtype)
    symbols = torch.randint(-1, classes, site, generator=g, dtype=torch.int32)
    return logits, symbols, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,classes,n,h,w", CASES)
def test_forward_and_alternatives(groups, classes, n, h, w, dtype):
    from deepvideocodec_amd import ops
    logits, symbols, _ = inputs(groups, classes, n, h, w, dtype)
    for top in {0, 1, min(5, classes), min(16, classes)}:
        given, ent, tl, ts, lp, p = definition(logits, symbols, top)
        r = ops.symbol_log_probs(logits.cuda(), symbols.cuda(), top)
        tol = step(classes, lp)
        # (a masked class at the type's lowest value has log p ~ -1e38: relative there)
        same(r.log_prob, given, tol + given.abs().nan_to_num(0, 0, 0) * 2.0 ** -23)
        same(r.entropy, ent, tol * (2 + ent))
        assert (r.top_log_prob is None) == (top == 0)
        if top:
            assert torch.equal(r.top_symbol.cpu(), ts)
            same(r.top_log_prob, tl, tol + tl.abs().nan_to_num(0, 0, 0) * 2.0 ** -23)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("groups,classes,n,h,w", CASES)
def test_gradient(groups, classes, n, h, w, dtype):
    from deepvideocodec_amd import autograd as A
    logits, symbols, g = inputs(groups, classes, n, h, w, dtype, 1)
    _, ent, _, _, lp, p = definition(logits, symbols)
    gl, gh = (torch.randn(symbols.shape, generator=g) for _ in range(2))
    x = logits.cuda().requires_grad_()
    tol = step(classes, lp)
    for use_l, use_h in ((True, True), (True, False), (False, True)):
        r = A.symbol_log_probs(x, symbols.cuda())
        outs = [r[0]] * use_l + [r[1]] * use_h
        seeds = [gl.cuda()] * use_l + [gh.cuda()] * use_h
        (got,) = torch.autograd.grad(outs, x, seeds)
        assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
        full = lambda t: t.double().view(lp.size(0), lp.size(1), 1, *lp.shape[3:])
        sym = full(symbols).long()
        a = torch.where(sym < 0, 0.0, full(gl)) * use_l
        b = full(gh) * use_h
        want = -p * a - b * torch.where(p == 0, 0.0, p * (lp + full(ent)))
        want = want + a * (torch.arange(classes).view(1, 1, -1, 1, 1) == sym)
        bound = tol * (a.abs() + b.abs() * (2 + 2 * full(ent))) + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal
        same(got, want.view(logits.shape), bound.expand(want.shape).reshape(logits.shape))


def test_gradient_against_differences():
    """In 64 bits by the definition, central differences of the returned quantities' definition."""
    from deepvideocodec_amd import autograd as A
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 2, 3, generator=g)
    sym = torch.randint(0, 3, (2, 2, 2, 3), generator=g, dtype=torch.int32)
    gl, gh = torch.randn(sym.shape, generator=g), torch.randn(sym.shape, generator=g)
    xc = x.cuda().requires_grad_()
    r = A.symbol_log_probs(xc, sym.cuda())
    (got,) = torch.autograd.grad((r[0], r[1]), xc, (gl.cuda(), gh.cuda()))

    def f(t):
        d = definition(t, sym)
        return float((d[0] * gl.double()).sum() + (d[1] * gh.double()).sum())

    eps = 2.0 ** -12
    for i in range(0, x.numel(), 5):
        up, dn = x.double().flatten().clone(), x.double().flatten().clone()
        up[i] += eps
        dn[i] -= eps
        # third derivatives of log-softmax and entropy are below 8 |g| here: eps^2 / 6 of that, plus fp32
        assert abs(float(got.flatten()[i]) - (f(up.view(x.shape)) - f(dn.view(x.shape))) / (2 * eps)) < 16 * eps * eps + 64 * 2.0 ** -23


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [True, False])
def test_masks_and_values_that_are_not_finite(dtype, rows):
    from deepvideocodec_amd import autograd as A, ops
    low = torch.finfo(dtype).min
    inf, nan = float("inf"), float("nan")
    sites = [[NEG] * 6, [low] * 6, [low, NEG, low, NEG, NEG, NEG], [NEG, NEG, 3.0, NEG, NEG, NEG], [0.0, -0.0, 0.0, -0.0, NEG, 0.0],
             [1.0, inf, 2.0, 0.0, 0.0, 0.0], [1.0, nan, 2.0, 3.0, nan, 0.0], [low, 0.0, low, 0.0, 1.0, low], [NEG, nan, NEG, NEG, NEG, NEG],
             [5e4, -5e4, 5e4, 5e4, -5e4, 0.0]]
    t = torch.tensor(sites).to(dtype)
    symbols = torch.tensor([2, 1, 1, 2, 3, 0, 0, 4, 0, 1], dtype=torch.int32)
    if not rows:
        t = t.t().reshape(1, 6, 2, 5).contiguous()
        symbols = symbols.view(1, 1, 2, 5)
    given, ent, tl, ts, lp, p = definition(t, symbols, 6)
    r = ops.symbol_log_probs(t.cuda(), symbols.cuda(), 6)
    same(r.log_prob, given, 1e-5 + given.abs().nan_to_num(0, 0, 0) * 2.0 ** -22)     # (2 * 104 + 81) 2^-23 < 4e-5: 1e-5 holds for D < 2
    same(r.entropy, ent, 1e-5)
    assert torch.equal(r.top_symbol.cpu(), ts)
    x = t.cuda().requires_grad_()
    o = A.symbol_log_probs(x, symbols.cuda())
    (grad,) = torch.autograd.grad((o[0], o[1]), x, (torch.ones_like(o[0]), torch.ones_like(o[1])))
    grad = (grad if rows else grad.view(6, 10).t()).cpu()
    assert bool(torch.isfinite(grad[[0, 1, 2, 3, 4, 7, 9]]).all()) and bool(grad[[5, 6, 8]].isnan().any(1).all())
    assert grad[0].tolist() == [0, 0, 1, 0, 0, 0]      # nothing may occur: only the given class's own term
    assert grad[3].tolist() == [0, 0, 0, 0, 0, 0]      # certain: no gradient


@pytest.mark.parametrize("dtype", TYPES)
def test_long_rows_of_every_kind(dtype):
    """Rows that are cut over workgroups: one value throughout, rising, falling, nothing allowed, one class allowed, a NaN, an
    infinity, the best classes in one place or at the ends."""
    from deepvideocodec_amd import ops
    v = 50003
    g = torch.Generator().manual_seed(11)
    noise = torch.randn(v, generator=g)
    rows = [torch.full((v,), 1.5), torch.arange(v) / 512.0, -torch.arange(v) / 512.0, torch.full((v,), NEG), torch.full((v,), NEG),
            noise.clone(), noise.clone(), noise.clone(), noise.clone(), torch.full((v,), torch.finfo(dtype).min)]
    rows[4][31007] = -3.0
    rows[5][40000] = float("nan")
    rows[6][123] = float("inf")
    rows[7][20000:20040] += 20
    rows[8][[0, 1, 2, v - 1, v - 2, v - 3]] += 30
    x = torch.stack(rows).to(dtype)
    sym = torch.tensor([5, v - 1, 0, 7, 31007, 3, 123, 20001, v - 1, 9], dtype=torch.int32)
    given, ent, tl, ts, lp, p = definition(x, sym, 16)
    for n in (10, 1):                     # in nine parts, in twelve
        r = ops.symbol_log_probs(x[:n].cuda(), sym[:n].cuda(), 16)
        tol = (2 * 104 + 16 + -(-v // 64) + 64) * 2.0 ** -23
        same(r.log_prob, given[:n], tol + given[:n].abs().nan_to_num(0, 0, 0) * 2.0 ** -23)
        same(r.entropy, ent[:n], tol * (2 + ent[:n].nan_to_num(0)))
        assert torch.equal(r.top_symbol.cpu(), ts[:n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", (1, 2, 3, 7, 31, 64, 65, 100, 128, 129, 255, 256))
def test_many_short_rows(classes, dtype):
    """Rows that share a wave: values, alternatives and gradient; masked rows, a NaN, an infinity; rows that follow each other on
    16 bytes, off them, and rows apart."""
    from deepvideocodec_amd import ops
    n = 8192 + 37
    logits, symbols, g = inputs(0, classes, n, 0, 0, dtype, 5)
    logits[100] = NEG
    logits[8191] = torch.finfo(dtype).min
    logits[8200, classes // 2] = float("nan")
    logits[n - 1, classes - 1] = float("inf")
    symbols[[0, 64, n - 2]] = classes
    top = min(classes, 8)
    given, ent, tl, ts, lp, p = definition(logits, symbols, top)
    tol = step(classes, lp)
    gl, gh = (torch.randn(n, generator=g) for _ in range(2))
    a, b = torch.where(symbols < 0, 0.0, gl.double())[:, None], gh.double()[:, None]
    pr, lpr = p.view(n, classes), lp.view(n, classes)
    want = -pr * a - b * torch.where(pr == 0, 0.0, pr * (lpr + ent[:, None])) + a * (torch.arange(classes)[None] == symbols[:, None])
    want[symbols == classes] = float("nan")
    bound = tol * (a.abs() + b.abs() * (2 + 2 * ent[:, None].nan_to_num(0))) + want.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal
    flat = torch.zeros(n * classes + 1, dtype=dtype).cuda()
    wide = torch.zeros(n, classes + 3, dtype=dtype).cuda()
    for x in (logits.cuda(), flat[1:].view(n, classes), wide[:, 1:1 + classes]):
        x.copy_(logits)
        for t in {0, 1, min(3, top), top, min(classes, 16)}:
            r = ops.symbol_log_probs(x, symbols.cuda(), t)
            same(r.log_prob, given, tol + given.abs().nan_to_num(0, 0, 0) * 2.0 ** -23)
            same(r.entropy, ent, tol * (2 + ent.nan_to_num(0)))
            if 0 < t <= top:
                assert torch.equal(r.top_symbol.cpu(), ts[:, :t])
                same(r.top_log_prob, tl[:, :t], tol + tl[:, :t].abs().nan_to_num(0, 0, 0) * 2.0 ** -23)
        got = ops.symbol_log_probs_backward(x, symbols.cuda(), r.stats, r.entropy, gl.cuda(), gh.cuda())
        same(got, want, bound)


@pytest.mark.parametrize("classes", [40, 65536, 65537, 70001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_alternatives_in_planes_of_very_many_classes(dtype, classes):
    """16-bit planes around 65536 classes: ties, signed zeros, an infinity, a NaN, minus infinity throughout."""
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(18)
    x = torch.randint(-3, 4, (1, classes, 2, 3), generator=g).to(dtype)
    x = torch.where((x == 0) & (torch.rand(x.shape, generator=g) < 0.5), -x, x)
    x[0, -1, 0, 0] = float("inf")
    x[0, classes // 2, 0, 1] = float("nan")
    x[0, :, 0, 2] = NEG
    x[0, :, 1, 0] = torch.where(torch.arange(classes) == classes - 2, 0.0, float("nan")).to(dtype)
    x[0, :, 1, 1] = -x[0, :, 1, 1].abs()
    sym = torch.randint(0, classes, (1, 1, 2, 3), generator=g, dtype=torch.int32)
    for top in (1, 3, 7, 16):
        given, ent, tl, ts, lp, p = definition(x, sym, top)
        r = ops.symbol_log_probs(x.cuda(), sym.cuda(), top)
        assert torch.equal(r.top_symbol.cpu(), ts)
        tol = (2 * 104 + 16 + classes + 64) * 2.0 ** -23
        same(r.log_prob, given, tol)
        same(r.top_log_prob, tl, tol)


def sums64(x):
    """float64, classes first: log p of all, entropies."""
    lp = x.double() - x.double().logsumexp(0, keepdim=True)
    return lp, -torch.where(lp == NEG, 0.0, lp.exp() * lp).sum(0)


@pytest.mark.parametrize("values", ["whole", "normal"])
@pytest.mark.parametrize("n,classes,top", [(2048, 131072, 0), (2048, 65536, 2), (64, 131072, 8), (1, 131072, 16), (1, 100003, 0)])
def test_sums_over_very_many_classes_in_planes(n, classes, top, values):
    """Sums over a hundred thousand classes keep fp32's accuracy whatever a lane has to add up (n samples of the same 8 x 8
    pixels: from 2048 on a lane takes every class): a lane adds at most 263 terms in fp32 in a row, its share is one of at
    most 16.  Whole logits: the terms repeat, so that the roundings of a long fp32 sum do not cancel."""
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(31 + classes)
    place = (1, classes, 8, 8)
    x = (torch.randint(-3, 4, place, generator=g) if values == "whole" else 3 * torch.randn(place, generator=g)).bfloat16().cuda()
    sym = torch.randint(0, classes, (1, 1, 8, 8), generator=g, dtype=torch.int32).cuda()
    lp, ent = sums64(x.view(classes, 64))
    given = lp.gather(0, sym.view(1, 64).long())
    r = ops.symbol_log_probs(x.expand(n, *place[1:]), sym.expand(n, 1, 8, 8).contiguous(), top)
    tol = (2 * float(lp.abs().max()) + 16 + 263 + 16) * 2.0 ** -23
    assert float((r.log_prob.view(n, 64) - given).abs().max()) <= tol
    assert bool(((r.entropy.view(n, 64) - ent).abs() <= tol * (2 + ent)).all())
    if top:
        best = torch.sort(x.view(classes, 64).float(), dim=0, descending=True, stable=True).indices[:top]
        assert torch.equal(r.top_symbol.view(n, top, 64), best.to(torch.int32).expand(n, top, 64))
        assert float((r.top_log_prob.view(n, top, 64) - lp.gather(0, best)).abs().max()) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,classes,top", [(512, (1 << 24) + 5, 0), (512, 1000003, 8), (1, (1 << 24) + 5, 8), (3, 300007, 1)])
def test_sums_over_very_long_rows(n, classes, top, dtype):
    """The same for rows (n sites over one row): with 512 of them a workgroup takes a whole row, 65536 classes a lane.  A lane adds
    at most 256 + 2 terms in a row, then come 64 lanes and at most 64 parts."""
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(33)
    x = torch.randint(-3, 4, (classes,), generator=g).to(dtype).cuda()
    sym = torch.randint(0, classes, (n,), generator=g, dtype=torch.int32).cuda()
    lp, ent = sums64(x.view(classes, 1))
    r = ops.symbol_log_probs(x.expand(n, classes), sym, top)
    tol = (2 * float(lp.abs().max()) + 16 + 258 + 16) * 2.0 ** -23
    assert float((r.log_prob - lp[sym.long(), 0]).abs().max()) <= tol
    assert float((r.entropy - ent).abs().max()) <= tol * (2 + float(ent))
    if top:
        best = torch.nonzero(x == 3)[:top, 0]
        assert torch.equal(r.top_symbol, best.to(torch.int32).expand(n, top))
        assert float((r.top_log_prob - lp[best, 0]).abs().max()) <= tol
    for bad in (float("nan"), float("inf")):
        x[classes - 3] = bad
        r = ops.symbol_log_probs(x.expand(n, classes), sym, top)
        assert bool(r.log_prob.isnan().all()) and bool(r.entropy.isnan().all())
        if top:
            assert bool((r.top_symbol[:, 0] == classes - 3).all()) and torch.equal(r.top_symbol[:, 1:], best[:top - 1].to(torch.int32).expand(n, top - 1))


def test_transposed_rows_of_very_many_classes():
    """(N, classes) logits whose classes lie apart: values and gradient, with a masked row, a NaN and an infinity."""
    from deepvideocodec_amd import ops
    v, n = 1 << 20, 64
    g = torch.Generator().manual_seed(32)
    xt = torch.randint(-3, 4, (v, n), generator=g).bfloat16()
    xt[:, 5] = NEG
    xt[77777, 6] = float("nan")
    xt[7, 7] = float("inf")
    xt[:, 8] = torch.where(torch.arange(v) == 900001, 2.0, NEG)
    xt[:, 9] = torch.arange(v) * (1.0 / 4096)                  # a maximum that keeps growing
    xt = xt.cuda()
    sym = torch.randint(0, v, (n,), generator=g, dtype=torch.int32).cuda()
    fine = [i for i in range(n) if i not in (5, 6, 7)]
    lp, ent = sums64(xt[:, fine])
    spread = float(lp[torch.isfinite(lp)].abs().max().clamp(max=104))
    # 263 terms in a row, 16 shares; the growing maximum rescales each of its 1024 stretches, a rounding each
    tol = (2 * spread + 16 + 263 + 16 + 1024) * 2.0 ** -23
    gl = torch.randn(n, generator=g).cuda()
    for top in (0, 8):
        r = ops.symbol_log_probs(xt.t(), sym, top)
        assert r.log_prob[5] == NEG and r.entropy[5] == 0 and bool(r.log_prob[6:8].isnan().all()) and bool(r.entropy[6:8].isnan().all())
        given = lp.gather(0, sym[fine].view(1, -1).long())[0]
        at = torch.isfinite(given)
        assert torch.equal(r.log_prob[fine][~at].double(), given[~at])
        assert bool(((r.log_prob[fine] - given)[at].abs() <= tol + given[at].abs() * 2.0 ** -23).all())
        assert bool(((r.entropy[fine] - ent).abs() <= tol * (2 + ent)).all())
        got = ops.symbol_log_probs_backward(xt.t(), sym, r.stats, r.entropy, gl, gl).t()[:, fine].double()
        p, a = lp.exp(), gl[fine].double()
        want = -p * a * (1 + torch.where(p == 0, 0.0, lp + ent)) + a * (torch.arange(v, device="cuda")[:, None] == sym[fine])
        bound = tol * a.abs() * (3 + 2 * ent) + want.abs() * 2.0 ** -8 + torch.finfo(torch.bfloat16).smallest_normal
        assert bool(((got - want).abs() <= bound).all())


def test_one_row_for_all_sites():
    """Expanded logits (no stride between rows), also where rows share waves."""
    from deepvideocodec_amd import ops
    for classes in (37, 300):
        g = torch.Generator().manual_seed(15)
        x = torch.randn(1, classes, generator=g).cuda().expand(9000, classes)
        sym = torch.randint(-1, classes, (9000,), generator=g, dtype=torch.int32).cuda()
        gl = torch.randn(9000, generator=g).cuda()
        res = [ops.symbol_log_probs(t, sym, 3) for t in (x, x.contiguous())]
        grads = [ops.symbol_log_probs_backward(t, sym, r.stats, r.entropy, gl, gl) for t, r in zip((x, x.contiguous()), res)]
        for a, b in zip((*res[0], grads[0]), (*res[1], grads[1])):
            assert torch.equal(a, b)


def test_no_second_derivative():
    from deepvideocodec_amd import autograd as A
    x = torch.randn(4, 9, generator=torch.Generator().manual_seed(16)).cuda().requires_grad_()
    lp = A.symbol_log_probs(x, torch.zeros(4, dtype=torch.int32).cuda())[0]
    (grad,) = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad"):
        grad.sum().backward()
    lp = A.symbol_log_probs(x, torch.zeros(4, dtype=torch.int32).cuda())[0]
    (grad,) = torch.autograd.grad((lp * lp).sum(), x, create_graph=True)      # (the seed depends on x)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


@pytest.mark.parametrize("n,groups,classes,h,w", [(70001, 0, 32768, 0, 0), (35000003, 0, 64, 0, 0), (2200001, 0, 1000, 0, 0), (9, 4, 64, 1024, 1024)])
def test_past_two_to_the_31_logits(n, groups, classes, h, w):
    """The last sites of a tensor of more than 2^31 logits are those of the last sites alone."""
    from deepvideocodec_amd import ops
    rows = groups == 0
    g = torch.Generator(device="cuda").manual_seed(17)
    x = torch.empty((n, classes) if rows else (n, groups * classes, h, w), dtype=torch.bfloat16, device="cuda").uniform_(-3, 3, generator=g)
    assert x.numel() > 1 << 31
    sym = torch.randint(0, classes, (n,) if rows else (n, groups, h, w), generator=g, dtype=torch.int32, device="cuda")
    gl = torch.empty(sym.shape, device="cuda").uniform_(-1, 1, generator=g)
    r = ops.symbol_log_probs(x, sym, 2)
    got = ops.symbol_log_probs_backward(x, sym, r.stats, r.entropy, gl, gl)
    last = lambda t: (t[-40:] if rows else t[-1:, :, -2:]).cpu()
    given, ent, tl, ts, lp, p = definition(last(x), last(sym), 2)
    tol = step(classes, lp)
    same(last(r.log_prob), given, tol)
    same(last(r.entropy), ent, tol * (2 + ent))
    assert torch.equal(last(r.top_symbol), ts)
    site = lambda t: last(t).double().view(lp.size(0), lp.size(1), 1, *lp.shape[3:])
    a, en = site(gl), ent.view(lp.size(0), lp.size(1), 1, *lp.shape[3:])
    want = -p * (a + a * (lp + en)) + a * (torch.arange(classes).view(1, 1, -1, 1, 1) == site(sym))
    bound = tol * a.abs() * (3 + 2 * en) + want.abs() * 2.0 ** -8 + torch.finfo(torch.bfloat16).smallest_normal
    same(last(got), want.view(last(x).shape), bound.expand(want.shape).reshape(last(x).shape))


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_in_long_rows(dtype):
    """Of tens of thousands of equally good classes the lowest, over all parts of a row."""
    from deepvideocodec_amd import ops
    x = torch.randint(0, 3, (9, 70000), generator=torch.Generator().manual_seed(13)).float()
    want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :16].to(torch.int32)
    r = ops.symbol_log_probs(x.to(dtype).cuda(), torch.zeros(9, dtype=torch.int32).cuda(), 16)
    assert torch.equal(r.top_symbol.cpu(), want)


def test_two_streams_at_once():
    """The same calls on two streams side by side: workspaces are each call's own."""
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(12)
    xs = [torch.randn(3, 60000, generator=g).cuda() for _ in range(2)]
    s = torch.randint(0, 60000, (3,), generator=g, dtype=torch.int32).cuda()
    acts = [ops.act_checkpoint(torch.randn(4, 64, 64, 64, generator=g).cuda()) for _ in range(2)]
    grads = [torch.randn(4, 64, 64, 64, generator=g).cuda() for _ in range(2)]
    work = lambda i: [*ops.symbol_log_probs(xs[i], s, 8), *ops.conv2d_wgrad_ckpt(acts[i], grads[i], (64, 64, 3, 3), with_bias=True)]
    want = [[t.clone() for t in work(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            for a, b in zip(out, want[i]):
                assert torch.equal(a, b)


def test_symbols_outside_the_classes():
    from deepvideocodec_amd import autograd as A, ops
    x = torch.randn(4, 10, generator=torch.Generator().manual_seed(0)).cuda().requires_grad_()
    sym = torch.tensor([-1, -2 ** 31, 10, 2 ** 31 - 1], dtype=torch.int32).cuda()
    r = ops.symbol_log_probs(x.detach(), sym)
    assert r.log_prob[:2].tolist() == [0.0, 0.0] and bool(r.log_prob[2:].isnan().all()) and bool(torch.isfinite(r.entropy).all())
    lp = A.symbol_log_probs(x, sym)[0]
    (g,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert bool((g[:2] == 0).all()) and bool(g[2:].isnan().all())


def test_ties_go_to_the_lowest_class():
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(2)
    for v in (70, 700, 7000):
        x = torch.randint(0, 3, (9, v), generator=g).float()
        want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :16].to(torch.int32)
        for dtype in TYPES:
            r = ops.symbol_log_probs(x.to(dtype).cuda(), torch.zeros(9, dtype=torch.int32).cuda(), 16)
            assert torch.equal(r.top_symbol.cpu(), want)
        planes = x.t().reshape(1, v, 3, 3).contiguous()
        r = ops.symbol_log_probs(planes.cuda(), torch.zeros(1, 1, 3, 3, dtype=torch.int32).cuda(), 16)
        assert torch.equal(r.top_symbol.view(16, 9).t().cpu(), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_are_read_in_place(dtype):
    from deepvideocodec_amd import autograd as A, ops
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(12, 203, generator=g).to(dtype).cuda()
    sym = torch.randint(0, 100, (6,), generator=g, dtype=torch.int32).cuda()
    big = torch.randn(4, 30, 5, 7, generator=g).to(dtype).cuda()
    s4 = torch.randint(0, 5, (2, 3, 5, 7), generator=g, dtype=torch.int32).cuda()
    views = [(wide[:6, :100], sym), (wide[::2, 1:102], sym), (wide[6:, 103:], sym), (wide.t()[3:103, :6].t(), sym), (wide[:1, :100].expand(6, 100), sym),
             (big[:2, 3:18], s4), (big[::2, ::2], s4), (big[1:3, 10:25], s4)]
    for x, s in views:
        a, b = ops.symbol_log_probs(x, s, 3), ops.symbol_log_probs(x.contiguous(), s, 3)
        tol = step(x.size(1), a.log_prob.cpu())
        for k in (0, 1, 3):
            assert float((a[k] - b[k]).abs().max()) <= 2 * tol
        assert torch.equal(a.top_symbol, b.top_symbol)
        y = x.detach().clone(memory_format=torch.preserve_format).requires_grad_()
        gl = torch.randn(s.shape, generator=g).cuda()
        got = ops.symbol_log_probs_backward(x, s, a.stats, a.entropy, gl, gl)
        o = A.symbol_log_probs(y, s)
        (want,) = torch.autograd.grad((o[0], o[1]), y, (gl, gl))
        assert float((got.float() - want.float()).abs().max()) <= 8 * tol * float(gl.abs().max()) * 8 + 2 * torch.finfo(dtype).eps * float(want.abs().max())


def test_no_sites():
    from deepvideocodec_amd import autograd as A, ops
    x = torch.empty(0, 7, device="cuda", requires_grad=True)
    s = torch.empty(0, dtype=torch.int32, device="cuda")
    r = ops.symbol_log_probs(x.detach(), s, 2)
    assert r.log_prob.shape == (0,) and r.top_symbol.shape == (0, 2)
    (g,) = torch.autograd.grad(A.symbol_log_probs(x, s)[0].sum(), x)
    assert g.shape == (0, 7)


def test_large_logits_keep_their_differences():
    """A common offset of 2^13 leaves the probabilities as they are where the logits are exact there."""
    from deepvideocodec_amd import autograd as A
    g = torch.Generator().manual_seed(6)
    base = torch.randint(-64, 64, (5, 300), generator=g).float() / 16
    sym = torch.randint(0, 300, (5,), generator=g, dtype=torch.int32).cuda()
    outs = []
    for off in (0.0, 8192.0):
        x = (base + off).cuda().requires_grad_()
        o = A.symbol_log_probs(x, sym)
        outs.append((o[0].detach(), o[1].detach(), torch.autograd.grad((o[0], o[1]), x, (torch.ones_like(o[0]),) * 2)[0]))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_refusals():
    from deepvideocodec_amd import ops
    x = torch.randn(3, 12, 4, 4, device="cuda")
    s = torch.zeros(3, 4, 4, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="match"):
        ops.symbol_log_probs(x, s[:2].contiguous())
    with pytest.raises(ValueError, match="match"):
        ops.symbol_log_probs(x, torch.zeros(3, 5, 4, 4, dtype=torch.int32, device="cuda"))
    with pytest.raises(TypeError, match="int32"):
        ops.symbol_log_probs(x, s.long())
    with pytest.raises(TypeError, match="fp32"):
        ops.symbol_log_probs(x.double(), s)
    with pytest.raises(ValueError, match="top"):
        ops.symbol_log_probs(x, s, 4)
    with pytest.raises(ValueError, match="top"):
        ops.symbol_log_probs(x, s, -1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.symbol_log_probs(x.transpose(2, 3), s)
    with pytest.raises(ValueError, match="contiguous"):
        ops.symbol_log_probs(x, s.transpose(2, 3))
    with pytest.raises(ValueError):
        ops.symbol_log_probs(x, s[:, 0])
    with pytest.raises(ValueError):
        ops.symbol_log_probs(x[0], s[0])
    r = ops.symbol_log_probs(x, s)
    with pytest.raises(ValueError, match="elements"):
        ops.symbol_log_probs_backward(x, s, r.stats[:1].contiguous(), r.entropy, r.entropy, None)
    with pytest.raises(TypeError):
        ops.symbol_log_probs_backward(x, s, r.stats, r.entropy, r.entropy.half(), None)


def test_side_stream_and_replayed_graph():
    from deepvideocodec_amd import ops
    g = torch.Generator().manual_seed(8)
    rows, s1 = torch.randn(5, 9001, generator=g).cuda(), torch.randint(0, 9001, (5,), generator=g, dtype=torch.int32).cuda()
    planes, s2 = torch.randn(2, 60, 8, 9, generator=g).cuda(), torch.randint(0, 20, (2, 3, 8, 9), generator=g, dtype=torch.int32).cuda()

    def passes():
        out = []
        for x, s in ((rows, s1), (planes, s2)):
            r = ops.symbol_log_probs(x, s, 4)
            out += [*r, ops.symbol_log_probs_backward(x, s, r.stats, r.entropy, r.log_prob, r.entropy)]
        return out

    want = [t.clone() for t in passes()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = passes()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes()
    for _ in range(4):
        rows.copy_(torch.randn(rows.shape, generator=g))
        planes.copy_(torch.randn(planes.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, passes()):
            assert torch.equal(a, b)


def test_forward_and_backward_in_a_replayed_graph():
    """The autograd form as a whole under capture, of a leaf that no eager graph holds."""
    from deepvideocodec_amd import autograd as A
    g = torch.Generator().manual_seed(14)
    sym = torch.randint(-1, 50, (3, 2, 4, 5), generator=g, dtype=torch.int32).cuda()
    gl, gh = (torch.randn(sym.shape, generator=g).cuda() for _ in range(2))

    def passes(x):
        r = A.symbol_log_probs(x, sym)
        (grad,) = torch.autograd.grad((r[0], r[1]), x, (gl, gh))
        return r[0].detach(), r[1].detach(), grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(torch.randn(3, 100, 4, 5, generator=g).cuda().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    leaf = torch.zeros(3, 100, 4, 5).cuda().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = passes(leaf)
    for _ in range(4):
        fresh = torch.randn(leaf.shape, generator=g).cuda()
        with torch.no_grad():
            leaf.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, passes(fresh.requires_grad_())):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_categorical_rate_behind_checkpointed_layers(fmt):
    """As used together: a stack of convolutions whose tape is 8-bit, logits for a small alphabet, bits as the loss.
    Gradients against 64 bits: the loss's own through the same (fp32) activations, each weight's from its stored operand."""
    import math
    import torch.nn.functional as F
    from deepvideocodec_amd import autograd as A, ops
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(2, 12, 16, 20, generator=gen)
    w1, b1 = torch.randn(24, 12, 3, 3, generator=gen) / 10, torch.randn(24, generator=gen)
    w2, b2 = torch.randn(3 * 9, 24, 1, 1, generator=gen) / 5, torch.randn(27, generator=gen)
    sym = torch.randint(0, 9, (2, 3, 16, 20), generator=gen, dtype=torch.int32)
    dev = [t.cuda().requires_grad_() for t in (x, w1, b1, w2, b2)]
    t = A.conv2d(dev[0], dev[1], dev[2], out_slope=0.01, storage=fmt)
    logits = A.conv2d(t, dev[3], dev[4], storage=fmt)
    lp, ent = A.symbol_log_probs(logits, sym.cuda())[:2]
    (-lp.sum() / math.log(2)).backward()
    # the same in 64 bits, the weight gradients' operands replaced by the stored ones
    ref = [q.double().requires_grad_() for q in (x, w1, b1, w2, b2)]
    t64 = F.leaky_relu(F.conv2d(ref[0], ref[1], ref[2], padding=1), 0.01)
    l64 = F.conv2d(t64, ref[3], ref[4])
    lp64 = F.log_softmax(l64.view(2, 3, 9, 16, 20), 2).gather(2, sym.long()[:, :, None])[:, :, 0]
    loss = -lp64.sum() / math.log(2)
    gx, gb1, gb2, gl, gt = torch.autograd.grad(loss, [ref[0], ref[2], ref[4], l64, t64])
    tq = ops.act_restore(ops.act_checkpoint(t.detach(), fmt=fmt)).cpu().double()
    xq = ops.act_restore(ops.act_checkpoint(x.cuda(), fmt=fmt)).cpu().double()
    g1 = gt * torch.where(t64 > 0, 1.0, 0.01)
    gw2 = torch.einsum("nohw,nihw->oi", gl, tq).view(27, 24, 1, 1)
    xp = F.pad(xq, (1, 1, 1, 1))
    gw1 = torch.stack([torch.stack([torch.einsum("nohw,nihw->oi", g1, xp[:, :, a:a + 16, b:b + 20]) for b in range(3)], -1) for a in range(3)], -2)
    # fp32 forward sums of at most 108 terms, a softmax, sums over 640 pixels: relative to the largest entry well below
    # (108 + 640 + 128) 2^-23 = 1.05e-4
    for got, want in ((dev[0].grad, gx), (dev[1].grad, gw1), (dev[2].grad, gb1), (dev[3].grad, gw2), (dev[4].grad, gb2)):
        assert float((got.cpu().double() - want).abs().max()) <= 1.1e-4 * float(want.abs().max())


@pytest.mark.parametrize("place,site", [((1, (1 << 32) + 5), (1,)), ((1, 1 << 31), (1,)), ((1, (1 << 32) + 6, 1, 1), (1, 2, 1, 1))])
def test_sizes_past_32_bits_are_refused(place, site):
    """A size of 2^31 or more does not fit the library's arguments: refused, not wrapped."""
    from deepvideocodec_amd import autograd as A, ops
    x, s = torch.zeros(place, dtype=torch.bfloat16, device="cuda"), torch.zeros(site, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        ops.symbol_log_probs(x, s)
    with pytest.raises(ValueError, match="2\\^31"):
        A.symbol_log_probs(x.requires_grad_(), s)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.symbol_log_probs_backward(x.detach(), s, torch.zeros((2, s.numel()), device="cuda"), torch.zeros(s.numel(), device="cuda"), None, None)
