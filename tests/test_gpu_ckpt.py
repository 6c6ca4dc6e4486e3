"""8-bit activation checkpoints against the format's definition in 64 bits: codes and scales bit for bit, restored
values, the sign-only adjoints, and weight gradients from checkpoints."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

FORMATS = ("int8", "e4m3")


def encode64(x, fmt):
    """codes, scales of a CPU tensor, from the definition, in float64."""
    n, c, h, w = x.shape
    v = F.pad(x.double().reshape(n, c, h * w), (0, -(h * w) % 32)).view(n, c, -1, 32)
    fine = torch.isfinite(v).all(-1, keepdim=True)
    v0 = torch.where(fine, v, 0.0)
    largest = 127.0 if fmt == "int8" else 448.0
    amax = v0.abs().amax(-1, keepdim=True)
    mant, expo = torch.frexp(amax / largest)                     # the smallest e with amax <= largest 2^e
    e = torch.where(amax == 0, -110, torch.where(mant == 0.5, expo - 1, expo)).clamp(min=-110)
    # amax / largest may round onto a power of two from above: settle it by an exact comparison
    e = torch.where(amax > largest * torch.exp2(e.double()), e + 1, e)
    y = v0.abs().clamp(max=63 * 2.0 ** 122 if fmt == "int8" else 240 * 2.0 ** 120) / torch.exp2(e.double())    # restores below 2^128
    if fmt == "int8":
        mag = torch.round(y)
    else:
        b = torch.floor(torch.log2(y.clamp(min=2.0 ** -30))).clamp(min=-6)
        b = torch.where(torch.exp2(b) > y, (b - 1).clamp(min=-6), b)
        q = torch.round(y / torch.exp2(b - 3))                   # in eighths of the binade (subnormals: of 2^-6)
        mag = torch.where(b == -6, q, (b + 7) * 8 + q - 8)       # q = 16 carries into the next binade by itself
    codes = torch.where(fine, mag, 0.0).to(torch.uint8) + (~(v > 0)).to(torch.uint8) * 128
    scales = torch.where(fine, e + 127, 255).to(torch.uint8)
    return codes.view(n, c, -1), scales.view(n, c, -1), fine


def values64(codes, scales, fmt, shape):
    n, c, h, w = shape
    k = torch.arange(128, dtype=torch.float64)
    mag = k if fmt == "int8" else torch.where(k < 8, k * 2.0 ** -9, (8 + k % 8) * torch.exp2(torch.floor(k / 8) - 10))
    table = torch.cat((mag, -mag))
    s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    v = table[codes.long()].view(n, c, -1, 32) * s[..., None]
    return v.reshape(n, c, -1)[:, :, :h * w].reshape(shape)


def leaky32(x, slope):
    return x if slope is None else torch.where(x > 0, x, x * torch.tensor(slope, dtype=torch.float32))


def sample(shape, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(6 * torch.randn(shape[:2], generator=g))[..., None, None]
    x[torch.rand(shape, generator=g) < 0.2] = 0.0                     # as behind a ReLU
    x[torch.rand(shape, generator=g) < 0.02] *= 2.0 ** -20            # far below their block's largest
    return x


SHAPES = [(1, 1, 1, 1), (1, 3, 1, 31), (2, 2, 4, 8), (1, 2, 3, 11), (2, 5, 16, 16), (1, 3, 7, 129), (3, 35, 20, 24), (1, 70, 33, 65)]


@pytest.mark.parametrize("slope", [None, 0.0, 0.1, 1.0])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_codes_and_scales_are_those_of_the_definition(shape, fmt, slope):
    from deepvideocodec_amd import ops
    x = sample(shape, sum(shape))
    ck = ops.act_checkpoint(x.cuda(), slope=slope, fmt=fmt)
    codes, scales, _ = encode64(leaky32(x, slope), fmt)
    assert ck.shape == shape and ck.fmt == fmt
    assert torch.equal(ck.scales.cpu(), scales)
    assert torch.equal(ck.codes.cpu(), codes)
    back = ops.act_restore(ck).cpu()
    assert torch.equal(back.double(), values64(codes, scales, fmt, shape))    # a code times a power of two is exact
    assert torch.equal(torch.signbit(back), ~(x > 0)) or slope == 0.0


@pytest.mark.parametrize("fmt", FORMATS)
def test_ranges_borders_and_ties(fmt):
    from deepvideocodec_amd import ops
    largest = 127.0 if fmt == "int8" else 448.0
    up = lambda v: math.ldexp(math.frexp(v)[0] + 2.0 ** -24, math.frexp(v)[1])     # the next fp32 number
    blocks = []
    for e in (-100, -3, 0, 5, 100):
        blocks += [[largest * 2.0 ** e], [up(largest) * 2.0 ** e], [2.0 ** e], [1.5 * 2.0 ** e, -2.0 ** (e - 30)]]
    # ties: halves of a step
    blocks += [[largest] + [k + 0.5 for k in range(0, 30)], [-largest] + [-(k + 0.5) for k in range(60, 90)],
               [largest] + [(8 + j + 0.5) * 2.0 ** s for j in range(8) for s in (-9, -5, 4)], [largest] + [(j + 0.5) * 2.0 ** -9 for j in range(9)]]
    # smallest and largest numbers
    blocks += [[2.0 ** -110], [2.0 ** -111, 2.0 ** -103], [1e-45], [2.0 ** -126, -1e-40], [3.4028234e38], [-3.4028234e38, 1.0], [0.0, -0.0]]
    x = torch.zeros(len(blocks), 32)
    for i, b in enumerate(blocks):
        x[i, :len(b)] = torch.tensor(b)
    x = x.view(1, len(blocks), 4, 8)
    ck = ops.act_checkpoint(x.cuda(), fmt=fmt)
    codes, scales, _ = encode64(x, fmt)
    assert torch.equal(ck.scales.cpu(), scales)
    assert torch.equal(ck.codes.cpu(), codes)
    v = ops.act_restore(ck).cpu()
    assert torch.equal(v.double(), values64(codes, scales, fmt, x.shape))
    # half a step of the block's scale (int8) or of the value (e4m3: 2^-4, subnormals half of 2^-9 scale steps)
    step = torch.exp2(scales.double() - 127).view(1, -1, 1, 1)
    bound = step / 2 if fmt == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)
    bound = torch.where(x.double().abs() > 1.875 * 2.0 ** 127, 2 * bound, bound)      # (rounded down, not to 2^128)
    assert bool(((v.double() - x.double()).abs() <= bound).all())


def test_int8_codes_of_the_topmost_binades():
    """The nearest of the scale's steps, and the one below only where that would restore to 2^128: 64 steps of 2^122, but none
    of the 127 steps of 2^121."""
    from deepvideocodec_amd import ops
    t = 2.0 ** 121
    blocks = [[127 * t], [126.75 * t, 126.5 * t, 126.25 * t, 125.5 * t], [-126.75 * t, 1.0], [127 * t, -126.5 * t, 63.5 * t],
              [127 * t + 2.0 ** 104, 126.5 * t, -127 * t, 126.984375 * t], [3.4028234e38, 126 * t, 125 * t, 127 * t], [127.5 * t, 3 * t]]
    x = torch.zeros(len(blocks), 32)
    for i, b in enumerate(blocks):
        x[i, :len(b)] = torch.tensor(b, dtype=torch.float64).float()
    v, a = x.double(), x.double().abs()
    e = torch.where(a.amax(1, keepdim=True) <= 127 * t, 121, 122)
    mag = torch.round(a / torch.exp2(e.double()))
    mag = torch.where(mag * torch.exp2(e.double()) >= 2.0 ** 128, mag - 1, mag)
    ck = ops.act_checkpoint(x.view(1, len(blocks), 4, 8).cuda(), fmt="int8")
    assert torch.equal(ck.scales.cpu().view(-1, 1), (e + 127).to(torch.uint8))
    assert torch.equal(ck.codes.cpu().view(-1, 32), mag.to(torch.uint8) + (~(v > 0)).to(torch.uint8) * 128)
    assert torch.equal(ops.act_restore(ck).cpu().double().view(-1, 32), torch.where(v > 0, 1.0, -1.0) * mag * torch.exp2(e.double()))


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_block_that_is_not_finite_restores_to_nan_and_keeps_to_itself(fmt):
    from deepvideocodec_amd import ops
    x = torch.randn(1, 3, 4, 32, generator=torch.Generator().manual_seed(0))
    for row, bad in enumerate((float("inf"), float("-inf"), float("nan"))):
        x[0, 1, row, 5 * row + 1] = bad
    v = ops.act_restore(ops.act_checkpoint(x.cuda(), fmt=fmt)).cpu()
    assert bool(v[0, 1, :3].isnan().all())
    assert bool(torch.isfinite(v[0, 1, 3]).all()) and bool(torch.isfinite(v[0, 0]).all()) and bool(torch.isfinite(v[0, 2]).all())


@pytest.mark.parametrize("fmt", FORMATS)
def test_views_and_unaligned_sources(fmt):
    """Channel slices, strided batches and planes off 16 bytes are read in place; restoring writes nothing else."""
    from deepvideocodec_amd import ops
    base = sample((3, 8, 6, 10), 7).cuda()
    for view in (base[:, 2:5], base[::2], base[1:2, 3:4], base[:, 1::3], base.view(3, 8, 60, 1)[:, :, 3:43].reshape(3, 8, 40, 1)[:, 1:4]):
        ck = ops.act_checkpoint(view, fmt=fmt)
        codes, scales, _ = encode64(view.cpu(), fmt)
        assert torch.equal(ck.codes.cpu(), codes) and torch.equal(ck.scales.cpu(), scales)
        assert torch.equal(ops.act_signs(view).cpu(), signs64(view.cpu()))
    flat = torch.zeros(4 * 63 + 1, device="cuda")
    odd = flat[1:].view(1, 4, 7, 9)                                    # 4 bytes past an aligned address
    odd.copy_(sample((1, 4, 7, 9), 8))
    assert torch.equal(ops.act_checkpoint(odd, fmt=fmt).codes.cpu(), encode64(odd.cpu(), fmt)[0])
    target = torch.full((3, 8, 6, 10), 5.0, device="cuda")
    ck = ops.act_checkpoint(base[:, 2:5], fmt=fmt)
    ops.act_restore(ck, out=target[:, 4:7])
    assert torch.equal(target[:, 4:7], ops.act_restore(ck))
    assert bool((target[:, :4] == 5).all()) and bool((target[:, 7:] == 5).all())


def signs64(x):
    n, c, h, w = x.shape
    v = F.pad((x > 0).reshape(n, c, h * w), (0, -(h * w) % 32)).view(n, c, -1, 32).long()
    return (v << torch.arange(32)).sum(-1).to(torch.int32)


@pytest.mark.parametrize("shape", SHAPES)
def test_sign_only_adjoints_equal_the_fp32_ones(shape):
    from deepvideocodec_amd import ops
    x = sample(shape, 3 + sum(shape)).cuda()
    g = torch.Generator().manual_seed(1)
    grad, plus = (torch.randn(shape, generator=g).cuda() for _ in range(2))
    signs = ops.act_signs(x)
    assert torch.equal(signs.cpu(), signs64(x.cpu()))
    for slope in (0.0, 0.01, 0.2):
        assert torch.equal(ops.act_grad_signs(grad, signs, slope, False, shape), ops.act_grad(grad, x, slope, False, shape))
        for fmt in FORMATS:
            ck = ops.act_checkpoint(x, slope=slope, fmt=fmt)
            assert torch.equal(ops.mul_act_grad_ckpt(grad, ck, slope), ops.mul_act_grad(grad, x, slope))
            assert torch.equal(ops.mul_act_grad_ckpt(grad, ck, slope, plus=plus), ops.mul_act_grad(grad, x, slope, plus=plus))
            into = grad.clone()
            ops.mul_act_grad_ckpt(into, ck, slope, out=into)            # in place
            assert torch.equal(into, ops.mul_act_grad(grad, x, slope))


@pytest.mark.parametrize("n,c,h,w", [(1, 4, 1, 1), (2, 8, 5, 7), (1, 12, 8, 16)])
def test_sign_only_adjoint_behind_a_pixel_shuffle(n, c, h, w):
    from deepvideocodec_amd import ops
    out = sample((n, c // 4, 2 * h, 2 * w), 5).cuda()
    grad = torch.randn(out.shape, generator=torch.Generator().manual_seed(2)).cuda()
    assert torch.equal(ops.act_grad_signs(grad, ops.act_signs(out), 0.1, True, (n, c, h, w)), ops.act_grad(grad, out, 0.1, True, (n, c, h, w)))


# ---------------------------------------------------------------------------------------- weight gradients
def wgrad64(x, g, k, stride):
    """(gw, gb) of float64 CPU tensors, tap by tap."""
    n, cout, ho, wo = g.shape
    p = k // 2
    xp = F.pad(x, (p, p, p, p))
    gw = torch.stack([torch.stack([torch.einsum("nopq,nipq->oi", g, xp[:, :, ky:ky + (ho - 1) * stride + 1:stride, kx:kx + (wo - 1) * stride + 1:stride])
                                   for kx in range(k)], -1) for ky in range(k)], -2)
    return gw, g.sum((0, 2, 3))


WGRAD = [
    # k, stride, cins, cout, h, w, batch
    (3, 1, (64,), 64, 36, 52, 2),
    (3, 1, (16, 8), 40, 17, 23, 1),
    (3, 1, (5, 7, 9, 11), 33, 21, 19, 2),
    (3, 1, (96,), 128, 12, 20, 1),
    (3, 1, (130,), 70, 8, 40, 1),
    (3, 1, (48,), 48, 16, 16, 3),
    (3, 1, (64,), 3, 9, 37, 1),
    (3, 1, (3,), 64, 20, 28, 1),
    (3, 1, (1,), 1, 1, 1, 1),
    (3, 1, (2,), 5, 1, 67, 2),
    (3, 1, (2,), 5, 67, 1, 2),
    (3, 1, (33,), 31, 70, 66, 1),
    (3, 1, (32, 32), 40, 12, 36, 2),         # a staging wave's channels in one source each ...
    (3, 1, (24, 40), 33, 12, 36, 2),         # ... and across two
    (3, 1, (33,), 64, 200, 12, 1),
    (3, 2, (67,), 64, 32, 48, 1),
    (3, 2, (16,), 24, 25, 31, 2),
    (3, 2, (4,), 6, 1, 2, 1),
    (3, 2, (40,), 72, 64, 130, 1),
    (7, 1, (8,), 32, 30, 50, 1),
    (7, 1, (16,), 2, 20, 37, 2),
    (7, 1, (32,), 64, 19, 70, 2),
    (7, 1, (40, 24), 16, 9, 33, 1),
    (7, 1, (3,), 33, 2, 3, 1),
    (1, 1, (64,), 32, 33, 47, 1),
    (1, 1, (7, 70), 65, 1, 5, 3),
    (1, 2, (12,), 64, 34, 50, 2),
    (1, 2, (33,), 34, 7, 9, 1),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,stride,cins,cout,h,w,batch", WGRAD)
def test_weight_gradient_of_whole_numbers_is_exact(k, stride, cins, cout, h, w, batch, fmt):
    """Whole numbers that both formats hold, small enough that every partial sum is below 2^24: no rounding happens
    anywhere, so every layout, padding or ragged edge that is wrong by one element shows."""
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(k + cout + h + w)
    # 15 steps of a block's scale: exact in both formats, whatever the block's largest value is
    xs = [torch.randint(-15, 16, (batch, c, h, w), generator=gen).float() for c in cins]
    p = k // 2
    ho, wo = (h + 2 * p - k) // stride + 1, (w + 2 * p - k) // stride + 1
    g = torch.randint(-8, 9, (batch, cout, ho, wo), generator=gen).float()
    assert batch * ho * wo * 15 * 8 < 1 << 24
    cks = [ops.act_checkpoint(x.cuda(), fmt=fmt) for x in xs]
    for x, ck in zip(xs, cks):
        assert torch.equal(ops.act_restore(ck).cpu(), x)
    gw, gb = ops.conv2d_wgrad_ckpt(cks, g.cuda(), (cout, sum(cins), k, k), stride, with_bias=True)
    want_w, want_b = wgrad64(torch.cat(xs, 1).double(), g.double(), k, stride)
    assert torch.equal(gw.cpu().double(), want_w)
    assert torch.equal(gb.cpu().double(), want_b)
    alone = ops.conv2d_wgrad_ckpt(cks, g.cuda(), (cout, sum(cins), k, k), stride)
    assert torch.equal(alone, gw)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,stride,cins,cout,h,w,batch", WGRAD)
def test_weight_gradient_of_real_numbers(k, stride, cins, cout, h, w, batch, fmt):
    """Against 64 bits with the stored operands.  Products are exact; n terms, each in three parts, are added in fp32, so
    a sum is off by at most 3 n 2^-24 of the sum of magnitudes (any order of addition)."""
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(3 * k + cout + h + w)
    xs = [sample((batch, c, h, w), 11 + c) for c in cins]
    p = k // 2
    ho, wo = (h + 2 * p - k) // stride + 1, (w + 2 * p - k) // stride + 1
    g = torch.randn(batch, cout, ho, wo, generator=gen) * torch.exp2(4 * torch.randn(1, cout, 1, 1, generator=gen) - 10)
    cks = [ops.act_checkpoint(x.cuda(), slope=0.1, fmt=fmt) for x in xs]
    x64 = torch.cat([values64(ck.codes.cpu(), ck.scales.cpu(), fmt, ck.shape) for ck in cks], 1)
    gw, gb = ops.conv2d_wgrad_ckpt(cks, g.cuda(), (cout, sum(cins), k, k), stride, with_bias=True)
    want_w, want_b = wgrad64(x64, g.double(), k, stride)
    most_w, most_b = wgrad64(x64.abs(), g.double().abs(), k, stride)
    n = batch * ho * wo
    assert bool(((gw.cpu().double() - want_w).abs() <= 3 * n * 2.0 ** -24 * most_w).all())
    assert bool(((gb.cpu().double() - want_b).abs() <= n * 2.0 ** -24 * most_b).all())
    again = ops.conv2d_wgrad_ckpt(cks, g.cuda(), (cout, sum(cins), k, k), stride, with_bias=True)
    assert torch.equal(again[0], gw) and torch.equal(again[1], gb)       # a fixed order of addition


@pytest.mark.parametrize("k,stride,cin,cout,h,w,batch", [
    (3, 1, 64, 64, 164, 256, 25),      # 8200 tiles over 256 workgroups: 33 for some (two slabs in time), 32 for most (one, and zeros)
    (3, 1, 64, 33, 100, 260, 24),      # 56 or 57 tiles each on odd tile counts
    (3, 1, 576, 576, 40, 160, 1),      # 81 blocks: four workgroups of 12 or 13 tiles each
    (1, 1, 1024, 1024, 68, 92, 1),     # one workgroup per block: all 51 tiles
    (7, 1, 32, 256, 132, 164, 2),      # 8 blocks, 12 or 13 tiles
    (3, 2, 256, 512, 130, 132, 2),
])
def test_weight_gradient_of_long_sums(k, stride, cin, cout, h, w, batch):
    """Many tiles per workgroup, several slabs in time, workgroups with one tile fewer than others: whole numbers, exact."""
    from deepvideocodec_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(k + cin)
    x = torch.randint(-1, 2, (batch, cin, h, w), generator=gen, device="cuda").float()
    p = k // 2
    ho, wo = (h + 2 * p - k) // stride + 1, (w + 2 * p - k) // stride + 1
    g = torch.randint(-1, 2, (batch, cout, ho, wo), generator=gen, device="cuda").float()
    assert batch * ho * wo < 1 << 24
    gw, gb = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x), g, (cout, cin, k, k), stride, with_bias=True)
    xp = F.pad(x, (p, p, p, p))
    rows = g.double().transpose(0, 1).reshape(cout, -1)
    for ky in range(k):
        for kx in range(k):
            cols = xp[:, :, ky:ky + (ho - 1) * stride + 1:stride, kx:kx + (wo - 1) * stride + 1:stride].double().transpose(0, 1).reshape(cin, -1)
            assert torch.equal(gw[:, :, ky, kx].double(), rows @ cols.t().contiguous()), (ky, kx)
    assert torch.equal(gb.double(), rows.sum(1))


def wgrad64_gpu(x, g, k, stride):
    """The same of fp32 GPU tensors, in float64, sample by sample."""
    n, cout, ho, wo = g.shape
    cin, p = x.size(1), k // 2
    gw = torch.zeros(cout, cin, k, k, dtype=torch.float64, device=x.device)
    for i in range(n):
        xp = F.pad(x[i], (p, p, p, p)).double()
        rows = g[i].double().reshape(cout, -1)
        for ky in range(k):
            for kx in range(k):
                cols = xp[:, ky:ky + (ho - 1) * stride + 1:stride, kx:kx + (wo - 1) * stride + 1:stride].reshape(cin, -1)
                gw[:, :, ky, kx] += rows @ cols.t().contiguous()
    return gw


@pytest.mark.parametrize("k,cin,cout,h,w,batch", [
    (3, 192, 192, 256, 256, 6),      # 106 tiles for each of 29 workgroups a block: four slabs in time, two launches of two
    (3, 192, 160, 256, 253, 7),      # five: of three and two
    (7, 64, 64, 42, 4740, 5),        # 8195 tiles over 64 workgroups: three slabs, in the second launch three tiles
    (7, 64, 64, 42, 4739, 5),
])
def test_weight_gradient_over_several_launches(k, cin, cout, h, w, batch):
    """Where the slabs would need more than 128 MiB, several launches add to the result: whole numbers, exact; a fixed order;
    also into memory that held something else, and in a replayed graph."""
    from deepvideocodec_amd import _lib, ops
    gen = torch.Generator(device="cuda").manual_seed(k + cin)
    x = torch.randint(-1, 2, (batch, cin, h, w), generator=gen, device="cuda").float()
    g = torch.randint(-1, 2, (batch, cout, h, w), generator=gen, device="cuda").float()
    assert batch * h * w < 1 << 24 and 4 * _lib.load().dvc_conv2d_wgrad_ckpt_scratch_floats(cout, cin, k, 1, batch, h, w) < 129 << 20
    ck = ops.act_checkpoint(x)
    want = wgrad64_gpu(x, g, k, 1)
    for _ in range(2):
        gw, gb = ops.conv2d_wgrad_ckpt(ck, g, (cout, cin, k, k), with_bias=True)
        assert torch.equal(gw.double(), want) and torch.equal(gb.double(), g.double().sum((0, 2, 3)))
        del gw, gb                            # (the next call's results lie where these were)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw, gb = ops.conv2d_wgrad_ckpt(ck, g, (cout, cin, k, k), with_bias=True)
    for _ in range(3):
        gw.fill_(float("nan"))
        gb.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gw.double(), want) and torch.equal(gb.double(), g.double().sum((0, 2, 3)))


def real_sums(k, stride, cin, cout, h, w, batch, fmt):
    """-> error of a weight gradient of random real numbers, in units of the gradient's root mean square."""
    from deepvideocodec_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(34)
    ho, wo = (h + 2 * (k // 2) - k) // stride + 1, (w + 2 * (k // 2) - k) // stride + 1
    ck = ops.act_checkpoint(torch.empty(batch, cin, h, w, device="cuda").normal_(generator=gen), fmt=fmt)
    g = torch.empty(batch, cout, ho, wo, device="cuda").normal_(generator=gen)
    want = wgrad64_gpu(ops.act_restore(ck), g, k, stride)
    return (ops.conv2d_wgrad_ckpt(ck, g, (cout, cin, k, k), stride).double() - want) / want.square().mean().sqrt()


@pytest.mark.parametrize("k,stride,cin,cout,h,w,batch,fmt", [
    (3, 1, 64, 64, 256, 256, 16, "int8"), (3, 1, 64, 64, 256, 256, 32, "e4m3"),      # one slab in time, two
    (3, 1, 64, 64, 255, 253, 8, "int8"), (3, 1, 96, 33, 128, 128, 8, "e4m3"), (3, 1, 32, 32, 256, 256, 16, "int8"),
    (3, 1, 40, 24, 255, 129, 8, "e4m3"), (3, 1, 3, 64, 256, 256, 16, "int8"), (3, 1, 64, 3, 256, 256, 8, "int8"),
    (3, 1, 128, 128, 16, 16, 64, "e4m3"), (3, 2, 64, 64, 256, 256, 8, "int8"), (3, 2, 32, 64, 255, 257, 8, "e4m3"),
    (1, 1, 64, 64, 256, 256, 32, "int8"), (1, 1, 32, 48, 255, 255, 8, "e4m3"), (1, 2, 64, 64, 256, 256, 8, "int8"),
    (7, 1, 32, 64, 128, 128, 32, "e4m3"), (7, 1, 16, 2, 255, 253, 4, "int8"), (1, 1, 1024, 1024, 96, 128, 1, "int8"),
    (3, 1, 192, 192, 256, 256, 8, "e4m3")])
def test_weight_gradient_of_long_sums_of_real_numbers(k, stride, cin, cout, h, w, batch, fmt):
    """All three parts of the gradient arrive in every form and at every place of a tile.  A slab is at most 512 row pieces of
    three matrix instructions that round twice: n = 6 x 512 roundings of a sum that grows like a random walk, 2^-24 / sqrt(3)
    of its size each, come to sqrt(n / 2) 2^-24 / sqrt(3) = 1.4e-6 of the result.  Without the third part every gradient is
    cut off by 2^-17 (5.5e-6 on average, all towards zero); without the second by 2^-9."""
    assert float(real_sums(k, stride, cin, cout, h, w, batch, fmt).square().mean().sqrt()) <= 3e-6


@pytest.mark.parametrize("k,stride,cin,cout,h,w,batch", [(3, 1, 64, 64, 256, 256, 32), (1, 1, 1024, 1024, 128, 128, 4), (1, 1, 1024, 512, 128, 128, 4),
                                                         (7, 1, 512, 512, 64, 256, 2)])
def test_weight_gradient_does_not_drift(k, stride, cin, cout, h, w, batch):
    """The matrix instruction's cuts are all downwards; over an even number of slabs -- over workgroups (the first: 256 of them, two
    slabs each) or in time (one workgroup per block, 16 slabs) -- they cancel.  Without the alternating signs the mean error is
    2e-6 and 2.3e-7 of the results' size; what chance leaves of it is 7e-7 / sqrt(results), 4e-9 or less."""
    assert abs(float(real_sums(k, stride, cin, cout, h, w, batch, "int8").mean())) <= 2e-8


@pytest.mark.parametrize("k,cin,cout,h,w,batch,chain", [
    (1, 1024, 1024, 512, 512, 1, 32 + 32 + 2), (1, 1024, 1024, 511, 511, 1, 64 + 32 + 2), (7, 256, 256, 512, 512, 1, 64 + 2 + 4),
    (3, 64, 64, 256, 256, 32, 32 + 2 + 1), (3, 576, 576, 128, 128, 16, 32 + 2 + 8), (3, 20, 24, 255, 253, 64, 256 + 1 + 1)])
def test_bias_gradient_of_long_sums(k, cin, cout, h, w, batch, chain):
    """One gradient per channel throughout: the terms of a sum are equal, so that the roundings of a long sum do not cancel.  `chain`:
    the terms that a lane adds up between two slabs' ends, the slabs in time of a launch, the launches; besides, a lane adds
    four pixels (2), 64 lanes are joined (6), then at most 16 groups of 16 workgroups (4 + 4 + 16)."""
    from deepvideocodec_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(35)
    g = torch.rand(1, cout, 1, 1, device="cuda", generator=gen).expand(batch, cout, h, w).contiguous()
    ck = ops.act_checkpoint(torch.zeros(batch, cin, h, w, device="cuda"))
    gw, gb = ops.conv2d_wgrad_ckpt(ck, g, (cout, cin, k, k), with_bias=True)
    want = g[0, :, 0, 0].double() * (batch * h * w)
    assert bool(((gb - want).abs() <= (chain + 32) * 2.0 ** -24 * want).all()) and not bool(gw.any())


@pytest.mark.parametrize("e", [-60, -100, -118, 60, 100])
def test_weight_gradient_of_very_small_and_large_gradients(e):
    """A power of two on the gradient is one on the result, as long as nothing leaves the normal numbers."""
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(8)
    x = torch.randint(-15, 16, (1, 40, 12, 20), generator=gen).float()
    g = torch.randint(-8, 9, (1, 36, 12, 20), generator=gen).float()
    ck = ops.act_checkpoint(x.cuda())
    a = ops.conv2d_wgrad_ckpt(ck, g.cuda(), (36, 40, 3, 3))
    b = ops.conv2d_wgrad_ckpt(ck, (g * 2.0 ** e).cuda(), (36, 40, 3, 3))
    assert torch.equal(a.double() * 2.0 ** e, b.double())


def test_weight_gradient_keeps_all_bits_of_the_gradient():
    """One pixel: the result is a single product of a 24-bit gradient and a code, correctly rounded parts and all."""
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(5)
    x = torch.exp2(torch.randint(-3, 4, (1, 40, 1, 1), generator=gen).float())          # powers of two: exact products
    g = torch.randn(1, 50, 1, 1, generator=gen)
    gw = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x.cuda()), g.cuda(), (50, 40, 1, 1))
    assert torch.equal(gw.cpu(), g.view(50, 1, 1, 1) * x.view(1, 40, 1, 1))


@pytest.mark.parametrize("k", [1, 3, 7])
def test_what_is_not_finite_reaches_the_weights_it_takes_part_in(k):
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(6)
    x, g = torch.randn(1, 40, 20, 40, generator=gen), torch.randn(1, 36, 20, 40, generator=gen)
    x[0, 7, 10, 20] = float("inf")
    gw = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x.cuda()), g.cuda(), (36, 40, k, k)).cpu()
    assert bool(gw[:, 7].isnan().all()) and bool(torch.isfinite(gw[:, :7]).all()) and bool(torch.isfinite(gw[:, 8:]).all())
    x[0, 7, 10, 20] = 0.0
    for bad in (float("nan"), float("inf")):
        g[0, 5, 3, 4] = bad
        gw, gb = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x.cuda()), g.cuda(), (36, 40, k, k), with_bias=True)
        gw, gb = gw.cpu(), gb.cpu()
        assert not bool(torch.isfinite(gw[5]).any()) and not bool(torch.isfinite(gb[5]))
        assert bool(torch.isfinite(gw[:5]).all()) and bool(torch.isfinite(gw[6:]).all()) and bool(torch.isfinite(gb[6:]).all())


def test_refusals_of_the_python_surface():
    from deepvideocodec_amd import ops
    x = torch.randn(2, 4, 8, 8, device="cuda")
    ck = ops.act_checkpoint(x)
    with pytest.raises(ValueError, match="slope"):
        ops.act_checkpoint(x, slope=1.5)
    with pytest.raises(ValueError, match="slope"):
        ops.act_checkpoint(x, slope=-0.5)
    with pytest.raises(TypeError):
        ops.act_checkpoint(x.half())
    with pytest.raises(ValueError, match="contiguous"):
        ops.act_checkpoint(x.transpose(2, 3)[:, :, :, ::2])
    with pytest.raises(ValueError, match="elements"):
        ops.act_restore(ck._replace(codes=ck.codes[:1].contiguous()))
    with pytest.raises(ValueError, match="contiguous"):
        ops.act_restore(ck._replace(codes=ck.codes.transpose(0, 1)))
    with pytest.raises(ValueError, match="shape"):
        ops.act_restore(ck, out=torch.empty(2, 4, 8, 9, device="cuda"))
    g = torch.randn(2, 6, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="grad_pre"):
        ops.conv2d_wgrad_ckpt(ck, g, (6, 4, 3, 3), 2)
    with pytest.raises(ValueError, match="weight shape"):
        ops.conv2d_wgrad_ckpt(ck, g, (6, 5, 3, 3))
    with pytest.raises(ValueError, match="contiguous"):
        ops.conv2d_wgrad_ckpt(ck, g.transpose(2, 3), (6, 4, 3, 3))
    with pytest.raises(ValueError, match="match"):
        ops.conv2d_wgrad_ckpt((ck, ops.act_checkpoint(x, fmt="e4m3")), g, (6, 8, 3, 3))
    with pytest.raises(_lib_error(), match="ksize"):
        ops.conv2d_wgrad_ckpt(ck, g, (6, 4, 5, 5))
    with pytest.raises(ValueError, match="elements"):
        ops.act_grad_signs(g, ops.act_signs(x), 0.1, False, tuple(g.shape))
    with pytest.raises(ValueError, match="shape"):
        ops.mul_act_grad_ckpt(g, ck, 0.1)
    # destinations whose planes share memory
    with pytest.raises(ValueError, match="overlapping"):
        ops.act_restore(ck, out=torch.empty(1, 4, 8, 8, device="cuda").expand(2, 4, 8, 8))
    with pytest.raises(ValueError, match="overlapping"):
        ops.act_restore(ck, out=torch.empty(2, 1, 8, 8, device="cuda").expand(2, 4, 8, 8))
    with pytest.raises(ValueError, match="overlapping"):
        ops.mul_act_grad_ckpt(x, ck, 0.1, out=torch.empty(1, 4, 8, 8, device="cuda").expand(2, 4, 8, 8))
    ops.act_restore(ck, out=torch.empty(4, 2, 8, 8, device="cuda").transpose(0, 1))      # interleaved samples do not


def test_sizes_past_32_bits_are_refused():
    """A size of 2^31 or more does not fit the library's arguments: refused, not wrapped, and before anything is allocated."""
    from deepvideocodec_amd import ops
    x = torch.zeros(1, 1, 4, 4, device="cuda")
    for shape in (((1 << 32) + 2, 1, 4, 4), (1, (1 << 32) + 2, 4, 4), (1 << 31, 1, 4, 4)):
        view = x.expand(shape)
        for call in (lambda: ops.act_checkpoint(view), lambda: ops.act_signs(view),
                     lambda: ops.act_grad_signs(view, torch.zeros(1, dtype=torch.int32, device="cuda"), 0.1, False, shape),
                     lambda: ops.mul_act_grad_ckpt(view, ops.act_checkpoint(x)._replace(shape=shape), 0.1, out=view),
                     lambda: ops.act_restore(ops.act_checkpoint(x)._replace(shape=shape)),
                     lambda: ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x)._replace(shape=shape), x, (1, shape[1], 3, 3))):
            with pytest.raises(ValueError):
                call()


def test_tensors_of_another_device_than_the_current_one_are_refused(monkeypatch):
    from deepvideocodec_amd import ops
    x = torch.randn(2, 4, 8, 8, device="cuda")
    ck = ops.act_checkpoint(x)
    monkeypatch.setattr(ops, "_on_current_device", lambda t, name: (_ for _ in ()).throw(ValueError(f"{name}: other device")))
    for call in (lambda: ops.act_checkpoint(x), lambda: ops.act_restore(ck), lambda: ops.act_signs(x),
                 lambda: ops.act_grad_signs(x, torch.zeros(2, 4, 2, dtype=torch.int32, device="cuda"), 0.1, False, (2, 4, 8, 8)),
                 lambda: ops.mul_act_grad_ckpt(x, ck, 0.1), lambda: ops.conv2d_wgrad_ckpt(ck, x, (4, 4, 3, 3)),
                 lambda: ops.symbol_log_probs(x, torch.zeros(2, 2, 8, 8, dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError, match="other device"):
            call()


def _lib_error():
    from deepvideocodec_amd import _lib
    return _lib.DvcError


def test_on_a_side_stream_and_in_a_replayed_graph():
    from deepvideocodec_amd import ops
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(2, 40, 24, 40, generator=gen).cuda()
    g = torch.randn(2, 48, 24, 40, generator=gen).cuda()

    def passes():
        ck = ops.act_checkpoint(x, slope=0.1)
        gp = ops.act_grad_signs(g, ops.act_signs(g), 0.1, False, tuple(g.shape))
        return ops.conv2d_wgrad_ckpt(ck, gp, (48, 40, 3, 3), with_bias=True) + (ops.mul_act_grad_ckpt(x, ck, 0.1),)

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
    for round_ in range(4):
        x.copy_(torch.randn(x.shape, generator=gen))
        g.copy_(torch.randn(g.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, passes()):
            assert torch.equal(a, b), round_


# ---------------------------------------------------------------------------------------- on the tape
CONV = [
    # k, stride, cins, cout, H, W, batch, in_slope, out_slope, shuffle
    (3, 1, (64,), 64, 36, 52, 2, None, None, False),
    (3, 1, (16, 8), 40, 17, 23, 1, 0.1, 0.01, False),
    (3, 2, (67,), 64, 32, 48, 1, None, 0.1, False),
    (7, 1, (16,), 2, 20, 37, 2, None, 0.0, False),
    (1, 1, (32,), 8, 9, 11, 1, 0.0, None, True),
    (3, 1, (24,), 32, 10, 14, 2, None, 0.01, True),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("k,stride,cins,cout,H,W,batch,in_slope,out_slope,shuffle", CONV)
def test_convolution_on_the_tape(k, stride, cins, cout, H, W, batch, in_slope, out_slope, shuffle, fmt):
    """With 8-bit storage outputs, data gradients and bias gradients keep their bits; the weight gradient is that of the
    restored operands."""
    from deepvideocodec_amd import autograd as A, ops
    gen = torch.Generator().manual_seed(k + cout + H)
    xs = [torch.randn(batch, c, H, W, generator=gen).cuda().requires_grad_() for c in cins]
    wt = (torch.randn(cout, sum(cins), k, k, generator=gen) / math.sqrt(sum(cins) * k * k)).cuda().requires_grad_()
    b = torch.randn(cout, generator=gen).cuda().requires_grad_()
    res = {}
    for storage in (None, fmt):
        y = A.conv2d(xs, wt, b, stride=stride, in_slope=in_slope, out_slope=out_slope, pixel_shuffle=shuffle, storage=storage)
        R = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).cuda()
        res[storage] = (y.detach(),) + torch.autograd.grad(y, [*xs, wt, b], R)
    n = len(xs)
    for a, c in zip(res[None][:1 + n], res[fmt][:1 + n]):
        assert torch.equal(a, c)
    cks = [ops.act_checkpoint(x.detach(), in_slope, fmt) for x in xs]
    p = k // 2
    ho, wo = (H + 2 * p - k) // stride + 1, (W + 2 * p - k) // stride + 1
    g = R if out_slope is None and not shuffle else ops.act_grad(R, res[None][0], 1.0 if out_slope is None else out_slope, shuffle, (batch, cout, ho, wo))
    x64 = torch.cat([ops.act_restore(ck).cpu().double() for ck in cks], 1)
    want, want_b = wgrad64(x64, g.cpu().double(), k, stride)
    most, most_b = wgrad64(x64.abs(), g.cpu().double().abs(), k, stride)
    pixels = batch * ho * wo
    assert bool(((res[fmt][1 + n].cpu().double() - want).abs() <= 3 * pixels * 2.0 ** -24 * most).all())
    assert bool(((res[fmt][2 + n].cpu().double() - want_b).abs() <= pixels * 2.0 ** -24 * most_b).all())
    # and no further from the weight gradient of the operands themselves than the storage's rounding takes it
    x32 = torch.cat([leaky32(x.detach().cpu(), in_slope) for x in xs], 1).double()
    off = wgrad64((x64 - x32).abs(), g.cpu().double().abs(), k, stride)[0]
    ref, most_ref = res[None][1 + n].cpu().double(), wgrad64(x32.abs(), g.cpu().double().abs(), k, stride)[0]
    assert bool(((res[fmt][1 + n].cpu().double() - ref).abs() <= off + 3 * pixels * 2.0 ** -24 * (most + 2 * most_ref)).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("kw", [dict(slope=0.01), dict(slope=0.0), dict(slope=0.1, start_from_relu=True, end_with_relu=True, bottleneck=True),
                                dict(slope=0.01, start_from_relu=False)])
def test_residual_block_on_the_tape(kw, fmt):
    """Outputs and data gradients keep their bits; the weight and bias gradients are those of the same two convolutions
    taken one by one with the same storage."""
    from deepvideocodec_amd import autograd as A
    from deepvideocodec_amd.models.layers import ResBlock
    torch.manual_seed(0)
    blk = ResBlock(32, **kw).cuda()
    x = torch.randn(2, 32, 18, 26).cuda().requires_grad_()
    plus = torch.randn(2, 32, 18, 26).cuda().requires_grad_()
    R = torch.randn(2, 32, 18, 26).cuda()
    params = [blk.conv1.weight, blk.conv1.bias, blk.conv2.weight, blk.conv2.bias]
    res = {}
    for storage in (None, fmt):
        blk.conv1.act_storage = blk.conv2.act_storage = storage
        y = blk(x, plus=plus)
        res[storage] = (y.detach(),) + torch.autograd.grad(y, [x, plus, *params], R)
    for i in (0, 1, 2):
        assert torch.equal(res[None][i], res[fmt][i]), i
    s_in, s_mid, s_out = blk.slope if blk.start_from_relu else None, blk.slope, blk.slope if blk.end_with_relu else None
    t = A.conv2d(x, blk.conv1.weight, blk.conv1.bias, in_slope=s_in, out_slope=s_mid, storage=fmt)
    y = A.conv2d(t, blk.conv2.weight, blk.conv2.bias, out_slope=s_out, residual=x, residual2=plus, storage=fmt)
    for a, c in zip(torch.autograd.grad(y, params, R), res[fmt][3:]):
        assert torch.equal(a, c)


@pytest.mark.parametrize("in_slope,out_slope", [(None, None), (0.1, None), (None, 0.01), (0.0, 0.2)])
@pytest.mark.parametrize("which", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (1, 1, 0), (0, 1, 1)])
def test_partly_frozen_convolution_on_the_tape(which, in_slope, out_slope):
    """Only some of input, weight and bias have gradients: those are the ones of the whole, and the tape keeps codes only where
    one of them reads them."""
    from deepvideocodec_amd import autograd as A
    gen = torch.Generator().manual_seed(9)
    x, wt, b = torch.randn(2, 20, 9, 12, generator=gen).cuda(), torch.randn(24, 20, 3, 3, generator=gen).cuda(), torch.randn(24, generator=gen).cuda()
    R = torch.randn(2, 24, 9, 12, generator=gen).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, wt, b)]
    whole = torch.autograd.grad(A.conv2d(*leaves, in_slope=in_slope, out_slope=out_slope, storage="int8"), leaves, R)
    some = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, wt, b), which)]
    y = A.conv2d(*some, in_slope=in_slope, out_slope=out_slope, storage="int8")
    codes = any(t is not None and t.dtype == torch.uint8 for t in y.grad_fn.saved_tensors)
    assert codes == bool(which[1] or (which[0] and in_slope is not None))
    got = torch.autograd.grad(y, [t for t in some if t.requires_grad], R)
    want = [t for t, w in zip(whole, which) if w]
    for a, c, t in zip(got, want, [t for t in some if t.requires_grad]):
        if t is some[2]:       # a bias alone is summed by another kernel
            assert float((a - c).abs().max()) <= 2 * 9 * 12 * 2.0 ** -24 * float(R.abs().sum((0, 2, 3)).max())
        else:
            assert torch.equal(a, c)


def test_frozen_convolution_stores_nothing(monkeypatch):
    """Where no gradient is asked for (a frozen layer behind frozen layers, under grad mode) nothing is coded, signs included."""
    from deepvideocodec_amd import autograd as A, ops
    gen = torch.Generator().manual_seed(10)
    x, wt, b = torch.randn(1, 8, 9, 12, generator=gen).cuda(), torch.randn(8, 8, 3, 3, generator=gen).cuda(), torch.randn(8, generator=gen).cuda()
    want = A.conv2d(x, wt, b, in_slope=0.1, out_slope=0.2)
    calls = []
    for name in ("act_signs", "act_checkpoint"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, f=getattr(ops, name), **k: (calls.append(name), f(*a, **k))[1])
    y = A.conv2d(x, wt, b, in_slope=0.1, out_slope=0.2, storage="int8")
    assert torch.equal(y, want) and not y.requires_grad and calls == []
    y = A.conv2d(x, wt, b.requires_grad_(), in_slope=0.1, out_slope=0.2, storage="int8")
    assert torch.equal(y, want) and calls == ["act_signs"]
    (gb,) = torch.autograd.grad(y, b, torch.ones_like(y))
    assert float((gb - torch.where(want > 0, 1.0, 0.2).sum((0, 2, 3))).abs().max()) <= 9 * 12 * 2.0 ** -24 * 9 * 12


@pytest.mark.parametrize("start", [True, False])
@pytest.mark.parametrize("which", [(), ("plus",), ("x",), ("x", "plus"), ("w1",), ("b1",), ("w2", "b2"), ("x", "w2"), ("b2",), ("x", "b1")])
def test_partly_frozen_residual_block_and_gate(which, start, monkeypatch):
    """The gradients that are asked for are those of the whole; codes are kept only of what one of them reads."""
    from deepvideocodec_amd import autograd as A, ops
    from deepvideocodec_amd.models.layers import ResBlock
    torch.manual_seed(0)
    blk = ResBlock(32, slope=0.1, start_from_relu=start, end_with_relu=True).cuda()
    blk.conv1.act_storage = blk.conv2.act_storage = "int8"
    x, plus, R = (torch.randn(2, 32, 9, 12).cuda() for _ in range(3))
    leaves = {"x": x, "plus": plus, "w1": blk.conv1.weight, "b1": blk.conv1.bias, "w2": blk.conv2.weight, "b2": blk.conv2.bias}
    for t in leaves.values():
        t.requires_grad_()
    whole = dict(zip(leaves, torch.autograd.grad(blk(x, plus=plus), list(leaves.values()), R)))
    for name, t in leaves.items():
        t.requires_grad_(name in which)
    calls = []
    for name in ("act_signs", "act_checkpoint", "plane_dot"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, f=getattr(ops, name), **k: (calls.append(name), f(*a, **k))[1])
    y = blk(x, plus=plus)
    inner = set(which) - {"plus"}
    reads_x = bool(inner & {"w1", "b1"}) or ("x" in inner and start)
    assert sorted(calls) == ["act_checkpoint"] * (bool(inner) + reads_x) + ["act_signs"] * bool(inner)
    if which:
        for name, got in zip(which, torch.autograd.grad(y, [leaves[n] for n in which], R)):
            assert torch.equal(got, whole[name]), name
    calls.clear()
    fc1, fc2 = torch.randn(4, 32).cuda(), torch.randn(32, 4).cuda()
    A.se_gate(x.detach(), fc1, fc2, "int8")
    assert calls == []


def test_squeeze_excite_pieces_on_the_tape():
    from deepvideocodec_amd import autograd as A, ops
    torch.manual_seed(0)
    a, b, g = (torch.randn(2, 32, 20, 24).cuda() for _ in range(3))
    scale = torch.rand(64).cuda().requires_grad_()
    fc1, fc2 = torch.randn(4, 32).cuda().requires_grad_(), torch.randn(32, 4).cuda().requires_grad_()
    b.requires_grad_()
    for storage in ("int8", "e4m3"):
        gb, gs = torch.autograd.grad(A.add_scaled(a, b, scale, storage=storage), [b, scale], g)
        assert torch.equal(gb, torch.autograd.grad(A.add_scaled(a, b, scale), b, g)[0])
        stored = ops.act_restore(ops.act_checkpoint(b.detach(), fmt=storage))
        assert torch.equal(gs, ops.plane_dot(g, stored).view_as(gs))
        r = torch.randn(64).cuda()
        for u, v in zip(torch.autograd.grad(A.se_gate(b, fc1, fc2, storage), [b, fc1, fc2], r), torch.autograd.grad(A.se_gate(b, fc1, fc2), [b, fc1, fc2], r)):
            assert torch.equal(u, v)


def test_training_step_on_8_bit_storage(seeded_sd):
    """The model's own training step with 8-bit storage: the same loss to the bit, gradients for the same parameters, less
    memory held by the tape.  (The layers' gradients are held to the definition above, layer by layer.)"""
    from deepvideocodec_amd import train as TR
    from deepvideocodec_amd.models import DMC
    from deepvideocodec_amd.testing import synthetic_gop
    frames = [f.cuda() for f in synthetic_gop(3, 128, 128, seed=3, batch=2)]
    res, held = {}, {}
    for storage in ("fp32", "int8", "e4m3"):
        net = DMC()
        net.load_state_dict(seeded_sd)
        net = net.cuda().train().set_act_storage(storage)
        torch.manual_seed(5)
        net(list(frames))                     # (weight images are built on first use and kept)
        torch.manual_seed(5)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = TR.RateDistortionLoss(lmbda=2048.0)(net(list(frames)), frames[1:])
        held[storage] = torch.cuda.memory_allocated() - before
        out["loss"].backward()
        res[storage] = (out["loss"].item(), {n: p.grad for n, p in net.named_parameters() if p.grad is not None})
        del net, out
    for storage in ("int8", "e4m3"):
        assert res[storage][0] == res["fp32"][0]
        assert set(res[storage][1]) == set(res["fp32"][1])
        assert all(bool(torch.isfinite(g).all()) for g in res[storage][1].values())
        assert held[storage] < held["fp32"], held


def test_recompute_with_8_bit_storage(seeded_sd):
    """Blocks that are recomputed in the backward pass store their operands in 8 bits while that runs: the same loss."""
    from deepvideocodec_amd import train as TR
    from deepvideocodec_amd.models import DMC
    from deepvideocodec_amd.testing import synthetic_gop
    frames = [f.cuda() for f in synthetic_gop(2, 64, 64, seed=3, batch=1)]
    res = []
    for recompute in (False, True):
        net = DMC()
        net.load_state_dict(seeded_sd)
        net = net.cuda().train().set_act_storage("int8")
        net.recompute = recompute
        torch.manual_seed(5)
        out = TR.RateDistortionLoss(lmbda=2048.0)(net(list(frames)), frames[1:])
        out["loss"].backward()
        res.append((out["loss"].item(), {n: p.grad for n, p in net.named_parameters() if p.grad is not None}))
    (l0, g0), (l1, g1) = res
    assert l0 == l1 and g0.keys() == g1.keys()
    assert all(bool(torch.isfinite(g).all()) for g in g1.values())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_past_two_to_the_31_values(fmt):
    """More than 2^31 values and 2^33 bytes: the last sample's checkpoint, signs, adjoints and weight gradient are its own."""
    from deepvideocodec_amd import ops
    g = torch.Generator(device="cuda").manual_seed(21)
    x = torch.empty((33, 64, 1024, 1024), device="cuda").uniform_(-1, 1, generator=g)
    assert x.numel() > 1 << 31
    ck, one = ops.act_checkpoint(x, 0.1, fmt), ops.act_checkpoint(x[-1:], 0.1, fmt)
    assert torch.equal(ck.codes[-1:], one.codes) and torch.equal(ck.scales[-1:], one.scales)
    signs = ops.act_signs(x)
    assert torch.equal(signs[-1:], ops.act_signs(x[-1:]))
    assert torch.equal(ops.act_grad_signs(x, signs, 0.5, False, x.shape)[-1:], ops.act_grad_signs(x[-1:], signs[-1:], 0.5, False, (1, *x.shape[1:])))
    assert torch.equal(ops.mul_act_grad_ckpt(x, ck, 0.5)[-1:], ops.mul_act_grad_ckpt(x[-1:], one, 0.5))
    out = ops.act_restore(ck, out=x)
    assert out is x and torch.equal(x[-1:], ops.act_restore(one))
    # whole numbers below 2^24: every order of the sums gives the same
    x.random_(-1, 2, generator=g)
    grad = torch.zeros((33, 64, 1024, 1024), device="cuda")
    grad[-1].random_(-1, 2, generator=g)
    gw, gb = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x, None, fmt), grad, (64, 64, 3, 3), with_bias=True)
    ow, ob = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x[-1:], None, fmt), grad[-1:].contiguous(), (64, 64, 3, 3), with_bias=True)
    assert torch.equal(gw, ow) and torch.equal(gb, ob) and float(gw.abs().max()) > 1000


def test_weight_gradient_of_one_huge_sample():
    """A sample's gradient of more than 2^31 bytes, against a product in 64 bits."""
    from deepvideocodec_amd import ops
    g = torch.Generator(device="cuda").manual_seed(22)
    h, w = 3001, 3000
    x = torch.empty((1, 64, h, w), device="cuda").random_(-1, 2, generator=g)
    grad = torch.empty((1, 64, h, w), device="cuda").random_(-1, 2, generator=g)
    assert grad.numel() * 4 > 1 << 31 and h * w < 1 << 24         # (whole numbers: exact sums)
    got = ops.conv2d_wgrad_ckpt(ops.act_checkpoint(x), grad, (64, 64, 1, 1)).view(64, 64)
    want = grad.view(64, -1).double() @ x.view(64, -1).double().t()
    assert torch.equal(got.double(), want)


def step_gradients(seeded_sd, storage, recompute=False, size=128):
    """One training step's gradients of the model with its seeded weights, the same noise every time."""
    from deepvideocodec_amd import train as TR
    from deepvideocodec_amd.models import DMC
    from deepvideocodec_amd.testing import synthetic_gop
    frames = [f.cuda() for f in synthetic_gop(3, size, size, seed=3, batch=2)]
    net = DMC()
    net.load_state_dict(seeded_sd)
    net = net.cuda().train().set_act_storage(storage)
    net.recompute = recompute
    torch.manual_seed(5)
    TR.RateDistortionLoss(lmbda=2048.0)(net(list(frames)), frames[1:])["loss"].backward()
    return {n: p.grad.double() for n, p in net.named_parameters() if p.grad is not None}


@pytest.mark.parametrize("fmt,most", [("int8", 0.1), ("e4m3", 0.15)])
def test_training_step_gradients_stay_close_to_those_of_fp32_storage(seeded_sd, fmt, most):
    """Every parameter's gradient against that of fp32 storage.  A stored operand's rounding is independent of the gradient it is
    multiplied with, so a weight gradient moves by the rounding's root mean square in units of the operand's: int8, half a
    step below 1/127 of the block's largest, which is at most sqrt(32) of its root mean square: sqrt(32) / 127 / sqrt(3) = 0.026;
    e4m3, half a step at most 2^-4 of the value: 2^-4 / sqrt(3) = 0.036.  Four times that is allowed, as products and
    operands are not quite uncorrelated; a wrong mask, scale or layout in any layer is off by the order of one."""
    want, got = step_gradients(seeded_sd, "fp32"), step_gradients(seeded_sd, fmt)
    assert want.keys() == got.keys()
    off = {n: float((got[n] - want[n]).norm() / want[n].norm()) for n in want if float(want[n].norm()) > 0}
    worst = sorted(off, key=off.get)[-3:]
    print(fmt, [(n, f"{off[n]:.1e}") for n in worst], f"median {sorted(off.values())[len(off) // 2]:.1e}")
    assert len(off) > 200 and off[worst[-1]] <= most


@pytest.mark.parametrize("fmt", FORMATS)
def test_recompute_with_8_bit_storage_gives_the_same_gradients(seeded_sd, fmt):
    """Recomputed blocks are stored from the same activations: the same gradients up to the order of sums (and the warp's
    atomics), as in fp32."""
    want, got = (step_gradients(seeded_sd, fmt, recompute, 64) for recompute in (False, True))
    assert want.keys() == got.keys()
    assert max(float((want[n] - got[n]).abs().max()) / max(float(want[n].abs().max()), 1e-20) for n in want) < 1e-4
