"""Refusals of the 8-bit checkpoint and symbol log-probability entry points, without a GPU: argument errors come back
as codes / exceptions before anything is launched."""
import ctypes as C

import pytest
import torch

from deepvideocodec_amd import _lib, ops
from deepvideocodec_amd._lib import DvcCkpt, DvcDst, DvcLogits, DvcSrc

P = 1 << 20      # stands for a device address: never dereferenced, every call below is refused first


def refused(rc, *words):
    assert rc == -1, rc
    for w in words:
        assert w in _lib.last_error(), _lib.last_error()


def src(ptr=P, cs=64, c=3):
    return C.byref(DvcSrc(ptr, c * cs, cs, c, 0))


def dst(ptr=P, cs=64):
    return C.byref(DvcDst(ptr, 3 * cs, cs))


def ck(codes=P, scales=P, c=3, fmt=0):
    return C.byref(DvcCkpt(codes, scales, c, fmt))


def lg(ptr=P, bs=1000, cs=64, groups=1, classes=5, dtype=0):
    return C.byref(DvcLogits(ptr, bs, cs, groups, classes, dtype, 0))


def test_checkpoint_refusals():
    lib = _lib.load()
    refused(lib.dvc_act_checkpoint(None, 0, 1.0, 0, P, P, 1, 8, 8, None), "source")
    refused(lib.dvc_act_checkpoint(src(cs=63), 0, 1.0, 0, P, P, 1, 8, 8, None), "stride")
    refused(lib.dvc_act_checkpoint(src(), 0, 1.0, 2, P, P, 1, 8, 8, None), "format")
    refused(lib.dvc_act_checkpoint(src(), 1, 1.5, 0, P, P, 1, 8, 8, None), "slope")
    refused(lib.dvc_act_checkpoint(src(), 1, -0.1, 0, P, P, 1, 8, 8, None), "slope")
    refused(lib.dvc_act_checkpoint(src(), 0, 1.0, 0, P + 4, P, 1, 8, 8, None), "16 bytes")
    refused(lib.dvc_act_checkpoint(src(), 0, 1.0, 0, None, P, 1, 8, 8, None), "null")
    refused(lib.dvc_act_checkpoint(src(), 0, 1.0, 0, P, P, 0, 8, 8, None), "dims")
    refused(lib.dvc_act_checkpoint(src(cs=1 << 40), 0, 1.0, 0, P, P, 1, 1 << 14, 1 << 14, None), "plane")
    refused(lib.dvc_act_restore(ck(fmt=7), dst(), 1, 8, 8, None), "format")
    refused(lib.dvc_act_restore(ck(codes=None), dst(), 1, 8, 8, None), "checkpoint")
    refused(lib.dvc_act_restore(ck(), dst(cs=10), 1, 8, 8, None), "destination")
    refused(lib.dvc_act_signs(src(), None, 1, 8, 8, None), "null")
    refused(lib.dvc_act_grad_signs(src(c=2), P, 0.1, 0, P, 1, 3, 8, 8, None), "channels")
    refused(lib.dvc_act_grad_signs(src(cs=256, c=1), P, 0.1, 1, P, 1, 6, 8, 8, None), "shuffled")
    refused(lib.dvc_mul_act_grad_ckpt(src(c=2), ck(c=3), 0.1, None, dst(), 1, 8, 8, None), "channels")
    refused(lib.dvc_mul_act_grad_ckpt(src(), ck(), 0.1, src(c=2), dst(), 1, 8, 8, None), "plus")


def test_weight_gradient_refusals():
    lib = _lib.load()

    def call(srcs, n=1, k=3, stride=1, grad=P, scratch=P, gw=P, h=8):
        return lib.dvc_conv2d_wgrad_ckpt(srcs, n, 1, h, 8, grad, 4, k, stride, scratch, gw, None, None)

    one = (DvcCkpt * 1)(DvcCkpt(P, P, 3, 0))
    refused(call(one, n=0), "n_src")
    refused(call(one, n=5), "n_src")
    refused(call(one, k=5), "ksize")
    refused(call(one, k=7, stride=2), "7x7")
    refused(call(one, stride=3), "stride")
    refused(call(one, grad=None), "null")
    refused(call(one, scratch=None), "null")
    refused(call(one, h=0), "dims")
    refused(call(one, scratch=P + 4), "16 bytes")
    refused(call((DvcCkpt * 1)(DvcCkpt(P + 1, P, 3, 0))), "16 bytes")
    refused(call((DvcCkpt * 2)(DvcCkpt(P, P, 3, 0), DvcCkpt(P, P, 3, 1)), n=2), "format")
    assert lib.dvc_conv2d_wgrad_ckpt_scratch_floats(4, 3, 5, 1, 1, 8, 8) == -1
    assert lib.dvc_conv2d_wgrad_ckpt_scratch_floats(4, 3, 3, 1, 1, 8, 8) > 0


@pytest.mark.parametrize("cout,cin,k,stride,n,h,w", [
    (64, 64, 3, 1, 32, 256, 256), (192, 192, 3, 1, 32, 256, 256), (512, 512, 3, 1, 32, 128, 128), (1024, 1024, 1, 1, 8, 512, 512),
    (64, 32, 7, 1, 32, 256, 256), (512, 512, 7, 1, 8, 256, 256), (40, 24, 3, 2, 64, 512, 512), (3, 64, 3, 1, 512, 256, 256), (2, 16, 7, 1, 4, 16, 16)])
def test_weight_gradient_scratch_does_not_grow_with_the_pixels(cout, cin, k, stride, n, h, w):
    """One block of every tap for each of about 256 workgroups (64 x 64, 7x7: 32 x 32; of weights that alone give more blocks than
    that, one block each) or 128 MiB, whichever is more, and a row of bias sums for each workgroup."""
    side = 32 if k == 7 else 64
    blocks = -(-cout // side) * -(-cin // side)
    most = max((256 + blocks) * side * side * k * k, 128 << 18) + (256 + blocks) * (cout + side)
    lib = _lib.load()
    for m in (n, 4 * n, 64 * n):
        assert 0 < lib.dvc_conv2d_wgrad_ckpt_scratch_floats(cout, cin, k, stride, m, h, w) <= most


def test_symbol_refusals():
    lib = _lib.load()

    def call(l, top=0, sym=P, lp=P, tl=P, ts=P, h=8):
        return lib.dvc_symbol_log_probs(l, sym, top, lp, P, P, tl, ts, None, 1, h, 8, None)

    refused(call(lg(ptr=None)), "null")
    refused(call(lg(classes=0)), "classes")
    refused(call(lg(groups=0)), "groups")
    refused(call(lg(dtype=3)), "type")
    refused(call(lg(cs=63)), "stride")
    refused(call(lg(), top=6), "top")
    refused(call(lg(classes=99), top=17), "top")
    refused(call(lg(), top=-1), "top")
    refused(call(lg(), top=2, tl=None), "null")
    refused(call(lg(), sym=None), "null")
    refused(call(lg(), lp=None), "null")
    refused(call(lg(), h=0), "dims")
    refused(lib.dvc_symbol_log_probs_backward(lg(), P, None, P, P, P, P, 1, 8, 8, None), "null")
    refused(lib.dvc_symbol_log_probs_backward(lg(), P, P, P, P, P, None, 1, 8, 8, None), "null")
    assert lib.dvc_symbol_log_probs_scratch_floats(lg(classes=0), 0, 1, 8, 8) == -1
    # one long row is cut over workgroups, which leave their parts in the scratch buffer
    long_row = lg(cs=1, classes=131072)
    assert lib.dvc_symbol_log_probs_scratch_floats(long_row, 8, 1, 1, 1) > 0
    assert lib.dvc_symbol_log_probs_scratch_floats(long_row, 17, 1, 1, 1) == -1
    refused(lib.dvc_symbol_log_probs(long_row, P, 8, P, P, P, P, P, None, 1, 1, 1, None), "scratch")
    assert lib.dvc_symbol_log_probs_scratch_floats(lg(cs=1, classes=1000), 8, 1, 1, 1) == 0
    # more threads than a launch has
    refused(lib.dvc_symbol_log_probs(lg(cs=1, classes=1000), P, 0, P, P, P, None, None, None, 1 << 27, 1, 1, None), "too many")
    refused(lib.dvc_symbol_log_probs(lg(cs=1, classes=5000), P, 0, P, P, P, None, None, None, 1 << 25, 1, 1, None), "too many")
    refused(lib.dvc_symbol_log_probs_backward(lg(cs=1, classes=5000), P, P, P, P, P, P, 1 << 25, 1, 1, None), "too many")
    refused(lib.dvc_symbol_log_probs(lg(cs=1 << 27, classes=4), P, 0, P, P, P, None, None, None, 64, 1 << 13, 1 << 14, None), "too many")
    refused(lib.dvc_symbol_log_probs_backward(lg(cs=1 << 27, classes=400), P, P, P, P, P, P, 64, 1 << 13, 1 << 14, None), "too many")


def test_python_surface_refuses_cpu_tensors_and_unknown_names():
    x = torch.zeros(1, 2, 4, 4)
    with pytest.raises(_lib.DvcError, match="no CPU fallback"):
        ops.act_checkpoint(x)
    with pytest.raises(_lib.DvcError, match="no CPU fallback"):
        ops.act_signs(x)
    with pytest.raises(ValueError, match="format"):
        ops.act_checkpoint(x, fmt="int4")
    with pytest.raises(_lib.DvcError, match="no CPU fallback"):
        ops.act_restore(ops.ActCheckpoint(torch.zeros(1, 2, 32, dtype=torch.uint8), torch.zeros(1, 2, 1, dtype=torch.uint8), (1, 2, 4, 4), "int8"))
    with pytest.raises(TypeError, match="ActCheckpoint"):
        ops.act_restore(x)
    with pytest.raises(_lib.DvcError, match="no CPU fallback"):
        ops.symbol_log_probs(torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32))
    from deepvideocodec_amd.models import DMC
    with pytest.raises(ValueError, match="storage"):
        DMC().set_act_storage("int4")


def test_storage_setting_reaches_every_layer():
    from deepvideocodec_amd.models import DMC
    from deepvideocodec_amd.models.layers import Conv2d, SELayer
    net = DMC()
    layers = [m for m in net.modules() if isinstance(m, (Conv2d, SELayer))]
    assert len(layers) > 80 and all(m.act_storage is None for m in layers)
    assert net.set_act_storage("int8") is net
    assert all(m.act_storage == "int8" for m in layers)
    net.set_act_storage("fp32")
    assert all(m.act_storage is None for m in layers)
