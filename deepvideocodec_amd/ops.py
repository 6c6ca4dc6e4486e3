"""Tensor-level wrappers over the libdvc_hip.so C ABI.

torch is used for device memory and stream plumbing only: every arithmetic op
here is a HIP kernel of this package launched on torch's current stream.
All tensors must be fp32 (int32 for symbols / indexes, uint8 for 8-bit checkpoints;
logits may be bf16 / fp16 as well) CUDA(HIP) tensors in NCHW with contiguous rows; batch / channel strides are free, so channel slices
of a larger buffer are accepted as sources, residuals and destinations.
"""
import ctypes as C
from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import DvcCkpt, DvcConv2d, DvcDst, DvcLogits, DvcSrc, check

Tensor = torch.Tensor
Srcs = Union[Tensor, Sequence[Tensor]]


def _stream() -> int:
    """The current stream of the current device (torch.cuda.current_stream().cuda_stream without the stream object: a
    tenth of a launch's host time instead of half of it)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _check4(t: Tensor, name: str, dtype=torch.float32):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t)}")
    if not t.is_cuda:
        raise _lib.DvcError(f"{name}: tensor is on {t.device}; the HIP path needs a GPU tensor (no CPU fallback)")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.dim() != 4:
        raise ValueError(f"{name}: expected NCHW, got shape {tuple(t.shape)}")
    if t.size(3) > 1 and t.stride(3) != 1 or (t.size(2) > 1 and t.stride(2) != t.size(3)):
        raise ValueError(f"{name}: rows must be contiguous (strides {t.stride()})")


def _check_vec(t: Optional[Tensor], numel: Optional[int], name: str, dtype=torch.float32, device=None):
    """A flat parameter-like operand handed to the library as a raw pointer (bias, gates, packed
    weights, tables): must be a contiguous GPU tensor of the stated dtype and element count, on the
    same device as the data -- anything else would be an out-of-bounds device read."""
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a tensor, got {type(t)}")
    if not t.is_cuda:
        raise _lib.DvcError(f"{name}: tensor is on {t.device}; the HIP path needs a GPU tensor (no CPU fallback)")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, the data is on {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous (strides {t.stride()})")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} elements, got {t.numel()} (shape {tuple(t.shape)})")


def _bs(t: Tensor) -> int:
    return t.stride(0) if t.size(0) > 1 else t.size(1) * max(t.stride(1), t.size(2) * t.size(3))


def _cs(t: Tensor) -> int:
    return t.stride(1) if t.size(1) > 1 else t.size(2) * t.size(3)


def _src(t: Tensor, name="src") -> DvcSrc:
    _check4(t, name)
    return DvcSrc(t.data_ptr(), _bs(t), _cs(t), t.size(1), 0)


def _dst(t: Tensor, name="out") -> DvcDst:
    _check4(t, name)
    return DvcDst(t.data_ptr(), _bs(t), _cs(t))


def _null_dst() -> DvcDst:
    return DvcDst(None, 0, 0)


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


PRECISIONS = {"fp32": 0, "bf16": 1, "bf16x2": 2, "fp16x2": 3}


def pack_conv_weight(weight: Tensor, stride: int = 1, precision: int = 0) -> Tensor:
    """OIHW weight -> the slab layout dvc_conv2d reads (re-pack whenever the weight changes).
    `precision` (PRECISIONS): 0 exact fp32; 1 bf16-rounded operands; 2 / 3 operands split into bf16 / fp16
    hi + lo parts (7x7: stride 1 only)."""
    if not (weight.is_cuda and weight.is_contiguous() and weight.dtype == torch.float32 and weight.dim() == 4):
        raise ValueError("pack_conv_weight: weight must be a contiguous fp32 OIHW GPU tensor")
    cout, cin, k, k2 = weight.shape
    if k != k2:
        raise ValueError("pack_conv_weight: square kernels only")
    lib = _lib.load()
    precision = int(precision)
    if precision:
        n = check(lib.dvc_conv2d_reduced_packed_weight_floats(cout, cin, k, stride, precision), "dvc_conv2d_reduced_packed_weight_floats")
        packed = torch.empty(n, dtype=torch.float32, device=weight.device)
        check(lib.dvc_conv2d_reduced_pack_weight(weight.data_ptr(), cout, cin, k, stride, precision, packed.data_ptr(), _stream()),
              "dvc_conv2d_reduced_pack_weight")
        return packed
    n = check(lib.dvc_conv2d_packed_weight_floats(cout, cin, k, stride), "dvc_conv2d_packed_weight_floats")
    packed = torch.empty(n, dtype=torch.float32, device=weight.device)
    check(lib.dvc_conv2d_pack_weight(weight.data_ptr(), cout, cin, k, stride, packed.data_ptr(), _stream()),
          "dvc_conv2d_pack_weight")
    return packed


def pack_conv_weight_dgrad(weight: Tensor) -> Tensor:
    """The packed image of the weight of `weight`'s data-gradient convolution (flipped taps, channel axes swapped),
    for conv2d(grad, (cin, cout, k, k), None, packed=...)."""
    if not (weight.is_cuda and weight.is_contiguous() and weight.dtype == torch.float32 and weight.dim() == 4):
        raise ValueError("pack_conv_weight_dgrad: weight must be a contiguous fp32 OIHW GPU tensor")
    cout, cin, k, _ = weight.shape
    lib = _lib.load()
    n = check(lib.dvc_conv2d_packed_weight_floats(cin, cout, k, 1), "dvc_conv2d_packed_weight_floats")
    packed = torch.empty(n, dtype=torch.float32, device=weight.device)
    check(lib.dvc_conv2d_pack_weight_dgrad(weight.data_ptr(), cout, cin, k, packed.data_ptr(), _stream()),
          "dvc_conv2d_pack_weight_dgrad")
    return packed


def conv2d(srcs: Srcs, weight: Tensor, bias: Optional[Tensor], stride: int = 1,
           in_slope: Optional[float] = None, out_slope: Optional[float] = None,
           residual: Optional[Tensor] = None, res_scale: Optional[Tensor] = None,
           residual2: Optional[Tensor] = None, pixel_shuffle: bool = False,
           out: Optional[Tensor] = None, packed: Optional[Tensor] = None, precision: int = 0,
           plane_sums: bool = False):
    """See DvcConv2d in include/dvc_hip.h.  `plane_sums=True` returns (out, sums): where the launch can emit per-tile
    sums of its output planes with its stores (dvc_conv2d_plane_sum_slots), `sums` is the (N, Cout, slots) tensor
    se_gate_from_sums() takes, otherwise None (use se_gate on `out`).  `precision`: see PRECISIONS; fp32 accumulation in every mode (`packed` must come from
    pack_conv_weight(..., precision=) with the same value). `srcs` are concatenated along C; slopes of
    None mean "no activation", 0.0 means ReLU.  `weight` is the OIHW tensor (its shape
    describes the layer); `packed` its pack_conv_weight() image -- packed on the fly if
    not given (callers that reuse a weight should cache it)."""
    if isinstance(srcs, torch.Tensor):
        srcs = (srcs,)
    if not 1 <= len(srcs) <= _lib.DVC_MAX_SRC:
        raise ValueError(f"conv2d: {len(srcs)} sources (1..{_lib.DVC_MAX_SRC} supported)")
    p = DvcConv2d()
    n, _, h, w = srcs[0].shape
    cin = 0
    for i, s in enumerate(srcs):
        if s.shape[0] != n or s.shape[2] != h or s.shape[3] != w:
            raise ValueError(f"conv2d: source {i} shape {tuple(s.shape)} does not match {(n, '*', h, w)}")
        p.src[i] = _src(s, f"conv2d src[{i}]")
        cin += s.size(1)
    if isinstance(weight, torch.Tensor):
        wshape, wdev = tuple(weight.shape), weight.device
        if not (weight.is_cuda and weight.is_contiguous() and weight.dtype == torch.float32):
            raise ValueError("conv2d: weight must be a contiguous fp32 GPU tensor")
    else:   # only the layer's (Cout, Cin, k, k): the caller brings the packed image
        wshape, wdev = tuple(weight), srcs[0].device
        if packed is None:
            raise ValueError("conv2d: a weight shape needs its packed image")
    cout, wcin, k, k2 = wshape
    if wcin != cin or k != k2:
        raise ValueError(f"conv2d: weight {wshape} does not match {cin} input channels")
    pad = k // 2
    ho = (h + 2 * pad - k) // stride + 1
    wo = (w + 2 * pad - k) // stride + 1
    oshape = (n, cout // 4, 2 * ho, 2 * wo) if pixel_shuffle else (n, cout, ho, wo)
    if out is None:
        out = torch.empty(oshape, dtype=torch.float32, device=wdev)
    elif tuple(out.shape) != oshape:
        raise ValueError(f"conv2d: out shape {tuple(out.shape)} != {oshape}")
    p.n_src = len(srcs)
    p.batch, p.in_h, p.in_w = n, h, w
    if packed is None:
        packed = pack_conv_weight(weight, stride, precision=precision)
    _check_vec(packed, None, "conv2d packed weight", device=wdev)
    _check_vec(bias, cout, "conv2d bias", device=wdev)
    p.weight_packed = packed.data_ptr()
    p.precision = int(precision)
    p.bias = _ptr(bias)
    p.out_channels = cout
    p.ksize = k
    p.stride = stride
    p.in_act = 0 if in_slope is None else 1
    p.out_act = 0 if out_slope is None else 1
    p.in_slope = 1.0 if in_slope is None else float(in_slope)
    p.out_slope = 1.0 if out_slope is None else float(out_slope)
    p.pixel_shuffle = 1 if pixel_shuffle else 0
    p.out = _dst(out)
    if residual is not None:
        if tuple(residual.shape) != oshape:
            raise ValueError(f"conv2d: residual shape {tuple(residual.shape)} != {oshape}")
        _check4(residual, "conv2d residual")
        p.residual = residual.data_ptr()
        p.res_batch_stride = _bs(residual)
        p.res_chan_stride = _cs(residual)
    if res_scale is not None:
        if residual is None:
            raise ValueError("conv2d: res_scale needs a residual")
        _check_vec(res_scale, n * oshape[1], "conv2d res_scale", device=wdev)
        p.res_scale = res_scale.data_ptr()
    if residual2 is not None:
        if residual is None or tuple(residual2.shape) != oshape:
            raise ValueError("conv2d: residual2 needs residual and the output shape")
        _check4(residual2, "conv2d residual2")
        p.residual2 = residual2.data_ptr()
        p.res2_batch_stride = _bs(residual2)
        p.res2_chan_stride = _cs(residual2)
    sums = None
    if plane_sums:
        slots = check(_lib.load().dvc_conv2d_plane_sum_slots(C.byref(p)), "dvc_conv2d_plane_sum_slots")
        if slots > 0:
            sums = torch.empty((n, cout, slots), dtype=torch.float32, device=wdev)
            p.plane_sums = sums.data_ptr()
    check(_lib.load().dvc_conv2d(C.byref(p), _stream()), "dvc_conv2d")
    return (out, sums) if plane_sums else out


def flow_warp(src: Tensor, flow: Tensor, out: Optional[Tensor] = None) -> Tensor:
    n, c, h, w = src.shape
    if tuple(flow.shape) != (n, 2, h, w):
        raise ValueError(f"flow_warp: flow shape {tuple(flow.shape)} != {(n, 2, h, w)}")
    if out is None:
        out = torch.empty_like(src, memory_format=torch.contiguous_format)
    elif tuple(out.shape) != (n, c, h, w):
        raise ValueError(f"flow_warp: out shape {tuple(out.shape)} != {(n, c, h, w)}")
    check(_lib.load().dvc_flow_warp(C.byref(_src(src)), C.byref(_src(flow, "flow")), C.byref(_dst(out)),
                                    n, h, w, _stream()), "dvc_flow_warp")
    return out


def avg_pool2(x: Tensor, scale: float = 1.0) -> Tensor:
    n, c, h, w = x.shape
    out = torch.empty((n, c, h // 2, w // 2), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_avg_pool2(C.byref(_src(x)), C.byref(_dst(out)), n, h, w, float(scale), _stream()),
          "dvc_avg_pool2")
    return out


def max_pool2(x: Tensor) -> Tensor:
    n, c, h, w = x.shape
    out = torch.empty((n, c, h // 2, w // 2), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_max_pool2(C.byref(_src(x)), C.byref(_dst(out)), n, h, w, _stream()), "dvc_max_pool2")
    return out


def bilinear_up2(x: Tensor, scale: float = 1.0) -> Tensor:
    n, c, h, w = x.shape
    out = torch.empty((n, c, 2 * h, 2 * w), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_bilinear_up2(C.byref(_src(x)), C.byref(_dst(out)), n, h, w, float(scale), _stream()),
          "dvc_bilinear_up2")
    return out


def spynet_level_input(im1: Tensor, im2: Tensor, flow_prev: Optional[Tensor]) -> Tensor:
    n, _, h, w = im1.shape
    out = torch.empty((n, 8, h, w), dtype=torch.float32, device=im1.device)
    fp = C.byref(_src(flow_prev, "flow_prev")) if flow_prev is not None else None
    check(_lib.load().dvc_spynet_level_input(C.byref(_src(im1, "im1")), C.byref(_src(im2, "im2")), fp,
                                             C.byref(_dst(out)), n, h, w, _stream()), "dvc_spynet_level_input")
    return out


def se_gate(x: Tensor, fc1: Tensor, fc2: Tensor) -> Tensor:
    """sigmoid(fc2 @ relu(fc1 @ mean_hw(x))) -> (N*C,) gate."""
    n, c, h, w = x.shape
    if fc1.dim() != 2 or fc1.size(1) != c:
        raise ValueError(f"se_gate: fc1 shape {tuple(fc1.shape)} does not match {c} channels")
    _check_vec(fc1, fc1.size(0) * c, "se_gate fc1", device=x.device)
    _check_vec(fc2, c * fc1.size(0), "se_gate fc2", device=x.device)
    if tuple(fc2.shape) != (c, fc1.size(0)):
        raise ValueError(f"se_gate: fc2 shape {tuple(fc2.shape)} != {(c, fc1.size(0))}")
    lib = _lib.load()
    partial = torch.empty(lib.dvc_se_scratch_floats(n, c), dtype=torch.float32, device=x.device)
    gate = torch.empty(n * c, dtype=torch.float32, device=x.device)
    check(lib.dvc_se_gate(C.byref(_src(x)), n, h, w, fc1.data_ptr(), fc2.data_ptr(), fc1.size(0),
                          partial.data_ptr(), gate.data_ptr(), _stream()), "dvc_se_gate")
    return gate


def se_gate_from_sums(sums: Tensor, h: int, w: int, fc1: Tensor, fc2: Tensor) -> Tensor:
    """se_gate of an (N, C, h, w) tensor whose per-tile plane sums `sums` (N, C, slots) a convolution wrote with
    its stores (conv2d(..., plane_sums=True)) -> (N*C,) gate."""
    if sums.dim() != 3:
        raise ValueError(f"se_gate_from_sums: sums shape {tuple(sums.shape)} is not (N, C, slots)")
    n, c, slots = sums.shape
    _check_vec(sums, n * c * slots, "se_gate_from_sums sums")
    if fc1.dim() != 2 or fc1.size(1) != c or tuple(fc2.shape) != (c, fc1.size(0)):
        raise ValueError(f"se_gate_from_sums: fc shapes {tuple(fc1.shape)}, {tuple(fc2.shape)} do not match {c} channels")
    _check_vec(fc1, fc1.size(0) * c, "se_gate_from_sums fc1", device=sums.device)
    _check_vec(fc2, c * fc1.size(0), "se_gate_from_sums fc2", device=sums.device)
    lib = _lib.load()
    partial = torch.empty(lib.dvc_se_scratch_floats(n, c), dtype=torch.float32, device=sums.device)
    gate = torch.empty(n * c, dtype=torch.float32, device=sums.device)
    check(lib.dvc_se_gate_from_sums(sums.data_ptr(), slots, n, c, h, w, fc1.data_ptr(), fc2.data_ptr(), fc1.size(0),
                                    partial.data_ptr(), gate.data_ptr(), _stream()), "dvc_se_gate_from_sums")
    return gate


def copy_into(src: Tensor, out: Tensor) -> Tensor:
    n, c, h, w = src.shape
    if tuple(out.shape) != tuple(src.shape):
        raise ValueError("copy_into: shape mismatch")
    check(_lib.load().dvc_copy(C.byref(_src(src)), C.byref(_dst(out)), n, h, w, _stream()), "dvc_copy")
    return out


def clamp(x: Tensor, lo: float, hi: float) -> Tensor:
    n, c, h, w = x.shape
    out = torch.empty((n, c, h, w), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_clamp(C.byref(_src(x)), C.byref(_dst(out)), n, h, w, float(lo), float(hi), _stream()),
          "dvc_clamp")
    return out


def eb_forward(z: Tensor, packed: Tensor, medians: Tensor, noise: Optional[Tensor] = None,
               want_likelihood=True, want_symbols=False):
    """-> (z_hat, likelihood | None, symbols | None)"""
    n, c, h, w = z.shape
    _check_vec(packed, c * _lib.EB_PARAMS_PER_CHANNEL, "eb_forward packed parameters", device=z.device)
    _check_vec(medians, c, "eb_forward medians", device=z.device)
    _check_vec(noise, n * c * h * w, "eb_forward noise", device=z.device)
    z_hat = torch.empty((n, c, h, w), dtype=torch.float32, device=z.device)
    lik = torch.empty_like(z_hat) if want_likelihood else None
    sym = torch.empty((n, c, h, w), dtype=torch.int32, device=z.device) if want_symbols else None
    if noise is not None and not (noise.is_contiguous() and tuple(noise.shape) == (n, c, h, w)):
        raise ValueError("eb_forward: noise must be contiguous and shaped like z")
    check(_lib.load().dvc_eb_forward(C.byref(_src(z, "z")), _ptr(noise), packed.data_ptr(), medians.data_ptr(),
                                     C.byref(_dst(z_hat)), C.byref(_dst(lik) if lik is not None else _null_dst()),
                                     _ptr(sym), n, h, w, _stream()), "dvc_eb_forward")
    return z_hat, lik, sym


def eb_dequantize(symbols: Tensor, medians: Tensor) -> Tensor:
    n, c, h, w = symbols.shape
    _check_vec(symbols, None, "eb_dequantize symbols", dtype=torch.int32)
    _check_vec(medians, c, "eb_dequantize medians", device=symbols.device)
    z_hat = torch.empty((n, c, h, w), dtype=torch.float32, device=symbols.device)
    check(_lib.load().dvc_eb_dequantize(symbols.data_ptr(), medians.data_ptr(), C.byref(_dst(z_hat)), n, c, h, w,
                                        _stream()), "dvc_eb_dequantize")
    return z_hat


def dual_prior_pass1(y: Tensor, means: Tensor, scales: Tensor) -> Tensor:
    n, c, h, w = y.shape
    out = torch.empty((n, c, h, w), dtype=torch.float32, device=y.device)
    check(_lib.load().dvc_dual_prior_pass1(C.byref(_src(y, "y")), C.byref(_src(means, "means")),
                                           C.byref(_src(scales, "scales")), C.byref(_dst(out)), n, h, w, _stream()),
          "dvc_dual_prior_pass1")
    return out


def process_with_mask(y: Tensor, means: Tensor, scales: Tensor, mask: Tensor):
    """-> (y_quant, y_hat, means_hat, scales_hat) of the reference's process_with_mask (video_model.py:161-167);
    `mask`: (1, 1, h, w) or (h, w) floats."""
    n, c, h, w = y.shape
    _check_vec(mask, h * w, "process_with_mask mask", device=y.device)
    outs = [torch.empty((n, c, h, w), dtype=torch.float32, device=y.device) for _ in range(4)]
    check(_lib.load().dvc_process_with_mask(C.byref(_src(y, "y")), C.byref(_src(means, "means")),
                                            C.byref(_src(scales, "scales")), mask.data_ptr(), *[C.byref(_dst(o)) for o in outs],
                                            n, h, w, _stream()), "dvc_process_with_mask")
    return tuple(outs)


def dual_prior_pass2(y: Tensor, means: Tensor, scales: Tensor, spatial: Tensor, noise: Optional[Tensor] = None,
                     want=("y_hat", "means_hat", "scales_hat", "likelihood"), scale_table: Optional[Tensor] = None):
    """-> dict with the requested tensors; 'symbols' in `want` also yields 'indexes'
    (both (2, N, C/2, h, w) int32: plane 0 = first-pass sites, plane 1 = second-pass sites)."""
    n, c, h, w = y.shape
    res = {}
    dsts = {}
    for k in ("y_hat", "means_hat", "scales_hat", "likelihood"):
        if k in want:
            res[k] = torch.empty((n, c, h, w), dtype=torch.float32, device=y.device)
            dsts[k] = _dst(res[k])
        else:
            dsts[k] = _null_dst()
    sym = idx = None
    if "symbols" in want:
        if scale_table is None:
            raise ValueError("dual_prior_pass2: scale_table required for symbols/indexes")
        _check_vec(scale_table, None, "dual_prior_pass2 scale_table", device=y.device)
        sym = torch.empty((2, n, c // 2, h, w), dtype=torch.int32, device=y.device)
        idx = torch.empty_like(sym)
        res["symbols"], res["indexes"] = sym, idx
    if noise is not None and not (noise.is_contiguous() and tuple(noise.shape) == (n, c, h, w)):
        raise ValueError("dual_prior_pass2: noise must be contiguous and shaped like y")
    check(_lib.load().dvc_dual_prior_pass2(
        C.byref(_src(y, "y")), C.byref(_src(means, "means")), C.byref(_src(scales, "scales")),
        C.byref(_src(spatial, "spatial")), _ptr(noise), C.byref(dsts["y_hat"]), C.byref(dsts["means_hat"]),
        C.byref(dsts["scales_hat"]), C.byref(dsts["likelihood"]), _ptr(sym), _ptr(idx), _ptr(scale_table),
        0 if scale_table is None else scale_table.numel(), n, h, w, _stream()), "dvc_dual_prior_pass2")
    return res


def dual_prior_dec_indexes(s: Tensor, plane: int, channels: int, scale_table: Tensor) -> Tensor:
    n, _, h, w = s.shape
    _check_vec(scale_table, None, "dual_prior_dec_indexes scale_table", device=s.device)
    idx = torch.empty((n, channels // 2, h, w), dtype=torch.int32, device=s.device)
    check(_lib.load().dvc_dual_prior_dec_indexes(C.byref(_src(s)), plane, idx.data_ptr(), scale_table.data_ptr(),
                                                 scale_table.numel(), n, channels, h, w, _stream()),
          "dvc_dual_prior_dec_indexes")
    return idx


def dual_prior_dec_apply(symbols: Tensor, m: Tensor, plane: int, channels: int,
                         yhat1: Optional[Tensor] = None) -> Tensor:
    n, _, h, w = m.shape
    out = torch.empty((n, channels, h, w), dtype=torch.float32, device=m.device)
    if symbols.dtype != torch.int32 or not symbols.is_contiguous() or symbols.numel() != n * (channels // 2) * h * w:
        raise ValueError("dual_prior_dec_apply: symbols must be contiguous int32 (N, C/2, h, w)")
    y1 = C.byref(_src(yhat1, "yhat1")) if yhat1 is not None else None
    check(_lib.load().dvc_dual_prior_dec_apply(symbols.data_ptr(), C.byref(_src(m)), plane, y1, C.byref(_dst(out)),
                                               n, channels, h, w, _stream()), "dvc_dual_prior_dec_apply")
    return out


def likelihood_bits(lik: Tensor) -> Tensor:
    """(N,) tensor: sum over (C,H,W) of -log2(lik)."""
    n, c, h, w = lik.shape
    lib = _lib.load()
    partial = torch.empty(lib.dvc_bits_scratch_floats(n), dtype=torch.float32, device=lik.device)
    bits = torch.empty(n, dtype=torch.float32, device=lik.device)
    check(lib.dvc_likelihood_bits(C.byref(_src(lik)), n, h, w, partial.data_ptr(), bits.data_ptr(), _stream()),
          "dvc_likelihood_bits")
    return bits


def sq_err_sum(a: Tensor, b: Tensor) -> Tensor:
    n, c, h, w = a.shape
    if tuple(b.shape) != tuple(a.shape):
        raise ValueError("sq_err_sum: shape mismatch")
    lib = _lib.load()
    partial = torch.empty(lib.dvc_bits_scratch_floats(n), dtype=torch.float32, device=a.device)
    sse = torch.empty(n, dtype=torch.float32, device=a.device)
    check(lib.dvc_sq_err_sum(C.byref(_src(a)), C.byref(_src(b)), n, h, w, partial.data_ptr(), sse.data_ptr(),
                             _stream()), "dvc_sq_err_sum")
    return sse


# ------------------------------------------------------------------------------------ gradients
def conv2d_wgrad(srcs: Srcs, grad_pre: Tensor, wshape, stride: int = 1, in_slope: Optional[float] = None,
                 with_bias: bool = False):
    """Weight gradient (OIHW) of conv2d; grad_pre = contiguous (N, Cout, ho, wo) gradient before the
    output activation (see act_grad).  `with_bias`: also return the bias gradient (sum of grad_pre over
    batch and pixels, from the same pass) as a second tensor."""
    if isinstance(srcs, torch.Tensor):
        srcs = (srcs,)
    cout, cin, k, _ = wshape
    n, _, h, w = srcs[0].shape
    if not grad_pre.is_contiguous() or grad_pre.dtype != torch.float32 or grad_pre.size(1) != cout:
        raise ValueError("conv2d_wgrad: grad_pre must be a contiguous fp32 (N, Cout, ho, wo) tensor")
    arr = (DvcSrc * len(srcs))(*[_src(s, f"wgrad src[{i}]") for i, s in enumerate(srcs)])
    if sum(s.size(1) for s in srcs) != cin:
        raise ValueError("conv2d_wgrad: sources do not add up to the weight's input channels")
    lib = _lib.load()
    nfl = check(lib.dvc_conv2d_wgrad_scratch_floats(cout, cin, k, stride, n, h, w), "dvc_conv2d_wgrad_scratch_floats")
    scratch = torch.empty(nfl, dtype=torch.float32, device=grad_pre.device)
    gw = torch.empty((cout, cin, k, k), dtype=torch.float32, device=grad_pre.device)
    gb = torch.empty(cout, dtype=torch.float32, device=grad_pre.device) if with_bias else None
    check(lib.dvc_conv2d_wgrad(arr, len(srcs), n, h, w, 0 if in_slope is None else 1,
                               1.0 if in_slope is None else float(in_slope), grad_pre.data_ptr(), cout, k, stride,
                               scratch.data_ptr(), gw.data_ptr(), gb.data_ptr() if with_bias else None, _stream()),
          "dvc_conv2d_wgrad")
    return (gw, gb) if with_bias else gw


def act_grad(grad: Tensor, act_out: Optional[Tensor], slope: float, pixel_shuffle: bool, conv_shape) -> Tensor:
    n, c, ho, wo = conv_shape
    out = torch.empty((n, c, ho, wo), dtype=torch.float32, device=grad.device)
    ao = C.byref(_src(act_out, "act_out")) if act_out is not None else None
    check(_lib.load().dvc_act_grad(C.byref(_src(grad, "grad")), ao, float(slope), 1 if pixel_shuffle else 0,
                                   out.data_ptr(), n, c, ho, wo, _stream()), "dvc_act_grad")
    return out


def mul_act_grad(grad: Tensor, x: Tensor, slope: float, out: Optional[Tensor] = None,
                 plus: Optional[Tensor] = None) -> Tensor:
    """grad * (x > 0 ? 1 : slope) (+ plus)."""
    n, c, h, w = grad.shape
    if out is None:
        out = torch.empty((n, c, h, w), dtype=torch.float32, device=grad.device)
    if plus is not None and tuple(plus.shape) != (n, c, h, w):
        raise ValueError(f"mul_act_grad: plus shape {tuple(plus.shape)} != {(n, c, h, w)}")
    check(_lib.load().dvc_mul_act_grad_add(C.byref(_src(grad, "grad")), C.byref(_src(x, "x")), float(slope),
                                           C.byref(_src(plus, "plus")) if plus is not None else None,
                                           C.byref(_dst(out)), n, h, w, _stream()), "dvc_mul_act_grad")
    return out


def zero_upsample2(x: Tensor, out_h: int, out_w: int) -> Tensor:
    n, c, h, w = x.shape
    out = torch.empty((n, c, out_h, out_w), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_zero_upsample2(C.byref(_src(x)), C.byref(_dst(out)), n, h, w, out_h, out_w, _stream()),
          "dvc_zero_upsample2")
    return out


def add_scaled(a: Tensor, b: Tensor, scale: Optional[Tensor] = None, c: Optional[Tensor] = None) -> Tensor:
    """a + b * scale[n*C + ch] (+ c)."""
    n, ch, h, w = a.shape
    out = torch.empty((n, ch, h, w), dtype=torch.float32, device=a.device)
    cc = C.byref(_src(c, "c")) if c is not None else None
    check(_lib.load().dvc_add_scaled(C.byref(_src(a, "a")), C.byref(_src(b, "b")), _ptr(scale), cc, C.byref(_dst(out)),
                                     n, h, w, _stream()), "dvc_add_scaled")
    return out


def scale_planes(x: Tensor, scale: Tensor) -> Tensor:
    n, ch, h, w = x.shape
    out = torch.empty((n, ch, h, w), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_scale_planes(C.byref(_src(x)), scale.data_ptr(), C.byref(_dst(out)), n, h, w, _stream()),
          "dvc_scale_planes")
    return out


def plane_dot(a: Tensor, b: Optional[Tensor] = None, sum_batch: bool = False) -> Tensor:
    """(N*C,) plane sums of a*b (or of a); (C,) summed over the batch too when sum_batch."""
    n, ch, h, w = a.shape
    lib = _lib.load()
    scratch = torch.empty(lib.dvc_plane_dot_scratch_floats(n, ch), dtype=torch.float32, device=a.device)
    out = torch.empty(ch if sum_batch else n * ch, dtype=torch.float32, device=a.device)
    bb = C.byref(_src(b, "b")) if b is not None else None
    check(lib.dvc_plane_dot(C.byref(_src(a, "a")), bb, n, h, w, 1 if sum_batch else 0, scratch.data_ptr(),
                            out.data_ptr(), _stream()), "dvc_plane_dot")
    return out


def flow_warp_backward(src: Tensor, flow: Tensor, grad_out: Tensor, want_src=True, want_flow=True):
    n, ch, h, w = src.shape
    gs = torch.zeros((n, ch, h, w), dtype=torch.float32, device=src.device) if want_src else None
    gf = torch.empty((n, 2, h, w), dtype=torch.float32, device=src.device) if want_flow else None
    check(_lib.load().dvc_flow_warp_backward(
        C.byref(_src(src, "src")), C.byref(_src(flow, "flow")), C.byref(_src(grad_out, "grad_out")),
        C.byref(_dst(gs)) if gs is not None else None, C.byref(_dst(gf)) if gf is not None else None,
        n, h, w, _stream()), "dvc_flow_warp_backward")
    return gs, gf


def avg_pool2_backward(grad_out: Tensor, h: int, w: int, scale: float = 1.0) -> Tensor:
    n, ch = grad_out.shape[:2]
    out = torch.empty((n, ch, h, w), dtype=torch.float32, device=grad_out.device)
    check(_lib.load().dvc_avg_pool2_backward(C.byref(_src(grad_out)), C.byref(_dst(out)), n, h, w, float(scale),
                                             _stream()), "dvc_avg_pool2_backward")
    return out


def max_pool2_backward(x: Tensor, grad_out: Tensor) -> Tensor:
    n, ch, h, w = x.shape
    out = torch.empty((n, ch, h, w), dtype=torch.float32, device=x.device)
    check(_lib.load().dvc_max_pool2_backward(C.byref(_src(x, "x")), C.byref(_src(grad_out, "grad_out")),
                                             C.byref(_dst(out)), n, h, w, _stream()), "dvc_max_pool2_backward")
    return out


def bilinear_up2_backward(grad_out: Tensor, h: int, w: int, scale: float = 1.0) -> Tensor:
    n, ch = grad_out.shape[:2]
    out = torch.empty((n, ch, h, w), dtype=torch.float32, device=grad_out.device)
    check(_lib.load().dvc_bilinear_up2_backward(C.byref(_src(grad_out)), C.byref(_dst(out)), n, h, w, float(scale),
                                                _stream()), "dvc_bilinear_up2_backward")
    return out


def eb_backward(x_eval: Tensor, packed: Tensor, grad_lik: Tensor, want_gx: bool = True):
    """-> (grad wrt x_eval | None, grad wrt the raw packed parameters (C, 58))."""
    n, c, h, w = x_eval.shape
    lib = _lib.load()
    gx = torch.empty((n, c, h, w), dtype=torch.float32, device=x_eval.device) if want_gx else None
    scratch = torch.empty(lib.dvc_eb_backward_scratch_floats(c), dtype=torch.float32, device=x_eval.device)
    gp = torch.empty((c, _lib.EB_PARAMS_PER_CHANNEL), dtype=torch.float32, device=x_eval.device)
    check(lib.dvc_eb_backward(C.byref(_src(x_eval, "x_eval")), packed.data_ptr(), C.byref(_src(grad_lik, "grad_lik")),
                              C.byref(_dst(gx)) if gx is not None else None, scratch.data_ptr(), gp.data_ptr(),
                              n, h, w, _stream()), "dvc_eb_backward")
    return gx, gp


def dual_prior_pass1_backward(grad_yhat1: Tensor) -> Tensor:
    n, c, h, w = grad_yhat1.shape
    gy = torch.empty((n, c, h, w), dtype=torch.float32, device=grad_yhat1.device)
    check(_lib.load().dvc_dual_prior_pass1_backward(C.byref(_src(grad_yhat1)), C.byref(_dst(gy)), n, h, w, _stream()),
          "dvc_dual_prior_pass1_backward")
    return gy


def dual_prior_pass2_backward(y: Tensor, means: Tensor, scales: Tensor, spatial: Tensor, noise: Optional[Tensor],
                              grad_yhat: Optional[Tensor], grad_lik: Optional[Tensor]):
    n, c, h, w = y.shape
    dev = y.device
    gy = torch.empty((n, c, h, w), dtype=torch.float32, device=dev)
    gm = torch.empty_like(gy)
    gs = torch.empty_like(gy)
    gsp = torch.empty((n, 2 * c, h, w), dtype=torch.float32, device=dev)
    gyh = C.byref(_src(grad_yhat, "grad_yhat")) if grad_yhat is not None else None
    gl = C.byref(_src(grad_lik, "grad_lik")) if grad_lik is not None else None
    check(_lib.load().dvc_dual_prior_pass2_backward(
        C.byref(_src(y, "y")), C.byref(_src(means, "means")), C.byref(_src(scales, "scales")),
        C.byref(_src(spatial, "spatial")), _ptr(noise), gyh, gl, C.byref(_dst(gy)), C.byref(_dst(gm)),
        C.byref(_dst(gs)), C.byref(_dst(gsp)), n, h, w, _stream()), "dvc_dual_prior_pass2_backward")
    return gy, gm, gs, gsp


def likelihood_bits_backward(lik: Tensor, grad_bits: Tensor) -> Tensor:
    n, c, h, w = lik.shape
    out = torch.empty((n, c, h, w), dtype=torch.float32, device=lik.device)
    check(_lib.load().dvc_likelihood_bits_backward(C.byref(_src(lik)), grad_bits.data_ptr(), C.byref(_dst(out)),
                                                   n, h, w, _stream()), "dvc_likelihood_bits_backward")
    return out


def sq_err_backward(a: Tensor, b: Tensor, grad_sse: Tensor) -> Tensor:
    n, c, h, w = a.shape
    out = torch.empty((n, c, h, w), dtype=torch.float32, device=a.device)
    check(_lib.load().dvc_sq_err_backward(C.byref(_src(a, "a")), C.byref(_src(b, "b")), grad_sse.data_ptr(),
                                          C.byref(_dst(out)), n, h, w, _stream()), "dvc_sq_err_backward")
    return out


# ------------------------------------------------------------------------------------ 8-bit activation checkpoints
class ActCheckpoint(NamedTuple):
    """An activation kept in 8 bits between the forward and the backward pass (format: include/dvc_hip.h): one byte
    per value and one power-of-two scale per 32 adjacent values of a channel plane."""
    codes: Tensor        # uint8 (N, C, blocks * 32), contiguous
    scales: Tensor       # uint8 (N, C, blocks), contiguous
    shape: Tuple[int, int, int, int]
    fmt: str             # "int8" or "e4m3"


def _blocks(h: int, w: int) -> int:
    return (h * w + 31) // 32


def _on_current_device(t: Tensor, name: str):
    if t.get_device() != torch._C._cuda_getDevice():
        raise ValueError(f"{name}: on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


def _sizes_fit(shape, name: str):
    """The library takes sizes as 32-bit integers, into which ctypes would wrap a larger one without a word."""
    if max(shape) >> 31:
        raise ValueError(f"{name}: shape {tuple(shape)}, every size must be below 2^31")


def _ckpt_format(fmt: str) -> int:
    if fmt not in _lib.CKPT_FORMATS:
        raise ValueError(f"unknown checkpoint format {fmt!r} (one of {', '.join(_lib.CKPT_FORMATS)})")
    return _lib.CKPT_FORMATS[fmt]


def _ckpt(ck: ActCheckpoint, name: str, device=None) -> DvcCkpt:
    if not isinstance(ck, ActCheckpoint):
        raise TypeError(f"{name}: expected an ActCheckpoint, got {type(ck)}")
    codes, scales, (n, c, h, w), fmt = ck
    fmt = _ckpt_format(fmt)
    if n < 1 or c < 1 or h < 1 or w < 1:
        raise ValueError(f"{name}: empty shape {tuple(ck.shape)}")
    _sizes_fit(ck.shape, name)
    blocks = n * c * ((h * w + 31) // 32)
    _check_vec(codes, blocks * 32, f"{name} codes" if device is not None else name, dtype=torch.uint8, device=device)
    _check_vec(scales, blocks, name, dtype=torch.uint8, device=codes.device)
    _on_current_device(codes, name)
    return DvcCkpt(codes.data_ptr(), scales.data_ptr(), c, fmt)


def _distinct(t: Tensor, name: str):
    """A destination whose samples or channels share memory (expanded views) would be written by several at once."""
    n, c, h, w = t.shape
    hw, s0, s1 = h * w, t.stride(0), t.stride(1) if t.size(1) > 1 else 0
    samples = n == 1 or s0 >= (c - 1) * s1 + hw or (s0 >= hw and s0 * (n - 1) + hw <= s1)
    if not samples or c > 1 and s1 < hw:
        raise ValueError(f"{name}: overlapping planes (strides {t.stride()})")


def _slope(slope: float, name: str) -> float:
    """LeakyReLU slopes outside [0, 1] do not keep the sign a derivative is read off (nor max(x, slope x))."""
    if not 0.0 <= float(slope) <= 1.0:
        raise ValueError(f"{name}: slope {slope} outside [0, 1]")
    return float(slope)


def act_checkpoint(x: Tensor, slope: Optional[float] = None, fmt: str = "int8") -> ActCheckpoint:
    """The 8-bit checkpoint of x, or of LeakyReLU(slope)(x) (0.0: ReLU), in `fmt`: "int8" (64 to 127
    steps up to the block's largest magnitude) or "e4m3" (4 significant bits each, down to 2^-14 of it).  act_restore() gives
    the values back; the weight gradient (conv2d_wgrad_ckpt) and the input activation's derivative (mul_act_grad_ckpt) read
    the codes themselves."""
    code = _ckpt_format(fmt)
    src = _src(x, "act_checkpoint x")
    _on_current_device(x, "act_checkpoint x")
    _sizes_fit(x.shape, "act_checkpoint x")
    n, c, h, w = x.shape
    blocks = (h * w + 31) // 32
    codes = x.new_empty((n, c, blocks * 32), dtype=torch.uint8)
    scales = x.new_empty((n, c, blocks), dtype=torch.uint8)
    check(_lib.load().dvc_act_checkpoint(C.byref(src), 0 if slope is None else 1,
                                         1.0 if slope is None else _slope(slope, "act_checkpoint"), code, codes.data_ptr(),
                                         scales.data_ptr(), n, h, w, _stream()), "dvc_act_checkpoint")
    return ActCheckpoint(codes, scales, (n, c, h, w), fmt)


def act_restore(ck: ActCheckpoint, out: Optional[Tensor] = None) -> Tensor:
    """The fp32 tensor a checkpoint stands for."""
    c = _ckpt(ck, "act_restore")
    n, ch, h, w = ck.shape
    if out is None:
        out = ck.codes.new_empty(ck.shape, dtype=torch.float32)
        dst = DvcDst(out.data_ptr(), ch * h * w, h * w)
    else:
        if tuple(out.shape) != tuple(ck.shape):
            raise ValueError(f"act_restore: out shape {tuple(out.shape)} != {tuple(ck.shape)}")
        dst = _dst(out)
        _distinct(out, "act_restore out")
        if out.device != ck.codes.device:
            raise ValueError(f"act_restore: out on {out.device}, the checkpoint is on {ck.codes.device}")
    check(_lib.load().dvc_act_restore(C.byref(c), C.byref(dst), n, h, w, _stream()), "dvc_act_restore")
    return out


def act_signs(x: Tensor) -> Tensor:
    """One bit per value, x > 0, as int32 words of 32 adjacent values of a channel plane: (N, C, blocks)."""
    src = _src(x, "act_signs x")
    _on_current_device(x, "act_signs x")
    _sizes_fit(x.shape, "act_signs x")
    n, c, h, w = x.shape
    signs = torch.empty((n, c, _blocks(h, w)), dtype=torch.int32, device=x.device)
    check(_lib.load().dvc_act_signs(C.byref(src), signs.data_ptr(), n, h, w, _stream()), "dvc_act_signs")
    return signs


def act_grad_signs(grad: Tensor, signs: Tensor, slope: float, pixel_shuffle: bool, conv_shape) -> Tensor:
    """act_grad() with the activation's output given by its signs (act_signs of the stored tensor)."""
    n, c, ho, wo = conv_shape
    stored = (n, c // 4, 2 * ho, 2 * wo) if pixel_shuffle else (n, c, ho, wo)
    if tuple(grad.shape) != stored or (pixel_shuffle and c % 4):
        raise ValueError(f"act_grad_signs: grad shape {tuple(grad.shape)} != {stored}")
    src = _src(grad, "act_grad_signs grad")
    _on_current_device(grad, "act_grad_signs grad")
    _sizes_fit(grad.shape, "act_grad_signs grad")
    _check_vec(signs, n * stored[1] * _blocks(*stored[2:]), "act_grad_signs signs", dtype=torch.int32, device=grad.device)
    out = torch.empty((n, c, ho, wo), dtype=torch.float32, device=grad.device)
    check(_lib.load().dvc_act_grad_signs(C.byref(src), signs.data_ptr(), float(slope), 1 if pixel_shuffle else 0,
                                         out.data_ptr(), n, c, ho, wo, _stream()), "dvc_act_grad_signs")
    return out


def mul_act_grad_ckpt(grad: Tensor, ck: ActCheckpoint, slope: float, out: Optional[Tensor] = None,
                      plus: Optional[Tensor] = None) -> Tensor:
    """mul_act_grad() with x given by its checkpoint: grad * (x > 0 ? 1 : slope) (+ plus)."""
    n, c, h, w = grad.shape
    if tuple(ck.shape) != (n, c, h, w):
        raise ValueError(f"mul_act_grad_ckpt: checkpoint shape {tuple(ck.shape)} != {(n, c, h, w)}")
    if out is None:
        out = torch.empty((n, c, h, w), dtype=torch.float32, device=grad.device)
    for t, name in ((out, "out"), (plus, "plus")):
        if t is not None and (tuple(t.shape) != (n, c, h, w) or t.device != grad.device):
            raise ValueError(f"mul_act_grad_ckpt: {name} {tuple(t.shape)} on {t.device} does not match grad {(n, c, h, w)}")
    _check4(out, "mul_act_grad_ckpt out")
    _distinct(out, "mul_act_grad_ckpt out")
    check(_lib.load().dvc_mul_act_grad_ckpt(C.byref(_src(grad, "grad")), C.byref(_ckpt(ck, "mul_act_grad_ckpt", grad.device)),
                                            float(slope), C.byref(_src(plus, "plus")) if plus is not None else None,
                                            C.byref(_dst(out)), n, h, w, _stream()), "dvc_mul_act_grad_ckpt")
    return out


def conv2d_wgrad_ckpt(cks: Union[ActCheckpoint, Sequence[ActCheckpoint]], grad_pre: Tensor, wshape, stride: int = 1,
                      with_bias: bool = False):
    """conv2d_wgrad() with the (activated, concatenated) sources given by checkpoints of one format."""
    if isinstance(cks, ActCheckpoint):
        cks = (cks,)
    if not 1 <= len(cks) <= _lib.DVC_MAX_SRC:
        raise ValueError(f"conv2d_wgrad_ckpt: {len(cks)} sources (1..{_lib.DVC_MAX_SRC} supported)")
    cout, cin, k, k2 = wshape
    n, _, h, w = cks[0].shape
    for i, ck in enumerate(cks):
        if (ck.shape[0], ck.shape[2], ck.shape[3]) != (n, h, w) or ck.fmt != cks[0].fmt:
            raise ValueError(f"conv2d_wgrad_ckpt: source {i} ({tuple(ck.shape)}, {ck.fmt}) does not match {(n, '*', h, w)}, {cks[0].fmt}")
    if sum(ck.shape[1] for ck in cks) != cin or k != k2:
        raise ValueError(f"conv2d_wgrad_ckpt: weight shape {tuple(wshape)} does not match {sum(ck.shape[1] for ck in cks)} input channels")
    pad = k // 2
    want = (n, cout, (h + 2 * pad - k) // stride + 1, (w + 2 * pad - k) // stride + 1)
    if tuple(grad_pre.shape) != want:
        raise ValueError(f"conv2d_wgrad_ckpt: grad_pre shape {tuple(grad_pre.shape)} != {want}")
    _check_vec(grad_pre, None, "conv2d_wgrad_ckpt grad_pre", device=cks[0].codes.device)
    arr = (DvcCkpt * len(cks))(*[_ckpt(ck, f"conv2d_wgrad_ckpt source {i}", grad_pre.device) for i, ck in enumerate(cks)])
    lib = _lib.load()
    nfl = check(lib.dvc_conv2d_wgrad_ckpt_scratch_floats(cout, cin, k, stride, n, h, w), "dvc_conv2d_wgrad_ckpt_scratch_floats")
    scratch = torch.empty(nfl, dtype=torch.float32, device=grad_pre.device)
    gw = torch.empty((cout, cin, k, k), dtype=torch.float32, device=grad_pre.device)
    gb = torch.empty(cout, dtype=torch.float32, device=grad_pre.device) if with_bias else None
    check(lib.dvc_conv2d_wgrad_ckpt(arr, len(cks), n, h, w, grad_pre.data_ptr(), cout, k, stride, scratch.data_ptr(),
                                    gw.data_ptr(), _ptr(gb), _stream()), "dvc_conv2d_wgrad_ckpt")
    return (gw, gb) if with_bias else gw


# ------------------------------------------------------------------------------------ symbols under given logits
class SymbolLogProbs(NamedTuple):
    """log_prob / entropy: fp32, shaped like the symbols; stats: (2, sites), for symbol_log_probs_backward;
    top_log_prob / top_symbol: fp32 / int32 (N, C * top, h, w) (rows: (N, top)), or None."""
    log_prob: Tensor
    entropy: Tensor
    stats: Tensor
    top_log_prob: Optional[Tensor]
    top_symbol: Optional[Tensor]


_LOGIT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _logits(logits: Tensor, symbols: Tensor, name: str):
    """-> (DvcLogits or None without sites, n, groups, h, w, 2-D?)"""
    if not isinstance(logits, torch.Tensor) or not isinstance(symbols, torch.Tensor):
        raise TypeError(f"{name}: expected tensors, got {type(logits)} and {type(symbols)}")
    if not logits.is_cuda:
        raise _lib.DvcError(f"{name} logits: tensor is on {logits.device}; the HIP path needs a GPU tensor (no CPU fallback)")
    dtype = _LOGIT_TYPES.get(logits.dtype)
    if dtype is None:
        raise TypeError(f"{name} logits: expected fp32, bf16 or fp16, got {logits.dtype}")
    shape, site, strides = logits.shape, symbols.shape, logits.stride()
    rows = len(shape) == 2
    if rows and len(site) == 1:
        (n, v), groups, h, w = shape, 1, 1, 1
        match = site[0] == n
    elif len(shape) == 4 and len(site) == 4:
        n, groups, h, w = site
        v = shape[1] // groups if groups else 0
        match = shape[0] == n and shape[1] == groups * v and shape[2] == h and shape[3] == w
        if w > 1 and strides[3] != 1 or h > 1 and strides[2] != w:
            raise ValueError(f"{name} logits: rows must be contiguous (strides {strides})")
    else:
        raise ValueError(f"{name}: expected logits (N, C * classes, h, w) with symbols (N, C, h, w), or (N, classes) with (N,), "
                         f"got {tuple(shape)} with {tuple(site)}")
    if not match or v < 1:
        raise ValueError(f"{name}: symbols {tuple(site)} do not match logits {tuple(shape)}")
    _check_vec(symbols, None, name, dtype=torch.int32, device=logits.device)
    _on_current_device(logits, name)
    _sizes_fit(shape, f"{name} logits")
    if n * h * w == 0:
        return None, n, groups, h, w, rows
    return DvcLogits(logits.data_ptr(), strides[0], strides[1] if shape[1] > 1 else h * w, groups, v, dtype, 0), n, groups, h, w, rows


def symbol_log_probs(logits: Tensor, symbols: Tensor, top: int = 0) -> SymbolLogProbs:
    """Log probabilities (nats) of given symbols under softmax(logits), the distributions' entropies and, for `top` > 0
    (at most 16), the `top` most likely classes in falling order (equal logits: the lower class first).

    logits (N, C * classes, h, w), symbols (N, C, h, w) int32: channel c's classes are the channels c * classes ...;
    or rows, logits (N, classes), symbols (N,).  fp32, bf16 or fp16 logits with free batch and class strides; sums are
    fp32 (over more than 256 classes a lane of the GPU, 64 bits).  A symbol < 0 means "none here" (log probability 0); one
    past the last class gives NaN.  Classes that may not occur have logits of -inf; a site without any other has log
    probability -inf and entropy 0.  Rows of more than 1024 classes: below 2^24 of them, of more than 256: below 2^26."""
    lg, n, groups, h, w, rows = _logits(logits, symbols, "symbol_log_probs")
    classes = logits.size(1) // groups
    top = int(top)
    if not 0 <= top <= min(_lib.MAX_TOP, classes):
        raise ValueError(f"symbol_log_probs: top={top} (0..{_lib.MAX_TOP}, at most the {classes} classes)")
    site = tuple(symbols.shape)
    log_prob = symbols.new_empty(site, dtype=torch.float32)
    entropy = torch.empty_like(log_prob)
    stats = log_prob.new_empty((2, n * groups * h * w))
    tl = ts = None
    if top:
        shape = (n, top) if rows else (n, groups * top, h, w)
        tl = log_prob.new_empty(shape)
        ts = symbols.new_empty(shape)
    if lg is not None:
        lib = _lib.load()
        nfl = 0
        if h * w == 1:      # only rows are ever cut into parts
            nfl = check(lib.dvc_symbol_log_probs_scratch_floats(C.byref(lg), top, n, h, w), "dvc_symbol_log_probs_scratch_floats")
        scratch = log_prob.new_empty(nfl) if nfl else None
        check(lib.dvc_symbol_log_probs(C.byref(lg), symbols.data_ptr(), top, log_prob.data_ptr(), entropy.data_ptr(),
                                       stats.data_ptr(), _ptr(tl), _ptr(ts), _ptr(scratch), n, h, w, _stream()), "dvc_symbol_log_probs")
    return SymbolLogProbs(log_prob, entropy, stats, tl, ts)


def symbol_log_probs_backward(logits: Tensor, symbols: Tensor, stats: Tensor, entropy: Tensor,
                              grad_log_prob: Optional[Tensor], grad_entropy: Optional[Tensor]) -> Tensor:
    """The gradient with respect to the logits (contiguous, their type) of what symbol_log_probs returned."""
    lg, n, groups, h, w, rows = _logits(logits, symbols, "symbol_log_probs_backward")
    dev, sites = logits.device, symbols.numel()
    _check_vec(stats, 2 * sites, "symbol_log_probs_backward stats", device=dev)
    _check_vec(entropy, sites, "symbol_log_probs_backward entropy", device=dev)
    _check_vec(grad_log_prob, sites, "symbol_log_probs_backward grad_log_prob", device=dev)
    _check_vec(grad_entropy, sites, "symbol_log_probs_backward grad_entropy", device=dev)
    out = torch.empty(tuple(logits.shape), dtype=logits.dtype, device=dev)
    if lg is not None:
        check(_lib.load().dvc_symbol_log_probs_backward(C.byref(lg), symbols.data_ptr(), stats.data_ptr(), entropy.data_ptr(),
                                                        _ptr(grad_log_prob), _ptr(grad_entropy), out.data_ptr(), n, h, w, _stream()),
              "dvc_symbol_log_probs_backward")
    return out
