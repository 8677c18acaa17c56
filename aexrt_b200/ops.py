"""Tensor-level wrappers of the C ABI (torch is used only for device memory and streams).

The functions mirror the steps of the reference's int8 conv branch
(``record_replay_conv``, native/aexrt_d3d12_runtime.cpp:23935-24318):

* :func:`quantize_conv_weight_int8` — layout-8 weight quantizer (engine.py:2418-2465)
* :func:`act_amax`                   — aexrt_int8_quant_zero + _amax (runtime.cpp:3159-3275)
* :func:`act_quantize`               — aexrt_int8_quant_pack[_pg] (runtime.cpp:3277-3361)
* :class:`ConvPlan` / :meth:`ConvPlan.run` — prequant conv kernels 51/52/53 (runtime.cpp:4614-4923)
* :func:`conv_w8a8_layer`            — the whole branch: amax -> quantize -> conv
* :func:`yolo_nms_topk`              — decode-filter + NMS + top-k (runtime.cpp:27104-27219)

Every device call goes through ``libaexrt_b200.so``; there is no CPU or
PyTorch fallback for any of them.
"""
from __future__ import annotations

import contextlib
import ctypes
import struct
from dataclasses import dataclass
from typing import Optional, Tuple

import numpy as np

from . import _native
from ._native import AexrtB200ConvPlanInfo, AexrtConv2DDesc, check

KIND_CONV = 1
KIND_CONV_SILU = 2
PLAN_FLAG_INT8_PERGROUP = 1 << 4
PLAN_FLAG_QUANT_ON_LOAD = 1 << 8
LAYOUT_NHWC_F16 = 0
LAYOUT_NCHW_F16 = 1
LAYOUT_NCHW_F32 = 2
SCALE_PER_TENSOR = 0
SCALE_PG16 = 1
NMS_MARK = 0
NMS_GREEDY = 1
NMS_CTAS_SHIFT = 8  # AEXRT_B200_NMS_CTAS_SHIFT: mode bits 8-11 = CTAs per image


def _torch():
    import torch

    return torch


def _stream(stream=None) -> int:
    torch = _torch()
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    return int(getattr(stream, "cuda_stream", stream))


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def quantize_conv_weight_int8(weight: np.ndarray, fp16_engine: bool = False) -> Tuple[np.ndarray, np.ndarray]:
    """Layout-8 weight quantization on the host (bit-identical to engine.py:2447-2457)."""
    w = np.ascontiguousarray(weight, dtype=np.float32)
    oc = w.shape[0]
    kk = int(np.prod(w.shape[2:])) if w.ndim > 2 else 1
    ic = w.shape[1] if w.ndim > 1 else 1
    codes = np.empty((oc, ic * kk), dtype=np.int8)
    scale = np.empty(oc, dtype=np.float32)
    check(_native.load().aexrt_b200_quantize_conv_weight_int8(
        w.ctypes.data, oc, ic, kk, int(bool(fp16_engine)), codes.ctypes.data, scale.ctypes.data), "quantize weights")
    return codes, scale


def conv_desc(n, ic, h, w, oc, k, s, p) -> AexrtConv2DDesc:
    oh = (h + 2 * p - k) // s + 1
    ow = (w + 2 * p - k) // s + 1
    return AexrtConv2DDesc(n, ic, h, w, oc, oh, ow, k, k, s, s, p, p, 1, 1, 1)


def kernel_id_for(k: int, s: int) -> int:
    """The reference's int8 kernel ids: 51 = 1x1, 52 = 3x3 s1, 53 = 3x3 s2 (runtime.cpp:8881-8940)."""
    if k == 1 and s == 1:
        return 51
    if k == 3 and s == 1:
        return 52
    if k == 3 and s == 2:
        return 53
    raise ValueError(f"no int8 kernel for k={k} s={s}")


def amax_groups_tensor(n: int, groups: int, device="cuda"):
    torch = _torch()
    return torch.zeros((n, groups), dtype=torch.int32, device=device)


def act_amax(x, layout: int = LAYOUT_NCHW_F16, c: Optional[int] = None, ldc: Optional[int] = None, coff: int = 0,
             out=None, groups_total: Optional[int] = None, group_offset: int = 0, zero_first: bool = True, stream=None):
    """Per-image amax of |x| per 16-channel group, as uint32 float bits in an int32 tensor [N, G]."""
    if layout == LAYOUT_NHWC_F16:
        n, h, w, cc = x.shape
        c = c or (cc - coff)
        ldc = ldc or cc
    else:
        n, c, h, w = x.shape
        ldc = c
    g = (c + 15) // 16
    groups_total = groups_total or g
    if out is None:
        out = amax_groups_tensor(n, groups_total, x.device)
    check(_native.load().aexrt_b200_act_amax_f16(
        x.data_ptr(), n, c, h, w, layout, ldc, coff, out.data_ptr(), groups_total, group_offset, int(zero_first),
        _stream(stream)), "act_amax")
    return out


def packed_act_shape(n: int, c: int, h: int, w: int, stride: int = 1):
    hp = h + (h & 1 if stride == 2 else 0)
    wp = w + (w & 1 if stride == 2 else 0)
    return (n, (c + 15) // 16, hp, wp, 16)


def act_quantize(x, amax_groups, mode: int = SCALE_PER_TENSOR, layout: int = LAYOUT_NCHW_F16, consumer_stride: int = 1,
                 c: Optional[int] = None, ldc: Optional[int] = None, coff: int = 0, group_offset: int = 0,
                 q_out=None, rec_out=None, stream=None):
    """int8 codes in the slab16 layout + per-image scale record [N, 1 + slabs] (fp32 amax values)."""
    torch = _torch()
    if layout == LAYOUT_NHWC_F16:
        n, h, w, cc = x.shape
        c = c or (cc - coff)
        ldc = ldc or cc
    else:
        n, c, h, w = x.shape
        ldc = c
    shape = packed_act_shape(n, c, h, w, consumer_stride)
    if q_out is None:
        q_out = torch.empty(shape, dtype=torch.int8, device=x.device)
    if rec_out is None:
        rec_out = torch.empty((n, 1 + shape[1]), dtype=torch.float32, device=x.device)
    check(_native.load().aexrt_b200_act_quantize_f16(
        x.data_ptr(), n, c, h, w, layout, ldc, coff, amax_groups.data_ptr(), amax_groups.shape[1], group_offset, mode,
        consumer_stride, q_out.data_ptr(), rec_out.data_ptr(), _stream(stream)), "act_quantize")
    return q_out, rec_out


def act_amax_quantize(x, mode: int = SCALE_PER_TENSOR, amax_out=None, q_out=None, rec_out=None, stream=None):
    """Standalone amax + quantize of an fp16 NCHW tensor for a stride-1 consumer in one call:
    returns (codes slab16, scale record, amax slots [n, ceil(c/16)])."""
    torch = _torch()
    n, c, h, w = x.shape
    groups = (c + 15) // 16
    if amax_out is None:
        amax_out = torch.empty((n, groups), dtype=torch.int32, device=x.device)
    if q_out is None:
        q_out = torch.empty(packed_act_shape(n, c, h, w, 1), dtype=torch.int8, device=x.device)
    if rec_out is None:
        rec_out = torch.empty((n, 1 + groups), dtype=torch.float32, device=x.device)
    check(_native.load().aexrt_b200_act_amax_quantize_f16(x.data_ptr(), n, c, h, w, mode, amax_out.data_ptr(),
                                                          amax_out.shape[1], 0, q_out.data_ptr(), rec_out.data_ptr(),
                                                          _stream(stream)), "act_amax_quantize")
    return q_out, rec_out, amax_out


def act_status() -> int:
    """Reads and clears the activation kernels' status word of the current device."""
    v = ctypes.c_uint32(0)
    check(_native.load().aexrt_b200_act_status(ctypes.byref(v)), "act_status")
    return v.value


def pack_f16(x, layout: int = LAYOUT_NHWC_F16, consumer_stride: int = 1, c: Optional[int] = None,
             ldc: Optional[int] = None, coff: int = 0, out=None, stream=None):
    """fp16 slab8 repack [N, ceil(C/8), Hp, Wp, 8] for the fp16 convs."""
    torch = _torch()
    if layout == LAYOUT_NHWC_F16:
        n, h, w, cc = x.shape
        c = c or (cc - coff)
        ldc = ldc or cc
    else:
        n, c, h, w = x.shape
        ldc = c
    hp = h + (h & 1 if consumer_stride == 2 else 0)
    wp = w + (w & 1 if consumer_stride == 2 else 0)
    if out is None:
        out = torch.empty((n, (c + 7) // 8, hp, wp, 8), dtype=torch.float16, device=x.device)
    check(_native.load().aexrt_b200_pack_f16(x.data_ptr(), n, c, h, w, layout, ldc, coff, consumer_stride,
                                             out.data_ptr(), _stream(stream)), "pack_f16")
    return out


@dataclass
class PlanInfo:
    kernel_id: int
    flags: int
    kind: int
    is_f16: bool
    tile_w: int
    tile_h: int
    block_n: int
    k_slots: int
    stages: int
    smem_bytes: int
    grid_m: int
    grid_n: int
    in_hp: int
    in_wp: int
    grid: int = 0
    variant: int = 0
    pitch: int = 0
    image_input: int = 0
    quant_on_load: int = 0
    staged_out: int = 0

    @staticmethod
    def from_c(i: AexrtB200ConvPlanInfo) -> "PlanInfo":
        return PlanInfo(i.kernel_id, i.flags, i.kind, bool(i.is_f16), i.tile_w, i.tile_h, i.block_n, i.k_slots,
                        i.stages, i.smem_bytes, i.grid_m, i.grid_n, i.in_hp, i.in_wp, i.grid, i.variant, i.pitch,
                        i.image_input, i.quant_on_load, i.staged_out)


class ConvPlan:
    """A device-resident conv plan: one reference kernel-plan command (kind, kernel, flags).

    ``ConvPlan.int8(...)`` takes layout-8 codes/scales (the reference's packed
    weights) and builds kernel 51/52/53 per ``can_use_conv_int8``;
    ``ConvPlan.fp16(...)`` builds the fp16 conv used for the stem and head.
    """

    def __init__(self, handle: int, desc: AexrtConv2DDesc, is_f16: bool):
        self._h = handle
        self.desc = desc
        self.is_f16 = is_f16
        self.info = self._info()

    @classmethod
    def int8(cls, n, ic, h, w, oc, k, s, codes, w_scale, bias, silu=True, pg16=False, block_n=0,
             quant_on_load=False):
        p = k // 2
        desc = conv_desc(n, ic, h, w, oc, k, s, p)
        codes = np.ascontiguousarray(codes, dtype=np.int8)
        w_scale = np.ascontiguousarray(w_scale, dtype=np.float32)
        bias = np.ascontiguousarray(bias, dtype=np.float32)
        flags = (PLAN_FLAG_INT8_PERGROUP if pg16 else 0) | (PLAN_FLAG_QUANT_ON_LOAD if quant_on_load else 0)
        h_ = _native.load().aexrt_b200_conv_plan_create(
            ctypes.byref(desc), KIND_CONV_SILU if silu else KIND_CONV, kernel_id_for(k, s), flags, codes.ctypes.data,
            w_scale.ctypes.data, bias.ctypes.data, block_n)
        if not h_:
            raise _native.AexrtError("conv_plan_create failed: " + _native.last_error())
        return cls(h_, desc, False)

    @classmethod
    def fp16(cls, n, ic, h, w, oc, k, s, weight, bias, silu=True, block_n=0):
        p = k // 2
        desc = conv_desc(n, ic, h, w, oc, k, s, p)
        weight = np.ascontiguousarray(weight, dtype=np.float32)
        bias = np.ascontiguousarray(bias, dtype=np.float32)
        h_ = _native.load().aexrt_b200_conv_plan_create_f16(
            ctypes.byref(desc), KIND_CONV_SILU if silu else KIND_CONV, weight.ctypes.data, bias.ctypes.data, block_n)
        if not h_:
            raise _native.AexrtError("conv_plan_create_f16 failed: " + _native.last_error())
        return cls(h_, desc, True)

    def _info(self) -> PlanInfo:
        i = AexrtB200ConvPlanInfo()
        check(_native.load().aexrt_b200_conv_plan_info(self._h, ctypes.byref(i)), "conv_plan_info")
        return PlanInfo.from_c(i)

    @property
    def out_shape(self):
        d = self.desc
        return (d.batch, d.out_h, d.out_w, d.out_channels)

    def run(self, x, rec=None, out=None, out_coff: int = 0, residual=None, res_coff: int = 0, amax_out=None,
            amax_goff: int = 0, acc_dump=None, stream=None):
        """Launches the conv; ``out`` is an fp16 NHWC tensor whose last dim is the channel stride."""
        torch = _torch()
        if out is None:
            out = torch.empty(self.out_shape, dtype=torch.float16, device=x.device)
        out_ldc = out.shape[-1]
        res_ldc = residual.shape[-1] if residual is not None else 0
        amax_stride = amax_out.shape[-1] if amax_out is not None else 0
        lib = _native.load()
        if self.is_f16:
            check(lib.aexrt_b200_conv_f16(self._h, x.data_ptr(), _ptr(residual), res_ldc, res_coff, out.data_ptr(),
                                          out_ldc, out_coff, _ptr(amax_out), amax_stride, amax_goff, _stream(stream)),
                  "conv_f16")
        else:
            check(lib.aexrt_b200_conv_w8a8(self._h, x.data_ptr(), rec.data_ptr(), _ptr(residual), res_ldc, res_coff,
                                           out.data_ptr(), out_ldc, out_coff, _ptr(amax_out), amax_stride, amax_goff,
                                           _ptr(acc_dump), _stream(stream)), "conv_w8a8")
        return out

    def run_sources(self, srcs, out=None, out_coff: int = 0, residual=None, res_coff: int = 0, amax_out=None,
                    amax_goff: int = 0, acc_dump=None, stream=None, device=None):
        """Quantize-on-load plans: the conv reads the fp16 NHWC sources (a ctypes array of
        AexrtB200ActSource with their amax slots) and quantizes them in shared memory."""
        torch = _torch()
        if out is None:
            out = torch.empty(self.out_shape, dtype=torch.float16, device=device or "cuda")
        res_ldc = residual.shape[-1] if residual is not None else 0
        amax_stride = amax_out.shape[-1] if amax_out is not None else 0
        check(_native.load().aexrt_b200_conv_w8a8_sources(self._h, srcs, len(srcs), _ptr(residual), res_ldc, res_coff,
                                                          out.data_ptr(), out.shape[-1], out_coff, _ptr(amax_out),
                                                          amax_stride, amax_goff, _ptr(acc_dump), _stream(stream)),
              "conv_w8a8_sources")
        return out

    def run_nhwc(self, x, x_coff: int = 0, out=None, out_coff: int = 0, residual=None, res_coff: int = 0,
                 amax_out=None, amax_goff: int = 0, stream=None):
        """fp16 stride-1 halo plans: the conv reads channels x_coff .. x_coff + in_channels of the fp16
        NHWC tensor ``x`` directly (no slab8 copy)."""
        torch = _torch()
        if out is None:
            out = torch.empty(self.out_shape, dtype=torch.float16, device=x.device)
        amax_stride = amax_out.shape[-1] if amax_out is not None else 0
        res_ldc = residual.shape[-1] if residual is not None else 0
        check(_native.load().aexrt_b200_conv_f16_nhwc(self._h, x.data_ptr(), x.shape[-1], x_coff, _ptr(residual),
                                                      res_ldc, res_coff, out.data_ptr(), out.shape[-1], out_coff,
                                                      _ptr(amax_out), amax_stride, amax_goff, _stream(stream)),
              "conv_f16_nhwc")
        return out

    def run_image(self, images, out=None, out_coff: int = 0, amax_out=None, amax_goff: int = 0, stream=None):
        """The image stem: fp16 or fp32 NCHW ``images`` straight into the fp16 NHWC ``out``
        (plans with info.image_input)."""
        torch = _torch()
        if out is None:
            out = torch.empty(self.out_shape, dtype=torch.float16, device=images.device)
        amax_stride = amax_out.shape[-1] if amax_out is not None else 0
        layout = LAYOUT_NCHW_F16 if images.dtype == torch.float16 else LAYOUT_NCHW_F32
        check(_native.load().aexrt_b200_conv_f16_image(self._h, images.data_ptr(), layout, out.data_ptr(),
                                                       out.shape[-1], out_coff, _ptr(amax_out), amax_stride,
                                                       amax_goff, _stream(stream)), "conv_f16_image")
        return out

    def status(self) -> int:
        v = ctypes.c_uint32(0)
        check(_native.load().aexrt_b200_conv_status(self._h, ctypes.byref(v)), "conv_status")
        return v.value

    def close(self):
        if self._h:
            _native.load().aexrt_b200_conv_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def conv_w8a8_layer(plan: ConvPlan, x_nhwc, mode: int = SCALE_PER_TENSOR, residual=None, out=None, amax_out=None,
                    stream=None):
    """The reference's int8 conv branch on an fp16 NHWC input: amax -> quantize -> conv."""
    d = plan.desc
    amax = act_amax(x_nhwc, LAYOUT_NHWC_F16, stream=stream)
    q, rec = act_quantize(x_nhwc, amax, mode, LAYOUT_NHWC_F16, consumer_stride=d.stride_h, stream=stream)
    return plan.run(q, rec, out=out, residual=residual, amax_out=amax_out, stream=stream)


def yolo_nms_topk(output0, nc: int, conf: float = 0.25, iou: float = 0.45, max_candidates: int = 512,
                  max_detections: int = 100, mode: int = NMS_MARK, has_objectness: bool = False,
                  channels_last: bool = False, dets=None, counts=None, stream=None, ctas_per_image: int = 0):
    """Detections of a batch of fp32 output0 tensors ([n, 4 + nc, anchors], or [n, anchors, 4 + nc]
    when `channels_last`): returns (dets [n, max_detections, 6] fp32 rows x1, y1, x2, y2, score,
    class; counts [n] int32).  Rows at and beyond counts[i] are zero.

    Defaults are the reference model's (runtime.cpp:551-561): 512 candidates, 100 detections,
    conf 0.25, IoU 0.45, the GPU path's NMS rule; ``mode=NMS_GREEDY`` gives yolo_postprocess's.
    ``ctas_per_image`` (0 automatic, else 1, 2, 4 or 8): the thread-block cluster that shares one
    image's pair tests; the detections do not depend on it."""
    torch = _torch()
    n = output0.shape[0]
    channels = output0.shape[2] if channels_last else output0.shape[1]
    anchors = output0.shape[1] if channels_last else output0.shape[2]
    if dets is None:
        dets = torch.zeros((n, max_detections, 6), dtype=torch.float32, device=output0.device)
    if counts is None:
        counts = torch.zeros((n,), dtype=torch.int32, device=output0.device)
    check(_native.load().aexrt_b200_yolo_nms_topk(
        output0.data_ptr(), n, channels, anchors, nc, int(has_objectness), 2 if channels_last else 1, conf, iou,
        max_candidates, max_detections, mode | (ctas_per_image << NMS_CTAS_SHIFT), dets.data_ptr(), counts.data_ptr(),
        _stream(stream)), "yolo_nms_topk")
    return dets, counts


# ---------------------------------------------------------------- attention over token sequences
DTYPE_F16 = 0
DTYPE_BF16 = 1
ATTENTION_BAD_PAGE = 1  # attention_status bits
ATTENTION_TIMEOUT = 2
# AexrtB200AttentionDesc as bytes: packing takes a fraction of filling the ctypes structure field by field, and
# these calls are short
_DESC = struct.Struct("@9If4I10Q")
assert _DESC.size == ctypes.sizeof(_native.AexrtB200AttentionDesc)


def _dtype16(t, what: str, torch) -> int:
    dtype = t.dtype
    if dtype is torch.bfloat16:
        return DTYPE_BF16
    if dtype is torch.float16:
        return DTYPE_F16
    raise ValueError(f"{what}: float16 or bfloat16 tensors, not {dtype}")


def _pack(what: str, *fields) -> bytes:
    """An AexrtB200AttentionDesc of these fields (those behind struct_size)."""
    try:
        return _DESC.pack(_DESC.size, *fields)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"{what}: a size or the scale is out of range ({e})") from None


def _entries(t, what: str, name: str) -> int:
    """The entries of a vector."""
    if t.dim() != 1:
        raise ValueError(f"{what}: {name} must have one dimension")
    return t.shape[0]


def _heads(t, what: str, name: str, dims: int):
    """Shape and strides of a [..., heads, head_dim] tensor with contiguous heads (the library ignores the stride of a
    dimension of size 1, which torch leaves arbitrary)."""
    shape, strides = t.shape, t.stride()
    if len(shape) != dims:
        raise ValueError(f"{what}: {name} must have {dims} dimensions")
    if strides[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{what}: each head of {name} must be contiguous")
    return shape, strides


def _index(t, what: str, name: str, size: int, int32) -> int:
    """Checks a contiguous int32 vector and returns its address."""
    if t.dtype is not int32 or t.dim() != 1 or t.numel() != size or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous int32 tensor of {size} entries")
    return t.data_ptr()


def _table(t, what: str, rows: int, int32):
    """Checks a block table and returns (address, columns, stride of its rows)."""
    shape, strides = t.shape, t.stride()
    if t.dtype is not int32 or len(shape) != 2 or shape[0] != rows or (strides[1] != 1 and shape[1] > 1):
        raise ValueError(f"{what}: block_table must be int32 [{rows}, columns] with contiguous rows")
    return t.data_ptr(), shape[1], strides[0] if rows > 1 else shape[1]


def _call(fn, what: str, torch, tensors, stream, args):
    """Calls a C entry point on the tensors' device (which must be one CUDA device) with `args` and the stream."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != index or index < 0):
            raise ValueError(f"{what}: CUDA tensors on one device, not on {tensors[0].device} and {t.device}")
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _call(fn, what, torch, tensors, stream, args)
    # the current stream's handle as torch keeps it, without a Stream object around it (3 us)
    handle = torch._C._cuda_getCurrentRawStream(index) if stream is None else _stream(stream)
    return fn(*args, handle)


def _allocating(torch, stream, device):
    """The context in which a call on `stream` allocates: that stream's own, since memory from the current one's pool may
    still be used by work that is queued there.  (Tensors that are not on a GPU are refused by the call.)"""
    if stream is None or device.type != "cuda":
        return contextlib.nullcontext()
    return torch.cuda.stream(stream if isinstance(stream, torch.cuda.Stream)
                             else torch.cuda.ExternalStream(_stream(stream), device=device))


def _made(torch, stream, shape, dtype, device):
    """A tensor that a call on `stream` writes and returns: not reused before both that stream and the current one have
    passed its last use."""
    with _allocating(torch, stream, device):
        t = torch.empty(shape, dtype=dtype, device=device)
    if stream is not None and t.is_cuda:
        t.record_stream(torch.cuda.current_stream(device))
    return t


def _outputs(what: str, torch, q, q_shape, out, lse, return_lse, stream):
    """The outputs given or made: (out, its strides, lse)."""
    if out is None:
        out = _made(torch, stream, q_shape, q.dtype, q.device)
    shape, strides = _heads(out, what, "out", 3)
    if shape != q_shape or out.dtype is not q.dtype:
        raise ValueError(f"{what}: out must have q's shape and type")
    if lse is None:
        if return_lse:
            lse = _made(torch, stream, q_shape[:2], torch.float32, q.device)
    elif lse.dtype is not torch.float32 or lse.dim() != 2 or lse.shape != q_shape[:2] or not lse.is_contiguous():
        raise ValueError(f"{what}: lse must be a contiguous float32 tensor [tokens, heads]")
    return out, strides, lse


def attention_packed(q, k, v, cu_q, cu_k, causal: bool = True, scale: Optional[float] = None, out=None, lse=None,
                     return_lse: bool = False, stream=None):
    """Softmax attention over packed sequences: ``q`` [q_tokens, q_heads, d], ``k`` and ``v`` [k_tokens, kv_heads, d]
    (fp16 or bf16, any token and head strides), sequence s in rows cu_q[s] .. cu_q[s + 1] and
    cu_k[s] .. cu_k[s + 1] (int32 on the device).  Causal: the last query token sees every key of its
    sequence.  ``scale`` defaults to d ** -0.5.  Returns out, or (out, lse) with ``return_lse`` or a
    given ``lse`` (fp32 [q_tokens, q_heads], natural logarithm).  Rows behind the last sequence are left as they were."""
    what, torch = "attention_packed", _torch()
    q_shape, qs = _heads(q, what, "q", 3)
    tokens, heads, dim = q_shape
    k_shape, ks = _heads(k, what, "k", 3)
    v_shape, vs = _heads(v, what, "v", 3)
    out, os_, lse = _outputs(what, torch, q, q_shape, out, lse, return_lse, stream)
    if k_shape != v_shape or k_shape[2] != dim or not q.dtype is k.dtype is v.dtype:
        raise ValueError(f"{what}: k and v must have one shape, and q's type and head size")
    num_seqs = _entries(cu_q, what, "cu_q") - 1
    if num_seqs < 0:
        raise ValueError(f"{what}: cu_q must have at least one entry")
    desc = _pack(what, _dtype16(q, what, torch), num_seqs, tokens, 0, heads, k_shape[1], dim, 1 if causal else 0,
                      max(dim, 1) ** -0.5 if scale is None else scale, k_shape[0], 0, 0, 0, qs[0], qs[1], os_[0], os_[1],
                      ks[0], ks[1], 0, vs[0], vs[1], 0)
    check(_call(_native.load().aexrt_b200_attention_packed, what, torch, (q, k, v, cu_q, cu_k, out, lse), stream,
                (desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), _index(cu_q, what, "cu_q", num_seqs + 1, torch.int32),
                 _index(cu_k, what, "cu_k", num_seqs + 1, torch.int32), out.data_ptr(), _ptr(lse))), what)
    return out if lse is None else (out, lse)


def attention_paged_workspace(q, k_cache, num_seqs: int, max_q: int):
    """A workspace tensor for :func:`attention_paged` calls of these shapes (any lengths and tables).  Calls that can
    overlap on the GPU each need their own."""
    what, torch = "attention_paged", _torch()
    (tokens, heads, dim), qs = _heads(q, what, "q", 3)
    k_shape, ks = _heads(k_cache, what, "k_cache", 4)
    if max_q < 0:
        raise ValueError(f"{what}: max_q must not be negative")
    desc = _pack(what, _dtype16(q, what, torch), num_seqs, tokens, max_q, heads, k_shape[2], dim, 1, 1.0, k_shape[0],
                      k_shape[1], 0, 0, qs[0], qs[1], heads * dim, dim, ks[1], ks[2], ks[0], ks[1], ks[2], ks[0])
    n = _call(lambda desc, stream: _native.load().aexrt_b200_attention_paged_workspace(desc), what, torch, (q, k_cache), 0, (desc,))
    check(n != 2 ** 64 - 1, what)
    return torch.empty((n,), dtype=torch.uint8, device=q.device)


def attention_paged(q, k_cache, v_cache, block_table, cu_q, kv_lens, max_q: int, causal: bool = True,
                    scale: Optional[float] = None, out=None, lse=None, return_lse: bool = False, workspace=None,
                    stream=None):
    """Attention of new tokens over a paged cache: ``q`` [q_tokens, q_heads, d] with sequence s in rows
    cu_q[s] .. cu_q[s + 1] (at most ``max_q`` each), caches [pages, page_size, kv_heads, d] (any strides; page_size
    a power of two from 8 to 1024), ``block_table`` [num_seqs, columns] int32, ``kv_lens`` [num_seqs] int32: cached keys
    of each sequence, the new tokens' own among them (see :func:`page_tables` and :func:`kv_append`).  ``workspace``:
    from :func:`attention_paged_workspace`; without one the call allocates it."""
    what, torch = "attention_paged", _torch()
    q_shape, qs = _heads(q, what, "q", 3)
    tokens, heads, dim = q_shape
    k_shape, ks = _heads(k_cache, what, "k_cache", 4)
    v_shape, vs = _heads(v_cache, what, "v_cache", 4)
    out, os_, lse = _outputs(what, torch, q, q_shape, out, lse, return_lse, stream)
    if k_shape != v_shape or k_shape[3] != dim or not q.dtype is k_cache.dtype is v_cache.dtype:
        raise ValueError(f"{what}: the caches must have one shape, and q's type and head size")
    num_seqs = _entries(kv_lens, what, "kv_lens")
    if max_q < 0:
        raise ValueError(f"{what}: max_q must not be negative")
    table, columns, table_stride = _table(block_table, what, num_seqs, torch.int32)
    if workspace is None:
        with _allocating(torch, stream, q.device):
            workspace = attention_paged_workspace(q, k_cache, num_seqs, max_q)
    elif not workspace.is_contiguous():
        raise ValueError(f"{what}: workspace must be contiguous")
    desc = _pack(what, _dtype16(q, what, torch), num_seqs, tokens, max_q, heads, k_shape[2], dim, 1 if causal else 0,
                      max(dim, 1) ** -0.5 if scale is None else scale, k_shape[0], k_shape[1], columns, table_stride,
                      qs[0], qs[1], os_[0], os_[1], ks[1], ks[2], ks[0], vs[1], vs[2], vs[0])
    check(_call(_native.load().aexrt_b200_attention_paged, what, torch,
                (q, k_cache, v_cache, block_table, cu_q, kv_lens, out, lse, workspace), stream,
                (desc, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), table,
                 _index(cu_q, what, "cu_q", num_seqs + 1, torch.int32), _index(kv_lens, what, "kv_lens", num_seqs, torch.int32), out.data_ptr(),
                 _ptr(lse), workspace.data_ptr(), workspace.numel() * workspace.element_size())), what)
    return out if lse is None else (out, lse)


def attention_status() -> int:
    """Reads and clears the attention kernels' status word of the current device (ATTENTION_* bits), after all work on it, on any stream."""
    v = ctypes.c_uint32(0)
    check(_native.load().aexrt_b200_attention_status(ctypes.byref(v)), "attention_status")
    return v.value


def page_tables(ctx_lens, new_lens, block_table, free_pages, free_state, page_size: int,
                max_tokens: Optional[int] = None, cu_q=None, kv_lens=None, slot_map=None, free_state_out=None, stream=None):
    """The tables of a serving step on the GPU: request s holds ctx_lens[s] cached tokens and brings new_lens[s].

    Takes the pages that the new tokens need from the free stack (``free_pages``, its top in ``free_state[0]``) into
    ``block_table`` [num_seqs, columns] in place, and returns (cu_q [num_seqs + 1], kv_lens [num_seqs],
    slot_map [max_tokens], free_state_out [2] = new top and pages missing), all int32.  slot_map holds each new
    token's slot, -1 where it has no page and behind the last token.  ``kv_lens`` may be ``ctx_lens`` and
    ``free_state_out`` may be ``free_state``: updated in place, as a captured step wants them."""
    what, torch = "page_tables", _torch()
    n = _entries(ctx_lens, what, "ctx_lens")

    def ints(size):
        return _made(torch, stream, (size,), torch.int32, ctx_lens.device)

    if slot_map is None:
        if max_tokens is None:
            raise ValueError(f"{what}: give max_tokens or slot_map")
        slot_map = ints(max_tokens)
    cu_q = ints(n + 1) if cu_q is None else cu_q
    kv_lens = ints(n) if kv_lens is None else kv_lens
    free_state_out = ints(2) if free_state_out is None else free_state_out
    table, columns, table_stride = _table(block_table, what, n, torch.int32)
    free, slots = _entries(free_pages, what, "free_pages"), _entries(slot_map, what, "slot_map")
    if (n | page_size | columns | table_stride | free | slots) >> 32:  # a C uint32_t would cut it; negative ones too
        raise ValueError(f"{what}: a size is out of range")
    check(_call(_native.load().aexrt_b200_page_tables, what, torch,
                (ctx_lens, new_lens, block_table, free_pages, free_state, cu_q, kv_lens, slot_map, free_state_out), stream,
                (_index(ctx_lens, what, "ctx_lens", n, torch.int32), _index(new_lens, what, "new_lens", n, torch.int32), n, page_size, table, columns,
                 table_stride, _index(free_pages, what, "free_pages", free, torch.int32), free, _index(free_state, what, "free_state", 2, torch.int32),
                 _index(free_state_out, what, "free_state_out", 2, torch.int32), _index(cu_q, what, "cu_q", n + 1, torch.int32),
                 _index(kv_lens, what, "kv_lens", n, torch.int32), _index(slot_map, what, "slot_map", slots, torch.int32), slots)), what)
    return cu_q, kv_lens, slot_map, free_state_out


def kv_append(k, v, slot_map, k_cache, v_cache, stream=None):
    """Writes rows ``k``, ``v`` [tokens, kv_heads, d] to their slots (page * page_size + row) of the paged caches
    [pages, page_size, kv_heads, d], in place; slots outside the cache (-1) are skipped.  Slots of one call are
    distinct, or each 16-byte piece of a shared slot comes from one of its tokens."""
    what, torch = "kv_append", _torch()
    k_shape, ks = _heads(k, what, "k", 3)
    v_shape, vs = _heads(v, what, "v", 3)
    kc_shape, kcs = _heads(k_cache, what, "k_cache", 4)
    vc_shape, vcs = _heads(v_cache, what, "v_cache", 4)
    _dtype16(k, what, torch)
    if k_shape != v_shape or kc_shape != vc_shape or k_shape[1:] != kc_shape[2:]:
        raise ValueError(f"{what}: k and v, and the caches, must agree in heads and head size")
    if not k.dtype is v.dtype is k_cache.dtype is v_cache.dtype:
        raise ValueError(f"{what}: one type for k, v and the caches")
    if (k_shape[0] | k_shape[1] | k_shape[2] | kc_shape[0] | kc_shape[1]) >> 32:  # a C uint32_t would cut it
        raise ValueError(f"{what}: a size is out of range")
    check(_call(_native.load().aexrt_b200_kv_append, what, torch, (k, v, slot_map, k_cache, v_cache), stream,
                (k.data_ptr(), v.data_ptr(), k_shape[0], k_shape[1], k_shape[2], ks[0], ks[1], vs[0], vs[1],
                 _index(slot_map, what, "slot_map", k_shape[0], torch.int32), k_cache.data_ptr(), v_cache.data_ptr(), kc_shape[0],
                 kc_shape[1], kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2])), what)
