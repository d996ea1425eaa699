"""Op-level API over ``libldx.so``: the drop-in replacements for the reference's
``nax_conv3d`` / ``pack_weight`` / ``pack_upsample_weight`` / ``conv3d_ncdhw`` /
``flash_attention`` / ``mx.fast.scaled_dot_product_attention`` /
``group_norm_affine`` / ``mx.fast.layer_norm``.

Tensors are ``torch`` CUDA (HIP) tensors used only as device memory; every op runs a
hand-written gfx950 kernel through the C ABI on torch's current stream. Activations
are channels-last NDHWC ``(B, D, H, W, C)`` float16, optionally a channel slice of a
wider tensor (the voxel pitch is read from the strides). Argument errors raise
``ValueError`` before anything is launched; HIP errors raise ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import (ACT_GELU, ACT_NONE, ACT_SILU, BLOCK4, BLOCK8, PAGE4, PAGE8, ROTARY_AXES, AttnArgs, Cache4AppendArgs,
                   Cache4AttentionArgs, Cache4ReadArgs, Cache8AppendArgs, Cache8AttentionArgs, Cache8Block,
                   ConvArgs, Dense8Args, RmsNormArgs, RotateHeadsArgs, SourceConvArgs, check, filler, lib)

__all__ = [
    "PackedWeight", "pack_weight", "pack_upsample_weight", "nax_conv3d", "conv3d", "dense",
    "group_norm_affine", "layer_norm", "attention", "flash_attention", "timestep_embedding",
    "silu", "upsample_nearest2", "resize_nearest", "output_extent", "count_flops", "squared_norms4",
    "nearest_codebook4", "conv3d_half", "group_norm_half", "Quantized8", "quantize8", "rms_norm", "dense8",
    "Cache8", "cache8_append", "cache8_attention", "Rotary", "rotate_heads", "Cache4", "cache4_append", "cache4_read",
    "cache4_attention",
]


class count_flops:
    """Context manager tallying the algorithmic FLOPs (2 x real multiply-adds, no
    padding; a folded upsample conv counts its 8 taps) of the convs, dense layers and
    attention launched inside it -- for throughput figures. ``cache8_attention`` and
    ``cache4_attention`` are not counted: how many tokens their queries see stands on the device alone."""

    active: "count_flops | None" = None

    def __init__(self) -> None:
        self.conv = 0.0
        self.dense = 0.0
        self.attention = 0.0

    @property
    def total(self) -> float:
        return self.conv + self.dense + self.attention

    def __enter__(self) -> "count_flops":
        count_flops.active = self
        return self

    def __exit__(self, *exc) -> None:
        count_flops.active = None


# A small op's time is its host path: on MI355X hosts the launch itself takes 4 us, the
# allocation of its result 1.8, and the helpers below and the argument blocks the rest (a dense
# layer 15.4 us before they were written without stream objects, pointer wrappers and tensor
# views, 11.1 now; an attention call 19.3, 10.9 now).

def _stream() -> int:
    """Handle of torch's current stream on the current device, read without building a stream
    object (2.9 -> 0.2 us)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _f32(t: torch.Tensor) -> torch.Tensor:
    """``t`` as contiguous fp32: ``t`` itself where it is that already."""
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


# Element types of the conv / attention kernels (the C ABI's LDX_DTYPE_*): fp16 and bf16, and
# fp32 for the FP32 networks (the exact split-fp16 mode).
ELEM_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
ALL_DTYPES = {**ELEM_DTYPES, torch.float32: _lib.DTYPE_F32}


def _require_cuda(t: torch.Tensor, name: str, dtype: torch.dtype | tuple | None = torch.float16) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor (got {t.device}); there is no CPU path")
    allowed = dtype if isinstance(dtype, tuple) else (dtype,)
    if dtype is not None and t.dtype not in allowed:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in allowed)}, got {t.dtype}")


def _same_elem(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    """``t`` is a device tensor of the call's element type ``dtype``."""
    _require_cuda(t, name, dtype)


def voxel_pitch(x: torch.Tensor, name: str = "x") -> int:
    """Voxel pitch (elements) of an NDHWC tensor whose voxels are evenly spaced and
    whose channels are contiguous -- a contiguous tensor or a channel slice of one."""
    if x.dim() != 5:
        raise ValueError(f"{name} must be NDHWC (B, D, H, W, C), got shape {tuple(x.shape)}")
    if x.is_contiguous() and x.numel():
        return x.shape[4]
    b, d, h, w, c = x.shape
    st = x.stride()
    if c > 1 and st[4] != 1:
        raise ValueError(f"{name}: channels must be contiguous")
    pitch = st[3] if w > 1 else (st[2] // max(w, 1) if h > 1 else (st[1] // (h * w) if d > 1 else (
        st[0] // (d * h * w) if b > 1 else c)))
    if pitch < c:
        raise ValueError(f"{name}: voxel pitch {pitch} < channels {c}")
    if ((w > 1 and st[3] != pitch) or (h > 1 and st[2] != w * pitch)
            or (d > 1 and st[1] != h * w * pitch) or (b > 1 and st[0] != d * h * w * pitch)):
        raise ValueError(f"{name}: voxels must be evenly spaced (strides {st})")
    return int(pitch)


def output_extent(n: int, *, stride: int = 1, upsample: bool = False) -> int:
    """``n`` (stride 1), ``(n - 1) // 2 + 1`` (stride 2), ``2 n`` (upsample)
    (_nax_conv.py:513-516, 552)."""
    if upsample:
        return 2 * n
    if stride == 1:
        return n
    if stride == 2:
        return (n - 1) // 2 + 1
    raise ValueError("stride must be 1 or 2")


# ------------------------------------------------------------------ weights

@dataclass
class PackedWeight:
    """A conv/dense weight in the kernel's fragment-major layout (a flat fp16 tensor of
    ``ldx_packed_weight_elems`` values; see ``include/ldx.h``), or folded into the
    8 parity filters of a nearest-2x-upsampled conv."""

    data: torch.Tensor
    out_channels: int
    in_channels: int
    ksize: int
    upsample: bool = False
    # FP32 weight in the exact mode's split: hi and lo fp16 planes
    # (``ldx_packed_weight_exact_elems`` values; an upsample conv keeps its unfolded 3x3x3
    # taps and runs on the upsampled grid).
    exact: bool = False


def pack_weight(weight: torch.Tensor) -> PackedWeight:
    """Pack a Torch-layout ``(O, C, K, K, K)`` (K = 1 or 3) or dense ``(O, C)`` fp16 or
    bf16 weight (the reference's ``pack_weight``, _nax_conv.py:350-364, in this library's
    layout); the packed tensor keeps the weight's dtype. An fp32 weight is packed for the
    exact mode (its hi / lo fp16 split, _nax_conv.py:343-364)."""
    _require_cuda(weight, "weight", tuple(ALL_DTYPES))
    if weight.dim() == 2:
        weight = weight.reshape(*weight.shape, 1, 1, 1)
    if weight.dim() != 5 or weight.shape[2] != weight.shape[3] or weight.shape[3] != weight.shape[4] \
            or weight.shape[2] not in (1, 3):
        raise ValueError(f"weight must be (O, C, K, K, K) with K in (1, 3), got {tuple(weight.shape)}")
    o, c, k = int(weight.shape[0]), int(weight.shape[1]), int(weight.shape[2])
    w = weight.contiguous()
    if w.dtype == torch.float32:
        return _pack_exact(w, o, c, k, False)
    out = torch.empty(lib.ldx_packed_weight_elems(o, c, k, 0), dtype=w.dtype, device=weight.device)
    check(lib.ldx_pack_weight(_ptr(w), o, c, k, _ptr(out), _stream()), "pack_weight")
    return PackedWeight(out, o, c, k, False)


def _pack_exact(w: torch.Tensor, o: int, c: int, k: int, upsample: bool) -> PackedWeight:
    out = torch.empty(lib.ldx_packed_weight_exact_elems(o, c, k), dtype=torch.float16, device=w.device)
    check(lib.ldx_pack_weight_exact(_ptr(w), o, c, k, _ptr(out), _stream()), "pack_weight_exact")
    return PackedWeight(out, o, c, k, upsample, exact=True)


def pack_upsample_weight(weight: torch.Tensor) -> PackedWeight:
    """Fold a ``(O, C, 3, 3, 3)`` fp16 weight into 8 parity 2x2x2 filters for a conv of a
    nearest 2x upsampling (_nax_conv.py:367-405), in the weight's dtype (fp16 or bf16). An
    fp32 weight keeps its 3x3x3 taps, split for the exact mode (the conv runs on the
    upsampled grid)."""
    _require_cuda(weight, "weight", tuple(ALL_DTYPES))
    if weight.dim() != 5 or tuple(weight.shape[2:]) != (3, 3, 3):
        raise ValueError(f"weight must be (O, C, 3, 3, 3), got {tuple(weight.shape)}")
    o, c = int(weight.shape[0]), int(weight.shape[1])
    w = weight.contiguous()
    if w.dtype == torch.float32:
        return _pack_exact(w, o, c, 3, True)
    out = torch.empty(lib.ldx_packed_weight_elems(o, c, 3, 1), dtype=w.dtype, device=weight.device)
    check(lib.ldx_pack_upsample_weight(_ptr(w), o, c, ELEM_DTYPES[w.dtype], _ptr(out), _stream()),
          "pack_upsample_weight")
    return PackedWeight(out, o, c, 3, True)


def unpack_weight(packed: PackedWeight) -> "np.ndarray":
    """Host copy of a packed weight in the plain ``(parities, O, taps, C)`` order (a test
    and debugging aid; the kernels read the fragment-major form)."""
    import numpy as np

    taps = 8 if packed.upsample else packed.ksize ** 3
    par = 8 if packed.upsample else 1
    nob = -(-packed.out_channels // 128) * 4
    nkc = -(-packed.in_channels // 64) * 4
    f = packed.data.cpu().numpy().reshape(par, nob, taps, nkc, 2, 32, 8)  # lane = g*32 + r
    # -> (par, ob, r, taps, kc, g, e) -> (par, O', taps, C')
    full = f.transpose(0, 1, 5, 2, 3, 4, 6).reshape(par, nob * 32, taps, nkc * 16)
    return full[:, :packed.out_channels, :, :packed.in_channels]


def _bias32(bias: torch.Tensor | None, batch: int, out_c: int) -> tuple[torch.Tensor | None, int]:
    if bias is None:
        return None, 0
    if not bias.is_cuda:
        raise ValueError("bias must be a device tensor")
    if bias.shape[-1] != out_c or bias.dim() not in (1, 2) or (bias.dim() == 2 and bias.shape[0] != batch):
        raise ValueError(f"bias shape {tuple(bias.shape)} does not fit ({batch}, {out_c})")
    return _f32(bias), int(bias.dim() == 2)


# ------------------------------------------------------------------ conv3d

MOMENTS_MAX_BLOCKS = 16384


def nax_conv3d(x: torch.Tensor, packed: PackedWeight, bias: torch.Tensor | None = None, *,
               affine: torch.Tensor | None = None, silu: bool = False, stride: int = 1,
               upsample: bool = False, output_scale: float = 1.0,
               residual: torch.Tensor | None = None, x1: torch.Tensor | None = None,
               act: str | None = None, out: torch.Tensor | None = None,
               shift: torch.Tensor | None = None,
               ln: tuple[torch.Tensor, torch.Tensor, float] | None = None,
               moments: bool | str = False) -> torch.Tensor:
    """Fused conv of NDHWC ``x`` (optionally ``concat([x, x1], channels)``) with a packed
    weight: ``half((conv(prep(x)) + bias + shift) * output_scale + residual)``, ``prep`` =
    the per-(b, c) ``affine`` then SiLU, rounded to fp16 once (nax_conv3d,
    _nax_conv.py:451-500). ``shift`` is an fp16 ``(B, O)`` per-batch term (a row slice of
    a wider tensor is fine). ``act="gelu"`` / ``"silu"`` additionally stores
    ``half(act(y))``. ``ln = (gamma, beta, eps)`` (pointwise convs of one input only)
    layer-normalizes each input row first, in the same launch (ldx_dense_ln).
    ``moments=True`` also keeps the GroupNorm partial moments of the output, reduced in
    the conv's epilogue (ldx_conv3d_stats), where the plan allows it and pays (not on
    split-K plans; ``moments="always"`` keeps them there too): a later
    ``group_norm_affine`` of the returned tensor then merges them instead of reading it.

    Element type: fp16 or bf16 (``x``'s dtype; ``x1``, the packed weight, ``shift``,
    ``residual`` and ``out`` must share it; bias and affine are fp32 either way), or fp32:
    the exact split-fp16 mode of the FP32 networks (a weight packed from fp32; no moments,
    no fused LayerNorm).

    Returns NDHWC ``(B, D', H', W', O)`` in ``x``'s dtype (written into ``out`` when given,
    which may be a channel slice of a wider tensor).
    """
    _require_cuda(x, "x", tuple(ALL_DTYPES))
    et = x.dtype
    exact = et == torch.float32
    if packed.exact != exact or (not exact and packed.data.dtype != et):
        raise ValueError(f"packed weight is {'an fp32 (exact) packing' if packed.exact else packed.data.dtype} "
                         f"but x is {et}")
    if exact and (ln is not None or moments == "always"):
        raise ValueError("the fp32 mode has no fused LayerNorm and keeps no moments")
    xp = voxel_pitch(x, "x")
    b, d, h, w, c0 = (int(s) for s in x.shape)
    c1, x1p = 0, 0
    if x1 is not None:
        _same_elem(x1, "x1", et)
        x1p = voxel_pitch(x1, "x1")
        if tuple(x1.shape[:4]) != (b, d, h, w):
            raise ValueError(f"x1 grid {tuple(x1.shape[:4])} != x grid {(b, d, h, w)}")
        c1 = int(x1.shape[4])
    if packed.in_channels != c0 + c1:
        raise ValueError(f"packed weight expects {packed.in_channels} input channels, got {c0 + c1}")
    if packed.upsample != bool(upsample):
        raise ValueError("upsample convs need pack_upsample_weight weights (and only they)")
    if packed.ksize == 1 and (stride != 1 or upsample):
        raise ValueError("pointwise conv supports stride 1 only")
    o = packed.out_channels
    if upsample:
        grid = (2 * d, 2 * h, 2 * w)
    elif packed.ksize == 3:
        grid = tuple(output_extent(n, stride=stride) for n in (d, h, w))
    else:
        grid = (d, h, w)
    bias32, batched = _bias32(bias, b, o)
    aff = None
    if affine is not None:
        if affine.dtype != torch.float32 or not affine.is_cuda or affine.numel() != b * (c0 + c1) * 2:
            raise ValueError("affine must be device float32 with batch * C * 2 values")
        aff = affine.contiguous()
    resp = 0
    if residual is not None:
        _same_elem(residual, "residual", et)
        if tuple(residual.shape) != (b, *grid, o):
            raise ValueError(f"residual shape {tuple(residual.shape)} != output {(b, *grid, o)}")
        resp = voxel_pitch(residual, "residual")
    if out is None:
        out = torch.empty((b, *grid, o), dtype=et, device=x.device)
    else:
        _same_elem(out, "out", et)
        if tuple(out.shape) != (b, *grid, o):
            raise ValueError(f"out shape {tuple(out.shape)} != {(b, *grid, o)}")
    yp = voxel_pitch(out, "out")
    a = ConvArgs()
    a.batch, a.in_d, a.in_h, a.in_w = b, d, h, w
    a.c0, a.c1, a.out_c = c0, c1, o
    a.ksize, a.stride, a.upsample = packed.ksize, stride, int(bool(upsample))
    a.x0, a.x0_pitch = x.data_ptr(), xp
    a.x1, a.x1_pitch = (x1.data_ptr() if x1 is not None else None), x1p
    a.weight = packed.data.data_ptr()
    a.bias, a.bias_batched = (bias32.data_ptr() if bias32 is not None else None), batched
    a.affine, a.silu = (aff.data_ptr() if aff is not None else None), int(bool(silu))
    a.residual, a.residual_pitch = (residual.data_ptr() if residual is not None else None), resp
    a.output_scale = float(output_scale)
    a.act = {None: ACT_NONE, "gelu": ACT_GELU, "silu": ACT_SILU}[act]
    a.dtype = ALL_DTYPES[et]
    if shift is not None:
        _same_elem(shift, "shift", et)
        if shift.dim() != 2 or tuple(shift.shape) != (b, o) or shift.stride(1) != 1:
            raise ValueError(f"shift must be (B, O) = {(b, o)} with contiguous channels")
        a.shift, a.shift_pitch = shift.data_ptr(), shift.stride(0) if b > 1 else o
    a.y, a.y_pitch = out.data_ptr(), yp
    if count_flops.active is not None:
        taps = 8 if upsample else packed.ksize ** 3
        flops = 2.0 * b * grid[0] * grid[1] * grid[2] * o * (c0 + c1) * taps
        if packed.ksize == 1 and d == 1 and h == 1:
            count_flops.active.dense += flops
        else:
            count_flops.active.conv += flops
    ws_bytes = lib.ldx_conv3d_workspace_bytes(ctypes.byref(a))
    ws = None
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws_bytes
    if ln is not None:
        gamma, beta, eps = ln
        for t, name in ((gamma, "ln gamma"), (beta, "ln beta")):
            if t.dtype != torch.float32 or not t.is_cuda or t.numel() != c0 or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous device float32 with {c0} values")
        check(lib.ldx_dense_ln(ctypes.byref(a), gamma.data_ptr(), beta.data_ptr(), float(eps), _stream()),
              "dense_ln")
        _set_moments(out, None)
        return out
    # Split-K plans (a workspace was asked for) keep no moments here: on the small tensors
    # that split, the reduce with moments (6.5 us) and their merge cost more than the
    # plain reduce plus a one-launch GroupNorm pass (measured on MI355X, config 5).
    # Nor do outputs of more than MOMENTS_MAX_BLOCKS moment blocks per batch item (the VQ
    # decoder's 32-channel full-resolution convs, 10^5 blocks): one workgroup per group
    # merges the blocks, which there costs more (90 us) than the two-pass GroupNorm over
    # the tensor (measured on MI355X, config 4: caps of 2048 / 4096 / 16384 blocks gave
    # 19.67 / 19.70 / 19.59 ms).
    if exact:
        check(lib.ldx_conv3d(ctypes.byref(a), _stream()), "conv3d (fp32)")
        _set_moments(out, None)
        return out
    # An inference-mode output keeps no moments (see _set_moments), so none are taken.
    want = (moments == "always" or (moments is True and not ws_bytes)) and not out.is_inference()
    chunks = lib.ldx_conv3d_stats_chunks(ctypes.byref(a)) if want else 0
    if moments != "always" and chunks > MOMENTS_MAX_BLOCKS:
        chunks = 0
    if chunks > 0:
        m = torch.empty((b, chunks, o // 2, 3), dtype=torch.float32, device=x.device)
        check(lib.ldx_conv3d_stats(ctypes.byref(a), m.data_ptr(), _stream()), "conv3d_stats")
        _set_moments(out, m)
        return out
    check(lib.ldx_conv3d(ctypes.byref(a), _stream()), "conv3d")
    _set_moments(out, None)
    return out


def _wrote(t: torch.Tensor) -> None:
    """Record that a kernel wrote ``t`` through its data pointer. Torch counts in-place
    writes in a version counter shared by every view of the same storage, but a write by
    a kernel launched through the C ABI is invisible to it; bumping the counter here
    makes every write -- by this library or by torch -- invalidate moments kept of any
    view of that storage. Inference tensors (``torch.inference_mode``) carry no version
    counter; nothing is recorded for them, and no moments are kept of them."""
    if not t.is_inference():
        increment_version(t)


def _set_moments(t: torch.Tensor, m: torch.Tensor | None) -> None:
    """Attach (or clear) the GroupNorm partial moments a conv kept of ``t`` as written,
    tagged with the storage's write version after that write. An inference tensor has no
    write version to validate moments against later, so none are kept of it (its
    GroupNorm then reduces the tensor itself)."""
    _wrote(t)
    if m is None or t.is_inference():
        if hasattr(t, "_ldx_moments"):
            del t._ldx_moments
    else:
        t._ldx_moments = (m, t._version)


def moments_of(t: torch.Tensor | None) -> torch.Tensor | None:
    """The ``(B, chunks, C / 2, 3)`` moments a conv kept of ``t`` (``nax_conv3d(...,
    moments=True)``), or None -- also when anything has written to ``t``'s storage since
    (a torch in-place op, another op's ``out=``, a write through another view)."""
    kept = getattr(t, "_ldx_moments", None) if t is not None else None
    if kept is None or t.is_inference():
        return None
    m, version = kept
    if t._version != version or t.dim() != 5 or m.shape[0] != t.shape[0] or 2 * m.shape[2] != t.shape[4]:
        return None
    return m


def conv3d(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           stride: int = 1, padding: int | None = None) -> torch.Tensor:
    """The reference's op-level ``conv3d(x, w, b, stride, pad)`` on NDHWC ``x`` with a
    Torch-layout ``(O, C, K, K, K)`` weight: K = 3 with padding 1, or K = 1 with
    padding 0 (mlx_model.py:159-202). Packs the weight on each call; modules prepack."""
    k = int(weight.shape[2]) if weight.dim() == 5 else 1
    pad = k // 2 if padding is None else padding
    if pad != k // 2:
        raise ValueError(f"only padding {k // 2} is supported for a {k}x{k}x{k} kernel")
    return nax_conv3d(x, pack_weight(weight), bias, stride=stride)


def dense(x: torch.Tensor, packed: PackedWeight, bias: torch.Tensor | None = None, *,
          residual: torch.Tensor | None = None, act: str | None = None,
          out: torch.Tensor | None = None, affine: torch.Tensor | None = None,
          ln: tuple[torch.Tensor, torch.Tensor, float] | None = None) -> torch.Tensor:
    """``half(x @ W^T + bias (+ residual))`` over the last axis of fp16 ``x`` with fp32
    accumulation and one rounding (SourceLayers.dense native path, mlx_model.py:204-217).
    ``ln = (gamma, beta, eps)`` applies ``layer_norm`` to ``x`` first, in the same launch."""
    if packed.ksize != 1:
        raise ValueError("dense needs a (O, C) weight packed with pack_weight")
    lead = x.shape[:-1]
    rows = math.prod(lead)
    x5 = x.reshape(1, 1, 1, rows, x.shape[-1])
    r5 = None if residual is None else residual.reshape(1, 1, 1, rows, packed.out_channels)
    o5 = None if out is None else out.reshape(1, 1, 1, rows, packed.out_channels)
    y = nax_conv3d(x5, packed, bias, residual=r5, act=act, out=o5, affine=affine, ln=ln)
    return y.reshape(*lead, packed.out_channels)


# ------------------------------------------------------------ normalisation

def group_norm_affine(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, *, groups: int,
                      eps: float, x1: torch.Tensor | None = None) -> torch.Tensor:
    """Per-(b, c) ``(scale, offset)`` fp32 ``(B, C, 2)`` of GroupNorm over NDHWC ``x``
    (optionally ``concat([x, x1])``), ``scale = gamma * rsqrt(var + eps)``, ``offset =
    beta - scale * mean`` (medmlx_core group_norm_affine; mlx_model.py:328-335)."""
    _require_cuda(x, "x", (torch.float16, torch.float32))
    xp = voxel_pitch(x, "x")
    b, d, h, w, c0 = (int(s) for s in x.shape)
    c1, x1p = 0, 0
    if x1 is not None:
        _require_cuda(x1, "x1", x.dtype)
        x1p = voxel_pitch(x1, "x1")
        c1 = int(x1.shape[4])
    c = c0 + c1
    if c % groups:
        raise ValueError(f"groups {groups} must divide channels {c}")
    g32, b32 = _f32(gamma), _f32(beta)
    if x.dtype == torch.float32:
        out = torch.empty((b, c, 2), dtype=torch.float32, device=x.device)
        ws_bytes = lib.ldx_group_norm_f32_workspace_bytes(b, d * h * w, c, groups)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
        check(lib.ldx_group_norm_affine_f32_ws(_ptr(x), xp, c0, _ptr(x1), x1p, c1, b, d * h * w, groups, _ptr(g32),
                                               _ptr(b32), float(eps), _ptr(out), _ptr(ws), ws_bytes, _stream()),
              "group_norm_affine_f32")
        return out
    m0, m1 = moments_of(x), moments_of(x1)
    if m0 is not None and (x1 is None or m1 is not None) and (c // groups) % 2 == 0 and c0 % 2 == 0 \
            and c1 % 2 == 0:
        # Moments the producing convs kept: no pass over x.
        out = torch.empty((b, c, 2), dtype=torch.float32, device=x.device)
        n1 = int(m1.shape[1]) if m1 is not None else 0
        # Many blocks per group: the blocks are first folded by a pass over whole rows.
        ws_bytes = lib.ldx_group_norm_moments_workspace_bytes(int(m0.shape[1]), c0, n1, c1, b, groups)
        ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=x.device)
        check(lib.ldx_group_norm_affine_moments_ws(
            _ptr(m0), int(m0.shape[1]), c0, _ptr(m1), n1, c1, b, groups, _ptr(g32), _ptr(b32), float(eps),
            _ptr(out), _ptr(ws), ws_bytes, _stream()), "group_norm_affine_moments")
        return out
    voxels = d * h * w
    ws = torch.empty(max(1, lib.ldx_group_norm_workspace_bytes(b, voxels, c, groups)),
                     dtype=torch.uint8, device=x.device)
    out = torch.empty((b, c, 2), dtype=torch.float32, device=x.device)
    check(lib.ldx_group_norm_affine(_ptr(x), xp, c0, _ptr(x1), x1p, c1, b, voxels, groups,
                                    _ptr(g32), _ptr(b32), float(eps), _ptr(out), _ptr(ws), _stream()),
          "group_norm_affine")
    return out


def layer_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """LayerNorm over the last axis of fp16 or fp32 ``x`` (mx.fast.layer_norm,
    mlx_model.py:360-367)."""
    _require_cuda(x, "x", (torch.float16, torch.float32))
    f = int(x.shape[-1])
    x2 = x.reshape(-1, f)
    if x2.stride(-1) != 1:
        raise ValueError("layer_norm: features must be contiguous")
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _require_cuda(out, "out", x.dtype)
    o2 = out.reshape(-1, f)
    fn = lib.ldx_layer_norm_f32 if x.dtype == torch.float32 else lib.ldx_layer_norm
    g32, b32 = _f32(gamma), _f32(beta)
    check(fn(_ptr(x2), x2.stride(0), x2.shape[0], f, _ptr(g32), _ptr(b32), float(eps), _ptr(o2), o2.stride(0),
             _stream()), "layer_norm")
    _wrote(out)
    return out


# ----------------------------------------------------------------- attention

def _attn_block(b: int, h: int, lq: int, lk: int, d: int, q: tuple, k: tuple, v: tuple, o: tuple, scale: float,
                like: torch.Tensor, mask: torch.Tensor | None) -> AttnArgs:
    """The C arguments from dimensions and ``(pointer, (batch, token, head) strides)`` of each
    operand, with the workspace they ask for; ``like`` gives the element type and device."""
    a = AttnArgs(b, h, lq, lk, d, *q, *k, *v, *o, float(scale))
    a.dtype = ALL_DTYPES[like.dtype]
    if mask is not None:
        a.mask, a.mask_stride = mask.data_ptr(), mask.stride()
    ws_bytes = lib.ldx_attention_workspace_bytes(ctypes.byref(a))
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=like.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws_bytes
        a._keep = ws  # the buffer lives as long as the argument block
    return a


def _attn_args(q4: torch.Tensor, k4: torch.Tensor, v4: torch.Tensor, o4: torch.Tensor,
               scale: float, mask: torch.Tensor | None) -> AttnArgs:
    """Build the C arguments from (B, L, H, D) views."""
    b, lq, h, d = q4.shape
    views = []
    for name, t in (("q", q4), ("k", k4), ("v", v4), ("o", o4)):
        st = t.stride()
        if st[3] != 1:
            raise ValueError(f"attention: {name} head_dim must be contiguous")
        views.append((t.data_ptr(), st[:3]))
    return _attn_block(b, h, lq, int(k4.shape[1]), d, *views, scale, q4, mask)


def _interleaved(t: torch.Tensor, name: str, d: int) -> tuple[int, tuple[int, int, int]]:
    """``(pointer, strides)`` of a ``(B, L, heads * d)`` tensor's (B, L, heads, d) view."""
    sb, sl, sc = t.stride()
    if sc != 1:
        raise ValueError(f"attention: {name} head_dim must be contiguous")
    return t.data_ptr(), (sb, sl, d)


def _prepare_mask(mask: torch.Tensor | None, b: int, h: int, lq: int, lk: int,
                  device: torch.device) -> torch.Tensor | None:
    if mask is None:
        return None
    if not mask.is_cuda:
        raise ValueError("mask must be a device tensor")
    if mask.dtype == torch.bool:
        mask = torch.zeros(mask.shape, dtype=torch.float32, device=device).masked_fill(~mask, -math.inf)
    mask = mask.to(torch.float32)
    while mask.dim() < 4:
        mask = mask.unsqueeze(0)
    return mask.expand(b, h, lq, lk)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
              mask: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale + mask) v`` for fp16 ``(B, H, L, D)`` tensors, the contract
    of ``mx.fast.scaled_dot_product_attention`` (mlx_model.py:485-487, 860-862). ``mask``
    is additive (``-inf`` removes a key) or boolean (``True`` keeps a key), broadcast to
    ``(B, H, L, LK)``. fp16 or bf16 (all three alike; the probabilities are rounded to
    that type for the P V product), or fp32 (head widths 16 / 32 / 64, no mask; FP32
    throughout). Returns ``(B, H, L, D)``."""
    _require_cuda(q, "q", tuple(ALL_DTYPES))
    for name, t in (("q", q), ("k", k), ("v", v)):
        _same_elem(t, name, q.dtype)
        if t.dim() != 4:
            raise ValueError(f"{name} must be (B, H, L, D)")
    b, h, lq, d = (int(s) for s in q.shape)
    lk = int(k.shape[2])
    if tuple(k.shape) != (b, h, lk, d) or tuple(v.shape) != (b, h, lk, d):
        raise ValueError(f"k/v shapes {tuple(k.shape)}, {tuple(v.shape)} do not fit q {tuple(q.shape)}")
    out = torch.empty((b, h, lq, d), dtype=q.dtype, device=q.device)
    m = _prepare_mask(mask, b, h, lq, lk, q.device)
    a = _attn_args(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), out.transpose(1, 2), scale, m)
    if count_flops.active is not None:
        count_flops.active.attention += 4.0 * b * h * lq * lk * d
    check(lib.ldx_attention(ctypes.byref(a), _stream()), "attention")
    return out


def flash_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, heads: int, scale: float,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Multi-head attention on head-interleaved projections ``(B, L, heads * d)``
    (head ``h`` = columns ``h*d .. h*d+d-1``), returning that layout
    (flash_attention, _attention.py:331-351). Key length may differ from query length.
    fp16, bf16 or fp32 (as ``attention``)."""
    _require_cuda(q, "q", tuple(ALL_DTYPES))
    for name, t in (("q", q), ("k", k), ("v", v)):
        _same_elem(t, name, q.dtype)
        if t.dim() != 3:
            raise ValueError(f"{name} must be (B, L, heads * d)")
    b, lq, f = (int(s) for s in q.shape)
    if f % heads:
        raise ValueError(f"features {f} not divisible by heads {heads}")
    d = f // heads
    lk = int(k.shape[1])
    if tuple(k.shape) != (b, lk, f) or tuple(v.shape) != (b, lk, f):
        raise ValueError("k/v must be (B, LK, heads * d) matching q")
    views = _interleaved(q, "q", d), _interleaved(k, "k", d), _interleaved(v, "v", d)
    if out is None:
        out = torch.empty((b, lq, f), dtype=q.dtype, device=q.device)
    else:
        _same_elem(out, "out", q.dtype)
        out.unflatten(2, (heads, d))   # raises where the last axis is not heads * d
    a = _attn_block(b, heads, lq, lk, d, *views, _interleaved(out, "o", d), scale, q, None)
    if count_flops.active is not None:
        count_flops.active.attention += 4.0 * b * heads * lq * lk * d
    check(lib.ldx_attention(ctypes.byref(a), _stream()), "attention")
    _wrote(out)
    return out


# ---------------------------------------------------------------- small ops

def timestep_embedding(timesteps: torch.Tensor, channels: int, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``[cos(t f), sin(t f)]`` (mlx_model.py:609-612) for int32 ``timesteps``, fp16 (computed
    in fp32, rounded once) or fp32."""
    _require_cuda(timesteps, "timesteps", torch.int32)
    if dtype not in (torch.float16, torch.float32):
        raise ValueError(f"timestep features are fp16 or fp32, not {dtype}")
    t = timesteps.contiguous()
    out = torch.empty((t.shape[0], channels), dtype=dtype, device=t.device)
    fn = lib.ldx_timestep_embedding_f32 if dtype == torch.float32 else lib.ldx_timestep_embedding
    check(fn(_ptr(t), t.shape[0], channels, _ptr(out), _stream()), "timestep_embedding")
    return out


def silu(x: torch.Tensor) -> torch.Tensor:
    """``half(silu(float(x)))`` (LdmUnet.silu, mlx_model.py:409-413)."""
    _require_cuda(x, "x")
    xc = x.contiguous()
    out = torch.empty_like(xc)
    check(lib.ldx_silu(_ptr(xc), xc.numel(), _ptr(out), _stream()), "silu")
    return out


def upsample_nearest2(x: torch.Tensor) -> torch.Tensor:
    """Nearest 2x upsampling of NDHWC ``x`` (_spatial.py:41-57)."""
    _require_cuda(x, "x")
    xp = voxel_pitch(x)
    b, d, h, w, c = (int(s) for s in x.shape)
    out = torch.empty((b, 2 * d, 2 * h, 2 * w, c), dtype=torch.float16, device=x.device)
    check(lib.ldx_upsample_nearest2(_ptr(x), xp, b, d, h, w, c, _ptr(out), c, _stream()),
          "upsample_nearest2")
    return out


def resize_nearest(x: torch.Tensor, shape: tuple[int, int, int]) -> torch.Tensor:
    """Nearest resize of NDHWC ``x`` to spatial ``shape``; only the factor-two case the
    model uses runs on the device (_spatial.py:60-69)."""
    if len(shape) != 3:
        raise ValueError("nearest resizing needs three spatial axes")
    if tuple(shape) == tuple(2 * int(s) for s in x.shape[1:4]):
        return upsample_nearest2(x)
    raise ValueError("only nearest 2x resizing is supported")


# ------------------------------------------------------------ VQ codebook search

_VQ_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _vq_rows(t: torch.Tensor, name: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor; there is no CPU path")
    if t.dtype not in _VQ_DTYPES:
        raise ValueError(f"{name} must be float16 or float32, got {t.dtype}")
    if t.dim() != 2 or t.shape[1] != 4 or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous (rows, 4), got {tuple(t.shape)}")
    if t.shape[0] < 1:
        raise ValueError(f"{name} is empty")
    return int(t.shape[0])


def squared_norms4(x: torch.Tensor) -> torch.Tensor:
    """Per-row ``T(sum float32(T(x * x)))`` of ``(rows, 4)`` vectors, the squared norm the
    reference keeps per codebook entry (mlx_model.py:775-778)."""
    n = _vq_rows(x, "x")
    out = torch.empty(n, dtype=x.dtype, device=x.device)
    check(lib.ldx_vq_squared_norms4(_ptr(x), n, _VQ_DTYPES[x.dtype], _ptr(out), _stream()), "vq_squared_norms4")
    return out


def nearest_codebook4(z: torch.Tensor, codebook: torch.Tensor, codebook_norm: torch.Tensor, *,
                      quantized: torch.Tensor | None = None) -> torch.Tensor:
    """int32 index of the nearest codebook row for each ``(positions, 4)`` latent row:
    the reference's distance and rounding points, the first NaN distance else the first
    smallest (nearest_codebook4, _vq.py:63-82). ``quantized`` (same shape and dtype as
    ``z``), when given, receives the straight-through ``z + (selected - z)``."""
    p = _vq_rows(z, "z")
    e = _vq_rows(codebook, "codebook")
    if codebook.dtype != z.dtype or codebook_norm.dtype != z.dtype:
        raise ValueError("z, codebook and codebook_norm must share one dtype")
    if not codebook_norm.is_cuda or tuple(codebook_norm.shape) != (e,) or not codebook_norm.is_contiguous():
        raise ValueError(f"codebook_norm must be a contiguous device vector of {e} values")
    if quantized is not None and (tuple(quantized.shape) != (p, 4) or quantized.dtype != z.dtype
                                  or not quantized.is_contiguous() or not quantized.is_cuda):
        raise ValueError("quantized must be a contiguous device tensor shaped and typed like z")
    idx = torch.empty(p, dtype=torch.int32, device=z.device)
    check(lib.ldx_vq_nearest4(_ptr(z), None, _ptr(codebook), _ptr(codebook_norm), p, e, _VQ_DTYPES[z.dtype],
                              _ptr(idx), _ptr(quantized), _stream()), "vq_nearest4")
    if quantized is not None:
        _wrote(quantized)
    return idx


# --------------------------------------------------------------- source-order arithmetic


def _ncdhw_strides(x: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(batch, channel, voxel) element strides of a logical NCDHW tensor whose voxels are
    evenly spaced: NCDHW-contiguous (voxel stride 1) or channels-last 3-D (voxel stride C)."""
    if x.dim() != 5:
        raise ValueError(f"{name} must be NCDHW (B, C, D, H, W), got shape {tuple(x.shape)}")
    _, _, d, h, w = x.shape
    st = x.stride()
    sv = st[4] if w > 1 else (st[3] // w if h > 1 else (st[2] // (h * w) if d > 1 else 1))
    if (w > 1 and st[4] != sv) or (h > 1 and st[3] != w * sv) or (d > 1 and st[2] != h * w * sv):
        raise ValueError(f"{name}: voxels must be evenly spaced (strides {st})")
    return int(st[0]), int(st[1]), int(sv)


def _like(x: torch.Tensor, shape: tuple[int, ...]) -> torch.Tensor:
    """An empty fp16 tensor of ``shape`` in ``x``'s memory format (NCDHW or channels-last)."""
    fmt = (torch.channels_last_3d if not x.is_contiguous() and x.is_contiguous(memory_format=torch.channels_last_3d)
           else torch.contiguous_format)
    return torch.empty(shape, dtype=torch.float16, device=x.device, memory_format=fmt)


def conv3d_half(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, *, padding: int,
                stride: int) -> torch.Tensor:
    """Source-order fp16 conv3d (conv3d_half, _source_half.py:327-384): four fp32 partial
    sums in Torch-CPU's channel-major order, bias added, one fp16 rounding -- Torch-CPU's
    result bit for bit. ``x`` is NCDHW ``(B, C, D, H, W)`` (contiguous or channels-last),
    ``weight`` ``(O, C, KD, KH, KW)``, ``bias`` ``(O,)`` or None, all fp16; returns
    ``(B, O, OD, OH, OW)`` in ``x``'s memory format."""
    _require_cuda(x, "x")
    _require_cuda(weight, "weight")
    xs = _ncdhw_strides(x, "conv3d input")
    if weight.dim() != 5:
        raise ValueError(f"weight must be (O, C, KD, KH, KW), got {tuple(weight.shape)}")
    b, c, d, h, w = x.shape
    o, wc, kd, kh, kw = weight.shape
    if wc != c:
        raise ValueError("conv3d input channels differ from source weights")
    if bias is not None:
        _require_cuda(bias, "bias")
        if tuple(bias.shape) != (o,):
            raise ValueError("conv3d bias must have one value per output channel")
        bias = bias.contiguous()
    ext = [(n + 2 * padding - k) // stride + 1 for n, k in zip((d, h, w), (kd, kh, kw))]
    if min(ext) < 1:
        raise ValueError("conv3d kernel exceeds the padded input")
    weight = weight.contiguous()
    y = _like(x, (b, o, *ext))
    ys = _ncdhw_strides(y, "y")
    a = SourceConvArgs(batch=b, in_c=c, in_d=d, in_h=h, in_w=w, out_c=o, kd=kd, kh=kh, kw=kw, stride=stride,
                       padding=padding, x=_ptr(x), x_batch_stride=xs[0], x_channel_stride=xs[1],
                       x_voxel_stride=xs[2], weight=_ptr(weight), bias=_ptr(bias), y=_ptr(y),
                       y_batch_stride=ys[0], y_channel_stride=ys[1], y_voxel_stride=ys[2])
    check(lib.ldx_conv3d_source_half(ctypes.byref(a), _stream()), "conv3d_source_half")
    fc = count_flops.active
    if fc is not None:
        fc.conv += 2.0 * b * o * c * kd * kh * kw * ext[0] * ext[1] * ext[2]
    return y


def group_norm_half(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, *, groups: int, eps: float,
                    return_affine: bool = False):
    """Source-order fp16 GroupNorm (group_norm_half, _source_half.py:387-544): Torch-CPU's
    chunked Welford cascade per group, then ``fp16(scale * x + offset)`` with the
    per-channel fp32 affine. ``x`` is NCDHW (contiguous or channels-last) fp16, ``weight``
    and ``bias`` fp16 ``(C,)``. Returns the normalized tensor in ``x``'s memory format, and
    with ``return_affine`` also the fp32 ``(B, C, 2)`` (scale, offset)."""
    _require_cuda(x, "x")
    xs = _ncdhw_strides(x, "group_norm input")
    b, c = x.shape[:2]
    if groups < 1 or c % groups:
        raise ValueError(f"group_norm channels {c} must be divisible by num_groups {groups}")
    for t, nm in ((weight, "weight"), (bias, "bias")):
        _require_cuda(t, nm)
        if tuple(t.shape) != (c,):
            raise ValueError("group_norm affine must have one value per channel")
    weight, bias = weight.contiguous(), bias.contiguous()
    voxels = int(x.shape[2] * x.shape[3] * x.shape[4])
    y = _like(x, tuple(x.shape))
    ys = _ncdhw_strides(y, "y")
    affine = torch.empty((b, c, 2), dtype=torch.float32, device=x.device)
    ws_bytes = lib.ldx_group_norm_source_workspace_bytes(b, c, voxels, groups)
    ws = torch.empty(max(int(ws_bytes), 1), dtype=torch.uint8, device=x.device)
    check(lib.ldx_group_norm_source_half(_ptr(x), xs[0], xs[1], xs[2], b, c, voxels, groups, _ptr(weight),
                                         _ptr(bias), float(eps), _ptr(affine), _ptr(y), ys[0], ys[1], ys[2],
                                         _ptr(ws), int(ws.numel()), _stream()), "group_norm_source_half")
    return (y, affine) if return_affine else y


# ------------------------------------------------------------------ 8-bit operators

# Small calls are bound by this host path too: each check below is one comparison on the way through, and
# the helpers that name what is wrong run only where one failed. One call over and over on the same tensors: a
# token's norm with residual and 8-bit rows 11.5 us of host time, three allocations and the launch 8 of them, a
# quantize8 8.9, dense8 8.9, cache8_append 9.2, cache8_attention 10.8. A program that calls between other work and
# builds its operands' Quantized8 or Cache8 each time pays 3 to 4 more (14.7, 12.4, 13.0 and 14.1).

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


@dataclass
class Quantized8:
    """8-bit rows: e4m3 ``codes`` (..., features rounded up to whole blocks of 128, zero codes past
    ``features``) and E8M0 ``scales`` (..., blocks rounded up to four), one per row and 128 columns; a
    value is its code times its block's power of two. Both contiguous. What ``quantize8`` and
    ``rms_norm(..., quantize=True)`` return and ``dense8`` takes on both sides (a weight is quantized
    once, ``quantize8(weight)`` of the Torch-layout ``(O, C)``)."""

    codes: torch.Tensor
    scales: torch.Tensor
    features: int

    @staticmethod
    def empty(lead: tuple[int, ...], features: int, like: torch.Tensor) -> "Quantized8":
        """Uninitialised rows on ``like``'s device."""
        kb = -(-features // BLOCK8)
        return Quantized8(like.new_empty((*lead, kb * BLOCK8), dtype=E4M3),
                          like.new_empty((*lead, -(-kb // 4) * 4), dtype=E8M0), features)

    @property
    def shape(self) -> tuple[int, ...]:
        return (*self.codes.shape[:-1], self.features)

    def float(self) -> torch.Tensor:
        """The values as fp32 (a test and debugging aid)."""
        kb = self.codes.shape[-1] // BLOCK8
        s = self.scales.float()[..., :kb, None]
        v = self.codes.float().unflatten(-1, (kb, BLOCK8)) * s
        return v.flatten(-2)[..., :self.features]


_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch8(fn, args: tuple, device: int, what: str) -> None:
    """One C call on the current stream of device ``device``, made current for it where it is not."""
    if device == _device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        check(rc, what)


_ELEM, _ALL = tuple(ELEM_DTYPES), tuple(ALL_DTYPES)
_MOST = 0x7fffffff   # what a size in the C structs holds (ctypes drops the bits above)


def _need(t: torch.Tensor, name: str, dtype: torch.dtype | tuple | None, device: int) -> None:
    """``t`` is a tensor of ``dtype`` (one of several, or any with None) on device ``device`` (any with -1)."""
    if type(t) is torch.Tensor and (t.dtype is dtype or dtype is None or dtype.__class__ is tuple and t.dtype in dtype) \
            and (t.get_device() == device if device >= 0 else t.is_cuda):
        return
    _require_cuda(t, name, dtype)
    if device >= 0 and t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t`` and the pitch of its rows (the last axis): rows evenly spaced, features contiguous (a copy is
    made of one that is not)."""
    f = t.shape[-1]
    if t.is_contiguous():
        return t, f
    t2 = t if t.dim() == 2 else t.reshape(-1, f)
    if f > 1 and t2.stride(1) != 1 or t2.shape[0] > 1 and t2.stride(0) < f:
        return t2.contiguous(), f
    return t2, (t2.stride(0) if t2.shape[0] > 1 else f)


def _rows_in_place(t: torch.Tensor, name: str) -> int:
    """Row pitch of an output, which has to be viewable as ``(rows, features)``."""
    f = int(t.shape[-1])
    if t.is_contiguous():
        return f
    try:
        t2 = t.view(-1, f)
    except RuntimeError:
        raise ValueError(f"{name}: rows must be evenly spaced") from None
    if f > 1 and t2.stride(1) != 1 or t2.shape[0] > 1 and t2.stride(0) < f:
        raise ValueError(f"{name}: features must be contiguous and rows must not overlap")
    return t2.stride(0) if t2.shape[0] > 1 else f


def _out_like(out: torch.Tensor | None, x: torch.Tensor, name: str) -> tuple[torch.Tensor, int]:
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format), x.shape[-1]
    _need(out, name, x.dtype, x.get_device())
    if out.shape != x.shape:
        raise ValueError(f"{name} shape {tuple(out.shape)} != {tuple(x.shape)}")
    return out, _rows_in_place(out, name)


def quantize8(x: torch.Tensor) -> Quantized8:
    """fp16, bf16 or fp32 ``x`` as 8-bit rows: per row and 128 columns the least power of two with which
    the largest magnitude does not pass 448, codes rounded to nearest even."""
    _need(x, "x", _ALL, -1)
    n = x.numel()
    if x.dim() < 1 or not n:
        raise ValueError(f"quantize8: shape {tuple(x.shape)} holds no rows")
    f = x.shape[-1]
    if f > _MOST:
        raise ValueError(f"quantize8: {f} features")
    x2, pitch = _rows(x)
    q = Quantized8.empty(x.shape[:-1], f, x)
    _launch8(lib.ldx_quantize8, (x2.data_ptr(), pitch, n // f, f, ALL_DTYPES[x.dtype], q.codes.data_ptr(),
                                 q.codes.shape[-1], q.scales.data_ptr(), q.scales.shape[-1]), x.get_device(), "quantize8")
    return q


def rms_norm(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
             quantize: bool = False, out: torch.Tensor | None = None, sum_out: torch.Tensor | None = None):
    """``s / sqrt(mean(s^2) + eps) * gamma`` over the last axis of fp16, bf16 or fp32 ``x``, ``s`` being
    ``x``, or ``x + residual`` rounded to that type. Returns the norm in ``x``'s type (into ``out`` when
    given, which may be ``x``), or as ``Quantized8`` rows with ``quantize``; with a ``residual`` the pair
    ``(norm, s)``, ``s`` into ``sum_out`` when given, which may be ``x`` or ``residual``. Squares are
    summed in fp32, at most 32 at a time, and those sums in fp64; ``eps`` is at least 1e-30. One launch."""
    _need(x, "x", _ALL, -1)
    n, dev, shape = x.numel(), x.get_device(), x.shape
    if not shape or not n:
        raise ValueError(f"rms_norm: shape {tuple(shape)} holds no rows")
    f = shape[-1]
    if f > _MOST:
        raise ValueError(f"rms_norm: {f} features")
    _need(gamma, "gamma", None, dev)
    if gamma.shape != (f,):
        raise ValueError(f"gamma shape {tuple(gamma.shape)} != ({f},)")
    if quantize and out is not None:
        raise ValueError("rms_norm: out and quantize exclude each other")
    if sum_out is not None and residual is None:
        raise ValueError("rms_norm: sum_out needs a residual")
    x2, xp = _rows(x)
    g32 = _f32(gamma)
    s, r2, rp, sp = None, None, 0, 0
    if residual is not None:
        _need(residual, "residual", x.dtype, dev)
        if residual.shape != shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != {tuple(shape)}")
        r2, rp = _rows(residual)
        s, sp = _out_like(sum_out, x, "sum_out")
    a = RmsNormArgs(n // f, f, ALL_DTYPES[x.dtype], x2.data_ptr(), xp, _ptr(r2), rp, _ptr(s), sp, g32.data_ptr(), eps)
    if quantize:
        y = Quantized8.empty(shape[:-1], f, x)
        a.codes, a.codes_pitch = y.codes.data_ptr(), y.codes.shape[-1]
        a.scales, a.scales_pitch = y.scales.data_ptr(), y.scales.shape[-1]
    else:
        y, a.y_pitch = _out_like(out, x, "out")
        a.y = y.data_ptr()
        if s is not None and a.y == a.sum:
            raise ValueError("rms_norm: out and sum_out are the same tensor")
    _launch8(lib.ldx_rms_norm, (ctypes.byref(a),), dev, "rms_norm")
    if out is not None:
        _wrote(out)
    if sum_out is not None:
        _wrote(sum_out)
    return y if residual is None else (y, s)


def _rows8(q: Quantized8, name: str, device: int) -> tuple[torch.Tensor, torch.Tensor, int, int, tuple]:
    """Checks one operand of ``dense8``: its codes and scales, their pitches, and its leading axes."""
    if not isinstance(q, Quantized8):
        raise ValueError(f"{name} must be Quantized8 rows")
    codes, scales, f = q.codes, q.scales, q.features
    if not (type(codes) is type(scales) is torch.Tensor and codes.dtype is E4M3 and scales.dtype is E8M0
            and codes.get_device() == scales.get_device() >= 0 and (device < 0 or codes.get_device() == device)):
        _need(codes, f"{name} codes", E4M3, device)
        _need(scales, f"{name} scales", E8M0, codes.get_device())
    kb = -(-f // BLOCK8)
    cp, sp = kb * BLOCK8, -(-kb // 4) * 4
    cs = codes.shape
    lead = cs[:-1]
    if f < 1 or not cs or cs[-1] != cp or scales.shape != (*lead, sp):
        raise ValueError(f"{name}: codes {tuple(cs)} and scales {tuple(scales.shape)} do not hold rows of {f} features")
    if not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{name}: codes and scales must be contiguous")
    return codes, scales, cp, sp, lead


_ACTS = {None: ACT_NONE, "gelu": ACT_GELU, "silu": ACT_SILU}


def dense8(x: Quantized8, weight: Quantized8, bias: torch.Tensor | None = None, *,
           residual: torch.Tensor | None = None, act: str | None = None, out: torch.Tensor | None = None,
           dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """``act(x @ weight^T + bias + residual)`` of 8-bit rows ``x`` (..., C) and an 8-bit weight (O, C),
    fp32 sums and one rounding to ``dtype`` (fp16, bf16 or fp32; ``residual`` and ``out`` share it).
    ``act`` is None, ``"gelu"`` or ``"silu"``. fp16 and bf16 results come from the e4m3 matrix
    instruction, whose sums are within 2^-10 of the terms' magnitudes (about 1.5e-5 of the result for
    ordinary data); fp32 results are summed to fp32 accuracy at half its rate: round those where a 16-bit
    result has to have it, too."""
    xc, xs, xp, xsp, lead = _rows8(x, "x", -1)
    dev = xc.get_device()
    wc, ws, wp, wsp, outs = _rows8(weight, "weight", dev)
    if len(outs) != 1:
        raise ValueError(f"weight must be (O, C) rows, got {weight.shape}")
    m, o = math.prod(lead), outs[0]
    if x.features != weight.features:
        raise ValueError(f"weight expects {weight.features} features, got {x.features}")
    if dtype not in ALL_DTYPES:
        raise ValueError(f"dtype must be fp16, bf16 or fp32, not {dtype}")
    if act not in _ACTS:
        raise ValueError(f"act must be None, 'gelu' or 'silu', not {act!r}")
    if not m or not o:
        raise ValueError(f"dense8: {m} rows and {o} outputs")
    shape = (*lead, o)
    if bias is not None:
        _need(bias, "bias", None, dev)
        if bias.shape != (o,):
            raise ValueError(f"bias shape {tuple(bias.shape)} != ({o},)")
        bias = _f32(bias)
    given = out is not None
    if given:
        _need(out, "out", dtype, dev)
        if out.shape != shape:
            raise ValueError(f"out shape {tuple(out.shape)} != {shape}")
        yp = _rows_in_place(out, "out")
    else:
        out, yp = xc.new_empty(shape, dtype=dtype), o
    r2, rp = None, 0
    if residual is not None:
        _need(residual, "residual", dtype, dev)
        if residual.shape != shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != {shape}")
        r2, rp = _rows(residual)
    a = Dense8Args(m, x.features, o, xc.data_ptr(), xp, xs.data_ptr(), xsp, wc.data_ptr(), wp, ws.data_ptr(), wsp,
                   _ptr(bias), _ptr(r2), rp, _ACTS[act], ALL_DTYPES[dtype], out.data_ptr(), yp)
    if count_flops.active is not None:
        count_flops.active.dense += 2.0 * m * o * x.features
    _launch8(lib.ldx_dense8, (ctypes.byref(a),), dev, "dense8")
    if given:
        _wrote(out)
    return out


@dataclass
class Cache8:
    """Keys and values in 8 bits, in pages of 64 tokens: e4m3 codes ``k`` (pages, heads, 64, D) and ``v``
    (pages, heads, D, 64) and E8M0 scales ``k_scales``, ``v_scales`` (pages, heads), all contiguous. Pages
    belong to no sequence by themselves: an int32 ``table`` (batch, pages per sequence) says which hold
    a sequence's tokens, in order."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    @staticmethod
    def empty(pages: int, heads: int, head_dim: int, device: torch.device | str = "cuda") -> "Cache8":
        """A cache of zero codes."""
        codes = [torch.zeros(s, dtype=torch.uint8, device=device).view(E4M3)
                 for s in ((pages, heads, PAGE8, head_dim), (pages, heads, head_dim, PAGE8))]
        scales = [torch.full((pages, heads), 127, dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)]
        return Cache8(*codes, *scales)


def _cache_block(cache: Cache8, what: str) -> tuple[Cache8Block, int]:
    """The C view of a cache and its device."""
    if not isinstance(cache, Cache8):
        raise ValueError(f"{what}: cache must be a Cache8")
    k, v, ks, vs = cache.k, cache.v, cache.k_scales, cache.v_scales
    if not (type(k) is type(v) is type(ks) is type(vs) is torch.Tensor and k.dtype is v.dtype is E4M3
            and ks.dtype is vs.dtype is E8M0 and k.get_device() == v.get_device() == ks.get_device() == vs.get_device() >= 0):
        _need(k, "cache k", E4M3, -1)
        _need(v, "cache v", E4M3, k.get_device())
        _need(ks, "cache k_scales", E8M0, k.get_device())
        _need(vs, "cache v_scales", E8M0, k.get_device())
    dev, shape = k.get_device(), k.shape
    if len(shape) != 4 or shape[2] != PAGE8:
        raise ValueError(f"cache k must be (pages, heads, {PAGE8}, D), got {tuple(shape)}")
    pages, heads, _, d = shape
    if v.shape != (pages, heads, d, PAGE8) or ks.shape != (pages, heads) or vs.shape != (pages, heads):
        raise ValueError(f"cache v {tuple(v.shape)} or scales {tuple(ks.shape)}, {tuple(vs.shape)} do not fit k "
                         f"{tuple(shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    return Cache8Block(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, d), dev


def _cache_ints(t: torch.Tensor, name: str, batch: int, device: int) -> int:
    """Pointer of ``batch`` int32 values on the device."""
    _need(t, name, torch.int32, device)
    if t.shape != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 ({batch},), got {tuple(t.shape)}")
    return t.data_ptr()


def _cache_table(table: torch.Tensor, batch: int, device: int) -> tuple[int, int, int]:
    """``(pointer, pitch, width)`` of a page table (a column range of a wider one is fine)."""
    _need(table, "table", torch.int32, device)
    shape = table.shape
    if len(shape) != 2 or shape[0] != batch or not shape[1] or (shape[1] > 1 and table.stride(1) != 1) \
            or (batch > 1 and table.stride(0) < shape[1]):
        raise ValueError(f"table must be int32 ({batch}, pages) with contiguous rows, got {tuple(shape)}")
    if shape[1] > _MOST:
        raise ValueError(f"table of {shape[1]} pages a sequence")
    return table.data_ptr(), (table.stride(0) if batch > 1 else shape[1]), shape[1]


def _head_strides(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(batch, token, head) strides of a ``(B, H, L, D)`` tensor with contiguous channels."""
    b, h, l, d = t.stride()
    if d != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")
    return b, l, h


def _distinct(t: torch.Tensor, name: str) -> None:
    """No two values of ``t`` stand in one place (sizes within strides, from the innermost axis out)."""
    span = 1
    for stride, size in sorted((stride, size) for stride, size in zip(t.stride(), t.shape) if size > 1):
        if stride < span:
            raise ValueError(f"{name} of strides {t.stride()} overlaps itself")
        span = stride * size


def cache8_append(cache: Cache8, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, *,
                  counts: torch.Tensor | None = None) -> None:
    """Write ``k``, ``v`` (B, heads, L, D; fp16, bf16 or fp32, any strides with contiguous channels) into
    ``cache`` at positions ``starts[b] ..`` of each sequence: its first ``counts[b]`` tokens (all ``L``
    without). Each page of 64 tokens has one power of two for a head's keys and one for its values; it
    rises with the largest token written, and older codes of the page are then rounded to it. Tokens
    past the table's width, of a negative start or in a page that the cache does not have are left out;
    a page that is written stands once in the table. ``table``, ``starts`` and ``counts`` are int32 on the
    device, so a captured graph appends where they say at each replay."""
    block, dev = _cache_block(cache, "cache8_append")
    _need(k, "k", _ALL, dev)
    _need(v, "v", k.dtype, dev)
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[1] != block.heads or shape[3] != block.head_dim or not shape[0] \
            or not shape[2]:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} must be (B, {block.heads}, L, {block.head_dim})")
    b, _, n, _ = shape
    if b > _MOST or n > _MOST:
        raise ValueError(f"cache8_append: {b} x {n} tokens")
    a = Cache8AppendArgs(block, b, n, k.data_ptr(), _head_strides(k, "k"), v.data_ptr(), _head_strides(v, "v"),
                         ALL_DTYPES[k.dtype], *_cache_table(table, b, dev), _cache_ints(starts, "starts", b, dev),
                         None if counts is None else _cache_ints(counts, "counts", b, dev))
    _launch8(lib.ldx_cache8_append, (ctypes.byref(a),), dev, "cache8_append")
    if not cache.k.is_inference():
        increment_version((cache.k, cache.v, cache.k_scales, cache.v_scales))


def cache8_attention(q: torch.Tensor, cache: Cache8, table: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                     starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` over the first ``lengths[b]`` tokens that ``cache`` holds of each
    sequence. ``q`` is fp16 or bf16 ``(B, heads, L, D)``, its heads a multiple of the cache's (query head
    ``j`` reads the cache's head ``j // group``). With ``starts`` query ``i`` sees tokens up to position
    ``starts[b] + i`` (causal); without, all ``lengths[b]``. A query that sees no token gives 0; tokens that
    it does not see, and pages behind the length, do not touch its result. A page that the cache does
    not have, or a length past the table, gives NaN. Scores, softmax and sums are fp32; probabilities are
    rounded to fp16 (2^-11 of each, those below 2^-21 of a query's largest to 2^-32 of it). Returns
    ``(B, heads, L, D)`` in ``q``'s type (into ``out`` when given, which may be ``q``); ``table``,
    ``lengths`` and ``starts`` are int32 on the device."""
    block, dev = _cache_block(cache, "cache8_attention")
    _need(q, "q", _ELEM, dev)
    shape = q.shape
    if len(shape) != 4 or shape[3] != block.head_dim or shape[1] % block.heads or not q.numel():
        raise ValueError(f"q {tuple(shape)} must be (B, a multiple of {block.heads}, L, {block.head_dim})")
    b, hq, lq, _ = shape
    if b > _MOST or hq > _MOST or lq > _MOST:
        raise ValueError(f"cache8_attention: {b} x {hq} x {lq} queries")
    given = out is not None
    if given:
        _need(out, "out", q.dtype, dev)
        if out.shape != shape:
            raise ValueError(f"out shape {tuple(out.shape)} != {tuple(shape)}")
        if not out.is_contiguous():
            _distinct(out, "out")
    else:
        out = q.new_empty(shape)
    a = Cache8AttentionArgs(block, b, hq, lq, q.data_ptr(), _head_strides(q, "q"), out.data_ptr(),
                            _head_strides(out, "out"), ALL_DTYPES[q.dtype], scale, *_cache_table(table, b, dev),
                            _cache_ints(lengths, "lengths", b, dev),
                            None if starts is None else _cache_ints(starts, "starts", b, dev))
    ref = ctypes.byref(a)
    ws_bytes = lib.ldx_cache8_attention_workspace_bytes(ref)
    if ws_bytes:
        ws = q.new_empty(ws_bytes, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws_bytes
    _launch8(lib.ldx_cache8_attention, (ref,), dev, "cache8_attention")
    if given:
        _wrote(out)
    return out


# ------------------------------------------------------------------ rotation of heads, 4-bit cache

@dataclass
class Rotary:
    """The plan of a position rotation: ``axes`` are the widths (even) of a head's sections, one for each
    axis of positions, in order; what a head has behind them is not turned. ``turns`` (fp64, on the device)
    holds every pair's full turns per position, the sections' one after another. Pair ``i`` of a section of
    ``w`` channels is its channels ``(i, i + w / 2)``, or ``(2 i, 2 i + 1)`` where ``interleaved``."""

    turns: torch.Tensor
    axes: tuple[int, ...]
    interleaved: bool = False

    @staticmethod
    def make(axes: tuple[int, ...] | int, *, theta: float = 10000.0, interleaved: bool = False,
             scale: float | tuple[float, ...] = 1.0, device: torch.device | str = "cuda") -> "Rotary":
        """The usual frequencies, ``theta^(-2 i / w)`` for pair ``i`` of an axis of ``w`` channels, times ``scale``
        (of every axis, or one each: positions of a finer or coarser grid than the model's)."""
        axes = (axes,) if isinstance(axes, int) else tuple(axes)
        scales = tuple(scale) if isinstance(scale, (tuple, list)) else (scale,) * len(axes)
        if not axes or len(scales) != len(axes) or any(w < 2 or w % 2 for w in axes):
            raise ValueError(f"Rotary: axes {axes} must be even widths, with a scale each, got {scales}")
        if not theta > 0:
            raise ValueError(f"Rotary: theta {theta} must be above 0")
        turns = [s * theta ** (-2.0 * i / w) / (2 * math.pi) for w, s in zip(axes, scales) for i in range(w // 2)]
        return Rotary(torch.tensor(turns, dtype=torch.float64, device=device), axes, interleaved)


def _head_gamma(gamma: torch.Tensor, name: str, d: int, device: int) -> torch.Tensor:
    """A head's ``d`` factors as contiguous fp32."""
    _need(gamma, name, None, device)
    if gamma.shape != (d,):
        raise ValueError(f"{name} shape {tuple(gamma.shape)} != ({d},)")
    return _f32(gamma)


def _heads_out(out: torch.Tensor | None, x: torch.Tensor, name: str) -> torch.Tensor:
    """``out``, checked, or a new (B, H, L, D) tensor whose tokens hold their heads side by side."""
    if out is None:
        b, h, l, d = x.shape
        return x.new_empty_strided((b, h, l, d), (l * h * d, d, h * d, 1))
    _need(out, name, x.dtype, x.get_device())
    if out.shape != x.shape:
        raise ValueError(f"{name} shape {tuple(out.shape)} != {tuple(x.shape)}")
    if not out.is_contiguous():
        _distinct(out, name)
    return out


_rotate_heads_args = filler(RotateHeadsArgs)
_NO_KEYS, _NO_AXES = (0,) * 8, (0,) * ROTARY_AXES


def _in_place(out: torch.Tensor, x: torch.Tensor, name: str) -> None:
    """An output that begins where its input does is that input, value for value."""
    if out.data_ptr() == x.data_ptr() and any(n > 1 and s != t for n, s, t in zip(x.shape, out.stride(), x.stride())):
        raise ValueError(f"{name} stands in its input's place with strides {out.stride()}, not {x.stride()}")


def rotate_heads(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: Rotary, *,
                 q_gamma: torch.Tensor | None = None, k_gamma: torch.Tensor | None = None, eps: float = 1e-6,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Queries and keys before an attention, in one launch: each head divided by its root mean square and
    times ``q_gamma`` / ``k_gamma`` (D,) where given, then turned by its token's position. ``q`` (B, H, L, D)
    and ``k`` (B, H', L, D; or None) are fp16, bf16 or fp32, any strides with contiguous channels (slices of one
    projection, say); D is even and at most 512. ``positions`` is int32 on the device, (B, L) for one axis,
    (axes, B, L) for several (a volume's depth, height and width), any strides, so that one row expanded serves
    the batch; ``rotary`` says how an axis turns (at most four). Angles are reduced in fp64: position 10^9
    has its own. Norm and rotation are fp32, rounded once. Returns ``(q, k)``, or ``q`` without keys, in the
    inputs' type: into ``q_out`` and ``k_out`` when given, each of which may be its own input and overlaps nothing else of the
    call, else with a token's heads side by side in memory (``(B, L, H * D)`` is a view)."""
    _need(q, "q", _ALL, -1)
    dev, shape, dtype = q.get_device(), q.shape, q.dtype
    if len(shape) != 4 or not q.numel():
        raise ValueError(f"q {tuple(shape)} must be (B, heads, L, D)")
    b, h, l, d = shape
    if not isinstance(rotary, Rotary):
        raise ValueError("rotate_heads: rotary must be a Rotary")
    turns, axes = rotary.turns, rotary.axes
    n, turned = len(axes), sum(axes)
    _need(turns, "rotary turns", torch.float64, dev)
    if not 1 <= n <= ROTARY_AXES or turned > d or turns.shape != (turned // 2,) or not turns.is_contiguous():
        raise ValueError(f"rotary: axes {axes} (at most {ROTARY_AXES}) with {tuple(turns.shape)} turns do not fit heads of {d}")
    _need(positions, "positions", torch.int32, dev)
    ps, at = positions.shape, positions.stride()
    if n == 1 and ps == (b, l):
        at = (0, *at)
    elif ps != (n, b, l):
        raise ValueError(f"positions {tuple(ps)} must be ({n}, {b}, {l})")
    if b > _MOST or h > _MOST or l > _MOST:
        raise ValueError(f"rotate_heads: {b} x {h} x {l} heads")
    if q_gamma is not None:
        q_gamma = _head_gamma(q_gamma, "q_gamma", d, dev)
    if k_gamma is not None:
        k_gamma = _head_gamma(k_gamma, "k_gamma", d, dev)
    qo = _heads_out(q_out, q, "q_out")
    if q_out is not None:
        _in_place(qo, q, "q_out")
    ko, kh, keys = None, 0, _NO_KEYS
    if k is None:
        if k_out is not None or k_gamma is not None:
            raise ValueError("rotate_heads: k_out and k_gamma need keys")
    else:
        _need(k, "k", dtype, dev)
        kshape = k.shape
        if len(kshape) != 4 or kshape[0] != b or kshape[2] != l or kshape[3] != d or not 0 < kshape[1] <= _MOST:
            raise ValueError(f"k {tuple(kshape)} does not fit q {tuple(shape)}")
        ko, kh = _heads_out(k_out, k, "k_out"), kshape[1]
        if k_out is not None:
            _in_place(ko, k, "k_out")
        at_q, at_k = qo.data_ptr(), ko.data_ptr()
        if at_k == at_q:
            raise ValueError("rotate_heads: q_out and k_out are the same tensor")
        if at_q == k.data_ptr() or at_k == q.data_ptr():
            raise ValueError("rotate_heads: an output may be its own input, not the other")
        keys = (k.data_ptr(), *_head_strides(k, "k"), at_k, *_head_strides(ko, "k_out"))
    a = _rotate_heads_args(b, l, h, kh, d, ALL_DTYPES[dtype], q.data_ptr(), *_head_strides(q, "q"), qo.data_ptr(),
                           *_head_strides(qo, "q_out"), *keys, 0 if q_gamma is None else q_gamma.data_ptr(),
                           0 if k_gamma is None else k_gamma.data_ptr(), eps, n, *axes, *_NO_AXES[n:],
                           rotary.interleaved, positions.data_ptr(), *at, turns.data_ptr())
    _launch8(lib.ldx_rotate_heads, (ctypes.byref(a),), dev, "rotate_heads")
    if q_out is not None:
        _wrote(q_out)
    if k_out is not None:
        _wrote(k_out)
    return qo if k is None else (qo, ko)


@dataclass
class Cache4:
    """Keys and values in 4 bits, in pages of 64 tokens: e2m1 codes ``k`` and ``v`` (pages, heads, 64, D / 2; uint8, two
    channels in a byte, the even one in its lower half) and E8M0 scales ``k_scales``, ``v_scales`` (pages, heads, D /
    32, 64), one for each 32 channels of a token, all contiguous: 17 bytes for 32 values. Pages belong to no
    sequence by themselves: an int32 ``table`` (batch, pages per sequence) says which hold a sequence's tokens, in
    order."""

    k: torch.Tensor
    v: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor

    @staticmethod
    def empty(pages: int, heads: int, head_dim: int, device: torch.device | str = "cuda") -> "Cache4":
        """A cache of zeros."""
        codes = [torch.zeros((pages, heads, PAGE4, head_dim // 2), dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.full((pages, heads, head_dim // BLOCK4, PAGE4), 127, dtype=torch.uint8, device=device).view(E8M0)
                  for _ in range(2)]
        return Cache4(*codes, *scales)


_cache4_append_args, _cache4_read_args = filler(Cache4AppendArgs), filler(Cache4ReadArgs)
_cache4_attention_args = filler(Cache4AttentionArgs)


def _cache4_block(cache: Cache4, what: str) -> tuple[tuple[int, ...], int]:
    """What the C view of a cache holds (its pointers, pages, heads and head width), and its device."""
    if not isinstance(cache, Cache4):
        raise ValueError(f"{what}: cache must be a Cache4")
    k, v, ks, vs = cache.k, cache.v, cache.k_scales, cache.v_scales
    if not (type(k) is type(v) is type(ks) is type(vs) is torch.Tensor and k.dtype is v.dtype is torch.uint8
            and ks.dtype is vs.dtype is E8M0 and k.get_device() == v.get_device() == ks.get_device() == vs.get_device() >= 0):
        _need(k, "cache k", torch.uint8, -1)
        _need(v, "cache v", torch.uint8, k.get_device())
        _need(ks, "cache k_scales", E8M0, k.get_device())
        _need(vs, "cache v_scales", E8M0, k.get_device())
    dev, shape = k.get_device(), k.shape
    if len(shape) != 4 or shape[2] != PAGE4:
        raise ValueError(f"cache k must be (pages, heads, {PAGE4}, D / 2), got {tuple(shape)}")
    pages, heads, _, half = shape
    each = (pages, heads, half // (BLOCK4 // 2), PAGE4)
    if v.shape != shape or ks.shape != each or vs.shape != each:
        raise ValueError(f"cache v {tuple(v.shape)} or scales {tuple(ks.shape)}, {tuple(vs.shape)} do not fit k "
                         f"{tuple(shape)}")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError("cache tensors must be contiguous")
    if not 0 < pages <= _MOST or not 0 < heads <= _MOST:
        raise ValueError(f"{what}: {pages} pages of {heads} heads")
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pages, heads, 2 * half), dev


def cache4_append(cache: Cache4, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, *,
                  counts: torch.Tensor | None = None) -> None:
    """Write ``k``, ``v`` (B, heads, L, D; fp16, bf16 or fp32, any strides with contiguous channels) into
    ``cache`` at positions ``starts[b] ..`` of each sequence: its first ``counts[b]`` tokens (all ``L``
    without). Each 32 channels of a token get the least power of two (up to 2^125) with which their largest
    magnitude does not pass 6, and codes rounded to nearest even; 32 channels with a NaN or an infinity among them
    become NaN. No other token changes. Tokens past the table's width, of a negative start or in a page that the
    cache does not have are left out; no token is written by two sequences. ``table``, ``starts`` and ``counts``
    are int32 on the device, so a captured graph appends where they say at each replay."""
    block, dev = _cache4_block(cache, "cache4_append")
    heads, d = block[5:]
    _need(k, "k", _ALL, dev)
    _need(v, "v", k.dtype, dev)
    shape = k.shape
    if len(shape) != 4 or shape != v.shape or shape[1] != heads or shape[3] != d or not shape[0] \
            or not shape[2]:
        raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} must be (B, {heads}, L, {d})")
    b, _, n, _ = shape
    if b > _MOST or n > _MOST:
        raise ValueError(f"cache4_append: {b} x {n} tokens")
    a = _cache4_append_args(*block, b, n, k.data_ptr(), *_head_strides(k, "k"), v.data_ptr(), *_head_strides(v, "v"),
                            ALL_DTYPES[k.dtype], *_cache_table(table, b, dev), _cache_ints(starts, "starts", b, dev),
                            0 if counts is None else _cache_ints(counts, "counts", b, dev))
    _launch8(lib.ldx_cache4_append, (ctypes.byref(a),), dev, "cache4_append")
    if not cache.k.is_inference():
        increment_version((cache.k, cache.v, cache.k_scales, cache.v_scales))


def cache4_read(cache: Cache4, table: torch.Tensor, lengths: torch.Tensor, tokens: int, *,
                starts: torch.Tensor | None = None, dtype: torch.dtype = torch.float16,
                out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """What ``cache`` holds of ``tokens`` tokens of each sequence, from ``starts[b]`` on (from its first one without):
    ``(k, v)``, (B, heads, tokens, D) each, in ``dtype`` (fp16, bf16 or fp32; rounded to it). Rows from ``lengths[b]``
    on, and before token 0, are zeros; with ``out``, a pair of that type and shape (any strides with contiguous
    channels), they are left as they were. A page that the cache does not have, or a token past the table, gives
    NaN. ``table``, ``lengths`` and ``starts`` are int32 on the device."""
    block, dev = _cache4_block(cache, "cache4_read")
    heads, d = block[5:]
    if dtype not in ALL_DTYPES:
        raise ValueError(f"dtype must be fp16, bf16 or fp32, not {dtype}")
    if not isinstance(tokens, int) or not 0 < tokens <= _MOST:
        raise ValueError(f"cache4_read: {tokens} tokens")
    b = lengths.shape[0] if isinstance(lengths, torch.Tensor) and lengths.dim() == 1 else 0
    if not 0 < b <= _MOST:
        raise ValueError("lengths must be int32 (B,)")
    shape = (b, heads, tokens, d)
    if out is None:
        k, v = (cache.k.new_empty(shape, dtype=dtype) for _ in range(2))
    else:
        k, v = out
        for t, name in ((k, "out k"), (v, "out v")):
            _need(t, name, dtype, dev)
            if t.shape != shape:
                raise ValueError(f"{name} shape {tuple(t.shape)} != {shape}")
            if not t.is_contiguous():
                _distinct(t, name)
        if k.data_ptr() == v.data_ptr():
            raise ValueError("cache4_read: out's k and v are the same tensor")
    a = _cache4_read_args(*block, b, tokens, k.data_ptr(), *_head_strides(k, "out k"), v.data_ptr(),
                          *_head_strides(v, "out v"), ALL_DTYPES[dtype], *_cache_table(table, b, dev),
                          _cache_ints(lengths, "lengths", b, dev),
                          0 if starts is None else _cache_ints(starts, "starts", b, dev), out is None)
    _launch8(lib.ldx_cache4_read, (ctypes.byref(a),), dev, "cache4_read")
    if out is not None:
        _wrote(k)
        _wrote(v)
    return k, v


def cache4_attention(q: torch.Tensor, cache: Cache4, table: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                     starts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` over the first ``lengths[b]`` tokens that ``cache`` holds of each
    sequence. ``q`` is fp16 or bf16 ``(B, heads, L, D)``, its heads a multiple of the cache's (query head
    ``j`` reads the cache's head ``j // group``). With ``starts`` query ``i`` sees tokens up to position
    ``starts[b] + i`` (causal); without, all ``lengths[b]``. A query that sees no token gives 0; tokens that
    it does not see, and pages behind the length, do not touch its result. A page that the cache does
    not have, or a length past the table, gives NaN. Scores, softmax and sums are fp32; probabilities are
    rounded to 16 bits, or to fp16 (2^-11 of each, those below 2^-21 of a query's largest to 2^-32 of it) where
    many queries share pages. Returns ``(B, heads, L, D)`` in ``q``'s type (into ``out`` when given, which may be
    ``q``); ``table``, ``lengths`` and ``starts`` are int32 on the device."""
    block, dev = _cache4_block(cache, "cache4_attention")
    heads, d = block[5:]
    _need(q, "q", _ELEM, dev)
    shape = q.shape
    if len(shape) != 4 or shape[3] != d or shape[1] % heads or not q.numel():
        raise ValueError(f"q {tuple(shape)} must be (B, a multiple of {heads}, L, {d})")
    b, hq, lq, _ = shape
    if b > _MOST or hq > _MOST or lq > _MOST:
        raise ValueError(f"cache4_attention: {b} x {hq} x {lq} queries")
    given = out is not None
    if given:
        _need(out, "out", q.dtype, dev)
        if out.shape != shape:
            raise ValueError(f"out shape {tuple(out.shape)} != {tuple(shape)}")
        if not out.is_contiguous():
            _distinct(out, "out")
        _in_place(out, q, "out")
    else:
        out = q.new_empty(shape)
    a = _cache4_attention_args(*block, b, hq, lq, q.data_ptr(), *_head_strides(q, "q"), out.data_ptr(),
                               *_head_strides(out, "out"), ALL_DTYPES[q.dtype], scale, *_cache_table(table, b, dev),
                               _cache_ints(lengths, "lengths", b, dev),
                               0 if starts is None else _cache_ints(starts, "starts", b, dev), 0, 0)
    ref = ctypes.byref(a)
    ws_bytes = lib.ldx_cache4_attention_workspace_bytes(ref)
    if ws_bytes:
        ws = q.new_empty(ws_bytes, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws_bytes
    _launch8(lib.ldx_cache4_attention, (ref,), dev, "cache4_attention")
    if given:
        _wrote(out)
    return out
